"""Rotary positions without a GPU: frequencies, refusals, the C entry's checks."""
import ctypes
import math

import numpy as np
import pytest
import torch


def test_frequencies_and_scalings():
    import poly_attention_b200 as P
    inv, m = P.rotary_frequencies(64)
    want = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    # one rounding to fp32
    np.testing.assert_allclose(inv.numpy().astype(np.float64), want, rtol=2.0 ** -24)
    assert m == 1.0
    lin, m = P.rotary_frequencies(64, scaling="linear", factor=4.0)
    np.testing.assert_allclose(lin.numpy().astype(np.float64), want / 4, rtol=2.0 ** -24)
    assert m == 1.0
    ntk, m = P.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and m == 1.0
    # the slowest frequency is stretched by the whole factor
    assert abs(float(ntk[-1]) / (want[-1] / 4) - 1) < 1e-6
    yarn, m = P.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=2048)
    turns = 2048 * want / (2 * math.pi)
    got = yarn.numpy()
    assert np.all(got[turns >= 32] == want[turns >= 32].astype(np.float32))
    assert np.all(got[turns <= 1] == (want[turns <= 1] / 4).astype(np.float32))
    assert abs(m - (0.1 * math.log(4) + 1)) < 1e-12


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, scaling="yarn"),
                                dict(dim=8, factor=0.5), dict(dim=8, theta=-1.0),
                                dict(dim=8, scaling="yarn", original_length=64, fast_turns=1.0)])
def test_frequency_refusals(kw):
    import poly_attention_b200 as P
    with pytest.raises(ValueError):
        P.rotary_frequencies(kw.pop("dim"), **kw)


def test_cpu_tensors_are_refused():
    import poly_attention_b200 as P
    inv, _ = P.rotary_frequencies(8)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.apply_rotary(torch.randn(1, 2, 3, 8), inv)
    assert P.apply_rotary([], inv) == []
    with pytest.raises(ValueError, match=r"\[b, h, n, d\]"):
        P.apply_rotary(torch.randn(3, 8), inv)


def test_c_entry_checks_before_launching():
    from poly_attention_b200 import _lib
    lib, err = _lib.lib, lambda: _lib.lib.poly_last_error().decode()
    assert lib.poly_sizeof_rotary_args() == ctypes.sizeof(_lib.PolyRotaryArgs)
    assert lib.poly_rotary(None, None) == _lib.POLY_EINVAL

    def args(**kw):
        a = _lib.PolyRotaryArgs()
        a.batch, a.rows, a.dim, a.rot, a.n, a.factor, a.inv_freq = 1, 4, 64, 64, 1, 1.0, 256
        a.t[0].src, a.t[0].dst, a.t[0].heads = 256, 512, 2
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, word in ((dict(n=9), "n must"), (dict(n=-1), "n must"), (dict(dim=300), "dim"), (dict(rot=63), "rot"),
                     (dict(rot=66), "rot"), (dict(rot=0), "rot"), (dict(dtype=9), "dtype"), (dict(inv_freq=None), "either"),
                     (dict(angles=256), "either"), (dict(positions=256, cu_seqlens=256, seqs=1), "exclude"),
                     (dict(cu_seqlens=256, seqs=0), "cu_seqlens"), (dict(cu_seqlens=256, seqs=2, batch=2), "cu_seqlens")):
        assert lib.poly_rotary(args(**kw), None) == _lib.POLY_EINVAL, kw
        assert word in err(), (kw, err())
    bad = args()
    bad.t[0].dst = None
    assert lib.poly_rotary(bad, None) == _lib.POLY_EINVAL
    # nothing to do: no launch
    assert lib.poly_rotary(args(rows=0), None) == _lib.POLY_OK
    assert lib.poly_rotary(args(n=0), None) == _lib.POLY_OK


def test_embedding_keeps_fp32_frequencies():
    import poly_attention_b200 as P
    attn = P.PolyAttention(dim=32, heads=2, dim_head=16, use_rotary_embed=True)
    want = attn.rotary_emb.freqs.clone()
    assert "rotary_emb.freqs" in attn.state_dict() and not attn.rotary_emb.freqs.requires_grad
    attn = attn.bfloat16().half().double().float()
    assert attn.rotary_emb.freqs.dtype == torch.float32 and torch.equal(attn.rotary_emb.freqs, want)


def test_frequencies_of_an_unfrozen_module_stay_constants():
    import poly_attention_b200 as P
    attn = P.PolyAttention(dim=32, heads=2, dim_head=16, use_rotary_embed=True)
    attn.requires_grad_(False).requires_grad_(True)
    assert not attn.rotary_emb.freqs.requires_grad and all(p.requires_grad for p in attn.parameters())
    other = P.PolyAttention(dim=32, heads=2, dim_head=16, use_rotary_embed=True)
    with torch.no_grad():
        other.rotary_emb.freqs.zero_()
    other.load_state_dict(attn.state_dict())
    assert torch.equal(other.rotary_emb.freqs, attn.rotary_emb.freqs)
