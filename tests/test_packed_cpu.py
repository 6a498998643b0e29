"""Packed passes without a GPU: offsets, refusals, the C entries' checks, the slot numbering."""
import ctypes
import random

import pytest
import torch


def test_offsets():
    import poly_attention_b200 as P
    cu, longest = P.packed_offsets([3, 0, 5], device="cpu")
    assert cu.tolist() == [0, 3, 3, 8] and cu.dtype == torch.int32 and longest == 5
    assert P.packed_offsets([], device="cpu")[0].tolist() == [0]
    with pytest.raises(ValueError):
        P.packed_offsets([3, -1], device="cpu")


def test_cpu_tensors_are_refused():
    import poly_attention_b200 as P
    t = torch.randn(8, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.pass_fwd_packed(t, t, t, torch.tensor([0, 8], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.poly_attention_order2_packed(t, t, t, t, torch.tensor([0, 8], dtype=torch.int32))
    attn = P.PolyAttention(dim=16, heads=2, dim_head=8)
    with pytest.raises(ValueError, match="packed"):
        attn(torch.randn(2, 4, 16), cu_seqlens=torch.tensor([0, 4]))


def test_dual_tensors_are_refused():
    """A forward-mode tangent would be lost: the refusal comes before the one of CPU tensors."""
    import torch.autograd.forward_ad as fw

    import poly_attention_b200 as P
    cu = torch.tensor([0, 8], dtype=torch.int32)
    t, inv = torch.randn(8, 2, 64), P.rotary_frequencies(64)[0]
    with fw.dual_level():
        d = fw.make_dual(t, torch.ones_like(t))
        for call in (lambda: P.poly_attention_order2_packed(d, t, t, t, cu),
                     lambda: P.poly_attention_chain_packed([t, t, t], [t, t, t], [t, d], cu),
                     lambda: P.pass_fwd_packed(t, t, d, cu),
                     lambda: P.pass_bwd_packed(t, t, t, cu, t, torch.zeros(2, 8), d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA"):       # a plain tensor inside the level is not refused
            P.pass_fwd_packed(t, t, t, cu)


def test_c_entries_check_before_launching():
    from poly_attention_b200 import _lib
    lib = _lib.lib
    assert lib.poly_sizeof_packed_args() == ctypes.sizeof(_lib.PolyPackedArgs)
    assert lib.poly_sizeof_packed_bwd_args() == ctypes.sizeof(_lib.PolyPackedBwdArgs)
    assert lib.poly_packed_pass_fwd(None, None) == _lib.POLY_EINVAL
    assert lib.poly_packed_pass_bwd(None, None) == _lib.POLY_EINVAL
    assert lib.poly_packed_pass_bwd_workspace_size(None) == 0

    def args(cls, **kw):
        a = cls()
        f = a.fwd if cls is _lib.PolyPackedArgs else a.bwd.fwd
        f.batch, f.heads, f.kv_heads, f.seq_q, f.seq_k, f.head_dim, f.scale = 1, 2, 1, 16, 16, 64, 0.1
        f.q = f.k = f.v = f.out = 256
        a.cu_seqlens, a.seqs = 256, 2
        for k, v in kw.items():
            setattr(f if hasattr(f, k) else a, k, v)
        return a

    for cls, call in ((_lib.PolyPackedArgs, lib.poly_packed_pass_fwd), (_lib.PolyPackedBwdArgs, lib.poly_packed_pass_bwd)):
        for kw, rc in ((dict(batch=2), _lib.POLY_EINVAL), (dict(seq_k=8), _lib.POLY_EINVAL), (dict(heads=3, kv_heads=2), _lib.POLY_EINVAL),
                       (dict(dtype=7), _lib.POLY_EINVAL), (dict(head_dim=129), _lib.POLY_EUNSUPPORTED),
                       (dict(key_mask=256), _lib.POLY_EUNSUPPORTED), (dict(query_mask=256), _lib.POLY_EUNSUPPORTED),
                       (dict(v_mul=256), _lib.POLY_EUNSUPPORTED), (dict(causal_offset=128), _lib.POLY_EUNSUPPORTED),
                       (dict(seqs=-1), _lib.POLY_EINVAL), (dict(max_len=-1), _lib.POLY_EINVAL), (dict(cu_seqlens=None), _lib.POLY_EINVAL),
                       (dict(q=None), _lib.POLY_EINVAL), (dict(scale=float("nan")), _lib.POLY_EINVAL),
                       (dict(epi_out=256), _lib.POLY_EINVAL), (dict(seq_q=2 ** 31 - 1, seq_k=2 ** 31 - 1), _lib.POLY_EUNSUPPORTED)):
            assert call(args(cls, **kw), None) == rc, kw
        assert call(args(cls, seq_q=0, seq_k=0), None) == _lib.POLY_OK
        assert call(args(cls, seqs=0), None) == _lib.POLY_OK
    # the backward's own needs: its tensors, then its workspace
    assert lib.poly_packed_pass_bwd(args(_lib.PolyPackedBwdArgs), None) == _lib.POLY_EINVAL
    b = args(_lib.PolyPackedBwdArgs, lse=256)
    b.bwd.dout = b.bwd.dq = b.bwd.dk = b.bwd.dv = 256
    assert lib.poly_packed_pass_bwd(b, None) == _lib.POLY_EINVAL
    assert "workspace" in lib.poly_last_error().decode()


@pytest.mark.parametrize("block", [8, 64, 128, 256])
def test_slot_numbering_covers_every_tile_once(block):
    """The search of csrc/packed.cuh restated: every tile of every sequence has one slot, every slot stays inside."""
    def locate(cu, total, slot):
        at = lambda s: min(max(cu[s], 0), total)   # noqa: E731
        lo, hi = 0, len(cu) - 1
        while hi - lo > 1:
            mid = (lo + hi) >> 1
            if at(mid) // block + mid <= slot:
                lo = mid
            else:
                hi = mid
        start, length = at(lo), at(lo + 1) - at(lo)
        tile = slot - (start // block + lo)
        return (lo, start, length, tile) if tile >= 0 and tile * block < length else None

    rng = random.Random(block)
    for _ in range(300):
        lens = [rng.choice([0, 1, rng.randrange(3 * block), block, block - 1, block + 1]) for _ in range(rng.randrange(1, 12))]
        lead = rng.choice([0, 0, 5, 300])
        cu = [lead]
        for n in lens:
            cu.append(cu[-1] + n)
        total = cu[-1] + rng.choice([0, 0, 7, 500])
        found = [t for t in (locate(cu, total, s) for s in range(total // block + len(lens))) if t]
        want = [(s, cu[s], n, t) for s, n in enumerate(lens) for t in range((n + block - 1) // block)]
        assert sorted((a, b, c, d) for a, b, c, d in found) == sorted(want)
        # tiles of different sequences never share a slot, so slot-addressed rows do not overlap
        wild = [rng.randrange(-1000, 2000) for _ in range(len(cu))]
        for s in range(total // block + len(lens)):
            t = locate(wild, total, s)
            if t:
                assert 0 <= t[1] and t[1] + t[2] <= total and t[1] + t[3] * block < total


def test_workspace_rows_of_sequences_are_apart():
    """csrc/packed.cuh's workspace rows restated: a sequence owns 8 (start / 8 + its number) and on, whole blocks of 8."""
    rng = random.Random(1)
    for _ in range(2000):
        lens = [rng.choice([0, 0, 1, 2, 3, 4, 5, rng.randrange(300)]) for _ in range(rng.randrange(1, 40))]
        cu = [rng.choice([0, 0, 1, 7])]
        for n in lens:
            cu.append(cu[-1] + n)
        total = cu[-1] + rng.choice([0, 0, 1, 50])
        end = 0
        for s, n in enumerate(lens):
            row = 8 * (cu[s] // 8 + s)
            assert row >= end
            end = row + (n + 7) // 8 * 8
        assert end <= 8 * (total // 8 + len(lens))
        # offsets that break the contract: a sequence's rows lie within [0, total], so its workspace rows stay inside too
        for s in range(len(lens)):
            start = rng.randrange(total + 1)
            n = rng.randrange(total - start + 1)
            assert 8 * (start // 8 + s) + (n + 7) // 8 * 8 <= 8 * (total // 8 + len(lens))


@pytest.mark.parametrize("d", [64, 128])
def test_backward_workspace_follows_the_tokens(d):
    """Many short sequences without a length bound: scratch for the tokens, not for a tile of rows a sequence."""
    from poly_attention_b200 import _lib

    def need(total, seqs):
        a = _lib.PolyPackedBwdArgs()
        f = a.bwd.fwd
        f.batch, f.heads, f.kv_heads, f.seq_q, f.seq_k, f.head_dim, f.scale, f.dtype = 1, 16, 16, total, total, d, 0.1, _lib.POLY_BF16
        for x, names in ((f, ("q", "k", "v", "out")), (a.bwd, ("dout", "dq", "dk", "dv"))):
            for name in names:
                setattr(x, name, 256)
                st = getattr(x, name + "_stride")
                st[1], st[2] = d, 16 * d
        a.cu_seqlens, a.seqs = 256, seqs
        assert _lib.lib.poly_packed_pass_bwd_kernel_name(a) == b"tc100"
        return _lib.lib.poly_packed_pass_bwd_workspace_size(a)

    for total, seqs in ((32768, 4096), (160000, 20000), (100, 1), (1, 1), (16411, 12)):
        # dq of the rows and 8 more a sequence; lse and delta in slots of 128; an order of 8192 slots at most
        slots = total // 128 + seqs
        assert need(total, seqs) <= 16 * ((total + 8 * seqs) * d + slots * 128 * 2) * 4 + 4 * 8192


@pytest.mark.parametrize("dtype,d,bound,want", [
    (torch.bfloat16, 64, None, ("tc100", "tc100")), (torch.float16, 128, 129, ("tc100", "tc100")),
    (torch.bfloat16, 64, 128, ("small", "small")), (torch.float16, 128, 1, ("small", "small")),
    (torch.float32, 64, 128, ("tf32x3", "simt")), (torch.float32, 128, None, ("simt", "simt")),
    (torch.bfloat16, 32, 16, ("simt", "simt"))])
def test_kernel_choice(dtype, d, bound, want):
    """The kernels that the GPU tests mean to reach (the choice looks at sizes and addresses only)."""
    from poly_attention_b200.packed import packed_kernel_names
    q, k = torch.empty(400, 4, d, dtype=dtype), torch.empty(400, 2, d, dtype=dtype)
    assert packed_kernel_names(q, k, k, bound) == want
