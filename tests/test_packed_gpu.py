"""Passes and chains over packed sequences against 64 bits (tolerances: pass_reference.py)."""
import pytest
import torch

import pass_reference as R

pytestmark = pytest.mark.gpu

LENGTHS = {
    "tiny": [1, 2, 0, 5],
    "small": [64, 1, 37, 0, 128, 16, 17, 100],
    "edges": [127, 128, 129, 255, 256, 257, 1, 0],
    "ragged": [500, 3, 77, 0, 641, 130],
    "one": [333],
}


def make(lens, h, g, d, dtype, seed=0, rest=0, bias=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(lens) + rest
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    q, k, v, do = (rnd(n, x, d).to(dtype) for x in (h, g, g, h))
    b = rnd(g, n) * 2 if bias else None
    return q, k, v, do, b, rnd(h, n)


def seqs(lens):
    a = 0
    for n in lens:
        if n:
            yield slice(a, a + n)
        a += n


def causal_keep(n, causal):
    return torch.ones(n, n, dtype=torch.bool, device="cuda").tril() if causal else None


def t64(x, sl):
    return x[sl].double().transpose(0, 1)


def check_pass(lens, h, g, d, dtype, causal, bias=False, clamp=None, seed=0, rest=0, max_seqlen=None, data=None, backward=True):
    import poly_attention_b200 as P
    q, k, v, do, b, dl = data or make(lens, h, g, d, dtype, seed, rest, bias)
    cu, _ = P.packed_offsets(lens)
    kw = dict(causal=causal, softclamp=clamp, bias=b, max_seqlen=max_seqlen)
    out, lse = P.pass_fwd_packed(q, k, v, cu, **kw)
    assert out.dtype == dtype and lse.dtype == torch.float32
    if backward:
        dq, dk, dv, db = P.pass_bwd_packed(q, k, v, cu, out, lse, do, dlse=dl, want_dbias=True, **kw)
    for sl in seqs(lens):
        n, scale = sl.stop - sl.start, d ** -0.5
        ref = [t64(x, sl) for x in (q, k, v)]
        bb = None if b is None else b[:, sl].double()
        (o, ot), (l, lt), st = R.forward(*ref, bb, causal_keep(n, causal), scale, clamp, dtype)
        what = f"length {n} at {sl.start}"
        R.assert_within(out[sl].transpose(0, 1), o, ot, "out " + what)
        R.assert_within(lse[:, sl], l, lt, "lse " + what)
        if not backward:
            continue
        res = R.backward(*ref, o, t64(do, sl), dl[:, sl].double(), st, scale, clamp, dtype)
        for name, got, (want, tol) in zip(("dq", "dk", "dv"), (dq, dk, dv), res):
            R.assert_within(got[sl].transpose(0, 1), want, tol, f"{name} {what}")
        R.assert_within(db[:, sl], *res[3], "dbias " + what)
    end = sum(lens)
    if out.shape[0] > end:
        for x in (out, lse.T) + ((dq, dk, dv, db.T) if backward else ()):
            assert (x[end:] == 0).all()
    return out, lse


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,g,d", [(2, 2, 64), (4, 1, 128), (4, 2, 32), (3, 3, 20)])
@pytest.mark.parametrize("lens", list(LENGTHS))
def test_pass(lens, h, g, d, causal, dtype):
    check_pass(LENGTHS[lens], h, g, d, dtype, causal, bias=lens != "small")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("bias", [True, False])
def test_softclamp(dtype, d, bias):
    check_pass(LENGTHS["ragged"], 4, 2, d, dtype, True, bias=bias, clamp=3.0)
    check_pass(LENGTHS["small"], 4, 2, d, dtype, False, bias=bias, clamp=3.0, max_seqlen=128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_short_sequences_with_their_bound(dtype, d, causal):
    for lens, bound in (([64, 1, 37, 0, 128, 16, 17, 100], 128), ([5, 16, 0, 1, 3], 16), ([33] * 40, 33), ([80, 65], 100)):
        for bias in (False, True):
            check_pass(lens, 4, 2, d, dtype, causal, bias=bias, max_seqlen=bound)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.float32, 40)])
@pytest.mark.parametrize("bound", [None, 128])
def test_rows_outside_the_sequences(dtype, d, bound):
    """Rows behind the last sequence hold NaN: they reach no result and come out as zeros."""
    lens = [100, 0, 28]
    data = make(lens, 4, 2, d, dtype, rest=70, bias=True)
    for x in data[:4]:
        x[128:] = float("nan")
    data[4][:, 128:] = float("nan")
    data[5][:, 128:] = float("nan")
    check_pass(lens, 4, 2, d, dtype, True, rest=70, data=data, max_seqlen=bound)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_short_sequences_without_their_bound(dtype, d, causal):
    """Sequences of no whole 8 rows, beside one another in the backward's dQ accumulator."""
    check_pass([(i * 7) % 17 for i in range(60)] + [129, 3, 64], 4, 2, d, dtype, causal, bias=True)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.float32, 40)])
@pytest.mark.parametrize("bound", [None, 130])
def test_a_sequence_of_nan_and_infinity_stays_alone(dtype, d, bound):
    import poly_attention_b200 as P
    lens = [100, 30, 130, 5]
    data = make(lens, 4, 2, d, dtype, bias=True)
    bad = slice(100, 130)
    for i, x in enumerate(data[:4]):
        x[bad] = float("nan") if i % 2 else float("inf")
    q, k, v, do, b, dl = data
    b[:, bad], dl[:, bad] = float("inf"), float("nan")
    cu, _ = P.packed_offsets(lens)
    out, lse = P.pass_fwd_packed(q, k, v, cu, causal=True, bias=b, max_seqlen=bound)
    grads = P.pass_bwd_packed(q, k, v, cu, out, lse, do, causal=True, bias=b, dlse=dl, want_dbias=True, max_seqlen=bound)
    for x in (out, lse.T, *grads[:3], grads[3].T):
        assert torch.isfinite(x[:100].float()).all() and torch.isfinite(x[130:].float()).all()
    for x in data[:4]:
        x[bad] = 0
    b[:, bad], dl[:, bad] = 0, 0
    clean, _ = P.pass_fwd_packed(q, k, v, cu, causal=True, bias=b, max_seqlen=bound)
    assert torch.equal(out[:100], clean[:100]) and torch.equal(out[130:], clean[130:])


# fp32 operands are split into two parts that together have to keep every kind of NaN
NANS32 = [(torch.float32, 64, None, bits) for bits in (0x7fffffff, 0x7fc00000, -1, 0x7f800001, -0x400000)]


@pytest.mark.parametrize("dtype,d,bound,bits", NANS32 + [
    (torch.bfloat16, 64, None, 0x7fff), (torch.float16, 128, None, 0x7e00), (torch.bfloat16, 64, 80, 0x7fff), (torch.float16, 64, 128, -1),
    (torch.float16, 128, 128, 0x7e00), (torch.bfloat16, 24, None, 0x7fff), (torch.float32, 24, None, 0x7fffffff)])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_every_nan_reaches_the_rows_that_see_it(which, dtype, d, bound, bits):
    import poly_attention_b200 as P
    t = {name: torch.randn(90, 2, d, device="cuda").to(dtype) for name in "qkv"}
    t[which].view(torch.int32 if dtype == torch.float32 else torch.int16)[70, 1, 5] = bits
    cu = torch.tensor([0, 20, 90], dtype=torch.int32, device="cuda")
    out, lse = P.pass_fwd_packed(t["q"], t["k"], t["v"], cu, causal=True, max_seqlen=bound)
    bad = out.isnan()
    assert not bad[:, 0].any() and not bad[:20].any()
    if which == "q":
        assert bad[70, 1].all() and bad.sum() == d and lse[1, 70].isnan()
    elif which == "k":
        assert bad[70:, 1].all() and not bad[:70].any() and lse[1, 70:].isnan().all()
    else:
        # (0 * NaN may reach the rows before it, as in a matrix product)
        assert bad[70:, 1, 5].all() and not bad[:, :, :5].any() and not bad[:, :, 6:].any() and not lse.isnan().any()


@pytest.mark.parametrize("dtype,d,bound", [
    (torch.bfloat16, 64, None), (torch.float16, 64, 300), (torch.float16, 128, None), (torch.bfloat16, 128, None),
    (torch.bfloat16, 64, 80), (torch.float16, 128, 128), (torch.float32, 64, None), (torch.bfloat16, 24, None)])
@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("bias", [False, True])
def test_every_nan_survives_the_softclamp(which, dtype, d, bound, bias):
    import poly_attention_b200 as P
    t = {name: torch.randn(90, 2, d, device="cuda").to(dtype) for name in "qkv"}
    t[which][70, 1, 5] = float("nan")
    b = torch.randn(2, 90, device="cuda") if bias else None
    cu = torch.tensor([0, 20, 90], dtype=torch.int32, device="cuda")
    out, lse = P.pass_fwd_packed(t["q"], t["k"], t["v"], cu, causal=True, max_seqlen=bound, softclamp=3.0, bias=b)
    seen = slice(70, 71 if which == "q" else 90)
    assert out[seen, 1].isnan().all() and lse[1, seen].isnan().all()
    assert out.isnan().sum() == d * (seen.stop - 70) and lse.isnan().sum() == seen.stop - 70


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bias", [True, False])
def test_softclamp_fp16(d, bias):
    check_pass(LENGTHS["ragged"], 4, 2, d, torch.float16, True, bias=bias, clamp=3.0)
    check_pass(LENGTHS["edges"], 4, 4, d, torch.float16, False, bias=bias, clamp=0.5)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 24)])
@pytest.mark.parametrize("bound", [None, 100])
def test_dead_keys(dtype, d, bound):
    """Keys of bias <= -FLT_MAX / 2 are out; a row that sees no other key is zero with lse -FLT_MAX and no gradient."""
    import poly_attention_b200 as P
    lens = [70, 100]
    q, k, v, do, b, dl = make(lens, 2, 1, d, dtype, bias=True)
    low = torch.finfo(torch.float32).min
    b[:, :40] = low
    b[:, 40:50] = float("-inf")
    b[:, 120] = low * 0.6
    cu, _ = P.packed_offsets(lens)
    out, lse = P.pass_fwd_packed(q, k, v, cu, causal=True, bias=b, max_seqlen=bound)
    dq, dk, dv, db = P.pass_bwd_packed(q, k, v, cu, out, lse, do, causal=True, bias=b, dlse=dl, want_dbias=True, max_seqlen=bound)
    assert (out[:50] == 0).all() and (lse[:, :50] == low).all() and (dq[:50] == 0).all()
    for x in (dk, dv, db.T):
        assert (x[:50] == 0).all() and (x[120] == 0).all()
    for sl, dead in ((slice(0, 70), slice(0, 50)), (slice(70, 170), slice(50, 51))):
        n = sl.stop - sl.start
        keep = causal_keep(n, True).clone()
        keep[:, dead] = False
        live = slice(50, n) if sl.start == 0 else slice(0, n)
        ref = [t64(x, sl) for x in (q, k, v)]
        (o, ot), (l, lt), st = R.forward(*ref, b[:, sl].double().clamp(min=-1e30), keep, d ** -0.5, None, dtype)
        R.assert_within(out[sl].transpose(0, 1)[:, live], o[:, live], ot[:, live], "out")
        R.assert_within(lse[:, sl][:, live], l[:, live], lt[:, live], "lse")
        p, rel, slope, tol = st
        gone = torch.ones(n, 1, device="cuda").double()
        gone[live] = 0
        st = tuple(torch.where(gone.bool(), torch.zeros_like(x), x) if x is not slope else x for x in st)
        o = torch.where(gone.bool(), torch.zeros_like(o), o)
        res = R.backward(*ref, o, t64(do, sl), dl[:, sl].double(), st, d ** -0.5, None, dtype)
        for name, got, (want, t) in zip(("dq", "dk", "dv"), (dq, dk, dv), res):
            R.assert_within(got[sl].transpose(0, 1), want, t, name)


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.7])
@pytest.mark.parametrize("dtype,bound", [(torch.bfloat16, None), (torch.bfloat16, 100), (torch.float32, None)])
def test_scales(scale, dtype, bound):
    import poly_attention_b200 as P
    lens = [70, 100]
    q, k, v, do, b, dl = make(lens, 2, 1, 64, dtype, bias=True)
    cu, _ = P.packed_offsets(lens)
    kw = dict(causal=True, scale=scale, bias=b, max_seqlen=bound)
    out, lse = P.pass_fwd_packed(q, k, v, cu, **kw)
    dq, dk, dv, _ = P.pass_bwd_packed(q, k, v, cu, out, lse, do, **kw)
    for sl in seqs(lens):
        ref = [t64(x, sl) for x in (q, k, v)]
        (o, ot), (l, lt), st = R.forward(*ref, b[:, sl].double(), causal_keep(sl.stop - sl.start, True), scale, None, dtype)
        R.assert_within(out[sl].transpose(0, 1), o, ot, "out")
        R.assert_within(lse[:, sl], l, lt, "lse")
        for name, got, (want, t) in zip(("dq", "dk", "dv"), (dq, dk, dv), R.backward(*ref, o, t64(do, sl), None, st, scale, None, dtype)):
            R.assert_within(got[sl].transpose(0, 1), want, t.abs() + 1e-30, name)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 128)])
def test_strides_and_alignment(dtype, d):
    """Head-split views of one projection, head-major tensors, odd offsets, features not contiguous."""
    import poly_attention_b200 as P
    lens = [60, 200, 1]
    q, k, v, do, b, dl = make(lens, 4, 2, d, dtype, bias=True)
    cu, _ = P.packed_offsets(lens)
    n = sum(lens)
    want, lw = P.pass_fwd_packed(q, k, v, cu, causal=True, bias=b)
    fused = torch.randn(n, 3 * 4 * d, device="cuda").to(dtype)
    fused[:, :4 * d], fused[:, 4 * d:6 * d], fused[:, 8 * d:10 * d] = q.reshape(n, -1), k.reshape(n, -1), v.reshape(n, -1)
    views = (fused[:, :4 * d].unflatten(1, (4, d)), fused[:, 4 * d:6 * d].unflatten(1, (2, d)), fused[:, 8 * d:10 * d].unflatten(1, (2, d)))
    major = tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))

    def shift(x):
        buf = torch.empty(x.numel() + 1, device="cuda", dtype=dtype)
        buf[1:] = x.reshape(-1)
        return buf[1:].view(x.shape)

    spread = tuple(torch.stack((x, x), -1).flatten(-2)[..., ::2] for x in (q, k, v))
    bt = b.T.contiguous().T
    for kind, ts in (("views", views), ("head-major", major), ("odd", tuple(shift(x) for x in (q, k, v))), ("spread", spread)):
        out, lse = P.pass_fwd_packed(*ts, cu, causal=True, bias=bt)
        if kind == "odd":       # other kernels
            data = (*ts, do, bt, dl)
            check_pass(lens, 4, 2, d, dtype, True, data=data)
        else:
            assert torch.equal(out, want) and torch.equal(lse, lw), kind
    g0 = P.pass_bwd_packed(q, k, v, cu, want, lw, do, causal=True, bias=b)
    g1 = P.pass_bwd_packed(*views, cu, want, lw, do.transpose(0, 1).contiguous().transpose(0, 1), causal=True, bias=bt)
    for x, y in zip(g0[1:3], g1[1:3]):
        assert torch.equal(x, y)


def exact_chain(qs, vs, h, causal, clamp, lens, scale):
    """64-bit autograd over every sequence: qs [total, heads, d]."""
    order = len(qs) - 1
    outs = torch.zeros_like(qs[0])
    for sl in seqs(lens):
        n = sl.stop - sl.start
        q = [x[sl].transpose(0, 1) for x in qs]
        v = [x[sl].transpose(0, 1) for x in vs]
        val, bias = v[-1], None
        for t in range(order - 1, -1, -1):
            r = q[t].shape[0] // q[t + 1].shape[0]
            s = q[t] @ q[t + 1].repeat_interleave(r, 0).transpose(1, 2) * scale
            if clamp:
                s = clamp * torch.tanh(s / clamp)
            if bias is not None:
                s = s + bias.repeat_interleave(r, 0)[:, None]
            if causal:
                s = s.masked_fill(~causal_keep(n, True), float("-inf"))
            lse = torch.logsumexp(s, -1)
            msg = torch.softmax(s, -1) @ val.repeat_interleave(r, 0)
            val, bias = (v[t - 2] * msg if t >= 2 else msg), lse
        outs = outs.index_copy(0, torch.arange(sl.start, sl.stop, device="cuda"), msg.transpose(0, 1))
    return outs


@pytest.mark.parametrize("order", [2, 3, 4])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 16])
def test_chain_gradients_fp32(order, causal, d):
    """fp32 chains against 64-bit autograd: errors of 2^-20 a product through 2 order passes and values of size
    about 4 stay below 1e-4 of the largest gradient."""
    import poly_attention_b200 as P
    lens, h, g = [70, 0, 1, 33, 150], 4, 2
    gen = torch.Generator(device="cuda").manual_seed(order)
    n = sum(lens)
    leaves = [torch.randn(n, h if i == 0 else g, d, generator=gen, device="cuda", requires_grad=True) for i in range(2 * order)]
    qs, vs = leaves[:order + 1], leaves[order + 1:]
    cu, longest = P.packed_offsets(lens)
    clamp = 5.0 if order == 3 else None
    out, lses, msgs = P.poly_attention_chain_packed(qs[:-1], qs[1:], vs, cu, causal=causal, softclamp_value=clamp, max_seqlen=longest)
    do = torch.randn(n, h, d, generator=gen, device="cuda")
    grads = torch.autograd.grad(out, leaves, do)
    wide = [x.detach().double().requires_grad_(True) for x in leaves]
    ref = exact_chain(wide[:order + 1], wide[order + 1:], h, causal, clamp, lens, d ** -0.5)
    rg = torch.autograd.grad(ref, wide, do.double())
    assert (out.double() - ref).abs().max() < 1e-4 * ref.abs().max()
    for i, (a, b) in enumerate(zip(grads, rg)):
        assert (a.double() - b).abs().max() < 1e-4 * b.abs().max(), i
    assert len(lses) == len(msgs) == order - 1 and lses[0].shape == (g, n) and msgs[0].shape == (n, g, d)


def test_chain_gradient_against_differences():
    import poly_attention_b200 as P
    lens, d = [9, 4], 16
    gen = torch.Generator(device="cuda").manual_seed(3)
    leaves = [torch.randn(13, 2, d, generator=gen, device="cuda", requires_grad=True) for _ in range(4)]
    w = torch.randn(13, 2, d, generator=gen, device="cuda").double()
    cu, _ = P.packed_offsets(lens)
    f = lambda ts: (P.poly_attention_order2_packed(*ts, cu, causal=True)[0].double() * w).sum()   # noqa: E731
    grads = torch.autograd.grad(f(leaves), leaves)
    eps = 2.0 ** -6
    for i, (x, g) in enumerate(zip(leaves, grads)):
        step = torch.randn(x.shape, generator=gen, device="cuda")
        with torch.no_grad():
            moved = lambda s: [t + s * eps * step if j == i else t for j, t in enumerate(leaves)]   # noqa: E731
            diff = float(f(moved(1)) - f(moved(-1))) / (2 * eps)
        want = float((g.double() * step.double()).sum())
        # central differences: eps^2 / 6 of a third derivative of some 10 |gradient|, and 2^-20 / eps of |f|'s terms
        size = float(g.abs().double().pow(2).sum().sqrt()) * 14 + float(w.abs().sum()) * 2.0 ** -20 / eps
        assert abs(diff - want) < 10 * eps ** 2 / 6 * size + size * 1e-3, i


@pytest.mark.parametrize("dtype,d,bound", [(torch.bfloat16, 64, None), (torch.float16, 128, None), (torch.bfloat16, 64, 128)])
@pytest.mark.parametrize("order", [2, 3])
def test_chain_is_its_passes(dtype, d, bound, order):
    """The chain's results are the passes' own, whose errors test_pass bounds."""
    import poly_attention_b200 as P
    lens, h, g = [100, 0, 128, 3], 4, 2
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = sum(lens)
    leaves = [torch.randn(n, h if i == 0 else g, d, generator=gen, device="cuda").to(dtype).requires_grad_(True)
              for i in range(2 * order)]
    qs, vs = leaves[:order + 1], leaves[order + 1:]
    cu, _ = P.packed_offsets(lens)
    kw = dict(causal=True, max_seqlen=bound)
    out, lses, msgs = P.poly_attention_chain_packed(qs[:-1], qs[1:], vs, cu, **kw)
    do = torch.randn(n, h, d, generator=gen, device="cuda").to(dtype)
    grads = torch.autograd.grad(out, leaves, do)
    with torch.no_grad():
        val, bias, st = vs[-1], None, {}
        for t in range(order - 1, -1, -1):
            res = P.pass_fwd_packed(qs[t], qs[t + 1], val, cu, bias=bias, epi_mul=vs[t - 2] if t >= 2 else None, out_lo=True, **kw)
            st[t] = (val, bias, res[0], res[1], res[-1])
            # out + out_lo is out in more bits, and the epilogue's product is made from it
            wide = res[0].double() + res[-1].double()
            half = torch.finfo(dtype).eps / 2 * res[0].double().abs() + 2.0 ** -25
            assert (res[-1].double().abs() <= half).all() and (res[-1] != 0).any()
            if t >= 2:
                step = torch.finfo(dtype).eps / 2
                want = vs[t - 2].double() * wide
                tol = (step + 2 * step ** 2) * want.abs() + (2.0 ** -24 * (1 + vs[t - 2].double().abs()) if dtype == torch.float16 else 0)
                assert ((res[2].double() - want).abs() <= tol).all()
            val, bias = res[2] if t >= 2 else res[0], res[1]
        assert torch.equal(out, st[0][2])
        for i, t in enumerate(range(order - 1, 0, -1)):
            assert torch.equal(msgs[i], st[t][2]) and torch.equal(lses[i], st[t][3])
        g_out, g_lse, dk = do, None, None
        for t in range(order):
            fac = (vs[t - 1], st[t + 1][2]) if 0 < t < order - 1 else None
            dq, dkn, dv, db = P.pass_bwd_packed(qs[t], qs[t + 1], st[t][0], cu, st[t][2], st[t][3], g_out, bias=st[t][1],
                                                dlse=g_lse, dq=dk, want_dbias=True, out_lo=st[t][4], factors=fac, **kw)
            if fac is not None:
                # the factors' gradients are the values' times the other factor, rounded once more
                plain = P.pass_bwd_packed(qs[t], qs[t + 1], st[t][0], cu, st[t][2], st[t][3], g_out, bias=st[t][1],
                                          dlse=g_lse, want_dbias=True, out_lo=st[t][4], **kw)[2].double()
                for got, other in zip(dv, (fac[1], fac[0])):
                    want = plain * other.double()
                    floor = 2.0 ** -24 * (1 + other.double().abs()) if dtype == torch.float16 else 0
                    assert ((got.double() - want).abs() <= 1.01 * torch.finfo(dtype).eps * want.abs() + floor).all()
            # dq sums its key tiles in 32 bits in any order: one step of the type
            near = lambda a, b: bool(((a.float() - b.float()).abs() <= 2 * torch.finfo(dtype).eps * b.float().abs() + 1e-3).all())   # noqa: E731
            assert near(grads[t], dq)
            if t == order - 1:
                assert near(grads[t + 1], dkn) and near(grads[2 * order - 1], dv)
            if fac is not None:
                assert near(grads[order + 1 + t - 1], dv[0])
            g_out, g_lse, dk = (dv if fac is None else dv[1]), db, dkn


@pytest.mark.parametrize("kind", ["order2", "order3"])
@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_modules_on_packed_sequences(kind, rotary, dtype):
    """A packed batch through the module equals its sequences one by one, positions, gates and gradients included."""
    import poly_attention_b200 as P
    torch.manual_seed(0)
    kw = dict(dim=64, heads=4, kv_heads=2, dim_head=64, causal=True, use_rotary_embed=rotary, prenorm=True, attn_gate=True,
              multiply_root_value=True)
    attn = (P.PolyAttention(**kw) if kind == "order2" else P.NPolyAttention(order=3, **kw)).cuda().to(dtype)
    lens = [40, 1, 0, 150]
    cu, longest = P.packed_offsets(lens)
    x = torch.randn(1, sum(lens) + 5, 64, device="cuda").to(dtype).requires_grad_(True)
    y = attn(x, cu_seqlens=cu, max_seqlen=longest)
    parts = [attn(x[:, sl]) for sl in seqs(lens)]
    end = sum(lens)
    want = torch.cat(parts, 1)
    # the same mathematics by other kernels: fp32 within 1e-4; bf16 within the modules' bar (2e-2 + 1e-2 |x|)
    tol = 1e-4 if dtype == torch.float32 else 2e-2
    assert ((y[:, :end] - want).abs() <= tol + (0 if dtype == torch.float32 else 1e-2) * want.abs()).all()
    w = torch.randn_like(want)
    params = [p for p in attn.parameters() if p.requires_grad]
    ga = torch.autograd.grad((y[:, :end] * w).sum(), [x, *params])
    gb = torch.autograd.grad((want * w).sum(), [x, *params])
    for a, b in zip(ga, gb):
        assert torch.isfinite(a).all()
        assert (a.float() - b.float()).norm() <= (1e-4 if dtype == torch.float32 else 3e-2) * b.float().norm() + 1e-6


@pytest.mark.parametrize("order", [2, 3])
def test_a_checkpointed_packed_module(order):
    """Activations formed again in the backward: the same kernels on the same inputs."""
    from torch.utils.checkpoint import checkpoint

    import poly_attention_b200 as P
    torch.manual_seed(0)
    kw = dict(dim=64, heads=2, dim_head=64, causal=True, use_rotary_embed=True, prenorm=True)
    attn = (P.PolyAttention(**kw) if order == 2 else P.NPolyAttention(order=3, **kw)).cuda()
    cu, longest = P.packed_offsets([7, 0, 30])
    x = torch.randn(1, 37, 64, device="cuda")
    grads = []
    for call in (attn, lambda *a, **k: checkpoint(attn, *a, use_reentrant=False, **k)):
        y = x.clone().requires_grad_(True)
        call(y, cu_seqlens=cu, max_seqlen=longest).square().sum().backward()
        grads.append(y.grad)
    assert torch.equal(*grads)


def test_module_refusals():
    import poly_attention_b200 as P
    attn = P.PolyAttention(dim=64, heads=2, dim_head=64).cuda()
    x = torch.randn(1, 20, 64, device="cuda")
    cu, _ = P.packed_offsets([20])
    mask = torch.ones(1, 20, dtype=torch.bool, device="cuda")
    for kw in (dict(mask=mask), dict(context=x), dict(context_mask=mask), dict(return_cache=True)):
        with pytest.raises(ValueError, match="packed"):
            attn(x, cu_seqlens=cu, **kw)
    with pytest.raises(ValueError, match="packed"):
        attn(torch.randn(2, 20, 64, device="cuda"), cu_seqlens=cu)


def test_refusals():
    import poly_attention_b200 as P
    q, k, v, do, b, dl = make([8, 8], 4, 2, 64, torch.bfloat16, bias=True)
    cu, _ = P.packed_offsets([8, 8])
    fwd = lambda *a, **kw: P.pass_fwd_packed(*a, **kw)   # noqa: E731
    for err, args, kw in [
        (TypeError, (q, k.float(), v, cu), {}), (TypeError, (q.double(), k.double(), v.double(), cu), {}),
        (ValueError, (q, k[:8], v[:8], cu), {}), (ValueError, (q, k, v[:, :1], cu), {}), (ValueError, (q[None], k, v, cu), {}),
        (ValueError, (q[:, :3], k, v, cu), {}), (ValueError, (q, k, v, cu[None]), {}), (ValueError, (q, k, v, cu.float()), {}),
        (RuntimeError, (q, k, v, cu.cpu()), {}), (RuntimeError, (q.cpu(), k, v, cu), {}),
        (ValueError, (q, k, v, cu), dict(bias=b[:, :5])), (ValueError, (q, k, v, cu), dict(epi_mul=q[:8])),
        (ValueError, (q, k, v, cu), dict(max_seqlen=-1)),
        (NotImplementedError, (torch.randn(16, 2, 160, device="cuda"),) * 3 + (cu,), {}),
    ]:
        with pytest.raises(err):
            fwd(*args, **kw)
    out, lse = fwd(q, k, v, cu)
    with pytest.raises(ValueError):
        P.pass_bwd_packed(q, k, v, cu, out, lse[:, :4], do)
    with pytest.raises(ValueError):
        P.pass_bwd_packed(q, k, v, cu, out, lse, do[:4])
    with pytest.raises(ValueError):
        P.poly_attention_chain_packed([q], [k], [], cu)


def test_offsets_that_break_the_contract_stay_inside():
    """Offsets out of range, decreasing or past the rows: any result, no access outside, no error."""
    import poly_attention_b200 as P
    for dtype, d in ((torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.float32, 24)):
        q, k, v, do, b, dl = make([300], 4, 2, d, dtype, bias=True)
        for cu in ([0, 400], [-50, 100, 300], [0, 200, 100, 300], [300, 0], [250, 250], [0, 2 ** 31 - 1, -2 ** 31, 300]):
            cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
            for bound in (None, 100):
                out, lse = P.pass_fwd_packed(q, k, v, cu, causal=True, bias=b, max_seqlen=bound)
                P.pass_bwd_packed(q, k, v, cu, torch.zeros_like(q), torch.zeros_like(lse), do, causal=True, bias=b, max_seqlen=bound)
        torch.cuda.synchronize()


@pytest.mark.parametrize("bound", [60, 100])
def test_a_wrong_length_bound_gives_nan(bound):
    import poly_attention_b200 as P
    lens = [50, 130, 7]
    q, k, v, do, b, dl = make(lens, 4, 2, 64, torch.bfloat16, bias=True)
    cu, _ = P.packed_offsets(lens)
    kw = dict(causal=True, bias=b, max_seqlen=bound)
    out, lse, epi, lo = P.pass_fwd_packed(q, k, v, cu, epi_mul=q, out_lo=True, **kw)
    dq, (dv, dr), dk, db = [P.pass_bwd_packed(q, k, v, cu, q, lse, do, want_dbias=True, factors=(k, v), **kw)[i] for i in (0, 2, 1, 3)]
    for x in (out, lse.T, epi, lo, dq, dk, dv, dr, db.T):
        assert torch.isnan(x[50:180]).all() and torch.isfinite(x[:50]).all() and torch.isfinite(x[180:]).all()


def test_long_rest_and_odd_rows():
    import poly_attention_b200 as P
    for dtype, d in ((torch.bfloat16, 64), (torch.float32, 64), (torch.float16, 20)):
        lens = [40]
        data = make(lens, 2, 1, d, dtype, rest=3000, bias=True)
        check_pass(lens, 2, 1, d, dtype, True, rest=3000, data=data)


def test_empty():
    import poly_attention_b200 as P
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, do, b, dl = make([0], 4, 2, 64, dtype, bias=True)
        for lens in ([], [0], [0, 0, 0]):
            cu, longest = P.packed_offsets(lens)
            assert longest == 0
            out, lse = P.pass_fwd_packed(q, k, v, cu, bias=b)
            assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
            P.pass_bwd_packed(q, k, v, cu, out, lse, do, bias=b, want_dbias=True)
        q, k, v, do, b, dl = make([10], 4, 2, 64, dtype, bias=True)
        for lens in ([], [0, 0]):
            cu, _ = P.packed_offsets(lens)
            out, lse = P.pass_fwd_packed(q, k, v, cu, bias=b)
            assert (out == 0).all() and (lse == 0).all()
            for x in P.pass_bwd_packed(q, k, v, cu, out, lse, do, bias=b, want_dbias=True):
                assert (x == 0).all()


def test_streams_graphs_and_two_calls_at_once():
    import poly_attention_b200 as P
    lens = [200, 56, 300]
    q, k, v, do, b, dl = make(lens, 4, 2, 64, torch.bfloat16, bias=True)
    cu, _ = P.packed_offsets(lens)

    def call():
        out, lse = P.pass_fwd_packed(q, k, v, cu, causal=True, bias=b)
        return (out, lse, *P.pass_bwd_packed(q, k, v, cu, out, lse, do, causal=True, bias=b, want_dbias=True)[1:])

    want = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want))
    # captured once, replayed on other sequences of the same rows
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(held, want))
    other = [1, 555, 0]
    cu.copy_(P.packed_offsets(other)[0])
    graph.replay()
    again = call()
    assert all(torch.equal(x, y) for x, y in zip(held, again)) and not torch.equal(again[0], want[0])
