"""Rotary positions on the GPU against the rotation in 64 bits.

Tolerance of an element of the pair (a, b): the angle is rounded once to fp32
as a fraction of half a turn (at most 2^-25, i.e. pi 2^-25 rad), sincospif is
good to 2 units in the last place (2^-22 of 1), the amplitude's and the two
products' roundings add 3 2^-24: (|x_a| + |x_b|) m 6e-7 in all, and the result
is rounded once to the tensors' type (eps / 2 of it).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(x, ang, m, interleaved, inverse=False):
    """x [b, h, n, d] and ang [b, n, rot / 2] in 64 bits; also the size |x_a| + |x_b| of every element."""
    x = x.detach().double().cpu().numpy()
    rot, half = 2 * ang.shape[-1], ang.shape[-1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = np.cos(ang)[:, None] * m, np.sin(ang)[:, None] * m * (-1 if inverse else 1)
    y, size = x.copy(), np.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    assert rot <= x.shape[-1]
    return y, size


def check(got, want, size, m, dtype):
    tol = 6e-7 * m * size + torch.finfo(dtype).eps / 2 * np.abs(want) * (1 + 1e-6) + 1e-7 * (dtype == torch.float16)
    err = np.abs(got.detach().double().cpu().numpy() - want)
    assert got.dtype == dtype
    assert np.all(err <= tol), float((err - tol).max())


def angles(pos, inv):
    return pos.double().cpu().numpy()[..., None] * inv.double().cpu().numpy()


def tensors(shapes, dtype, token_major=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for b, h, n, d in shapes:
        t = torch.randn(b, n, h, d, generator=g, device="cuda").to(dtype).permute(0, 2, 1, 3)
        out.append(t if token_major else t.contiguous())
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,h,n,d,rot", [(1, 1, 1, 64, 64), (2, 3, 37, 64, 32), (3, 4, 129, 128, 128), (1, 2, 700, 128, 16),
                                         (2, 2, 5, 24, 12), (1, 1, 3, 7, 2), (2, 5, 33, 256, 256), (40, 2, 1, 96, 48)])
def test_rotation(dtype, interleaved, b, h, n, d, rot):
    import poly_attention_b200 as P
    inv, _ = P.rotary_frequencies(rot)
    inv = inv.cuda()
    xs = tensors([(b, h, n, d), (b, 1, n, d), (b, 2 * h, n, d)], dtype, token_major=bool(n & 1))
    before = [x.clone() for x in xs]
    ys = P.apply_rotary(xs, inv, positions=11, interleaved=interleaved, attention_factor=1.25)
    ang = angles(torch.arange(11, 11 + n).expand(b, n), inv)
    for x, y, x0 in zip(xs, ys, before):
        want, size = reference(x, ang, 1.25, interleaved)
        check(y, want, size, 1.25, dtype)
        assert torch.equal(y[..., rot:], x[..., rot:]) and torch.equal(x, x0)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_far_positions_keep_their_angle(wide):
    import poly_attention_b200 as P
    inv, m = P.rotary_frequencies(64, scaling="yarn", factor=16.0, original_length=4096)
    inv = inv.cuda()
    b, n = 3, 50
    g = torch.Generator(device="cuda").manual_seed(1)
    pos = torch.randint(0, 1 << 24, (b, n), generator=g, device="cuda").to(wide)
    pos[0, 0], pos[0, 1] = 0, -5
    for p in (pos, pos[:1], pos[1]):
        x, = tensors([(b, 2, n, 64)], torch.float32)
        y = P.apply_rotary(x, inv, positions=p, attention_factor=m)
        want, size = reference(x, angles(p.expand(b, n), inv), m, True)
        check(y, want, size, m, torch.float32)


@pytest.mark.parametrize("shape", [(30, 8), (2, 30, 8)])
def test_given_angles(shape):
    import poly_attention_b200 as P
    g = torch.Generator(device="cuda").manual_seed(2)
    ang = 50 * torch.randn(*shape, generator=g, device="cuda")
    x, = tensors([(2, 3, 30, 20)], torch.float32)
    want, size = reference(x, ang.double().cpu().numpy().reshape(-1, 30, 8) * np.ones((2, 1, 1)), 1.0, False)
    check(P.apply_rotary(x, angles=ang, interleaved=False), want, size, 1.0, torch.float32)


def test_packed_positions():
    import poly_attention_b200 as P
    lens = [5, 0, 1, 200, 33, 0]
    cu = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
    total = sum(lens) + 3                                  # rows behind the last sequence count on
    inv = P.rotary_frequencies(32)[0].cuda()
    x = torch.randn(total, 4, 64, device="cuda", dtype=torch.bfloat16)
    y = P.apply_rotary(x, inv, cu_seqlens=cu)
    pos = np.concatenate([np.arange(n) for n in lens] + [np.arange(3)])
    want, size = reference(x.transpose(0, 1)[None], angles(torch.tensor(pos)[None], inv), 1.0, True)
    n = sum(lens)
    check(y[:n].transpose(0, 1)[None], want[:, :, :n], size[:, :, :n], 1.0, torch.bfloat16)
    assert y.shape == x.shape and y.is_contiguous()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
def test_gradient_is_the_transpose(dtype, interleaved):
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(32)[0].cuda()
    xs = [x.requires_grad_(True) for x in tensors([(2, 4, 65, 48), (2, 2, 65, 48)], dtype)]
    ys = P.apply_rotary(xs, inv, positions=3, interleaved=interleaved, attention_factor=0.75)
    dys = tensors([(2, 4, 65, 48), (2, 2, 65, 48)], dtype, token_major=False, seed=9)
    grads = torch.autograd.grad(ys, xs, dys)
    ang = angles(torch.arange(3, 68).expand(2, 65), inv)
    for g, dy in zip(grads, dys):
        want, size = reference(dy, ang, 0.75, interleaved, inverse=True)
        check(g, want, size, 0.75, dtype)
    # one output used only, through a broadcast gradient
    y0, _ = P.apply_rotary(xs, inv, positions=3, interleaved=interleaved, attention_factor=0.75)
    g0, = torch.autograd.grad(y0.sum(), xs[:1])
    want, size = reference(torch.ones_like(xs[0]), ang, 0.75, interleaved, inverse=True)
    check(g0, want, size, 0.75, dtype)


def test_gradient_against_differences():
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(8)[0].cuda()
    x = torch.randn(1, 2, 5, 8, device="cuda", requires_grad=True)
    w = torch.randn(1, 2, 5, 8, device="cuda")
    f = lambda t: (P.apply_rotary(t, inv, positions=2).double() * w.double()).sum()   # noqa: E731
    g, = torch.autograd.grad(f(x), x)
    with torch.no_grad():
        for i in (0, 9, 33, 79):
            e = torch.zeros_like(x).view(-1)
            e[i] = 0.5
            diff = float(f(x + e.view_as(x)) - f(x - e.view_as(x)))
            # the map is linear: only fp32 roundings of about 20 terms of size 4 remain
            assert abs(diff - float(g.reshape(-1)[i])) < 20 * 4 * 2 * 6e-7


def test_positions_changed_before_the_backward_are_refused():
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(16)[0].cuda()
    x = torch.randn(1, 2, 5, 16, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda")
    y = P.apply_rotary(x, inv, positions=pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    with pytest.raises(TypeError):
        P.apply_rotary(x, inv, positions=1.5)


def test_offsets_as_the_packed_passes_take_them():
    """No sequence at all is a batch, offsets that are no integers are not."""
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(16)[0].cuda()
    x = torch.randn(5, 2, 16, device="cuda")
    none, longest = P.packed_offsets([])
    assert P.apply_rotary(x[:0], inv, cu_seqlens=none).shape == (0, 2, 16)
    assert torch.equal(P.apply_rotary(x, inv, cu_seqlens=none), P.apply_rotary(x, inv))
    assert torch.equal(P.apply_rotary(x, inv, cu_seqlens=torch.tensor([0, 2, 5], device="cuda")),
                       P.apply_rotary(x, inv, cu_seqlens=torch.tensor([0, 2, 5], device="cuda", dtype=torch.int32)))
    for bad in (torch.tensor([0.0, 5.0], device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda"),
                torch.empty(0, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            P.apply_rotary(x, inv, cu_seqlens=bad)
    for kw in (dict(use_rotary_embed=True), {}):
        attn = P.PolyAttention(dim=64, heads=2, dim_head=64, causal=True, **kw).cuda()
        for n in (0, 3):
            y = attn(torch.randn(1, n, 64, device="cuda"), cu_seqlens=none, max_seqlen=longest)
            assert y.shape == (1, n, 64)


def test_strides_alignment_and_empty():
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(16)[0].cuda()
    base = torch.randn(2, 9, 3, 3, 33, device="cuda", dtype=torch.bfloat16)
    x = base[:, :, 1, :, 1:33].permute(0, 2, 1, 3)        # odd strides and an odd offset
    want, size = reference(x, angles(torch.arange(9).expand(2, 9), inv), 1.0, True)
    check(P.apply_rotary(x, inv), want, size, 1.0, torch.bfloat16)
    wide = torch.randn(2, 3, 9, 64, device="cuda")[..., ::2]   # features not contiguous
    want, size = reference(wide, angles(torch.arange(9).expand(2, 9), inv), 1.0, True)
    check(P.apply_rotary(wide, inv), want, size, 1.0, torch.float32)
    assert P.apply_rotary(torch.empty(2, 3, 0, 32, device="cuda"), inv).shape == (2, 3, 0, 32)
    assert P.apply_rotary(torch.empty(0, 3, 4, 32, device="cuda"), inv).shape == (0, 3, 4, 32)
    many = [torch.randn(1, 2, 4, 16, device="cuda") for _ in range(11)]   # more tensors than one launch takes
    for x, y in zip(many, P.apply_rotary(many, inv)):
        want, size = reference(x, angles(torch.arange(4)[None], inv), 1.0, True)
        check(y, want, size, 1.0, torch.float32)


def test_refusals():
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(16)[0].cuda()
    x = torch.randn(2, 3, 4, 16, device="cuda")
    bad = [(TypeError, dict(xs=x.double())), (TypeError, dict(xs=[x, x.half()])), (ValueError, dict(xs=[x, x[:1]])),
           (ValueError, dict(inv_freq=None)), (ValueError, dict(angles=torch.zeros(4, 8, device="cuda"))),
           (ValueError, dict(inv_freq=P.rotary_frequencies(32)[0].cuda())), (ValueError, dict(positions=torch.arange(5, device="cuda"))),
           (TypeError, dict(positions=torch.zeros(4, device="cuda"))), (RuntimeError, dict(positions=torch.arange(4))),
           (ValueError, dict(cu_seqlens=torch.tensor([0, 4], device="cuda", dtype=torch.int32))),
           (ValueError, dict(xs=torch.randn(2, 3, 4, 512, device="cuda"))),
           (NotImplementedError, dict(inv_freq=inv.clone().requires_grad_(True)))]
    for err, kw in bad:
        args = dict(xs=x, inv_freq=inv)
        args.update(kw)
        with pytest.raises(err):
            P.apply_rotary(args.pop("xs"), args.pop("inv_freq"), **args)


def test_dual_tensors_are_refused():
    import torch.autograd.forward_ad as fw

    import poly_attention_b200 as P
    inv = P.rotary_frequencies(16)[0].cuda()
    x = torch.randn(2, 3, 4, 16, device="cuda")
    with fw.dual_level():
        for xs in (fw.make_dual(x, x), [x, fw.make_dual(x, x)]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                P.apply_rotary(xs, inv)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            P.apply_rotary(x, fw.make_dual(inv, inv))
        P.apply_rotary(x, inv)


def test_stream_and_graph():
    import poly_attention_b200 as P
    inv = P.rotary_frequencies(64)[0].cuda()
    x = torch.randn(2, 4, 33, 64, device="cuda", dtype=torch.float16)
    pos = torch.arange(33, device="cuda")
    want = P.apply_rotary(x, inv, positions=pos + 7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = P.apply_rotary(x, inv, positions=pos + 7)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    p = pos.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = P.apply_rotary(x, inv, positions=p)
    p.add_(7)
    graph.replay()
    assert torch.equal(y, want)


@pytest.mark.parametrize("kind", ["order2", "order3"])
def test_modules_step_by_step_equals_parallel(kind):
    """use_rotary_embed: a causal prompt equals its tokens one by one over the cache
    (fp32: two orders of the same sums, and the 3xTF32 products: 1e-4)."""
    import poly_attention_b200 as P
    torch.manual_seed(0)
    kw = dict(dim=64, heads=4, kv_heads=2, dim_head=64, causal=True, use_rotary_embed=True)
    attn = (P.PolyAttention(**kw) if kind == "order2" else P.NPolyAttention(order=3, **kw)).cuda()
    x = torch.randn(2, 13, 64, device="cuda")
    plain = (P.PolyAttention(**{**kw, "use_rotary_embed": False}) if kind == "order2"
             else P.NPolyAttention(order=3, **{**kw, "use_rotary_embed": False})).cuda()
    plain.load_state_dict(attn.state_dict(), strict=False)
    with torch.no_grad():
        full = attn(x)
        _, cache = attn(x[:, :6], return_cache=True)
        rows = []
        for i in range(6, 13):
            y, cache = attn(x[:, i:i + 1], cache=cache, return_cache=True)
            rows.append(y)
        assert (torch.cat(rows, 1) - full[:, 6:]).abs().max() < 1e-4
        # positions matter
        assert (plain(x) - full).abs().max() > 1e-3


def test_module_given_angles_and_gradients():
    import poly_attention_b200 as P
    torch.manual_seed(0)
    attn = P.PolyAttention(dim=64, heads=2, dim_head=64, causal=True, use_rotary_embed=True).cuda()
    x = torch.randn(1, 20, 64, device="cuda", requires_grad=True)
    ang = (torch.arange(20, device="cuda")[:, None] * attn.rotary_emb.freqs).repeat_interleave(2, -1)
    want = attn(x)
    got = attn(x, rotary_pos_emb=ang)
    # the given angles are rounded to fp32 before the rotation (20 rad: 2^-20), else the same calls
    assert (got - want).abs().max() < 1e-4
    gw, = torch.autograd.grad(want.square().sum(), x)
    gg, = torch.autograd.grad(got.square().sum(), x)
    assert (gw - gg).abs().max() < 1e-3 * gw.abs().max()


def test_a_table_of_angles_serves_tensors_of_every_length():
    """Its last rows, as the last tokens of a sequence want them; one launch for the tensors of a length."""
    import poly_attention_b200 as P
    from poly_attention_b200 import _lib
    from poly_attention_b200.poly_attention import rotate_by_angles
    g = torch.Generator(device="cuda").manual_seed(4)
    table = torch.randn(13, 16, generator=g, device="cuda").repeat_interleave(2, -1)
    qs = [torch.randn(2, 3, n, 64, generator=g, device="cuda") for n in (5, 13, 1, 5, 13)]
    for t in (table, table.expand(2, 13, 32), table.expand(2, 1, 13, 32)):
        before = _lib.lib.poly_launch_count()
        ys = rotate_by_angles(t, qs)
        assert _lib.lib.poly_launch_count() == before + 3
        for q, y in zip(qs, ys):
            assert torch.equal(y, P.apply_rotary(q, angles=table[13 - q.shape[2]:, ::2].contiguous()))
    one, = rotate_by_angles(table[:1], qs[:1])
    assert torch.equal(one, P.apply_rotary(qs[0], angles=table[:1, ::2].expand(5, 16)))
    for bad in (table[:4], table[..., :31], table.expand(2, 3, 13, 32), table[0]):
        with pytest.raises(ValueError):
            rotate_by_angles(bad, qs[:1])


def test_pairs_of_two_angles_are_nan():
    from poly_attention_b200.poly_attention import rotate_by_angles
    half = torch.arange(1.0, 17.0, device="cuda").expand(5, 16).contiguous()
    q = torch.randn(2, 3, 5, 64, device="cuda")
    y, = rotate_by_angles(torch.cat((half, half), -1), [q])         # the half-and-half layout: no pair is equal
    assert y[..., :32].isnan().all() and torch.equal(y[..., 32:], q[..., 32:])


@pytest.mark.parametrize("order", [2, 3])
def test_given_angles_step_by_step(order):
    """Cached steps with the angles so far equal the parallel call (fp32: 1e-4, as test_modules_step_by_step_equals_parallel)."""
    import poly_attention_b200 as P
    torch.manual_seed(0)
    kw = dict(dim=64, heads=2, dim_head=64, causal=True)
    attn = (P.PolyAttention(**kw) if order == 2 else P.NPolyAttention(order=3, **kw)).cuda()
    x = torch.randn(1, 20, 64, device="cuda")
    ang = (torch.arange(20, device="cuda")[:, None] * P.rotary_frequencies(64)[0].cuda()).repeat_interleave(2, -1)
    with torch.no_grad():
        full = attn(x, rotary_pos_emb=ang)
        _, cache = attn(x[:, :7], rotary_pos_emb=ang[:7], return_cache=True)
        for i in range(7, 20):
            y, cache = attn(x[:, i:i + 1], rotary_pos_emb=ang[:i + 1], cache=cache, return_cache=True)
            assert (y[:, 0] - full[:, i]).abs().max() < 1e-4


def test_given_angles_with_contexts_of_other_lengths():
    import poly_attention_b200 as P
    torch.manual_seed(0)
    attn = P.PolyAttention(dim=64, heads=2, dim_head=64).cuda()
    x, c1, c2 = (torch.randn(1, n, 64, device="cuda") for n in (4, 9, 13))
    ang = torch.randn(13, 32, device="cuda").repeat_interleave(2, -1)
    y = attn(x, context=(c1, c2), rotary_pos_emb=ang)
    assert y.shape == x.shape and torch.isfinite(y).all()


def test_an_unfrozen_module_runs():
    import poly_attention_b200 as P
    attn = P.PolyAttention(dim=64, heads=2, dim_head=64, causal=True, use_rotary_embed=True).cuda().requires_grad_(True)
    attn(torch.randn(1, 5, 64, device="cuda")).square().sum().backward()
    assert all(p.grad is not None for p in attn.parameters())


def test_compile_and_opcheck():
    import poly_attention_b200 as P
    attn = P.PolyAttention(dim=64, heads=2, dim_head=64, causal=True, use_rotary_embed=True).cuda().bfloat16()
    x = torch.randn(1, 20, 64, device="cuda", dtype=torch.bfloat16)
    want = attn(x)
    got = torch.compile(attn, fullgraph=True)(x)
    assert (got - want).abs().max() < 2e-2
    xs = [torch.randn(1, 2, 6, 16, device="cuda", requires_grad=True)]
    inv = P.rotary_frequencies(16)[0].cuda()
    torch.library.opcheck(torch.ops.poly_b200.rotary, (xs, inv, None, 3, None, None, True, 1.0, False))
