"""Decoding over trees of drafted tokens: every level against 64 bits (tolerances:
pass_reference.py, on the rows that the level read), the step against decoding
token by token, commits, graphs, refusals."""
import random

import pytest
import torch

import pass_reference as R

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.float32).min


def tree(kind, n, rng):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] * n
    return [-1 if i == 0 else rng.randrange(-1, i) for i in range(n)]


def visible(parents):
    """Truth values [T, T] and which nodes are not padding."""
    n = len(parents)
    see = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parents):
        ok = -1 <= p < i and (p < 0 or bool(see[p, p]))
        if ok:
            see[i, i] = True
            if p >= 0:
                see[i] |= see[p]
    return see.cuda()


class Case:
    def __init__(self, *, order, h, g, d, dtype, lens, parents, cap=None, seed=0, clamp=None, max_nodes=None, stale=None):
        import poly_attention_b200 as P
        b, t = len(lens), len(parents[0])
        cap = cap or max(lens) + t
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
        self.lens, self.parents, self.clamp, self.d, self.dtype, self.order = lens, parents, clamp, d, dtype, order
        self.dec = P.TreeDecoder(batch=b, order=order, heads=h, kv_heads=g, dim_head=d, capacity=cap, max_nodes=max_nodes or t,
                                 dtype=dtype, softclamp_value=clamp)
        n = max(lens)
        rows = [rnd(b, g, n, d).to(dtype) for _ in range(3 * order - 2)]
        lses = [2 + rnd(b, g, n) for _ in range(order - 1)]
        self.dec.load(rows[:order], rows[order:2 * order - 1], lses, rows[2 * order - 1:], lens)
        if stale is not None:      # whatever lies behind the lengths
            for c in self.dec.keys + self.dec.vals + self.dec.msgs + self.dec.lses:
                for i, m in enumerate(lens):
                    c[i, :, m:] = stale
        self.q1 = rnd(b, h, t, d).to(dtype)
        self.nk = [rnd(b, g, t, d).to(dtype) for _ in range(order)]
        self.nv = [rnd(b, g, t, d).to(dtype) for _ in range(order - 1)]
        self.par = torch.tensor(parents, dtype=torch.int32, device="cuda")

    def step(self, **kw):
        return self.dec.step(self.q1, self.nk, self.nv, self.par, **kw)

    def check(self):
        dec, order, t = self.dec, self.order, self.q1.shape[2]
        out, msgs, lses = self.step(return_rows=True)
        for i, n in enumerate(self.lens):
            see = visible(self.parents[i])
            live = see.diagonal()
            end = n + t
            keep = torch.cat((torch.ones(t, n, dtype=torch.bool, device="cuda"), see), 1)
            for new, cache in zip(self.nk + self.nv, dec.keys + dec.vals):
                assert torch.equal(cache[i, :, n:end][:, live], new[i][:, live]) and (cache[i, :, n:end][:, ~live] == 0).all()
            for lvl in range(order - 1, -1, -1):
                at = order - 1 - lvl
                q = (self.q1 if lvl == 0 else self.nk[lvl - 1])[i].double()
                k = dec.keys[lvl][i, :, :end].double()
                if lvl == order - 1:
                    v = dec.vals[-1][i, :, :end].double()
                elif lvl:
                    v = (dec.vals[lvl - 1][i, :, :end] * dec.msgs[order - 2 - lvl][i, :, :end]).double()
                else:
                    v = dec.msgs[order - 2][i, :, :end].double()
                bias = None if lvl == order - 1 else dec.lses[order - 2 - lvl][i, :, :end].double()
                seen = keep
                if bias is not None:
                    dead = bias <= LOW / 2
                    assert torch.equal(dead, dead[:1].expand_as(dead))
                    seen = keep & ~dead[:1]
                    bias = bias.masked_fill(dead, 0.0)
                some = live & seen.any(1)
                (o, ot), (l, lt), _ = R.forward(q[:, some], k, v, bias, seen[some], self.d ** -0.5, self.clamp, self.dtype)
                what = f"level {lvl} sequence {i}"
                got = out[i] if lvl == 0 else msgs[at][i]
                R.assert_within(got[:, some], o, ot, "rows " + what)
                assert (got[:, ~some] == 0).all()
                if lvl:
                    R.assert_within(lses[at][i][:, some], l, lt, "lse " + what)
                    assert (lses[at][i][:, ~some] == LOW).all()
                    assert torch.equal(dec.msgs[at][i, :, n:end], msgs[at][i]) and torch.equal(dec.lses[at][i, :, n:end], lses[at][i])
        return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("order", [2, 3])
@pytest.mark.parametrize("h,g,d", [(4, 4, 64), (4, 1, 128), (6, 2, 64), (4, 2, 24), (32, 2, 128)])
@pytest.mark.parametrize("lens,nodes", [([0], 1), ([1, 5], 3), ([63, 64, 65, 0], 7), ([300, 17], 16), ([130, 700], 33), ([1000], 64)])
def test_step(lens, nodes, h, g, d, order, dtype):
    rng = random.Random(nodes)
    kinds = ["random", "chain", "star", "random"]
    Case(order=order, h=h, g=g, d=d, dtype=dtype, lens=lens, parents=[tree(kinds[i], nodes, rng) for i in range(len(lens))]).check()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 32)])
def test_order_four_and_softclamp(dtype, d):
    rng = random.Random(1)
    Case(order=4, h=4, g=2, d=d, dtype=dtype, lens=[100, 41], parents=[tree("random", 9, rng) for _ in range(2)]).check()
    Case(order=3, h=4, g=2, d=d, dtype=dtype, lens=[100, 41], parents=[tree("random", 9, rng) for _ in range(2)], clamp=3.0).check()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("order", [2, 3])
def test_padding_nodes_and_stale_rows(dtype, d, order):
    """Trees of different sizes in one call; NaN behind the lengths and in the padding's rows reaches nothing."""
    rng = random.Random(2)
    parents = [tree("random", 20, rng), tree("random", 20, rng), [-2] * 20, [-1, 0, -2, 1, 2, 4] + [-2] * 14, [3, 9] + [-2] * 18]
    for i in range(7, 20):
        parents[1][i] = -2
    c = Case(order=order, h=4, g=2, d=d, dtype=dtype, lens=[90, 128, 33, 0, 5], parents=parents, cap=200, stale=float("nan"))
    for i in range(5):
        live = visible(parents[i]).diagonal()
        for x in [c.q1] + c.nk + c.nv:
            x[i][:, ~live] = float("nan")
    out = c.check()
    assert torch.isfinite(out).all()


def test_dead_cached_keys():
    for dtype, d in ((torch.bfloat16, 64), (torch.float32, 40)):
        c = Case(order=3, h=4, g=2, d=d, dtype=dtype, lens=[70, 12], parents=[[-1, 0, 0], [-1, 0, -2]])
        for x in c.dec.lses:
            x[0, :, :33] = LOW
            x[1, :, :12] = float("-inf")
        c.check()


def test_many_splits_and_groups():
    """One sequence over many key ranges, and more groups than fit at once (no split)."""
    rng = random.Random(3)
    Case(order=2, h=8, g=2, d=128, dtype=torch.bfloat16, lens=[5003], parents=[tree("random", 5, rng)]).check()
    Case(order=2, h=8, g=2, d=128, dtype=torch.bfloat16, lens=[5003, 4000], parents=[tree("random", 60, rng) for _ in range(2)]).check()
    Case(order=3, h=4, g=4, d=64, dtype=torch.float16, lens=[2100], parents=[tree("random", 50, rng)], max_nodes=64).check()
    Case(order=2, h=2, g=2, d=64, dtype=torch.float16, lens=[rng.randrange(200) for _ in range(170)],
         parents=[tree("random", 4, rng) for _ in range(170)], cap=1000).check()


def test_strides_and_shared_tree():
    rng = random.Random(4)
    shared = tree("random", 8, rng)
    c = Case(order=2, h=4, g=2, d=64, dtype=torch.bfloat16, lens=[50, 77], parents=[shared, shared])
    want = c.step().clone()
    one = c.dec.step(c.q1, c.nk, c.nv, torch.tensor(shared, dtype=torch.int32, device="cuda"))
    assert torch.equal(one, want)
    token_major = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)   # noqa: E731
    assert torch.equal(c.dec.step(token_major(c.q1), [token_major(t) for t in c.nk], [token_major(t) for t in c.nv], c.par), want)
    spread = lambda t: torch.stack((t, t), -1).flatten(-2)[..., ::2]   # noqa: E731
    assert torch.equal(c.dec.step(spread(c.q1), [spread(t) for t in c.nk], [spread(t) for t in c.nv], c.par), want)

    def odd(t):     # an address that is a multiple of 2 bytes only
        buf = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)
    got = c.dec.step(odd(c.q1), [odd(t) for t in c.nk], [odd(t) for t in c.nv], c.par)
    # other kernels, the same roundings of 16-bit operands: two steps of the type
    assert ((got - want).abs() <= 2 * torch.finfo(torch.bfloat16).eps * want.abs() + 4e-3).all()


@pytest.mark.parametrize("order", [2, 3])
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
def test_a_path_of_the_tree_is_decoding_token_by_token(order, dtype, tol):
    """Every node's output is that of ChainDecoder fed its path (the framework's bars: fp32 1e-4, bf16 2e-2 + 1e-2 |x|)."""
    from poly_attention_b200.decode import ChainDecoder
    n = 37
    parents = [-1, 0, 0, 1, 3, 2]
    c = Case(order=order, h=4, g=2, d=64, dtype=dtype, lens=[n], parents=[parents])
    dec = c.dec
    keep = [x[:, :, :n].clone() for x in dec.keys + dec.vals + dec.lses + dec.msgs]
    out = c.step()
    for leaf in (4, 5):
        path, p = [], leaf
        while p >= 0:
            path.insert(0, p)
            p = parents[p]
        cd = ChainDecoder(batch=1, order=order, heads=4, kv_heads=2, dim_head=64, capacity=n + 8, dtype=dtype)
        for dst, src in zip(cd.qs + cd.vs + cd.lses + cd.msgs, keep):
            dst[:, :, :n] = src
        cd.length = n
        for node in path:
            at = slice(node, node + 1)
            cd.append_kv([t[:, :, at] for t in c.nk], [t[:, :, at] for t in c.nv])
            y = cd.step(c.q1[:, :, at])
            assert ((out[:, :, at] - y).abs() <= tol + (1e-2 if dtype != torch.float32 else 0) * y.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_commit(dtype):
    rng = random.Random(5)
    lens = [20, 0, 64, 9]
    parents = [tree("random", 12, rng) for _ in lens]
    c = Case(order=3, h=4, g=2, d=64, dtype=dtype, lens=lens, parents=parents, cap=100)
    c.step()
    caches = c.dec.keys + c.dec.vals + c.dec.msgs + c.dec.lses
    before = [x.clone() for x in caches]
    paths = []
    for p in parents:
        node, path = rng.randrange(12), []
        while node >= 0:
            path.insert(0, node)
            node = p[node]
        paths.append(path)
    paths[3] = []
    path = torch.full((4, 12), 99, dtype=torch.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    c.dec.commit(path.cuda(), torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda"))
    assert c.dec.lengths.tolist() == [n + len(p) for n, p in zip(lens, paths)]
    for x, old in zip(caches, before):
        for i, (n, p) in enumerate(zip(lens, paths)):
            assert torch.equal(x[i, :, :n], old[i, :, :n])
            assert torch.equal(x[i, :, n:n + len(p)], old[i, :, [n + j for j in p]])
    # the next step continues from the kept rows
    c.lens = c.dec.lengths.tolist()
    c.check()


def test_commit_of_bad_paths_stays_inside():
    c = Case(order=2, h=2, g=2, d=64, dtype=torch.bfloat16, lens=[5, 96], parents=[[-1, 0, 1]] * 2, cap=99)
    c.step()
    rest = [x[0, :, 8:].clone() for x in c.dec.keys]
    c.dec.commit(torch.tensor([[2, 0, -7], [1 << 30, 2, 2]], dtype=torch.int32, device="cuda"),
                 torch.tensor([1 << 30, 50], dtype=torch.int32, device="cuda"))
    assert c.dec.lengths.tolist() == [8, 99]
    for x, r in zip(c.dec.keys, rest):
        assert torch.equal(x[0, :, 8:], r)
    with pytest.raises(ValueError, match="since the last commit"):
        c.dec.commit(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.tensor([1, 1], dtype=torch.int32, device="cuda"))
    c.dec.lengths.fill_(5)
    c.dec.refresh()
    c.step()
    c.dec.commit(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.tensor([-3, 3], dtype=torch.int32, device="cuda"))
    assert c.dec.lengths.tolist() == [5, 6]


def test_full_cache():
    c = Case(order=2, h=2, g=2, d=64, dtype=torch.bfloat16, lens=[10, 4], parents=[[-1, 0, 1]] * 2, cap=13)
    c.check()
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    c.dec.commit(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), one)
    with pytest.raises(ValueError, match="capacity"):
        c.step()
    c.dec.lengths.fill_(3)
    c.dec.refresh()
    c.lens = [3, 3]
    c.check()
    # past the host's check (lengths changed on the device, as in a replayed graph): nodes without room are padding
    guard = [x[1].clone() for x in c.dec.keys]
    c.dec.lengths.copy_(torch.tensor([12, 1 << 30], dtype=torch.int32))
    out = c.step()
    assert (out[0, :, 1:] == 0).all() and (out[0, :, 0] != 0).any() and (out[1] == 0).all()
    for x, old in zip(c.dec.keys, guard):
        assert torch.equal(x[1], old)
    c.dec.lengths.fill_(-5)
    c.dec.refresh()
    c.lens = [0, 0]
    c.check()


def test_positions():
    c = Case(order=2, h=2, g=2, d=64, dtype=torch.bfloat16, lens=[10, 4], parents=[[-1, 0, 1, 0], [-1, -1, -2, 2]], cap=50)
    assert c.dec.positions(c.par).tolist() == [[10, 11, 12, 11], [4, 4, 4, 4]]


def test_graph_replays_follow_the_lengths():
    rng = random.Random(6)
    lens = [100, 30]
    c = Case(order=3, h=4, g=2, d=64, dtype=torch.bfloat16, lens=lens, parents=[tree("random", 6, rng) for _ in lens], cap=400)
    other = Case(order=3, h=4, g=2, d=64, dtype=torch.bfloat16, lens=lens, parents=c.parents, cap=400)
    path = torch.tensor([[0, 3, 5, 0], [1, 2, 4, 0]], dtype=torch.int32, device="cuda")
    count = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    c.step()          # before capture: first-launch settings
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.step()
        c.dec.commit(path, count)
    assert c.dec.lengths.tolist() == lens
    for it in range(5):
        for x, y in zip([c.q1] + c.nk + c.nv, [other.q1] + other.nk + other.nv):
            x.copy_(torch.randn(x.shape, device="cuda"))
            y.copy_(x)
        graph.replay()
        want = other.step()
        other.dec.commit(path, count)
        assert torch.equal(out, want)
    assert c.dec.lengths.tolist() == [115, 40]
    # after replays the host looks the lengths up again before an eager step
    c.dec.lengths.fill_(396)
    with pytest.raises(ValueError, match="capacity"):
        c.step()
    c.dec.lengths.copy_(torch.tensor([115, 40], dtype=torch.int32))
    for x, y in zip(c.dec.keys + c.dec.msgs + c.dec.lses, other.dec.keys + other.dec.msgs + other.dec.lses):
        assert torch.equal(x[0, :, :115], y[0, :, :115]) and torch.equal(x[1, :, :40], y[1, :, :40])


@pytest.mark.parametrize("h,g,d,nodes,longest,dtype", [
    (4, 4, 64, 5, 300, torch.bfloat16), (16, 4, 128, 16, 300, torch.bfloat16), (8, 2, 128, 60, 9000, torch.float16), (4, 2, 64, 6, 40000, torch.bfloat16),
    (32, 2, 64, 20, 100, torch.float16), (4, 2, 24, 5, 100, torch.float32), (4, 2, 64, 5, 100, torch.float32)])
@pytest.mark.parametrize("part", ["row", "feature"])
def test_nan_of_a_query_stays_and_stays_its_own(h, g, d, nodes, longest, dtype, part):
    rng = random.Random(3)
    c = Case(order=2, h=h, g=g, d=d, dtype=dtype, lens=[longest, 3], parents=[tree("random", nodes, rng)] * 2, cap=longest + nodes)
    want = c.step().clone()
    c.q1[0, 1, nodes - 1, slice(None) if part == "row" else slice(3, 4)] = float("nan")
    out, msgs, lses = c.step(return_rows=True)
    assert out[0, 1, nodes - 1].isnan().all()
    out[0, 1, nodes - 1] = want[0, 1, nodes - 1]
    assert torch.equal(out, want)
    c.nk[0][0, 0, nodes - 1] = float("nan")      # the last node's query of the top level
    out, msgs, lses = c.step(return_rows=True)
    assert lses[0][0, 0, nodes - 1].isnan() and msgs[0][0, 0, nodes - 1].isnan().all() and lses[0].isnan().sum() == 1
    assert out[0, 0, nodes - 1].isnan().all()


@pytest.mark.parametrize("h,g,d,nodes,longest", [
    (16, 4, 128, 16, 300), (8, 2, 128, 60, 9000), (4, 4, 64, 40, 90), (32, 2, 64, 20, 100), (4, 2, 64, 33, 2000), (4, 4, 64, 5, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nan_of_a_query_survives_the_softclamp(h, g, d, nodes, longest, dtype):
    rng = random.Random(3)
    c = Case(order=2, h=h, g=g, d=d, dtype=dtype, lens=[longest, 3], parents=[tree("random", nodes, rng)] * 2, cap=longest + nodes,
             clamp=4.0)
    want, _, lses = c.step(return_rows=True)
    want, lse = want.clone(), lses[0].clone()
    c.q1[0, 1, nodes - 1, 3] = float("nan")
    c.nk[0][1, 0, nodes - 1, 3] = float("nan")     # the last node's query of the top level, of the other sequence
    out, _, lses = c.step(return_rows=True)
    assert out[0, 1, nodes - 1].isnan().all() and lses[0][1, 0, nodes - 1].isnan()
    out[0, 1, nodes - 1], lses[0][1, 0, nodes - 1] = want[0, 1, nodes - 1], lse[1, 0, nodes - 1]
    assert torch.equal(out[0], want[0]) and torch.equal(lses[0], lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,g,nodes,lens", [
    (4, 4, 40, [300, 17]), (4, 2, 33, [4000]), (16, 4, 16, [130, 0, 700]), (32, 2, 20, [100, 2500]), (6, 2, 64, [77]),
    (2, 2, 36, [50 + i for i in range(80)])])
def test_softclamp_with_many_rows_a_key(h, g, nodes, lens, d, dtype):
    """The tcgen05 kernel's own tanh, with bias and dead keys: one and two row tiles, one and several key ranges."""
    from poly_attention_b200 import _lib
    rng = random.Random(nodes)
    c = Case(order=2, h=h, g=g, d=d, dtype=dtype, lens=lens, parents=[tree("random", nodes, rng) for _ in lens], clamp=3.0)
    for x in c.dec.lses:
        x[0, :, :lens[0] // 3] = LOW
    c.check()
    assert _lib.lib.poly_tree_kernel_name(c.dec._passes[1]) == b"tc100"


def test_commits_between_replays_of_a_captured_step():
    lens, parents = [40, 7], [[-1, 0, 1, 1]] * 2
    c, other = (Case(order=2, h=4, g=2, d=64, dtype=torch.bfloat16, lens=lens, parents=parents, cap=100) for _ in range(2))
    c.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.step()
    path = torch.tensor([[0, 1, 3], [0, 1, 2]], dtype=torch.int32, device="cuda")
    count = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    for _ in range(4):     # the host sees no step between these commits
        graph.replay()
        assert torch.equal(out, other.step())
        c.dec.commit(path, count)
        other.dec.commit(path, count)
    assert c.dec.lengths.tolist() == other.dec.lengths.tolist() == [52, 15]
    for x, y in zip(c.dec.keys + c.dec.msgs, other.dec.keys + other.dec.msgs):
        assert torch.equal(x[0, :, :52], y[0, :, :52]) and torch.equal(x[1, :, :15], y[1, :, :15])


def test_dual_tensors_are_refused():
    import torch.autograd.forward_ad as fw
    c = Case(order=2, h=2, g=2, d=64, dtype=torch.bfloat16, lens=[3], parents=[[-1]])
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            c.dec.step(fw.make_dual(c.q1, c.q1), c.nk, c.nv, c.par)
    c.check()


def test_a_commit_keeps_nodes_of_the_last_step_only():
    """Captured, replayed and eager steps of different sizes: what follows each is held to its nodes."""
    c = Case(order=2, h=4, g=2, d=64, dtype=torch.bfloat16, lens=[40, 7], parents=[[-1, 0, 1, 1, 2, 4]] * 2, cap=200)
    dec = c.dec
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    two = lambda t: t[:, :, :2].contiguous()   # noqa: E731
    path = i32([[0, 1, 2, 3, 4, 5], [1, 5, 5, 5, 5, 5]])
    c.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step()
    small = [two(c.q1), [two(t) for t in c.nk], [two(t) for t in c.nv], i32([-1, 0])]
    graph.replay()
    dec.step(*small)                      # fewer nodes than the captured step
    rows = [x[1, :, 8].clone() for x in dec.keys]
    dec.commit(path, i32([6, 6]))
    assert dec.lengths.tolist() == [42, 9]
    for x, row in zip(dec.keys, rows):    # entries 1 and (past the nodes) 5 are both the last node
        assert torch.equal(x[1, :, 7], row) and torch.equal(x[1, :, 8], row)
    dec.commit(path, i32([6, 6]))         # no step since
    assert dec.lengths.tolist() == [42, 9]
    dec.step(*small)
    graph.replay()                        # the last step, not seen by the host
    dec.commit(path, i32([5, 3]))
    assert dec.lengths.tolist() == [47, 12]
    graph.replay()
    n = 3
    dec.load([x[:, :, :n] for x in dec.keys], [x[:, :, :n] for x in dec.vals], [x[:, :, :n] for x in dec.lses],
             [x[:, :, :n] for x in dec.msgs], [3, 1])
    dec.commit(path, i32([2, 2]))         # a load drops the step's rows
    assert dec.lengths.tolist() == [3, 1]


def test_packed_prompts_of_no_tokens():
    import poly_attention_b200 as P
    dec = P.TreeDecoder(batch=2, order=2, heads=2, kv_heads=2, dim_head=64, capacity=10, max_nodes=4)
    none = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    dec.load_packed([none] * 2, [none], [torch.empty(2, 0, device="cuda")], [none], torch.zeros(3, dtype=torch.int32, device="cuda"), 0)
    assert dec.lengths.tolist() == [0, 0]


def test_a_refused_load_changes_nothing():
    c = Case(order=2, h=2, g=2, d=64, dtype=torch.bfloat16, lens=[5], parents=[[-1]], cap=20)
    caches = c.dec.keys + c.dec.vals + c.dec.lses + c.dec.msgs
    before = [x.clone() for x in caches]
    rows, lse = torch.zeros(1, 2, 10, 64, device="cuda"), torch.zeros(1, 2, 10, device="cuda")
    for bad in (([rows] * 2, [rows], [lse], [rows[..., :32]], [7]), ([rows] * 2, [rows], [lse], [lse], [7]),
                ([rows, rows[:, :, :6]], [rows], [lse], [rows], [7])):
        with pytest.raises(ValueError):
            c.dec.load(*bad)
        assert all(torch.equal(x, y) for x, y in zip(caches, before)) and c.dec.lengths.tolist() == [5]
    for lens in ([6.5], torch.tensor([True])):
        with pytest.raises(TypeError, match="integers"):
            c.dec.load([rows] * 2, [rows], [lse], [rows], lens)
        assert c.dec.lengths.tolist() == [5]
    c.check()


def test_a_decoder_of_no_sequences():
    import poly_attention_b200 as P
    none, longest = P.packed_offsets([])
    attn = P.PolyAttention(dim=64, heads=2, dim_head=64, causal=True, use_rotary_embed=True).cuda()
    y, dec = attn.tree_prefill(torch.randn(1, 0, 64, device="cuda"), none, max_seqlen=longest, capacity=8, max_nodes=2)
    parents = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    assert y.shape == (1, 0, 64)
    assert attn.tree_step(torch.randn(0, 2, 64, device="cuda"), dec, parents).shape == (0, 2, 64)
    dec.commit(parents, torch.empty(0, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="since the last commit"):
        dec.commit(parents, torch.empty(0, dtype=torch.int32, device="cuda"))
    row = torch.randn(0, 2, 2, 64, device="cuda")
    out, msgs, lses = dec.step(row, [row] * 2, [row], parents, return_rows=True)
    assert out.shape == msgs[0].shape == (0, 2, 2, 64) and lses[0].shape == (0, 2, 2)


def test_two_decoders_on_two_streams():
    rng = random.Random(7)
    cases = [Case(order=3, h=8, g=2, d=128, dtype=torch.bfloat16, lens=[3000 + i, 500], parents=[tree("random", 10, rng)] * 2, seed=i)
             for i in range(2)]
    want = [c.step().clone() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(3):
        got = []
        for c, s in zip(cases, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(c.step())
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals():
    c = Case(order=2, h=4, g=2, d=64, dtype=torch.bfloat16, lens=[10, 4], parents=[[-1, 0, 1]] * 2, cap=50)
    q, nk, nv, par = c.q1, c.nk, c.nv, c.par
    wide = torch.randn(2, 4, 9, 64, device="cuda").bfloat16()
    for err, args in ((ValueError, (q[0], nk, nv, par)), (ValueError, (wide, nk, nv, par)), (ValueError, (q, nk[:1], nv, par)),
                      (ValueError, (q, nk, [nv[0][:, :1]], par)), (TypeError, (q.float(), nk, nv, par)), (TypeError, (q, [nk[0].half(), nk[1]], nv, par)),
                      (TypeError, (q, nk, nv, par.long())), (ValueError, (q, nk, nv, par[:, :2])), (RuntimeError, (q, nk, nv, par.cpu())),
                      (RuntimeError, (q.cpu(), nk, nv, par))):
        with pytest.raises(err):
            c.dec.step(*args)
    with pytest.raises(ValueError):
        c.dec.step(q, nk, nv, par, out=torch.empty(2, 4, 3, 32, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="nothing to commit"):
        Case(order=2, h=2, g=2, d=64, dtype=torch.bfloat16, lens=[3], parents=[[-1]]).dec.commit(par[:1], torch.ones(1, dtype=torch.int32, device="cuda"))
    c.step()
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    for err, args in ((TypeError, (par.long(), one)), (ValueError, (par[:1], one)), (ValueError, (par, one[:1])), (RuntimeError, (par.cpu(), one))):
        with pytest.raises(err):
            c.dec.commit(*args)
    rows = [torch.zeros(2, 2, 20, 64, device="cuda")] * 2
    for lens in ([21, 0], [-1, 0], [3]):
        with pytest.raises(ValueError):
            c.dec.load(rows, rows[:1], [torch.zeros(2, 2, 20, device="cuda")], rows[:1], lens)
