"""Tree decoding without a GPU: the C entries' checks, the refusals, the ancestor search."""
import ctypes
import random

import pytest
import torch


def test_struct_sizes_and_checks():
    from poly_attention_b200 import _lib
    lib, err = _lib.lib, lambda: _lib.lib.poly_last_error().decode()
    assert lib.poly_sizeof_tree_pass() == ctypes.sizeof(_lib.PolyTreePass)
    assert lib.poly_sizeof_tree_append() == ctypes.sizeof(_lib.PolyTreeAppend)
    assert lib.poly_sizeof_tree_commit() == ctypes.sizeof(_lib.PolyTreeCommit)

    def args(**kw):
        a = _lib.PolyTreePass()
        a.batch, a.heads, a.kv_heads, a.nodes, a.head_dim, a.dtype, a.capacity, a.scale = 2, 4, 2, 8, 64, _lib.POLY_BF16, 20000, 0.1
        a.q = a.k = a.v = a.lengths = a.parents = 256
        for n in ("q", "k", "v"):
            st = getattr(a, n + "_stride")
            st[0], st[1], st[2] = 12800, 6400, 64
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, rc in ((dict(nodes=65), _lib.POLY_EINVAL), (dict(nodes=-1), _lib.POLY_EINVAL), (dict(heads=3), _lib.POLY_EINVAL),
                   (dict(heads=0), _lib.POLY_EINVAL), (dict(head_dim=160), _lib.POLY_EUNSUPPORTED), (dict(dtype=5), _lib.POLY_EINVAL),
                   (dict(capacity=-1), _lib.POLY_EINVAL), (dict(q=None), _lib.POLY_EINVAL), (dict(lengths=None), _lib.POLY_EINVAL),
                   (dict(parents=None), _lib.POLY_EINVAL), (dict(scale=float("nan")), _lib.POLY_EINVAL),
                   (dict(batch=40000), _lib.POLY_EUNSUPPORTED)):
        a = args(**kw)
        assert lib.poly_tree_chain(None, a, 1, None) == rc, kw
        assert lib.poly_tree_kernel_name(a) == b"invalid" and lib.poly_tree_workspace_size(a) == 0
    assert lib.poly_tree_kernel_name(args()) == b"tree"
    assert lib.poly_tree_kernel_name(args(dtype=_lib.POLY_F32)) == b"simt"
    assert lib.poly_tree_kernel_name(args(head_dim=96)) == b"simt"
    assert lib.poly_tree_kernel_name(args(k=258)) == b"simt"
    assert lib.poly_tree_kernel_name(args(nodes=17)) == b"tc100" and lib.poly_tree_kernel_name(args(nodes=17, q=264)) == b"tree"
    # the workspace does not depend on where q is
    assert lib.poly_tree_workspace_size(args(nodes=17)) == lib.poly_tree_workspace_size(args(nodes=17, q=264)) > 0
    need = lib.poly_tree_workspace_size(args())
    assert need > 0
    assert lib.poly_tree_chain(None, args(workspace=256, workspace_bytes=need - 1), 1, None) == _lib.POLY_EINVAL
    assert "workspace" in err()
    assert lib.poly_tree_chain(None, None, 1, None) == _lib.POLY_EINVAL
    assert lib.poly_tree_chain(None, None, -1, None) == _lib.POLY_EINVAL
    assert lib.poly_tree_chain(None, None, 0, None) == _lib.POLY_OK
    # nothing to do: no launch
    for kw in (dict(batch=0), dict(nodes=0), dict(capacity=0)):
        assert lib.poly_tree_chain(None, args(**kw), 1, None) == _lib.POLY_OK
    ap = _lib.PolyTreeAppend()
    ap.batch, ap.kv_heads, ap.nodes, ap.row_bytes, ap.capacity, ap.n = 1, 1, 4, 128, 10, 1
    assert lib.poly_tree_chain(ap, None, 0, None) == _lib.POLY_EINVAL           # no lengths
    ap.lengths = ap.parents = 256
    assert lib.poly_tree_chain(ap, None, 0, None) == _lib.POLY_EINVAL           # null tensor
    ap.n = 17
    assert lib.poly_tree_chain(ap, None, 0, None) == _lib.POLY_EINVAL
    ap.n, ap.row_bytes = 1, 127
    assert lib.poly_tree_chain(ap, None, 0, None) == _lib.POLY_EINVAL
    co = _lib.PolyTreeCommit()
    assert lib.poly_tree_commit(None, None) == _lib.POLY_EINVAL
    co.batch, co.kv_heads, co.nodes, co.capacity, co.n = 1, 1, 4, 10, 1
    assert lib.poly_tree_commit(co, None) == _lib.POLY_EINVAL
    co.lengths = co.path = co.count = 256
    assert lib.poly_tree_commit(co, None) == _lib.POLY_EINVAL                   # bad cache
    assert lib.poly_tree_positions(None, None, 0, 1, 4, None, 0, None) == _lib.POLY_EINVAL
    assert lib.poly_tree_positions(None, None, 0, 1, 65, None, 0, None) == _lib.POLY_EINVAL
    assert lib.poly_tree_positions(None, None, 0, 0, 4, None, 0, None) == _lib.POLY_OK


def test_counted_entries_check_like_the_plain_ones():
    from poly_attention_b200 import _lib
    lib = _lib.lib
    assert lib.poly_tree_chain_counted(None, None, 0, 256, None) == _lib.POLY_EINVAL     # nothing would write the count
    assert lib.poly_tree_chain_counted(None, None, 0, None, None) == _lib.POLY_OK
    assert lib.poly_tree_chain_counted(_lib.PolyTreeAppend(), None, 0, 256, None) == _lib.POLY_EINVAL
    assert lib.poly_tree_commit_counted(None, 256, None) == _lib.POLY_EINVAL
    assert lib.poly_tree_commit_counted(_lib.PolyTreeCommit(), 256, None) == _lib.POLY_EINVAL


@pytest.mark.parametrize("kw,err", [(dict(order=1), ValueError), (dict(heads=3), ValueError), (dict(max_nodes=0), ValueError),
                                    (dict(max_nodes=65), ValueError), (dict(order=5), ValueError), (dict(dtype=torch.float64), TypeError),
                                    (dict(dim_head=160), NotImplementedError)])
def test_decoder_refusals(kw, err):
    import poly_attention_b200 as P
    args = dict(batch=1, order=2, heads=4, kv_heads=2, dim_head=64, capacity=16, max_nodes=4, device="cpu")
    args.update(kw)
    with pytest.raises(err):
        P.TreeDecoder(**args)


def test_ancestor_search():
    """The pointer jumping of csrc/tree.cu restated, against walking up."""
    def jump(parents, room):
        n = 64
        up = [p if i < room and -1 <= p < i else -2 for i, p in enumerate(parents)] + [-2] * (n - len(parents))
        mask = [0 if up[i] == -2 else 1 << i for i in range(n)]
        for _ in range(6):
            m2, u2 = list(mask), list(up)
            for i in range(n):
                p = up[i]
                if p >= 0:
                    m2[i] = mask[i] | mask[p] if mask[p] else 0
                    u2[i] = up[p] if mask[p] else -2
            mask, up = m2, u2
        return mask

    def walk(parents, room):
        out = [0] * 64
        for i, p in enumerate(parents):
            ok = i < room and -1 <= p < i
            if ok and p >= 0:
                ok = out[p] != 0
            out[i] = (out[p] if p >= 0 else 0) | 1 << i if ok else 0
        return out

    rng = random.Random(0)
    for case in range(400):
        n = rng.randrange(1, 65)
        kind = case % 4
        parents = [i - 1 if kind == 0 else -1 if kind == 1 else rng.randrange(-1, i) if kind == 2 else rng.randrange(-2, max(i, 1) + 1)
                   for i in range(n)]
        if kind == 0 and rng.random() < 0.5:
            parents[rng.randrange(n)] = -2
        room = rng.choice([n, 64, rng.randrange(n + 1)])
        assert jump(parents, room) == walk(parents, room)
