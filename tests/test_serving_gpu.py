"""The packed, rotary and tree operators as a model uses them together: a packed
prompt batch through a module fills a decoder, drafted trees run through it,
accepted paths are kept; against the module on the sequences one by one."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(kind, rotary, dtype, **kw):
    import poly_attention_b200 as P
    torch.manual_seed(0)
    args = dict(dim=64, heads=4, kv_heads=2, dim_head=64, causal=True, use_rotary_embed=rotary, **kw)
    attn = P.PolyAttention(**args) if kind == 2 else P.NPolyAttention(order=kind, **args)
    return attn.cuda().to(dtype)


@pytest.mark.parametrize("kind", [2, 3])
@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("kw", [{}, dict(prenorm=True, attn_gate=True, multiply_root_value=True, softclamp_value=4.0),
                                dict(shared_kv=True, prenorm=True, separate_context_norms=True)])
def test_prompt_drafts_commit(kind, rotary, dtype, tol, kw):
    """fp32: two orders of the same sums through the layer, about 2^-20 a product (2e-4 of values of size 1);
    bf16: the modules' bar of 2e-2 + 1e-2 |x| for one layer, on both sides of the comparison 3e-2."""
    import poly_attention_b200 as P
    attn = build(kind, rotary, dtype, **kw)
    rng = random.Random(kind)
    lens = [17, 1, 130]
    cu, longest = P.packed_offsets(lens)
    tokens = [torch.randn(n, 64, device="cuda").to(dtype) for n in lens]
    y, dec = attn.tree_prefill(torch.cat(tokens)[None], cu, max_seqlen=longest, capacity=longest + 30, max_nodes=8)
    at = 0
    with torch.no_grad():
        for t in tokens:
            want = attn(t[None])[0]
            assert ((y[0, at:at + len(t)] - want).abs() <= tol + tol / 2 * want.abs()).all()
            at += len(t)
        for step in range(3):
            nodes = [5, 8, 1][step]
            parents = [[-1 if i == 0 else rng.randrange(-1, i) for i in range(nodes)] for _ in lens]
            x = torch.randn(3, nodes, 64, device="cuda").to(dtype)
            y = attn.tree_step(x, dec, torch.tensor(parents, dtype=torch.int32, device="cuda"))
            path = torch.zeros(3, nodes, dtype=torch.int32)
            count = []
            for s, par in enumerate(parents):
                # the whole sequence to a node in one go, for every node
                for node in range(nodes):
                    line, p = [], node
                    while p >= 0:
                        line.insert(0, p)
                        p = par[p]
                    full = torch.cat((tokens[s], x[s, line]))
                    want = attn(full[None])[0, -1]
                    assert ((y[s, node] - want).abs() <= tol + tol / 2 * want.abs()).all(), (step, s, node)
                keep = line if s != 1 else []
                path[s, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
                count.append(len(keep))
                tokens[s] = torch.cat((tokens[s], x[s, keep]))
            dec.commit(path.cuda(), torch.tensor(count, dtype=torch.int32, device="cuda"))
            assert dec.lengths.tolist() == [len(t) for t in tokens]


def test_a_bound_above_the_capacity():
    """max_seqlen is a bound: the prompts have to fit the cache, it does not."""
    import poly_attention_b200 as P
    attn = build(2, False, torch.float32)
    cu, _ = P.packed_offsets([5, 16])
    x = torch.randn(1, 21, 64, device="cuda")
    y, dec = attn.tree_prefill(x, cu, max_seqlen=4096, capacity=16, max_nodes=2)
    want, other = attn.tree_prefill(x, cu, max_seqlen=16, capacity=16, max_nodes=2)
    assert dec.lengths.tolist() == [5, 16]
    assert (y - want).abs().max() < 1e-4      # (another kernel: fp32, 3xTF32 products)
    for a, b in zip(dec.keys + dec.vals, other.keys + other.vals):
        assert torch.equal(a[0, :, :5], b[0, :, :5]) and torch.equal(a[1], b[1])
    for bound, cap in ((4096, 15), (15, 20)):     # a sequence that does not fit, a bound that is none
        with pytest.raises(ValueError, match="do not fit"):
            attn.tree_prefill(x, cu, max_seqlen=bound, capacity=cap, max_nodes=2)


def test_host_threads_at_once():
    """Several host threads, a stream each, through all three operators: every one gets the single thread's results."""
    import threading

    import poly_attention_b200 as P
    attn = build(2, True, torch.bfloat16)
    cu, longest = P.packed_offsets([30, 200])
    x, drafts = (torch.randn(*s, 64, device="cuda").bfloat16() for s in ((1, 230), (2, 3)))
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device="cuda")

    def work(out):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                y, dec = attn.tree_prefill(x, cu, max_seqlen=longest, capacity=210, max_nodes=3)
                out.append((y, attn.tree_step(drafts, dec, parents)))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    results = [[] for _ in range(5)]
    work(results[0])
    threads = [threading.Thread(target=work, args=(r,)) for r in results[1:]]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in results:
        assert len(r) == 5 and all(torch.equal(a, b) for pair in r for a, b in zip(pair, results[0][0]))


def test_training_step_of_packed_rotary_module():
    """Gradients of a packed layer with positions are those of its sequences one by one (fp32, 1e-4 of the largest)."""
    import poly_attention_b200 as P
    attn = build(3, True, torch.float32, prenorm=True)
    lens = [30, 70, 0, 5]
    cu, longest = P.packed_offsets(lens)
    x = torch.randn(1, sum(lens), 64, device="cuda")
    params = [p for p in attn.parameters() if p.requires_grad]
    w = torch.randn_like(x)
    ga = torch.autograd.grad((attn(x, cu_seqlens=cu, max_seqlen=longest) * w).sum(), params)
    total, at = 0.0, 0
    for n in lens:
        if n:
            total = total + (attn(x[:, at:at + n]) * w[:, at:at + n]).sum()
        at += n
    gb = torch.autograd.grad(total, params)
    for a, b in zip(ga, gb):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max() + 1e-6


def test_a_captured_step_serves_growing_sequences():
    import poly_attention_b200 as P
    attn = build(2, True, torch.bfloat16)
    lens = [40, 9]
    cu, longest = P.packed_offsets(lens)
    prompt = torch.randn(1, sum(lens), 64, device="cuda").bfloat16()
    decs = [attn.tree_prefill(prompt, cu, max_seqlen=longest, capacity=200, max_nodes=4)[1] for _ in range(2)]
    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    x = torch.randn(2, 4, 64, device="cuda").bfloat16()
    path = torch.tensor([[0, 1, 3, 0], [0, 2, 0, 0]], dtype=torch.int32, device="cuda")
    count = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    attn.tree_step(x, decs[0], parents)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = attn.tree_step(x, decs[0], parents)
        decs[0].commit(path, count)
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        graph.replay()
        want = attn.tree_step(x, decs[1], parents)
        decs[1].commit(path, count)
        assert torch.equal(y, want)
    assert decs[0].lengths.tolist() == [52, 17]


def test_a_captured_training_step():
    """Forward and backward of the packed chain with positions in one graph; the replay gives the eager gradients.
    (No eager graph of the same leaves may live during the capture: torch's engine then joins the streams of both,
    which ends a capture of any operator's backward, plain products included.)"""
    import poly_attention_b200 as P
    lens = [60, 140]
    cu, longest = P.packed_offsets(lens)
    inv = P.rotary_frequencies(64)[0].cuda()
    leaves = [torch.randn(200, 2, 64, device="cuda").bfloat16().requires_grad_(True) for _ in range(4)]
    do = torch.randn(200, 2, 64, device="cuda").bfloat16()

    def step():
        qs = P.apply_rotary(leaves[:3], inv, cu_seqlens=cu)
        out = P.poly_attention_order2_packed(*qs, leaves[3], cu, causal=True, max_seqlen=longest)[0]
        return out, torch.autograd.grad(out, leaves, do)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out, grads = step()
    graph.replay()
    torch.cuda.synchronize()
    want, wg = step()
    assert torch.equal(out, want)
    for a, b in zip(grads, wg):
        # dq sums its key tiles in 32 bits in any order: one step of the type
        assert ((a - b).abs().float() <= 2 * torch.finfo(torch.bfloat16).eps * b.abs().float() + 1e-3).all()
