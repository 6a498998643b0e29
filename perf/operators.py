"""Timing cases for the packed-sequence, rotary and tree-decoding operators.

``listed()`` and ``draw()`` give cases, ``prepare()`` makes a case's inputs on
the GPU, ``run()`` makes one pass: through the framework's public calls when
``own`` is true, else through elementary torch operations in 32 bits (the plain
form). ``exact()`` restates the operators in 64 bits and ``work()`` counts the
bytes and operations that a pass cannot do without.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "poly-attention_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import poly_attention_b200
    return poly_attention_b200


# ---------------------------------------------------------------------------
# cases

def _packed(name, **kw):
    c = dict(op="packed", order=2, dtype="bf16", heads=16, kv_heads=16, dim=64, causal=True, softclamp=0.0,
             backward=False, seqs=8, total=1024, spread=0.8, layout=1)
    c.update(kw, name=name)
    return c


def _rotary(name, **kw):
    c = dict(op="rotary", dtype="bf16", batch=8, heads=16, kv_heads=16, keys=2, length=1024, dim=64, rot=64,
             interleaved=True, scaling="none", start=0, ragged=False, backward=False)
    c.update(kw, name=name)
    return c


def _tree(name, **kw):
    c = dict(op="tree", order=2, dtype="bf16", batch=4, heads=16, kv_heads=4, dim=128, nodes=8, longest=2048,
             softclamp=0.0, layout=1)
    c.update(kw, name=name)
    return c


def listed():
    return [
        # a few very short requests answered at once: the call's latency
        _packed("packed_tiny", heads=4, kv_heads=4, seqs=3, total=37, layout=3),
        # images of different sizes cut into patches, both directions: many short sequences, no causal mask
        _packed("packed_images", dtype="fp16", causal=False, backward=True, seqs=256, total=14001, spread=0.25, layout=5),
        # a training step on documents of unequal lengths packed into one row
        _packed("packed_train", backward=True, seqs=12, total=16411, layout=7),
        # the same for the order-3 chain at its decoding head shape (grouped heads of 128)
        _packed("packed_train_chain", order=3, kv_heads=4, dim=128, backward=True, seqs=9, total=12289, layout=11),
        # a prompt batch with one long request among short ones
        _packed("packed_prompt", dtype="fp16", seqs=6, total=32768, spread=1.0, layout=19),
        # a full-precision evaluation of packed sequences
        _packed("packed_fp32", dtype="fp32", heads=8, kv_heads=8, seqs=7, total=4099, layout=17),
        # positions of one new token of each sequence of a decoding batch: latency
        _rotary("rotary_step", batch=32, kv_heads=4, keys=3, length=1, dim=128, rot=128, start=2049, ragged=True),
        # queries and keys of a training batch, both directions
        _rotary("rotary_train", length=4096, backward=True),
        # a long prompt far into the context: half layout on part of the head, frequencies scaled for it
        _rotary("rotary_long", dtype="fp16", batch=1, kv_heads=4, keys=2, length=32768, dim=128, rot=64,
                interleaved=False, scaling="yarn", start=98304),
        # one sequence, a short chain of drafted tokens: latency
        _tree("tree_one", batch=1, nodes=6, longest=1021, layout=3),
        # a serving batch of the order-3 chain, a tree of 16 nodes each
        _tree("tree_batch", order=3, batch=32, nodes=16, longest=2304, layout=5),
        # few long sequences with wide trees
        _tree("tree_long", dtype="fp16", batch=4, nodes=60, longest=40001, layout=7),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_packed(rng):
    while True:
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
        backward = dtype != "fp32" and rng.random() < 0.6
        dim = 64 if dtype == "fp32" else rng.choice([64, 64, 128])
        heads = rng.choice([4, 8, 16])
        total = _log_int(rng, 33, 4200 if dtype == "fp32" else (17000 if backward else 33000))
        c = _packed("", order=rng.choice([2, 2, 3]), dtype=dtype, heads=heads, dim=dim,
                    kv_heads=rng.choice([heads, heads // 2, heads // 4]), causal=rng.random() < 0.7,
                    softclamp=rng.choice([0.0, 0.0, 0.0, 20.0]), backward=backward,
                    seqs=_log_int(rng, 1, max(1, min(300, total // 8))), total=total,
                    spread=rng.uniform(0.2, 1.4), layout=rng.randrange(1 << 30))
        scores = c["heads"] * sum(n * n for n in _lengths(c)) * c["order"]
        if scores <= (4.5e9 if backward else 2.0e10 if dtype != "fp32" else 4e8):
            return c


def _draw_rotary(rng):
    while True:
        dim = rng.choice([64, 128])
        heads = rng.choice([4, 8, 16])
        length = _log_int(rng, 1, 32768)
        batch = _log_int(rng, 1, max(1, min(32, 32768 // length)))
        c = _rotary("", dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=batch, heads=heads,
                    kv_heads=rng.choice([heads, heads // 2, heads // 4]), keys=rng.choice([2, 3]), length=length, dim=dim,
                    rot=rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), start=_log_int(rng, 1, 900000) - 1,
                    ragged=rng.random() < 0.5, backward=length > 1 and rng.random() < 0.5)
        if work(c)["bytes"] <= 8.0e8:
            return c


def _draw_tree(rng):
    while True:
        heads = rng.choice([4, 8, 16])
        c = _tree("", order=rng.choice([2, 2, 3]), dtype=rng.choice(["bf16", "fp16"]), batch=_log_int(rng, 1, 32),
                  heads=heads, kv_heads=rng.choice([heads, heads // 2, heads // 4]), dim=rng.choice([64, 128]),
                  nodes=_log_int(rng, 1, 64), longest=_log_int(rng, 1, 40001), softclamp=rng.choice([0.0, 0.0, 0.0, 20.0]),
                  layout=rng.randrange(1 << 30))
        rows = c["batch"] * c["longest"]
        if rows * c["kv_heads"] * c["dim"] * c["order"] <= 1.6e8 and rows * c["nodes"] * heads * c["order"] <= 3e8:
            return c


def draw(rng):
    kind = rng.choice(["packed", "packed", "rotary", "tree"])
    c = {"packed": _draw_packed, "rotary": _draw_rotary, "tree": _draw_tree}[kind](rng)
    c.pop("name")
    return c


def _lengths(case):
    """Sequence lengths of a packed case: lognormal shares of ``total``, some of them 0 or 1."""
    r = random.Random(case["layout"])
    s, total = case["seqs"], case["total"]
    w = [r.lognormvariate(0.0, case["spread"]) for _ in range(s)]
    n = [int(total * x / sum(w)) for x in w]
    if s > 2 and r.random() < 0.5:
        n[r.randrange(s)] = r.randrange(2)
    rest = total - sum(n)
    if rest:
        some = [i for i in range(s) if n[i] > 1] or [0]
        for i in range(rest):
            n[some[i % len(some)]] += 1
    return n


def _tree_layout(case):
    """Cached lengths and the parents of every sequence's tree (-1: child of the cached tokens)."""
    r = random.Random(case["layout"])
    b, t, longest = case["batch"], case["nodes"], case["longest"]
    lens = [longest] + [r.randrange(longest // 2, longest + 1) for _ in range(b - 1)]
    parents = [[-1 if i == 0 else r.randrange(-1, i) if r.random() < 0.5 else i - 1 for i in range(t)] for _ in range(b)]
    return lens, parents


# ---------------------------------------------------------------------------
# inputs

def _unit(t):
    """Queries and keys leave the modules' head norms: unit mean square over the features."""
    return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6)


def _frequencies(case):
    """Inverse frequencies and the factor of the amplitude, in 64 bits."""
    rot, kind, theta, factor, old = case["rot"], case["scaling"], 10000.0, 8.0, 8192.0
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if kind == "ntk":
        theta = theta * factor ** (rot / max(rot - 2, 1))
    inv = theta ** (-i / rot)
    m = 1.0
    if kind == "linear":
        inv = inv / factor
    if kind == "yarn":
        turns = old * inv / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        inv = inv / factor * (1.0 - keep) + inv * keep
        m = 0.1 * math.log(factor) + 1.0
    return inv.float(), m


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    st = dict(case=case)
    if case["op"] == "packed":
        n, h, k, d, order = case["total"], case["heads"], case["kv_heads"], case["dim"], case["order"]
        lens = _lengths(case)
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        st["cu_host"], st["longest"] = cu, max(lens)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        st["qs"] = [_unit(rnd(n, h if i == 0 else k, d)).to(dt).requires_grad_(case["backward"]) for i in range(order + 1)]
        st["vs"] = [rnd(n, k, d).to(dt).requires_grad_(case["backward"]) for _ in range(order - 1)]
        if case["backward"]:
            st["dout"] = rnd(n, h, d).to(dt)
    elif case["op"] == "rotary":
        b, n, d = case["batch"], case["length"], case["dim"]
        heads = [case["heads"]] + [case["kv_heads"]] * case["keys"]
        # head-split views of projections: [b, n, h, d] in memory
        st["xs"] = [_unit(rnd(b, n, h, d)).to(dt).permute(0, 2, 1, 3).requires_grad_(case["backward"]) for h in heads]
        if case["backward"]:
            st["dys"] = [rnd(b, n, h, d).to(dt).permute(0, 2, 1, 3) for h in heads]
        inv, st["factor"] = _frequencies(case)
        st["inv"] = inv.cuda()
        pos = case["start"] + torch.arange(n, device="cuda").expand(b, n)
        if case["ragged"]:
            pos = pos + torch.randint(0, 64, (b, 1), generator=g, device="cuda")
        st["pos"] = pos.to(torch.int32).contiguous()
    else:
        b, h, k, d, t, order = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "nodes", "order"))
        lens, parents = _tree_layout(case)
        cap = case["longest"] + t
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
        st["keys"] = [_unit(rnd(b, k, cap, d)).to(dt) for _ in range(order)]
        st["vals"] = [rnd(b, k, cap, d).to(dt) for _ in range(order - 1)]
        # what the earlier steps left: messages, and log-sum-exps that grow with the length
        st["msgs"] = [(0.3 * rnd(b, k, cap, d)).to(dt) for _ in range(order - 1)]
        st["lses"] = [0.2 * rnd(b, k, cap) + math.log(max(case["longest"], 2)) for _ in range(order - 1)]
        st["q1"] = _unit(rnd(b, h, t, d)).to(dt)
        st["new_keys"] = [_unit(rnd(b, k, t, d)).to(dt) for _ in range(order)]
        st["new_vals"] = [rnd(b, k, t, d).to(dt) for _ in range(order - 1)]
        if own:
            dec = _package().TreeDecoder(batch=b, order=order, heads=h, kv_heads=k, dim_head=d, capacity=cap, max_nodes=t,
                                         dtype=dt, device="cuda", softclamp_value=case["softclamp"] or None)
            dec.load(st["keys"], st["vals"], st["lses"], st["msgs"], st["lens"])
            st["decoder"] = dec
            for x in ("keys", "vals", "msgs", "lses"):
                del st[x]
    return st


# ---------------------------------------------------------------------------
# the framework's calls

def _own_packed(st):
    P, case = _package(), st["case"]
    qs, vs = st["qs"], st["vs"]
    kw = dict(causal=case["causal"], softclamp_value=case["softclamp"] or None, max_seqlen=st["longest"])
    if case["order"] == 2:
        out = P.poly_attention_order2_packed(qs[0], qs[1], qs[2], vs[0], st["cu"], **kw)[0]
    else:
        out = P.poly_attention_chain_packed(qs[:-1], qs[1:], vs, st["cu"], **kw)[0]
    if not case["backward"]:
        return [out]
    return [out, *torch.autograd.grad(out, [*qs, *vs], st["dout"])]


def _own_rotary(st):
    P, case = _package(), st["case"]
    ys = P.apply_rotary(st["xs"], st["inv"], positions=st["pos"], interleaved=case["interleaved"],
                        attention_factor=st["factor"])
    if not case["backward"]:
        return list(ys)
    return [*ys, *torch.autograd.grad(ys, st["xs"], st["dys"])]


def _own_tree(st):
    out, msgs, lses = st["decoder"].step(st["q1"], st["new_keys"], st["new_vals"], st["parents"], return_rows=True)
    return [out, *msgs, *lses]


# ---------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits

def _plain_pass(q, k, v, bias, keep, scale, clamp):
    """q [.., r, d], k / v [.., n, d], bias [.., n], keep: allowed entries. Returns out, lse."""
    s = (q @ k.transpose(-1, -2)) * scale
    if clamp:
        s = clamp * torch.tanh(s / clamp)
    if bias is not None:
        s = s + bias.unsqueeze(-2)
    if keep is not None:
        s = s.masked_fill(~keep, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    return (p @ v) / total, (m + torch.log(total)).squeeze(-1)


def _plain_chain(qs, vs, causal, scale, clamp):
    """One sequence: qs[0] [g, r, n, d], other tensors [g, n, d] (32 bits). Returns the chain's output."""
    order, n = len(qs) - 1, qs[0].shape[-2]
    keep = None
    if causal:
        at = torch.arange(n, device=qs[0].device)
        keep = at[None, :] <= at[:, None]
    val, bias = vs[-1], None
    for t in range(order - 1, 0, -1):
        msg, lse = _plain_pass(qs[t], qs[t + 1], val, bias, keep, scale, clamp)
        val, bias = (vs[t - 2] * msg if t >= 2 else msg), lse
    g, r, _, d = qs[0].shape
    out = _plain_pass(qs[0], qs[1].unsqueeze(1), val.unsqueeze(1), bias.unsqueeze(1), keep, scale, clamp)[0]
    return out


def _plain_packed(st):
    case = st["case"]
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    r, scale = h // g, case["dim"] ** -0.5
    leaves = [*st["qs"], *st["vs"]]
    nq = len(st["qs"])
    outs = [torch.empty_like(st["qs"][0], requires_grad=False)]
    if case["backward"]:
        outs += [torch.empty_like(x, requires_grad=False) for x in leaves]
    cu = st["cu_host"]
    for a, e in zip(cu[:-1], cu[1:]):
        n = e - a
        if n == 0:
            continue
        step = max(1, min(g, (1 << 28) // (r * n * n)))
        for k0 in range(0, g, step):
            k1 = min(g, k0 + step)
            with torch.set_grad_enabled(case["backward"]):
                parts = [x.detach()[a:e, (k0 * r if i == 0 else k0):(k1 * r if i == 0 else k1)].float().transpose(0, 1)
                         for i, x in enumerate(leaves)]
                if case["backward"]:
                    parts = [x.contiguous().requires_grad_(True) for x in parts]
                q1 = parts[0].reshape(k1 - k0, r, n, d)
                out = _plain_chain([q1, *parts[1:nq]], parts[nq:], case["causal"], scale, case["softclamp"])
                out = out.reshape((k1 - k0) * r, n, d)
                if case["backward"]:
                    dout = st["dout"][a:e, k0 * r:k1 * r].float().transpose(0, 1)
                    grads = torch.autograd.grad(out, parts, dout)
            outs[0][a:e, k0 * r:k1 * r] = out.detach().transpose(0, 1)
            if case["backward"]:
                for i, x in enumerate(grads):
                    w = r if i == 0 else 1
                    outs[1 + i][a:e, k0 * w:k1 * w] = x.transpose(0, 1)
    return outs


def _plain_rotate(x, cos, sin, rot, interleaved):
    xf = x.detach().float()
    head, rest = xf[..., :rot], xf[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1).to(x.dtype)


def _plain_rotary(st):
    case = st["case"]
    # a far position times a frequency needs more than 32 bits to keep its angle
    ang = st["pos"].double()[:, None, :, None] * st["inv"].double()
    cos, sin = (torch.cos(ang) * st["factor"]).float(), (torch.sin(ang) * st["factor"]).float()
    outs = [_plain_rotate(x, cos, sin, case["rot"], case["interleaved"]) for x in st["xs"]]
    if case["backward"]:
        outs += [_plain_rotate(x, cos, -sin, case["rot"], case["interleaved"]) for x in st["dys"]]
    return outs


def _ancestors(parents):
    """[b, T, T] truth values: node j is node i or one of its ancestors."""
    b, t = parents.shape
    seen = torch.zeros(b, t, t, dtype=torch.bool, device=parents.device)
    node = torch.arange(t, device=parents.device).expand(b, t)
    live = torch.ones_like(node, dtype=torch.bool)
    for _ in range(t):
        seen |= live.unsqueeze(-1) & (torch.arange(t, device=parents.device) == node.unsqueeze(-1))
        up = torch.gather(parents.long(), 1, node.clamp(min=0))
        node, live = up.clamp(min=0), live & (up >= 0)
    return seen


def _plain_tree(st):
    case = st["case"]
    b, h, g, d, t, order = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "nodes", "order"))
    scale, clamp, r, dt = d ** -0.5, case["softclamp"], h // g, _DT[case["dtype"]]
    n = case["longest"]
    old = (torch.arange(n, device="cuda")[None] < st["lens"][:, None])[:, None].expand(b, t, n)
    keep = torch.cat((old, _ancestors(st["parents"])), -1)[:, None]           # [b, 1, T, n + T]
    rows = lambda cache, new: torch.cat((cache[:, :, :n].float(), new.float()), 2)   # noqa: E731
    msgs, lses = [None] * (order - 1), [None] * (order - 1)
    val, bias = rows(st["vals"][-1], st["new_vals"][-1]), None
    for lvl in range(order - 1, 0, -1):
        at = (order - 1) - lvl
        msg, lse = _plain_pass(st["new_keys"][lvl - 1].float(), rows(st["keys"][lvl], st["new_keys"][lvl]), val, bias, keep,
                               scale, clamp)
        msgs[at], lses[at] = msg, lse
        full = rows(st["msgs"][at], msg)
        bias = torch.cat((st["lses"][at][:, :, :n], lse), -1)
        val = rows(st["vals"][lvl - 2], st["new_vals"][lvl - 2]) * full if lvl >= 2 else full
    q1 = st["q1"].float().reshape(b, g, r * t, d)
    out = _plain_pass(q1, rows(st["keys"][0], st["new_keys"][0]), val, bias, keep.repeat(1, 1, r, 1), scale, clamp)[0]
    return [out.reshape(b, h, t, d).to(dt), *[m.to(dt) for m in msgs], *lses]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"packed": _own_packed, "rotary": _own_rotary, "tree": _own_tree}[op](state)
    return {"packed": _plain_packed, "rotary": _plain_rotary, "tree": _plain_tree}[op](state)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions

def _exact_scores(q, k, bias, i0, causal, scale, clamp):
    """Rows i0.. of one head: x (the biased scores) and the softclamp's derivative."""
    s = torch.einsum("id,jd->ij", q, k) * scale
    slope = None
    if clamp:
        th = torch.tanh(s / clamp)
        s, slope = clamp * th, 1.0 - th * th
    if bias is not None:
        s = s + bias[None]
    if causal:
        i = torch.arange(i0, i0 + q.shape[0], device=q.device)
        s[torch.arange(k.shape[0], device=q.device)[None] > i[:, None]] = -math.inf
    return s, slope


def _exact_fwd(q, k, v, bias, causal, scale, clamp, block):
    out, lse = torch.empty_like(q), q.new_empty(q.shape[0])
    for i in range(0, q.shape[0], block):
        x, _ = _exact_scores(q[i:i + block], k, bias, i, causal, scale, clamp)
        lse[i:i + block] = torch.logsumexp(x, -1)
        out[i:i + block] = torch.exp(x - lse[i:i + block, None]) @ v
    return out, lse


def _exact_bwd(q, k, v, bias, out, lse, dout, dlse, causal, scale, clamp, block):
    dq, dk, dv, db = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), k.new_zeros(k.shape[0])
    for i in range(0, q.shape[0], block):
        sl = slice(i, i + block)
        x, slope = _exact_scores(q[sl], k, bias, i, causal, scale, clamp)
        p = torch.exp(x - lse[sl, None])
        row = (dout[sl] * out[sl]).sum(-1) - (0.0 if dlse is None else dlse[sl])
        ds = p * (dout[sl] @ v.T - row[:, None])
        dv += p.T @ dout[sl]
        db += ds.sum(0)
        dz = ds * scale if slope is None else ds * slope * scale
        dq[sl] = dz @ k
        dk += dz.T @ q[sl]
    return dq, dk, dv, db


def _exact_packed(st):
    case = st["case"]
    h, g, order, nq = case["heads"], case["kv_heads"], case["order"], case["order"] + 1
    args = (case["causal"], case["dim"] ** -0.5, case["softclamp"])
    leaves = [x.detach() for x in (*st["qs"], *st["vs"])]
    outs = [torch.zeros(leaves[0].shape, dtype=torch.float64, device="cuda")]
    if case["backward"]:
        outs += [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in leaves]
    for a, e in zip(st["cu_host"], st["cu_host"][1:]):
        if e == a:
            continue
        block = max(1, (1 << 26) // (e - a))
        for kh in range(g):
            q = [None] + [x[a:e, kh].double() for x in leaves[1:nq]]
            v = [x[a:e, kh].double() for x in leaves[nq:]]
            # level t attends q[t] to q[t + 1]; its values: the message above it, times v below the top level
            val, bias, msg, lse = {order - 1: v[-1]}, {order - 1: None}, {}, {}
            for t in range(order - 1, 0, -1):
                msg[t], lse[t] = _exact_fwd(q[t], q[t + 1], val[t], bias[t], *args, block)
                bias[t - 1] = lse[t]
                val[t - 1] = v[t - 2] * msg[t] if t >= 2 else msg[t]
            dval, dbias = torch.zeros_like(val[0]), torch.zeros_like(bias[0])
            for hh in range(kh * (h // g), (kh + 1) * (h // g)):
                q1 = leaves[0][a:e, hh].double()
                o, l = _exact_fwd(q1, q[1], val[0], bias[0], *args, block)
                outs[0][a:e, hh] = o
                if case["backward"]:
                    dq, dk, dv, db = _exact_bwd(q1, q[1], val[0], bias[0], o, l, st["dout"][a:e, hh].double(), None, *args, block)
                    outs[1][a:e, hh] = dq
                    outs[2][a:e, kh] += dk
                    dval += dv
                    dbias += db
            if not case["backward"]:
                continue
            dmsg = dval
            for t in range(1, order):
                dq, dk, dv, db = _exact_bwd(q[t], q[t + 1], val[t], bias[t], msg[t], lse[t], dmsg, dbias, *args, block)
                outs[1 + t][a:e, kh] += dq
                outs[2 + t][a:e, kh] += dk
                if t == order - 1:
                    outs[1 + nq + order - 2][a:e, kh] = dv
                else:
                    outs[1 + nq + t - 1][a:e, kh] = dv * msg[t + 1]
                    dmsg, dbias = dv * v[t - 1], db
    return outs


def _exact_rotary(st):
    case = st["case"]
    rot = case["rot"]
    half = rot // 2
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    turn = torch.polar(torch.full((), st["factor"], dtype=torch.float64, device="cuda"),
                       torch.einsum("bn,f->bnf", st["pos"].double(), st["inv"].double()))[:, None]

    def go(x, w):
        y = x.detach().double().clone()
        z = torch.complex(y[..., first], y[..., second]) * w
        y[..., first], y[..., second] = z.real, z.imag
        return y

    outs = [go(x, turn) for x in st["xs"]]
    if case["backward"]:
        outs += [go(x, turn.conj()) for x in st["dys"]]
    return outs


def _exact_tree(st):
    case = st["case"]
    b, h, g, order, t = (case[x] for x in ("batch", "heads", "kv_heads", "order", "nodes"))
    lens, parents = _tree_layout(case)
    scale, clamp = case["dim"] ** -0.5, case["softclamp"]
    out = torch.zeros(st["q1"].shape, dtype=torch.float64, device="cuda")
    msgs = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in st["new_vals"]]
    lses = [torch.zeros(x.shape[:3], dtype=torch.float64, device="cuda") for x in st["new_vals"]]
    for s in range(b):
        n = lens[s]
        hide = torch.zeros(t, n + t, dtype=torch.bool)
        for i in range(t):
            hide[i, n:] = True
            j = i
            while j >= 0:
                hide[i, n + j] = False
                j = parents[s][j]
        hide = hide.cuda()

        def attend(q, k, v, bias):
            x, _ = _exact_scores(q, k, bias, 0, False, scale, clamp)
            x[hide] = -math.inf
            lse = torch.logsumexp(x, -1)
            return torch.exp(x - lse[:, None]) @ v, lse

        for kh in range(g):
            key = [torch.cat((c[s, kh, :n], w[s, kh])).double() for c, w in zip(st["keys"], st["new_keys"])]
            v = [torch.cat((c[s, kh, :n], w[s, kh])).double() for c, w in zip(st["vals"], st["new_vals"])]
            val, bias = v[-1], None
            for lvl in range(order - 1, 0, -1):
                at = order - 1 - lvl
                m, l = attend(st["new_keys"][lvl - 1][s, kh].double(), key[lvl], val, bias)
                msgs[at][s, kh], lses[at][s, kh] = m, l
                m, bias = torch.cat((st["msgs"][at][s, kh, :n].double(), m)), torch.cat((st["lses"][at][s, kh, :n].double(), l))
                val = v[lvl - 2] * m if lvl >= 2 else m
            for hh in range(kh * (h // g), (kh + 1) * (h // g)):
                out[s, hh] = attend(st["q1"][s, hh].double(), key[0], val, bias)[0]
    return [out, *msgs, *lses]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return {"packed": _exact_packed, "rotary": _exact_rotary, "tree": _exact_tree}[case["op"]](st)


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    es = _ES[case["dtype"]]
    if case["op"] == "rotary":
        rows = case["batch"] * case["length"] * (case["heads"] + case["keys"] * case["kv_heads"])
        ways = 2 if case["backward"] else 1
        size = rows * case["dim"] * ways
        return {"bytes": 2 * size * es + 4 * case["batch"] * case["length"], "flops": 3 * rows * case["rot"] * ways}
    h, g, d, order = case["heads"], case["kv_heads"], case["dim"], case["order"]
    if case["op"] == "packed":
        lens = _lengths(case)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        heads = h + (order - 1) * g
        tokens = case["total"]
        per_token = (h + (2 * order - 1) * g) * d * es          # inputs
        size = tokens * (per_token + h * d * es)
        flops = 4 * pairs * heads * d
        if case["backward"]:
            size += tokens * (per_token + h * d * es)           # gradients written, output gradient read
            flops += 8 * pairs * heads * d
        return {"bytes": size, "flops": flops}
    lens, _ = _tree_layout(case)
    t, b = case["nodes"], case["batch"]
    cached = (3 * order - 2) * g * d * es + (order - 1) * g * 4    # keys, values, messages and log-sum-exps of a token
    rows = sum(n + t for n in lens)
    new = b * t * ((2 * h + (2 * order - 1) * g) * d * es + (order - 1) * g * (d * es + 4))
    return {"bytes": sum(lens) * cached + new, "flops": 4 * d * t * rows * (h + (order - 1) * g)}
