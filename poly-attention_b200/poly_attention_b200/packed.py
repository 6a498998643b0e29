"""Poly attention over sequences of different lengths packed end to end.

Tensors are [total, heads, d] (tokens of all sequences, no batch axis) and
``cu_seqlens`` (int32 [s + 1] on the device) holds each sequence's first row and
the row behind the last. A sequence's tokens attend that sequence alone, so the
result of each is that of ``poly_attention_order2`` / ``poly_attention_chain`` on
it by itself (poly_attention/poly_attention.py:48-116,
n_poly_attention.py:263-313), without the padding that a [b, n, ...] batch of
unequal lengths needs. Rows outside every sequence come out as zeros and get
zero gradients.

The offsets stay on the device and are not checked there: they must not
decrease and must lie in [0, total] (others give wrong rows, never an access
outside the tensors). ``max_seqlen`` is an upper bound of the lengths, if the
caller has one: up to 128 it selects kernels that hold a whole sequence per CTA, and
a longer sequence then comes out as NaN. Without it the 16-bit backward (heads of 64 or 128 features) takes
4 d bytes of scratch per row and head, for 8 rows more a sequence, and 1 KB a sequence and head; with it none.

Gradients of queries over several key tiles are summed in 32 bits in no fixed order
(16-bit tensors with heads of 64 or 128 features and no bound of 128): equal calls may
differ in their last bit. Everything else is the same from call to call.
"""
from __future__ import annotations

import operator

import torch

from . import _lib
from ._lib import PolyPackedArgs, PolyPackedBwdArgs, check, lib
from .core import _autocast, _sc
from .ops import _DTYPES, _no_tangents, _on, _require_cuda, _stream, packed_cu


def split_heads(t, split, heads):
    """'b n (split h d) -> split b h n d' as strided views (no copy)."""
    b, n, f = t.shape
    d = f // (split * heads)
    return t.view(b, n, split, heads, d).permute(2, 0, 3, 1, 4)


def token_rows(t):
    """[1, heads, total, d] -> [total, heads, d] (a view)."""
    return t.squeeze(0).transpose(0, 1)


def check_packed(x, context=None, mask=None, context_mask=None, cache=None, return_cache=False):
    """A module's arguments with cu_seqlens."""
    if x.dim() != 3 or x.shape[0] != 1:
        raise ValueError("packed sequences (cu_seqlens) come as one row: x [1, total, dim]")
    if any(t is not None for t in (context, mask, context_mask, cache)) or return_cache:
        raise ValueError("packed sequences (cu_seqlens) take no context, masks or cache")


def packed_offsets(lengths, device="cuda"):
    """(cu_seqlens, max_seqlen) of a list of sequence lengths."""
    lengths = [int(n) for n in lengths]
    if any(n < 0 for n in lengths):
        raise ValueError("sequence lengths must be non-negative")
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32).to(device), max(lengths, default=0)


def _tensors(q, k, v, *same):
    dtype, device = q.dtype, q.device
    if dtype not in _DTYPES or k.dtype != dtype or v.dtype != dtype:
        _require_cuda(q, k, v)
        raise TypeError(f"q, k, v must share one of {list(_DTYPES)}; got {dtype}, {k.dtype}, {v.dtype}")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[::2] != k.shape[::2]:
        raise ValueError(f"packed tensors are q [total, h, d] and k, v [total, g, d]; got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if device.type != "cuda":
        _require_cuda(q)
    for t in (k, v, *same):
        if t is not None and t.device != device:
            _require_cuda(t)
            raise ValueError("packed tensors must be on one device")


def _bound(max_seqlen):
    if max_seqlen is None:
        return 0
    max_seqlen = operator.index(max_seqlen)
    if max_seqlen < 0:
        raise ValueError("max_seqlen must be non-negative")
    return min(max_seqlen, 1 << 30)


def _rows(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _vec(t, heads, total, what):
    if t.shape != (heads, total):
        raise ValueError(f"{what} must be [{heads}, {total}], got {tuple(t.shape)}")
    return _rows(t.float())


_FWD = _lib.packer(PolyPackedArgs)


def _forward(q, k, v, cu, bias, epi_mul, causal, softclamp, scale, max_seqlen, out_lo):
    """pass_fwd_packed on checked tensors: (out, lse, epi or None, out_lo or None)."""
    total, h, d = q.shape
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = q.new_empty(total, h, d)
    lse = q.new_empty(h, total, dtype=torch.float32)
    epi = lo = None
    if epi_mul is not None:
        epi_mul, epi = _rows(epi_mul), torch.empty_like(out)
    if out_lo and q.dtype != torch.float32:
        lo = torch.empty_like(out)
    seqs = cu.shape[0] - 1
    if seqs == 0 and total:
        for t in (out, lse, epi, lo):
            if t is not None:
                t.zero_()
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    ms = epi_mul.stride() if epi is not None else (0, 0)
    # PolyPackedArgs in its order; tensors as pointer and (batch, head, row) strides
    a = PolyPackedArgs.from_buffer_copy(_FWD.pack(
        1, h, k.shape[1], total, total, d, _DTYPES[q.dtype], bool(causal), d ** -0.5 if scale is None else scale, _sc(softclamp),
        q.data_ptr(), 0, qs[1], qs[0], k.data_ptr(), 0, ks[1], ks[0], v.data_ptr(), 0, vs[1], vs[0], 0, 0, 0, 0,
        0 if bias is None else bias.data_ptr(), 0, 0 if bias is None else bias.stride(0), 0, 0, 0, 0,
        out.data_ptr(), 0, d, h * d, lse.data_ptr(), 0, total,
        0 if epi is None else epi_mul.data_ptr(), 0, ms[1], ms[0], 0 if epi is None else epi.data_ptr(), 0, d, h * d, 0, 0, 0, 0,
        cu.data_ptr(), seqs, max_seqlen, 1, 0, 0 if lo is None else lo.data_ptr()))
    with _on(q.device):
        check(lib.poly_packed_pass_fwd(a, _stream(q.device)), "poly_packed_pass_fwd")
    return out, lse, epi, lo


@torch.compiler.disable   # library calls through ctypes: dynamo runs them eagerly
def pass_fwd_packed(q, k, v, cu_seqlens, *, causal=False, softclamp=None, scale=None, bias=None, epi_mul=None,
                    max_seqlen=None, out_lo=False):
    """One attention pass over packed sequences (see PolyPackedArgs in include/poly_attention.h).

    q [total, h, d]; k, v [total, g, d] with g | h; bias [g, total] fp32; epi_mul
    [total, h, d]. Returns (out, lse[, epi_mul * out][, out_lo]) with out like q and lse
    fp32 [h, total]; out_lo is what rounding took off out, which ``pass_bwd_packed`` takes
    (None for float32).
    """
    _no_tangents((q, k, v, bias, epi_mul))
    _tensors(q, k, v, bias, epi_mul)
    cu = packed_cu(cu_seqlens, q)
    if bias is not None:
        bias = _vec(bias, k.shape[1], q.shape[0], "bias")
    if q.shape[1] % max(k.shape[1], 1):
        raise ValueError("heads must be divisible by kv_heads")
    if epi_mul is not None and (epi_mul.shape != q.shape or epi_mul.dtype != q.dtype):
        raise ValueError("epi_mul must have q's shape and dtype")
    out, lse, epi, lo = _forward(q, k, v, cu, bias, epi_mul, causal, softclamp, scale, _bound(max_seqlen), out_lo)
    return (out, lse) + ((epi,) if epi is not None else ()) + ((lo,) if out_lo else ())


_BWD = _lib.packer(PolyPackedBwdArgs)


def _backward(q, k, v, cu, out, lse, dout, bias, dlse, dq, want_dbias, out_lo, factors, causal, softclamp, scale, max_seqlen):
    """pass_bwd_packed on checked tensors."""
    q, k, v, out, dout = _rows(q), _rows(k), _rows(v), _rows(out), _rows(dout)
    total, h, d = q.shape
    g = k.shape[1]
    if any(st <= 0 for st in dout.stride()):
        dout = dout.contiguous()        # broadcast gradients (out.sum().backward())
    left = right = dright = None
    if factors is not None:
        left, right = (_rows(t) for t in factors)
        dright = v.new_empty(total, g, d)
    accumulate = dq is not None
    if dq is None:
        dq = q.new_empty(total, h, d)
    dk, dv = k.new_empty(total, g, d), v.new_empty(total, g, d)
    dbias = q.new_empty(g, total, dtype=torch.float32) if want_dbias else None
    seqs = cu.shape[0] - 1
    if seqs == 0 and total:
        for t in (dk, dv, dbias, dright, None if accumulate else dq):
            if t is not None:
                t.zero_()
    qs, ks, vs, os, gs, dqs = q.stride(), k.stride(), v.stride(), out.stride(), dout.stride(), dq.stride()
    ls, rs = (left.stride(), right.stride()) if left is not None else ((0, 0), (0, 0))
    ptr = lambda t: 0 if t is None else t.data_ptr()   # noqa: E731
    # PolyPackedBwdArgs in its order
    a = PolyPackedBwdArgs.from_buffer_copy(_BWD.pack(
        1, h, g, total, total, d, _DTYPES[q.dtype], bool(causal), d ** -0.5 if scale is None else scale, _sc(softclamp),
        q.data_ptr(), 0, qs[1], qs[0], k.data_ptr(), 0, ks[1], ks[0], v.data_ptr(), 0, vs[1], vs[0], 0, 0, 0, 0,
        ptr(bias), 0, 0 if bias is None else bias.stride(0), 0, 0, 0, 0,
        out.data_ptr(), 0, os[1], os[0], lse.data_ptr(), 0, lse.stride(0), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
        dout.data_ptr(), 0, gs[1], gs[0], ptr(dlse), 0, 0 if dlse is None else dlse.stride(0),
        dq.data_ptr(), 0, dqs[1], dqs[0], dk.data_ptr(), 0, d, g * d, dv.data_ptr(), 0, d, g * d, ptr(dbias), 0, total,
        accumulate, 0, 0, 0, cu.data_ptr(), seqs, max_seqlen, 1, 0, ptr(out_lo),
        ptr(left), ls[1], ls[0], ptr(right), rs[1], rs[0], ptr(dright), d, g * d))
    b = a.bwd
    with _on(q.device):
        need = lib.poly_packed_pass_bwd_workspace_size(a)
        ws = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
        if need:
            b.workspace, b.workspace_bytes = ws.data_ptr(), need
        check(lib.poly_packed_pass_bwd(a, _stream(q.device)), "poly_packed_pass_bwd")
    return dq, dk, dv if dright is None else (dv, dright), dbias


@torch.compiler.disable
def pass_bwd_packed(q, k, v, cu_seqlens, out, lse, dout, *, causal=False, softclamp=None, scale=None, bias=None,
                    dlse=None, dq=None, want_dbias=False, max_seqlen=None, out_lo=None, factors=None):
    """Backward of ``pass_fwd_packed``. Returns (dq, dk, dv, dbias-or-None). With ``dq`` given the
    query gradient is added to it in place. With ``factors`` = (left, right), whose product the
    values were, dv is the pair of their gradients."""
    _no_tangents((q, k, v, out, lse, dout, bias, dlse, dq, out_lo), *(factors or ()))
    _tensors(q, k, v, out, lse, dout, bias, dlse, dq, out_lo, *(factors or ()))
    cu = packed_cu(cu_seqlens, q)
    total, h = q.shape[:2]
    g = k.shape[1]
    if h % max(g, 1):
        raise ValueError("heads must be divisible by kv_heads")
    if out.shape != q.shape or dout.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out and dout must have q's shape, out its dtype")
    if dq is not None and (dq.shape != q.shape or dq.dtype != q.dtype or dq.stride(-1) != 1):
        raise ValueError("dq must have q's shape and dtype and a contiguous last dim")
    if out_lo is not None and (out_lo.shape != out.shape or out_lo.dtype != out.dtype or out_lo.stride() != out.stride()):
        raise ValueError("out_lo must have out's shape, dtype and strides")
    if out_lo is not None and out.stride(-1) != 1:
        raise ValueError("out and out_lo must have a contiguous last dim")
    if factors is not None and any(t.shape != v.shape or t.dtype != v.dtype for t in factors):
        raise ValueError("the values' factors must have their shape and dtype")
    lse = _vec(lse, h, total, "lse")
    bias = None if bias is None else _vec(bias, g, total, "bias")
    dlse = None if dlse is None else _vec(dlse, h, total, "dlse")
    return _backward(q, k, v, cu, out, lse, dout.to(q.dtype), bias, dlse, dq, want_dbias, out_lo, factors, causal, softclamp,
                     scale, _bound(max_seqlen))


def packed_kernel_names(q, k, v, max_seqlen=None):
    """(forward, backward) kernel family the library picks for these packed tensors."""
    a, b = PolyPackedArgs(), PolyPackedBwdArgs()

    def put(x, name, t):
        setattr(x, name, t.data_ptr())
        st = getattr(x, name + "_stride")
        st[1], st[2] = t.stride(1), t.stride(0)

    for x, f in ((a, a.fwd), (b, b.bwd.fwd)):
        f.batch, f.heads, f.kv_heads, f.head_dim, f.dtype = 1, q.shape[1], k.shape[1], q.shape[2], _DTYPES[q.dtype]
        f.seq_q = f.seq_k = q.shape[0]
        f.scale = q.shape[2] ** -0.5
        for name, t in (("q", q), ("k", k), ("v", v), ("out", q)):
            put(f, name, t)
        x.cu_seqlens, x.seqs, x.max_len = 1, 1, int(max_seqlen or 0)
    for name, t in (("dout", q), ("dq", q), ("dk", k), ("dv", v)):
        put(b.bwd, name, t)
    return lib.poly_packed_pass_fwd_kernel_name(a).decode(), lib.poly_packed_pass_bwd_kernel_name(b).decode()


def _chain_forward(order, cu, opts, ql, qr, vs, keep):
    """Per level: values, biases, messages, log-sum-exps, rounding residues (if ``keep``)."""
    vals, biases, msgs, lses, los = ([None] * order for _ in range(5))
    val, bias = vs[-1], None
    for t in range(order - 1, -1, -1):
        vals[t], biases[t] = val, bias
        # V' = v * msg is written by the pass that makes msg (n_poly_attention.py:287)
        msgs[t], lses[t], epi, los[t] = _forward(ql[t], qr[t], val, cu, bias, vs[t - 2] if t >= 2 else None, *opts, keep)
        val, bias = epi if t >= 2 else msgs[t], lses[t]
    return vals, biases, msgs, lses, los


class _PackedChain(torch.autograd.Function):
    """The order-n chain. Inputs: order queries ql, order keys qr and order - 1 values; shared[t] says
    that ql[t] is qr[t - 1], whose two gradients are then summed inside the kernel."""

    @staticmethod
    def forward(ctx, order, shared, cu, opts, *tensors):
        ql, qr, vs = tensors[:order], tensors[order:2 * order], tensors[2 * order:]
        vals, biases, msgs, lses, los = _chain_forward(order, cu, opts, ql, qr, vs, True)
        ctx.order, ctx.shared, ctx.opts = order, shared, opts
        ctx.has = [[x is not None for x in xs] for xs in (biases, los)]
        ctx.save_for_backward(cu, *tensors, *vals, *msgs, *lses, *(x for x in (*biases, *los) if x is not None))
        extra = (*lses[:0:-1], *msgs[:0:-1])        # level order - 1 first, as in the caches
        ctx.mark_non_differentiable(*extra)
        return (msgs[0], *extra)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, *_unused):
        n, saved = ctx.order, iter(ctx.saved_tensors)
        take = lambda k: [next(saved) for _ in range(k)]   # noqa: E731
        cu, = take(1)
        ql, qr, vs, vals, msgs, lses = take(n), take(n), take(n - 1), take(n), take(n), take(n)
        biases, los = ([next(saved) if x else None for x in has] for has in ctx.has)
        causal, softclamp, scale, max_seqlen = ctx.opts
        dql, dqr, dvs = [None] * n, [None] * n, [None] * (n - 1)
        g_out, g_lse = dout.to(ql[0].dtype), None
        for t in range(n):
            # a key tensor that is the next level's query keeps one gradient: the second part is added in the
            # kernel to the first, which was rounded once to the tensors' type
            dq, dqr[t], dv, g_lse = _backward(ql[t], qr[t], vals[t], cu, msgs[t], lses[t], g_out, biases[t], g_lse,
                                              dqr[t - 1] if ctx.shared[t] else None, t < n - 1, los[t],
                                              (vs[t - 1], msgs[t + 1]) if 0 < t < n - 1 else None, causal, softclamp, scale,
                                              max_seqlen)
            if not ctx.shared[t]:
                dql[t] = dq
            if t == n - 1:
                dvs[-1] = dv
            elif t == 0:
                g_out = dv
            else:
                dvs[t - 1], g_out = dv
        return (None, None, None, None, *dql, *dqr, *dvs)


def _chain(q_left, q_right, vs, cu_seqlens, softclamp_value, causal, max_seqlen):
    order = len(q_left)
    if order < 2 or len(q_right) != order or len(vs) != order - 1:
        raise ValueError("a chain of order n >= 2 takes n queries, n keys and n - 1 values")
    shared = tuple(t >= 1 and q_left[t] is q_right[t - 1] for t in range(order))
    ql, qr, vv = _autocast(*q_left), _autocast(*q_right), _autocast(*vs)
    ql = [qr[t - 1] if shared[t] else ql[t] for t in range(order)]
    _no_tangents((*ql, *qr, *vv))
    _tensors(ql[0], qr[0], vv[0], *ql[1:], *qr[1:], *vv[1:])
    shape, dtype = qr[0].shape, qr[0].dtype
    for t in (*ql[1:], *qr[1:], *vv):
        if t.shape != shape or t.dtype != dtype:
            raise ValueError("key, value and lower query tensors must share one shape and dtype")
    if ql[0].shape[1] % max(qr[0].shape[1], 1):
        raise ValueError("heads must be divisible by kv_heads")
    cu = packed_cu(cu_seqlens, ql[0])
    opts = (bool(causal), softclamp_value, None, _bound(max_seqlen))
    if torch.is_grad_enabled() and any(t.requires_grad for t in (*ql, *qr, *vv)):
        res = _PackedChain.apply(order, shared, cu, opts, *ql, *qr, *vv)
        return res[0], res[1:order], res[order:]
    _, _, msgs, lses, _ = _chain_forward(order, cu, opts, ql, qr, vv, False)
    return msgs[0], tuple(lses[:0:-1]), tuple(msgs[:0:-1])


@torch.compiler.disable
def poly_attention_chain_packed(q_left, q_right, vs, cu_seqlens, *, softclamp_value=None, causal=False, max_seqlen=None):
    """Order-n chain over packed sequences (n = len(q_left)), as ``poly_attention_chain``.

    q_left[0] = q1 [total, h, d]; q_left[t >= 1], q_right[t] and vs[t] are [total, g, d]. Returns
    (out [total, h, d], lses [g, total], msgs [total, g, d]), lses / msgs in the caches' order.
    """
    return _chain(q_left, q_right, vs, cu_seqlens, softclamp_value, causal, max_seqlen)


@torch.compiler.disable
def poly_attention_order2_packed(q1, q2, q3, v3, cu_seqlens, *, q2_pass1=None, softclamp_value=None, causal=False,
                                 max_seqlen=None):
    """Order-2 poly attention over packed sequences, as ``poly_attention_order2``: q1 [total, h, d];
    q2, q3, v3 [total, g, d]. Returns (out, lse23 [g, total], msg [total, g, d])."""
    out, lses, msgs = _chain((q1, q2 if q2_pass1 is None else q2_pass1), (q2, q3), (v3,), cu_seqlens, softclamp_value, causal,
                             max_seqlen)
    return out, lses[0], msgs[0]


__all__ = ["packed_offsets", "pass_fwd_packed", "pass_bwd_packed", "poly_attention_order2_packed",
           "poly_attention_chain_packed"]
