"""Rotary positions (``poly_rotary``): queries and keys of a layer rotated in one
launch, straight from the strided head-split views, with gradients.

``apply_rotary`` is the operator, ``rotary_frequencies`` its frequencies (with
the usual scalings for contexts longer than a model was trained on) and
``RotaryEmbedding`` the module that ``use_rotary_embed=True`` puts into the
attention modules (``rotary_emb``, poly_attention/poly_attention.py:202,
302-304; n_poly_attention.py:118, 226).

There is no CPU implementation: CPU tensors raise.
"""
from __future__ import annotations

import ctypes
import math
import operator
from typing import List, Optional

import torch
from torch import nn

from . import _lib
from ._lib import PolyRotaryArgs, PolyRotaryTensor, check, lib
from .ops import _DTYPES, _no_tangents, _on, _require_cuda, _stream, packed_cu


def rotary_frequencies(dim, *, theta=10000.0, scaling=None, factor=1.0, original_length=None, fast_turns=32.0,
                       slow_turns=1.0):
    """Inverse frequencies [dim / 2] (fp32) and the attention factor that goes with them.

    ``theta ** (-2 i / dim)``, computed in 64 bits. ``scaling`` stretches the
    context by ``factor``: "linear" divides every frequency by it, "ntk" raises
    theta to ``theta * factor ** (dim / (dim - 2))``, "yarn" divides only the
    frequencies that turn less than ``slow_turns`` times in ``original_length``
    positions, keeps those that turn more than ``fast_turns`` times, mixes the
    ones between, and returns the attention factor ``0.1 ln(factor) + 1``.
    """
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary dim must be positive and even, got {dim}")
    if not (theta > 0 and factor >= 1.0):
        raise ValueError("theta must be positive and factor at least 1")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling == "ntk":
        theta = theta * factor ** (dim / max(dim - 2, 1))
    elif scaling not in (None, "linear", "yarn"):
        raise ValueError(f"unknown rotary scaling {scaling!r}")
    inv = theta ** (-i / dim)
    if scaling == "linear":
        return (inv / factor).float(), 1.0
    if scaling == "yarn":
        if not original_length or not fast_turns > slow_turns:
            raise ValueError("yarn scaling needs original_length and fast_turns > slow_turns")
        turns = inv * (original_length / (2.0 * math.pi))
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        return (inv * keep + inv / factor * (1.0 - keep)).float(), 0.1 * math.log(factor) + 1.0
    return inv.float(), 1.0


def _empty_like(x):
    """Output with x's axis order in memory (token-major views stay token-major), dense."""
    b, h, n, d = x.shape
    s = x.stride()
    token_major = s[1] <= s[2]
    return torch.empty_strided((b, h, n, d), (h * n * d, d, h * d, 1) if token_major else (h * n * d, n * d, d, 1),
                               dtype=x.dtype, device=x.device)


_HEAD = _lib.packer(PolyRotaryArgs, before="t")
_TENSOR = _lib.packer(PolyRotaryTensor)


def _rotate(xs, inv_freq, positions, start, cu_seqlens, angles, interleaved, factor, inverse):
    xs = [x if x.stride(-1) == 1 else x.contiguous() for x in xs]
    outs = [_empty_like(x) for x in xs]
    x0 = xs[0]
    b, _, n, d = x0.shape
    rot = 2 * (inv_freq if angles is None else angles).shape[-1]
    ps = positions.stride() if positions is not None else (0, 0)
    an = angles.stride() if angles is not None else (0, 0)
    with _on(x0.device):
        stream = _stream(x0.device)
        for i0 in range(0, len(xs), _lib.MAX_ROTARY):
            part = xs[i0:i0 + _lib.MAX_ROTARY]
            buf = bytearray(ctypes.sizeof(PolyRotaryArgs))
            _HEAD.pack_into(buf, 0, b, n, d, rot, _DTYPES[x0.dtype], interleaved, inverse, len(part), factor,
                            positions is not None and positions.dtype == torch.int64,
                            positions.data_ptr() if positions is not None else 0, ps[0], ps[1], start,
                            inv_freq.data_ptr() if angles is None else 0, 0 if angles is None else angles.data_ptr(), an[0], an[1],
                            cu_seqlens.data_ptr() if cu_seqlens is not None else 0,
                            cu_seqlens.shape[0] - 1 if cu_seqlens is not None else 0, 0)
            at = PolyRotaryArgs.t.offset
            for x, y in zip(part, outs[i0:]):
                s, t = x.stride(), y.stride()
                _TENSOR.pack_into(buf, at, x.data_ptr(), y.data_ptr(), x.shape[1], 0, s[0], s[1], s[2], t[0], t[1], t[2])
                at += ctypes.sizeof(PolyRotaryTensor)
            check(lib.poly_rotary(PolyRotaryArgs.from_buffer(buf), stream), "poly_rotary")
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, args, *xs):
        inv_freq, positions, ctx.start, cu_seqlens, angles, ctx.interleaved, ctx.factor = args
        # saved, not kept: changing them in place before the backward is an error then, not another gradient
        ctx.save_for_backward(inv_freq, positions, cu_seqlens, angles)
        ctx.dtype = xs[0].dtype
        ctx.set_materialize_grads(False)
        return tuple(_rotate(xs, *args, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *dys):
        # the rotation's transpose: the same launch with sin negated
        live = [i for i, g in enumerate(dys) if g is not None]
        out = [None] * len(dys)
        if live:
            inv_freq, positions, cu_seqlens, angles = ctx.saved_tensors
            for i, g in zip(live, _rotate([dys[i].to(ctx.dtype) for i in live], inv_freq, positions, ctx.start, cu_seqlens, angles,
                                          ctx.interleaved, ctx.factor, True)):
                out[i] = g
        return (None, *out)


# Under torch.compile the rotation is one opaque node with a shape function;
# eager calls skip the dispatcher.
@torch.library.custom_op("poly_b200::rotary", mutates_args=())
def _rotary_op(xs: List[torch.Tensor], inv_freq: Optional[torch.Tensor], positions: Optional[torch.Tensor], start: int,
               cu_seqlens: Optional[torch.Tensor], angles: Optional[torch.Tensor], interleaved: bool, factor: float,
               inverse: bool) -> List[torch.Tensor]:
    return _rotate(xs, inv_freq, positions, start, cu_seqlens, angles, interleaved, factor, inverse)


@_rotary_op.register_fake
def _(xs, inv_freq, positions, start, cu_seqlens, angles, interleaved, factor, inverse):
    return [_empty_like(x) for x in xs]


def _op_setup(ctx, inputs, output):
    xs, inv_freq, positions, ctx.start, cu_seqlens, angles, ctx.interleaved, ctx.factor, ctx.inverse = inputs
    ctx.save_for_backward(inv_freq, positions, cu_seqlens, angles)
    ctx.shapes = [x.shape for x in xs]


def _op_backward(ctx, grads):
    inv_freq, positions, cu_seqlens, angles = ctx.saved_tensors
    live = [i for i, g in enumerate(grads) if g is not None]
    out = [None] * len(grads)
    if live:
        res = _rotary_op([grads[i] for i in live], inv_freq, positions, ctx.start, cu_seqlens, angles, ctx.interleaved,
                         ctx.factor, not ctx.inverse)
        for i, g in zip(live, res):
            out[i] = g
    return out, None, None, None, None, None, None, None, None


_rotary_op.register_autograd(_op_backward, setup_context=_op_setup)


def apply_rotary(xs, inv_freq=None, *, positions=0, cu_seqlens=None, angles=None, interleaved=True, attention_factor=1.0):
    """Rotate queries / keys by their positions; a tensor gives a tensor, a list a list.

    xs: tensors [b, h, n, d] (any strides with a contiguous feature axis; heads
    may differ) or packed [total, h, d], of one dtype, batch and length. The
    first ``rot`` features are rotated, the rest copied.

    The angles are ``position * inv_freq`` (fp32 [rot / 2]; the product is taken
    in 64 bits, so far positions keep their angle) or ``angles`` (fp32 [n, rot / 2] or
    [b, n, rot / 2]). ``positions`` is the first row's position (rows count up from
    it), or an int32 / int64 tensor [n] or [b, n]; with ``cu_seqlens`` (int32 [s + 1],
    packed sequences, batch 1) every sequence counts from 0, and rows behind the last
    count on. ``interleaved`` pairs
    features (2i, 2i + 1), otherwise (i, i + rot / 2). ``attention_factor``
    multiplies cos and sin. Gradients reach xs; frequencies and angles get none.
    """
    single = torch.is_tensor(xs)
    xs = [xs] if single else list(xs)
    if not xs:
        return []
    x0 = xs[0]
    packed = x0.dim() == 3
    if packed:
        xs = [x.transpose(0, 1).unsqueeze(0) if x.dim() == 3 else x for x in xs]
        x0 = xs[0]
    if x0.dim() != 4:
        raise ValueError("apply_rotary takes tensors [b, h, n, d] or [total, h, d]")
    b, _, n, d = x0.shape
    dtype, device = x0.dtype, x0.device
    if device.type != "cuda":
        _require_cuda(x0)
    if dtype not in _DTYPES:
        raise TypeError(f"rotary tensors must be one of {list(_DTYPES)}; got {dtype}")
    grad = False
    for x in xs:
        if x.dtype != dtype:
            raise TypeError(f"rotary tensors must share one dtype; got {[x.dtype for x in xs]}")
        s = x.shape
        if len(s) != 4 or s[0] != b or s[2] != n or s[3] != d or x.device != device:
            _require_cuda(x)
            raise ValueError("rotary tensors must share batch, length, features and device")
        grad = grad or x.requires_grad
    _require_cuda(inv_freq, angles, cu_seqlens)
    if (inv_freq is None) == (angles is None):
        raise ValueError("give either inv_freq or angles")
    _no_tangents(xs, inv_freq, angles)
    table = inv_freq if angles is None else angles
    if table.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("rotary frequencies and angles have no gradient")
    rot = 2 * table.shape[-1]
    if rot == 0 or rot > d or d > 256:
        raise ValueError(f"rotary features ({rot}) must be in [2, {d}] and the head at most 256")
    if table.device != device:
        raise ValueError("rotary frequencies must be on the tensors' device")
    start = 0
    if angles is not None:
        if cu_seqlens is not None or torch.is_tensor(positions) or positions != 0:
            raise ValueError("angles already hold the positions")
        angles = angles.float()
        if angles.dim() == 2:
            angles = angles.unsqueeze(0)
        if angles.dim() != 3 or angles.shape[0] not in (1, b) or angles.shape[1] != n:
            raise ValueError(f"angles must be [{n}, rot / 2] or [{b}, {n}, rot / 2], got {tuple(angles.shape)}")
        if angles.stride(-1) != 1:
            angles = angles.contiguous()
        angles = angles.expand(b, -1, -1)
        positions = None
    else:
        if inv_freq.dim() != 1:
            raise ValueError("inv_freq must be [rot / 2]")
        if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
            inv_freq = inv_freq.float().contiguous()
        if cu_seqlens is not None:
            if torch.is_tensor(positions) or positions != 0:
                raise ValueError("positions and cu_seqlens exclude one another")
            if b != 1:
                raise ValueError("packed sequences (cu_seqlens) are rotated with batch 1")
            cu_seqlens = packed_cu(cu_seqlens, x0)
            if cu_seqlens.shape[0] == 1:
                cu_seqlens = None          # no sequence: rows behind the last one count on, here from 0
            positions = None
        elif torch.is_tensor(positions):
            _require_cuda(positions)
            if positions.dtype not in (torch.int32, torch.int64) or positions.device != x0.device:
                raise TypeError("positions must be an int or an int32 / int64 tensor on the tensors' device")
            if positions.dim() == 1:
                positions = positions.unsqueeze(0)
            if positions.dim() != 2 or positions.shape[0] not in (1, b) or positions.shape[1] != n:
                raise ValueError(f"positions must be [{n}] or [{b}, {n}], got {tuple(positions.shape)}")
            positions = positions.expand(b, -1)
        else:
            start, positions = operator.index(positions), None
    args = (inv_freq, positions, start, cu_seqlens, angles, bool(interleaved), float(attention_factor))
    if b == 0 or n == 0:
        ys = [x.clone() for x in xs]
    elif torch.compiler.is_compiling():
        ys = _rotary_op(xs, *args, False)
    elif grad and torch.is_grad_enabled():
        ys = _Rotary.apply(args, *xs)
    else:
        ys = _rotate(xs, *args, False)
    if packed:
        ys = [y.squeeze(0).transpose(0, 1) for y in ys]
    return ys[0] if single else list(ys)


class RotaryEmbedding(nn.Module):
    """Rotary positions of one head size; ``freqs`` [dim / 2] is a constant (a buffer:
    ``requires_grad_`` of a surrounding module does not reach it), kept in fp32
    whatever dtype that module is cast to (a frequency rounded to 16
    bits is off by whole turns after a few hundred positions)."""

    def __init__(self, dim, *, theta=10000.0, interleaved=True, scaling=None, factor=1.0, original_length=None):
        super().__init__()
        freqs, self.attention_factor = rotary_frequencies(dim, theta=theta, scaling=scaling, factor=factor,
                                                          original_length=original_length)
        self.register_buffer("freqs", freqs)
        self.interleaved = interleaved

    def _apply(self, fn, recurse=True):
        keep = self.freqs
        super()._apply(fn, recurse)
        if self.freqs.dtype != torch.float32:
            self.freqs = keep.float().to(self.freqs.device)
        return self

    def forward(self, xs, positions=0, cu_seqlens=None):
        return apply_rotary(xs, self.freqs, positions=positions, cu_seqlens=cu_seqlens, interleaved=self.interleaved,
                            attention_factor=self.attention_factor)

    def rotate_queries_with_cached_keys(self, q, k):
        """Queries are the last rows of the keys' sequence."""
        if q.shape[-2] == k.shape[-2]:
            return tuple(self([q, k]))
        if q.shape[-2] > k.shape[-2]:
            raise ValueError("more queries than keys")
        return self(q, positions=k.shape[-2] - q.shape[-2]), self(k)


__all__ = ["apply_rotary", "rotary_frequencies", "RotaryEmbedding"]
