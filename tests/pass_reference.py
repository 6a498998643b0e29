"""One attention pass in 64 bits, with the error that a kernel may make.

``forward`` and ``backward`` take 64-bit tensors of one sequence (q [h, i, d],
k / v [g, j, d], bias [g, j]) and return each result with a bound, summed from
the roundings of a kernel that keeps scores, softmax and sums in 32 bits and
multiplies its operands in type T (r = eps(T) / 2; 2^-20 for fp32 operands, whose
3xTF32 products drop lo * lo terms of 2^-22 and carry three roundings):

  score       dx_ij = 2^-20 scale sum|q||k| + 2^-20 |x_ij|   (sums of d products in
              fp32, the scale's, bias's and exponent's roundings)
  log-sum-exp dl_i = max_j dx_ij + 2^-20 (1 + |lse_i|)
  probability p_ij (dx_ij + dl_i), and r p_ij more where it is an operand
  out         sum_j p_ij (dx_ij + dl_i + r) |v_j| + r |out|
  ds          p_ij ((dx_ij + dl_i) |dp - row| + 2^-20 sum|dout||v| + sum|dout| err(out)) and r |ds| as operand
"""
import math

import torch

F32 = 2.0 ** -20


def unit(dtype):
    return F32 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _tiny(dtype, n):
    # probabilities below 2^-25 vanish in fp16; results below its smallest number round to steps of 2^-24
    return n * 2.0 ** -25 if dtype == torch.float16 else 0.0


def scores(q, k, bias, keep, scale, clamp):
    r = q.shape[0] // k.shape[0]
    k = k.repeat_interleave(r, 0)
    s = q @ k.transpose(1, 2) * scale
    size = q.abs() @ k.abs().transpose(1, 2) * abs(scale)
    slope = torch.ones_like(s)
    if clamp:
        th = torch.tanh(s / clamp)
        s, slope = clamp * th, 1 - th * th
        size = size + clamp      # the clamp's own rounding: a few 2^-23 of its value
    x = s if bias is None else s + bias.repeat_interleave(r, 0)[:, None]
    dx = F32 * (size + x.abs())
    if keep is not None:
        x = x.masked_fill(~keep, -math.inf)
        dx = dx.masked_fill(~keep, 0.0)
    return x, dx, slope


def forward(q, k, v, bias, keep, scale, clamp, dtype):
    """(out, tol), (lse, tol), and what backward needs."""
    x, dx, slope = scores(q, k, bias, keep, scale, clamp)
    vr = v.repeat_interleave(q.shape[0] // k.shape[0], 0)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[..., None]).nan_to_num(0.0)
    dl = dx.amax(-1) + F32 * (1 + lse.abs())
    out = p @ vr
    rel = dx + dl[..., None]
    tol = (p * (rel + unit(dtype))) @ vr.abs() + unit(dtype) * out.abs() + _tiny(dtype, k.shape[1]) * (1 + vr.abs().amax())
    return (out, tol), (lse, dl), (p, rel, slope, tol)


def backward(q, k, v, out, dout, dlse, state, scale, clamp, dtype):
    """(dq, tol), (dk, tol), (dv, tol), (dbias, tol); out is the pass's exact result."""
    p, rel, slope, out_tol = state
    h, g = q.shape[0], k.shape[0]
    r, u = h // g, unit(dtype)
    kr, vr = k.repeat_interleave(r, 0), v.repeat_interleave(r, 0)
    group = lambda t: t.view(g, r, *t.shape[1:]).sum(1)   # noqa: E731
    dp = dout @ vr.transpose(1, 2)
    row = (dout * out).sum(-1) - (0 if dlse is None else dlse)
    gap = dp - row[..., None]
    ds = p * gap
    err = p * (rel * gap.abs() + F32 * (dout.abs() @ vr.abs().transpose(1, 2) + row.abs()[..., None])
               + (dout.abs() * out_tol).sum(-1)[..., None])
    tiny = _tiny(dtype, max(p.shape[1], p.shape[2]))
    dz = ds * slope
    ez = err * slope + u * dz.abs() + tiny
    if clamp:
        ez = ez + ds.abs() * 2 * rel / clamp
    ez = ez * scale
    dz = dz * scale
    dq, dk = dz @ kr, group(dz.transpose(1, 2) @ q)
    dv = group(p.transpose(1, 2) @ dout)
    # accumulation of the products in fp32: 2^-20 of the sum of their sizes
    dq_t = (ez + F32 * dz.abs()) @ kr.abs() + u * dq.abs() + tiny
    dk_t = group((ez + F32 * dz.abs()).transpose(1, 2) @ q.abs()) + u * dk.abs() + tiny
    dv_t = group((p * (rel + u + F32) + tiny).transpose(1, 2) @ dout.abs()) + u * dv.abs() + tiny
    db, db_t = group(ds.sum(1)), group((err + F32 * ds.abs()).sum(1))
    return (dq, dq_t), (dk, dk_t), (dv, dv_t), (db, db_t)


def assert_within(got, want, tol, what):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = ((got - want).abs() - tol)
    bad = ~(over <= 0)
    if bad.any():
        i = int(torch.where(bad, over.nan_to_num(math.inf), torch.full_like(over, -math.inf)).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {i}: got {float(got.reshape(-1)[i])}, "
                             f"want {float(want.reshape(-1)[i])}, tolerance {float(tol.reshape(-1)[i])}")
