// Pieces shared by the tcgen05 backward kernels (bwd_tc100.cu: head_dim 64,
// bwd_tc128.cu: head_dim 128): kernel parameters, the per-element softmax
// backward, the dS^T tile store, and the prep / dQ-convert kernels around
// them.
#pragma once

#include "common.cuh"
#include "packed.cuh"
#include "tc_ptx.cuh"

namespace poly {
namespace bwdc {
using namespace tc;

struct BwdParams {
  int seq_q, seq_k, heads, kv_heads, nq_pad, q_tiles, k_tiles, causal;
  float scale, sl2, sc_in, sc_out;
  const float* bias; int64_t bias_stride[2];
  float* dq_acc;                 // [b*heads][seq_q][head_dim] fp32
  const float* lse2;             // [b*heads][nq_pad] log2-domain lse (+inf padding)
  const float* delta;            // [b*heads][nq_pad]
  void* dk; int64_t dk_stride[3];
  void* dv; int64_t dv_stride[3];
  float* dbias; int64_t dbias_stride[2];
  PackedSeqs pk;                 // packed sequences: rows from packed_row0 on in dq_acc, of slots of 128 in lse2 and delta
  const int* order;              // and the slots, longest walk first (NULL: as they are)
};

template <typename T>
__device__ __forceinline__ uint32_t pk(float a, float b);
template <>
__device__ __forceinline__ uint32_t pk<__nv_bfloat16>(float a, float b) { return pack_bf16(a, b); }
template <>
__device__ __forceinline__ uint32_t pk<__half>(float a, float b) { return pack_f16(a, b); }

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer() - t0 > kWaitNs) return;
}

// Writes 32 consecutive 16-bit values (one 32-query chunk c of row r) into a
// [128 rows][128 cols] tile stored as two 128-byte-swizzled 64-column atoms.
__device__ __forceinline__ void store_chunk(uint8_t* tile, int r, int c, const uint32_t (&w)[16]) {
  const int atom = c >> 1;
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4) {
    const int idx = (c & 1) * 4 + q4;
    uint4 val = make_uint4(w[q4 * 4 + 0], w[q4 * 4 + 1], w[q4 * 4 + 2], w[q4 * 4 + 3]);
    *reinterpret_cast<uint4*>(tile + atom * (128 * 128) + r * 128 + ((idx ^ (r & 7)) << 4)) = val;
  }
}

// One 32-query chunk of the softmax backward for this thread's key row.
// x = s * scale * log2(e) + bias - lse (log2 domain), p = 2^x,
// ds = p (dp - delta), d-bias += ds, dS = ds * softclamp'(s). MASK adds the
// causal diagonal (queries il < diag_row) and invalid-key masks; the
// unmasked variant is the common case and carries no per-element selects.
template <typename T, bool SOFTCLAMP, bool HAS_BIAS, bool MASK, bool DB>
__device__ __forceinline__ void softmax_bwd_chunk(const uint32_t (&sv)[32], const uint32_t (&dv)[32],
                                                  const float* nl, const float* dl, float b2, const BwdParams& p,
                                                  bool key_ok, int il0, int diag_row, float& dbias,
                                                  uint32_t (&pw)[16], uint32_t (&dw)[16]) {
  const float4* l4 = reinterpret_cast<const float4*>(nl);
  const float4* d4 = reinterpret_cast<const float4*>(dl);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float4 lq = l4[q], dq = d4[q];
    const float lv[4] = {lq.x, lq.y, lq.z, lq.w};
    const float dd4[4] = {dq.x, dq.y, dq.z, dq.w};
    float pp[4], dd[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int u = q * 4 + e;
      const float sr = __uint_as_float(sv[u]);
      const float off = HAS_BIAS ? lv[e] + b2 : lv[e];
      float x, dfac = 1.f;
      if (SOFTCLAMP) {
        const float th = tanhf(sr * p.sc_in);
        dfac = 1.f - th * th;
        x = fmaf(th, p.sc_out, off);
      } else {
        x = fmaf(sr, p.sl2, off);
      }
      float pr = ex2(x);
      if (MASK && (!key_ok || il0 + u < diag_row)) pr = 0.f;
      const float ds = pr * (__uint_as_float(dv[u]) - dd4[e]);
      if (DB) dbias += ds;   // only when the caller wants the key-bias gradient
      pp[e] = pr;
      dd[e] = SOFTCLAMP ? ds * dfac : ds;
    }
    pw[2 * q] = pk<T>(pp[0], pp[1]);
    pw[2 * q + 1] = pk<T>(pp[2], pp[3]);
    dw[2 * q] = pk<T>(dd[0], dd[1]);
    dw[2 * q + 1] = pk<T>(dd[2], dd[3]);
  }
}

// delta_i = dout_i . out_i - dlse_i and nlse2_i = -lse_i * log2(e), padded to
// nq_pad rows per (batch, head) with (delta 0, nlse2 -inf) so padded queries
// get p = 0. Eight lanes per row, 16-byte loads (D / 64 per lane).
template <typename T, int D>
__global__ void bwd_prep_kernel(const PolyPassBwdArgs a, float* lse2, float* delta, int nq_pad) {
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
  const int sub = threadIdx.x & 7;
  const int64_t rows = (int64_t)a.fwd.batch * a.fwd.heads * nq_pad;
  if (w >= rows) return;
  const int i = (int)(w % nq_pad);
  const int bh = (int)(w / nq_pad);
  const int b = bh / a.fwd.heads, h = bh - b * a.fwd.heads;
  float s = 0.f;
  if (i < a.fwd.seq_q) {
    const T* o = (const T*)a.fwd.out + b * a.fwd.out_stride[0] + h * a.fwd.out_stride[1] +
                 (int64_t)i * a.fwd.out_stride[2] + sub * (D / 8);
    const T* g = (const T*)a.dout + b * a.dout_stride[0] + h * a.dout_stride[1] + (int64_t)i * a.dout_stride[2] +
                 sub * (D / 8);
#pragma unroll
    for (int v8 = 0; v8 < D / 64; ++v8) {
      const uint4 ov = *reinterpret_cast<const uint4*>(o + v8 * 8);
      const uint4 gv = *reinterpret_cast<const uint4*>(g + v8 * 8);
      const T* op = reinterpret_cast<const T*>(&ov);
      const T* gp = reinterpret_cast<const T*>(&gv);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += to_f32(op[e]) * to_f32(gp[e]);
    }
  }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  s += __shfl_xor_sync(0xffffffffu, s, 4);
  if (sub == 0) {
    if (i >= a.fwd.seq_q) {
      lse2[w] = -INFINITY;      // stored negated: padded queries get p = 2^-inf = 0
      delta[w] = 0.f;
    } else {
      if (a.dlse) s -= a.dlse[b * a.dlse_stride[0] + h * a.dlse_stride[1] + i];
      delta[w] = s;
      lse2[w] = -a.fwd.lse[b * a.fwd.lse_stride[0] + h * a.fwd.lse_stride[1] + i] * kLog2e;
    }
  }
}

// dq = scale * dq_acc (+ dq when accumulating), 8 elements per thread.
template <typename T, int D>
__global__ void bwd_dq_convert_kernel(const PolyPassBwdArgs a, const float* dq_acc) {
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t total = (int64_t)a.fwd.batch * a.fwd.heads * a.fwd.seq_q * (D / 8);
  if (idx >= total) return;
  const int c8 = (int)(idx % (D / 8));
  const int64_t row = idx / (D / 8);
  const int i = (int)(row % a.fwd.seq_q);
  const int bh = (int)(row / a.fwd.seq_q);
  const int b = bh / a.fwd.heads, h = bh - b * a.fwd.heads;
  const float* src = dq_acc + row * D + c8 * 8;
  T* dst = (T*)a.dq + b * a.dq_stride[0] + h * a.dq_stride[1] + (int64_t)i * a.dq_stride[2] + c8 * 8;
  const float4 x0 = *reinterpret_cast<const float4*>(src);
  const float4 x1 = *reinterpret_cast<const float4*>(src + 4);
  float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  const float sc = a.fwd.scale;
  if (a.dq_accumulate) {
    const uint4 old = *reinterpret_cast<const uint4*>(dst);
    const uint32_t* ow = &old.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T* pr = reinterpret_cast<const T*>(&ow[e]);
      v[2 * e] = v[2 * e] * sc + to_f32(pr[0]);
      v[2 * e + 1] = v[2 * e + 1] * sc + to_f32(pr[1]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= sc;
  }
  uint4 out;
  uint32_t* w = &out.x;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pk<T>(v[2 * e], v[2 * e + 1]);
  *reinterpret_cast<uint4*>(dst) = out;
}

// Packed sequences. The kernels' row statistics are laid out by slots of 128 rows
// (packed.cuh), so every sequence owns whole tiles of them, 16-byte aligned. The dQ
// accumulator, 64 or 128 times as wide, has whole blocks of 8 rows for a sequence: a
// query tile cut by its sequence's end is added in such blocks, and what its rows past
// the end hold (0 * NaN) lands in rows that nobody reads. So the workspace follows the
// tokens: 160000 of them in 20000 sequences, h16 d64, take 1.7 GB (11.5 GB with dQ in slots).
// One block per 32 rows of a slot and head: delta and -log2 lse as above, and
// the accumulator's rows as zeros. A row that saw no live key gets p = 0.
template <typename T, int D>
__global__ void __launch_bounds__(256) packed_bwd_prep_kernel(const PolyPassBwdArgs a, const PackedSeqs q, float* dq_acc,
                                                              float* lse2, float* delta, int64_t nq_pad, int64_t dq_rows,
                                                              int* order) {
  if (order) {   // CTA 0 of every head is extra: the first sorts the slots
    if (blockIdx.x == 0) {
      if (blockIdx.y == 0) packed_order<128>(q, q.total / 128 + q.seqs, a.fwd.causal != 0, order);
      return;
    }
  }
  const int bx = blockIdx.x - (order ? 1 : 0);
  const int own = (q.total / 128 + q.seqs) * 4;   // the CTAs behind these zero the rows outside the sequences
  if (bx >= own) {
    if (blockIdx.y == 0) packed_zero_rest(q, bx - own);
    return;
  }
  PackedTile t;
  const int slot = bx >> 2;
  if (!packed_tile<128>(q.cu, q.seqs, q.total, slot, t)) return;
  const int h = blockIdx.y, sub = threadIdx.x & 7;
  const int r = (bx & 3) * 32 + (threadIdx.x >> 3);   // row of the slot
  const int i = t.tile * 128 + r;                              // row of the sequence
  const int64_t w = h * nq_pad + (int64_t)slot * 128 + r;
  const bool live = i < t.len;
  const int64_t row = (int64_t)t.start + i;
  float s = 0.f;
  if (live) {
    float* acc = dq_acc + (h * dq_rows + packed_row0(t) + i) * D + sub * (D / 8);
#pragma unroll
    for (int v4 = 0; v4 < D / 32; ++v4) *reinterpret_cast<float4*>(acc + v4 * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
    const T* o = (const T*)a.fwd.out + h * a.fwd.out_stride[1] + row * a.fwd.out_stride[2] + sub * (D / 8);
    const T* g = (const T*)a.dout + h * a.dout_stride[1] + row * a.dout_stride[2] + sub * (D / 8);
    const T* ol = q.out_lo ? (const T*)q.out_lo + h * a.fwd.out_stride[1] + row * a.fwd.out_stride[2] + sub * (D / 8) : nullptr;
#pragma unroll
    for (int v8 = 0; v8 < D / 64; ++v8) {
      const uint4 ov = *reinterpret_cast<const uint4*>(o + v8 * 8);
      const uint4 gv = *reinterpret_cast<const uint4*>(g + v8 * 8);
      uint4 lv = make_uint4(0u, 0u, 0u, 0u);
      if (ol) lv = *reinterpret_cast<const uint4*>(ol + v8 * 8);
      const T* op = reinterpret_cast<const T*>(&ov);
      const T* gp = reinterpret_cast<const T*>(&gv);
      const T* lp = reinterpret_cast<const T*>(&lv);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (to_f32(op[e]) + to_f32(lp[e])) * to_f32(gp[e]);
    }
  }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  s += __shfl_xor_sync(0xffffffffu, s, 4);
  if (sub == 0) {
    const float l = live ? a.fwd.lse[h * a.fwd.lse_stride[1] + row] : -FLT_MAX;
    if (l <= kDeadBias) {
      lse2[w] = -INFINITY;
      delta[w] = 0.f;
    } else {
      if (a.dlse) s -= a.dlse[h * a.dlse_stride[1] + row];
      delta[w] = s;
      lse2[w] = -l * kLog2e;
    }
  }
}

// dq = scale * dq_acc (+ dq), from the accumulator's rows to the sequences'.
template <typename T, int D>
__global__ void __launch_bounds__(256) packed_bwd_dq_kernel(const PolyPassBwdArgs a, const PackedSeqs q,
                                                            const float* dq_acc, int64_t dq_rows) {
  PackedTile t;
  const int slot = blockIdx.x >> 2;
  if (!packed_tile<128>(q.cu, q.seqs, q.total, slot, t)) return;
  const int h = blockIdx.y, r0 = (blockIdx.x & 3) * 32;
  const float sc = a.fwd.scale;
  for (int idx = threadIdx.x; idx < 32 * (D / 8); idx += 256) {
    const int r = r0 + idx / (D / 8), c = (idx % (D / 8)) * 8;
    const int i = t.tile * 128 + r;
    if (i >= t.len) return;
    const float* src = dq_acc + (h * dq_rows + packed_row0(t) + i) * D + c;
    T* dst = (T*)a.dq + h * a.dq_stride[1] + ((int64_t)t.start + i) * a.dq_stride[2] + c;
    const float4 x0 = *reinterpret_cast<const float4*>(src);
    const float4 x1 = *reinterpret_cast<const float4*>(src + 4);
    float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    if (a.dq_accumulate) {
      const uint4 old = *reinterpret_cast<const uint4*>(dst);
      const T* pr = reinterpret_cast<const T*>(&old);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * sc + to_f32(pr[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= sc;
    }
    uint4 out;
    uint32_t* w = &out.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pk<T>(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<uint4*>(dst) = out;
  }
}

struct BwdWs {
  float* dq_acc;
  float* lse2;
  float* delta;
  int nq_pad;
  size_t bytes;
};

// 32 features of dV = a[] as the gradients of a product's two factors (packed
// sequences whose values were v_left * v_right): dv for v_left, dv_right for v_right.
template <typename T>
__device__ __forceinline__ void store_dv_factors(const PackedSeqs& q, int kvh, int64_t row, int col, const uint32_t (&a)[32],
                                                 T* dv) {
  const T* vl = (const T*)q.v_left + kvh * q.v_left_stride[0] + row * q.v_left_stride[1] + col;
  const T* vr = (const T*)q.v_right + kvh * q.v_right_stride[0] + row * q.v_right_stride[1] + col;
  T* dr = (T*)q.dv_right + kvh * q.dv_right_stride[0] + row * q.dv_right_stride[1] + col;
#pragma unroll
  for (int q8 = 0; q8 < 4; ++q8) {
    const uint4 l4 = *reinterpret_cast<const uint4*>(vl + q8 * 8), r4 = *reinterpret_cast<const uint4*>(vr + q8 * 8);
    const T* lp = reinterpret_cast<const T*>(&l4);
    const T* rp = reinterpret_cast<const T*>(&r4);
    uint4 x4, y4;
    uint32_t *xp = &x4.x, *yp = &y4.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float g0 = __uint_as_float(a[q8 * 8 + 2 * e]), g1 = __uint_as_float(a[q8 * 8 + 2 * e + 1]);
      xp[e] = pk<T>(g0 * to_f32(rp[2 * e]), g1 * to_f32(rp[2 * e + 1]));
      yp[e] = pk<T>(g0 * to_f32(lp[2 * e]), g1 * to_f32(lp[2 * e + 1]));
    }
    *reinterpret_cast<uint4*>(dv + q8 * 8) = x4;
    *reinterpret_cast<uint4*>(dr + q8 * 8) = y4;
  }
}

// Workspace: fp32 dQ accumulator [b * heads][seq_q][D], then the log2-domain
// lse and delta rows padded to the query tile BQ.
template <int D, int BQ>
BwdWs bwd_ws(const PolyPassBwdArgs& a) {
  BwdWs w{};
  w.nq_pad = (a.fwd.seq_q + BQ - 1) / BQ * BQ;
  const size_t bh = (size_t)a.fwd.batch * a.fwd.heads;
  const size_t acc = (bh * a.fwd.seq_q * D * 4 + 255) / 256 * 256;
  const size_t vec = (bh * w.nq_pad * 4 + 255) / 256 * 256;
  w.bytes = acc + 2 * vec;
  char* base = (char*)a.workspace;
  w.dq_acc = (float*)base;
  w.lse2 = (float*)(base + acc);
  w.delta = (float*)(base + acc + vec);
  return w;
}

// The same for packed sequences: per head, dq_rows rows of dq_acc and nq_pad rows of slots of the statistics.
struct PackedBwdWs {
  float* dq_acc;
  float* lse2;
  float* delta;
  int* order;
  int slots;
  int64_t nq_pad, dq_rows;
  size_t bytes;
};

inline PackedBwdWs packed_bwd_ws(const PolyPassBwdArgs& a, int seqs) {
  PackedBwdWs w{};
  w.slots = a.fwd.seq_q / 128 + seqs;
  w.nq_pad = (int64_t)w.slots * 128;
  w.dq_rows = packed_rows(a.fwd.seq_q, seqs);
  const size_t rows = (size_t)a.fwd.heads * w.nq_pad, acc = (size_t)a.fwd.heads * w.dq_rows * a.fwd.head_dim;
  const bool sorted = w.slots <= kOrderSlots;
  w.bytes = (acc + rows * 2) * 4 + (sorted ? (size_t)w.slots * 4 : 0);
  w.dq_acc = (float*)a.workspace;
  w.lse2 = w.dq_acc + acc;
  w.delta = w.lse2 + rows;
  w.order = sorted ? (int*)(w.delta + rows) : nullptr;
  return w;
}

}  // namespace bwdc
}  // namespace poly
