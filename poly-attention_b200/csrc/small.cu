// Attention pass for short sequences (seq_q, seq_k <= 128): one CTA per
// (batch, head), one warp per 16 query rows. PolyViT's 64-token images
// (poly_vit.py:42-101 calling poly_attention.py:63-114) are the case: there a
// 128 x 128 tcgen05 tile pair would be >85% padding. The whole key range fits
// in shared memory (cp.async, 16-byte chunks XOR-swizzled by row so ldmatrix
// is conflict-free), a row's scores stay in registers, so the softmax needs no
// running rescale: S = Q K^T and O = P V on mma.sync m16n8k16 (fp32
// accumulation), exact row max, one normalisation. Same semantics as the other
// pass kernels: scale, softclamp, causal (top-left aligned), per-key bias in
// the log2 domain with dead keys (bias <= -FLT_MAX / 2) dropped, lse in
// natural-log units.
//
// PACKED: one CTA per (packed sequence, head) where the caller bounds the
// lengths by 128; the CTA takes the rows of its sequence. Sequences of up to 64
// and of 65 to 128 rows have a launch each (NMAX): the warps and score registers
// of 128 rows, idle in a short sequence, left one CTA per SM.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "mma_sync.cuh"
#include "packed.cuh"
#include "tc_ptx.cuh"

namespace poly {
namespace {
using namespace ms;

constexpr int kMaxN = 128;

// A packed sequence's output row: out, its rounding residue, the epilogue's product.
template <typename T>
struct PackedRow {
  T *out, *lo, *eo;
  const T* em;
  __device__ __forceinline__ PackedRow(const PolyPassArgs& a, const PackedSeqs& pk, int h, int64_t first, int row) {
    const int64_t at = h * a.out_stride[1] + row * a.out_stride[2];   // a's pointers are at the sequence
    out = (T*)a.out + at;
    lo = pk.out_lo ? (T*)pk.out_lo + first * a.out_stride[2] + at : nullptr;
    eo = a.epi_out ? (T*)a.epi_out + h * a.epi_out_stride[1] + row * a.epi_out_stride[2] : nullptr;
    em = a.epi_out ? (const T*)a.epi_mul + h * a.epi_mul_stride[1] + row * a.epi_mul_stride[2] : nullptr;
  }
  // Half hf of accumulator fragments o of features c0 .. c0 + 31, times `by`. Every lane of the warp
  // calls; rows that are not live are not touched.
  __device__ __forceinline__ void put(int c0, const float (&o)[4][4], int hf, float by, bool live) const {
    const int c = c0 + 8 * (threadIdx.x & 3);
    uint32_t w[4], m[4], r[4];
    if (eo) quad_load(m, em + c, live);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pk2<T>(o[i][2 * hf] * by, o[i][2 * hf + 1] * by);
    if (lo) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T* e = reinterpret_cast<const T*>(&w[i]);
        r[i] = pk2<T>(o[i][2 * hf] * by - to_f32(e[0]), o[i][2 * hf + 1] * by - to_f32(e[1]));
      }
      quad_store(lo + c, r, live);
    }
    quad_store(out + c, w, live);
    if (eo) {
      quad_transpose(m);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T* e = reinterpret_cast<const T*>(&m[i]);
        r[i] = pk2<T>(o[i][2 * hf] * by * to_f32(e[0]), o[i][2 * hf + 1] * by * to_f32(e[1]));
      }
      quad_store(eo + c, r, live);
    }
  }
};

// packed, d = 64: bound by latency, so six (three) CTAs an SM. 256 sequences of 14001 tokens: 36 us for those of
// up to 64 tokens and 33 for the longer ones (39 at two CTAs, which spills nothing); 37 and 38 with O in one piece
template <typename T, int D, bool HAS_BIAS, bool SOFTCLAMP, bool PACKED, int NMAX>
__global__ void __launch_bounds__(2 * NMAX, D != 64 ? 1 : !PACKED ? 2 : NMAX == 64 ? 6 : 3)
pass_small_kernel(PolyPassArgs a, const PackedSeqs pk) {
  constexpr int KS = D / 16, NB = D / 8, CH = D / 8;
  constexpr int KNB = NMAX / 8;   // key n-blocks
  const int bh = blockIdx.x;
  const int b = PACKED ? 0 : bh / a.heads, h = bh - (PACKED ? bh / a.heads : b) * a.heads;
  int nq = a.seq_q, nk = a.seq_k;
  int64_t first_row = 0;
  // packed: the launch for 65 to 128 rows starts while the one for up to 64 drains (their
  // sequences differ) and ends after it
  if (PACKED && NMAX == 64) pdl_launch();
  const EndAfterPrevious<PACKED && NMAX != 64> order;
  if constexpr (PACKED) {
    if (bh >= pk.seqs * a.heads) {   // the CTAs behind the sequences' zero the rows outside them
      packed_zero_rest(pk, bh - pk.seqs * a.heads);
      return;
    }
    const int first = packed_at(pk.cu, bh / a.heads, pk.total);
    nq = nk = packed_at(pk.cu, bh / a.heads + 1, pk.total) - first;
    if (nk > pk.max_len) {   // the caller's bound is wrong: NaN, once
      if (NMAX != 64) return;
      packed_nan_rows(a.out, h * a.out_stride[1], a.out_stride[2], first, nk, D);
      packed_nan_rows(pk.out_lo, h * a.out_stride[1], a.out_stride[2], first, nk, D);
      packed_nan_rows(a.epi_out, h * a.epi_out_stride[1], a.epi_out_stride[2], first, nk, D);
      for (int i = threadIdx.x; a.lse && i < nk; i += blockDim.x) a.lse[h * a.lse_stride[1] + first + i] = NAN;
      return;
    }
    if (nk <= 0 || (NMAX == 64 ? nk > 64 : nk <= 64)) return;
    const int64_t f = first_row = first;
    a.q = (const T*)a.q + f * a.q_stride[2];
    a.k = (const T*)a.k + f * a.k_stride[2];
    a.v = (const T*)a.v + f * a.v_stride[2];
    a.out = (T*)a.out + f * a.out_stride[2];
    if (HAS_BIAS) a.bias += f;
    if (a.lse) a.lse += f;
    if (a.epi_out) {
      a.epi_mul = (const T*)a.epi_mul + f * a.epi_mul_stride[2];
      a.epi_out = (T*)a.epi_out + f * a.epi_out_stride[2];
    }
  }
  const int kp = (nk + 15) & ~15;   // keys padded to the P.V K step
  // shared memory sized to the keys present: K [kp][D], V [kp][D], bias [kp]
  extern __shared__ __align__(16) uint8_t sm[];
  const uint32_t sK = tc::smem_u32(sm), sV = sK + kp * D * 2;
  float* sB = reinterpret_cast<float*>(sm + 2 * kp * D * 2);

  const int g = h / (a.heads / a.kv_heads);
  const T* kg = (const T*)a.k + b * a.k_stride[0] + g * a.k_stride[1];
  const T* vg = (const T*)a.v + b * a.v_stride[0] + g * a.v_stride[1];
  for (int c = threadIdx.x; c < kp * CH; c += blockDim.x) {
    const int r = c / CH, ch = c - r * CH;
    const bool ok = r < nk;
    const int rr = ok ? r : 0;
    cp16(sK + soff<D>(r, ch), kg + (int64_t)rr * a.k_stride[2] + ch * 8, ok);
    cp16(sV + soff<D>(r, ch), vg + (int64_t)rr * a.v_stride[2] + ch * 8, ok);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (HAS_BIAS)
    for (int j = threadIdx.x; j < kp; j += blockDim.x) {
      float x = -INFINITY;
      if (j < nk) {
        const float raw = a.bias[b * a.bias_stride[0] + g * a.bias_stride[1] + j];
        x = raw <= kDeadBias ? -INFINITY : raw * kLog2e;
      }
      sB[j] = x;
    }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gq = lane >> 2, tq = lane & 3;
  const int r0 = warp * 16 + gq, r1 = r0 + 8;   // this thread's two query rows
  // Q fragments (rows r0 / r1, K step ks): loaded while the keys stream in
  uint32_t qa[KS][4];
  {
    const T* qb = (const T*)a.q + b * a.q_stride[0] + h * a.q_stride[1];
    const T* q0 = qb + (int64_t)(r0 < nq ? r0 : 0) * a.q_stride[2];
    const T* q1 = qb + (int64_t)(r1 < nq ? r1 : 0) * a.q_stride[2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c0 = ks * 16 + 2 * tq;
      qa[ks][0] = r0 < nq ? *reinterpret_cast<const uint32_t*>(q0 + c0) : 0u;
      qa[ks][1] = r1 < nq ? *reinterpret_cast<const uint32_t*>(q1 + c0) : 0u;
      qa[ks][2] = r0 < nq ? *reinterpret_cast<const uint32_t*>(q0 + c0 + 8) : 0u;
      qa[ks][3] = r1 < nq ? *reinterpret_cast<const uint32_t*>(q1 + c0 + 8) : 0u;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  if (warp * 16 >= nq) return;

  // S = Q K^T over every key block; scores of rows r0 (e = 0, 1) and r1 (e = 2, 3)
  float s[KNB][4];
  const float qk = SOFTCLAMP ? a.scale / a.softclamp : a.scale * kLog2e;
  const float sc_out = SOFTCLAMP ? a.softclamp * kLog2e : 0.f;
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int nb = 0; nb < KNB; ++nb) {
    s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
    if (nb * 8 < kp) {
      const int key = nb * 8 + (lane & 7);
#pragma unroll
      for (int ks = 0; ks < KS; ks += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm4(sK + soff<D>(key, ks * 2 + (lane >> 3)), b0, b1, b2, b3);
        mma<T>(s[nb], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
        mma<T>(s[nb], qa[ks + 1][0], qa[ks + 1][1], qa[ks + 1][2], qa[ks + 1][3], b2, b3);
      }
      // packed: scores stay raw without a bias or clamp (the scale, positive here, goes into the
      // exponent's FFMA), and only blocks on the diagonal or at the end test their entries
      const bool plain = PACKED && nb * 8 + 8 <= nk && !(a.causal && nb * 8 + 7 > warp * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = nb * 8 + 2 * tq + (e & 1);
        const int row = e < 2 ? r0 : r1;
        if constexpr (PACKED) {
          float x = s[nb][e];
          if (SOFTCLAMP) x = HAS_BIAS ? fmaf(tanhf(x * qk), sc_out, sB[j]) : tanhf(x * qk) * sc_out;
          else if (HAS_BIAS) x = fmaf(x, qk, sB[j]);
          if (!plain && (j >= nk || (a.causal && j > row))) x = -INFINITY;
          s[nb][e] = x;
          continue;
        }
        float x = s[nb][e] * qk;
        if (SOFTCLAMP) x = tanhf(x) * sc_out;
        if (HAS_BIAS) x += sB[j];
        if (j >= nk || (a.causal && j > row)) x = -INFINITY;
        s[nb][e] = x;
      }
      m0 = fmaxf(m0, fmaxf(s[nb][0], s[nb][1]));
      m1 = fmaxf(m1, fmaxf(s[nb][2], s[nb][3]));
    }
  }
  m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
  m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
  float l0 = 0.f, l1 = 0.f;
  const float mul = PACKED && !HAS_BIAS && !SOFTCLAMP ? qk : 1.f;
  if (PACKED) {
    m0 *= mul;
    m1 *= mul;
  }
  const float s0 = m0 == -INFINITY ? 0.f : m0, s1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
  for (int nb = 0; nb < KNB; ++nb) {
    if (nb * 8 < kp) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (PACKED) {
          const float p = tc::ex2(fmaf(s[nb][e], mul, e < 2 ? -s0 : -s1));
          s[nb][e] = p;
          if (e < 2) l0 += p; else l1 += p;
          continue;
        }
        const float m = e < 2 ? m0 : m1;
        const float p = s[nb][e] == -INFINITY ? 0.f : exp2f(s[nb][e] - m);
        s[nb][e] = p;
        if (e < 2) l0 += p; else l1 += p;
      }
    }
  }
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

  if constexpr (PACKED) {
    // P as operands first, then O 32 features at a time, written as it is done: scores and O
    // never live together, which leaves registers for more CTAs per SM
    uint32_t pa[NMAX / 16][4];
#pragma unroll
    for (int kk = 0; kk < NMAX / 16; ++kk) {
      pa[kk][0] = pk2<T>(s[2 * kk][0], s[2 * kk][1]);
      pa[kk][1] = pk2<T>(s[2 * kk][2], s[2 * kk][3]);
      pa[kk][2] = pk2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
      pa[kk][3] = pk2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
    }
    const float j0 = l0 > 0.f ? 1.f / l0 : 0.f, j1 = l1 > 0.f ? 1.f / l1 : 0.f;
    const PackedRow<T> row0(a, pk, h, first_row, r0), row1(a, pk, h, first_row, r1);
#pragma unroll
    for (int n4 = 0; n4 < NB; n4 += 4) {
      float o[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < NMAX / 16; ++kk) {
        if (kk * 16 < kp) {
          const int vkey = kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            uint32_t v0, v1, v2, v3;
            ldsm4t(sV + soff<D>(vkey, n4 + n2 * 2 + (lane >> 4)), v0, v1, v2, v3);
            mma<T>(o[2 * n2], pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3], v0, v1);
            mma<T>(o[2 * n2 + 1], pa[kk][0], pa[kk][1], pa[kk][2], pa[kk][3], v2, v3);
          }
        }
      }
      row0.put(n4 * 8, o, 0, j0, r0 < nq);
      row1.put(n4 * 8, o, 1, j1, r1 < nq);
    }
    if (a.lse && tq == 0) {
      float* lb = a.lse + h * a.lse_stride[1];
      if (r0 < nq) lb[r0] = l0 == 0.f ? -FLT_MAX : (m0 + __log2f(l0)) * kLn2;
      if (r1 < nq) lb[r1] = l1 == 0.f ? -FLT_MAX : (m1 + __log2f(l1)) * kLn2;
    }
  } else {
    // O = P V, K steps of 16 keys (P from the score registers, V via ldmatrix.trans)
    float o[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < NMAX / 16; ++kk) {
      if (kk * 16 < kp) {
        const uint32_t pa0 = pk2<T>(s[2 * kk][0], s[2 * kk][1]), pa1 = pk2<T>(s[2 * kk][2], s[2 * kk][3]);
        const uint32_t pa2 = pk2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
        const uint32_t pa3 = pk2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
        const int vkey = kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int n2 = 0; n2 < NB / 2; ++n2) {
          uint32_t v0, v1, v2, v3;
          ldsm4t(sV + soff<D>(vkey, n2 * 2 + (lane >> 4)), v0, v1, v2, v3);
          mma<T>(o[2 * n2], pa0, pa1, pa2, pa3, v0, v1);
          mma<T>(o[2 * n2 + 1], pa0, pa1, pa2, pa3, v2, v3);
        }
      }
    }
    bool fb0 = false, fb1 = false;   // row took the fully-excluded result
    // A row whose every key is excluded (only dead keys can do that here) gets
    // the reference's -finfo.max result: the uniform average over the keys that
    // are not both causally masked and dead, lse = -FLT_MAX.
    if (HAS_BIAS && (m0 == -INFINITY || m1 == -INFINITY)) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int row = hf ? r1 : r0;
        if ((hf ? m1 : m0) != -INFINITY) continue;
        int count = 0;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[n][2 * hf] = o[n][2 * hf + 1] = 0.f;
        for (int j = 0; j < nk; ++j) {
          if (a.causal && j > row && sB[j] == -INFINITY) continue;
          ++count;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(sm + kp * D * 2 + soff<D>(j, n) + 4 * tq);
            const T* e = reinterpret_cast<const T*>(&w);
            o[n][2 * hf] += to_f32(e[0]);
            o[n][2 * hf + 1] += to_f32(e[1]);
          }
        }
        if (hf) { l1 = (float)count; fb1 = true; } else { l0 = (float)count; fb0 = true; }
      }
    }
    const float j0 = l0 > 0.f ? 1.f / l0 : 0.f, j1 = l1 > 0.f ? 1.f / l1 : 0.f;
    T* ob = (T*)a.out + b * a.out_stride[0] + h * a.out_stride[1];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int c = n * 8 + 2 * tq;
      if (r0 < nq) *reinterpret_cast<uint32_t*>(ob + (int64_t)r0 * a.out_stride[2] + c) = pk2<T>(o[n][0] * j0, o[n][1] * j0);
      if (r1 < nq) *reinterpret_cast<uint32_t*>(ob + (int64_t)r1 * a.out_stride[2] + c) = pk2<T>(o[n][2] * j1, o[n][3] * j1);
    }
    if (a.lse && tq == 0) {
      float* lb = a.lse + b * a.lse_stride[0] + h * a.lse_stride[1];
      if (r0 < nq) lb[r0] = fb0 ? -FLT_MAX : (m0 + __log2f(l0)) * kLn2;
      if (r1 < nq) lb[r1] = fb1 ? -FLT_MAX : (m1 + __log2f(l1)) * kLn2;
    }
  }
}

template <typename T, int D, bool B, bool C, bool PACKED, int NMAX>
int launch_n(const PolyPassArgs& a, const PackedSeqs* pk, cudaStream_t s) {
  constexpr int smem = 2 * NMAX * D * 2 + NMAX * 4;
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_smem((const void*)pass_small_kernel<T, D, B, C, PACKED, NMAX>, smem, done,
                                "cudaFuncSetAttribute(small)")) return rc;
  const int nq = PACKED ? std::min(pk->max_len, NMAX) : a.seq_q, nk = PACKED ? nq : a.seq_k;
  const int threads = 32 * ((nq + 15) / 16);
  const int kp = (nk + 15) & ~15;
  const int bytes = 2 * kp * D * 2 + kp * 4;   // <= smem (the attribute's maximum)
  PackedSeqs q{};
  if (PACKED) q = *pk;
  if (PACKED && NMAX != 64) q.zero.n = 0;   // done by the first launch
  const unsigned grid = (unsigned)((PACKED ? pk->seqs : a.batch) * a.heads) + zero_ctas(q);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute dep = dependent_launch();
  cfg.attrs = &dep;
  cfg.numAttrs = PACKED && NMAX != 64 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, pass_small_kernel<T, D, B, C, PACKED, NMAX>, a, q);
  note_launch(1);
  return cuda_status(e, "pass_small launch");
}

template <typename T, int D, bool B, bool C, bool PACKED>
int launch_t(const PolyPassArgs& a, const PackedSeqs* pk, cudaStream_t s) {
  if (PACKED) {
    const int rc = launch_n<T, D, B, C, true, 64>(a, pk, s);
    if (rc || pk->max_len <= 64) return rc;
  } else if (a.seq_q <= 64 && a.seq_k <= 64) {
    // half the score registers: an order-2 forward of 256 x 64 tokens, 16 heads, in 95 us at d = 64 (108 with those
    // of 128 keys) and 168 us at d = 128 (235)
    return launch_n<T, D, B, C, false, 64>(a, pk, s);
  }
  return launch_n<T, D, B, C, PACKED, kMaxN>(a, pk, s);
}

template <typename T, int D, bool PACKED>
int launch_d(const PolyPassArgs& a, const PackedSeqs* pk, cudaStream_t s) {
  const bool bias = a.bias != nullptr, sc = a.softclamp > 0.f;
  if (sc) return bias ? launch_t<T, D, true, true, PACKED>(a, pk, s) : launch_t<T, D, false, true, PACKED>(a, pk, s);
  return bias ? launch_t<T, D, true, false, PACKED>(a, pk, s) : launch_t<T, D, false, false, PACKED>(a, pk, s);
}

template <bool PACKED>
int launch_any(const PolyPassArgs& a, const PackedSeqs* pk, cudaStream_t s) {
  if (a.dtype == POLY_BF16)
    return a.head_dim == 64 ? launch_d<__nv_bfloat16, 64, PACKED>(a, pk, s) : launch_d<__nv_bfloat16, 128, PACKED>(a, pk, s);
  return a.head_dim == 64 ? launch_d<__half, 64, PACKED>(a, pk, s) : launch_d<__half, 128, PACKED>(a, pk, s);
}

bool al(const void* p, int bytes) { return ((uintptr_t)p % bytes) == 0; }

}  // namespace

bool pass_small_eligible(const PolyPassArgs& a) {
  if (a.seq_q < 1 || a.seq_q > kMaxN || a.seq_k < 1 || a.seq_k > kMaxN) return false;
  if (a.dtype != POLY_BF16 && a.dtype != POLY_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  if (a.key_mask || a.query_mask || a.v_mul || a.epi_out) return false;
  if (!al(a.k, 16) || !al(a.v, 16) || !al(a.q, 4) || !al(a.out, 4)) return false;
  if ((a.k_stride[0] | a.k_stride[1] | a.k_stride[2] | a.v_stride[0] | a.v_stride[1] | a.v_stride[2]) & 7)
    return false;
  if ((a.q_stride[0] | a.q_stride[1] | a.q_stride[2] | a.out_stride[0] | a.out_stride[1] | a.out_stride[2]) & 1)
    return false;
  return true;
}

int launch_pass_small(const PolyPassArgs& a, cudaStream_t s) { return launch_any<false>(a, nullptr, s); }
int launch_packed_fwd_small(const PolyPassArgs& a, const PackedSeqs& q, cudaStream_t s) {
  return launch_any<true>(a, &q, s);
}

}  // namespace poly
