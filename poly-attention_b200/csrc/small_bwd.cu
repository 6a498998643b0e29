// Backward of a pass over packed sequences of at most 128 rows: one CTA per
// (sequence, kv head) holds the whole sequence, where the 128-key tcgen05 tiles
// would be mostly padding and their fp32 dQ accumulator most of the traffic.
//
// In 16 x 16 blocks (mma.sync m16n8k16), for every query head of the group:
//   S^T = K Q^T, dP^T = V dO^T; p = 2^(s + bias - lse), ds = p (dp - delta),
//   dbias_j += ds, dV += P^T dO, dK += dS^T Q, dQ = dS K.
// Every sum has a fixed order (no atomics), every output is written once, and delta
// and the log2-domain lse are formed here: one launch and no workspace.
//
// Bound by latency and, next, by the path to memory: per CTA some 10 us of dependent
// loads, products and stores, 12 tensors of the sequence moved through it. So several
// CTAs have to share an SM, global accesses are 16 bytes a lane, and sequences of
// up to 64 and of 65 to 128 rows have a kernel each. 256 sequences of 14001 tokens, 16
// heads of 64 (200 of them up to 64), fp16: 78 + 60 us a pass with the
// value's factors, 74 + 50 without. P and dS in registers of one warp per 16 keys took
// 93 us instead of the 78, four CTAs an SM (64 registers, spills) 88.
#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "mma_sync.cuh"
#include "packed.cuh"

namespace poly {
namespace {
using namespace ms;

constexpr int kMaxN = 128;

struct SmallBwd {
  PolyPassBwdArgs a;
  PackedSeqs pk;
  int rows;   // shared-memory rows: the length bound, padded to 16
};

// delta = dout . out - dlse and -log2 lse of every row, 8 lanes a row and at most U rows a lane,
// their loads issued together; rows past the end, and rows that saw no live key, get p = 0.
template <typename T, int D, int U>
__device__ __forceinline__ void row_sums(const SmallBwd& P, int h, int64_t first, int n, int np, float* sLse, float* sDel) {
  const PolyPassBwdArgs& a = P.a;
  const PolyPassArgs& f = a.fwd;
  const T* gb = (const T*)a.dout + h * a.dout_stride[1] + first * a.dout_stride[2];
  const int row = threadIdx.x >> 3, step = blockDim.x >> 3, lane8 = threadIdx.x & 7;
  float sum[U], l[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = row + u * step;
    sum[u] = 0.f;
    l[u] = r < n ? f.lse[h * f.lse_stride[1] + first + r] : -FLT_MAX;
  }
#pragma unroll
  for (int c = 0; c < D; c += 64) {
    uint4 ov[U], gv[U], lv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row + u * step;
      const int64_t at = h * f.out_stride[1] + (first + r) * f.out_stride[2] + c + lane8 * 8;
      ov[u] = gv[u] = lv[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < n) {
        ov[u] = *reinterpret_cast<const uint4*>((const T*)f.out + at);
        gv[u] = *reinterpret_cast<const uint4*>(gb + (int64_t)r * a.dout_stride[2] + c + lane8 * 8);
        if (P.pk.out_lo) lv[u] = *reinterpret_cast<const uint4*>((const T*)P.pk.out_lo + at);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T *op = reinterpret_cast<const T*>(&ov[u]), *gp = reinterpret_cast<const T*>(&gv[u]);
      const T* lp = reinterpret_cast<const T*>(&lv[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[u] += (to_f32(op[e]) + to_f32(lp[e])) * to_f32(gp[e]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = row + u * step;
    sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 1);
    sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 2);
    sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 4);
    if (lane8 == 0 && r < np) {
      const bool dead = l[u] <= kDeadBias;
      sLse[r] = dead ? -INFINITY : -l[u] * kLog2e;
      sDel[r] = dead ? 0.f : sum[u] - (a.dlse ? a.dlse[h * a.dlse_stride[1] + first + r] : 0.f);
    }
  }
}

// A wrong length bound: every gradient of the sequence is NaN.
__device__ __noinline__ void nan_sequence(const SmallBwd& P, int g, int64_t first, int n) {
  const PolyPassBwdArgs& a = P.a;
  const PackedSeqs& pk = P.pk;
  const int rep = a.fwd.heads / a.fwd.kv_heads, d = a.fwd.head_dim;
  for (int r = 0; r < rep; ++r) packed_nan_rows(a.dq, (g * rep + r) * a.dq_stride[1], a.dq_stride[2], first, n, d);
  packed_nan_rows(a.dk, g * a.dk_stride[1], a.dk_stride[2], first, n, d);
  packed_nan_rows(a.dv, g * a.dv_stride[1], a.dv_stride[2], first, n, d);
  if (pk.v_left) packed_nan_rows(pk.dv_right, g * pk.dv_right_stride[0], pk.dv_right_stride[1], first, n, d);
  for (int i = threadIdx.x; a.dbias && i < n; i += blockDim.x) a.dbias[g * a.dbias_stride[1] + first + i] = NAN;
}

// Probabilities and score gradients of 16 keys x 16 queries: fragments of S^T = K Q^T and dP^T = V dO^T
// in s and dp, p over s and ds (of the scores before the clamp) over dp. k0, k1: the thread's keys,
// b0, b1 their terms of the exponent; db0, db1 collect the bias's gradient.
template <bool SOFTCLAMP>
__device__ __forceinline__ void probabilities(float (&s)[2][4], float (&dp)[2][4], const float* sLse, const float* sDel, int q0,
                                              int k0, int k1, float b0, float b1, bool diag, float qk, float sc_out, float& db0,
                                              float& db1) {
  const int tq = threadIdx.x & 3;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = q0 + nb * 8 + 2 * tq + (e & 1), j = e < 2 ? k0 : k1;
      const float off = sLse[i] + (e < 2 ? b0 : b1);
      float x, slope = 1.f;
      if (SOFTCLAMP) {
        const float th = tanhf(s[nb][e] * qk);
        slope = 1.f - th * th;
        x = fmaf(th, sc_out, off);
      } else {
        x = fmaf(s[nb][e], qk, off);
      }
      if (diag && j > i) x = -INFINITY;
      const float p = tc::ex2(x);
      const float d = p * (dp[nb][e] - sDel[i]);
      if (e < 2) db0 += d; else db1 += d;
      s[nb][e] = p;
      dp[nb][e] = SOFTCLAMP ? d * slope : d;
    }
  }
}

// S^T and dP^T of 16 keys (strip ks) x 16 queries (strip qs)
template <typename T, int D>
__device__ __forceinline__ void scores(float (&s)[2][4], float (&dp)[2][4], uint32_t sK, uint32_t sV, uint32_t sQ, uint32_t sG,
                                       int ks, int qs) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = dp[nb][0] = dp[nb][1] = dp[nb][2] = dp[nb][3] = 0.f;
  // A fragments of K and V; B fragments: queries, features of this step (two n-blocks)
  const int arow = ks * 16 + (lane & 15), row = qs * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const int ach = c * 2 + (lane >> 4), ch = c * 2 + ((lane >> 3) & 1);
    uint32_t ka[4], va[4], x[4];
    ldsm4(sK + soff<D>(arow, ach), ka[0], ka[1], ka[2], ka[3]);
    ldsm4(sV + soff<D>(arow, ach), va[0], va[1], va[2], va[3]);
    ldsm4(sQ + soff<D>(row, ch), x[0], x[1], x[2], x[3]);
    mma<T>(s[0], ka[0], ka[1], ka[2], ka[3], x[0], x[1]);
    mma<T>(s[1], ka[0], ka[1], ka[2], ka[3], x[2], x[3]);
    ldsm4(sG + soff<D>(row, ch), x[0], x[1], x[2], x[3]);
    mma<T>(dp[0], va[0], va[1], va[2], va[3], x[0], x[1]);
    mma<T>(dp[1], va[0], va[1], va[2], va[3], x[2], x[3]);
  }
}

// 32 features of a row of dQ from half hf of accumulator fragments, added to what is there if the caller
// wants that. Every lane of the warp calls; rows that are not live are not touched.
template <typename T>
__device__ __forceinline__ void put_dq(T* row, const float (&o)[4][4], int hf, float scale, bool add, bool live) {
  T* at = row + 8 * (threadIdx.x & 3);
  uint32_t w[4], old[4];
  if (add) {
    quad_load(old, at, live);
    quad_transpose(old);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = o[i][2 * hf] * scale, y = o[i][2 * hf + 1] * scale;
    if (add) {
      const T* e = reinterpret_cast<const T*>(&old[i]);
      x += to_f32(e[0]);
      y += to_f32(e[1]);
    }
    w[i] = pk2<T>(x, y);
  }
  quad_store(at, w, live);
}

// 32 features from c0 of one key's dK and dV, likewise; where the values were a product, its factors
// are loaded before the first store
template <typename T>
__device__ __forceinline__ void put_dkv(const SmallBwd& P, int g, int64_t r, int c0, const float (&dk)[4][4],
                                        const float (&dv)[4][4], int hf, bool live) {
  const PolyPassBwdArgs& a = P.a;
  const PackedSeqs& pk = P.pk;
  const int64_t c = c0 + 8 * (threadIdx.x & 3);
  uint32_t x[4], y[4], w[4];
  if (pk.v_left) {
    quad_load(x, (const T*)pk.v_left + g * pk.v_left_stride[0] + r * pk.v_left_stride[1] + c, live);
    quad_load(y, (const T*)pk.v_right + g * pk.v_right_stride[0] + r * pk.v_right_stride[1] + c, live);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pk2<T>(dk[i][2 * hf] * a.fwd.scale, dk[i][2 * hf + 1] * a.fwd.scale);
  quad_store((T*)a.dk + g * a.dk_stride[1] + r * a.dk_stride[2] + c, w, live);
  T* dvp = (T*)a.dv + g * a.dv_stride[1] + r * a.dv_stride[2] + c;
  if (pk.v_left) {
    quad_transpose(x);
    quad_transpose(y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T *left = reinterpret_cast<const T*>(&x[i]), *right = reinterpret_cast<const T*>(&y[i]);
      const float v0 = dv[i][2 * hf], v1 = dv[i][2 * hf + 1];
      w[i] = pk2<T>(v0 * to_f32(right[0]), v1 * to_f32(right[1]));
      x[i] = pk2<T>(v0 * to_f32(left[0]), v1 * to_f32(left[1]));
    }
    quad_store((T*)pk.dv_right + g * pk.dv_right_stride[0] + r * pk.dv_right_stride[1] + c, x, live);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pk2<T>(dv[i][2 * hf], dv[i][2 * hf + 1]);
  }
  quad_store(dvp, w, live);
}

// Up to 64 rows: eight warps, P and dS of the whole sequence through shared memory. First one
// 16 x 16 block of them per warp and turn; then a warp has 16 rows and 32 features (D / 64 such
// pieces) of dV = P^T dO, dK = dS^T Q and dQ = dS K. Few registers, so that CTAs enough to hide the
// latencies fit an SM.
template <typename T, int D, bool HAS_BIAS, bool SOFTCLAMP>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) small_bwd64_kernel(const __grid_constant__ SmallBwd P) {
  constexpr int CH = D / 8, NF = D / 64, SP = 128;   // SP: bytes of a row of P and dS
  const PolyPassBwdArgs& a = P.a;
  const PolyPassArgs& f = a.fwd;
  const PackedSeqs& pk = P.pk;
  pdl_launch();   // the launch for longer sequences
  if ((int)blockIdx.x >= pk.seqs * f.kv_heads) {   // the CTAs behind the sequences' zero the rows outside them
    packed_zero_rest(pk, blockIdx.x - pk.seqs * f.kv_heads);
    return;
  }
  const int seq = blockIdx.x / f.kv_heads, g = blockIdx.x - seq * f.kv_heads;
  const int64_t first = packed_at(pk.cu, seq, pk.total);
  const int n = packed_at(pk.cu, seq + 1, pk.total) - (int)first;
  if (n > pk.max_len) return nan_sequence(P, g, first, n);
  if (n <= 0 || n > 64) return;
  const int ns = (n + 15) >> 4, np = ns * 16;
  extern __shared__ __align__(16) uint8_t sm[];
  const int tile = P.rows * D * 2;
  uint8_t *pP = sm + 4 * tile, *pS = pP + P.rows * SP;
  float* sLse = reinterpret_cast<float*>(pS + P.rows * SP);   // -lse in the log2 domain
  float* sDel = sLse + P.rows;
  float* sDb = sDel + P.rows;   // [query strip][row]: parts of the bias's gradient
  const uint32_t sK = tc::smem_u32(sm), sV = sK + tile, sQ = sV + tile, sG = sQ + tile, sP = sG + tile, sS = sP + P.rows * SP;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int rep = f.heads / f.kv_heads;

  auto fill = [&](uint32_t dst, const T* src, int64_t stride) {
    for (int c = threadIdx.x; c < np * CH; c += 256) {
      const int r = c / CH, ch = c - r * CH;
      const bool ok = r < n;
      cp16(dst + soff<D>(r, ch), src + (int64_t)(ok ? r : 0) * stride + ch * 8, ok);
    }
  };
  fill(sK, (const T*)f.k + g * f.k_stride[1] + first * f.k_stride[2], f.k_stride[2]);
  fill(sV, (const T*)f.v + g * f.v_stride[1] + first * f.v_stride[2], f.v_stride[2]);
  const float qk = SOFTCLAMP ? f.scale / f.softclamp : f.scale * kLog2e;
  const float sc_out = SOFTCLAMP ? f.softclamp * kLog2e : 0.f;
  const int strip = warp & 3, fg = warp >> 2;   // this warp's rows and features of the gradients
  float dk[NF][4][4], dv[NF][4][4], db = 0.f;   // db: of key threadIdx.x
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) dk[j][i][e] = dv[j][i][e] = 0.f;

  for (int hr = 0; hr < rep; ++hr) {
    const int h = g * rep + hr;
    fill(sQ, (const T*)f.q + h * f.q_stride[1] + first * f.q_stride[2], f.q_stride[2]);
    fill(sG, (const T*)a.dout + h * a.dout_stride[1] + first * a.dout_stride[2], a.dout_stride[2]);
    asm volatile("cp.async.commit_group;" ::: "memory");
    row_sums<T, D, 2>(P, h, first, n, np, sLse, sDel);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    for (int u = warp; u < ns * ns; u += 8) {
      const int ks = u % ns, qs = u / ns, k0 = ks * 16 + gq, k1 = k0 + 8;
      if (f.causal && qs < ks) continue;   // none of these keys seen; the products skip the block too
      // the keys' term of the exponent; -inf (p = 0) for keys past the end and dead ones
      float b0 = k0 < n ? 0.f : -INFINITY, b1 = k1 < n ? 0.f : -INFINITY;
      if (HAS_BIAS) {
        const float* bias = f.bias + g * f.bias_stride[1] + first;
        if (k0 < n) b0 = bias[k0] <= kDeadBias ? -INFINITY : bias[k0] * kLog2e;
        if (k1 < n) b1 = bias[k1] <= kDeadBias ? -INFINITY : bias[k1] * kLog2e;
      }
      float s[2][4], dp[2][4], db0 = 0.f, db1 = 0.f;
      scores<T, D>(s, dp, sK, sV, sQ, sG, ks, qs);
      probabilities<SOFTCLAMP>(s, dp, sLse, sDel, qs * 16, k0, k1, b0, b1, f.causal && ks == qs, qk, sc_out, db0, db1);
      // rounded once, as matrix operands
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int at0 = k0 * SP + (((qs * 2 + hf) ^ (k0 & 7)) << 4) + 4 * tq, at1 = at0 + 8 * SP;   // k1 & 7 == k0 & 7
        *reinterpret_cast<uint32_t*>(pP + at0) = pk2<T>(s[hf][0], s[hf][1]);
        *reinterpret_cast<uint32_t*>(pP + at1) = pk2<T>(s[hf][2], s[hf][3]);
        *reinterpret_cast<uint32_t*>(pS + at0) = pk2<T>(dp[hf][0], dp[hf][1]);
        *reinterpret_cast<uint32_t*>(pS + at1) = pk2<T>(dp[hf][2], dp[hf][3]);
      }
      if (a.dbias) {
        db0 += __shfl_xor_sync(0xffffffffu, db0, 1);
        db0 += __shfl_xor_sync(0xffffffffu, db0, 2);
        db1 += __shfl_xor_sync(0xffffffffu, db1, 1);
        db1 += __shfl_xor_sync(0xffffffffu, db1, 2);
        if (tq == 0) {
          sDb[qs * P.rows + k0] = db0;
          sDb[qs * P.rows + k1] = db1;
        }
      }
    }
    __syncthreads();
    if (a.dbias && (int)threadIdx.x < n)
      for (int qs = f.causal ? (int)threadIdx.x >> 4 : 0; qs < ns; ++qs) db += sDb[qs * P.rows + threadIdx.x];
    if (strip < ns) {
      const int brow = (lane & 7) + ((lane >> 3) & 1) * 8, bch = lane >> 4;
      // dV and dK: keys of this strip, A = P^T and dS^T as stored
      for (int qs = f.causal ? strip : 0; qs < ns; ++qs) {
        const int r = strip * 16 + (lane & 15), ch = qs * 2 + bch;
        const uint32_t at = r * SP + ((ch ^ (r & 7)) << 4);
        uint32_t pa[4], da[4], x[4];
        ldsm4(sP + at, pa[0], pa[1], pa[2], pa[3]);
        ldsm4(sS + at, da[0], da[1], da[2], da[3]);
#pragma unroll
        for (int j = 0; j < NF; ++j) {
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            const uint32_t b = soff<D>(qs * 16 + brow, (fg + 2 * j) * 4 + n2 * 2 + bch);
            ldsm4t(sG + b, x[0], x[1], x[2], x[3]);
            mma<T>(dv[j][2 * n2], pa[0], pa[1], pa[2], pa[3], x[0], x[1]);
            mma<T>(dv[j][2 * n2 + 1], pa[0], pa[1], pa[2], pa[3], x[2], x[3]);
            ldsm4t(sQ + b, x[0], x[1], x[2], x[3]);
            mma<T>(dk[j][2 * n2], da[0], da[1], da[2], da[3], x[0], x[1]);
            mma<T>(dk[j][2 * n2 + 1], da[0], da[1], da[2], da[3], x[2], x[3]);
          }
        }
      }
      // dQ: queries of this strip, A = dS^T read transposed
      T* dq = (T*)a.dq + h * a.dq_stride[1] + first * a.dq_stride[2];
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        float o[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        for (int ks = 0; ks < (f.causal ? strip + 1 : ns); ++ks) {
          const int r = ks * 16 + (lane & 7) + (lane >> 4) * 8, ch = strip * 2 + ((lane >> 3) & 1);
          uint32_t x[4], y[4];
          ldsm4t(sS + r * SP + ((ch ^ (r & 7)) << 4), x[0], x[1], x[2], x[3]);
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            ldsm4t(sK + soff<D>(ks * 16 + brow, (fg + 2 * j) * 4 + n2 * 2 + bch), y[0], y[1], y[2], y[3]);
            mma<T>(o[2 * n2], x[0], x[1], x[2], x[3], y[0], y[1]);
            mma<T>(o[2 * n2 + 1], x[0], x[1], x[2], x[3], y[2], y[3]);
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = strip * 16 + gq + 8 * hf;
          put_dq(dq + (int64_t)row * a.dq_stride[2] + (fg + 2 * j) * 32, o, hf, f.scale, a.dq_accumulate, row < n);
        }
      }
    }
    if (hr + 1 < rep) __syncthreads();   // the next head overwrites Q, dO, P, dS and the row statistics
  }
  if (a.dbias && (int)threadIdx.x < n) a.dbias[g * a.dbias_stride[1] + first + threadIdx.x] = db;
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int row = strip * 16 + gq + 8 * hf;
      put_dkv<T>(P, g, first + row, (fg + 2 * j) * 32, dk[j], dv[j], hf, row < n);
    }
}

// 65 to 128 rows: one warp per 16 keys with its dK and dV in registers, where P of the whole sequence
// beside dS would leave one CTA per SM.
template <typename T, int D, bool HAS_BIAS, bool SOFTCLAMP>
__global__ void __launch_bounds__(2 * kMaxN, D == 64 ? 2 : 1) small_bwd128_kernel(const __grid_constant__ SmallBwd P) {
  constexpr int NF = D / 32, CH = D / 8;
  constexpr int SP = kMaxN * 2;   // bytes of a dS row
  const PolyPassBwdArgs& a = P.a;
  const PolyPassArgs& f = a.fwd;
  const PackedSeqs& pk = P.pk;
  const EndAfterPrevious<true> order;   // started while the launch for up to 64 rows drains; ends after it
  const int seq = blockIdx.x / f.kv_heads, g = blockIdx.x - seq * f.kv_heads;
  const int64_t first = packed_at(pk.cu, seq, pk.total);
  const int n = packed_at(pk.cu, seq + 1, pk.total) - (int)first;
  if (n <= 64 || n > pk.max_len) return;
  const int np = (n + 15) & ~15;
  extern __shared__ __align__(16) uint8_t sm[];
  const int tile = P.rows * D * 2;
  uint8_t *pK = sm, *pV = sm + tile, *pQ = sm + 2 * tile, *pG = sm + 3 * tile, *pS = sm + 4 * tile;   // pS [rows][kMaxN]
  float* sLse = reinterpret_cast<float*>(pS + P.rows * SP);   // -lse in the log2 domain
  float* sDel = sLse + P.rows;
  const uint32_t sK = tc::smem_u32(pK), sV = tc::smem_u32(pV), sQ = tc::smem_u32(pQ), sG = tc::smem_u32(pG), sS = tc::smem_u32(pS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int rep = f.heads / f.kv_heads;

  auto fill = [&](uint32_t dst, const T* src, int64_t stride) {
    for (int c = threadIdx.x; c < np * CH; c += blockDim.x) {
      const int r = c / CH, ch = c - r * CH;
      const bool ok = r < n;
      cp16(dst + soff<D>(r, ch), src + (int64_t)(ok ? r : 0) * stride + ch * 8, ok);
    }
  };
  fill(sK, (const T*)f.k + g * f.k_stride[1] + first * f.k_stride[2], f.k_stride[2]);
  fill(sV, (const T*)f.v + g * f.v_stride[1] + first * f.v_stride[2], f.v_stride[2]);

  const int k0 = warp * 16 + gq, k1 = k0 + 8;   // this thread's two keys
  const bool active = warp * 16 < n;
  // the keys' term of the exponent; -inf (p = 0) for keys past the end and dead ones
  float b0 = k0 < n ? 0.f : -INFINITY, b1 = k1 < n ? 0.f : -INFINITY;
  if (HAS_BIAS) {
    const float* bias = f.bias + g * f.bias_stride[1] + first;
    if (k0 < n) b0 = bias[k0] <= kDeadBias ? -INFINITY : bias[k0] * kLog2e;
    if (k1 < n) b1 = bias[k1] <= kDeadBias ? -INFINITY : bias[k1] * kLog2e;
  }
  const float qk = SOFTCLAMP ? f.scale / f.softclamp : f.scale * kLog2e;
  const float sc_out = SOFTCLAMP ? f.softclamp * kLog2e : 0.f;
  float dk[NF][4][4], dv[NF][4][4], db0 = 0.f, db1 = 0.f;
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) dk[j][i][e] = dv[j][i][e] = 0.f;

  for (int hr = 0; hr < rep; ++hr) {
    const int h = g * rep + hr;
    fill(sQ, (const T*)f.q + h * f.q_stride[1] + first * f.q_stride[2], f.q_stride[2]);
    fill(sG, (const T*)a.dout + h * a.dout_stride[1] + first * a.dout_stride[2], a.dout_stride[2]);
    asm volatile("cp.async.commit_group;" ::: "memory");
    row_sums<T, D, 4>(P, h, first, n, np, sLse, sDel);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    if (active) {
      // causal: queries before this warp's first key see none of its keys (and dQ
      // below reads no such block of dS)
      const int c0 = f.causal ? warp : 0;
      for (int c = c0; c < np / 16; ++c) {
        float s[2][4], ds[2][4];
        scores<T, D>(s, ds, sK, sV, sQ, sG, warp, c);
        probabilities<SOFTCLAMP>(s, ds, sLse, sDel, c * 16, k0, k1, b0, b1, f.causal && c == warp, qk, sc_out, db0, db1);
        // probabilities and score gradients, rounded once as matrix operands
        uint32_t pa[4], da[4];
        pa[0] = pk2<T>(s[0][0], s[0][1]); pa[1] = pk2<T>(s[0][2], s[0][3]);
        pa[2] = pk2<T>(s[1][0], s[1][1]); pa[3] = pk2<T>(s[1][2], s[1][3]);
        da[0] = pk2<T>(ds[0][0], ds[0][1]); da[1] = pk2<T>(ds[0][2], ds[0][3]);
        da[2] = pk2<T>(ds[1][0], ds[1][1]); da[3] = pk2<T>(ds[1][2], ds[1][3]);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int ch = c * 2 + hf;
          *reinterpret_cast<uint32_t*>(pS + k0 * SP + ((ch ^ (k0 & 7)) << 4) + 4 * tq) = da[2 * hf];
          *reinterpret_cast<uint32_t*>(pS + k1 * SP + ((ch ^ (k1 & 7)) << 4) + 4 * tq) = da[2 * hf + 1];
        }
        const int brow = c * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, bch = lane >> 4;
#pragma unroll
        for (int n2 = 0; n2 < 2 * NF; ++n2) {
          uint32_t x[4];
          ldsm4t(sG + soff<D>(brow, n2 * 2 + bch), x[0], x[1], x[2], x[3]);
          mma<T>(dv[n2 / 2][n2 % 2 * 2], pa[0], pa[1], pa[2], pa[3], x[0], x[1]);
          mma<T>(dv[n2 / 2][n2 % 2 * 2 + 1], pa[0], pa[1], pa[2], pa[3], x[2], x[3]);
          ldsm4t(sQ + soff<D>(brow, n2 * 2 + bch), x[0], x[1], x[2], x[3]);
          mma<T>(dk[n2 / 2][n2 % 2 * 2], da[0], da[1], da[2], da[3], x[0], x[1]);
          mma<T>(dk[n2 / 2][n2 % 2 * 2 + 1], da[0], da[1], da[2], da[3], x[2], x[3]);
        }
      }
    }
    __syncthreads();
    if (active) {
      // dQ of queries warp*16 .. + 15: A = dS (stored [key][query], read transposed), B = K
      float o[NF][4][4];
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
      const int kend = f.causal ? warp + 1 : np / 16;
      for (int kk = 0; kk < kend; ++kk) {
        uint32_t x[4], y[4];
        const int r = kk * 16 + (lane & 7) + (lane >> 4) * 8, ch = warp * 2 + ((lane >> 3) & 1);
        ldsm4t(sS + r * SP + ((ch ^ (r & 7)) << 4), x[0], x[1], x[2], x[3]);
        const int brow = kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, bch = lane >> 4;
#pragma unroll
        for (int n2 = 0; n2 < 2 * NF; ++n2) {
          ldsm4t(sK + soff<D>(brow, n2 * 2 + bch), y[0], y[1], y[2], y[3]);
          mma<T>(o[n2 / 2][n2 % 2 * 2], x[0], x[1], x[2], x[3], y[0], y[1]);
          mma<T>(o[n2 / 2][n2 % 2 * 2 + 1], x[0], x[1], x[2], x[3], y[2], y[3]);
        }
      }
      T* dq = (T*)a.dq + h * a.dq_stride[1] + first * a.dq_stride[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int row = hf ? k1 : k0;
#pragma unroll
        for (int j = 0; j < NF; ++j)
          put_dq(dq + (int64_t)row * a.dq_stride[2] + j * 32, o[j], hf, f.scale, a.dq_accumulate, row < n);
      }
    }
    __syncthreads();   // the next head overwrites Q, dO, dS and the row statistics
  }
  if (!active) return;
  db0 += __shfl_xor_sync(0xffffffffu, db0, 1);
  db0 += __shfl_xor_sync(0xffffffffu, db0, 2);
  db1 += __shfl_xor_sync(0xffffffffu, db1, 1);
  db1 += __shfl_xor_sync(0xffffffffu, db1, 2);
  if (a.dbias && tq == 0) {
    float* d = a.dbias + g * a.dbias_stride[1] + first;
    if (k0 < n) d[k0] = db0;
    if (k1 < n) d[k1] = db1;
  }
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int row = hf ? k1 : k0;
#pragma unroll
    for (int j = 0; j < NF; ++j) put_dkv<T>(P, g, first + row, j * 32, dk[j], dv[j], hf, row < n);
  }
}

template <typename T, int D, bool B, bool C>
int launch_t(SmallBwd p, cudaStream_t s) {
  // bytes of one row: K, V, Q, dO, dS (and P and four parts of dbias), lse and delta
  constexpr int row64 = 4 * D * 2 + 2 * 128 + 4 * 4 + 8, row128 = 4 * D * 2 + kMaxN * 2 + 8;
  static std::atomic<uint64_t> done64{0}, done128{0};
  int rc = allow_smem((const void*)small_bwd64_kernel<T, D, B, C>, 64 * row64, done64, "cudaFuncSetAttribute(small bwd)");
  if (!rc) rc = allow_smem((const void*)small_bwd128_kernel<T, D, B, C>, kMaxN * row128, done128, "cudaFuncSetAttribute(small bwd)");
  if (rc) return rc;
  const int rows = p.rows, groups = p.pk.seqs * p.a.fwd.kv_heads;
  p.rows = std::min(rows, 64);
  small_bwd64_kernel<T, D, B, C><<<groups + zero_ctas(p.pk), 256, p.rows * row64, s>>>(p);
  note_launch(1);
  rc = cuda_status(cudaGetLastError(), "small_bwd launch");
  if (rc || rows <= 64) return rc;
  p.rows = rows;
  p.pk.zero.n = 0;   // done by the first launch
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)groups);
  cfg.blockDim = dim3(2 * rows);
  cfg.dynamicSmemBytes = rows * row128;
  cfg.stream = s;
  cudaLaunchAttribute dep = dependent_launch();
  cfg.attrs = &dep;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, small_bwd128_kernel<T, D, B, C>, p);
  note_launch(1);
  return cuda_status(e, "small_bwd launch");
}

template <typename T, int D>
int launch_d(const SmallBwd& p, cudaStream_t s) {
  const bool bias = p.a.fwd.bias != nullptr, sc = p.a.fwd.softclamp > 0.f;
  if (sc) return bias ? launch_t<T, D, true, true>(p, s) : launch_t<T, D, false, true>(p, s);
  return bias ? launch_t<T, D, true, false>(p, s) : launch_t<T, D, false, false>(p, s);
}

}  // namespace

int launch_packed_bwd_small(const PolyPassBwdArgs& a, const PackedSeqs& q, cudaStream_t s) {
  SmallBwd p{a, q, (q.max_len + 15) & ~15};
  if (a.fwd.dtype == POLY_BF16)
    return a.fwd.head_dim == 64 ? launch_d<__nv_bfloat16, 64>(p, s) : launch_d<__nv_bfloat16, 128>(p, s);
  return a.fwd.head_dim == 64 ? launch_d<__half, 64>(p, s) : launch_d<__half, 128>(p, s);
}

}  // namespace poly
