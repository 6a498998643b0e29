// Backward of a pass over packed sequences of at most 128 rows: one CTA per
// (sequence, kv head) holds the whole sequence, where the 128-key tcgen05 tiles
// would be mostly padding and their fp32 dQ accumulator most of the traffic.
//
// One warp per 16 keys (mma.sync m16n8k16). For every query head of the group and
// 16 queries at a time:
//   S^T = K Q^T, dP^T = V dO^T; p = 2^(s + bias - lse), ds = p (dp - delta),
//   dbias_j += ds, dV += P^T dO, dK += dS^T Q (accumulators in registers; the
//   score fragments are the A operands as they are), dS^T -> shared memory;
// then, one warp per 16 queries, dQ = dS K from that tile read transposed. Every sum
// has a fixed order (no atomics), every output is written once, and delta and
// the log2-domain lse are formed here: one launch and no workspace.
//
// Bound by latency: per CTA a few microseconds of dependent loads, products and
// stores, so several CTAs have to share an SM. Sequences of up to 64 and of 65 to
// 128 rows therefore have a launch each (NMAX), the first with half the threads
// and 40 KB of shared memory at d = 64.
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

template <typename T, int D, bool HAS_BIAS, bool SOFTCLAMP, int NMAX>
__global__ void __launch_bounds__(2 * NMAX, D == 64 ? 256 / NMAX : 1) small_bwd_kernel(const __grid_constant__ SmallBwd P) {
  constexpr int KS = D / 16, NB = D / 8, CH = D / 8;
  constexpr int SP = NMAX * 2;   // bytes of a dS row
  const PolyPassBwdArgs& a = P.a;
  const PolyPassArgs& f = a.fwd;
  const PackedSeqs& pk = P.pk;
  // the launch for 65 to 128 rows starts while the one for up to 64 drains (their sequences differ)
  // and ends after it
  if (NMAX == 64) pdl_launch();
  const EndAfterPrevious<NMAX != 64> order;
  if ((int)blockIdx.x >= pk.seqs * f.kv_heads) {   // the CTAs behind the sequences' zero the rows outside them
    packed_zero_rest(pk, blockIdx.x - pk.seqs * f.kv_heads);
    return;
  }
  const int seq = blockIdx.x / f.kv_heads, g = blockIdx.x - seq * f.kv_heads;
  const int64_t first = packed_at(pk.cu, seq, pk.total);
  const int n = packed_at(pk.cu, seq + 1, pk.total) - (int)first;
  if (n > pk.max_len) {   // the caller's bound is wrong: NaN, once
    if constexpr (NMAX == 64) {
      for (int r = 0; r < f.heads / f.kv_heads; ++r)
        packed_nan_rows(a.dq, (g * (f.heads / f.kv_heads) + r) * a.dq_stride[1], a.dq_stride[2], first, n, D);
      packed_nan_rows(a.dk, g * a.dk_stride[1], a.dk_stride[2], first, n, D);
      packed_nan_rows(a.dv, g * a.dv_stride[1], a.dv_stride[2], first, n, D);
      if (pk.v_left) packed_nan_rows(pk.dv_right, g * pk.dv_right_stride[0], pk.dv_right_stride[1], first, n, D);
      for (int i = threadIdx.x; a.dbias && i < n; i += blockDim.x) a.dbias[g * a.dbias_stride[1] + first + i] = NAN;
    }
    return;
  }
  if (n <= 0 || (NMAX == 64 ? n > 64 : n <= 64)) return;
  const int np = (n + 15) & ~15;
  extern __shared__ __align__(16) uint8_t sm[];
  const int tile = P.rows * D * 2;
  uint8_t *pK = sm, *pV = sm + tile, *pQ = sm + 2 * tile, *pG = sm + 3 * tile, *pS = sm + 4 * tile;   // pS [rows][NMAX]
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
  float dk[NB][4], dv[NB][4], db0 = 0.f, db1 = 0.f;
#pragma unroll
  for (int i = 0; i < NB; ++i) dk[i][0] = dk[i][1] = dk[i][2] = dk[i][3] = dv[i][0] = dv[i][1] = dv[i][2] = dv[i][3] = 0.f;

  for (int hr = 0; hr < rep; ++hr) {
    const int h = g * rep + hr;
    const T* gb = (const T*)a.dout + h * a.dout_stride[1] + first * a.dout_stride[2];
    fill(sQ, (const T*)f.q + h * f.q_stride[1] + first * f.q_stride[2], f.q_stride[2]);
    fill(sG, gb, a.dout_stride[2]);
    asm volatile("cp.async.commit_group;" ::: "memory");
    // delta = dout . out - dlse and -log2 lse of every row, 8 lanes a row and at most four rows a
    // lane, their loads issued together; rows past the end, and rows that saw no live key, get p = 0
    {
      const int row = threadIdx.x >> 3, step = blockDim.x >> 3, lane8 = threadIdx.x & 7;
      float sum[4] = {0.f, 0.f, 0.f, 0.f}, l[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = row + u * step;
        l[u] = r < n ? f.lse[h * f.lse_stride[1] + first + r] : -FLT_MAX;
      }
#pragma unroll
      for (int c = 0; c < D; c += 64) {
        uint4 ov[4], gv[4], lv[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = row + u * step;
          const int64_t at = h * f.out_stride[1] + (first + r) * f.out_stride[2] + c + lane8 * 8;
          ov[u] = gv[u] = lv[u] = make_uint4(0u, 0u, 0u, 0u);
          if (r < n) {
            ov[u] = *reinterpret_cast<const uint4*>((const T*)f.out + at);
            gv[u] = *reinterpret_cast<const uint4*>(gb + (int64_t)r * a.dout_stride[2] + c + lane8 * 8);
            if (pk.out_lo) lv[u] = *reinterpret_cast<const uint4*>((const T*)pk.out_lo + at);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const T *op = reinterpret_cast<const T*>(&ov[u]), *gp = reinterpret_cast<const T*>(&gv[u]), *lp = reinterpret_cast<const T*>(&lv[u]);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[u] += (to_f32(op[e]) + to_f32(lp[e])) * to_f32(gp[e]);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
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
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    if (active) {
      // causal: queries before this warp's first key see none of its keys (and dQ
      // below reads no such block of dS)
      const int c0 = f.causal ? warp : 0;
      const int arow = warp * 16 + (lane & 15), ach = lane >> 4;   // A fragments of K and V
      for (int c = c0; c < np / 16; ++c) {
        float s[2][4], dp[2][4];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = dp[nb][0] = dp[nb][1] = dp[nb][2] = dp[nb][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t ka[4], va[4], x[4];
          ldsm4(sK + soff<D>(arow, ks * 2 + ach), ka[0], ka[1], ka[2], ka[3]);
          ldsm4(sV + soff<D>(arow, ks * 2 + ach), va[0], va[1], va[2], va[3]);
          // B fragments: queries c*16 .. + 15, features of this step (two n-blocks)
          const int row = c * 16 + (lane & 7) + (lane >> 4) * 8, ch = ks * 2 + ((lane >> 3) & 1);
          ldsm4(sQ + soff<D>(row, ch), x[0], x[1], x[2], x[3]);
          mma<T>(s[0], ka[0], ka[1], ka[2], ka[3], x[0], x[1]);
          mma<T>(s[1], ka[0], ka[1], ka[2], ka[3], x[2], x[3]);
          ldsm4(sG + soff<D>(row, ch), x[0], x[1], x[2], x[3]);
          mma<T>(dp[0], va[0], va[1], va[2], va[3], x[0], x[1]);
          mma<T>(dp[1], va[0], va[1], va[2], va[3], x[2], x[3]);
        }
        float ds[2][4];
        const bool diag = f.causal && c == warp;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = c * 16 + nb * 8 + 2 * tq + (e & 1), j = e < 2 ? k0 : k1;
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
            ds[nb][e] = SOFTCLAMP ? d * slope : d;
          }
        }
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
        for (int n2 = 0; n2 < NB / 2; ++n2) {
          uint32_t x[4];
          ldsm4t(sG + soff<D>(brow, n2 * 2 + bch), x[0], x[1], x[2], x[3]);
          mma<T>(dv[2 * n2], pa[0], pa[1], pa[2], pa[3], x[0], x[1]);
          mma<T>(dv[2 * n2 + 1], pa[0], pa[1], pa[2], pa[3], x[2], x[3]);
          ldsm4t(sQ + soff<D>(brow, n2 * 2 + bch), x[0], x[1], x[2], x[3]);
          mma<T>(dk[2 * n2], da[0], da[1], da[2], da[3], x[0], x[1]);
          mma<T>(dk[2 * n2 + 1], da[0], da[1], da[2], da[3], x[2], x[3]);
        }
      }
    }
    __syncthreads();
    if (active) {
      // dQ of queries warp*16 .. + 15: A = dS (stored [key][query], read transposed), B = K
      float o[NB][4];
#pragma unroll
      for (int i = 0; i < NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      const int kend = f.causal ? warp + 1 : np / 16;
      for (int kk = 0; kk < kend; ++kk) {
        uint32_t x[4], y[4];
        const int r = kk * 16 + (lane & 7) + (lane >> 4) * 8, ch = warp * 2 + ((lane >> 3) & 1);
        ldsm4t(sS + r * SP + ((ch ^ (r & 7)) << 4), x[0], x[1], x[2], x[3]);
        const int brow = kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, bch = lane >> 4;
#pragma unroll
        for (int n2 = 0; n2 < NB / 2; ++n2) {
          ldsm4t(sK + soff<D>(brow, n2 * 2 + bch), y[0], y[1], y[2], y[3]);
          mma<T>(o[2 * n2], x[0], x[1], x[2], x[3], y[0], y[1]);
          mma<T>(o[2 * n2 + 1], x[0], x[1], x[2], x[3], y[2], y[3]);
        }
      }
      T* dq = (T*)a.dq + h * a.dq_stride[1] + first * a.dq_stride[2];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = hf ? k1 : k0;
          if (row >= n) continue;
          uint32_t* at = reinterpret_cast<uint32_t*>(dq + (int64_t)row * a.dq_stride[2] + i * 8 + 2 * tq);
          float x0 = o[i][2 * hf] * f.scale, x1 = o[i][2 * hf + 1] * f.scale;
          if (a.dq_accumulate) {
            const uint32_t old = *at;
            const T* e = reinterpret_cast<const T*>(&old);
            x0 += to_f32(e[0]);
            x1 += to_f32(e[1]);
          }
          *at = pk2<T>(x0, x1);
        }
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
    if (row >= n) continue;
    const int64_t r = first + row;
    T* dkp = (T*)a.dk + g * a.dk_stride[1] + r * a.dk_stride[2];
    T* dvp = (T*)a.dv + g * a.dv_stride[1] + r * a.dv_stride[2];
    const T* vl = pk.v_left ? (const T*)pk.v_left + g * pk.v_left_stride[0] + r * pk.v_left_stride[1] : nullptr;
    const T* vr = pk.v_left ? (const T*)pk.v_right + g * pk.v_right_stride[0] + r * pk.v_right_stride[1] : nullptr;
    T* dr = pk.v_left ? (T*)pk.dv_right + g * pk.dv_right_stride[0] + r * pk.dv_right_stride[1] : nullptr;
    uint32_t fl[NB], fr[NB];   // the value's factors: loaded before the first store
    if (vl) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        fl[i] = *reinterpret_cast<const uint32_t*>(vl + i * 8 + 2 * tq);
        fr[i] = *reinterpret_cast<const uint32_t*>(vr + i * 8 + 2 * tq);
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int c = i * 8 + 2 * tq;
      *reinterpret_cast<uint32_t*>(dkp + c) = pk2<T>(dk[i][2 * hf] * f.scale, dk[i][2 * hf + 1] * f.scale);
      const float v0 = dv[i][2 * hf], v1 = dv[i][2 * hf + 1];
      if (vl) {
        const T *x = reinterpret_cast<const T*>(&fl[i]), *y = reinterpret_cast<const T*>(&fr[i]);
        *reinterpret_cast<uint32_t*>(dvp + c) = pk2<T>(v0 * to_f32(y[0]), v1 * to_f32(y[1]));
        *reinterpret_cast<uint32_t*>(dr + c) = pk2<T>(v0 * to_f32(x[0]), v1 * to_f32(x[1]));
      } else {
        *reinterpret_cast<uint32_t*>(dvp + c) = pk2<T>(v0, v1);
      }
    }
  }
}

template <typename T, int D, bool B, bool C, int NMAX>
int launch_n(SmallBwd p, cudaStream_t s) {
  constexpr int row = 4 * D * 2 + NMAX * 2 + 8;   // K, V, Q, dO, dS, lse and delta of one row
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_smem((const void*)small_bwd_kernel<T, D, B, C, NMAX>, NMAX * row, done,
                                "cudaFuncSetAttribute(small bwd)")) return rc;
  p.rows = std::min(p.rows, NMAX);
  if (NMAX != 64) p.pk.zero.n = 0;   // done by the first launch
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.pk.seqs * p.a.fwd.kv_heads) + zero_ctas(p.pk));
  cfg.blockDim = dim3(2 * p.rows);
  cfg.dynamicSmemBytes = p.rows * row;
  cfg.stream = s;
  cudaLaunchAttribute dep = dependent_launch();
  cfg.attrs = &dep;
  cfg.numAttrs = NMAX != 64 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, small_bwd_kernel<T, D, B, C, NMAX>, p);
  note_launch(1);
  return cuda_status(e, "small_bwd launch");
}

template <typename T, int D, bool B, bool C>
int launch_t(const SmallBwd& p, cudaStream_t s) {
  const int rc = launch_n<T, D, B, C, 64>(p, s);
  return rc || p.rows <= 64 ? rc : launch_n<T, D, B, C, kMaxN>(p, s);
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
