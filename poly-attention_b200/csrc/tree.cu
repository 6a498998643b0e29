// Decoding passes over trees of drafted tokens (contract: poly_attention.h).
//
// A pass has M = nodes * R rows per (sequence, kv head), R query heads sharing a
// kv head, against lengths[b] + nodes keys. For the trees of speculative decoding
// the cache is read once and everything else is small beside it: HBM-bound like
// the single-token decode kernel, until M reaches some hundred rows.
//
// Up to 32 rows, and where values are a product, tree_kernel here; more rows go to
// the tcgen05 kernel of tree_tc100.cu.
//
// tree_kernel (16-bit, d = 64 / 128): a CTA takes 16 WR rows (WR = 1, 2, 4) of one
// (sequence, kv head) and one of `splits` key ranges. Warp 4 fills a ring of
// 64-key stages with TMA (128-byte swizzle) and the bias by cp.async; warps 0-3
// form a WR x 4 / WR grid, each 16 rows by 16 WR keys of a stage: S = Q K^T and
// O += P V' on mma.sync m16n8k16, online softmax in the log2 domain with a lazy
// maximum. Few rows are spread over the keys, many rows over the warps, so no
// product is spent on padding while there are 64 rows to fill. The warps' states
// merge in shared memory; up to 8 splits are a cluster and join through distributed
// shared memory, more (few groups, a long cache) go through the workspace and
// tree_combine_kernel. Key ranges follow the lengths on the device, so the grid
// needs the capacity only.
//
// The kernels of a step are programmatic dependents of one another: a pass
// streams the cached rows while its predecessor drains, and waits for it
// (griddepcontrol.wait) before it loads the first tile with a row >= lengths[b],
// and before it writes anything.
//
// tree_simt_kernel serves the other types and head sizes: one warp per row, 32-key
// tiles in shared memory, fp32.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "mma_sync.cuh"
#include "tc_host.cuh"
#include "tc_ptx.cuh"
#include "tree_common.cuh"

namespace cg = cooperative_groups;

namespace poly {

static __device__ int g_tree_error[2] = {0, 0};

int read_device_error_tree(int* out, bool reset) {
  int rc = cuda_status(cudaMemcpyFromSymbol(out, g_tree_error, sizeof(int)), "read device error word");
  if (rc == POLY_OK && reset) {
    const int zero = 0;
    rc = cuda_status(cudaMemcpyToSymbol(g_tree_error, &zero, sizeof(int)), "reset device error word");
  }
  return rc;
}

namespace {
using namespace treec;

constexpr int kKeys = 64;                     // keys per stage
constexpr int kWarps = 4;                     // consumer warps
constexpr int kThreads = (kWarps + 1) * 32;

template <int D, int NARR>
struct Ring {
  static constexpr int kArr = kKeys * D * 2;
  static constexpr int kStage = NARR * kArr;
  // ~100 KB a CTA: two CTAs per SM
  static constexpr int kStages = 100 * 1024 / kStage > 4 ? 4 : 100 * 1024 / kStage;
  static constexpr int kRecords = 2 * kWarps * 16 * kRecord<D> * 4;   // the warps' and the CTA's records reuse the ring
  static constexpr int kBias = kStages * kStage > kRecords ? kStages * kStage : kRecords;
  static constexpr int kMask = kBias + kStages * kKeys * 4;
  static constexpr int kUp = kMask + kNodes * 8;
  static constexpr int kBar = kUp + kNodes * 4;
  static constexpr int kBytes = kBar + 2 * kStages * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
};

__device__ __forceinline__ void cp_async4(uint32_t sa, const void* gmem, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sa), "l"(gmem), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = tc::globaltimer();
  while (!tc::mbar_try_wait(bar, parity))
    if (tc::globaltimer() - t0 > tc::kWaitNs) return;
}
template <typename T>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {   // one rounding: the product is exact in 32 bits
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 p = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&p);
  } else {
    const __half2 p = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&p);
  }
}
// 16-byte chunk ch of key row key in a TMA-swizzled array (boxes of 64 features)
__device__ __forceinline__ uint32_t swz(int key, int ch) {
  return (uint32_t)((ch >> 3) * (kKeys * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
}

template <typename T, int D, int WR, bool VMUL>
__global__ void __launch_bounds__(kThreads, 2) tree_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                        const __grid_constant__ CUtensorMap tm_v,
                                                        const __grid_constant__ CUtensorMap tm_m,
                                                        const __grid_constant__ PolyTreePass a, const TreeGeom geo) {
  using R_ = Ring<D, VMUL ? 3 : 2>;
  constexpr int NST = R_::kStages, KS = D / 16, NB = D / 8;
  constexpr int WK = kWarps / WR, KW = kKeys / WK, NKB = KW / 8;   // keys of a warp in a stage, in n8 blocks
  extern __shared__ uint8_t dsm_raw[];
  uint8_t* dsm = dsm_raw + ((1024 - (tc::smem_u32(dsm_raw) & 1023)) & 1023);
  const uint32_t sbase = tc::smem_u32(dsm);
  float* sbias = reinterpret_cast<float*>(dsm + R_::kBias);
  uint64_t* anc = reinterpret_cast<uint64_t*>(dsm + R_::kMask);
  uint64_t* full = reinterpret_cast<uint64_t*>(dsm + R_::kBar);
  uint64_t* empty = full + NST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + NST);
  int* err = g_tree_error;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int split = blockIdx.x % geo.splits, rb = blockIdx.x / geo.splits;
  const int b = blockIdx.y / a.kv_heads, g = blockIdx.y - b * a.kv_heads;
  const int R = a.heads / a.kv_heads, rows = R * a.nodes;
  const int len = seq_length(a.lengths, b, a.capacity);
  const int nkeys = min(len + a.nodes, a.capacity);
  const int tiles = (nkeys + kKeys - 1) / kKeys;
  const int t0 = (int)((int64_t)tiles * split / geo.splits), t1 = (int)((int64_t)tiles * (split + 1) / geo.splits);

  pdl_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      tc::mbar_init(&full[s], a.bias ? 33 : 1);   // producer lane 0 (+ tx), + 32 bias lanes
      tc::mbar_init(&empty[s], kWarps);
    }
    tc::abort_init(abort_flag, err);
    tc::fence_barrier_init();
  }
  ancestors(a.parents + b * a.parents_stride, a.nodes, a.capacity - len, anc, reinterpret_cast<int*>(dsm + R_::kUp));

  const int wr = warp % WR, wk = warp / WR;
  const int m0 = rb * 16 * WR + wr * 16 + gq, m1 = m0 + 8;   // this thread's two rows of the group
  float mx0 = -INFINITY, mx1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float o[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    const float* bg = a.bias ? a.bias + b * a.bias_stride[0] + g * a.bias_stride[1] : nullptr;
    bool waited = false;
    int issued = 0;
    for (int t = 0; t < t1 - t0; ++t) {
      const int s = t % NST, kb = (t0 + t) * kKeys;
      if (t >= NST && !tc::mbar_wait_warp(&empty[s], ((t / NST) - 1) & 1, abort_flag, err, 71)) break;
      if (!waited && kb + kKeys > len) {   // rows that the previous kernels of the step write
        pdl_wait();
        waited = true;
      }
      uint8_t* st = dsm + s * R_::kStage;
      if (lane == 0) {
        tc::mbar_arrive_expect_tx(&full[s], R_::kStage);
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
          tc::tma_load_4d(st + hf * (kKeys * 128), &tm_k, &full[s], hf * 64, kb, g, b);
          tc::tma_load_4d(st + R_::kArr + hf * (kKeys * 128), &tm_v, &full[s], hf * 64, kb, g, b);
          if (VMUL) tc::tma_load_4d(st + 2 * R_::kArr + hf * (kKeys * 128), &tm_m, &full[s], hf * 64, kb, g, b);
        }
      }
      if (bg) {
#pragma unroll
        for (int e = 0; e < kKeys / 32; ++e) {
          const int kl = lane + 32 * e, j = kb + kl;
          cp_async4(tc::smem_u32(sbias + s * kKeys + kl), bg + (j < nkeys ? j : 0), j < nkeys);
        }
        cp_async_arrive(&full[s]);
      }
      issued = t + 1;
    }
    if (*abort_flag) {   // let every copy in flight land before the CTA moves on
      for (int t = max(0, issued - NST); t < issued; ++t) drain_wait(&full[t % NST], (t / NST) & 1);
    }
  } else {
    // ------------------------------------------------------------ consumers
    uint32_t qa[KS][4];
    const int i0 = min(m0, rows - 1), i1 = min(m1, rows - 1);
    const uint64_t see0 = m0 < rows ? anc[i0 / R] : 0ull, see1 = m1 < rows ? anc[i1 / R] : 0ull;
    {
      const T* q = (const T*)a.q + b * a.q_stride[0];
      const T* q0 = q + (int64_t)(g * R + i0 % R) * a.q_stride[1] + (int64_t)(i0 / R) * a.q_stride[2];
      const T* q1 = q + (int64_t)(g * R + i1 % R) * a.q_stride[1] + (int64_t)(i1 / R) * a.q_stride[2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qa[ks][0] = *reinterpret_cast<const uint32_t*>(q0 + ks * 16 + 2 * tq);
        qa[ks][1] = *reinterpret_cast<const uint32_t*>(q1 + ks * 16 + 2 * tq);
        qa[ks][2] = *reinterpret_cast<const uint32_t*>(q0 + ks * 16 + 8 + 2 * tq);
        qa[ks][3] = *reinterpret_cast<const uint32_t*>(q1 + ks * 16 + 8 + 2 * tq);
      }
    }
    const bool clamp = a.softclamp > 0.f;
    const float qk = clamp ? a.scale / a.softclamp : a.scale * kLog2e, sc_out = a.softclamp * kLog2e;
    for (int t = 0; t < t1 - t0; ++t) {
      const int s = t % NST, kb = (t0 + t) * kKeys;
      if (!tc::mbar_wait_warp(&full[s], (t / NST) & 1, abort_flag, err, 72)) break;
      const uint32_t sK = sbase + s * R_::kStage, sV = sK + R_::kArr, sM = sV + R_::kArr;
      float x[NKB][4];
#pragma unroll
      for (int nb = 0; nb < NKB; ++nb) {
        x[nb][0] = x[nb][1] = x[nb][2] = x[nb][3] = 0.f;
        const int key = wk * KW + nb * 8 + (lane & 7);
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          uint32_t b0, b1, b2, b3;
          ms::ldsm4(sK + swz(key, ks * 2 + (lane >> 3)), b0, b1, b2, b3);
          ms::mma<T>(x[nb], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
          ms::mma<T>(x[nb], qa[ks + 1][0], qa[ks + 1][1], qa[ks + 1][2], qa[ks + 1][3], b2, b3);
        }
      }
      const bool tail = kb + kKeys > len;   // holds rows of the tree, or past it
      float t0m = -INFINITY, t1m = -INFINITY;
#pragma unroll
      for (int nb = 0; nb < NKB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kl = wk * KW + nb * 8 + 2 * tq + (e & 1);
          float v = x[nb][e] * qk;
          if (clamp) v = tanhf(v) * sc_out;
          if (a.bias) {
            const float braw = sbias[s * kKeys + kl];
            v = braw <= kDeadBias ? -INFINITY : v + braw * kLog2e;
          }
          if (tail) {
            const int node = kb + kl - len;
            if (node >= 0 && (node >= kNodes || !(((e < 2 ? see0 : see1) >> node) & 1))) v = -INFINITY;
          }
          if (e < 2 ? !see0 : !see1) v = -INFINITY;   // padding
          x[nb][e] = v;
          if (e < 2) t0m = fmaxf(t0m, v); else t1m = fmaxf(t1m, v);
        }
      }
      t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, 1));
      t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, 2));
      t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, 1));
      t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, 2));
      // the reference maximum moves when the row's grows by more than 2^8 (the sums stay exact)
      if (t0m > mx0 + 8.f) {
        const float f = mx0 == -INFINITY ? 0.f : exp2f(mx0 - t0m);
        mx0 = t0m;
        l0 *= f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[n][0] *= f;
          o[n][1] *= f;
        }
      }
      if (t1m > mx1 + 8.f) {
        const float f = mx1 == -INFINITY ? 0.f : exp2f(mx1 - t1m);
        mx1 = t1m;
        l1 *= f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[n][2] *= f;
          o[n][3] *= f;
        }
      }
#pragma unroll
      for (int nb = 0; nb < NKB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = x[nb][e] == -INFINITY ? 0.f : tc::ex2(x[nb][e] - (e < 2 ? mx0 : mx1));
          x[nb][e] = p;
          if (e < 2) l0 += p; else l1 += p;
        }
      const bool cut = kb + kKeys > nkeys;   // rows past the tree hold whatever was there: 0 * NaN
#pragma unroll
      for (int kk = 0; kk < KW / 16; ++kk) {
        const uint32_t pa0 = ms::pk2<T>(x[2 * kk][0], x[2 * kk][1]), pa1 = ms::pk2<T>(x[2 * kk][2], x[2 * kk][3]);
        const uint32_t pa2 = ms::pk2<T>(x[2 * kk + 1][0], x[2 * kk + 1][1]);
        const uint32_t pa3 = ms::pk2<T>(x[2 * kk + 1][2], x[2 * kk + 1][3]);
        const int k16 = wk * KW + kk * 16, vkey = k16 + (lane & 7) + ((lane >> 3) & 1) * 8;
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;   // this thread's key pairs of a B fragment
        if (cut) {
          const int j = kb + k16 + 2 * tq;
          keep0 = (j < nkeys ? 0xffffu : 0u) | (j + 1 < nkeys ? 0xffff0000u : 0u);
          keep1 = (j + 8 < nkeys ? 0xffffu : 0u) | (j + 9 < nkeys ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int n2 = 0; n2 < NB / 2; ++n2) {
          const uint32_t off = swz(vkey, n2 * 2 + (lane >> 4));
          uint32_t v[4];
          ms::ldsm4t(sV + off, v[0], v[1], v[2], v[3]);
          if (VMUL) {
            uint32_t w[4];
            ms::ldsm4t(sM + off, w[0], w[1], w[2], w[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = mul2<T>(v[e], w[e]);
          }
          if (cut) {
            v[0] &= keep0;
            v[1] &= keep1;
            v[2] &= keep0;
            v[3] &= keep1;
          }
          ms::mma<T>(o[2 * n2], pa0, pa1, pa2, pa3, v[0], v[1]);
          ms::mma<T>(o[2 * n2 + 1], pa0, pa1, pa2, pa3, v[2], v[3]);
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[s]);
    }
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  }
  __syncthreads();   // the ring is idle (every issued stage consumed or drained): it takes the warps' records
  constexpr int RS = kRecord<D>;
  float* rec = reinterpret_cast<float*>(dsm);
  if (warp < kWarps) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float* r = rec + ((wk * WR + wr) * 16 + gq + hf * 8) * RS;
#pragma unroll
      for (int n = 0; n < NB; ++n)
        *reinterpret_cast<float2*>(r + n * 8 + 2 * tq) = make_float2(o[n][2 * hf], o[n][2 * hf + 1]);
      if (tq == 0) {
        r[D] = hf ? mx1 : mx0;
        r[D + 1] = hf ? l1 : l0;
      }
    }
  }
  __syncthreads();
  pdl_wait();   // nothing is written before the previous kernel of the step is done (a shared workspace, the caches)
  // rows' states over the WK warps that share them; with several splits a record of them
  auto merge = [&](int rr, int c, auto at, int count, float& M, float& x, float& y, float& L) {
    M = -INFINITY;
    for (int w = 0; w < count; ++w) M = fmaxf(M, at(w)[rr * RS + D]);
    x = y = L = 0.f;
    for (int w = 0; w < count; ++w) {
      const float* r = at(w) + rr * RS;
      const float f = r[D] == -INFINITY ? 0.f : exp2f(r[D] - M);
      x = fmaf(r[c], f, x);
      y = fmaf(r[c + 1], f, y);
      L = fmaf(r[D + 1], f, L);
    }
  };
  auto put = [&](int rr, int c, float M, float x, float y, float L) {
    const int m = rb * 16 * WR + rr;
    if (m >= rows) return;
    const int h = g * R + m % R, node = m / R;
    const float inv = L == 0.f ? 0.f : 1.f / L;   // (NaN stays)
    write_row<T>(a, b, h, node, len, c, x * inv, y * inv);
    if (c == 0) write_lse(a, b, h, node, len, L == 0.f ? -FLT_MAX : (M + __log2f(L)) * kLn2);
  };
  float* crec = rec + kWarps * 16 * RS;   // this CTA's
  const bool local = geo.splits == 1 || geo.cluster;
  for (int idx = threadIdx.x; idx < 16 * WR * (D / 2); idx += kThreads) {
    const int rr = idx / (D / 2), c = (idx - rr * (D / 2)) * 2;
    float M, x, y, L;
    merge(rr, c, [&](int w) { return rec + w * WR * 16 * RS; }, WK, M, x, y, L);
    if (geo.splits == 1) {
      put(rr, c, M, x, y, L);
      continue;
    }
    const int m = rb * 16 * WR + rr;
    if (!local && m >= rows) break;
    float* p = local ? crec + rr * RS : geo.part + (((int64_t)blockIdx.y * rows + m) * geo.splits + split) * RS;
    *reinterpret_cast<float2*>(p + c) = make_float2(x, y);
    if (c == 0) {
      p[D] = M;
      p[D + 1] = L;
    }
  }
  if (geo.cluster) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();   // every CTA's records are visible to the cluster
    // CTA `split` joins and writes its share of the rows
    for (int idx = split * kThreads + threadIdx.x; idx < 16 * WR * (D / 2); idx += geo.splits * kThreads) {
      const int rr = idx / (D / 2), c = (idx - rr * (D / 2)) * 2;
      float M, x, y, L;
      merge(rr, c, [&](int w) { return (const float*)cluster.map_shared_rank(crec, w); }, geo.splits, M, x, y, L);
      put(rr, c, M, x, y, L);
    }
    cluster.sync();   // no CTA leaves while its records may still be read
  }
}

// One warp per row: the splits' records (m, l, acc[D]) into out and lse.
template <typename T, int D>
__global__ void __launch_bounds__(128) tree_combine_kernel(const __grid_constant__ PolyTreePass a, const TreeGeom geo) {
  const int lane = threadIdx.x & 31;
  const int R = a.heads / a.kv_heads, rows = R * a.nodes;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_launch();
  pdl_wait();
  if (row >= (int64_t)a.batch * a.kv_heads * rows) return;
  const int group = (int)(row / rows), m = (int)(row - (int64_t)group * rows);
  const int b = group / a.kv_heads, g = group - b * a.kv_heads;
  const float* p = geo.part + row * geo.splits * kRecord<D>;
  float M = -INFINITY;
  for (int s = lane; s < geo.splits; s += 32) M = fmaxf(M, p[s * kRecord<D> + D]);
  M = warp_max(M);
  float L = 0.f, acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t) acc[t] = 0.f;
#pragma unroll 4
  for (int s = 0; s < geo.splits; ++s) {
    const float* r = p + s * kRecord<D>;
    const float f = r[D] == -INFINITY ? 0.f : exp2f(r[D] - M);
    L = fmaf(r[D + 1], f, L);
#pragma unroll
    for (int t = 0; t < D / 64; ++t) {
      const float2 v = *reinterpret_cast<const float2*>(r + t * 64 + 2 * lane);
      acc[2 * t] = fmaf(v.x, f, acc[2 * t]);
      acc[2 * t + 1] = fmaf(v.y, f, acc[2 * t + 1]);
    }
  }
  const int len = seq_length(a.lengths, b, a.capacity), h = g * R + m % R, node = m / R;
  const float inv = L == 0.f ? 0.f : 1.f / L;   // (NaN stays)
#pragma unroll
  for (int t = 0; t < D / 64; ++t) write_row<T>(a, b, h, node, len, t * 64 + 2 * lane, acc[2 * t] * inv, acc[2 * t + 1] * inv);
  if (lane == 0) write_lse(a, b, h, node, len, L == 0.f ? -FLT_MAX : (M + __log2f(L)) * kLn2);
}

// ---------------------------------------------------------------- CUDA cores
constexpr int kSimtWarps = 8, kSimtKeys = 32;

template <typename T, int DMAX>
__global__ void __launch_bounds__(kSimtWarps * 32) tree_simt_kernel(const __grid_constant__ PolyTreePass a) {
  constexpr int NT = DMAX / 32;
  __shared__ float Ks[kSimtKeys][DMAX + 1], Vs[kSimtKeys][DMAX + 1], Qs[kSimtWarps][DMAX];
  __shared__ uint64_t anc[kNodes];
  __shared__ int up[kNodes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.head_dim;
  const int b = blockIdx.y / a.kv_heads, g = blockIdx.y - b * a.kv_heads;
  const int R = a.heads / a.kv_heads, rows = R * a.nodes, m = blockIdx.x * kSimtWarps + warp;
  const int len = seq_length(a.lengths, b, a.capacity), nkeys = min(len + a.nodes, a.capacity);
  pdl_launch();
  pdl_wait();
  ancestors(a.parents + b * a.parents_stride, a.nodes, a.capacity - len, anc, up);
  const bool ok = m < rows;
  const int node = ok ? m / R : 0, h = g * R + (ok ? m % R : 0);
  const uint64_t see = ok ? anc[node] : 0ull;
  const T* q = (const T*)a.q + b * a.q_stride[0] + h * a.q_stride[1] + node * a.q_stride[2];
  for (int t = lane; t < DMAX; t += 32) Qs[warp][t] = t < d ? to_f32(q[t]) : 0.f;
  const T* k = (const T*)a.k + b * a.k_stride[0] + g * a.k_stride[1];
  const T* v = (const T*)a.v + b * a.v_stride[0] + g * a.v_stride[1];
  const T* vm = a.v_mul ? (const T*)a.v_mul + b * a.v_mul_stride[0] + g * a.v_mul_stride[1] : nullptr;
  const float* bias = a.bias ? a.bias + b * a.bias_stride[0] + g * a.bias_stride[1] : nullptr;
  float mx = -INFINITY, l = 0.f, acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = 0.f;
  for (int j0 = 0; j0 < nkeys; j0 += kSimtKeys) {
    __syncthreads();
    for (int i = threadIdx.x; i < kSimtKeys * DMAX; i += kSimtWarps * 32) {
      const int r = i / DMAX, c = i - r * DMAX;
      const bool in = j0 + r < nkeys && c < d;
      Ks[r][c] = in ? to_f32(k[(int64_t)(j0 + r) * a.k_stride[2] + c]) : 0.f;
      float x = in ? to_f32(v[(int64_t)(j0 + r) * a.v_stride[2] + c]) : 0.f;
      if (vm && in) x = to_f32(from_f32<T>(x * to_f32(vm[(int64_t)(j0 + r) * a.v_mul_stride[2] + c])));
      Vs[r][c] = x;
    }
    __syncthreads();
    const int j = j0 + lane, n = j - len;
    float s = 0.f;
#pragma unroll 8
    for (int t = 0; t < DMAX; ++t) s = fmaf(Qs[warp][t], Ks[lane][t], s);
    s *= a.scale;
    if (a.softclamp > 0.f) s = a.softclamp * tanhf(s / a.softclamp);
    bool keep = see && j < nkeys && (n < 0 || ((see >> n) & 1));
    if (keep && bias) {
      const float bj = bias[j];
      keep = !(bj <= kDeadBias);
      s += bj;
    }
    s = keep ? s : -INFINITY;
    const float mn = fmaxf(mx, warp_max(s));
    if (mn == -INFINITY && !__any_sync(0xffffffffu, s != s)) continue;   // (a row of NaN scores has a sum)
    const float p = keep ? exp2f((s - mn) * kLog2e) : 0.f, f = exp2f((mx - mn) * kLog2e);
    l = l * f + warp_sum(p);
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] *= f;
#pragma unroll 4
    for (int jj = 0; jj < kSimtKeys; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, p, jj);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = fmaf(pj, Vs[jj][lane + 32 * t], acc[t]);
    }
    mx = mn;
  }
  if (!ok) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = lane + 32 * t;
    if (c >= d) continue;
    const T x = from_f32<T>(acc[t] * inv);
    if (a.out) ((T*)a.out)[b * a.out_stride[0] + h * a.out_stride[1] + node * a.out_stride[2] + c] = x;
    if (a.cache_out && len + node < a.capacity)
      ((T*)a.cache_out)[b * a.cache_out_stride[0] + h * a.cache_out_stride[1] + (int64_t)(len + node) * a.cache_out_stride[2] + c] = x;
  }
  if (lane == 0) write_lse(a, b, h, node, len, l == 0.f ? -FLT_MAX : mx + logf(l));
}

// ---------------------------------------------------------------- rows in and out
// One CTA per (cache, sequence, head): nodes rows of row_bytes.
template <typename W>
__global__ void __launch_bounds__(128) tree_append_kernel(const __grid_constant__ PolyTreeAppend a, int32_t* step_nodes) {
  __shared__ uint64_t anc[kNodes];
  __shared__ int up[kNodes];
  const int k = blockIdx.y, b = blockIdx.x / a.kv_heads, g = blockIdx.x - b * a.kv_heads;
  const int len = seq_length(a.lengths, b, a.capacity);
  pdl_launch();
  if (step_nodes && blockIdx.x == 0 && k == 0 && threadIdx.x == 0) *step_nodes = a.nodes;
  ancestors(a.parents + b * a.parents_stride, a.nodes, a.capacity - len, anc, up);
  const auto& t = a.t[k];
  const char* src = (const char*)t.src + b * t.src_stride[0] + g * t.src_stride[1];
  char* dst = (char*)t.cache + b * t.cache_stride[0] + g * t.cache_stride[1] + (int64_t)len * t.cache_stride[2];
  const int words = a.row_bytes / (int)sizeof(W), n = min(a.nodes, a.capacity - len);
  for (int i = threadIdx.x; i < n * words; i += 128) {
    const int node = i / words, w = i - node * words;
    W x{};
    if (anc[node]) x = *reinterpret_cast<const W*>(src + node * t.src_stride[2] + w * sizeof(W));   // padding: zeros
    *reinterpret_cast<W*>(dst + node * t.cache_stride[2] + w * sizeof(W)) = x;
  }
}

// Nodes that a commit may keep: those of the last step, where the step left their number.
__device__ __forceinline__ int kept_nodes(const PolyTreeCommit& a, const int32_t* step_nodes) {
  return step_nodes ? min(max(*step_nodes, 0), a.nodes) : a.nodes;
}

// One CTA per (cache, sequence, head). A thread owns its words of every row and
// moves them in path order; an entry's row is at or behind its place, so nothing
// is overwritten before it is read.
template <typename W>
__global__ void __launch_bounds__(64) tree_commit_kernel(const __grid_constant__ PolyTreeCommit a, const int32_t* step_nodes) {
  const int k = blockIdx.y, b = blockIdx.x / a.kv_heads, g = blockIdx.x - b * a.kv_heads;
  const int len = seq_length(a.lengths, b, a.capacity);
  const int room = min(kept_nodes(a, step_nodes), a.capacity - len), n = min(max(a.count[b], 0), min(room, a.path_len));
  const auto& t = a.t[k];
  char* base = (char*)t.cache + b * t.cache_stride[0] + g * t.cache_stride[1] + (int64_t)len * t.cache_stride[2];
  const int32_t* path = a.path + b * a.path_stride;
  for (int w = threadIdx.x; w < (int)(t.row_bytes / sizeof(W)); w += 64)
    for (int i = 0; i < n; ++i) {
      const int p = min(max(path[i], i), room - 1);
      if (p != i)
        *reinterpret_cast<W*>(base + i * t.cache_stride[2] + w * sizeof(W)) =
            *reinterpret_cast<const W*>(base + p * t.cache_stride[2] + w * sizeof(W));
    }
}

__global__ void __launch_bounds__(kNodes) tree_positions_kernel(const int32_t* lengths, const int32_t* parents, int64_t stride,
                                                                int nodes, int32_t* positions, int64_t pstride) {
  __shared__ uint64_t anc[kNodes];
  __shared__ int up[kNodes];
  const int b = blockIdx.x, i = threadIdx.x;
  ancestors(parents + b * stride, nodes, nodes, anc, up);
  if (i < nodes) positions[b * pstride + i] = lengths[b] + (anc[i] ? __popcll(anc[i]) - 1 : 0);
}

// One CTA: every thread has the step's number of nodes before it is taken back.
__global__ void __launch_bounds__(128) tree_lengths_kernel(const __grid_constant__ PolyTreeCommit a, int32_t* step_nodes) {
  const int nodes = min(kept_nodes(a, step_nodes), a.path_len);
  for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
    const int len = seq_length(a.lengths, b, a.capacity);
    a.lengths[b] = len + min(max(a.count[b], 0), min(nodes, a.capacity - len));
  }
  if (!step_nodes) return;
  __syncthreads();
  if (threadIdx.x == 0) *step_nodes = 0;
}

// ---------------------------------------------------------------- host
int fail(int code, const std::string& m) {
  set_error(m);
  return code;
}

int sm_count() {
  static std::mutex mu;
  static int dev_sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  std::lock_guard<std::mutex> lk(mu);
  if (!dev_sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    dev_sms[dev] = n;
  }
  return dev_sms[dev];
}

bool on_tensor_cores(const PolyTreePass& a) {
  if (a.dtype != POLY_BF16 && a.dtype != POLY_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  auto rows_ok = [](const void* p, const int64_t* st) {
    return !p || (aligned16(p) && st[0] > 0 && st[1] > 0 && st[2] > 0 && !((st[0] | st[1] | st[2]) & 7));
  };
  auto pairs_ok = [](const void* p, const int64_t* st) {   // 4-byte accesses
    return !p || (((uintptr_t)p & 3) == 0 && !((st[0] | st[1] | st[2]) & 1));
  };
  return rows_ok(a.k, a.k_stride) && rows_ok(a.v, a.v_stride) && rows_ok(a.v_mul, a.v_mul_stride) &&
         pairs_ok(a.q, a.q_stride) && pairs_ok(a.out, a.out_stride) && pairs_ok(a.cache_out, a.cache_out_stride);
}

int warp_rows(const PolyTreePass& a) {
  const int rows = a.nodes * (a.heads / a.kv_heads);
  return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}

// Key ranges per (sequence, kv head), at least one key tile of the capacity each. tcgen05
// kernel: as many as fill the CTAs that fit at once, one per SM. tree_kernel, of which two fit:
// up to 8 that join in a cluster, filling both places (16 sequences of up to 9000 tokens,
// 8 nodes, h16 g4 d128: 133 us a step, 155 with 3 CTAs per 2 SMs; 8 sequences: 80 and 91; 32 of
// up to 2304: 82 and 80). More than 8, which go through the workspace, fill 3 places of 4:
// 2 sequences of up to 40001 tokens take 96 us a step so, 121 with every place filled.
TreeGeom geometry(const PolyTreePass& a, bool may_tc = true) {
  TreeGeom geo{};
  const int rows = a.nodes * (a.heads / a.kv_heads), wr = warp_rows(a);
  geo.row_blocks = may_tc ? tree_tc_row_blocks(a) : 0;
  geo.tcgen05 = geo.row_blocks > 0;
  if (!geo.tcgen05) geo.row_blocks = (rows + 16 * wr - 1) / (16 * wr);
  const int64_t ctas = (int64_t)a.batch * a.kv_heads * geo.row_blocks;
  const int keys = geo.tcgen05 ? 128 : kKeys, tiles = (a.capacity + keys - 1) / keys;
  auto fill = [&](int slots) { return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(kMaxSplits, tiles), slots / ctas)); };
  if (geo.tcgen05) {
    geo.splits = fill(sm_count());
  } else {
    // a cluster's 8 splits, or more of at least 16 tiles each (a second launch and the records' way through
    // L2 cost about 5 us)
    const int long_splits = std::min(fill(sm_count() * 3 / 2), tiles / 16);
    geo.splits = long_splits > 8 ? long_splits : std::min(fill(sm_count() * 2), 8);
    geo.cluster = geo.splits > 1 && geo.splits <= 8;
  }
  return geo;
}

int check_pass(const PolyTreePass* a) {
  if (!a) return fail(POLY_EINVAL, "null tree pass");
  if (a->batch < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->nodes < 0 || a->nodes > kNodes || a->head_dim <= 0 || a->capacity < 0)
    return fail(POLY_EINVAL, "tree pass: bad sizes (nodes <= 64)");
  if (a->heads % a->kv_heads) return fail(POLY_EINVAL, "tree pass: heads must be divisible by kv_heads");
  if (a->dtype != POLY_F32 && a->dtype != POLY_F16 && a->dtype != POLY_BF16) return fail(POLY_EINVAL, "tree pass: unknown dtype");
  if (a->head_dim > 128) return fail(POLY_EUNSUPPORTED, "tree pass: head_dim > 128 is not supported");
  if (!(a->scale == a->scale)) return fail(POLY_EINVAL, "tree pass: scale is NaN");
  if (!a->q || !a->k || !a->v || !a->lengths || !a->parents)
    return fail(POLY_EINVAL, "tree pass: q, k, v, lengths and parents are required");
  if ((int64_t)a->batch * a->kv_heads > 65535) return fail(POLY_EUNSUPPORTED, "tree pass: batch * kv_heads > 65535");
  return POLY_OK;
}

// A kernel of a step: a programmatic dependent of the one before it.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, bool dependent, int cluster,
                   A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (dependent) attr[n++] = dependent_launch();
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  note_launch(1);
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int D>
int launch_combine(const PolyTreePass& a, const TreeGeom& geo, cudaStream_t s) {
  const int64_t rows = (int64_t)a.batch * a.heads * a.nodes;
  return cuda_status(launch(tree_combine_kernel<T, D>, dim3((unsigned)((rows + 3) / 4)), 128, 0, s, true, 0, a, geo), "tree launch");
}

template <typename T, int D, int WR, bool VMUL>
int launch_tree(const PolyTreePass& a, cudaStream_t s, bool dep) {
  using R_ = Ring<D, VMUL ? 3 : 2>;
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_smem((const void*)tree_kernel<T, D, WR, VMUL>, R_::kAlloc, done,
                                "cudaFuncSetAttribute(tree)")) return rc;
  TreeGeom geo = geometry(a);
  geo.part = (float*)a.workspace;
  CUtensorMap tk, tv, tm;
  memset(&tm, 0, sizeof(tm));
  int rc = make_map(&tk, a.k, a.dtype, D, a.capacity, a.kv_heads, a.batch, a.k_stride, kKeys);
  if (!rc) rc = make_map(&tv, a.v, a.dtype, D, a.capacity, a.kv_heads, a.batch, a.v_stride, kKeys);
  if (!rc && VMUL) rc = make_map(&tm, a.v_mul, a.dtype, D, a.capacity, a.kv_heads, a.batch, a.v_mul_stride, kKeys);
  if (rc) return rc;
  const int groups = a.batch * a.kv_heads;
  cudaError_t e = launch(tree_kernel<T, D, WR, VMUL>, dim3(geo.splits * geo.row_blocks, groups), kThreads, R_::kAlloc, s, dep,
                         geo.cluster ? geo.splits : 0, tk, tv, tm, a, geo);
  rc = cuda_status(e, "tree launch");
  return rc || geo.splits <= 1 || geo.cluster ? rc : launch_combine<T, D>(a, geo, s);
}

template <typename T, int D>
int launch_rows(const PolyTreePass& a, cudaStream_t s, bool dep) {
  TreeGeom geo = geometry(a);
  if (geo.tcgen05) {
    geo.part = (float*)a.workspace;
    const int rc = launch_tree_tc(a, geo, s, dep);
    return rc || geo.splits <= 1 ? rc : launch_combine<T, D>(a, geo, s);
  }
  const bool vm = a.v_mul != nullptr;
  switch (warp_rows(a)) {
    case 1: return vm ? launch_tree<T, D, 1, true>(a, s, dep) : launch_tree<T, D, 1, false>(a, s, dep);
    case 2: return vm ? launch_tree<T, D, 2, true>(a, s, dep) : launch_tree<T, D, 2, false>(a, s, dep);
    default: return vm ? launch_tree<T, D, 4, true>(a, s, dep) : launch_tree<T, D, 4, false>(a, s, dep);
  }
}

template <typename T, int DMAX>
int launch_simt(const PolyTreePass& a, cudaStream_t s, bool dep) {
  const int rows = a.nodes * (a.heads / a.kv_heads);
  return cuda_status(launch(tree_simt_kernel<T, DMAX>, dim3((rows + kSimtWarps - 1) / kSimtWarps, a.batch * a.kv_heads),
                            kSimtWarps * 32, 0, s, dep, 0, a), "tree launch");
}

template <typename T>
int launch_simt_d(const PolyTreePass& a, cudaStream_t s, bool dep) {
  if (a.head_dim <= 32) return launch_simt<T, 32>(a, s, dep);
  return a.head_dim <= 64 ? launch_simt<T, 64>(a, s, dep) : launch_simt<T, 128>(a, s, dep);
}

int launch_pass(const PolyTreePass& a, cudaStream_t s, bool dep) {
  if (on_tensor_cores(a)) {
    if (a.dtype == POLY_BF16) return a.head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(a, s, dep) : launch_rows<__nv_bfloat16, 128>(a, s, dep);
    return a.head_dim == 64 ? launch_rows<__half, 64>(a, s, dep) : launch_rows<__half, 128>(a, s, dep);
  }
  if (a.dtype == POLY_F32) return launch_simt_d<float>(a, s, dep);
  return a.dtype == POLY_F16 ? launch_simt_d<__half>(a, s, dep) : launch_simt_d<__nv_bfloat16>(a, s, dep);
}

int check_append(const PolyTreeAppend& a) {
  if (a.batch < 0 || a.kv_heads <= 0 || a.nodes < 0 || a.nodes > kNodes || a.capacity < 0 || a.row_bytes <= 0 || (a.row_bytes & 1))
    return fail(POLY_EINVAL, "tree append: bad sizes (nodes <= 64, rows of whole 16-bit words)");
  if (a.n < 0 || a.n > POLY_MAX_TREE_CACHES) return fail(POLY_EINVAL, "tree append: at most 16 caches");
  if (!a.lengths || !a.parents) return fail(POLY_EINVAL, "tree append: lengths and parents are required");
  for (int i = 0; i < a.n; ++i)
    if (!a.t[i].src || !a.t[i].cache) return fail(POLY_EINVAL, "tree append: null tensor");
  return POLY_OK;
}

int launch_append(const PolyTreeAppend& a, int32_t* step_nodes, cudaStream_t s) {
  uint64_t bits = (uint64_t)a.row_bytes;
  for (int i = 0; i < a.n; ++i) {
    bits |= (uint64_t)(uintptr_t)a.t[i].src | (uint64_t)(uintptr_t)a.t[i].cache;
    for (int x = 0; x < 3; ++x) bits |= (uint64_t)a.t[i].src_stride[x] | (uint64_t)a.t[i].cache_stride[x];
  }
  const dim3 grid(a.batch * a.kv_heads, a.n);
  const cudaError_t e = bits & 15 ? launch(tree_append_kernel<uint16_t>, grid, 128, 0, s, false, 0, a, step_nodes)
                                  : launch(tree_append_kernel<uint4>, grid, 128, 0, s, false, 0, a, step_nodes);
  return cuda_status(e, "tree append launch");
}

}  // namespace
}  // namespace poly

using namespace poly;

extern "C" {

size_t poly_sizeof_tree_pass(void) { return sizeof(PolyTreePass); }
size_t poly_sizeof_tree_append(void) { return sizeof(PolyTreeAppend); }
size_t poly_sizeof_tree_commit(void) { return sizeof(PolyTreeCommit); }

const char* poly_tree_kernel_name(const PolyTreePass* a) {
  if (check_pass(a) != POLY_OK) return "invalid";
  if (!on_tensor_cores(*a)) return "simt";
  return a->nodes > 0 && tree_tc_row_blocks(*a) ? "tc100" : "tree";
}

size_t poly_tree_workspace_size(const PolyTreePass* a) {
  if (check_pass(a) != POLY_OK || !on_tensor_cores(*a) || a->batch == 0 || a->nodes == 0 || a->capacity == 0) return 0;
  // enough for either kernel: which one runs depends on q's address and strides, which may change from step to step
  PolyTreePass any = *a;
  any.q = nullptr;
  any.q_stride[0] = any.q_stride[1] = any.q_stride[2] = 8;
  any.out = any.cache_out = nullptr;
  size_t need = 0;
  for (const bool tc : {false, true}) {
    const TreeGeom geo = geometry(any, tc);
    if (geo.splits > 1 && !geo.cluster)
      need = std::max(need, (size_t)a->batch * a->heads * a->nodes * geo.splits * (a->head_dim + 4) * sizeof(float));
  }
  return need;
}

int poly_tree_chain(const PolyTreeAppend* append, const PolyTreePass* passes, int n, void* stream) {
  return poly_tree_chain_counted(append, passes, n, nullptr, stream);
}

int poly_tree_chain_counted(const PolyTreeAppend* append, const PolyTreePass* passes, int n, int32_t* step_nodes, void* stream) {
  if (n < 0 || (n > 0 && !passes)) return fail(POLY_EINVAL, "poly_tree_chain: null passes or negative count");
  if (step_nodes && !append) return fail(POLY_EINVAL, "poly_tree_chain_counted: step_nodes is written by the append");
  int rc;
  if (append && (rc = check_append(*append))) return rc;
  for (int i = 0; i < n; ++i) {
    if ((rc = check_pass(&passes[i]))) return rc;
    const size_t need = poly_tree_workspace_size(&passes[i]);
    if (need && (!passes[i].workspace || passes[i].workspace_bytes < need))
      return fail(POLY_EINVAL, "tree pass " + std::to_string(i) + " needs a workspace of " + std::to_string(need) + " bytes");
    if ((uintptr_t)passes[i].workspace & 15) return fail(POLY_EINVAL, "tree pass: workspace must be 16-byte aligned");
  }
  cudaStream_t s = (cudaStream_t)stream;
  bool dep = false;
  if (append && append->n > 0 && append->batch > 0 && append->nodes > 0 && append->capacity > 0) {
    if ((rc = launch_append(*append, step_nodes, s))) return rc;
    dep = true;
  }
  for (int i = 0; i < n; ++i) {
    if (passes[i].batch == 0 || passes[i].nodes == 0 || passes[i].capacity == 0) continue;
    if ((rc = launch_pass(passes[i], s, dep))) return rc;
    dep = true;
  }
  return POLY_OK;
}

int poly_tree_positions(const int32_t* lengths, const int32_t* parents, int64_t parents_stride, int batch, int nodes,
                        int32_t* positions, int64_t positions_stride, void* stream) {
  if (batch < 0 || nodes < 0 || nodes > kNodes) return fail(POLY_EINVAL, "tree positions: bad sizes (nodes <= 64)");
  if (batch == 0 || nodes == 0) return POLY_OK;
  if (!lengths || !parents || !positions) return fail(POLY_EINVAL, "tree positions: null pointer");
  tree_positions_kernel<<<batch, kNodes, 0, (cudaStream_t)stream>>>(lengths, parents, parents_stride, nodes, positions,
                                                                    positions_stride);
  note_launch(1);
  return cuda_status(cudaGetLastError(), "tree positions launch");
}

int poly_tree_commit(const PolyTreeCommit* args, void* stream) { return poly_tree_commit_counted(args, nullptr, stream); }

int poly_tree_commit_counted(const PolyTreeCommit* args, int32_t* step_nodes, void* stream) {
  if (!args) return fail(POLY_EINVAL, "null tree commit");
  const PolyTreeCommit& a = *args;
  if (a.batch < 0 || a.kv_heads <= 0 || a.nodes < 0 || a.nodes > kNodes || a.path_len < 0 || a.capacity < 0 || a.n < 0 ||
      a.n > POLY_MAX_TREE_CACHES)
    return fail(POLY_EINVAL, "tree commit: bad sizes (nodes <= 64, at most 16 caches)");
  if (!a.lengths || !a.path || !a.count) return fail(POLY_EINVAL, "tree commit: lengths, path and count are required");
  uint64_t bits = 0;
  for (int i = 0; i < a.n; ++i) {
    if (!a.t[i].cache || a.t[i].row_bytes <= 0 || (a.t[i].row_bytes & 1)) return fail(POLY_EINVAL, "tree commit: bad cache");
    bits |= (uint64_t)(uintptr_t)a.t[i].cache | (uint64_t)a.t[i].row_bytes;
    for (int x = 0; x < 3; ++x) bits |= (uint64_t)a.t[i].cache_stride[x];
  }
  if (a.batch == 0 || a.nodes == 0) return POLY_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (a.n > 0) {
    const dim3 grid(a.batch * a.kv_heads, a.n);
    if (bits & 3) tree_commit_kernel<uint16_t><<<grid, 64, 0, s>>>(a, step_nodes);
    else tree_commit_kernel<uint32_t><<<grid, 64, 0, s>>>(a, step_nodes);
    note_launch(1);
    const int rc = cuda_status(cudaGetLastError(), "tree commit launch");
    if (rc) return rc;
  }
  tree_lengths_kernel<<<1, 128, 0, s>>>(a, step_nodes);
  note_launch(1);
  return cuda_status(cudaGetLastError(), "tree lengths launch");
}

}  // extern "C"
