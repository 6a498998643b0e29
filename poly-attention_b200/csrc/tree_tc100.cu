// tcgen05 tree pass (sm_100a, 16-bit, d = 64 / 128, no v_mul): the pass of the
// order-n step that has the query heads (R rows a node), and the widest trees of the
// others, whose 33 to some hundred rows per cached key the mma.sync kernel of tree.cu
// cannot multiply at the rate at which the cache arrives.
//
// A CTA takes one (sequence, kv head), one range of 128-key tiles, and its rows as
// 128-row tiles: head r, node i at row r * Tp + i (Tp: the nodes padded to 8, so that
// one TMA box per head lands on the swizzle's 8-row period). Two softmax warpgroups
// keep the tensor core busy:
//   ROWS2   two row tiles, one warpgroup each, over the same K / V stages;
//   else    one row tile, whose even and odd key tiles go to the two warpgroups, each
//           with its own maximum, sum and O; they merge through shared memory.
// Warps: 0 TMA, 1 TMEM + MMA issue, 2 bias (cp.async cannot drop dead keys; plain loads
// a few tiles ahead can), 3 zeroes the value rows behind the tree in the last tile
// (whatever they hold: 0 * NaN), 4-7 and 8-11 softmax. TMEM: S / P of the two
// warpgroups at 0 and 128 (P, 16-bit, over the first half of its S), O at 256 and
// 256 + D. P V(i) precedes S(i + 1) of a warpgroup in issue order, so a full S says
// that O is at rest and P's columns are free.
//
// Measured (4 sequences of up to 40001 tokens, 128492 in all, d 128): 60 rows 67 us for 263 MB,
// 60 % of the measured copy rate (the longest sequence's ranges set the time); 240 rows 121 us,
// bound by the chain score - softmax - product of a tile, about 3 us, with two tiles in flight. Items of 64 keys
// with S, P and O side by side in TMEM, so that S(i + 1) is formed during softmax(i),
// were slower (84 and 159 us): the hand-offs per item cost more than they hid.
#include <algorithm>
#include <cstring>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "tc_host.cuh"
#include "tc_ptx.cuh"
#include "tree_common.cuh"

namespace poly {

static __device__ int g_tree_tc_error[2] = {0, 0};

int read_device_error_tree_tc(int* out, bool reset) {
  int rc = cuda_status(cudaMemcpyFromSymbol(out, g_tree_tc_error, sizeof(int)), "read device error word");
  if (rc == POLY_OK && reset) {
    const int zero = 0;
    rc = cuda_status(cudaMemcpyToSymbol(g_tree_tc_error, &zero, sizeof(int)), "reset device error word");
  }
  return rc;
}

namespace {
using namespace tc;
using namespace treec;

constexpr int BM = 128, BN = 128, kThreads = 384;
constexpr int kAtom = 128 * 128;   // bytes of 64 columns of a 128-row tile

template <int D, bool ROWS2>
struct Lay {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kTiles = ROWS2 ? 2 : 1;          // row tiles
  static constexpr int S = D == 64 ? 4 : ROWS2 ? 2 : 3;  // key stages
  static constexpr int kQ = 0;
  static constexpr int kK = kTiles * kTile;
  static constexpr int kV = kK + S * kTile;
  static constexpr int kB = kV + S * kTile;              // bias [S][128]; before it, the nodes' ancestors
  static constexpr int kUp = kB + kNodes * 8;
  static constexpr int kBar = kB + S * BN * 4;
  static constexpr int kNumBars = 1 + 4 * S + 2 + 2 + 2 + 3;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kAlloc = kMisc + 16 + 1024;
  static_assert(S * BN * 4 >= kNodes * 12 && kAlloc <= 227 * 1024, "shared memory");
};

struct TreeTcParams {
  PolyTreePass a;
  TreeGeom geo;          // splits, row_blocks, part
  int tp, heads_tile;    // rows of a head, heads of a row tile
};

template <typename T>
__device__ __forceinline__ uint32_t pk2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack_bf16(a, b);
  else return pack_f16(a, b);
}
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer() - t0 > kWaitNs) return;
}
// bits [0, 64) of: all ones below place -base, then `see` from there on
__device__ __forceinline__ uint64_t window(uint64_t see, int base) {
  if (base <= -64) return ~0ull;
  if (base < 0) return ((1ull << -base) - 1) | (see << -base);
  return base < 64 ? see >> base : 0ull;
}

template <typename T, int D, bool ROWS2, bool SOFTCLAMP>
__global__ void __launch_bounds__(kThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TreeTcParams P) {
  using L = Lay<D, ROWS2>;
  constexpr int S = L::S;
  constexpr int kIsBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  const PolyTreePass& a = P.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sK = smem + L::kK;
  uint8_t* sV = smem + L::kV;
  float* sB = (float*)(smem + L::kB);
  uint64_t* anc = (uint64_t*)(smem + L::kB);
  uint64_t* bars = (uint64_t*)(smem + L::kBar);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* v_full = bars + 1 + S;
  uint64_t* k_empty = bars + 1 + 2 * S;   // keys: free once their scores are formed
  uint64_t* v_empty = bars + 1 + 3 * S;   // values and bias: once multiplied
  uint64_t* s_full = bars + 1 + 4 * S;    // [2]
  uint64_t* p_full = bars + 3 + 4 * S;    // [2]
  uint64_t* o_done = bars + 5 + 4 * S;    // [2]
  uint64_t* v_cut = bars + 7 + 4 * S;     // the last value tile arrives here if it has rows behind the tree ...
  uint64_t* v_clean = bars + 8 + 4 * S;   // ... and is without them here
  uint64_t* drain = bars + 9 + 4 * S;
  uint32_t* tmem_slot = (uint32_t*)(smem + L::kMisc);
  volatile int* abort_flag = (volatile int*)(smem + L::kMisc + 4);
  int* err = g_tree_tc_error;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % P.geo.splits, rb = blockIdx.x / P.geo.splits;
  const int b = blockIdx.y / a.kv_heads, g = blockIdx.y - b * a.kv_heads;
  const int R = a.heads / a.kv_heads;
  const int len = seq_length(a.lengths, b, a.capacity);
  const int nkeys = min(len + a.nodes, a.capacity);
  const int tiles = (nkeys + BN - 1) / BN;
  const int t0 = (int)((int64_t)tiles * split / P.geo.splits), t1 = (int)((int64_t)tiles * (split + 1) / P.geo.splits);
  const int n = t1 - t0;
  const int cut_tile = (nkeys % BN) != 0 && t1 == tiles ? n - 1 : -1;
  const int head0 = rb * P.heads_tile * L::kTiles;   // the block's first head of the group

  pdl_launch();
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < S; ++s) {
      mbar_init(&k_full[s], 33);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 128);
      mbar_init(&o_done[x], 1);
    }
    mbar_init(v_cut, 1);
    mbar_init(v_clean, 32);
    mbar_init(drain, 1);
    abort_init(abort_flag, err);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  ancestors(a.parents + b * a.parents_stride, a.nodes, a.capacity - len, anc, (int*)(smem + L::kUp));
  // the softmax threads' rows, and what their nodes see (read before the bias takes its place)
  const int x = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
  const int hl = r / P.tp, node = r - hl * P.tp, head = head0 + (ROWS2 ? x * P.heads_tile : 0) + hl;
  const bool row_ok = warp >= 4 && hl < P.heads_tile && head < R && node < a.nodes;
  const uint64_t see = row_ok ? anc[node] : 0ull;
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // key tiles of warpgroup x: every one (ROWS2) or those of its parity
  auto items = [&](int x) { return ROWS2 ? n : (n + 1 - x) >> 1; };
  auto tile_of = [&](int x, int i) { return ROWS2 ? i : 2 * i + x; };

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      // ------------------------------------------------ TMA producer
      int rows = 0;
      for (int x = 0; x < L::kTiles; ++x)
        rows += min(max(R - head0 - x * P.heads_tile, 0), P.heads_tile);
      mbar_arrive_expect_tx(q_full, rows * a.nodes * D * 2);
      for (int x = 0; x < L::kTiles; ++x)
        for (int r = 0; r < P.heads_tile && head0 + x * P.heads_tile + r < R; ++r)
#pragma unroll
          for (int hf = 0; hf < D / 64; ++hf)
            tma_load_4d(smem + L::kQ + x * L::kTile + hf * kAtom + r * P.tp * 128, &tm_q, q_full, hf * 64, 0,
                        g * R + head0 + x * P.heads_tile + r, b);
      int k_issued = 0, issued = 0;
      bool waited = false;
      for (int j = 0; j < n; ++j) {
        const int s = j % S, kb = (t0 + j) * BN;
        if (j >= S && !mbar_wait(&k_empty[s], ((j / S) - 1) & 1, abort_flag, err, 81)) break;
        if (!waited && kb + BN > len) {   // rows that the previous kernels of the step write
          pdl_wait();
          waited = true;
        }
        mbar_arrive_expect_tx(&k_full[s], L::kTile);
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf)
          tma_load_4d(sK + s * L::kTile + hf * kAtom, &tm_k, &k_full[s], hf * 64, kb, g, b);
        k_issued = j + 1;
        if (j >= S && !mbar_wait(&v_empty[s], ((j / S) - 1) & 1, abort_flag, err, 92)) break;
        uint64_t* v_bar = j == cut_tile ? v_cut : &v_full[s];
        mbar_arrive_expect_tx(v_bar, L::kTile);
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf)
          tma_load_4d(sV + s * L::kTile + hf * kAtom, &tm_v, v_bar, hf * 64, kb, g, b);
        issued = j + 1;
      }
      if (*abort_flag) {
        drain_wait(q_full, 0);
        for (int j = max(0, k_issued - S); j < k_issued; ++j) drain_wait(&k_full[j % S], (j / S) & 1);
        for (int j = max(0, issued - S); j < issued; ++j) {
          if (j == cut_tile) drain_wait(v_cut, 0);
          else drain_wait(&v_full[j % S], (j / S) & 1);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      // ------------------------------------------------ MMA issuer
      constexpr uint32_t idS = idesc_f16(BM, BN, kIsBf16, 0, 0);
      constexpr uint32_t idO = idesc_f16(BM, D, kIsBf16, 0, 1);
      const uint32_t qa = smem_u32(smem + L::kQ), ka = smem_u32(sK), va = smem_u32(sV);
      auto issue_s = [&](int x, int j) -> bool {
        const int s = j % S;
        if (!mbar_wait(&k_full[s], (j / S) & 1, abort_flag, err, 82)) return false;
        tc_fence_after();
        const uint32_t q = qa + (ROWS2 ? x * L::kTile : 0);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk >> 2) * kAtom + (uint32_t)(kk & 3) * 32;
          mma_f16_ss(tmem + x * BN, smem_desc_sw128(q + off, 16, 1024), smem_desc_sw128(ka + s * L::kTile + off, 16, 1024),
                     idS, kk > 0);
        }
        mma_commit(&s_full[x]);
        if (!ROWS2 || x == 1) mma_commit(&k_empty[s]);
        return true;
      };
      bool ok = mbar_wait(q_full, 0, abort_flag, err, 83) && issue_s(0, tile_of(0, 0));
      if (ok && items(1) > 0) ok = issue_s(1, tile_of(1, 0));
      for (int w = 0; ok && w < (ROWS2 ? 2 * n : n); ++w) {
        const int x = w & 1, i = w >> 1, j = tile_of(x, i), s = j % S;
        if (!(ok = mbar_wait(&p_full[x], i & 1, abort_flag, err, 84))) break;
        if (!ROWS2 || x == 0) {
          ok = j == cut_tile ? mbar_wait(v_clean, 0, abort_flag, err, 85) : mbar_wait(&v_full[s], (j / S) & 1, abort_flag, err, 86);
          if (!ok) break;
        }
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          mma_f16_ts(tmem + 256 + x * D, tmem + x * BN + kk * 8, smem_desc_sw128(va + s * L::kTile + kk * 2048, BN * 128, 1024),
                     idO, i > 0 || kk > 0);
        mma_commit(&o_done[x]);
        if (!ROWS2 || x == 1) mma_commit(&v_empty[s]);
        if (i + 1 < items(x)) ok = issue_s(x, tile_of(x, i + 1));
      }
      mma_commit(drain);
      drain_wait(drain, 0);
    }
  } else if (warp == 2) {
    // -------------------------------------------------- bias (k_full counts these 32 threads too)
    const float* bias = a.bias ? a.bias + b * a.bias_stride[0] + g * a.bias_stride[1] : nullptr;
    bool waited = false;
    for (int j = 0; j < n; ++j) {
      const int s = j % S, kb = (t0 + j) * BN;
      if (!waited && kb + BN > len) {
        pdl_wait();
        waited = true;
      }
      float x[BN / 32];
#pragma unroll
      for (int e = 0; e < BN / 32; ++e) {
        const int key = kb + e * 32 + lane;
        x[e] = key >= nkeys ? -INFINITY : bias ? bias[key] : 0.f;
      }
      if (j >= S && !mbar_wait_warp(&v_empty[s], ((j / S) - 1) & 1, abort_flag, err, 87)) break;
#pragma unroll
      for (int e = 0; e < BN / 32; ++e) sB[s * BN + e * 32 + lane] = x[e] <= kDeadBias ? -INFINITY : x[e];
      mbar_arrive(&k_full[s]);
    }
  } else if (warp == 3) {
    // -------------------------------------------------- values behind the tree
    if (cut_tile >= 0 && mbar_wait_warp(v_cut, 0, abort_flag, err, 88)) {
      zero_tile_rows<BN, D / 64>(sV + (cut_tile % S) * L::kTile, nkeys - (t0 + cut_tile) * BN, lane, 32);
      fence_proxy_async_smem();
      mbar_arrive(v_clean);
    }
  } else {
    // -------------------------------------------------- softmax (thread = row)
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + x * BN, o_addr = tmem + lane_base + 256 + x * D;
    const int cnt = items(x);
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    const float sc_in = SOFTCLAMP ? a.scale / a.softclamp : 0.f;
    for (int i = 0; i < cnt; ++i) {
      const int j = tile_of(x, i), s = j % S, kb = (t0 + j) * BN;
      if (!mbar_wait_warp(&s_full[x], i & 1, abort_flag, err, 89)) { ok = false; break; }
      tc_fence_after();
      uint32_t v[BN];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
      tmem_wait_ld();
      if (!mbar_wait_warp(&k_full[s], (j / S) & 1, abort_flag, err, 91)) { ok = false; break; }   // the bias (long there)
      // scaled scores with their bias, natural units; log2(e) goes into the exponent's FFMA
      const float4* b4 = reinterpret_cast<const float4*>(sB + s * BN);
#pragma unroll
      for (int q = 0; q < BN / 4; ++q) {
        const float4 bb = b4[q];
        const float be[4] = {bb.x, bb.y, bb.z, bb.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = __uint_as_float(v[4 * q + e]);
          v[4 * q + e] = __float_as_uint(SOFTCLAMP ? fmaf(tanh_ex2(z * sc_in), a.softclamp, be[e]) : fmaf(z, a.scale, be[e]));
        }
      }
      if (kb + BN > len) {
        const uint64_t w0 = window(see, kb - len), w1 = window(see, kb - len + 64);
#pragma unroll
        for (int c = 0; c < BN; ++c)
          if (!(((c < 64 ? w0 : w1) >> (c & 63)) & 1)) v[c] = __float_as_uint(-INFINITY);
      }
      float mx[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) mx[u] = __uint_as_float(v[u]);
#pragma unroll
      for (int c = 4; c < BN; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(v[c]));
      const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kLog2e;
      const bool grow = tmax > m_run + 8.f;   // the reference maximum moves when the row's grows by more than 2^8
      const float m_new = grow ? tmax : m_run;
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = ex2(m_run - m_use);
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int c = 0; c < BN; c += 2) {
        const float e0 = ex2(fmaf(__uint_as_float(v[c]), kLog2e, -m_use));
        const float e1 = ex2(fmaf(__uint_as_float(v[c + 1]), kLog2e, -m_use));
        sum0 += e0;
        sum1 += e1;
        v[c >> 1] = pk2<T>(e0, e1);
      }
      l_run = l_run * alpha + (sum0 + sum1);
      m_run = m_new;
      if (i > 0 && __any_sync(0xffffffffu, grow)) {   // S(i) is full: P V(i - 1) is done
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int t = 0; t < 32; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * alpha);
          tmem_st32(o_addr + c * 32, o);
        }
        tmem_wait_st();
      }
      tmem_st32(s_addr, *reinterpret_cast<const uint32_t(*)[32]>(&v[0]));
      tmem_st32(s_addr + 32, *reinterpret_cast<const uint32_t(*)[32]>(&v[32]));
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }
    const bool have = ok && cnt > 0 && mbar_wait_warp(&o_done[x], (cnt - 1) & 1, abort_flag, err, 90);
    if (have) tc_fence_after();
    if (!see || !have) {   // padding, or no key: nothing is kept
      m_run = -INFINITY;
      l_run = 0.f;
    }
    pdl_wait();   // nothing is written before the previous kernel of the step is done
    // one row tile: the second warpgroup's sums go through shared memory (the stages are idle: both
    // warpgroups' products are done) to the first
    constexpr int RS = D + 4;
    float* side = (float*)(smem + L::kK) + r * RS;
    float m2 = -INFINITY, f0 = 1.f, f1 = 0.f;
    if (!ROWS2) {
      // both warpgroups' products have to be done before the stages are overwritten
      named_bar_sync(1, 256);
      if (x == 1) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (have) {
            tmem_ld32(o_addr + c * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<uint4*>(side + c * 32 + q * 4) =
                have ? make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]) : make_uint4(0u, 0u, 0u, 0u);
        }
        side[D] = m_run;
        side[D + 1] = l_run;
      }
      named_bar_sync(1, 256);
      if (x == 0) {
        m2 = side[D];
        const float M = fmaxf(m_run, m2);
        f0 = m_run == -INFINITY ? 0.f : ex2(m_run - M);
        f1 = m2 == -INFINITY ? 0.f : ex2(m2 - M);
        l_run = l_run * f0 + side[D + 1] * f1;
        m_run = M;
      }
    }
    if (ROWS2 || x == 0) {
      const int rows = R * a.nodes, m = node * R + head;
      float* rec = P.geo.splits > 1 ? P.geo.part + (((int64_t)blockIdx.y * rows + m) * P.geo.splits + split) * kRecord<D> : nullptr;
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;   // (NaN stays)
      const bool keep0 = have && f0 != 0.f && l_run != 0.f, keep1 = !ROWS2 && f1 != 0.f && l_run != 0.f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (have) {   // warp-uniform
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int t = 0; t < 32; t += 8) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = keep0 ? __uint_as_float(o[t + e]) * f0 : 0.f;
          if (keep1) {
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              const float4 z = *reinterpret_cast<const float4*>(side + c * 32 + t + e);
              y[e] = fmaf(z.x, f1, y[e]);
              y[e + 1] = fmaf(z.y, f1, y[e + 1]);
              y[e + 2] = fmaf(z.z, f1, y[e + 2]);
              y[e + 3] = fmaf(z.w, f1, y[e + 3]);
            }
          }
          if (!row_ok) continue;
          if (rec) {
            *reinterpret_cast<float4*>(rec + c * 32 + t) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(rec + c * 32 + t + 4) = make_float4(y[4], y[5], y[6], y[7]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= inv;
            write_row8<T>(a, b, g * R + head, node, len, c * 32 + t, y);
          }
        }
      }
      if (row_ok) {
        if (rec) {
          rec[D] = m_run;
          rec[D + 1] = l_run;
        } else {
          write_lse(a, b, g * R + head, node, len, l_run == 0.f ? -FLT_MAX : (m_run + __log2f(l_run)) * kLn2);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

int padded_nodes(const PolyTreePass& a) { return (a.nodes + 7) & ~7; }

template <typename T, int D, bool ROWS2, bool SC>
int launch_t(const PolyTreePass& a, const TreeGeom& geo, cudaStream_t s, bool dependent) {
  using L = Lay<D, ROWS2>;
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_smem((const void*)tree_tc_kernel<T, D, ROWS2, SC>, L::kAlloc, done,
                                "cudaFuncSetAttribute(tree tc)")) return rc;
  CUtensorMap tq, tk, tv;
  int rc = make_map(&tq, a.q, a.dtype, D, a.nodes, a.heads, a.batch, a.q_stride, a.nodes);
  if (!rc) rc = make_map(&tk, a.k, a.dtype, D, a.capacity, a.kv_heads, a.batch, a.k_stride, BN);
  if (!rc) rc = make_map(&tv, a.v, a.dtype, D, a.capacity, a.kv_heads, a.batch, a.v_stride, BN);
  if (rc) return rc;
  TreeTcParams p{};
  p.a = a;
  p.geo = geo;
  p.tp = padded_nodes(a);
  p.heads_tile = BM / p.tp;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(geo.splits * geo.row_blocks, a.batch * a.kv_heads);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = s;
  cudaLaunchAttribute attr = dependent_launch();
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  note_launch(1);
  return cuda_status(cudaLaunchKernelEx(&cfg, tree_tc_kernel<T, D, ROWS2, SC>, tq, tk, tv, p), "tree tc launch");
}

template <typename T, int D>
int launch_d(const PolyTreePass& a, const TreeGeom& geo, cudaStream_t s, bool dep) {
  const bool rows2 = a.heads / a.kv_heads > BM / padded_nodes(a), sc = a.softclamp > 0.f;
  if (rows2) return sc ? launch_t<T, D, true, true>(a, geo, s, dep) : launch_t<T, D, true, false>(a, geo, s, dep);
  return sc ? launch_t<T, D, false, true>(a, geo, s, dep) : launch_t<T, D, false, false>(a, geo, s, dep);
}

}  // namespace

// Row blocks of the tcgen05 pass, or 0 where the mma.sync kernel serves: its 16-row
// tiles keep up with the cache to about 32 rows; q has to suit a
// TMA box per head and the outputs 16-byte stores.
int tree_tc_row_blocks(const PolyTreePass& a) {
  const int R = a.heads / a.kv_heads;
  if (a.v_mul || a.nodes * R <= 32 || a.scale < 0.f) return 0;
  if (!aligned16(a.q) || !strides_ok(a.q_stride, 3)) return 0;
  if (a.out && (!aligned16(a.out) || !strides_ok(a.out_stride, 3))) return 0;
  if (a.cache_out && (!aligned16(a.cache_out) || !strides_ok(a.cache_out_stride, 3))) return 0;
  const int per_tile = BM / padded_nodes(a), per_block = R > per_tile ? 2 * per_tile : per_tile;
  return (R + per_block - 1) / per_block;
}

int launch_tree_tc(const PolyTreePass& a, const TreeGeom& geo, cudaStream_t s, bool dependent) {
  if (a.dtype == POLY_BF16)
    return a.head_dim == 64 ? launch_d<__nv_bfloat16, 64>(a, geo, s, dependent) : launch_d<__nv_bfloat16, 128>(a, geo, s, dependent);
  return a.head_dim == 64 ? launch_d<__half, 64>(a, geo, s, dependent) : launch_d<__half, 128>(a, geo, s, dependent);
}

}  // namespace poly
