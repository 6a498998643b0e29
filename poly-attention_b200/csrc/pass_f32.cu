// fp32 attention pass on the tensor cores with 3xTF32 (config 1's fp32
// PolyAttention forward, poly_attention/poly_attention.py:63-114): every
// product a.b is formed as a_hi.b_hi + a_hi.b_lo + a_lo.b_hi from the TF32
// split x_hi = tf32(x), x_lo = tf32(x - x_hi), which keeps the error near fp32
// rounding (the fp32 parity bar is 1e-4; plain TF32 would miss it).
//
// CTA = 64 query rows of one (batch, head), 4 warps x 16 rows; key tiles of 64
// through a 2-stage cp.async ring (rows padded to 68 floats: the fragment
// loads below are bank-conflict free). mma.sync m16n8k8 tf32. The score
// accumulator pairs keys (2t, 2t + 1) per lane; P.V uses that pairing as its
// K order (V rows are read in the same order), so P never moves between lanes.
// Online softmax in the log2 domain. Rows whose every key is excluded get the
// reference's -finfo.max result: a uniform average over the keys that are not
// both masked (causal) and dead (bias <= -FLT_MAX / 2), lse = -FLT_MAX.
//
// PACKED: sequences laid end to end, one CTA per 64-row slot (packed.cuh) and
// head; slots are taken from the last to the first, so that of a causal sequence
// the rows with the most keys start first. Three groups of 4 warps share the CTA's
// rows, each with every third key tile, and join at the end: sequences of unequal
// lengths leave few CTAs for the longest one's last rows. The MMAs alone (8 cycles an
// m16n8k8 on a quarter of an SM, measured) would take 42 of the 105 us of a pass of
// 4099 tokens in 7 sequences, h8 d64; the rest is the splits and the softmax that the
// same warps do between them. A split in four instructions took an order-2 forward from 231 us
// to 204; a fourth group with 32-key tiles or an exact order by keys gave no more than 3%.
#include <cfloat>

#include "common.cuh"
#include "packed.cuh"

namespace poly {
namespace {

constexpr int D = 64, BM = 64, LD = D + 4;   // padded row pitch (floats)
// groups of 4 warps over the key tiles, keys of a tile, bytes of a group's two-stage ring (K, V, bias)
template <bool PACKED>
struct Shape {
  static constexpr int KG = PACKED ? 3 : 1, BN = 64, kRing = (4 * BN * LD + 2 * BN) * 4;
  static constexpr int kSmem = KG * kRing;
};

__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = tf32(x);
  lo = tf32(x - __uint_as_float(hi));
}
// x_hi rounded to nearest (ties away) by integer arithmetic, x_lo cut off: 2^-21 of x is lost instead of
// 2^-22, for 4 instructions instead of about 10; with lo rounded too (6) the results are no nearer to 64 bits (8.2e-7
// both) and the time is that of before (234 us against 204). NaN and infinity leave a NaN in lo.
__device__ __forceinline__ void split_fast(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
template <bool PACKED>
__device__ __forceinline__ void split_for(float x, uint32_t& hi, uint32_t& lo) {
  if constexpr (PACKED) split_fast(x, hi, lo);
  else split(x, hi, lo);
}
__device__ __forceinline__ void mma8(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t sa, const void* g, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sa), "l"(g), "r"(ok ? 16 : 0) : "memory");
}

template <bool HAS_BIAS, bool SOFTCLAMP, bool PACKED>
__global__ void __launch_bounds__(Shape<PACKED>::KG * 128) pass_f32_kernel(PolyPassArgs a, const PackedSeqs pk) {
  constexpr int KG = Shape<PACKED>::KG, BN = Shape<PACKED>::BN;
  extern __shared__ __align__(16) float smf[];
  const int kg = PACKED ? threadIdx.x >> 7 : 0, tid = threadIdx.x & 127;
  float* ring = smf + kg * (Shape<PACKED>::kRing / 4);
  float(*sK)[BN * LD] = reinterpret_cast<float(*)[BN * LD]>(ring);
  float(*sV)[BN * LD] = reinterpret_cast<float(*)[BN * LD]>(ring + 2 * BN * LD);
  float(*sB)[BN] = reinterpret_cast<float(*)[BN]>(ring + 4 * BN * LD);
  auto sync = [&] {   // the group's warps
    if constexpr (PACKED) asm volatile("bar.sync %0, 128;" ::"r"(1 + kg) : "memory");
    else __syncthreads();
  };
  // packed: heads fastest, so that CTAs running together share a sequence's keys
  const int bh = PACKED ? blockIdx.x : blockIdx.y;
  const int b = PACKED ? 0 : bh / a.heads, h = bh - b * a.heads, g = h / (a.heads / a.kv_heads);
  int tile = blockIdx.x;
  if constexpr (PACKED) {
    const int own = pk.total / BM + pk.seqs;   // the CTAs behind these zero the rows outside the sequences
    if ((int)blockIdx.y >= own) {
      if (bh == 0) packed_zero_rest(pk, blockIdx.y - own);
      return;
    }
    PackedTile t;
    if (!packed_tile<BM>(pk.cu, pk.seqs, pk.total, own - 1 - blockIdx.y, t)) return;
    tile = t.tile;
    a.seq_q = a.seq_k = t.len;
    const int64_t f = t.start;
    a.q = (const float*)a.q + f * a.q_stride[2];
    a.k = (const float*)a.k + f * a.k_stride[2];
    a.v = (const float*)a.v + f * a.v_stride[2];
    a.out = (float*)a.out + f * a.out_stride[2];
    if (HAS_BIAS) a.bias += f;
    if (a.lse) a.lse += f;
    if (a.epi_out) {
      a.epi_mul = (const float*)a.epi_mul + f * a.epi_mul_stride[2];
      a.epi_out = (float*)a.epi_out + f * a.epi_out_stride[2];
    }
  }
  const int warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
  const int i0 = tile * BM + warp * 16 + gq, i1 = i0 + 8;   // this thread's two rows
  const int nq = a.seq_q, nk = a.seq_k;
  const float* kp = (const float*)a.k + b * a.k_stride[0] + g * a.k_stride[1];
  const float* vg = (const float*)a.v + b * a.v_stride[0] + g * a.v_stride[1];
  const float* bg = HAS_BIAS ? a.bias + b * a.bias_stride[0] + g * a.bias_stride[1] : nullptr;
  const int kend = a.causal ? min(nk, tile * BM + BM) : nk;
  const int ntile = (kend + BN - 1) / BN;

  auto issue = [&](int t) {
    const int st = (t / KG) & 1, j0 = t * BN;
    for (int c = tid; c < BN * (D / 4); c += 128) {
      const int r = c / (D / 4), ch = c - r * (D / 4);
      const bool ok = j0 + r < nk;
      const int rr = ok ? j0 + r : 0;
      cp16((uint32_t)__cvta_generic_to_shared(&sK[st][r * LD + ch * 4]), kp + (int64_t)rr * a.k_stride[2] + ch * 4, ok);
      cp16((uint32_t)__cvta_generic_to_shared(&sV[st][r * LD + ch * 4]), vg + (int64_t)rr * a.v_stride[2] + ch * 4, ok);
    }
    if (tid < BN) {
      const int j = j0 + tid;
      float x = 0.f;
      if (HAS_BIAS && j < nk) {
        const float raw = bg[j];
        x = raw <= kDeadBias ? -INFINITY : raw * kLog2e;
      }
      sB[st][tid] = x;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // A fragments of Q split into TF32 hi / lo (rows i0 / i1, K steps of 8)
  uint32_t qh[D / 8][4], ql[D / 8][4];
  {
    const float* qb = (const float*)a.q + b * a.q_stride[0] + h * a.q_stride[1];
    const float* q0 = qb + (int64_t)(i0 < nq ? i0 : 0) * a.q_stride[2];
    const float* q1 = qb + (int64_t)(i1 < nq ? i1 : 0) * a.q_stride[2];
#pragma unroll
    for (int ks = 0; ks < D / 8; ++ks) {
      const float x[4] = {i0 < nq ? q0[ks * 8 + tq] : 0.f, i1 < nq ? q1[ks * 8 + tq] : 0.f,
                          i0 < nq ? q0[ks * 8 + tq + 4] : 0.f, i1 < nq ? q1[ks * 8 + tq + 4] : 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) split_for<PACKED>(x[e], qh[ks][e], ql[ks][e]);
    }
  }
  const float qk = SOFTCLAMP ? a.scale / a.softclamp : a.scale * kLog2e;
  const float sc_out = SOFTCLAMP ? a.softclamp * kLog2e : 0.f;
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  if (kg < ntile) issue(kg);
  for (int t = kg; t < ntile; t += KG) {
    if (t + KG < ntile) {
      issue(t + KG);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    sync();
    const int st = (t / KG) & 1, j0 = t * BN;
    const float* K = sK[st];
    const float* V = sV[st];
    // S = Q K^T: n-block nb = keys j0 + 8 nb .. + 7. The three products of a step go
    // round all n-blocks in turn: MMAs on one accumulator wait for one another (about
    // 33 cycles), eight accumulators hide that. Each accumulator's order of sums is kept.
    float s[BN / 8][4];
#pragma unroll
    for (int nb = 0; nb < BN / 8; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 8; ++ks) {
      uint32_t bh[BN / 8][2], bl[BN / 8][2];
#pragma unroll
      for (int nb = 0; nb < BN / 8; ++nb) {
        const float* kr = K + (nb * 8 + gq) * LD + ks * 8 + tq;
        split_for<PACKED>(kr[0], bh[nb][0], bl[nb][0]);
        split_for<PACKED>(kr[4], bh[nb][1], bl[nb][1]);
      }
#pragma unroll
      for (int nb = 0; nb < BN / 8; ++nb) mma8(s[nb], ql[ks][0], ql[ks][1], ql[ks][2], ql[ks][3], bh[nb][0], bh[nb][1]);
#pragma unroll
      for (int nb = 0; nb < BN / 8; ++nb) mma8(s[nb], qh[ks][0], qh[ks][1], qh[ks][2], qh[ks][3], bl[nb][0], bl[nb][1]);
#pragma unroll
      for (int nb = 0; nb < BN / 8; ++nb) mma8(s[nb], qh[ks][0], qh[ks][1], qh[ks][2], qh[ks][3], bh[nb][0], bh[nb][1]);
    }
    float mx0 = m0, mx1 = m1;
    const bool edge = !PACKED || j0 + BN > nk || (a.causal && j0 + BN - 1 > tile * BM);   // keys that some row does not see
#pragma unroll
    for (int nb = 0; nb < BN / 8; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int jl = nb * 8 + 2 * tq + (e & 1), j = j0 + jl;
        const int row = e < 2 ? i0 : i1;
        float x = s[nb][e] * qk;
        if (SOFTCLAMP) x = tanhf(x) * sc_out;
        if (HAS_BIAS) x += sB[st][jl];
        if (edge && (j >= nk || (a.causal && j > row))) x = -INFINITY;
        s[nb][e] = x;
        if (e < 2) mx0 = fmaxf(mx0, x); else mx1 = fmaxf(mx1, x);
      }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float a0 = mx0 == -INFINITY ? 1.f : exp2f(m0 - mx0), a1 = mx1 == -INFINITY ? 1.f : exp2f(m1 - mx1);
    m0 = mx0;
    m1 = mx1;
    l0 *= a0;
    l1 *= a1;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      o[n][0] *= a0;
      o[n][1] *= a0;
      o[n][2] *= a1;
      o[n][3] *= a1;
    }
#pragma unroll
    for (int nb = 0; nb < BN / 8; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float m = e < 2 ? m0 : m1;
        const float p = s[nb][e] == -INFINITY ? 0.f : exp2f(s[nb][e] - m);
        s[nb][e] = p;
        if (e < 2) l0 += p; else l1 += p;
      }
    // O += P V: K step = n-block nb, element (row, t) <-> key 8 nb + 2t, (row, t + 4) <-> key 8 nb + 2t + 1
#pragma unroll
    for (int nb = 0; nb < BN / 8; ++nb) {
      uint32_t ph[4], pl[4];
      split_for<PACKED>(s[nb][0], ph[0], pl[0]);
      split_for<PACKED>(s[nb][2], ph[1], pl[1]);
      split_for<PACKED>(s[nb][1], ph[2], pl[2]);
      split_for<PACKED>(s[nb][3], ph[3], pl[3]);
      const float* v0 = V + (nb * 8 + 2 * tq) * LD;
      const float* v1 = v0 + LD;
      uint32_t bh[D / 8][2], bl[D / 8][2];
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        split_for<PACKED>(v0[n * 8 + gq], bh[n][0], bl[n][0]);
        split_for<PACKED>(v1[n * 8 + gq], bh[n][1], bl[n][1]);
      }
#pragma unroll
      for (int n = 0; n < D / 8; ++n) mma8(o[n], pl[0], pl[1], pl[2], pl[3], bh[n][0], bh[n][1]);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) mma8(o[n], ph[0], ph[1], ph[2], ph[3], bl[n][0], bl[n][1]);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) mma8(o[n], ph[0], ph[1], ph[2], ph[3], bh[n][0], bh[n][1]);
    }
    sync();   // the stage is refilled next iteration
  }
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  if constexpr (PACKED) {
    // the other groups' sums, thread by thread, through shared memory (the rings are idle)
    constexpr int kSide = (D / 2 + 4) * 128;   // [4 D / 8 + 4][128 threads]
    __syncthreads();
    if (kg) {
      float* side = smf + (kg - 1) * kSide + tid;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) side[(n * 4 + e) * 128] = o[n][e];
      side[D / 2 * 128] = m0;
      side[(D / 2 + 1) * 128] = m1;
      side[(D / 2 + 2) * 128] = l0;
      side[(D / 2 + 3) * 128] = l1;
    }
    __syncthreads();
    if (kg) return;
    for (int k = 0; k < KG - 1; ++k) {
      const float* side = smf + k * kSide + tid;
      const float y0 = side[D / 2 * 128], y1 = side[(D / 2 + 1) * 128];
      const float n0 = fmaxf(m0, y0), n1 = fmaxf(m1, y1);
      const float f0 = m0 == -INFINITY ? 0.f : exp2f(m0 - n0), f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - n1);
      const float g0 = y0 == -INFINITY ? 0.f : exp2f(y0 - n0), g1 = y1 == -INFINITY ? 0.f : exp2f(y1 - n1);
      m0 = n0;
      m1 = n1;
      l0 = l0 * f0 + side[(D / 2 + 2) * 128] * g0;
      l1 = l1 * f1 + side[(D / 2 + 3) * 128] * g1;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = o[n][e] * (e < 2 ? f0 : f1) + side[(n * 4 + e) * 128] * (e < 2 ? g0 : g1);
    }
  }

  float* ob = (float*)a.out + b * a.out_stride[0] + h * a.out_stride[1];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int row = hf ? i1 : i0;
    const float m = hf ? m1 : m0, l = hf ? l1 : l0;
    if (row >= nq) continue;
    float lse;
    float r[D / 8][2];
    if (PACKED ? l == 0.f : m == -INFINITY) {   // (a row of NaN scores has no maximum, but a sum)
      // every key excluded: uniform average over keys not both masked and dead
      // (packed rows: zero)
      int count = 0;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) r[n][0] = r[n][1] = 0.f;
      for (int j = 0; j < (PACKED ? 0 : nk); ++j) {
        const bool masked = a.causal && j > row;
        const bool dead = HAS_BIAS && bg[j] <= kDeadBias;
        if (masked && dead) continue;
        ++count;
        const float* vr = vg + (int64_t)j * a.v_stride[2];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          r[n][0] += vr[n * 8 + 2 * tq];
          r[n][1] += vr[n * 8 + 2 * tq + 1];
        }
      }
      const float inv = count ? 1.f / (float)count : 0.f;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        r[n][0] *= inv;
        r[n][1] *= inv;
      }
      lse = -FLT_MAX;
    } else {
      const float inv = 1.f / l;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        r[n][0] = o[n][2 * hf] * inv;
        r[n][1] = o[n][2 * hf + 1] * inv;
      }
      lse = (m + __log2f(l)) * kLn2;
    }
    float* orow = ob + (int64_t)row * a.out_stride[2];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(orow + n * 8 + 2 * tq) = make_float2(r[n][0], r[n][1]);
    if (PACKED && a.epi_out) {
      const float* em = (const float*)a.epi_mul + h * a.epi_mul_stride[1] + (int64_t)row * a.epi_mul_stride[2];
      float* eo = (float*)a.epi_out + h * a.epi_out_stride[1] + (int64_t)row * a.epi_out_stride[2];
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const int c = n * 8 + 2 * tq;
        eo[c] = em[c] * r[n][0];
        eo[c + 1] = em[c + 1] * r[n][1];
      }
    }
    if (a.lse && tq == 0) a.lse[b * a.lse_stride[0] + h * a.lse_stride[1] + row] = lse;
  }
}

bool al(const void* p, int bytes) { return ((uintptr_t)p % bytes) == 0; }

}  // namespace

bool pass_f32_eligible(const PolyPassArgs& a) {
  if (a.dtype != POLY_F32 || a.head_dim != D || a.seq_q < 1 || a.seq_k < 1) return false;
  if (a.key_mask || a.query_mask || a.v_mul || a.epi_out) return false;
  if (!al(a.k, 16) || !al(a.v, 16) || !al(a.out, 8)) return false;
  if ((a.k_stride[0] | a.k_stride[1] | a.k_stride[2] | a.v_stride[0] | a.v_stride[1] | a.v_stride[2]) & 3) return false;
  if ((a.out_stride[0] | a.out_stride[1] | a.out_stride[2]) & 1) return false;
  return true;
}

namespace {
template <bool B, bool C, bool PACKED>
int launch_t(const PolyPassArgs& a, const PackedSeqs* pk, cudaStream_t s) {
  using S = Shape<PACKED>;
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_smem((const void*)pass_f32_kernel<B, C, PACKED>, S::kSmem, done,
                                "cudaFuncSetAttribute(f32)")) return rc;
  const dim3 grid = PACKED ? dim3(a.heads, a.seq_q / BM + pk->seqs + zero_ctas(*pk)) : dim3((a.seq_q + BM - 1) / BM, a.batch * a.heads);
  pass_f32_kernel<B, C, PACKED><<<grid, S::KG * 128, S::kSmem, s>>>(a, PACKED ? *pk : PackedSeqs{});
  note_launch(1);
  return cuda_status(cudaGetLastError(), "pass_f32 launch");
}

template <bool PACKED>
int launch_any(const PolyPassArgs& a, const PackedSeqs* pk, cudaStream_t s) {
  const bool bias = a.bias != nullptr, sc = a.softclamp > 0.f;
  if (sc) return bias ? launch_t<true, true, PACKED>(a, pk, s) : launch_t<false, true, PACKED>(a, pk, s);
  return bias ? launch_t<true, false, PACKED>(a, pk, s) : launch_t<false, false, PACKED>(a, pk, s);
}
}  // namespace

int launch_pass_f32(const PolyPassArgs& a, cudaStream_t s) { return launch_any<false>(a, nullptr, s); }

// The slots are the grid's second axis, which holds 65535.
bool packed_f32_eligible(const PolyPackedArgs& pa) {
  const PolyPassArgs& a = pa.pass;
  if (a.dtype != POLY_F32 || a.head_dim != D || a.seq_q / BM + pa.seqs > 65535 - kZeroCtas) return false;
  if (!al(a.k, 16) || !al(a.v, 16) || !al(a.out, 8)) return false;
  return !((a.k_stride[1] | a.k_stride[2] | a.v_stride[1] | a.v_stride[2]) & 3) && !((a.out_stride[1] | a.out_stride[2]) & 1);
}
int launch_packed_fwd_f32(PolyPassArgs a, const PackedSeqs& q, cudaStream_t s) {
  return launch_any<true>(a, &q, s);
}

}  // namespace poly
