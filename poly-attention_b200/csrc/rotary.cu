// Rotary positions of query / key tensors read straight from strided
// head-split views, up to POLY_MAX_ROTARY tensors of one call in one launch.
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_b cos t + x_a sin t)
//
// for the pairs (a, b) = (2i, 2i + 1) (interleaved) or (i, i + rot / 2) (half
// layout) of the first rot features, t = position * inv_freq_i or a given
// angle; features past rot are copied. The transpose (the gradient) is the same
// rotation with sin negated.
//
// Bound by HBM: every tensor is read and written once. The angles are the only
// arithmetic of weight and depend on (row, pair) alone, so a CTA owns a few rows of
// every head of every tensor, forms their cos / sin once in shared memory with the
// addresses of its rows and heads, and its threads walk (row, head) pairs in the
// order in which they lie in memory, four 16-byte loads ahead. Measured at b8 h16
// n4096 d64 (three tensors, 403 MB moved), ways that were left: addresses by division
// per 16 bytes, one load ahead: 116 us; a thread per row with its angles in
// registers, walking the heads: 85 us, but neighbouring threads 2 KB apart.
#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "packed.cuh"

namespace poly {
namespace {

constexpr int kThreads = 256;
constexpr int kTableBytes = 16 * 1024;   // cos / sin pairs of a CTA's rows
constexpr int kMaxRows = 16;             // rows per CTA
constexpr int kMaxHeads = 128;           // heads per CTA

struct RotaryPlan {
  PolyRotaryArgs a;
  int units;             // threads of a row: a run of features each
  int rows_per_cta;      // rows (of all batch elements)
  int heads_total;
  int head_split;        // CTAs that share their rows' heads
  int rows_first;        // walk the rows of a head before the next head (head-major tensors)
};

// cos and sin of an angle of any size: reduced to a turn in 64 bits, because an
// fp32 product position * inv_freq is off by 0.03 rad at position 2^19 already.
__device__ __forceinline__ float2 turn(double ang, float m, bool inverse) {
  double r = ang * 0.15915494309189533577;   // 1 / (2 pi)
  r -= rint(r);
  float s, c;
  sincospif((float)(2.0 * r), &s, &c);
  return make_float2(c * m, inverse ? -s * m : s * m);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// two neighbouring elements as fp32 and back, one conversion for both
template <typename T>
__device__ __forceinline__ float2 get2(const T* p) {
  if constexpr (std::is_same<T, float>::value) {
    return make_float2(p[0], p[1]);
  } else if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(p));
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}
template <typename T>
__device__ __forceinline__ void put2(T* p, float a, float b) {
  if constexpr (std::is_same<T, float>::value) {
    p[0] = a;
    p[1] = b;
  } else if constexpr (std::is_same<T, __half>::value) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
  } else {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
  }
}

// V elements per access: 16 bytes when every row and pointer allows it; else one
// element of a pair (V = 1).
// TWO: a unit is two runs.
template <typename T, int V, bool TWO>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const __grid_constant__ RotaryPlan P) {
  using X = Vec<T, V>;
  constexpr int kAhead = TWO ? 2 : 4;      // (row, head) pairs in flight per thread
  extern __shared__ __align__(16) float2 cs[];                // [rows][half]
  __shared__ struct { const T* src; T* dst; } head_at[kMaxHeads];
  __shared__ uint8_t head_k[kMaxHeads];                        // the head's tensor
  __shared__ struct { int64_t src, dst; } row_at[kMaxRows][POLY_MAX_ROTARY];
  const PolyRotaryArgs& a = P.a;
  const int half = a.rot >> 1, part = blockIdx.x % P.head_split;
  const int64_t flat0 = (int64_t)(blockIdx.x / P.head_split) * P.rows_per_cta, all = (int64_t)a.batch * a.rows;
  const int nrows = (int)min((int64_t)P.rows_per_cta, all - flat0);
  const int h0 = (int)((int64_t)P.heads_total * part / P.head_split);
  const int nh = (int)((int64_t)P.heads_total * (part + 1) / P.head_split) - h0;
  for (int i = threadIdx.x; i < nh; i += kThreads) {
    int h = h0 + i, k = 0;
    while (h >= a.t[k].heads) h -= a.t[k++].heads;
    head_at[i].src = (const T*)a.t[k].src + h * a.t[k].src_stride[1];
    head_at[i].dst = (T*)a.t[k].dst + h * a.t[k].dst_stride[1];
    head_k[i] = (uint8_t)k;
  }
  for (int i = threadIdx.x; i < nrows * a.n; i += kThreads) {
    const int r = i / a.n, k = i - r * a.n;
    const int64_t b = (flat0 + r) / a.rows, row = (flat0 + r) - b * a.rows;
    row_at[r][k].src = b * a.t[k].src_stride[0] + row * a.t[k].src_stride[2];
    row_at[r][k].dst = b * a.t[k].dst_stride[0] + row * a.t[k].dst_stride[2];
  }
  for (int i = threadIdx.x; i < nrows * half; i += kThreads) {
    const int r = i / half, f = i - r * half;
    const int64_t b = (flat0 + r) / a.rows, row = (flat0 + r) - b * a.rows;
    double ang;
    if (a.angles) {
      ang = (double)a.angles[b * a.angle_stride[0] + row * a.angle_stride[1] + f];
    } else {
      int64_t pos = a.pos_start;
      if (a.cu_seqlens)
        pos += row - packed_start(a.cu_seqlens, a.seqs, a.rows, (int)row);
      else if (a.positions)
        pos += a.pos_wide ? ((const int64_t*)a.positions)[b * a.pos_stride[0] + row * a.pos_stride[1]]
                          : (int64_t)((const int32_t*)a.positions)[b * a.pos_stride[0] + row * a.pos_stride[1]];
      else
        pos += row;
      ang = (double)pos * (double)a.inv_freq[f];
    }
    cs[i] = turn(ang, a.factor, a.inverse != 0);
  }
  __syncthreads();

  // A unit is one run of interleaved pairs, a run of first halves with its run of
  // second halves, or what lies past rot: there a run, or two where a unit is two.
  const bool il = a.interleaved != 0;
  const int rot_units = V == 1 ? half : (il ? a.rot : half) / V;
  const int groups = kThreads / P.units, grp = threadIdx.x / P.units, u = threadIdx.x - grp * P.units;
  if (grp >= groups) return;
  const bool turns = u < rot_units;
  int c0, c1 = -1;
  if (turns) {
    c0 = V == 1 && il ? 2 * u : u * V;
    if (TWO) c1 = V == 1 && il ? 2 * u + 1 : half + u * V;
  } else {
    c0 = a.rot + (u - rot_units) * (TWO ? 2 * V : V);
    if (TWO && c0 + V < a.dim) c1 = c0 + V;
  }
  const int pair0 = V == 1 ? u : il ? u * (V / 2) : u * V;
  const int total = nrows * nh, inner = P.rows_first ? nrows : nh;
  int o = grp / inner, in = grp - o * inner;   // outer and inner place of this thread's next pair
  const int step_o = groups / inner, step_in = groups - step_o * inner;
  for (int it = grp; it < total; it += groups * kAhead) {
    X x[kAhead], y[kAhead];
    T* dst[kAhead];
    int row[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (it + i * groups < total) {
        const int r = P.rows_first ? in : o, h = P.rows_first ? o : in, k = head_k[h];
        const T* src = head_at[h].src + row_at[r][k].src;
        dst[i] = head_at[h].dst + row_at[r][k].dst;
        row[i] = r;
        x[i] = *reinterpret_cast<const X*>(src + c0);
        if (TWO && c1 >= 0) y[i] = *reinterpret_cast<const X*>(src + c1);
        in += step_in;
        o += step_o;
        if (in >= inner) {
          in -= inner;
          ++o;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (it + i * groups < total) {
        if (turns) {
          const float2* w = cs + row[i] * half + pair0;
          if constexpr (!TWO) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
              const float4 q = *reinterpret_cast<const float4*>(w + (e >> 1));   // two pairs
              const float2 p0 = get2(&x[i].e[e]), p1 = get2(&x[i].e[e + 2]);
              put2(&x[i].e[e], p0.x * q.x - p0.y * q.y, p0.y * q.x + p0.x * q.y);
              put2(&x[i].e[e + 2], p1.x * q.z - p1.y * q.w, p1.y * q.z + p1.x * q.w);
            }
          } else if constexpr (V > 1) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float4 q = *reinterpret_cast<const float4*>(w + e);
              const float2 p0 = get2(&x[i].e[e]), p1 = get2(&y[i].e[e]);
              put2(&x[i].e[e], p0.x * q.x - p1.x * q.y, p0.y * q.z - p1.y * q.w);
              put2(&y[i].e[e], p1.x * q.x + p0.x * q.y, p1.y * q.z + p0.y * q.w);
            }
          } else {
            const float p0 = to_f32(x[i].e[0]), p1 = to_f32(y[i].e[0]);
            x[i].e[0] = from_f32<T>(p0 * w->x - p1 * w->y);
            y[i].e[0] = from_f32<T>(p1 * w->x + p0 * w->y);
          }
        }
        *reinterpret_cast<X*>(dst[i] + c0) = x[i];
        if (TWO && c1 >= 0) *reinterpret_cast<X*>(dst[i] + c1) = y[i];
      }
    }
  }
}

bool vector_ok(const PolyRotaryArgs& a, int v, int es) {
  const int run = a.interleaved ? a.rot : a.rot / 2;
  if (run % v || (a.dim - a.rot) % v || a.dim % v) return false;
  for (int k = 0; k < a.n; ++k) {
    const PolyRotaryTensor& t = a.t[k];
    if (((uintptr_t)t.src | (uintptr_t)t.dst) & 15) return false;
    for (int i = 0; i < 3; ++i)
      if ((t.src_stride[i] * es) & 15 || (t.dst_stride[i] * es) & 15) return false;
  }
  return true;
}

int fail(const std::string& m) {
  set_error("poly_rotary: " + m);
  return POLY_EINVAL;
}

template <typename T>
int launch_t(RotaryPlan& p, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  PolyRotaryArgs& a = p.a;
  const int half = a.rot / 2;
  static std::atomic<int> sms[64] = {};   // per device; host threads may call at once
  int dev = 0;
  if (const int rc = cuda_status(cudaGetDevice(&dev), "cudaGetDevice")) return rc;
  int n_sm = dev < 64 ? sms[dev].load(std::memory_order_relaxed) : 0;
  if (!n_sm) {
    if (cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n_sm <= 0) n_sm = 148;
    if (dev < 64) sms[dev].store(n_sm, std::memory_order_relaxed);
  }
  const bool vec = vector_ok(a, V, sizeof(T));
  const int v = vec ? V : 1, run = a.interleaved && vec ? a.rot : half, rest = a.dim - a.rot;
  const int span = a.interleaved && vec ? v : 2 * v;   // features of a unit
  p.units = run / v + (rest + span - 1) / span;
  p.rows_first = 0;
  for (int k = 0; k < a.n; ++k) p.rows_first |= a.t[k].heads > 1 && a.t[k].src_stride[2] < a.t[k].src_stride[1];
  // rows of a CTA: as many as the table holds, fewer while that leaves SMs idle
  const int64_t rows = (int64_t)a.batch * a.rows;
  p.rows_per_cta = std::max(1, std::min(kMaxRows, kTableBytes / (int)sizeof(float2) / half));
  while (p.rows_per_cta > 1 && (rows + p.rows_per_cta - 1) / p.rows_per_cta < 4 * n_sm) p.rows_per_cta = (p.rows_per_cta + 1) / 2;
  const int64_t tiles = (rows + p.rows_per_cta - 1) / p.rows_per_cta;
  // few rows, or more heads than a CTA holds: several CTAs share the heads (each forms the same angles)
  p.head_split = (p.heads_total + kMaxHeads - 1) / kMaxHeads;
  if (tiles < 2 * n_sm)
    p.head_split = (int)std::max<int64_t>(p.head_split, std::min<int64_t>((p.heads_total + 3) / 4, (2 * n_sm + tiles - 1) / tiles));
  const int64_t grid = tiles * p.head_split;
  if (grid > 0x7fffffff) return fail("too many rows for one call");
  const size_t smem = sizeof(float2) * (size_t)p.rows_per_cta * half;
  if (!vec)
    rotary_kernel<T, 1, true><<<(unsigned)grid, kThreads, smem, s>>>(p);
  else if (a.interleaved)
    rotary_kernel<T, V, false><<<(unsigned)grid, kThreads, smem, s>>>(p);
  else
    rotary_kernel<T, V, true><<<(unsigned)grid, kThreads, smem, s>>>(p);
  note_launch(1);
  return cuda_status(cudaGetLastError(), "rotary launch");
}

}  // namespace

int rotary(const PolyRotaryArgs* args, cudaStream_t s) {
  if (!args) return fail("null args");
  const PolyRotaryArgs& a = *args;
  if (a.n < 0 || a.n > POLY_MAX_ROTARY) return fail("n must be in [0, " + std::to_string(POLY_MAX_ROTARY) + "]");
  if (a.batch < 0 || a.rows < 0 || a.dim <= 0 || a.dim > 256) return fail("bad sizes (dim <= 256)");
  if (a.rot <= 0 || a.rot > a.dim || (a.rot & 1)) return fail("rot must be even and in [2, dim]");
  if (a.dtype != POLY_F32 && a.dtype != POLY_F16 && a.dtype != POLY_BF16) return fail("unknown dtype");
  if (!a.inv_freq == !a.angles) return fail("give either inv_freq or angles");
  if ((a.positions != nullptr) + (a.cu_seqlens != nullptr) + (a.angles != nullptr) > 1)
    return fail("positions, cu_seqlens and angles exclude one another");
  if (a.cu_seqlens && (a.batch > 1 || a.seqs <= 0)) return fail("cu_seqlens needs batch 1 and at least one sequence");
  RotaryPlan p{};
  p.a = a;
  for (int k = 0; k < a.n; ++k) {
    if (!a.t[k].src || !a.t[k].dst || a.t[k].heads <= 0) return fail("null tensor or no heads");
    p.heads_total += a.t[k].heads;
  }
  if (a.n == 0 || a.batch == 0 || a.rows == 0) return POLY_OK;
  switch (a.dtype) {
    case POLY_F32: return launch_t<float>(p, s);
    case POLY_F16: return launch_t<__half>(p, s);
    default: return launch_t<__nv_bfloat16>(p, s);
  }
}

}  // namespace poly
