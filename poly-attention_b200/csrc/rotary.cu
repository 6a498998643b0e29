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
// arithmetic and depend on (row, pair) alone, so a CTA owns a few rows of every
// head of every tensor: it forms their cos / sin once in shared memory and
// streams the heads through 16-byte loads and stores.
#include <algorithm>
#include <string>

#include "common.cuh"
#include "packed.cuh"

namespace poly {
namespace {

constexpr int kThreads = 256;
constexpr int kTableBytes = 16 * 1024;   // cos / sin pairs of a CTA's rows

struct RotaryPlan {
  PolyRotaryArgs a;
  int rows_per_cta;      // consecutive rows whose cos / sin the CTA holds
  int row_tiles;         // per batch element
  int heads_total;
  int head_split;        // CTAs that share a row tile, each with its heads
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

// V elements per access: 16 bytes when every row and pointer allows it, else 1.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryPlan P) {
  extern __shared__ __align__(16) float2 cs[];   // [rows_per_cta][rot / 2]
  const PolyRotaryArgs& a = P.a;
  const int half = a.rot >> 1;
  const int part = blockIdx.x % P.head_split;
  const int tile = blockIdx.x / P.head_split;
  const int b = tile / P.row_tiles;
  const int row0 = (tile - b * P.row_tiles) * P.rows_per_cta;
  const int nrows = min(P.rows_per_cta, a.rows - row0);
  for (int i = threadIdx.x; i < nrows * half; i += kThreads) {
    const int r = i / half, f = i - r * half;
    const int64_t row = row0 + r;
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

  // a unit is a run of V features: a whole number of interleaved pairs, or a
  // run of first halves with its run of second halves, or a run past rot
  const int rot_units = (a.interleaved ? a.rot : half) / V;
  const int units = rot_units + (a.dim - a.rot) / V;
  const int h0 = (int)((int64_t)P.heads_total * part / P.head_split);
  const int h1 = (int)((int64_t)P.heads_total * (part + 1) / P.head_split);
  const int nh = h1 - h0, total = nrows * nh * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int u = i % units, rh = i / units;
    const int hh = rh % nh, r = rh / nh;
    int h = h0 + hh, k = 0;
    while (h >= a.t[k].heads) h -= a.t[k++].heads;
    const PolyRotaryTensor& t = a.t[k];
    const T* src = (const T*)t.src + b * t.src_stride[0] + h * t.src_stride[1] + (int64_t)(row0 + r) * t.src_stride[2];
    T* dst = (T*)t.dst + b * t.dst_stride[0] + h * t.dst_stride[1] + (int64_t)(row0 + r) * t.dst_stride[2];
    const float2* w = cs + r * half;
    if (u >= rot_units) {
      const int c = a.rot + (u - rot_units) * V;
      *reinterpret_cast<Vec<T, V>*>(dst + c) = *reinterpret_cast<const Vec<T, V>*>(src + c);
    } else if (a.interleaved) {
      if constexpr (V > 1) {
        Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(src + u * V);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 q = w[(u * V + e) >> 1];
          const float p0 = to_f32(x.e[e]), p1 = to_f32(x.e[e + 1]);
          x.e[e] = from_f32<T>(p0 * q.x - p1 * q.y);
          x.e[e + 1] = from_f32<T>(p1 * q.x + p0 * q.y);
        }
        *reinterpret_cast<Vec<T, V>*>(dst + u * V) = x;
      } else if ((u & 1) == 0) {   // one thread writes both of a pair (dst may be src)
        const float2 q = w[u >> 1];
        const float p0 = to_f32(src[u]), p1 = to_f32(src[u + 1]);
        dst[u] = from_f32<T>(p0 * q.x - p1 * q.y);
        dst[u + 1] = from_f32<T>(p1 * q.x + p0 * q.y);
      }
    } else {
      Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(src + u * V);
      Vec<T, V> y = *reinterpret_cast<const Vec<T, V>*>(src + half + u * V);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 q = w[u * V + e];
        const float p0 = to_f32(x.e[e]), p1 = to_f32(y.e[e]);
        x.e[e] = from_f32<T>(p0 * q.x - p1 * q.y);
        y.e[e] = from_f32<T>(p1 * q.x + p0 * q.y);
      }
      *reinterpret_cast<Vec<T, V>*>(dst + u * V) = x;
      *reinterpret_cast<Vec<T, V>*>(dst + half + u * V) = y;
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
  static int sms[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int n_sm = dev < 64 ? sms[dev] : 0;
  if (!n_sm) {
    if (cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n_sm <= 0) n_sm = 148;
    if (dev < 64) sms[dev] = n_sm;
  }
  // rows of a CTA: as many as the table holds, fewer while that leaves SMs idle
  p.rows_per_cta = std::max(1, std::min(16, kTableBytes / (int)sizeof(float2) / std::max(half, 1)));
  while (p.rows_per_cta > 1 && (int64_t)a.batch * ((a.rows + p.rows_per_cta - 1) / p.rows_per_cta) < 4 * n_sm)
    p.rows_per_cta = (p.rows_per_cta + 1) / 2;
  p.row_tiles = (a.rows + p.rows_per_cta - 1) / p.rows_per_cta;
  const int64_t tiles = (int64_t)a.batch * p.row_tiles;
  // few rows: several CTAs share a row tile's heads (each forms the same angles)
  p.head_split = 1;
  if (tiles < 2 * n_sm) p.head_split = (int)std::min<int64_t>(p.heads_total, (2 * n_sm + tiles - 1) / tiles);
  const int64_t grid = tiles * p.head_split;
  if (grid > 0x7fffffff) return fail("too many rows for one call");
  const size_t smem = sizeof(float2) * (size_t)p.rows_per_cta * std::max(half, 1);
  if (vector_ok(a, V, sizeof(T)))
    rotary_kernel<T, V><<<(unsigned)grid, kThreads, smem, s>>>(p);
  else
    rotary_kernel<T, 1><<<(unsigned)grid, kThreads, smem, s>>>(p);
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
