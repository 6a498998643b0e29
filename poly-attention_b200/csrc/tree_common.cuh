// Pieces shared by the tree decoding kernels (tree.cu: mma.sync and CUDA cores,
// tree_tc100.cu: tcgen05): programmatic dependence, the nodes' visibility, output rows.
#pragma once

#include "common.cuh"
#include "mma_sync.cuh"

namespace poly {
namespace treec {

constexpr int kNodes = POLY_MAX_TREE_NODES;
constexpr int kMaxSplits = 64;

// Visible tree nodes of every node as bits (0: padding), by pointer jumping: after
// round r a node knows its nearest 2^r ancestors. Callers with at least 64 threads.
__device__ __forceinline__ void ancestors(const int32_t* parents, int nodes, int room, uint64_t* mask, int* up) {
  const int i = threadIdx.x;
  if (i < kNodes) {
    int p = -2;
    if (i < nodes && i < room) {
      p = parents[i];
      if (p >= i || p < -1) p = -2;
    }
    mask[i] = p == -2 ? 0ull : 1ull << i;
    up[i] = p;
  }
  __syncthreads();
  for (;;) {   // at most 6 rounds: each doubles the distance
    uint64_t m = 0;
    int p = -2;
    if (i < kNodes) {
      m = mask[i];
      p = up[i];
      if (p >= 0) {
        // below a padding node: padding too
        m = mask[p] ? m | mask[p] : 0ull;
        p = mask[p] ? up[p] : -2;
      }
    }
    __syncthreads();
    if (i < kNodes) {
      mask[i] = m;
      up[i] = p;
    }
    if (!__syncthreads_or(p >= 0)) break;
  }
}

__device__ __forceinline__ int seq_length(const int32_t* lengths, int b, int capacity) {
  return min(max(lengths[b], 0), capacity);
}

// Row `m` of a group: query head g * R + m % R, node m / R.
template <typename T>
__device__ __forceinline__ void write_row(const PolyTreePass& a, int b, int h, int node, int len, int c, float x, float y) {
  const uint32_t w = ms::pk2<T>(x, y);
  if (a.out)
    *reinterpret_cast<uint32_t*>((T*)a.out + b * a.out_stride[0] + h * a.out_stride[1] + node * a.out_stride[2] + c) = w;
  if (a.cache_out && len + node < a.capacity)
    *reinterpret_cast<uint32_t*>((T*)a.cache_out + b * a.cache_out_stride[0] + h * a.cache_out_stride[1] +
                                 (int64_t)(len + node) * a.cache_out_stride[2] + c) = w;
}
// Eight features at once, where the outputs allow 16-byte stores.
template <typename T>
__device__ __forceinline__ void write_row8(const PolyTreePass& a, int b, int h, int node, int len, int c, const float (&x)[8]) {
  const uint4 w = make_uint4(ms::pk2<T>(x[0], x[1]), ms::pk2<T>(x[2], x[3]), ms::pk2<T>(x[4], x[5]), ms::pk2<T>(x[6], x[7]));
  if (a.out)
    *reinterpret_cast<uint4*>((T*)a.out + b * a.out_stride[0] + h * a.out_stride[1] + node * a.out_stride[2] + c) = w;
  if (a.cache_out && len + node < a.capacity)
    *reinterpret_cast<uint4*>((T*)a.cache_out + b * a.cache_out_stride[0] + h * a.cache_out_stride[1] +
                              (int64_t)(len + node) * a.cache_out_stride[2] + c) = w;
}
__device__ __forceinline__ void write_lse(const PolyTreePass& a, int b, int h, int node, int len, float v) {
  if (a.lse) a.lse[b * a.lse_stride[0] + h * a.lse_stride[1] + node] = v;
  if (a.cache_lse && len + node < a.capacity)
    a.cache_lse[b * a.cache_lse_stride[0] + h * a.cache_lse_stride[1] + len + node] = v;
}

// How a pass is cut over CTAs, and where its records go.
struct TreeGeom {
  int splits, row_blocks;
  bool tcgen05;  // the kernel of tree_tc100.cu
  bool cluster;  // tree_kernel: the splits are a cluster's CTAs and join through its shared memory
  float* part;   // records acc[D], m, l, 2 unused: [group][row of the group][split]
};
// floats of a record (16-byte aligned: a thread writes its row's in float4)
template <int D>
constexpr int kRecord = D + 4;

}  // namespace treec

int tree_tc_row_blocks(const PolyTreePass& a);
int launch_tree_tc(const PolyTreePass& a, const treec::TreeGeom& geo, cudaStream_t s, bool dependent);
}  // namespace poly
