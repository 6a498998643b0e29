// Finding a row or a tile in a batch of sequences packed end to end.
//
// cu_seqlens[s] is sequence s's first row, cu_seqlens[s + 1] the row behind it.
// The kernels that split every sequence into tiles of B rows number the tiles
// without a prefix sum: sequence s owns the slots floor(cu[s] / B) + s and up to
// (not including) floor(cu[s + 1] / B) + s + 1, which are at least ceil(len / B)
// of them, and total / B + seqs slots cover every sequence. So a CTA finds its
// sequence by one search over cu_seqlens; a slot past its sequence's last tile
// is empty. Offsets are clamped to [0, total]: offsets outside it or running
// backwards select wrong rows, never rows outside the tensors.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace poly {

__device__ __forceinline__ int packed_at(const int* cu, int s, int total) { return min(max(cu[s], 0), total); }

// first row of the sequence that row i belongs to
__device__ __forceinline__ int packed_start(const int* cu, int seqs, int total, int i) {
  int lo = 0, hi = seqs;   // the last s with cu[s] <= i
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (packed_at(cu, mid, total) <= i) lo = mid; else hi = mid;
  }
  return packed_at(cu, lo, total);
}

struct PackedTile {
  int seq, start, len;   // the sequence, its first row and its length
  int tile;              // tile of the sequence
  int slot0;             // the sequence's first slot
};

// The tile of slot `slot` (B rows a tile); false: the slot is empty.
template <int B>
__device__ __forceinline__ bool packed_tile(const int* cu, int seqs, int total, int slot, PackedTile& t) {
  int lo = 0, hi = seqs;   // the last s with cu[s] / B + s <= slot
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (packed_at(cu, mid, total) / B + mid <= slot) lo = mid; else hi = mid;
  }
  t.seq = lo;
  t.start = packed_at(cu, lo, total);
  t.len = packed_at(cu, lo + 1, total) - t.start;
  t.slot0 = t.start / B + lo;
  t.tile = slot - t.slot0;
  return t.tile >= 0 && t.tile * B < t.len;
}

// The same numbering in blocks of 8 rows, for a workspace in which every sequence has rows of its own: the
// first row of a tile's sequence, and the rows in all.
constexpr int kRowBlock = 8;
__device__ __forceinline__ int packed_row0(const PackedTile& t) { return (t.start / kRowBlock + t.seq) * kRowBlock; }
inline int64_t packed_rows(int total, int seqs) { return ((int64_t)(total / kRowBlock) + seqs) * kRowBlock; }

// Rows before the first and behind the last sequence of a pass's outputs, as zeros:
// CTA `part` of kZeroCtas that the pass's first kernel has for it beside its own.
// Usually there are none, and the CTA reads two offsets and leaves.
__device__ __forceinline__ void packed_zero_rest(const PackedSeqs& q, int part) {
  const int lo = packed_at(q.cu, 0, q.total), hi = max(packed_at(q.cu, q.seqs, q.total), lo);
  const int rest = lo + (q.total - hi);
  for (int r = part; r < rest; r += kZeroCtas) {
    const int64_t row = r < lo ? r : hi + (r - lo);
    for (int k = 0; k < q.zero.n; ++k) {
      const auto& t = q.zero.t[k];
      char* base = t.p + row * t.row_stride;
      if (t.wide) {
        const int words = t.row_bytes >> 4;
        for (int i = threadIdx.x; i < t.heads * words; i += blockDim.x)
          *reinterpret_cast<uint4*>(base + (i / words) * t.head_stride + (i % words) * 16) = make_uint4(0u, 0u, 0u, 0u);
      } else {   // rows need no more than their type's alignment
        const int words = t.row_bytes >> 1;
        for (int i = threadIdx.x; i < t.heads * words; i += blockDim.x)
          *reinterpret_cast<uint16_t*>(base + (i / words) * t.head_stride + (i % words) * 2) = 0;
      }
    }
  }
}

// Rows of one head as NaN (0x7fff is one in fp16 and in bf16): a sequence that is
// longer than the caller's bound said.
__device__ __forceinline__ void packed_nan_rows(void* p, int64_t head, int64_t row_stride, int64_t first, int rows, int dim) {
  if (!p) return;
  for (int64_t i = threadIdx.x; i < (int64_t)rows * dim; i += blockDim.x)
    ((uint16_t*)p)[head + (first + i / dim) * row_stride + i % dim] = 0x7fff;
}

// The slots of a launch by descending number of tiles to walk, `order`[slots], by one CTA:
// a launch that starts its longest CTAs first ends even. Empty slots go last. Equal
// ones come in any order (it decides when a CTA runs, not what it computes).
constexpr int kOrderSlots = 8192;   // more slots are left in their own order
template <int B>
__device__ __forceinline__ void packed_order(const PackedSeqs& q, int slots, bool causal, int* order) {
  constexpr int kBins = 512;
  __shared__ int at[kBins];
  auto bin = [&](int s) {
    PackedTile t;
    if (!packed_tile<B>(q.cu, q.seqs, q.total, s, t)) return kBins - 1;
    const int tiles = (t.len + B - 1) / B;
    return kBins - 1 - min(causal ? tiles - t.tile : tiles, kBins - 1);
  };
  for (int i = threadIdx.x; i < kBins; i += blockDim.x) at[i] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += blockDim.x) atomicAdd(&at[bin(s)], 1);
  __syncthreads();
  if (threadIdx.x == 0) {
    int sum = 0;
    for (int i = 0; i < kBins; ++i) {
      const int c = at[i];
      at[i] = sum;
      sum += c;
    }
  }
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += blockDim.x) order[atomicAdd(&at[bin(s)], 1)] = s;
}

}  // namespace poly
