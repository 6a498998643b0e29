// Warp-level tensor core pieces (mma.sync m16n8k16, ldmatrix, cp.async) of the
// kernels whose tiles are too small for tcgen05: short sequences (small.cu,
// small_bwd.cu) and drafted trees (tree.cu).
#pragma once

#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace poly {
namespace ms {

__device__ __forceinline__ void cp16(uint32_t sa, const void* g, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sa), "l"(g), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a));
}
template <typename T>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pk2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return tc::pack_bf16(lo, hi);
  else return tc::pack_f16(lo, hi);
}

// Four 8-feature blocks of a row as a quad of lanes holds them in accumulators (lane t: features 2t, 2t + 1
// of each) <-> whole blocks (lane t: block t), the form for 16-byte global accesses: 4-byte ones of
// such fragments cost eight times the wavefronts. Its own inverse; every lane of the warp takes part.
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4]) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
  const uint32_t a = __shfl_xor_sync(0xffffffffu, odd ? w[0] : w[1], 1), b = __shfl_xor_sync(0xffffffffu, odd ? w[2] : w[3], 1);
  const uint32_t w0 = odd ? a : w[0], w1 = odd ? w[1] : a, w2 = odd ? b : w[2], w3 = odd ? w[3] : b;
  const uint32_t c = __shfl_xor_sync(0xffffffffu, high ? w0 : w2, 2), d = __shfl_xor_sync(0xffffffffu, high ? w1 : w3, 2);
  w[0] = high ? c : w0;
  w[1] = high ? d : w1;
  w[2] = high ? w2 : c;
  w[3] = high ? w3 : d;
}
__device__ __forceinline__ void quad_load(uint32_t (&w)[4], const void* block, bool live) {
  uint4 x = make_uint4(0u, 0u, 0u, 0u);
  if (live) x = *reinterpret_cast<const uint4*>(block);
  w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
}
__device__ __forceinline__ void quad_store(void* block, uint32_t (&w)[4], bool live) {   // w as in accumulators
  quad_transpose(w);
  if (live) *reinterpret_cast<uint4*>(block) = make_uint4(w[0], w[1], w[2], w[3]);
}

// byte offset of 16-byte chunk ch of row r in a [rows][D] 16-bit tile, chunks XOR-swizzled by row
template <int D>
__device__ __forceinline__ uint32_t soff(int r, int ch) {
  return (uint32_t)(r * (D * 2) + ((ch ^ (r & 7)) << 4));
}

}  // namespace ms
}  // namespace poly
