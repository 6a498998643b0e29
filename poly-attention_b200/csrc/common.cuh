// Shared helpers for the poly-attention kernels (sm_100a).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cfloat>
#include <string>

#include "poly_attention.h"

namespace poly {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A key whose additive bias is at or below this is "dead": the reference adds
// a -finfo.max log-sum-exp there, which no finite score can lift back.
constexpr float kDeadBias = -FLT_MAX * 0.5f;

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Programmatic dependence between consecutive kernels: let the next one start, wait for the previous one.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A kernel that shares nothing with its predecessor may start early without waiting; held as a
// local of the kernel, this still makes it end after that one, so that what follows it in the
// stream follows both.
template <bool ON>
struct EndAfterPrevious {
  __device__ __forceinline__ ~EndAfterPrevious() {
    if (ON) pdl_wait();
  }
};

// Thread-local error message for poly_last_error().
void set_error(const std::string& msg);

// Counts kernel launches made by this library (poly_launch_count()).
void note_launch(int n = 1);

// Launch attribute of a programmatic dependent.
inline cudaLaunchAttribute dependent_launch() {
  cudaLaunchAttribute a;
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

inline int cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return POLY_OK;
  set_error(std::string(what) + ": " + cudaGetErrorString(e));
  return POLY_ECUDA;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device. The setting is the device's,
// so it is made once for each; `done` is the kernel's mask of devices that have it.
inline int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done, const char* what) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;   // a device past 64 is set every time
  if (e == cudaSuccess && !(done.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  }
  return cuda_status(e, what);
}

// Launchers implemented in the individual .cu files.
int launch_pass_fwd_simt(const PolyPassArgs& a, cudaStream_t s);
int launch_pass_bwd_simt(const PolyPassBwdArgs& a, cudaStream_t s);
int launch_lse_merge(const PolyMergeArgs& a, cudaStream_t s);

bool pass_fwd_tc_eligible(const PolyPassArgs& a);
int launch_pass_fwd_tc(const PolyPassArgs& a, cudaStream_t s);
size_t pass_fwd_tc_workspace(const PolyPassArgs& a);

bool pass_bwd_tc_eligible(const PolyPassBwdArgs& a);
int launch_pass_bwd_tc(const PolyPassBwdArgs& a, cudaStream_t s);
size_t pass_bwd_tc_workspace(const PolyPassBwdArgs& a);

int read_device_error_fwd(int* out, bool reset);
int read_device_error_bwd(int* out, bool reset);
int read_device_error_fwd2(int* out, bool reset);
int read_device_error_dec(int* out, bool reset);
int read_device_error_bwd128(int* out, bool reset);
int read_device_error_tree(int* out, bool reset);
int read_device_error_tree_tc(int* out, bool reset);
size_t pass_bwd_tc128_workspace(const PolyPassBwdArgs& a);
int launch_pass_bwd_tc128(const PolyPassBwdArgs& a, cudaStream_t s);
int selftest_wait_timeout(uint64_t limit_ns, int* result, cudaStream_t s);
bool pass_fwd_tc2_eligible(const PolyPassArgs& a);
int launch_pass_fwd_tc2(const PolyPassArgs& a, cudaStream_t s);

bool pass_f32_eligible(const PolyPassArgs& a);
int launch_pass_f32(const PolyPassArgs& a, cudaStream_t s);
bool pass_small_eligible(const PolyPassArgs& a);
int launch_pass_small(const PolyPassArgs& a, cudaStream_t s);
bool pass_decode_eligible(const PolyPassArgs& a);
int launch_pass_decode(const PolyPassArgs& a, cudaStream_t s, bool dependent = false);
size_t pass_decode_workspace(const PolyPassArgs& a);
int copy_rows(const PolyRowCopy* copies, int n, cudaStream_t s);
int head_rmsnorm(const PolyHeadNorm* norms, int n, cudaStream_t s);
int rotary(const PolyRotaryArgs* args, cudaStream_t s);

// Outputs whose rows outside every packed sequence are written as zeros (packed.cuh).
struct ZeroRest {
  struct {
    char* p;
    int heads, row_bytes;
    int64_t head_stride, row_stride;   // bytes
    bool wide;                          // 16-byte stores
  } t[5];
  int n;
};

// Sequences packed end to end (packed.cuh): device offsets, their number, rows in all.
struct PackedSeqs {
  const int* cu;
  int seqs, total, max_len;
  void* out_lo;         // rounding residue of out (forward: written, backward: read) | NULL
  // backward of values that are a product: the factors and the second gradient | NULL
  const void* v_left; int64_t v_left_stride[2];
  const void* v_right; int64_t v_right_stride[2];
  void* dv_right; int64_t dv_right_stride[2];
  ZeroRest zero;        // the work of kZeroCtas extra CTAs of the pass's first kernel (none if zero.n is 0)
};
constexpr int kZeroCtas = 32;
inline unsigned zero_ctas(const PackedSeqs& q) { return q.zero.n ? kZeroCtas : 0; }
int launch_packed_fwd_simt(const PolyPassArgs& a, const PackedSeqs& q, cudaStream_t s);
int launch_packed_bwd_simt(const PolyPassBwdArgs& a, const PackedSeqs& q, cudaStream_t s);
size_t packed_bwd_simt_workspace(const PolyPassBwdArgs& a);
bool packed_fwd_tc_eligible(const PolyPassArgs& a, const void* out_lo);
int launch_packed_fwd_tc(PolyPassArgs a, const PackedSeqs& q, cudaStream_t s);
bool packed_f32_eligible(const PolyPackedArgs& a);
int launch_packed_fwd_f32(PolyPassArgs a, const PackedSeqs& q, cudaStream_t s);
int launch_packed_fwd_small(const PolyPassArgs& a, const PackedSeqs& q, cudaStream_t s);
int launch_packed_bwd_small(const PolyPassBwdArgs& a, const PackedSeqs& q, cudaStream_t s);
bool packed_bwd_tc_eligible(const PolyPackedBwdArgs& a);
int launch_packed_bwd_tc(PolyPassBwdArgs a, const PackedSeqs& q, cudaStream_t s);
int launch_packed_bwd_tc128(const PolyPassBwdArgs& a, const PackedSeqs& q, cudaStream_t s);
size_t packed_bwd_tc_workspace(const PolyPassBwdArgs& a, int seqs);

}  // namespace poly
