// decode_common.cuh -- element types and cache addressing shared by the
// token-generation kernels (kv_append.cu, paged_attention.cu,
// logits_process.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "ct_internal.h"

namespace ct {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Calls f with a value of the C++ type that a CT_DTYPE_* code names.
template <class F>
inline int with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case CT_DTYPE_F32: return f(float{});
    case CT_DTYPE_BF16: return f(__nv_bfloat16{});
    case CT_DTYPE_F16: return f(__half{});
    default: return CT_ERR_INVALID_ARGUMENT;
  }
}

// Raises a kernel's limit of dynamic shared memory, once a device.
template <auto KERNEL>
inline int allow_shared(int bytes, const DeviceInfo& dev) {
  static std::atomic<bool> done[64];
  if (dev.device < 64 && done[dev.device].load(std::memory_order_acquire)) return CT_OK;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return CT_ERR_CUDA;
  if (dev.device < 64) done[dev.device].store(true, std::memory_order_release);
  return CT_OK;
}

inline int dtype_bytes(int dtype) { return dtype == CT_DTYPE_F32 ? 4 : 2; }

}  // namespace ct
