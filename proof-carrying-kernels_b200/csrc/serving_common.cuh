// What the serving operators (cache append and attention, adapters, logits) share: element types
// of their inputs, the device status bit of a bad index, and their error reports.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

#include "pck_b200.h"
#include "pck_common.cuh"

namespace pck {

// Device status: an index read from device memory (page, slot, adapter) was out of range; the
// kernel left the access out.
constexpr unsigned kDevIndex = 2u;

int report_error(int code, const char* message);

inline int report_cuda(const char* what, cudaError_t err) {
  char msg[160];
  snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(err));
  return report_error(PCK_ERR_CUDA, msg);
}

// Row strides of an input: rows of their own, or one row for all.
inline bool rows_apart(int64_t stride, int64_t width) { return stride >= width || stride == 0; }

inline bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

}  // namespace pck
