// cusort_float.cuh -- reading and writing 32- and 16-bit floating-point rows
// as 32-bit values, for the routing kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cusort_b200.h"

namespace cusort_b200 {
namespace dev {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// N elements moved by one load or store.
template <typename T, int N> struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

}  // namespace dev

// Calls f with a value of the element type; false for an unknown type.
template <typename F>
bool with_float_type(int type, F&& f) {
  switch (type) {
    case CUSORT_FLOAT_F32: f(float{}); return true;
    case CUSORT_FLOAT_F16: f(__half{}); return true;
    case CUSORT_FLOAT_BF16: f(__nv_bfloat16{}); return true;
    default: return false;
  }
}

inline int float_type_bytes(int type) {
  return type == CUSORT_FLOAT_F32 ? 4 : type == CUSORT_FLOAT_F16 || type == CUSORT_FLOAT_BF16 ? 2 : 0;
}

}  // namespace cusort_b200
