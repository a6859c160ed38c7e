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

// N elements as the machine word or words they lie in, so that loads are
// kept whole until their values are used.
template <int BYTES> struct BitsOf;
template <> struct BitsOf<2> { using type = uint16_t; };
template <> struct BitsOf<4> { using type = uint32_t; };
template <> struct BitsOf<8> { using type = uint2; };
template <> struct BitsOf<16> { using type = uint4; };
template <typename T, int N> using Bits = typename BitsOf<sizeof(T) * N>::type;

__device__ __forceinline__ float2 to_float2(uint32_t bits, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&bits));
}
__device__ __forceinline__ float2 to_float2(uint32_t bits, __nv_bfloat16) {
  return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
}
__device__ __forceinline__ uint32_t from_float2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t from_float2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int N>
__device__ __forceinline__ void unpack(Bits<T, N> bits, float (&x)[N]) {
  if constexpr (sizeof(T) * N == 2) {
    x[0] = to_float(*reinterpret_cast<const T*>(&bits));
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&bits);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * N / 4); ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = to_float2(w[i], T{});
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
}

template <typename T, int N>
__device__ __forceinline__ Bits<T, N> pack(const float (&x)[N]) {
  Bits<T, N> bits;
  if constexpr (sizeof(T) * N == 2) {
    *reinterpret_cast<T*>(&bits) = from_float<T>(x[0]);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&bits);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * N / 4); ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(x[i]);
      else w[i] = from_float2(x[2 * i], x[2 * i + 1], T{});
    }
  }
  return bits;
}

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
