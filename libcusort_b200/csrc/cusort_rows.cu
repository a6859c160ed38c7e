// cusort_rows.cu -- token rows to their experts' segments and back: dispatch
// copies every token's row to the rows of its pairs, combine adds the pairs'
// rows up with their weights, and the gradient of combine.  (The gradient of
// dispatch is combine without weights.)
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"
#include "cusort_float.cuh"

namespace {

using namespace cusort_b200;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxChosen = 32;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(kAll, x, d);
  return x;
}

struct DispatchArgs {
  const void* x;
  int64_t stride;  // vectors between rows
  const int32_t *sources, *positions;
  void* rows;
  int64_t tokens, capacity, vectors, chunks;  // vectors to a row, chunks of 32 * U of them
  int k;
};

// One warp per (token, chunk of its row): the chunk is read once and written k
// times.  The warps after those clear the rows that hold no pair, 32 each.
template <typename V, int U>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(DispatchArgs a) {
  const int lane = threadIdx.x & 31;
  int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const V* x = static_cast<const V*>(a.x);
  V* rows = static_cast<V*>(a.rows);
  if (w < a.tokens * a.chunks) {
    const int64_t t = w / a.chunks, first = (w - t * a.chunks) * (32 * U) + lane;
    const int at = lane < a.k ? a.positions[t * a.k + lane] : -1;
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * 32 < a.vectors) v[u] = x[t * a.stride + first + u * 32];
    for (int j = 0; j < a.k; ++j) {
      const int64_t r = __shfl_sync(kAll, at, j);
      if (r < 0 || r >= a.capacity) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + u * 32 < a.vectors) rows[r * a.vectors + first + u * 32] = v[u];
    }
    return;
  }
  const int64_t r0 = (w - a.tokens * a.chunks) * 32;
  if (r0 >= a.capacity) return;
  uint32_t empty = __ballot_sync(kAll, r0 + lane < a.capacity && a.sources[r0 + lane] < 0);
  const V zero{};
  for (; empty; empty &= empty - 1) {
    const int64_t r = r0 + __ffs(empty) - 1;
    for (int64_t i = lane; i < a.vectors; i += 32) rows[r * a.vectors + i] = zero;
  }
}

struct CombineArgs {
  const void* rows;
  const float* weights;  // null: ones
  const int32_t* positions;
  const void* residual;  // null: none
  int64_t residual_stride;  // elements between rows
  void* out;
  int64_t tokens, capacity, hidden, chunks;
  int k;
};

// One warp per (token, chunk of its row): sums in 32 bits, rounded once.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) combine_kernel(CombineArgs a) {
  using P = dev::Pack<T, N>;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= a.tokens * a.chunks) return;
  const int64_t t = w / a.chunks, e = ((w - t * a.chunks) * 32 + lane) * N;
  const int at = lane < a.k ? a.positions[t * a.k + lane] : -1;
  const float wt = a.weights == nullptr ? 1.f : lane < a.k ? a.weights[t * a.k + lane] : 0.f;
  const T* rows = static_cast<const T*>(a.rows);
  float sum[N];
#pragma unroll
  for (int n = 0; n < N; ++n) sum[n] = 0.f;
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) {
    const int64_t r = __shfl_sync(kAll, at, j);
    const float f = __shfl_sync(kAll, wt, j);
    if (r >= 0 && r < a.capacity && e < a.hidden) {
      const P v = *reinterpret_cast<const P*>(rows + r * a.hidden + e);
#pragma unroll
      for (int n = 0; n < N; ++n) sum[n] += f * dev::to_float(v.v[n]);
    }
  }
  if (e >= a.hidden) return;
  if (a.residual != nullptr) {
    const P v = *reinterpret_cast<const P*>(static_cast<const T*>(a.residual) + t * a.residual_stride + e);
#pragma unroll
    for (int n = 0; n < N; ++n) sum[n] += dev::to_float(v.v[n]);
  }
  P o;
#pragma unroll
  for (int n = 0; n < N; ++n) o.v[n] = dev::from_float<T>(sum[n]);
  *reinterpret_cast<P*>(static_cast<T*>(a.out) + t * a.hidden + e) = o;
}

struct CombineBackwardArgs {
  const void* grad_out;
  int64_t stride;
  const void* rows;
  const float* weights;
  const int32_t *sources, *positions;
  void* grad_rows;
  float* grad_weights;
  int64_t pairs, capacity, hidden;
  int k;
};

// One warp per pair: its row's gradient, and its weight's as a dot product.
// The warps after those clear the rows that hold no pair, 32 each.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) combine_backward_kernel(CombineBackwardArgs a) {
  using P = dev::Pack<T, N>;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  T* grad_rows = static_cast<T*>(a.grad_rows);
  if (w < a.pairs) {
    const int64_t r = a.positions[w];
    float dot = 0.f;
    if (r >= 0 && r < a.capacity) {
      const T* g = static_cast<const T*>(a.grad_out) + (w / a.k) * a.stride;
      const T* y = static_cast<const T*>(a.rows) + r * a.hidden;
      T* out = grad_rows + r * a.hidden;
      const float f = a.weights[w];
#pragma unroll 4
      for (int64_t e = lane * N; e < a.hidden; e += 32 * N) {
        const P gv = *reinterpret_cast<const P*>(g + e), yv = *reinterpret_cast<const P*>(y + e);
        P o;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float gf = dev::to_float(gv.v[n]);
          dot += gf * dev::to_float(yv.v[n]);
          o.v[n] = dev::from_float<T>(f * gf);
        }
        *reinterpret_cast<P*>(out + e) = o;
      }
    }
    dot = warp_sum(dot);
    if (lane == 0) a.grad_weights[w] = dot;
    return;
  }
  const int64_t r0 = (w - a.pairs) * 32;
  if (r0 >= a.capacity) return;
  uint32_t empty = __ballot_sync(kAll, r0 + lane < a.capacity && a.sources[r0 + lane] < 0);
  P zero;
#pragma unroll
  for (int n = 0; n < N; ++n) zero.v[n] = dev::from_float<T>(0.f);
  for (; empty; empty &= empty - 1) {
    const int64_t r = r0 + __ffs(empty) - 1;
    for (int64_t e = lane * N; e < a.hidden; e += 32 * N) *reinterpret_cast<P*>(grad_rows + r * a.hidden + e) = zero;
  }
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool bad_shape(int64_t tokens, int k, int64_t capacity) {
  return tokens < 0 || k < 1 || k > kMaxChosen || capacity < 0 || tokens > INT32_MAX / k || capacity > INT32_MAX;
}

template <typename V, int U>
cudaError_t dispatch(DispatchArgs a, size_t row_bytes, int64_t stride_bytes, cudaStream_t stream) {
  a.vectors = row_bytes / sizeof(V);
  a.stride = stride_bytes / (int64_t)sizeof(V);
  a.chunks = div_up(a.vectors, 32 * U);
  const int64_t grid = div_up(a.tokens * a.chunks + div_up(a.capacity, 32), kWarps);
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  dispatch_kernel<V, U><<<(int)grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

extern "C" cudaError_t cusort_dispatch_rows(const void* d_x, int64_t row_stride_bytes, size_t row_bytes,
                                            const int32_t* d_sources, const int32_t* d_positions, void* d_rows,
                                            int64_t num_tokens, int k, int64_t capacity, cudaStream_t stream) {
  if (bad_shape(num_tokens, k, capacity) || row_stride_bytes < 0 || row_bytes > (size_t)INT32_MAX)
    return cudaErrorInvalidValue;
  if (capacity == 0 || row_bytes == 0) return cudaSuccess;
  if (d_sources == nullptr || d_rows == nullptr || (num_tokens > 0 && (d_x == nullptr || d_positions == nullptr)))
    return cudaErrorInvalidValue;
  const DispatchArgs a{d_x, 0, d_sources, d_positions, d_rows, num_tokens, capacity, 0, 0, k};
  const uint64_t al = reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_rows) | row_bytes |
                      (uint64_t)row_stride_bytes;
  if ((al & 15) == 0) return dispatch<uint4, 4>(a, row_bytes, row_stride_bytes, stream);
  if ((al & 7) == 0) return dispatch<uint2, 4>(a, row_bytes, row_stride_bytes, stream);
  if ((al & 3) == 0) return dispatch<uint32_t, 4>(a, row_bytes, row_stride_bytes, stream);
  if ((al & 1) == 0) return dispatch<uint16_t, 4>(a, row_bytes, row_stride_bytes, stream);
  return dispatch<uint8_t, 4>(a, row_bytes, row_stride_bytes, stream);
}

extern "C" cudaError_t cusort_combine_rows(cusort_float_type type, const void* d_rows, const float* d_weights,
                                           const int32_t* d_positions, const void* d_residual,
                                           int64_t residual_stride, void* d_out, int64_t num_tokens, int k,
                                           int64_t capacity, int64_t hidden, cudaStream_t stream) {
  const int size = float_type_bytes(type);
  if (size == 0 || bad_shape(num_tokens, k, capacity) || hidden < 0 || hidden > INT32_MAX ||
      (d_residual != nullptr && residual_stride < 0))
    return cudaErrorInvalidValue;
  if (num_tokens == 0 || hidden == 0) return cudaSuccess;
  if ((capacity > 0 && d_rows == nullptr) || d_positions == nullptr || d_out == nullptr) return cudaErrorInvalidValue;
  CombineArgs a{d_rows, d_weights, d_positions, d_residual, residual_stride, d_out, num_tokens, capacity, hidden, 0, k};
  const uint64_t al = reinterpret_cast<uintptr_t>(d_rows) | reinterpret_cast<uintptr_t>(d_residual) |
                      reinterpret_cast<uintptr_t>(d_out) | (uint64_t)(hidden * size) |
                      (d_residual != nullptr ? (uint64_t)(residual_stride * size) : 0);
  cudaError_t err = cudaSuccess;
  with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    constexpr int kWide = 16 / sizeof(T);
    a.chunks = div_up(hidden, 32 * ((al & 15) == 0 ? kWide : 1));
    const int64_t grid = div_up(num_tokens * a.chunks, kWarps);
    if (grid > INT32_MAX) { err = cudaErrorInvalidValue; return; }
    if ((al & 15) == 0) combine_kernel<T, kWide><<<(int)grid, kThreads, 0, stream>>>(a);
    else combine_kernel<T, 1><<<(int)grid, kThreads, 0, stream>>>(a);
    err = cudaGetLastError();
  });
  return err;
}

extern "C" cudaError_t cusort_combine_rows_backward(cusort_float_type type, const void* d_grad_out,
                                                    int64_t grad_stride, const void* d_rows, const float* d_weights,
                                                    const int32_t* d_sources, const int32_t* d_positions,
                                                    void* d_grad_rows, float* d_grad_weights, int64_t num_tokens,
                                                    int k, int64_t capacity, int64_t hidden, cudaStream_t stream) {
  const int size = float_type_bytes(type);
  if (size == 0 || bad_shape(num_tokens, k, capacity) || hidden < 0 || hidden > INT32_MAX || grad_stride < 0)
    return cudaErrorInvalidValue;
  if ((num_tokens > 0 && (d_grad_weights == nullptr || d_positions == nullptr || d_weights == nullptr)) ||
      (num_tokens > 0 && hidden > 0 && d_grad_out == nullptr) ||
      (capacity > 0 && (d_sources == nullptr || (hidden > 0 && (d_rows == nullptr || d_grad_rows == nullptr)))))
    return cudaErrorInvalidValue;
  const int64_t pairs = num_tokens * k, grid = div_up(pairs + div_up(capacity, 32), kWarps);
  if (grid == 0) return cudaSuccess;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  const CombineBackwardArgs a{d_grad_out, grad_stride, d_rows, d_weights, d_sources, d_positions, d_grad_rows,
                              d_grad_weights, pairs, capacity, hidden, k};
  const uint64_t al = reinterpret_cast<uintptr_t>(d_grad_out) | reinterpret_cast<uintptr_t>(d_rows) |
                      reinterpret_cast<uintptr_t>(d_grad_rows) | (uint64_t)(hidden * size) |
                      (uint64_t)(grad_stride * size);
  cudaError_t err = cudaSuccess;
  with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    if ((al & 15) == 0) combine_backward_kernel<T, 16 / sizeof(T)><<<(int)grid, kThreads, 0, stream>>>(a);
    else combine_backward_kernel<T, 1><<<(int)grid, kThreads, 0, stream>>>(a);
    err = cudaGetLastError();
  });
  return err;
}
