// cusort_rows.cu -- token rows to their experts' segments and back: dispatch
// copies every token's row to the rows of its pairs, combine adds the pairs'
// rows up with their weights, and the gradient of combine.  (The gradient of
// dispatch is combine without weights.)
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/cusort_b200.h"
#include "cusort_float.cuh"
#include "cusort_overlap.cuh"

namespace {

using namespace cusort_b200;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kBackwardThreads = 128;  // 256: 187 us where it takes 181 (see combine_backward_kernel)
constexpr int kMaxChosen = 32;
constexpr int kEmptyRows = 8;           // rows that a warp looks at to clear those without a pair
constexpr int64_t kBusyWarps = 148 * 16;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(kAll, x, d);
  return x;
}

// Clears those of the kEmptyRows rows from r0 on that hold no pair.  Few rows
// to a warp: the rows after the last segment lie together, and a warp that
// clears 32 rows of 8 KB alone (as a first form did) is still at it 25 us
// after the others are done.
template <typename V>
__device__ __forceinline__ void clear_empty_rows(V* rows, const int32_t* sources, int64_t r0, int64_t capacity,
                                                 int64_t vectors, int lane) {
  const int64_t r = r0 + lane;
  uint32_t empty = __ballot_sync(kAll, lane < kEmptyRows && r < capacity && sources[r < capacity ? r : 0] < 0);
  const V zero{};
  constexpr int kPer16 = 16 / (int)sizeof(V);
  for (; empty; empty &= empty - 1) {
    // whole 16-byte words between what lies before the first and after the last of them
    V* row = rows + (r0 + __ffs(empty) - 1) * vectors;
    const int64_t before = (16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / sizeof(V), head = min(before, vectors);
    const int64_t words = (vectors - head) / kPer16, rest = vectors - head - words * kPer16;
    uint4* body = reinterpret_cast<uint4*>(row + head);
    if (lane < head) row[lane] = zero;
#pragma unroll 4
    for (int64_t i = lane; i < words; i += 32) body[i] = make_uint4(0, 0, 0, 0);
    if (lane < rest) row[head + words * kPer16 + lane] = zero;
  }
}

struct DispatchArgs {
  const void* x;
  int64_t stride;  // vectors between rows
  const int32_t *sources, *positions;
  void* rows;
  int64_t tokens, capacity, empty_warps, vectors, chunks;  // vectors to a row, chunks of 32 * U of them
  int k;
};

// One warp per (token, chunk of its row): the chunk is read once and written k
// times.  The first warps clear the rows that hold no pair.  Bound by memory;
// taking the output's rows in order instead (each read from its token) reads
// every token k times and came to 69 % of the copy rate where this comes to
// 94 %: 98 us, 6.1 TB/s (8192 tokens, k = 8, rows of 8 KB).
template <typename V, int U>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(DispatchArgs a) {
  dev::wait_for_previous();
  const int lane = threadIdx.x & 31;
  int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const V* x = static_cast<const V*>(a.x);
  V* rows = static_cast<V*>(a.rows);
  if (w < a.empty_warps) {
    clear_empty_rows(rows, a.sources, w * kEmptyRows, a.capacity, a.vectors, lane);
    return;
  }
  w -= a.empty_warps;
  if (w >= a.tokens * a.chunks) return;
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
}

struct CombineArgs {
  const void* rows;
  const float* weights;  // null: ones
  const int32_t* positions;
  const void* residual;     // null: none
  int64_t residual_stride;  // elements between rows
  void* out;
  int64_t tokens, capacity, hidden, chunks;
  int k;
};

// One warp per (token, chunk of its row): sums in 32 bits, rounded once.  The
// rows of K pairs and U vectors of each are in flight at a time: bound by
// memory, and by too few bytes in flight before that (8192 tokens, k = 8, rows
// of 8 KB: K x U = 4 x 1 85 % of the copy rate, 4 x 2 91 %, 4 x 4 97 %: 95 us,
// 6.3 TB/s; 4099 tokens, k = 6, rows of 4 KB 24 us, 74 %).
template <typename T, int N, int U>
__global__ void __launch_bounds__(kThreads) combine_kernel(CombineArgs a) {
  dev::wait_for_previous();
  using B = dev::Bits<T, N>;
  constexpr int K = 4;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= a.tokens * a.chunks) return;
  const int64_t t = w / a.chunks, e = ((w - t * a.chunks) * (32 * U) + lane) * N;
  const int at = lane < a.k ? a.positions[t * a.k + lane] : -1;
  const float wt = a.weights == nullptr ? 1.f : lane < a.k ? a.weights[t * a.k + lane] : 0.f;
  const T* rows = static_cast<const T*>(a.rows) + e;
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) in[u] = e + u * 32 * N < a.hidden;
  float sum[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int n = 0; n < N; ++n) sum[u][n] = 0.f;
  for (int j0 = 0; j0 < a.k; j0 += K) {
    B v[K][U];
    float f[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int64_t r = __shfl_sync(kAll, at, (j0 + j) & 31);  // -1 from k on: K divides 32
      f[j] = __shfl_sync(kAll, wt, (j0 + j) & 31);
      const bool there = r >= 0 && r < a.capacity;
      if (!there) f[j] = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[j][u] = B{};  // zeros where there is nothing: no branch between the loads and their use
        if (there && in[u]) v[j][u] = *reinterpret_cast<const B*>(rows + r * a.hidden + u * 32 * N);
      }
    }
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[N];
        dev::unpack<T, N>(v[j][u], x);
#pragma unroll
        for (int n = 0; n < N; ++n) sum[u][n] += f[j] * x[n];
      }
  }
  if (a.residual != nullptr) {
    const T* residual = static_cast<const T*>(a.residual) + t * a.residual_stride + e;
    B v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = B{};
      if (in[u]) v[u] = *reinterpret_cast<const B*>(residual + u * 32 * N);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
      dev::unpack<T, N>(v[u], x);
#pragma unroll
      for (int n = 0; n < N; ++n) sum[u][n] += x[n];
    }
  }
  T* out = static_cast<T*>(a.out) + t * a.hidden + e;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (in[u]) *reinterpret_cast<B*>(out + u * 32 * N) = dev::pack<T, N>(sum[u]);
}

struct CombineBackwardArgs {
  const void* grad_out;
  int64_t stride;
  const void* rows;
  const float* weights;
  const int32_t *sources, *positions;
  void* grad_rows;
  float* grad_weights;
  int64_t pairs, capacity, empty_warps, hidden;
  int k;
};

// One warp per pair: its row's gradient, and its weight's as a dot product.
// The pairs of a token lie side by side, so that its gradient comes from
// memory once and from the caches k - 1 times.  The first warps clear the rows
// that hold no pair.  Bound by memory: 8192 tokens, k = 8, rows of 8 KB 181 us
// (97 % of the copy rate); 4099 tokens, k = 6, rows of 4 KB 39 us (87 %).
template <typename T, int N, int U>
__global__ void __launch_bounds__(kBackwardThreads) combine_backward_kernel(CombineBackwardArgs a) {
  dev::wait_for_previous();
  using B = dev::Bits<T, N>;
  const int lane = threadIdx.x & 31;
  int64_t w = (int64_t)blockIdx.x * (kBackwardThreads / 32) + (threadIdx.x >> 5);
  T* grad_rows = static_cast<T*>(a.grad_rows);
  if (w < a.empty_warps) {
    clear_empty_rows(reinterpret_cast<B*>(grad_rows), a.sources, w * kEmptyRows, a.capacity, a.hidden / N, lane);
    return;
  }
  w -= a.empty_warps;
  if (w >= a.pairs) return;
  const int64_t r = a.positions[w];
  float dot = 0.f;
  if (r >= 0 && r < a.capacity) {
    const T* g = static_cast<const T*>(a.grad_out) + (w / a.k) * a.stride;
    const T* y = static_cast<const T*>(a.rows) + r * a.hidden;
    T* out = grad_rows + r * a.hidden;
    const float f = a.weights[w];
    for (int64_t e0 = lane * N; e0 < a.hidden; e0 += 32 * N * U) {
      B gv[U], yv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t e = e0 + u * 32 * N;
        yv[u] = gv[u] = B{};
        if (e < a.hidden) {
          yv[u] = *reinterpret_cast<const B*>(y + e);
          gv[u] = *reinterpret_cast<const B*>(g + e);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t e = e0 + u * 32 * N;
        float gx[N], yx[N];
        dev::unpack<T, N>(gv[u], gx);
        dev::unpack<T, N>(yv[u], yx);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          dot += gx[n] * yx[n];
          gx[n] *= f;
        }
        if (e < a.hidden) *reinterpret_cast<B*>(out + e) = dev::pack<T, N>(gx);
      }
    }
  }
  dot = warp_sum(dot);
  if (lane == 0) a.grad_weights[w] = dot;
}

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool bad_shape(int64_t tokens, int k, int64_t capacity) {
  return tokens < 0 || k < 1 || k > kMaxChosen || capacity < 0 || tokens > INT32_MAX / k || capacity > INT32_MAX;
}

// Bytes of the widest vector that every address is a multiple of.
int vector_bytes(uint64_t bits) { return (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1; }

// Vectors to a lane, for 16-byte ones: as few left over at the row's end as
// possible, then as many as possible, but no more than leave kBusyWarps warps
// (few tokens: latency counts, and shorter chunks are done sooner).
int vectors_per_lane(int64_t tokens, int64_t vectors) {
  int best = 1;
  int64_t waste = INT64_MAX;
  for (int u = 4; u >= 1; --u) {
    const int64_t chunks = div_up(vectors, 32 * u);
    if ((u == 1 || tokens * chunks >= kBusyWarps) && chunks * u < waste) waste = chunks * u, best = u;
  }
  return best;
}

template <typename V, int U>
cudaError_t dispatch(DispatchArgs a, size_t row_bytes, int64_t stride_bytes, cudaStream_t stream) {
  a.vectors = row_bytes / sizeof(V);
  a.stride = stride_bytes / (int64_t)sizeof(V);
  a.chunks = div_up(a.vectors, 32 * U);
  a.empty_warps = div_up(a.capacity, kEmptyRows);
  return launch_after_previous(dispatch_kernel<V, U>, div_up(a.empty_warps + a.tokens * a.chunks, kWarps), kThreads, 0,
                               a, stream);
}

template <typename T, int BYTES, int U>
cudaError_t combine(CombineArgs a, cudaStream_t stream) {
  constexpr int N = BYTES / (int)sizeof(T);
  a.chunks = div_up(a.hidden, 32 * N * U);
  return launch_after_previous(combine_kernel<T, N, U>, div_up(a.tokens * a.chunks, kWarps), kThreads, 0, a, stream);
}

template <typename T, int BYTES, int U>
cudaError_t combine_backward(CombineBackwardArgs a, cudaStream_t stream) {
  a.empty_warps = div_up(a.capacity, kEmptyRows);
  const int64_t grid = div_up(a.empty_warps + a.pairs, kBackwardThreads / 32);
  if (grid == 0) return cudaSuccess;
  return launch_after_previous(combine_backward_kernel<T, BYTES / (int)sizeof(T), U>, grid, kBackwardThreads, 0, a,
                               stream);
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
  const DispatchArgs a{d_x, 0, d_sources, d_positions, d_rows, num_tokens, capacity, 0, 0, 0, k};
  switch (vector_bytes(reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_rows) | row_bytes |
                       (uint64_t)row_stride_bytes)) {
    case 16:
      switch (vectors_per_lane(num_tokens, row_bytes / 16)) {
        case 4: return dispatch<uint4, 4>(a, row_bytes, row_stride_bytes, stream);
        case 3: return dispatch<uint4, 3>(a, row_bytes, row_stride_bytes, stream);
        case 2: return dispatch<uint4, 2>(a, row_bytes, row_stride_bytes, stream);
        default: return dispatch<uint4, 1>(a, row_bytes, row_stride_bytes, stream);
      }
    // narrower vectors, more of them in flight
    case 8: return dispatch<uint2, 4>(a, row_bytes, row_stride_bytes, stream);
    case 4: return dispatch<uint32_t, 8>(a, row_bytes, row_stride_bytes, stream);
    case 2: return dispatch<uint16_t, 8>(a, row_bytes, row_stride_bytes, stream);
    default: return dispatch<uint8_t, 8>(a, row_bytes, row_stride_bytes, stream);
  }
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
  const CombineArgs a{d_rows, d_weights, d_positions, d_residual, residual_stride, d_out, num_tokens, capacity, hidden,
                      0, k};
  const int bytes = vector_bytes(reinterpret_cast<uintptr_t>(d_rows) | reinterpret_cast<uintptr_t>(d_residual) |
                                 reinterpret_cast<uintptr_t>(d_out) | (uint64_t)(hidden * size) |
                                 (d_residual != nullptr ? (uint64_t)(residual_stride * size) : 0));
  cudaError_t err = cudaSuccess;
  with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    if (bytes == 16) {
      switch (vectors_per_lane(num_tokens, hidden * size / 16)) {
        case 4: err = combine<T, 16, 4>(a, stream); break;
        case 3: err = combine<T, 16, 3>(a, stream); break;
        case 2: err = combine<T, 16, 2>(a, stream); break;
        default: err = combine<T, 16, 1>(a, stream); break;
      }
    } else if (bytes == 8) {
      err = combine<T, 8, 4>(a, stream);
    } else if (bytes == 4 || sizeof(T) == 4) {
      err = combine<T, 4, 8>(a, stream);
    } else {
      err = combine<T, sizeof(T), 8>(a, stream);
    }
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
  const CombineBackwardArgs a{d_grad_out, grad_stride, d_rows, d_weights, d_sources, d_positions, d_grad_rows,
                              d_grad_weights, num_tokens * k, capacity, 0, hidden, k};
  const int bytes = vector_bytes(reinterpret_cast<uintptr_t>(d_grad_out) | reinterpret_cast<uintptr_t>(d_rows) |
                                 reinterpret_cast<uintptr_t>(d_grad_rows) | (uint64_t)(hidden * size) |
                                 (uint64_t)(grad_stride * size));
  cudaError_t err = cudaSuccess;
  with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    if (bytes == 16) {
      switch (vectors_per_lane(INT32_MAX, hidden * size / 16)) {  // a warp takes the whole row, however few they are
        case 4: err = combine_backward<T, 16, 4>(a, stream); break;
        case 3: err = combine_backward<T, 16, 3>(a, stream); break;
        case 2: err = combine_backward<T, 16, 2>(a, stream); break;
        default: err = combine_backward<T, 16, 1>(a, stream); break;
      }
    }
    else if (bytes == 8) err = combine_backward<T, 8, 4>(a, stream);
    else if (bytes == 4 || sizeof(T) == 4) err = combine_backward<T, 4, 8>(a, stream);
    else err = combine_backward<T, sizeof(T), 8>(a, stream);
  });
  return err;
}
