// cusort_route.cu -- routing of tokens to experts: scores, a bias for
// balance, groups, the k best, their weights; and the gradient of the logits.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"
#include "cusort_float.cuh"

namespace {

using namespace cusort_b200;

constexpr int kMaxExperts = 1024;
constexpr int kMaxChosen = 32;  // one lane per chosen expert
constexpr int kMaxGroups = 32;  // one lane per group
constexpr int kWarps = 4;       // tokens per CTA
constexpr uint32_t kAll = 0xffffffffu;

struct RouteArgs {
  const void* logits;
  int64_t stride;  // elements between rows
  const float* bias;
  float* weights;
  int32_t* experts;
  int64_t tokens;
  int num_experts, k, groups, groups_kept, per_group;
  bool softmax, renormalize, top2;
  float scale;
};

struct RouteBackwardArgs {
  const float* grad_weights;
  const void* logits;
  int64_t stride;
  const float* bias;
  const int32_t* experts;
  void* grad_logits;
  int64_t tokens;
  int num_experts, k;
  bool softmax, renormalize;
  float scale;
};

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// Unsigned order of the result = order of x; 0 is below every float's.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(kAll, x, d));
  return x;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(kAll, x, d);
  return x;
}

// exp(x - top), 1 at the top itself (an infinite one too).
__device__ __forceinline__ float exp_below(float x, float top) { return x == top ? 1.f : expf(x - top); }

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// A logit as the router sees it: -0 is +0; NaN, -inf and whatever the bias
// takes out is -inf.
template <typename T>
__device__ __forceinline__ float load_logit(const T* row, const float* bias, int e) {
  const float x = dev::to_float(row[e]) + 0.f;
  return x > neg_inf() && (bias == nullptr || bias[e] > neg_inf()) ? x : neg_inf();
}

// One warp per token; lane l holds experts l, l + 32, ...
template <typename T, int V>
__global__ void __launch_bounds__(32 * kWarps) route_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;

  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    x[i] = e < a.num_experts ? load_logit(row, a.bias, e) : neg_inf();
  }
  const bool grouped = a.groups_kept < a.groups;
  const bool need_total = a.softmax && (a.bias != nullptr || !a.renormalize);
  const bool need_score = a.bias != nullptr || (grouped && a.top2);
  float top = neg_inf(), total = 0.f;
  float s[V];
  if (a.softmax && (need_total || need_score)) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
    top = warp_max(top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = x[i] > neg_inf() ? exp_below(x[i], top) : 0.f;
      total += s[i];
    }
    total = warp_sum(total);
  } else if (need_score) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = x[i] > neg_inf() ? sigmoid(x[i]) : 0.f;
  }
  // What the experts are ordered by: the logit (both scores grow with it), or
  // the score plus the bias.
  float c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = x[i];
    if (a.bias != nullptr && x[i] > neg_inf()) c[i] = (a.softmax ? s[i] / total : s[i]) + a.bias[i * 32 + lane];
  }
  uint32_t kept = kAll;
  if (grouped) {
    float mine = neg_inf();  // lane g: group g's value
    for (int g = 0; g < a.groups; ++g) {
      float b1 = neg_inf(), b2 = neg_inf();
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if ((i * 32 + lane) / a.per_group == g && x[i] > neg_inf()) {
          const float v = a.top2 && a.bias == nullptr ? s[i] : c[i];
          b2 = fmaxf(b2, fminf(b1, v));
          b1 = fmaxf(b1, v);
        }
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        const float o1 = __shfl_xor_sync(kAll, b1, d), o2 = __shfl_xor_sync(kAll, b2, d);
        b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
        b1 = fmaxf(b1, o1);
      }
      const float v = a.top2 && b2 > neg_inf() ? b1 + b2 : b1;
      if (lane == g) mine = v;
    }
    int ahead = 0;
    for (int g = 0; g < a.groups; ++g) {
      const float v = __shfl_sync(kAll, mine, g);
      ahead += v > mine || (v == mine && g < lane);
    }
    kept = __ballot_sync(kAll, lane < a.groups && ahead < a.groups_kept);
  }
  uint32_t key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    const bool in = x[i] > neg_inf() && (!grouped || (kept >> (e / a.per_group) & 1));
    key[i] = in ? order_key(c[i]) : 0u;
  }
  // k rounds: the largest key, the lowest expert among equals.  Lane j keeps
  // the j-th.
  int chosen = -1;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (key[i] > best) best = key[i], at = i;
    const uint32_t most = __reduce_max_sync(kAll, best);
    if (most == 0) break;
    const uint32_t e = __reduce_min_sync(kAll, best == most ? (uint32_t)(at * 32 + lane) : kAll);
    if (lane == j) chosen = (int)e;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if ((uint32_t)(i * 32 + lane) == e) key[i] = 0;
  }
  const bool has = chosen >= 0;
  const float xc = has ? load_logit(row, (const float*)nullptr, chosen) : neg_inf();
  float w;
  if (a.softmax && a.renormalize) {
    const float m = warp_max(xc);
    w = has ? exp_below(xc, m) : 0.f;
  } else {
    w = has ? (a.softmax ? exp_below(xc, top) / total : sigmoid(xc)) : 0.f;
  }
  if (a.renormalize) {
    const float sum = warp_sum(w);
    w = sum > 0.f ? w / sum : 0.f;
  }
  if (lane < a.k) {
    a.experts[t * a.k + lane] = chosen;
    a.weights[t * a.k + lane] = w * a.scale;
  }
}

// One warp per token; the row of the gradient is put together in shared
// memory.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kWarps) route_backward_kernel(RouteBackwardArgs a) {
  __shared__ float s_row[kWarps][32 * V];
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  T* out = static_cast<T*>(a.grad_logits) + t * a.num_experts;
  float* buf = s_row[threadIdx.x >> 5];

  const int id = lane < a.k ? a.experts[t * a.k + lane] : -1;
  float xc = neg_inf();
  if (id >= 0 && id < a.num_experts) xc = load_logit(row, a.bias, id);
  const bool has = xc > neg_inf();
  const float g = has ? a.grad_weights[t * a.k + lane] : 0.f;

  const bool dense = a.softmax && !a.renormalize;
  float x[V], top = neg_inf(), total = 0.f;
  if (dense) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * 32 + lane;
      x[i] = e < a.num_experts ? load_logit(row, a.bias, e) : neg_inf();
      top = fmaxf(top, x[i]);
    }
    top = warp_max(top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = x[i] > neg_inf() ? exp_below(x[i], top) : 0.f;
      total += x[i];
    }
    total = warp_sum(total);
  }
  float at;         // the chosen experts' own part
  float used = 0.f; // sum over the chosen of g w (w without the scale)
  if (a.softmax) {
    float p;
    if (a.renormalize) {
      const float m = warp_max(xc);
      p = has ? exp_below(xc, m) : 0.f;
      const float sum = warp_sum(p);
      p = sum > 0.f ? p / sum : 0.f;
    } else {
      p = has ? exp_below(xc, top) / total : 0.f;
    }
    used = warp_sum(g * p);
    at = a.scale * p * (a.renormalize ? g - used : g);
  } else {
    const float e = expf(-fabsf(xc));
    const float slope = has ? e / ((1.f + e) * (1.f + e)) : 0.f;  // s (1 - s), without the difference
    at = g;
    if (a.renormalize) {
      const float s = has ? sigmoid(xc) : 0.f;
      const float sum = warp_sum(s);
      used = sum > 0.f ? warp_sum(g * (s / sum)) : 0.f;
      at = sum > 0.f ? (g - used) / sum : 0.f;
    }
    at *= a.scale * slope;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    buf[e] = dense && total > 0.f ? -(a.scale * used) * (x[i] / total) : 0.f;
  }
  __syncwarp();
  if (has) atomicAdd(&buf[id], at);  // ids of one token are distinct: no two lanes meet
  __syncwarp();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    if (e < a.num_experts) out[e] = dev::from_float<T>(buf[e]);
  }
}

template <template <typename, int> class K, typename Args>
cudaError_t launch(int type, int num_experts, int64_t tokens, const Args& a, cudaStream_t stream) {
  const int64_t grid = (tokens + kWarps - 1) / kWarps;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  const bool known = with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    const int v = (num_experts + 31) / 32;
    if (v <= 1) K<T, 1>::run((int)grid, a, stream);
    else if (v <= 2) K<T, 2>::run((int)grid, a, stream);
    else if (v <= 4) K<T, 4>::run((int)grid, a, stream);
    else if (v <= 8) K<T, 8>::run((int)grid, a, stream);
    else if (v <= 16) K<T, 16>::run((int)grid, a, stream);
    else K<T, 32>::run((int)grid, a, stream);
  });
  return known ? cudaGetLastError() : cudaErrorInvalidValue;
}

template <typename T, int V> struct Forward {
  static void run(int grid, const RouteArgs& a, cudaStream_t s) { route_kernel<T, V><<<grid, 32 * kWarps, 0, s>>>(a); }
};
template <typename T, int V> struct Backward {
  static void run(int grid, const RouteBackwardArgs& a, cudaStream_t s) {
    route_backward_kernel<T, V><<<grid, 32 * kWarps, 0, s>>>(a);
  }
};

bool bad_shape(int type, int64_t stride, int64_t tokens, int num_experts, int k, int score) {
  return float_type_bytes(type) == 0 || tokens < 0 || num_experts < 1 || num_experts > kMaxExperts || k < 1 ||
         k > std::min(kMaxChosen, num_experts) || stride < 0 ||
         (score != CUSORT_SCORE_SOFTMAX && score != CUSORT_SCORE_SIGMOID);
}

}  // namespace

extern "C" cudaError_t cusort_route(cusort_float_type type, const void* d_logits, int64_t row_stride,
                                    const float* d_bias, float* d_weights, int32_t* d_experts, int64_t num_tokens,
                                    int num_experts, int k, int groups, int groups_kept, cusort_score score,
                                    cusort_group_score group_score, int renormalize, float scale,
                                    cudaStream_t stream) {
  if (bad_shape(type, row_stride, num_tokens, num_experts, k, score)) return cudaErrorInvalidValue;
  if (groups < 1 || groups > kMaxGroups || num_experts % groups != 0 || groups_kept < 1 || groups_kept > groups ||
      k > groups_kept * (num_experts / groups))
    return cudaErrorInvalidValue;
  if (group_score != CUSORT_GROUP_MAX && group_score != CUSORT_GROUP_TOP2) return cudaErrorInvalidValue;
  if (num_tokens == 0) return cudaSuccess;
  if (d_logits == nullptr || d_weights == nullptr || d_experts == nullptr) return cudaErrorInvalidValue;
  const RouteArgs a{d_logits, row_stride, d_bias, d_weights, d_experts, num_tokens, num_experts, k, groups,
                    groups_kept, num_experts / groups, score == CUSORT_SCORE_SOFTMAX, renormalize != 0,
                    group_score == CUSORT_GROUP_TOP2, scale};
  return launch<Forward>(type, num_experts, num_tokens, a, stream);
}

extern "C" cudaError_t cusort_route_backward(cusort_float_type type, const float* d_grad_weights,
                                             const void* d_logits, int64_t row_stride, const float* d_bias,
                                             const int32_t* d_experts, void* d_grad_logits, int64_t num_tokens,
                                             int num_experts, int k, cusort_score score, int renormalize,
                                             float scale, cudaStream_t stream) {
  if (bad_shape(type, row_stride, num_tokens, num_experts, k, score)) return cudaErrorInvalidValue;
  if (num_tokens == 0) return cudaSuccess;
  if (d_grad_weights == nullptr || d_logits == nullptr || d_experts == nullptr || d_grad_logits == nullptr)
    return cudaErrorInvalidValue;
  const RouteBackwardArgs a{d_grad_weights, d_logits, row_stride, d_bias, d_experts, d_grad_logits, num_tokens,
                            num_experts, k, score == CUSORT_SCORE_SOFTMAX, renormalize != 0, scale};
  return launch<Backward>(type, num_experts, num_tokens, a, stream);
}
