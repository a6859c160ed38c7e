// cusort_route.cu -- routing of tokens to experts: scores, a bias for
// balance, groups, the k best, their weights; and the gradient of the logits.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

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
  int num_experts, k, k_lanes;  // k_lanes: the power of two from k on
  int groups, groups_kept, per_group, group_lanes;  // group_lanes: lanes to a group, 0 where groups end inside a lane
  bool wide;                                        // rows and their addresses are whole vectors
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
  int num_experts, k, k_lanes;
  bool wide;
  bool softmax, renormalize;
  float scale;
};

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// Unsigned order of the result = order of x; 0 is below every float's.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order_key(uint32_t u) {
  return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : 0xffffffffu));
}

// Over the first `lanes` lanes (a power of two) and every block of as many.
__device__ __forceinline__ float max_over(float x, int lanes) {
  for (int d = lanes >> 1; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(kAll, x, d));
  return x;
}
__device__ __forceinline__ float sum_over(float x, int lanes) {
  for (int d = lanes >> 1; d; d >>= 1) x += __shfl_xor_sync(kAll, x, d);
  return x;
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

// A logit as the router sees it: -0 is +0, and NaN is -inf.
template <typename T>
__device__ __forceinline__ float logit(T v) {
  const float x = dev::to_float(v) + 0.f;
  return x > neg_inf() ? x : neg_inf();
}
template <typename T>
__device__ __forceinline__ float logit_at(const T* row, const float* bias, int e) {
  const float x = logit(row[e]);
  return bias == nullptr || bias[e] > neg_inf() ? x : neg_inf();
}

template <typename T, int V> constexpr int vector_length() {
  return V * sizeof(T) <= 16 ? V : 16 / (int)sizeof(T);
}

// The lane's V consecutive logits, from expert lane * V on; -inf beyond the
// last.
template <typename T, int V>
__device__ __forceinline__ void load_logits(float (&x)[V], const T* row, int lane, int num_experts, bool wide) {
  constexpr int N = vector_length<T, V>();
  if (wide) {
#pragma unroll
    for (int c = 0; c < V; c += N) {
      if (lane * V + c < num_experts) {
        const auto p = *reinterpret_cast<const dev::Pack<T, N>*>(row + lane * V + c);
#pragma unroll
        for (int i = 0; i < N; ++i) x[c + i] = logit(p.v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[c + i] = neg_inf();
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = lane * V + i < num_experts ? logit(row[lane * V + i]) : neg_inf();
  }
}

// Which groups stay: lane's mask of its V experts (bit i: expert lane * V + i).
// value: what groups go by, -inf where not available.
template <int V>
__device__ uint32_t kept_experts(const RouteArgs& a, const float (&value)[V], int lane) {
  float mine = neg_inf();  // the value of the group that this lane stands for
  int group = lane;
  if (a.group_lanes != 0) {
    // a group is group_lanes whole lanes: its two best by exchange among them
    float b1 = value[0], b2 = neg_inf();
#pragma unroll
    for (int i = 1; i < V; ++i) {
      b2 = fmaxf(b2, fminf(b1, value[i]));
      b1 = fmaxf(b1, value[i]);
    }
    for (int d = 1; d < a.group_lanes; d <<= 1) {
      const float o1 = __shfl_xor_sync(kAll, b1, d), o2 = __shfl_xor_sync(kAll, b2, d);
      b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
      b1 = fmaxf(b1, o1);
    }
    mine = a.top2 && b2 > neg_inf() ? b1 + b2 : b1;
    group = lane / a.group_lanes;
    int ahead = 0;
    for (int g = 0; g < a.groups; ++g) {
      const float v = __shfl_sync(kAll, mine, g * a.group_lanes);
      ahead += v > mine || (v == mine && g < group);
    }
    return ahead < a.groups_kept ? kAll : 0u;
  }
  // groups of any length: one after the other, lane g keeps group g's
  for (int g = 0; g < a.groups; ++g) {
    float b1 = neg_inf(), b2 = neg_inf();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if ((lane * V + i) / a.per_group == g) {
        b2 = fmaxf(b2, fminf(b1, value[i]));
        b1 = fmaxf(b1, value[i]);
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const float o1 = __shfl_xor_sync(kAll, b1, d), o2 = __shfl_xor_sync(kAll, b2, d);
      b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
      b1 = fmaxf(b1, o1);
    }
    if (lane == g) mine = a.top2 && b2 > neg_inf() ? b1 + b2 : b1;
  }
  int ahead = 0;
  for (int g = 0; g < a.groups; ++g) {
    const float v = __shfl_sync(kAll, mine, g);
    ahead += v > mine || (v == mine && g < lane);
  }
  const uint32_t kept = __ballot_sync(kAll, lane < a.groups && ahead < a.groups_kept);
  uint32_t mask = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (lane * V + i) / a.per_group;
    mask |= (g < 32 ? kept >> g & 1u : 0u) << i;
  }
  return mask;
}

// One warp per token; a lane holds V consecutive experts, so that a lower lane
// means a lower expert and groups are runs of lanes.  k rounds choose the
// largest order key; lane j keeps the j-th.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kWarps) route_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;

  float x[V];
  load_logits<T, V>(x, row, lane, a.num_experts, a.wide);
  const bool biased = a.bias != nullptr, grouped = a.groups_kept < a.groups;
  uint32_t mask = kAll;  // experts of the lane that may be chosen
  float top = neg_inf(), total = 0.f;
  float c[V];  // what experts are ordered by: the logit (both scores grow with it), or the score plus the bias
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = x[i];
  const bool need_total = a.softmax && (biased || !a.renormalize);
  if (need_total || biased || (grouped && a.top2)) {
    float b[V], s[V];
    if (biased) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = lane * V + i;
        b[i] = e < a.num_experts ? a.bias[e] : 0.f;
        if (!(b[i] > neg_inf())) x[i] = neg_inf();
      }
    }
    if (a.softmax) {
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
      top = warp_max(top);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] = x[i] > neg_inf() ? exp_below(x[i], top) : 0.f;
        total += s[i];
      }
      total = warp_sum(total);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = sigmoid(x[i]);  // 0 at -inf
    }
    if (biased) {
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = x[i] > neg_inf() ? (a.softmax ? s[i] / total : s[i]) + b[i] : neg_inf();
    }
    if (grouped && a.top2 && !biased) {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = x[i] > neg_inf() ? s[i] : neg_inf();
      mask = kept_experts<V>(a, s, lane);
    } else if (grouped) {
      mask = kept_experts<V>(a, c, lane);
    }
  } else if (grouped) {
    mask = kept_experts<V>(a, c, lane);
  }

  int chosen = -1;
  float xc = neg_inf();  // the chosen expert's logit
  if (sizeof(T) == 2 && !biased) {
    // a 16-bit logit's order and its expert fit one word, lower experts above higher ones
    uint32_t key[V], mine = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // of the widened value the low 16 bits are zero (bf16), or the low 13 and the exponent's range is short (f16):
      // the narrow value's own bits are ordered
      const uint32_t bits = __float_as_uint(x[i]);
      uint32_t narrow;
      if constexpr (std::is_same_v<T, __nv_bfloat16>) narrow = bits >> 16;
      else narrow = __half_as_ushort(__float2half_rn(x[i]));
      narrow = (narrow ^ (narrow & 0x8000u ? 0xffffu : 0x8000u)) << 16;
      key[i] = x[i] > neg_inf() && (mask >> i & 1u) ? narrow | (0xffffu - (lane * V + i)) : 0u;
    }
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(kAll, best);
      if (best == 0) break;
      if (lane == j) mine = best;
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = key[i] == best ? 0u : key[i];
    }
    if (mine != 0) {
      chosen = 0xffff - (mine & 0xffffu);
      uint32_t narrow = mine >> 16;
      narrow ^= narrow & 0x8000u ? 0x8000u : 0xffffu;
      if constexpr (std::is_same_v<T, __nv_bfloat16>) xc = __uint_as_float(narrow << 16);
      else xc = __half2float(__ushort_as_half((unsigned short)narrow));
    }
  } else {
    uint32_t key[V], mine = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = c[i] > neg_inf() && (mask >> i & 1u) ? order_key(c[i]) : 0u;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) best = max(best, key[i]);
      const uint32_t most = __reduce_max_sync(kAll, best);
      if (most == 0) break;
      const int owner = __ffs(__ballot_sync(kAll, best == most)) - 1;  // equal ones: the lower lane
      int at = 0;
      if (lane == owner) {
        bool open = true;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (open && key[i] == most) {
            at = i;
            key[i] = 0;
            open = false;
          }
        }
      }
      at = __shfl_sync(kAll, at, owner) + owner * V;
      if (lane == j) chosen = at, mine = most;
    }
    if (chosen >= 0) xc = biased ? logit(row[chosen]) : from_order_key(mine);
  }
  const bool has = chosen >= 0;
  float w;
  if (a.softmax && a.renormalize) {
    const float m = max_over(xc, a.k_lanes);
    w = has ? exp_below(xc, m) : 0.f;
  } else {
    w = has ? (a.softmax ? exp_below(xc, top) / total : sigmoid(xc)) : 0.f;
  }
  if (a.renormalize) {
    const float sum = sum_over(w, a.k_lanes);
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
  __shared__ alignas(16) float s_row[kWarps][32 * V];
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  T* out = static_cast<T*>(a.grad_logits) + t * a.num_experts;
  float* buf = s_row[threadIdx.x >> 5];

  const int id = lane < a.k ? a.experts[t * a.k + lane] : -1;
  float xc = neg_inf();
  if (id >= 0 && id < a.num_experts) xc = logit_at(row, a.bias, id);
  const bool has = xc > neg_inf();
  const float g = has ? a.grad_weights[t * a.k + lane] : 0.f;

  const bool dense = a.softmax && !a.renormalize;
  float x[V], top = neg_inf(), total = 0.f;
  if (dense) {
    load_logits<T, V>(x, row, lane, a.num_experts, a.wide);
    if (a.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = lane * V + i;
        if (e < a.num_experts && !(a.bias[e] > neg_inf())) x[i] = neg_inf();
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
    top = warp_max(top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = x[i] > neg_inf() ? exp_below(x[i], top) : 0.f;
      total += x[i];
    }
    total = warp_sum(total);
  }
  float at;          // the chosen experts' own part
  float used = 0.f;  // sum over the chosen of g w (w without the scale)
  if (a.softmax) {
    float p;
    if (a.renormalize) {
      const float m = max_over(xc, a.k_lanes);
      p = has ? exp_below(xc, m) : 0.f;
      const float sum = sum_over(p, a.k_lanes);
      p = sum > 0.f ? p / sum : 0.f;
    } else {
      p = has ? exp_below(xc, top) / total : 0.f;
    }
    used = __shfl_sync(kAll, sum_over(g * p, a.k_lanes), 0);
    at = a.scale * p * (a.renormalize ? g - used : g);
  } else {
    const float e = expf(-fabsf(xc));
    const float slope = has ? e / ((1.f + e) * (1.f + e)) : 0.f;  // s (1 - s), without the difference
    at = g;
    if (a.renormalize) {
      const float s = has ? sigmoid(xc) : 0.f;
      const float sum = sum_over(s, a.k_lanes);
      used = sum_over(sum > 0.f ? g * (s / sum) : 0.f, a.k_lanes);
      at = sum > 0.f ? (g - used) / sum : 0.f;
    }
    at *= a.scale * slope;
  }
  const float each = dense && total > 0.f ? -(a.scale * used) / total : 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) buf[lane * V + i] = dense ? each * x[i] : 0.f;
  __syncwarp();
  if (has) atomicAdd(&buf[id], at);  // ids of one token are distinct: no two lanes meet
  __syncwarp();
  constexpr int N = vector_length<T, V>();
  if (a.wide) {
#pragma unroll
    for (int c = 0; c < V; c += N) {
      const int e = lane * V + c;
      dev::Pack<T, N> p;
#pragma unroll
      for (int i = 0; i < N; ++i) p.v[i] = dev::from_float<T>(buf[e + i]);
      if (e < a.num_experts) *reinterpret_cast<dev::Pack<T, N>*>(out + e) = p;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = i * 32 + lane;
      if (e < a.num_experts) out[e] = dev::from_float<T>(buf[e]);
    }
  }
}

int lanes_for(int k) {
  int n = 1;
  while (n < k) n *= 2;
  return n;
}

// Experts to a lane: the power of two with which 32 lanes hold them all.
int experts_per_lane(int num_experts) { return lanes_for((num_experts + 31) / 32); }

// Whether rows can be read and written as vectors of a lane's experts (of 16
// bytes where those are more).
bool whole_vectors(int type, int num_experts, std::initializer_list<const void*> bases, int64_t stride) {
  const int size = float_type_bytes(type), n = std::min(experts_per_lane(num_experts), 16 / size);
  uintptr_t bits = (uintptr_t)(stride * size);
  for (const void* p : bases) bits |= reinterpret_cast<uintptr_t>(p);
  return num_experts % n == 0 && bits % (n * size) == 0;
}

// Lanes to a group where groups are aligned runs of a power of two of whole
// lanes, else 0.
int lanes_per_group(int num_experts, int per_group) {
  const int v = experts_per_lane(num_experts), n = per_group / v;
  return per_group % v == 0 && (n & (n - 1)) == 0 ? n : 0;
}

template <template <typename, int> class K, typename Args>
cudaError_t launch(int type, int num_experts, int64_t tokens, const Args& a, cudaStream_t stream) {
  const int64_t grid = (tokens + kWarps - 1) / kWarps;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  const bool known = with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    switch (experts_per_lane(num_experts)) {
      case 1: K<T, 1>::run((int)grid, a, stream); break;
      case 2: K<T, 2>::run((int)grid, a, stream); break;
      case 4: K<T, 4>::run((int)grid, a, stream); break;
      case 8: K<T, 8>::run((int)grid, a, stream); break;
      case 16: K<T, 16>::run((int)grid, a, stream); break;
      default: K<T, 32>::run((int)grid, a, stream); break;
    }
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
  const int per_group = num_experts / groups;
  const RouteArgs a{d_logits, row_stride, d_bias, d_weights, d_experts, num_tokens, num_experts, k, lanes_for(k), groups,
                    groups_kept, per_group, lanes_per_group(num_experts, per_group),
                    whole_vectors(type, num_experts, {d_logits}, row_stride), score == CUSORT_SCORE_SOFTMAX,
                    renormalize != 0, group_score == CUSORT_GROUP_TOP2, scale};
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
                            num_experts, k, lanes_for(k),
                            whole_vectors(type, num_experts, {d_logits, d_grad_logits}, row_stride),
                            score == CUSORT_SCORE_SOFTMAX, renormalize != 0, scale};
  return launch<Backward>(type, num_experts, num_tokens, a, stream);
}
