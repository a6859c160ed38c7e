// cusort_route.cu -- routing of tokens to experts: scores, a bias for
// balance, groups, the k best, their weights; and the gradient of the logits.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/cusort_b200.h"
#include "cusort_float.cuh"
#include "cusort_overlap.cuh"

namespace {

using namespace cusort_b200;

constexpr int kMaxExperts = 1024;
constexpr int kMaxChosen = 32;  // one lane per chosen expert
constexpr int kMaxGroups = 32;  // one lane per group
constexpr int kWarps = 4;       // per CTA
constexpr int64_t kBusyWarps = 148 * 4 * 6;
constexpr uint32_t kAll = 0xffffffffu;

struct RouteArgs {
  const void* logits;
  int64_t stride;  // elements between rows
  const float* bias;
  float* weights;
  int32_t* experts;
  int64_t tokens;
  int num_experts, k, k_lanes;  // k_lanes: the power of two from k on
  int per_warp;                 // tokens to a warp, at most 32 / k_lanes
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
  int num_experts, k, k_lanes, per_warp;
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
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
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

// The lane's V consecutive values of a row, from expert lane * V on; -inf
// beyond the last.
template <typename T, int V>
__device__ __forceinline__ void load_row(T (&x)[V], const T* row, int lane, int num_experts, bool wide) {
  constexpr int N = vector_length<T, V>();
  const T none = dev::from_float<T>(neg_inf());
  if (wide) {
#pragma unroll
    for (int c = 0; c < V; c += N) {
      if (lane * V + c < num_experts) {
        const auto p = *reinterpret_cast<const dev::Pack<T, N>*>(row + lane * V + c);
#pragma unroll
        for (int i = 0; i < N; ++i) x[c + i] = p.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[c + i] = none;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = lane * V + i < num_experts ? row[lane * V + i] : none;
  }
}

// The k largest keys (0: none) of a warp whose lanes hold V consecutive
// experts each, in order, equal ones by their expert; lane base + j gets the
// j-th key and its expert.  UNIQUE: no two keys but 0 are equal.
//
// Few experts to a lane: k rounds over all keys.  More: the k-th largest of
// the lanes' own maxima is below no more than k - 1 keys in other lanes, so
// the k largest are among the keys from it on, seldom more than a few beyond
// k; these are gathered one to a lane and take the place that the number of
// those before them says.  Counting takes more exchanges than rounds would,
// but none waits for another (8192 x 256 f32, k = 8: 7.1 us in rounds, 6.4).
// Measured (us, all keys -> gathered): 32768 tokens of 128 experts, 32-bit
// logits, k = 8 20.2 -> 15.5, k = 4 12.6 -> 14.0 (not there); 16-bit logits,
// whose rounds are shorter, 256 experts, k = 8 14.1 -> 18.6 (not there).
template <int V, bool UNIQUE>
__device__ __forceinline__ void choose(uint32_t (&key)[V], int k, int lane, int base, uint2* scratch, uint32_t& mine,
                                       int& chosen) {
  if constexpr (V >= (UNIQUE ? 16 : 4)) {
    if (V > 4 || k > 4) {
      uint32_t m = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) m = max(m, key[i]);
      int above = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) above += __shfl_sync(kAll, m, i) > m;
      // lanes whose maximum has fewer than k above it hold the k largest; the smallest of them
      const uint32_t low = max(1u, __reduce_min_sync(kAll, above < k ? m : 0xffffffffu));
      uint32_t mask = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) mask |= (key[i] >= low ? 1u : 0u) << i;
      const int count = __popc(mask);
      const uint32_t b0 = __ballot_sync(kAll, count & 1), b1 = __ballot_sync(kAll, count & 2),
                     b2 = __ballot_sync(kAll, count & 4), b3 = __ballot_sync(kAll, count & ~7);
      const int total = __popc(b0) + 2 * __popc(b1) + 4 * __popc(b2);
      if (b3 == 0 && total <= 32) {
        const uint32_t below = dev::lanemask_lt();
        int at = __popc(b0 & below) + 2 * __popc(b1 & below) + 4 * __popc(b2 & below);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (mask >> i & 1u) scratch[at++] = make_uint2(key[i], lane * V + i);
        __syncwarp();
        uint2 c = lane < total ? scratch[lane] : make_uint2(0u, 0u);
        __syncwarp();
        // a candidate's place is the number of those before it
        int place = 0;
#pragma unroll 4
        for (int i = 0; i < total; ++i) {
          const uint32_t other = __shfl_sync(kAll, c.x, i);
          place += other > c.x || (other == c.x && i < lane);
        }
        if (lane < total) scratch[place] = c;
        __syncwarp();
        if (lane >= base && lane - base < min(k, total)) {
          c = scratch[lane - base];
          mine = c.x;
          chosen = (int)c.y;
        }
        __syncwarp();
        return;
      }
    }
  }
  if constexpr (UNIQUE) {
    // The next largest key is the one with the largest key - last, modulo 2^32: what is not below `last` comes out
    // smaller than what is, so nothing has to be taken out.
    uint32_t last = 0;
    for (int j = 0; j < k; ++j) {
      uint32_t best = key[0] - last;
#pragma unroll
      for (int i = 1; i < V; ++i) best = max(best, key[i] - last);
      last += __reduce_max_sync(kAll, best);
      if (last == 0) break;
      if (lane == base + j) mine = last;
    }
    if (lane >= base && mine != 0) chosen = 0xffff - (mine & 0xffffu);
  } else {
    for (int j = 0; j < k; ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) best = max(best, key[i]);
      const uint32_t most = __reduce_max_sync(kAll, best);
      if (most == 0) break;
      const int owner = __ffs(__ballot_sync(kAll, best == most)) - 1;  // equal ones: the lower lane
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) hits |= (key[i] == most ? 1u : 0u) << i;
      hits = lane == owner ? hits & (0u - hits) : 0u;
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = hits >> i & 1u ? 0u : key[i];
      const int e = __shfl_sync(kAll, __ffs(hits) - 1, owner) + owner * V;
      if (lane == base + j) mine = most, chosen = e;
    }
  }
}

// Order keys of 16-bit logits, unique: the logit's order above, the expert
// below (lower experts larger); 0 where the logit is -inf or NaN.  The signed
// order of two halves at once: negative ones inverted, the others with the
// sign bit set.
template <typename T, int V>
__device__ __forceinline__ void narrow_keys(uint32_t (&key)[V], const T (&x)[V], int lane) {
  using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
  constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
  constexpr uint32_t kLeast = (0x8000u - kInf) << 16;           // from the first above -inf
  constexpr uint32_t kSpan = (2 * kInf) << 16 | 0xffffu;        // to +inf itself; NaN lies beyond, on either side
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    T2 pair;
    pair.x = x[i];
    pair.y = x[i + 1 < V ? i + 1 : i];
    T2 zero;
    zero.x = zero.y = dev::from_float<T>(0.f);
    pair = __hadd2(pair, zero);  // -0 becomes +0
    uint32_t w = *reinterpret_cast<uint32_t*>(&pair);
    w ^= ((w & 0x80008000u) >> 15) * 0xffffu | 0x80008000u;
    key[i] = w << 16 | (0xffffu - (lane * V + i));
    if (i + 1 < V) key[i + 1] = (w & 0xffff0000u) | (0xffffu - (lane * V + i + 1));
  }
#pragma unroll
  for (int i = 0; i < V; ++i) key[i] = key[i] - kLeast <= kSpan ? key[i] : 0u;
}

// Which groups stay: lane's mask of its V experts (bit i: expert lane * V + i).
// value: what groups go by, -inf where not available.
template <int V>
__device__ __forceinline__ uint32_t kept_experts(const RouteArgs& a, const float (&value)[V], int lane) {
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
    const int shift = __ffs(a.group_lanes) - 1, group = lane >> shift;
    // groups_kept rounds: the largest, the lower lane among equals.  -inf has a key above 0, so that every round
    // takes one group.
    uint32_t key = group < a.groups ? order_key((a.top2 && b2 > neg_inf() ? b1 + b2 : b1) + 0.f) : 0u, kept = 0;
    for (int n = 0; n < a.groups_kept; ++n) {
      const uint32_t most = __reduce_max_sync(kAll, key);
      if (group == (__ffs(__ballot_sync(kAll, key == most)) - 1) >> shift) key = 0, kept = kAll;
    }
    return kept;
  }
  // groups of any length: one after the other, lane g keeps group g's
  float mine = neg_inf();
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

// A warp takes per_warp tokens one after the other; a lane holds V consecutive
// experts, so that a lower lane means a lower expert and groups are runs of
// lanes.  The chosen experts of its tokens lie k_lanes lanes apart, and their
// weights are computed for all tokens at once.
//
// Bound by instruction issue and, within a token, by the chain of its rounds
// (ncu: 54-61 % of the issue slots, 34-37 % of the warps, 6-8 % of the DRAM
// rate).  Measured: 8192 x 256 f32, sigmoid with a bias, 4 of 8 groups, k = 8:
// 12.2 us; 32768 x 128 bf16, renormalised softmax, k = 4: 7.8 us (1.2 TB/s);
// 16 x 64: 2.0 us.
//
// SCORED: scores of all experts are needed (a softmax's sum, a bias, groups by
// their scores); GROUPED: groups_kept < groups.  A kernel of its own for what
// needs neither holds half the registers.
// Seven CTAs to an SM instead of the four that the scored kernels would take
// (8192 x 256 f32 logits, us: softmax 9.5 -> 8.0, sigmoid, bias and groups 14.7
// -> 13.2, in spite of 44 bytes spilled; ten CTAs 14.8), and four instead of two
// from 257 experts on (8192 x 512, softmax: 20.6 -> 15.8).  Measured for 32-bit
// logits.  Of 8 and 16 experts to a lane the scored kernels of all types spill,
// up to 36 bytes, with groups 36 to 92; those of 32 with groups, at the 255
// registers that there are, 32 to 92.
template <typename T, int V, bool SCORED, bool GROUPED>
__global__ void __launch_bounds__(32 * kWarps, V <= 8 ? 7 : V == 16 ? 4 : 1) route_kernel(RouteArgs a) {
  dev::wait_for_previous();
  __shared__ uint2 s_scratch[kWarps][32];
  const int lane = threadIdx.x & 31;
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * a.per_warp;
  if (t0 >= a.tokens) return;
  const int tokens = (int)min((int64_t)a.per_warp, a.tokens - t0);
  const T* row = static_cast<const T*>(a.logits) + t0 * a.stride;
  const bool biased = SCORED && a.bias != nullptr;

  float b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = biased && lane * V + i < a.num_experts ? a.bias[lane * V + i] : 0.f;

  int chosen = -1;
  uint32_t mine = 0;
  float top = neg_inf(), total = 0.f;  // of the token whose chosen expert the lane holds
  T raw[V];
  load_row<T, V>(raw, row, lane, a.num_experts, a.wide);
  for (int n = 0; n < tokens; ++n) {
    const int base = n * a.k_lanes;
    T now[V];
#pragma unroll
    for (int i = 0; i < V; ++i) now[i] = raw[i];
    row += a.stride;
    if (n + 1 < tokens) load_row<T, V>(raw, row, lane, a.num_experts, a.wide);
    uint32_t mask = kAll;  // experts of the lane that may be chosen
    float c[V];  // what experts are ordered by: the logit (both scores grow with it), or the score plus the bias
    if constexpr (sizeof(T) == 4 || SCORED || GROUPED) {
      float x[V], value[V];  // value: what groups go by
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = x[i] = b[i] > neg_inf() ? logit(now[i]) : neg_inf();
      if constexpr (SCORED) {
        float s[V];
        if (a.softmax) {
          float m = x[0], sum = 0.f;
#pragma unroll
          for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
          m = warp_max(m);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            s[i] = x[i] > neg_inf() ? exp_below(x[i], m) : 0.f;
            sum += s[i];
          }
          sum = warp_sum(sum);
          if (lane >= base) top = m, total = sum;  // later tokens' lanes are set again
          if (biased) {
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = s[i] / sum;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) s[i] = sigmoid(x[i]);
          if (biased) {
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = s[i];
          }
        }
        if (biased) {
#pragma unroll
          for (int i = 0; i < V; ++i) c[i] = x[i] > neg_inf() ? c[i] + b[i] : neg_inf();
        }
        if (a.top2 && !biased) {
#pragma unroll
          for (int i = 0; i < V; ++i) value[i] = x[i] > neg_inf() ? s[i] : neg_inf();
        }
      }
      if (biased || !a.top2) {
#pragma unroll
        for (int i = 0; i < V; ++i) value[i] = c[i];
      }
      if constexpr (GROUPED) mask = kept_experts<V>(a, value, lane);
    }
    uint32_t key[V];
    if (sizeof(T) == 2 && !biased) {
      if constexpr (sizeof(T) == 2) narrow_keys<T, V>(key, now, lane);
      if constexpr (GROUPED) {
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = mask >> i & 1u ? key[i] : 0u;
      }
      choose<V, true>(key, a.k, lane, base, s_scratch[threadIdx.x >> 5], mine, chosen);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = c[i] > neg_inf() && (mask >> i & 1u) ? order_key(c[i]) : 0u;
      choose<V, false>(key, a.k, lane, base, s_scratch[threadIdx.x >> 5], mine, chosen);
    }
  }

  const int n = lane / a.k_lanes, j = lane - n * a.k_lanes;
  const int64_t t = t0 + n;
  const bool has = chosen >= 0;
  float xc = neg_inf();  // the chosen expert's logit
  if (has) {
    if (biased) {
      xc = logit(static_cast<const T*>(a.logits)[t * a.stride + chosen]);
    } else if constexpr (std::is_same_v<T, float>) {
      xc = from_order_key(mine);
    } else {
      uint32_t narrow = mine >> 16;
      narrow ^= narrow & 0x8000u ? 0x8000u : 0xffffu;
      if constexpr (std::is_same_v<T, __nv_bfloat16>) xc = __uint_as_float(narrow << 16);
      else xc = __half2float(__ushort_as_half((unsigned short)narrow));
    }
  }
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
  if (n < tokens && j < a.k) {
    a.experts[t * a.k + j] = chosen;
    a.weights[t * a.k + j] = w * a.scale;
  }
}

// Where an expert's value lies in a warp's row in shared memory: the lanes'
// 16-byte words side by side, so that none of them share a bank (as V values
// a lane in a run, 32768 x 1024 gradients took 81 us).
template <int V>
__device__ __forceinline__ int place_of(int expert) {
  if constexpr (V <= 4) return expert;
  const int lane = expert / V, i = expert % V;
  return (i / 4 * 32 + lane) * 4 + i % 4;
}

// A warp takes per_warp tokens: first the gradients at all their chosen
// experts, k_lanes lanes to a token, then row after row, put together in
// shared memory.  With w the weights, u = sum of g w, S the chosen scores' sum:
//   softmax, renormalised   dl = w (g - u / scale) at the chosen, 0 elsewhere
//   softmax                 dl = scale p g at the chosen, - p u everywhere
//   sigmoid                 dl = scale g s (1 - s), or
//                           (scale g - u) (s / S) (1 - s) renormalised
// Bound by latency (ncu: 45 % of the issue slots).  Measured, 32768 x 128 bf16,
// k = 4: 4.2 us where only the chosen have a gradient (2.0 TB/s), 11.4 us where
// all do.  Many experts: as many CTAs to an SM as keep all values in registers
// (32768 x 512 bf16, k = 8: 18.1 -> 12.4 and 38.5 -> 25.5 us).
template <typename T, int V>
__global__ void __launch_bounds__(32 * kWarps, V <= 4 ? 1 : V == 8 ? 10 : V == 16 ? 8 : 4) route_backward_kernel(RouteBackwardArgs a) {
  dev::wait_for_previous();
  __shared__ alignas(16) float s_row[kWarps][32 * V];
  const int lane = threadIdx.x & 31;
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * a.per_warp;
  if (t0 >= a.tokens) return;
  const int tokens = (int)min((int64_t)a.per_warp, a.tokens - t0);
  const int mine = lane / a.k_lanes, j = lane - mine * a.k_lanes;
  const T* row = static_cast<const T*>(a.logits) + t0 * a.stride;
  T* out = static_cast<T*>(a.grad_logits) + t0 * a.num_experts;
  float* buf = s_row[threadIdx.x >> 5];

  int id = -1;
  float xc = neg_inf(), g = 0.f;
  if (mine < tokens && j < a.k) {
    id = a.experts[(t0 + mine) * a.k + j];
    g = a.grad_weights[(t0 + mine) * a.k + j];
    if (id >= 0 && id < a.num_experts) xc = logit_at(row + mine * a.stride, a.bias, id);
  }
  const bool has = xc > neg_inf();
  if (!has) g = 0.f;

  const bool dense = a.softmax && !a.renormalize;
  float at = 0.f;  // the chosen experts' own part
  if (a.softmax && a.renormalize) {
    const float m = max_over(xc, a.k_lanes);
    float p = has ? exp_below(xc, m) : 0.f;
    const float sum = sum_over(p, a.k_lanes);
    p = sum > 0.f ? p / sum : 0.f;
    at = a.scale * p * (g - sum_over(g * p, a.k_lanes));
  } else if (!a.softmax) {
    const float e = expf(-fabsf(xc));
    if (a.renormalize) {
      // s / S before the product: a sum of subnormal scores would take 1 / S beyond the largest number
      const float s = has ? sigmoid(xc) : 0.f;
      const float sum = sum_over(s, a.k_lanes);
      const float share = sum > 0.f ? s / sum : 0.f;
      const float rest = (xc > 0.f ? e : 1.f) / (1.f + e);  // 1 - s, without the difference
      const float used = sum_over(sum > 0.f ? g * share : 0.f, a.k_lanes);
      at = sum > 0.f ? a.scale * share * rest * (g - used) : 0.f;
    } else {
      at = has ? g * (a.scale * (e / ((1.f + e) * (1.f + e)))) : 0.f;  // s (1 - s), without the difference
    }
  }
  T raw[V];
  if (dense) load_row<T, V>(raw, row, lane, a.num_experts, a.wide);
  for (int n = 0; n < tokens; ++n, out += a.num_experts) {
    float x[V];
    if (dense) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = logit(raw[i]);
      row += a.stride;
      if (n + 1 < tokens) load_row<T, V>(raw, row, lane, a.num_experts, a.wide);
      if (a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = lane * V + i;
          if (e < a.num_experts && !(a.bias[e] > neg_inf())) x[i] = neg_inf();
        }
      }
      float top = x[0], total = 0.f;
#pragma unroll
      for (int i = 1; i < V; ++i) top = fmaxf(top, x[i]);
      top = warp_max(top);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i] = x[i] > neg_inf() ? exp_below(x[i], top) : 0.f;
        total += x[i];
      }
      const float e = has && mine == n ? exp_below(xc, top) : 0.f;
      const float sum = warp_sum(total), used = warp_sum(g * e);
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      if (mine == n) at = a.scale * g * (e * inv);
      const float each = -(a.scale * inv) * (used * inv);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] *= each;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) buf[place_of<V>(lane * V + i)] = x[i];
    __syncwarp();
    if (has && mine == n) atomicAdd(&buf[place_of<V>(id)], at);  // lanes meet, in any order, only where a caller repeats an expert
    __syncwarp();
    constexpr int N = vector_length<T, V>();
    if (a.wide) {
#pragma unroll
      for (int c = 0; c < V; c += N) {
        const int e = lane * V + c;
        dev::Pack<T, N> p;
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = dev::from_float<T>(buf[place_of<V>(e + i)]);
        if (e < a.num_experts) *reinterpret_cast<dev::Pack<T, N>*>(out + e) = p;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = i * 32 + lane;
        if (e < a.num_experts) out[e] = dev::from_float<T>(buf[place_of<V>(e)]);
      }
    }
    __syncwarp();
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

// Tokens to a warp: what a warp does once for its tokens is the cheaper the
// more they are, as long as kBusyWarps warps are left (about six to each of
// the 592 schedulers).
int tokens_per_warp(int64_t tokens, int k) {
  int n = 32 / lanes_for(k);
  while (n > 1 && tokens / n < kBusyWarps) n /= 2;
  return n;
}

template <template <typename, int> class K, typename Args>
cudaError_t launch(int type, int num_experts, int64_t tokens, const Args& a, cudaStream_t stream) {
  const int64_t per_cta = (int64_t)kWarps * a.per_warp, grid = (tokens + per_cta - 1) / per_cta;
  cudaError_t err = cudaErrorInvalidValue;
  with_float_type(type, [&](auto zero) {
    using T = decltype(zero);
    switch (experts_per_lane(num_experts)) {
      case 1: err = K<T, 1>::run(grid, a, stream); break;
      case 2: err = K<T, 2>::run(grid, a, stream); break;
      case 4: err = K<T, 4>::run(grid, a, stream); break;
      case 8: err = K<T, 8>::run(grid, a, stream); break;
      case 16: err = K<T, 16>::run(grid, a, stream); break;
      default: err = K<T, 32>::run(grid, a, stream); break;
    }
  });
  return err;
}

template <typename T, int V> struct Forward {
  static cudaError_t run(int64_t grid, const RouteArgs& a, cudaStream_t s) {
    const bool grouped = a.groups_kept < a.groups;
    const bool scored = a.bias != nullptr || (a.softmax && !a.renormalize) || (grouped && a.top2);
    return launch_after_previous(grouped  ? route_kernel<T, V, true, true>
                                 : scored ? route_kernel<T, V, true, false>
                                          : route_kernel<T, V, false, false>,
                                 grid, 32 * kWarps, 0, a, s);
  }
};
template <typename T, int V> struct Backward {
  static cudaError_t run(int64_t grid, const RouteBackwardArgs& a, cudaStream_t s) {
    return launch_after_previous(route_backward_kernel<T, V>, grid, 32 * kWarps, 0, a, s);
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
  const RouteArgs a{d_logits, row_stride, d_bias, d_weights, d_experts, num_tokens, num_experts, k, lanes_for(k),
                    tokens_per_warp(num_tokens, k), groups, groups_kept, per_group, lanes_per_group(num_experts, per_group),
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
                            num_experts, k, lanes_for(k), tokens_per_warp(num_tokens, k),
                            whole_vectors(type, num_experts, {d_logits, d_grad_logits}, row_stride),
                            score == CUSORT_SCORE_SOFTMAX, renormalize != 0, scale};
  return launch<Backward>(type, num_experts, num_tokens, a, stream);
}
