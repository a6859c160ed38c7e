// cusort_experts_f32.cu -- the experts' matrix products of 32-bit operands, by
// multiply-adds in 32 bits: the tensor cores would round the operands.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "cusort_experts.cuh"
#include "cusort_overlap.cuh"

namespace {

using namespace cusort_b200;

constexpr int kThreads = 256;
constexpr int kSms = 148;
constexpr int kN = 128, kPad = 4;

// A CTA's tile of 16 U x 128 sums, U x 8 to a thread, K contracted elements to a step.
template <int U, int K> struct Shape {
  static constexpr int kM = 16 * U;
  static constexpr int kCtas = U == 1 ? 4 : 2;  // to an SM
  float a[2][K][kM + kPad], b[2][K][kN + kPad];
};

// Two multiply-adds: {d.x + a * b.x, d.y + a * b.y}.
__device__ __forceinline__ void add_twice(unsigned long long& d, unsigned long long a, unsigned long long b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ unsigned long long both(float x) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %1};" : "=l"(v) : "f"(x));
  return v;
}

// c (m x n) = a (m x k) x b (k x n), for each expert.  The elements' strides
// are free; one of a's and one of b's is 1.
struct FloatArgs {
  const float *a, *b;
  float* c;
  int64_t am, ak, bk, bn, b_expert, cm, c_expert;
  SegmentArgs segments;
  int m, n, k;
  uint32_t most;  // tiles along m of all experts
};

// RAGGED_K: the rows of a segment are what is contracted (the gradient of the
// weights); otherwise they are the rows of a and c, and rows of no segment are
// cleared.  A_ACROSS: a is contiguous along m, B_ALONG: b along k.
//
// Each step is loaded into registers while the one before is multiplied.
// Where experts have many rows, 8 x 8 sums to a thread: 32 experts of 1024
// rows, 1024 -> 2048, 3.3 ms, 41 TFLOP/s; 4 x 8, two multiply-adds at a time
// or not, 4.0 to 4.3 ms.  The multiply-adds bound it (55 % of their 74.4
// TFLOP/s), then the shared-memory loads beside them.  Few rows: smaller tiles,
// so that less is multiplied for nothing, and longer steps for more bytes in
// flight (64 experts of 16 rows 410 us, in tiles of 64 rows 605; of 40 rows
// 615).  The weights' bytes would take 82 of the 410: with one row of sums to a
// thread every weight that it reads from shared memory goes into a single
// multiply-add.  The gradient of the weights, 8 x 8 sums to a thread whatever
// the rows: 32 experts of 1024 rows, 1024 x 2048, 3.3 ms, 41 TFLOP/s; 64 experts
// of 16, 40 and 64 rows 305, 494 and 604 us (writing 537 MB).
template <int U, int K, bool RAGGED_K, bool B_ALONG>
__global__ void __launch_bounds__(kThreads, Shape<U, K>::kCtas)
    float_products_kernel(const __grid_constant__ FloatArgs a) {
  constexpr int kM = 16 * U, kLoadsA = kM * K / kThreads, kLoadsB = kN * K / kThreads;
  constexpr bool A_ACROSS = RAGGED_K;
  extern __shared__ uint4 raw[];
  __shared__ uint32_t sums[kThreads / 32];
  Shape<U, K>& sh = *reinterpret_cast<Shape<U, K>*>(raw);
  int32_t* s_segments = reinterpret_cast<int32_t*>(&sh + 1);
  const int experts = a.segments.experts, t = threadIdx.x;
  const Segments s{s_segments, s_segments + experts, s_segments + 2 * experts};
  dev::wait_for_previous();
  const int m_tiles = (a.m + kM - 1) / kM, n_tiles = (a.n + kN - 1) / kN;
  load_segments<kThreads>(a.segments, s, sums, a.most,
                          [&](int count) { return RAGGED_K ? m_tiles : (count + kM - 1) / kM; });
  const uint32_t tiles = (uint32_t)s.tiles[experts] * n_tiles;
  if (!RAGGED_K)
    clear_other_rows(reinterpret_cast<uint16_t*>(a.c), 2 * (int64_t)a.n, a.segments, s,
                     blockIdx.x * (kThreads / 32) + t / 32, gridDim.x * (kThreads / 32));
  const int tx = t % 16, ty = t / 16;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int e = find(s.tiles, experts, tile / n_tiles);
    const uint32_t before = s.tiles[e], of = s.tiles[e + 1] - before, local = tile - before * n_tiles;
    const int m0 = local % of * kM, n0 = local / of * kN, first = s.first[e], count = s.count[e];
    const int m = RAGGED_K ? a.m : count, k = RAGGED_K ? count : a.k;
    const float* pa = a.a + (RAGGED_K ? first * a.ak : first * a.am);
    const float* pb = a.b + (RAGGED_K ? first * a.bk : e * a.b_expert);
    float ra[kLoadsA], rb[kLoadsB];
    // consecutive threads take consecutive elements in memory
    const auto a_k = [&](int i) { return A_ACROSS ? t / kM + kThreads / kM * i : t % K; };
    const auto a_m = [&](int i) { return A_ACROSS ? t % kM : t / K + kThreads / K * i; };
    const auto b_k = [&](int i) { return B_ALONG ? t % K : t / kN + kThreads / kN * i; };
    const auto b_n = [&](int i) { return B_ALONG ? t / K + kThreads / K * i : t % kN; };
    const auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < kLoadsA; ++i)
        ra[i] = k0 + a_k(i) < k && m0 + a_m(i) < m ? pa[(m0 + a_m(i)) * a.am + (k0 + a_k(i)) * a.ak] : 0.f;
#pragma unroll
      for (int i = 0; i < kLoadsB; ++i)
        rb[i] = k0 + b_k(i) < k && n0 + b_n(i) < a.n ? pb[(k0 + b_k(i)) * a.bk + (n0 + b_n(i)) * a.bn] : 0.f;
    };
    const auto store = [&](int buffer) {
#pragma unroll
      for (int i = 0; i < kLoadsA; ++i) sh.a[buffer][a_k(i)][a_m(i)] = ra[i];
#pragma unroll
      for (int i = 0; i < kLoadsB; ++i) sh.b[buffer][b_k(i)][b_n(i)] = rb[i];
    };
    unsigned long long sum[U][4] = {};  // of pairs of columns
    load(0);
    store(0);
    __syncthreads();
    for (int k0 = 0, buffer = 0; k0 < k; k0 += K, buffer ^= 1) {
      if (k0 + K < k) load(k0 + K);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        float x[U];
        if constexpr (U == 1) {
          x[0] = sh.a[buffer][i][ty];
        } else {
#pragma unroll
          for (int u = 0; u < U; u += 4)
            *reinterpret_cast<float4*>(x + u) = *reinterpret_cast<const float4*>(&sh.a[buffer][i][ty * U + u]);
        }
        const ulonglong2 y0 = *reinterpret_cast<const ulonglong2*>(&sh.b[buffer][i][tx * 4]);
        const ulonglong2 y1 = *reinterpret_cast<const ulonglong2*>(&sh.b[buffer][i][64 + tx * 4]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const unsigned long long xx = both(x[u]);
          add_twice(sum[u][0], xx, y0.x);
          add_twice(sum[u][1], xx, y0.y);
          add_twice(sum[u][2], xx, y1.x);
          add_twice(sum[u][3], xx, y1.y);
        }
      }
      if (k0 + K < k) store(buffer ^ 1);
      __syncthreads();
    }
    float* pc = a.c + (RAGGED_K ? e * a.c_expert : first * a.cm);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int mm = m0 + ty * U + u;
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const int nn = n0 + v / 4 * 64 + tx * 4 + v % 4;
        const float x = __uint_as_float((uint32_t)(sum[u][v / 2] >> (v % 2 * 32)));
        if (mm < m && nn < a.n) pc[mm * a.cm + nn] = x;
      }
    }
  }
}

template <int U, int K, bool RAGGED_K, bool B_ALONG>
cudaError_t run(FloatArgs a, cudaStream_t stream) {
  constexpr int kM = 16 * U;
  const int64_t row_tiles = RAGGED_K ? (int64_t)a.segments.experts * ((a.m + kM - 1) / kM)
                                     : a.segments.capacity / kM + std::min(a.segments.experts, a.segments.capacity);
  const int64_t tiles = row_tiles * ((a.n + kN - 1) / kN);
  if (tiles > 1 << 30) return cudaErrorInvalidValue;
  a.most = (uint32_t)row_tiles;
  const auto kernel = float_products_kernel<U, K, RAGGED_K, B_ALONG>;
  // the limit is the kernel's, not the call's: the same one from every host thread
  constexpr size_t kMost = sizeof(Shape<U, K>) + 4 * (3 * kMaxExperts + 1);
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
  if (e) return e;
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(Shape<U, K>::kCtas * kSms, tiles));
  return launch_after_previous(kernel, grid, kThreads, sizeof(Shape<U, K>) + 4 * (3 * (size_t)a.segments.experts + 1), a,
                               stream);
}

// Rows an expert on average up to which tiles have 16 and 64 rows.  64 experts,
// 1024 -> 2048, in tiles of 16, 64 and 128 rows: 16 rows each 415, 608 and 846
// us; 24 752, 611, 848; 64 1430, 632, 886; 96 2132, 1076, 925.
constexpr int kFewestRows = 16, kFewRows = 64;

}  // namespace

namespace cusort_b200 {

cudaError_t float_products(const float* rows, int64_t row_stride, const float* weights, int64_t expert_stride,
                           int64_t in_stride, int64_t out_stride, const SegmentArgs& segments, float* out, int in,
                           int width, cudaStream_t stream) {
  const FloatArgs a{rows, weights, out, row_stride, 1, in_stride, out_stride, expert_stride, width, 0, segments, 0,
                    width, in, 0};
  const bool fewest = segments.capacity <= (int64_t)kFewestRows * segments.experts;
  const bool few = segments.capacity <= (int64_t)kFewRows * segments.experts, along = out_stride != 1;
  if (fewest) return along ? run<1, 32, false, true>(a, stream) : run<1, 32, false, false>(a, stream);
  if (few) return along ? run<4, 32, false, true>(a, stream) : run<4, 32, false, false>(a, stream);
  return along ? run<8, 16, false, true>(a, stream) : run<8, 16, false, false>(a, stream);
}

cudaError_t float_products_grad(const float* slow, int64_t slow_stride, const float* fast, int64_t fast_stride,
                                const SegmentArgs& segments, float* grad, int slow_width, int fast_width,
                                cudaStream_t stream) {
  const FloatArgs a{slow, fast, grad, 1, slow_stride, fast_stride, 1, 0, fast_width, (int64_t)slow_width * fast_width,
                    segments, slow_width, fast_width, 0, 0};
  return run<8, 16, true, false>(a, stream);
}

}  // namespace cusort_b200
