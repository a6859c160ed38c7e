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
constexpr int kM = 64, kN = 128, kK = 16;  // a CTA's tile; 4 x 8 sums to a thread
constexpr int kPad = 4;

// c (m x n) = a (m x k) x b (k x n), for each expert.  The elements' strides
// are free; one of a's and one of b's is 1.
struct FloatArgs {
  const float *a, *b;
  float* c;
  int64_t am, ak, bk, bn, b_expert, cm, c_expert;
  SegmentArgs segments;
  int m, n, k;
};

// RAGGED_K: the rows of a segment are what is contracted (the gradient of the
// weights); otherwise they are the rows of a and c, and rows of no segment are
// cleared.  A_ACROSS: a is contiguous along m, B_ALONG: b along k.
//
// Each step of 16 is loaded into registers while the one before is multiplied.
// Bound by the multiply-adds and the shared-memory loads that feed them: XXX
template <bool RAGGED_K, bool B_ALONG>
__global__ void __launch_bounds__(kThreads, 2) float_products_kernel(const __grid_constant__ FloatArgs a) {
  __shared__ float sa[2][kK][kM + kPad], sb[2][kK][kN + kPad];
  __shared__ uint32_t sums[kThreads / 32];
  extern __shared__ int32_t s_segments[];
  constexpr bool A_ACROSS = RAGGED_K;
  const int experts = a.segments.experts, t = threadIdx.x;
  const Segments s{s_segments, s_segments + experts, s_segments + 2 * experts};
  dev::wait_for_previous();
  const int m_tiles = (a.m + kM - 1) / kM, n_tiles = (a.n + kN - 1) / kN;
  load_segments<kThreads>(a.segments, s, sums, [&](int count) { return RAGGED_K ? m_tiles : (count + kM - 1) / kM; });
  const uint32_t tiles = (uint32_t)s.tiles[experts] * n_tiles;
  if (!RAGGED_K)
    clear_other_rows(reinterpret_cast<uint16_t*>(a.c), 2 * (int64_t)a.n, a.segments, s, blockIdx.x * (kThreads / 32) + t / 32,
                     gridDim.x * (kThreads / 32));
  const int tx = t % 16, ty = t / 16;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int e = find(s.tiles, experts, tile / n_tiles);
    const uint32_t before = s.tiles[e], of = s.tiles[e + 1] - before, local = tile - before * n_tiles;
    const int m0 = local % of * kM, n0 = local / of * kN, first = s.first[e], count = s.count[e];
    const int m = RAGGED_K ? a.m : count, k = RAGGED_K ? count : a.k;
    const float* pa = a.a + (RAGGED_K ? first * a.ak : first * a.am);
    const float* pb = a.b + (RAGGED_K ? first * a.bk : e * a.b_expert);
    float ra[4], rb[8];
    const auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int km = A_ACROSS ? t / kM + 4 * i : t % kK, mm = A_ACROSS ? t % kM : t / kK + 16 * i;
        ra[i] = k0 + km < k && m0 + mm < m ? pa[(m0 + mm) * a.am + (k0 + km) * a.ak] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int kn = B_ALONG ? t % kK : t / kN + 2 * i, nn = B_ALONG ? t / kK + 16 * i : t % kN;
        rb[i] = k0 + kn < k && n0 + nn < a.n ? pb[(k0 + kn) * a.bk + (n0 + nn) * a.bn] : 0.f;
      }
    };
    const auto store = [&](int buffer) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sa[buffer][A_ACROSS ? t / kM + 4 * i : t % kK][A_ACROSS ? t % kM : t / kK + 16 * i] = ra[i];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        sb[buffer][B_ALONG ? t % kK : t / kN + 2 * i][B_ALONG ? t / kK + 16 * i : t % kN] = rb[i];
    };
    float sum[4][8] = {};
    load(0);
    store(0);
    __syncthreads();
    for (int k0 = 0, buffer = 0; k0 < k; k0 += kK, buffer ^= 1) {
      if (k0 + kK < k) load(k0 + kK);
#pragma unroll
      for (int i = 0; i < kK; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(&sa[buffer][i][ty * 4]);
        const float4 y0 = *reinterpret_cast<const float4*>(&sb[buffer][i][tx * 4]);
        const float4 y1 = *reinterpret_cast<const float4*>(&sb[buffer][i][64 + tx * 4]);
        const float xs[4] = {x.x, x.y, x.z, x.w}, ys[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int v = 0; v < 8; ++v) sum[u][v] = fmaf(xs[u], ys[v], sum[u][v]);
      }
      if (k0 + kK < k) store(buffer ^ 1);
      __syncthreads();
    }
    float* pc = a.c + (RAGGED_K ? e * a.c_expert : first * a.cm);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int mm = m0 + ty * 4 + u;
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const int nn = n0 + v / 4 * 64 + tx * 4 + v % 4;
        if (mm < m && nn < a.n) pc[mm * a.cm + nn] = sum[u][v];
      }
    }
    __syncthreads();
  }
}

template <bool RAGGED_K, bool B_ALONG>
cudaError_t run(const FloatArgs& a, int64_t tiles, cudaStream_t stream) {
  if (tiles > INT32_MAX) return cudaErrorInvalidValue;
  const size_t smem = sizeof(int32_t) * (3 * (size_t)a.segments.experts + 1);
  return launch_after_previous(float_products_kernel<RAGGED_K, B_ALONG>,
                               std::max<int64_t>(1, std::min<int64_t>(2 * kSms, tiles)), kThreads, smem, a, stream);
}

}  // namespace

namespace cusort_b200 {

cudaError_t float_products(const float* rows, int64_t row_stride, const float* weights, int64_t expert_stride,
                           int64_t in_stride, int64_t out_stride, const SegmentArgs& segments, float* out, int in,
                           int width, cudaStream_t stream) {
  const FloatArgs a{rows, weights, out, row_stride, 1, in_stride, out_stride, expert_stride, width, 0, segments, 0, width, in};
  const int64_t tiles = ((int64_t)segments.capacity / kM + std::min(segments.experts, segments.capacity)) * ((width + kN - 1) / kN);
  return out_stride == 1 ? run<false, false>(a, tiles, stream) : run<false, true>(a, tiles, stream);
}

cudaError_t float_products_grad(const float* slow, int64_t slow_stride, const float* fast, int64_t fast_stride,
                                const SegmentArgs& segments, float* grad, int slow_width, int fast_width,
                                cudaStream_t stream) {
  const FloatArgs a{slow, fast, grad, 1, slow_stride, fast_stride, 1, 0, fast_width, (int64_t)slow_width * fast_width,
                    segments, slow_width, fast_width, 0};
  const int64_t tiles = (int64_t)segments.experts * ((slow_width + kM - 1) / kM) * ((fast_width + kN - 1) / kN);
  return run<true, false>(a, tiles, stream);
}

}  // namespace cusort_b200
