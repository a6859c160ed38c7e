// cusort_plan.cu -- grouping (token, expert) pairs by expert: counts, aligned
// segment offsets, the pair at every row and the row of every pair.  A stable
// counting sort over at most 1024 experts.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"
#include "cusort_device.cuh"

namespace {

using namespace cusort_b200;

constexpr int kMaxExperts = 1024;
constexpr int kThreads = 1024;     // per CTA; kSmallThreads where all pairs are few
constexpr int kSmallThreads = 256;
constexpr int64_t kSmallItems = 1024;
constexpr int64_t kOneTileItems = 8192;   // up to here one CTA does it all, in one launch
constexpr int64_t kMinTileItems = 2048;
constexpr int kMaxTiles = 148;            // one CTA per SM
constexpr uint32_t kAll = 0xffffffffu;

struct PlanArgs {
  const void* experts;
  int64_t items, capacity, tile_items;
  int num_experts, align;
  uint32_t* tile_counts;  // [tiles][num_experts]; null: one tile, counted in place
  int32_t *counts, *offsets, *sources, *positions;
};

// The item's expert; num_experts for items that belong to none.
template <typename I>
__device__ __forceinline__ int expert_of(const PlanArgs& a, int64_t i, int64_t end) {
  if (i >= end) return a.num_experts;
  const I e = static_cast<const I*>(a.experts)[i];
  return e >= 0 && e < (I)a.num_experts ? (int)e : a.num_experts;
}

template <typename I>
__global__ void __launch_bounds__(kThreads) plan_count_kernel(PlanArgs a) {
  __shared__ uint32_t s_count[kMaxExperts];
  dev::pdl_launch_dependents();
  for (int e = threadIdx.x; e < a.num_experts; e += kThreads) s_count[e] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * a.tile_items, end = min(begin + a.tile_items, a.items);
#pragma unroll 2
  for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) {
    const int e = expert_of<I>(a, i, end);
    if (e < a.num_experts) atomicAdd(&s_count[e], 1u);
  }
  __syncthreads();
  uint32_t* out = a.tile_counts + (int64_t)blockIdx.x * a.num_experts;
  for (int e = threadIdx.x; e < a.num_experts; e += kThreads) out[e] = s_count[e];
}

// Every CTA counts its tile warp by warp (a warp's items are one run), adds up
// the tiles before its own and all of them, scans the aligned totals, and
// gives its items their rows: in each 32 items the peers of an expert by their
// lanes.
template <typename I, int THREADS>
__global__ void __launch_bounds__(THREADS) plan_place_kernel(PlanArgs a) {
  constexpr int W = THREADS / 32;
  extern __shared__ uint32_t s_warp[];  // [W][num_experts]: the next item of an expert in a warp's run
  __shared__ uint32_t s_before[kMaxExperts], s_total[kMaxExperts], s_offset[kMaxExperts + 1], s_sums[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.num_experts;
  const int64_t begin = blockIdx.x * a.tile_items, end = min(begin + a.tile_items, a.items);
  const int64_t run = (a.tile_items + 32 * W - 1) / (32 * W) * 32;
  const int64_t wbegin = min(begin + warp * run, end), wend = min(wbegin + run, end);
  for (int i = threadIdx.x; i < W * E; i += THREADS) s_warp[i] = 0;
  for (int e = threadIdx.x; e < E; e += THREADS) s_before[e] = s_total[e] = 0;
  __syncthreads();
  uint32_t* mine = s_warp + warp * E;
#pragma unroll 4
  for (int64_t i = wbegin + lane; i < wend; i += 32) {
    const int e = expert_of<I>(a, i, wend);
    if (e < E) atomicAdd(&mine[e], 1u);
  }
  if (a.tile_counts != nullptr) {
    // columns of the tiles' counts: as many threads to an expert as there are
    dev::pdl_wait();
    const int parts = max(1, THREADS / E), tiles = gridDim.x;
    for (int i = threadIdx.x; i < parts * E; i += THREADS) {
      const int e = i % E;
      uint32_t before = 0, total = 0;
#pragma unroll 8
      for (int t = i / E; t < tiles; t += parts) {
        const uint32_t c = a.tile_counts[(int64_t)t * E + e];
        if (t < blockIdx.x) before += c;
        total += c;
      }
      atomicAdd(&s_before[e], before);
      atomicAdd(&s_total[e], total);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += THREADS) {
    uint32_t at = s_before[e];
#pragma unroll 8
    for (int w = 0; w < W; ++w) {
      const uint32_t c = s_warp[w * E + e];
      s_warp[w * E + e] = at;
      at += c;
    }
    if (a.tile_counts == nullptr) s_total[e] = at;
  }
  __syncthreads();
  // exclusive scan of the aligned totals, P experts to a thread
  {
    constexpr int P = kMaxExperts / THREADS;
    const uint32_t al = a.align;
    uint32_t v[P], sum = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = threadIdx.x * P + j;
      v[j] = sum;
      sum += e < E ? (s_total[e] + al - 1) / al * al : 0;
    }
    uint32_t in = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(kAll, in, d);
      if (lane >= d) in += o;
    }
    if (lane == 31) s_sums[warp] = in;
    __syncthreads();
    uint32_t before = lane < warp ? s_sums[lane] : 0;  // W <= 32
    before = __reduce_add_sync(kAll, before) + in - sum;
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (threadIdx.x * P + j < E) s_offset[threadIdx.x * P + j] = before + v[j];
    if (threadIdx.x == THREADS - 1) s_offset[E] = before + sum;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < E; e += THREADS) {
      a.counts[e] = (int32_t)s_total[e];
      a.offsets[e] = (int32_t)s_offset[e];
    }
    if (threadIdx.x == 0) a.offsets[E] = (int32_t)s_offset[E];
  }
#pragma unroll 4
  for (int64_t base = wbegin; base < wend; base += 32) {
    const int64_t i = base + lane;
    const int e = expert_of<I>(a, i, wend);
    const uint32_t peers = __match_any_sync(kAll, e);
    uint32_t at = 0;
    if (e < E) at = mine[e] + __popc(peers & dev::lanemask_lt());
    __syncwarp();
    if (e < E && (peers >> lane) == 1u) mine[e] = at + 1;  // the last peer
    __syncwarp();
    if (i < wend) {
      const int64_t row = e < E ? (int64_t)s_offset[e] + at : -1;
      a.positions[i] = (int32_t)row;
      if (e < E && row < a.capacity) a.sources[row] = (int32_t)i;
    }
  }
  // rows that hold no pair: the ends of the segments, and what follows the last
  if (a.align > 1) {
    for (int e = blockIdx.x * W + warp; e < E; e += gridDim.x * W)
      for (int64_t r = (int64_t)s_offset[e] + s_total[e] + lane; r < min((int64_t)s_offset[e + 1], a.capacity); r += 32)
        a.sources[r] = -1;
  }
  for (int64_t r = (int64_t)s_offset[E] + blockIdx.x * THREADS + threadIdx.x; r < a.capacity;
       r += (int64_t)gridDim.x * THREADS)
    a.sources[r] = -1;
}

struct PlanShape {
  int tiles;
  int64_t tile_items;
};

PlanShape shape_of(int64_t items) {
  if (items <= kOneTileItems) return {1, std::max<int64_t>(items, 1)};
  int64_t tile = std::max<int64_t>(kMinTileItems, (items + kMaxTiles - 1) / kMaxTiles);
  tile = (tile + kThreads - 1) / kThreads * kThreads;
  return {(int)((items + tile - 1) / tile), tile};
}

template <typename I, int THREADS>
cudaError_t place(const PlanArgs& a, int tiles, cudaStream_t stream) {
  const size_t smem = sizeof(uint32_t) * (THREADS / 32) * a.num_experts;
  if (smem > 32 * 1024) {  // beside the static arrays
    const cudaError_t e = cudaFuncSetAttribute(plan_place_kernel<I, THREADS>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = tiles > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, plan_place_kernel<I, THREADS>, a);
}

template <typename I>
cudaError_t run(const PlanArgs& a, int tiles, cudaStream_t stream) {
  if (tiles == 1 && a.items <= kSmallItems) return place<I, kSmallThreads>(a, 1, stream);
  if (tiles > 1) {
    plan_count_kernel<I><<<tiles, kThreads, 0, stream>>>(a);
    if (const cudaError_t e = cudaGetLastError()) return e;
  }
  return place<I, kThreads>(a, tiles, stream);
}

}  // namespace

extern "C" cudaError_t cusort_plan_dispatch(void* d_temp_storage, size_t* temp_storage_bytes, int expert_bytes,
                                            const void* d_experts, int64_t num_pairs, int num_experts, int align,
                                            int64_t capacity, int32_t* d_counts, int32_t* d_offsets,
                                            int32_t* d_sources, int32_t* d_positions, cudaStream_t stream) {
  if (temp_storage_bytes == nullptr || (expert_bytes != 4 && expert_bytes != 8) || num_pairs < 0 ||
      num_experts < 1 || num_experts > kMaxExperts || align < 1 || align > (1 << 20))
    return cudaErrorInvalidValue;
  // every row number fits 32 bits, and every pair a row
  const int64_t need = num_pairs + std::min<int64_t>(num_experts, num_pairs) * (align - 1);
  if (num_pairs > INT32_MAX || need > INT32_MAX || capacity < need || capacity > INT32_MAX)
    return cudaErrorInvalidValue;
  const PlanShape shape = shape_of(num_pairs);
  const size_t bytes = shape.tiles > 1 ? sizeof(uint32_t) * shape.tiles * num_experts : 1;
  if (d_temp_storage == nullptr) {
    *temp_storage_bytes = bytes;
    return cudaSuccess;
  }
  if (*temp_storage_bytes < bytes || (reinterpret_cast<uintptr_t>(d_temp_storage) & 15) != 0)
    return cudaErrorInvalidValue;
  if (d_counts == nullptr || d_offsets == nullptr ||
      (num_pairs > 0 && (d_experts == nullptr || d_positions == nullptr)) || (capacity > 0 && d_sources == nullptr))
    return cudaErrorInvalidValue;
  const PlanArgs a{d_experts, num_pairs, capacity, shape.tile_items, num_experts, align,
                   shape.tiles > 1 ? static_cast<uint32_t*>(d_temp_storage) : nullptr,
                   d_counts, d_offsets, d_sources, d_positions};
  return expert_bytes == 4 ? run<int32_t>(a, shape.tiles, stream) : run<int64_t>(a, shape.tiles, stream);
}
