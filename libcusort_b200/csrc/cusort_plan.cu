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
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTiles = 148;      // one CTA per SM
constexpr int kMinTileItems = 2048;  // below this a tile's fixed cost exceeds its items'
constexpr uint32_t kAll = 0xffffffffu;

struct PlanArgs {
  const void* experts;
  int64_t items, capacity, tile_items;  // tile_items: a multiple of 32 * kWarps
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
  for (int e = threadIdx.x; e < a.num_experts; e += kThreads) s_count[e] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * a.tile_items, end = min(begin + a.tile_items, a.items);
  for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) {
    const int e = expert_of<I>(a, i, end);
    if (e < a.num_experts) atomicAdd(&s_count[e], 1u);
  }
  __syncthreads();
  uint32_t* out = a.tile_counts + (int64_t)blockIdx.x * a.num_experts;
  for (int e = threadIdx.x; e < a.num_experts; e += kThreads) out[e] = s_count[e];
}

// Every CTA adds up the tiles before its own and all of them, scans the
// aligned totals, and gives its items their rows: warp by warp over
// contiguous runs, in each 32 items the peers of an expert by their lanes.
template <typename I>
__global__ void __launch_bounds__(kThreads) plan_place_kernel(PlanArgs a) {
  extern __shared__ uint32_t s_warp[];  // [kWarps][num_experts]: the next row of an expert in a warp's run
  __shared__ uint32_t s_total[kMaxExperts], s_offset[kMaxExperts + 1], s_sums[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.num_experts;
  const int64_t begin = blockIdx.x * a.tile_items, end = min(begin + a.tile_items, a.items);
  const int64_t run = a.tile_items / kWarps;
  const int64_t wbegin = min(begin + warp * run, end), wend = min(wbegin + run, end);
  for (int i = threadIdx.x; i < kWarps * E; i += kThreads) s_warp[i] = 0;
  __syncthreads();
  uint32_t* mine = s_warp + warp * E;
  for (int64_t i = wbegin + lane; i < wend; i += 32) {
    const int e = expert_of<I>(a, i, wend);
    if (e < E) atomicAdd(&mine[e], 1u);
  }
  __syncthreads();
  // each expert: items before this tile, its total
  for (int e = threadIdx.x; e < E; e += kThreads) {
    uint32_t before = 0, total = 0;
    if (a.tile_counts != nullptr) {
      for (int t = 0; t < gridDim.x; ++t) {
        const uint32_t c = a.tile_counts[(int64_t)t * E + e];
        if (t < blockIdx.x) before += c;
        total += c;
      }
    }
    uint32_t at = before;
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = s_warp[w * E + e];
      s_warp[w * E + e] = at;
      at += c;
    }
    s_total[e] = a.tile_counts != nullptr ? total : at;
  }
  __syncthreads();
  // exclusive scan of the aligned totals: four experts to a thread
  {
    const uint32_t al = a.align;
    uint32_t v[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = threadIdx.x * 4 + j;
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
    uint32_t before = in - sum;
    for (int w = 0; w < warp; ++w) before += s_sums[w];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (threadIdx.x * 4 + j < E) s_offset[threadIdx.x * 4 + j] = before + v[j];
    if (threadIdx.x == kThreads - 1) s_offset[E] = before + sum;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < E; e += kThreads) {
      a.counts[e] = (int32_t)s_total[e];
      a.offsets[e] = (int32_t)s_offset[e];
    }
    if (threadIdx.x == 0) a.offsets[E] = (int32_t)s_offset[E];
  }
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
    for (int e = blockIdx.x * kWarps + warp; e < E; e += gridDim.x * kWarps)
      for (int64_t r = (int64_t)s_offset[e] + s_total[e] + lane; r < min((int64_t)s_offset[e + 1], a.capacity); r += 32)
        a.sources[r] = -1;
  }
  for (int64_t r = (int64_t)s_offset[E] + blockIdx.x * kThreads + threadIdx.x; r < a.capacity;
       r += (int64_t)gridDim.x * kThreads)
    a.sources[r] = -1;
}

struct PlanShape {
  int tiles;
  int64_t tile_items;
};

PlanShape shape_of(int64_t items) {
  const int64_t step = 32 * kWarps;
  int64_t tile = std::max<int64_t>(kMinTileItems, (items + kMaxTiles - 1) / kMaxTiles);
  tile = (tile + step - 1) / step * step;
  return {(int)std::max<int64_t>(1, (items + tile - 1) / tile), tile};
}

template <typename I>
cudaError_t run(const PlanArgs& a, int tiles, cudaStream_t stream) {
  const size_t smem = sizeof(uint32_t) * kWarps * a.num_experts;
  if (tiles > 1) {
    plan_count_kernel<I><<<tiles, kThreads, 0, stream>>>(a);
    if (const cudaError_t e = cudaGetLastError()) return e;
  }
  plan_place_kernel<I><<<tiles, kThreads, smem, stream>>>(a);
  return cudaGetLastError();
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
