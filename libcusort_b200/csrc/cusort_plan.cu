// cusort_plan.cu -- grouping (token, expert) pairs by expert: counts, aligned
// segment offsets, the pair at every row and the row of every pair.  A stable
// counting sort over at most 1024 experts: row of pair i = offset of its expert
// + the pairs of that expert before i.
//
// Up to 2048 pairs one CTA does it in one launch; more are split into tiles,
// whose counts a first kernel leaves for the second to add up.  Bound by
// latency and by the ranking's issue slots (ncu: 37 % and 50 % of them), not by
// memory.  Measured: 512 pairs over 256 experts 3.9 us; 262144 over 128 9.7 us
// (0.5 us at the copy rate); 1M over 128 17 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"
#include "cusort_overlap.cuh"

namespace {

using namespace cusort_b200;

constexpr int kMaxExperts = 1024;
constexpr int kThreads = 1024;          // per CTA; kSmallThreads where all pairs are few
constexpr int kSmallThreads = 256;
constexpr int kItems = 4;               // to a thread, in registers
constexpr int64_t kSmallItems = kSmallThreads * kItems;
constexpr int64_t kOneTileItems = 2048;  // up to here one CTA does it all, in one launch
constexpr int kMaxTiles = 148;           // one CTA per SM
constexpr int kManyExperts = 512;
constexpr int kFewTiles = 64;  // from kManyExperts on, more tiles cost more in adding up their counts than they save
                               // (262144 pairs, us with 64 and 148 tiles: 128 experts 10.9 and 9.7, 256 experts 12.2
                               // and 11.6, 1024 experts 18.4 and 22.2)
constexpr uint32_t kAll = 0xffffffffu;

struct PlanArgs {
  const void* experts;
  int64_t items, capacity, tile_items;
  int num_experts, align;
  uint32_t* tile_counts;  // [tiles][num_experts]; null: one tile, counted in place
  int32_t *counts, *offsets, *sources, *positions;
};

// No row holds a pair until one is put there: the rows between and after the
// segments are never looked for.
__device__ __forceinline__ void clear_sources(const PlanArgs& a, int64_t thread, int64_t threads) {
  for (int64_t r = thread; r < a.capacity; r += threads) a.sources[r] = -1;
}

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
  dev::wait_for_previous();
  clear_sources(a, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)gridDim.x * kThreads);
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

// The lanes whose expert is the same; `bits` to an expert.  With
// __match_any_sync, 262144 pairs took 0.8 (64 experts) to 1.1 us (128) more.
__device__ __forceinline__ uint32_t peers_of(int expert, int bits) {
  uint32_t peers = kAll;
  for (int b = 0; b < bits; ++b) {
    const bool set = expert >> b & 1;
    const uint32_t lanes = __ballot_sync(kAll, set);
    peers &= set ? lanes : ~lanes;
  }
  return peers;
}

// Exclusive scan of one value per thread; its total in *sum.  s_sums: W words.
template <int W>
__device__ __forceinline__ uint32_t scan_cta(uint32_t v, uint32_t* s_sums, uint32_t* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t in = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(kAll, in, d);
    if (lane >= d) in += o;
  }
  if (lane == 31) s_sums[warp] = in;
  __syncthreads();
  const uint32_t s = lane < W ? s_sums[lane] : 0;
  *sum = __reduce_add_sync(kAll, s);
  const uint32_t before = __reduce_add_sync(kAll, lane < warp ? s : 0);
  __syncthreads();  // s_sums may be used again
  return before + in - v;
}

// A CTA's tile in steps of THREADS * kItems items, each warp a run of them.
// In each 32 items the peers of an expert rank by their lanes, the 32s of a
// run by a counter, the runs and the steps by a scan.  The pairs of a step are
// put in their rows' order in shared memory first: a store of 32 pairs to as
// many segments takes an SM 32 times as long as one to neighbouring rows.
template <typename I, int THREADS>
__global__ void __launch_bounds__(THREADS) plan_place_kernel(PlanArgs a) {
  constexpr int W = THREADS / 32, kStep = THREADS * kItems, P = kMaxExperts / THREADS;
  extern __shared__ uint2 s_pair[];  // [kStep] (row, item)
  uint16_t* s_warp = reinterpret_cast<uint16_t*>(s_pair + kStep);  // [W][num_experts]: items of an expert in a warp's
                                                                   // run, then in the runs before
  __shared__ uint32_t s_before[kMaxExperts], s_total[kMaxExperts], s_offset[kMaxExperts], s_local[kMaxExperts], s_sums[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.num_experts;
  const int64_t begin = blockIdx.x * a.tile_items, end = min(begin + a.tile_items, a.items);
  const bool alone = a.tile_counts == nullptr;
  const int bits = 32 - __clz(E);  // E itself stands for no expert
  uint16_t* mine = s_warp + warp * E;
  dev::wait_for_previous();
  if (alone) clear_sources(a, threadIdx.x, THREADS);  // else the count kernel's part
  for (int e = threadIdx.x; e < E; e += THREADS) s_before[e] = s_total[e] = 0;

  // Segments from all tiles' counts; with one tile from its own, once they are known.
  auto segments = [&]() {
    const uint32_t al = a.align;
    uint32_t v[P], sum = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = threadIdx.x * P + j;
      v[j] = sum;
      sum += e < E ? (s_total[e] + al - 1) / al * al : 0;
    }
    uint32_t all;
    const uint32_t before = scan_cta<W>(sum, s_sums, &all);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = threadIdx.x * P + j;
      if (e < E) {
        s_offset[e] = before + v[j];
        if (blockIdx.x == 0) {
          a.counts[e] = (int32_t)s_total[e];
          a.offsets[e] = (int32_t)(before + v[j]);
        }
      }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[E] = (int32_t)all;
  };
  if (!alone) {
    // columns of the tiles' counts: as many threads to an expert as there are
    __syncthreads();
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
    __syncthreads();
    segments();
  }
  for (int64_t step = begin; step < end || (alone && step == begin); step += kStep) {
    const int64_t left = min((int64_t)kStep, end - step);
    const int rounds = (int)((left + THREADS - 1) / THREADS);  // 32s to a run
    const int64_t first = step + (int64_t)warp * rounds * 32 + lane;
    int expert[kItems];
    uint32_t at[kItems];
#pragma unroll
    for (int g = 0; g < kItems; ++g) expert[g] = g < rounds ? expert_of<I>(a, first + g * 32, end) : E;
    for (int i = threadIdx.x; i < W * E; i += THREADS) s_warp[i] = 0;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kItems; ++g) {
      if (g >= rounds) break;
      const uint32_t peers = peers_of(expert[g], bits);
      at[g] = expert[g] < E ? mine[expert[g]] + __popc(peers & dev::lanemask_lt()) : 0;
      __syncwarp();
      if (expert[g] < E && (peers >> lane) == 1u) mine[expert[g]] = (uint16_t)(at[g] + 1);  // the last peer
      __syncwarp();
    }
    __syncthreads();
    // each expert: the runs before each run, and its items in this step
    uint32_t count[P], sum = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = threadIdx.x * P + j;
      count[j] = 0;
      if (e < E) {
#pragma unroll 8
        for (int w = 0; w < W; ++w) {
          const uint32_t c = s_warp[w * E + e];
          s_warp[w * E + e] = (uint16_t)count[j];
          count[j] += c;
        }
        if (alone) s_total[e] = count[j];
      }
      sum += count[j];
    }
    uint32_t kept;
    uint32_t local = scan_cta<W>(sum, s_sums, &kept);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = threadIdx.x * P + j;
      if (e < E) s_local[e] = local;
      local += count[j];
    }
    if (alone) segments();
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kItems; ++g) {
      const int64_t i = first + g * 32;
      const int e = expert[g];
      if (g >= rounds || i >= end) break;
      uint32_t row = 0xffffffffu;
      if (e < E) {
        const uint32_t in = mine[e] + at[g];
        row = s_offset[e] + s_before[e] + in;
        s_pair[s_local[e] + in] = make_uint2(row, (uint32_t)i);
      }
      a.positions[i] = (int32_t)row;
    }
    __syncthreads();
    for (uint32_t n = threadIdx.x; n < kept; n += THREADS) {
      const uint2 p = s_pair[n];
      if (p.x < a.capacity) a.sources[p.x] = (int32_t)p.y;
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (threadIdx.x * P + j < E) s_before[threadIdx.x * P + j] += count[j];
    __syncthreads();
  }
}

struct PlanShape {
  int tiles;
  int64_t tile_items;
};

PlanShape shape_of(int64_t items, int num_experts) {
  if (items <= kOneTileItems) return {1, std::max<int64_t>(items, 1)};
  const int64_t step = (int64_t)kThreads * kItems;
  const int tiles = num_experts < kManyExperts ? kMaxTiles : kFewTiles;
  int64_t tile = std::min(step, (items + tiles - 1) / tiles);
  tile = std::max(tile, (items + kMaxTiles - 1) / kMaxTiles);
  tile = (tile + kThreads - 1) / kThreads * kThreads;
  return {(int)((items + tile - 1) / tile), tile};
}

template <typename I, int THREADS>
cudaError_t place(const PlanArgs& a, int tiles, cudaStream_t stream) {
  const size_t pairs = sizeof(uint2) * THREADS * kItems, row = sizeof(uint16_t) * (THREADS / 32);
  const size_t smem = pairs + row * a.num_experts, most = pairs + row * kMaxExperts;
  if (smem + 17 * 1024 > 48 * 1024) {  // beside the static arrays
    const cudaError_t e = cudaFuncSetAttribute(plan_place_kernel<I, THREADS>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e) return e;
  }
  return launch_after_previous(plan_place_kernel<I, THREADS>, tiles, THREADS, smem, a, stream);
}

template <typename I>
cudaError_t run(const PlanArgs& a, int tiles, cudaStream_t stream) {
  if (tiles == 1 && a.items <= kSmallItems) return place<I, kSmallThreads>(a, 1, stream);
  if (tiles > 1) {
    if (const cudaError_t e = launch_after_previous(plan_count_kernel<I>, tiles, kThreads, 0, a, stream)) return e;
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
  const PlanShape shape = shape_of(num_pairs, num_experts);
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
