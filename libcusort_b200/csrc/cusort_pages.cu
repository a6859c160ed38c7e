// cusort_pages.cu -- blocks of a paged cache after they were given out:
// requests that go on from others' (forking), blocks given back, blocks
// copied, and a pool whose used blocks are moved together.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"
#include "cusort_overlap.cuh"

namespace {

using namespace cusort_b200;

constexpr int kMaxRequests = 16384;
constexpr int kMaxWidth = 1 << 30;  // entries of a table: for_rows numbers them, and some behind the last, in 32 bits
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kSms = 148;
constexpr int kTiles = kSms;                  // of the pool, a CTA each
// One CTA does it all in shared memory while tables and pool have up to so
// many entries.  In one CTA and in a launch for each phase: freeing 200 entries
// 3.8 and 6.8 us, 5000 6.0 and 7.2, 14000 9.0 and 6.9; forking 140 entries 6.7
// and 10.0, 9200 9.5 and 9.8, 12600 12.9 and 11.7; compacting 7500 9.8 and
// 12.1, 26900 24 and 12.
constexpr int64_t kFewEntries = 1 << 13;
constexpr uint32_t kAll = 0xffffffffu;

enum Op { kFork, kFree, kCompact };

struct PagesArgs {
  const int32_t* tables;
  int64_t table_stride;
  int width, requests, block_size, num_blocks;
  const int32_t* lens;
  const int32_t* parents;  // fork: of each child
  int children;
  const int32_t* keep;                             // free: tokens that a request keeps
  const int32_t *free_blocks, *num_free, *shares;  // fork and free
  // results
  int32_t *tables_out, *lens_out, *sources, *destinations, *shares_out, *free_out, *num_free_out;
  uint8_t* served;
  // workspace
  int32_t* tile_counts;    // [kTiles] blocks that a tile of the pool adds to the list; and the blocks taken
  // compact: [num_blocks] tables that hold a block, less one; the move that a block takes part in
  int32_t *holders, *map;
  int phase;               // of the form with a launch for each
  int row_lanes, row_parts;  // see for_rows
};

// Blocks that a length needs, and those of them that the table has.
__device__ __forceinline__ int blocks_of(const PagesArgs& a, int len) {
  return (int)(((uint32_t)max(len, 0) + (uint32_t)a.block_size - 1) / (uint32_t)a.block_size);
}
__device__ __forceinline__ int held_of(const PagesArgs& a, int len) { return min(a.width, blocks_of(a, len)); }
__device__ __forceinline__ bool in_pool(const PagesArgs& a, int block) { return block >= 0 && block < a.num_blocks; }

// Sum of the CTA's values before this thread's; total: of all.
__device__ __forceinline__ int scan(int v, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int in = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(kAll, in, d);
    if (lane >= d) in += u;
  }
  if (lane == 31) sums[warp] = in;
  __syncthreads();
  const int w = sums[lane];
  total = __reduce_add_sync(kAll, w);
  const int before = __reduce_add_sync(kAll, lane < warp ? w : 0);
  __syncthreads();
  return before + in - v;
}

// Blocks at the CTA's tile of the pool: a whole number of fours to a tile.
struct Tile {
  int begin, end;
};
__device__ __forceinline__ int tile_size(const PagesArgs& a) {
  return (int)((((int64_t)a.num_blocks + gridDim.x - 1) / gridDim.x + 3) / 4 * 4);
}
__device__ __forceinline__ Tile tile_of(const PagesArgs& a, int i) {
  const int64_t size = tile_size(a);
  return {(int)min((int64_t)a.num_blocks, i * size), (int)min((int64_t)a.num_blocks, (i + 1) * size)};
}

// What is counted for each block: the tables that hold it, less one.  ONE: in
// shared memory, else in global memory, by all SMs.
template <Op OP, bool ONE> struct Holders {
  int* of;
  int* tiles;  // in shared memory: what this CTA adds to the tiles' counts
  __device__ __forceinline__ int operator[](int block) const { return ONE ? of[block] : __ldcg(of + block); }
  // Whether a block goes on the list: one that nothing holds any more (fork, free), one that is held (compact).
  __device__ __forceinline__ bool listed(int block) const { return ((*this)[block] < 0) != (OP == kCompact); }
  // Adds, and keeps count of the listed blocks of each tile: however often a block gets on the list and off it again
  // meanwhile, in whatever order, its ups and downs come to what it is at the end.  All additions are under way before
  // the first one's result is looked at.
  template <int N>
  __device__ __forceinline__ void add(const PagesArgs& a, const int (&block)[N], const int (&n)[N]) const {
    int old[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (n[i] != 0 && in_pool(a, block[i])) old[i] = atomicAdd(of + block[i], n[i]);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!ONE && n[i] != 0 && in_pool(a, block[i]) && (old[i] < 0) != (old[i] + n[i] < 0))
        atomicAdd(tiles + block[i] / tile_size(a), (old[i] + n[i] < 0) != (OP == kCompact) ? 1 : -1);
  }
};

// Listed blocks of the tiles before tile i, and of all.
template <Op OP, bool ONE>
__device__ __forceinline__ int2 counts_before(const PagesArgs& a, const Holders<OP, ONE>& h, int i, int* sums) {
  int total = 0, unused;
  if (ONE) {
    int n = 0;
    for (int b = threadIdx.x; b < a.num_blocks; b += kThreads) n += h.listed(b);
    scan(n, sums, total);
    return make_int2(0, total);
  }
  const int mine = threadIdx.x < gridDim.x ? __ldcg(a.tile_counts + threadIdx.x) : 0;
  scan(mine, sums, total);
  scan(threadIdx.x < i ? mine : 0, sums, unused);
  return make_int2(unused, total);
}

// f(row, entries) for every thread's shares of the rows: kEach entries each, of which those below the width are any.
// A long row is shared by several warps, several short ones by a warp.
constexpr int kEach = 4;
template <typename F>
__device__ __forceinline__ void for_rows(const PagesArgs& a, int rows, F&& f) {
  const int shift = __ffs(a.row_lanes) - 1, lane = threadIdx.x & (a.row_lanes - 1);
  const int64_t all = gridDim.x * kThreads >> shift, units = (int64_t)rows * a.row_parts;
  for (int64_t u = (blockIdx.x * kThreads + threadIdx.x) >> shift; u < units; u += all) {
    // a long division where it has to be
    const int r = units <= INT32_MAX ? (int)((uint32_t)u / (uint32_t)a.row_parts) : (int)(u / a.row_parts);
    const int first = (int)(u - (int64_t)r * a.row_parts) * a.row_lanes * kEach + lane;
    int at[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) at[i] = first + i * a.row_lanes;
    f(r, at);
  }
}

// Of the num_free first free blocks, within the list.
__device__ __forceinline__ int free_of(const PagesArgs& a) { return min(max(*a.num_free, 0), a.num_blocks); }

// ------------------------------------------------------------------ forking

// Every CTA works the children out for itself (they are few): for a request
// its first child and the number of children that are served, for a child the
// number of blocks taken before its own.
struct Children {
  int *first, *count;  // [requests]; the count above two bits: kPart, kStays
  int* rank;           // [children] blocks taken before; -1: takes none, -2: no parent or not served
};
constexpr int kPart = 2;   // the request's last block is part-filled
constexpr int kStays = 1;  // and its first child keeps it: no other table holds it

// What is read first is on its way before anything else: a chain of a length,
// a table's entry and its shares beside that of the parents.
__device__ __forceinline__ int plan_children(const PagesArgs& a, const Children& c, int* sums) {
  const int t = threadIdx.x;
  const int parent0 = t < a.children ? a.parents[t] : -1, len0 = t < a.requests ? a.lens[t] : 0, left = free_of(a);
  for (int p = t; p < a.requests; p += kThreads) c.first[p] = a.children;
  __syncthreads();
  for (int p = t; p < a.requests; p += kThreads) {
    const int len = p == t ? len0 : a.lens[p], blocks = blocks_of(a, len);
    int bits = 0;
    if (len > 0 && len % a.block_size != 0 && blocks <= a.width) {
      const int last = a.tables[p * a.table_stride + blocks - 1];
      bits = in_pool(a, last) && a.shares[last] == 0 ? kPart | kStays : kPart;
    }
    c.count[p] = bits;
  }
  for (int r = t; r < a.children; r += kThreads) {
    const int p = r == t ? parent0 : a.parents[r];
    if (p >= 0 && p < a.requests) atomicMin(c.first + p, r);
  }
  __syncthreads();
  int taken = 0;
  for (int r0 = 0; r0 < a.children; r0 += kThreads) {
    const int r = r0 + t, p = r0 == 0 ? parent0 : r < a.children ? a.parents[r] : -1;
    const bool valid = p >= 0 && p < a.requests;
    bool need = false;
    if (valid) {
      const int bits = c.count[p] & (kPart | kStays);
      need = bits == kPart || (bits != 0 && c.first[p] != r);
    }
    int total;
    const int rank = taken + scan(need, sums, total);
    taken += total;
    if (r < a.children) {
      const bool ok = valid && (!need || rank < left);
      c.rank[r] = !ok ? -2 : need ? rank : -1;
      if (ok) atomicAdd(c.count + p, 4);
    }
  }
  __syncthreads();
  return min(taken, left);
}

// The children's results, their tables, and the holders that their parents' blocks win and lose.
template <bool ONE>
__device__ __forceinline__ void fork_tables(const PagesArgs& a, const Children& c, const Holders<kFork, ONE>& h) {
  const int left = free_of(a), me = blockIdx.x * kThreads + threadIdx.x, all = gridDim.x * kThreads;
  for (int r = me; r < a.children; r += all) {
    const int rank = c.rank[r], p = a.parents[r];
    const bool valid = p >= 0 && p < a.requests;
    const int len = rank == -2 ? 0 : max(a.lens[p], 0);
    a.lens_out[r] = len;
    a.sources[r] = rank >= 0 ? a.tables[p * a.table_stride + blocks_of(a, len) - 1] : -1;
    a.destinations[r] = rank >= 0 ? a.free_blocks[left - 1 - rank] : -1;
    a.served[r] = !valid || rank != -2;
  }
  for_rows(a, a.children, [&](int r, const int (&at)[kEach]) {
    const int rank = c.rank[r], p = rank == -2 ? 0 : a.parents[r], held = rank == -2 ? 0 : held_of(a, a.lens[p]);
    const int32_t* from = a.tables + p * a.table_stride;
    int32_t* to = a.tables_out + (int64_t)r * a.width;
    int block[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      block[i] = at[i] >= held ? -1 : rank >= 0 && at[i] == held - 1 ? a.free_blocks[left - 1 - rank] : from[at[i]];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (at[i] < a.width) to[at[i]] = block[i];
  });
  for_rows(a, a.requests, [&](int p, const int (&at)[kEach]) {
    const int held = held_of(a, a.lens[p]), count = c.count[p], more = (count >> 2) - 1;
    const int32_t* from = a.tables + p * a.table_stride;
    if (more == 0 && !(count & kPart)) return;
    // what becomes of a part-filled last block
    const int last = (count & kStays) && c.first[p] < a.children ? 0 : -1;
    int block[kEach], delta[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      block[i] = at[i] < held ? from[at[i]] : -1;
      delta[i] = (count & kPart) && at[i] == held - 1 ? last : more;
    }
    h.add(a, block, delta);
  });
}

// ------------------------------------------------------------ the phases

// 0: what later phases add to is set up.
template <Op OP, bool ONE>
__device__ __forceinline__ void set_up(const PagesArgs& a, const Holders<OP, ONE>& h) {
  const int me = blockIdx.x * kThreads + threadIdx.x, all = gridDim.x * kThreads;
#pragma unroll 4
  for (int b = me; b < a.num_blocks; b += all) h.of[b] = OP == kCompact ? -1 : a.shares[b];
  if (OP == kCompact)
    for (int i = me; i < a.num_blocks / 2; i += all) a.sources[i] = a.destinations[i] = -1;
  if (!ONE && me < kTiles) a.tile_counts[me] = 0;
}

// 1: holders are counted.
template <Op OP, bool ONE>
__device__ __forceinline__ void count_holders(const PagesArgs& a, const Children& c, const Holders<OP, ONE>& h) {
  if constexpr (OP == kFork) {
    fork_tables(a, c, h);
  } else {
    for_rows(a, a.requests, [&](int r, const int (&at)[kEach]) {
      const int len = a.lens[r], held = held_of(a, len);
      const int kept = OP == kFree ? held_of(a, min(a.keep[r], len)) : 0;
      const int32_t* from = a.tables + r * a.table_stride;
      int block[kEach], n[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        n[i] = OP == kFree ? -1 : 1;
        block[i] = at[i] >= kept && at[i] < held ? from[at[i]] : -1;
      }
      h.add(a, block, n);
    });
  }
}

// 2, fork and free: the free list, and behind what is left of it the blocks that nothing holds any more.
template <Op OP, bool ONE>
__device__ __forceinline__ void write_free(const PagesArgs& a, const Holders<OP, ONE>& h, int left, int* sums) {
  const Tile t = tile_of(a, blockIdx.x);
  const int2 before = counts_before(a, h, blockIdx.x, sums);
  int at = left + before.x;
  for (int b0 = t.begin; b0 < t.end; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const bool gone = b < t.end && h.listed(b);
    int total;
    const int place = at + scan(gone, sums, total);
    at += total;
    if (gone && place < a.num_blocks) a.free_out[place] = b;
    if (gone || (ONE && b < t.end)) a.shares_out[b] = gone ? 0 : h[b];
  }
  const int end = (int)min((int64_t)a.num_blocks, (int64_t)left + before.y);
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < a.num_blocks; i += gridDim.x * kThreads)
    if (i < left || i >= end) a.free_out[i] = i < left ? a.free_blocks[i] : -1;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.num_free_out = end;
}

// 2, compact: with U used blocks, those from U on are numbered in order, and so are the holes below it.
template <bool ONE>
__device__ __forceinline__ void write_moves(const PagesArgs& a, const Holders<kCompact, ONE>& h, int* map, int* sums) {
  const Tile t = tile_of(a, blockIdx.x);
  const int2 before = counts_before(a, h, blockIdx.x, sums);
  const int used = before.y;
  // used blocks below U: those of the tiles before U's, and those of its own before it
  const int of = min((int)(used / max(tile_size(a), 1)), (int)gridDim.x - 1);
  int inside = counts_before(a, h, of, sums).x, n = 0, total;
#pragma unroll 4
  for (int b = tile_of(a, of).begin + threadIdx.x; b < used; b += kThreads) n += h.listed(b);
  scan(n, sums, total);
  inside += total;
  int at = before.x;
  for (int b0 = t.begin; b0 < t.end; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const bool in = b < t.end && h.listed(b);
    const int below = at + scan(in, sums, total);  // used blocks below b
    at += total;
    if (b < t.end && in && b >= used) {
      a.sources[below - inside] = b;
      map[b] = below - inside;
    } else if (b < t.end && !in && b < used) {
      a.destinations[b - below] = b;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.num_free_out = a.num_blocks - used;
}

// 3, compact: tables, shares and free list by the new numbers.
template <bool ONE>
__device__ __forceinline__ void renumber(const PagesArgs& a, const Holders<kCompact, ONE>& h, const int* map) {
  const int me = blockIdx.x * kThreads + threadIdx.x, all = gridDim.x * kThreads;
  const int used = a.num_blocks - __ldcg(a.num_free_out);
  const auto moved = [&](int block) { return __ldcg(a.destinations + (ONE ? map[block] : __ldcg(map + block))); };
  for_rows(a, a.requests, [&](int r, const int (&at)[kEach]) {
    const int held = held_of(a, a.lens[r]);
    const int32_t* from = a.tables + r * a.table_stride;
    int32_t* to = a.tables_out + (int64_t)r * a.width;
    int block[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) block[i] = at[i] < held ? from[at[i]] : -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (block[i] >= used && block[i] < a.num_blocks) block[i] = moved(block[i]);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (at[i] < a.width) to[at[i]] = block[i];
  });
  for (int b = me; b < a.num_blocks; b += all) {
    const int holders = h[b];
    if (b >= used) {
      a.shares_out[b] = 0;
      if (holders >= 0) a.shares_out[moved(b)] = holders;
    } else if (holders >= 0) {
      a.shares_out[b] = holders;
    }
    a.free_out[b] = b < a.num_blocks - used ? a.num_blocks - 1 - b : -1;
  }
}

// ONE: all phases, in one CTA; otherwise the phase a.phase, over any number of
// them, a launch for each.  Bound by the latency of launches (2.3 us each) and
// of dependent loads: a child's parent, its length, its last block, that
// block's shares.  256 requests of up to 545 blocks freed in 7.9 us (before the
// entries of long rows were shared among warps, four at a time to a thread:
// 18), 2048 forked in 14.6, 1024 tables of up to 273 blocks compacted in 13.5.
// One cluster of eight CTAs for all phases took 6.3 to 12.6 us where one CTA
// takes 3.8 to 9.5.
template <Op OP, bool ONE>
__global__ void __launch_bounds__(kThreads, 1) pages_kernel(const __grid_constant__ PagesArgs a) {
  extern __shared__ int s_all[];  // ONE: holders, and for compact the map; the children
  __shared__ int sums[kWarps], tiles[kTiles];
  static_assert(kWarps == 32, "scan() takes a sum to a lane");
  int* const values = ONE ? s_all : OP == kCompact ? a.holders : a.shares_out;
  int* const map = ONE ? s_all + a.num_blocks : a.map;
  int* const s_children = s_all + (ONE ? a.num_blocks : 0);
  const Children c{s_children, s_children + a.requests, s_children + 2 * a.requests};
  const Holders<OP, ONE> h{values, tiles};
  dev::wait_for_previous();
  if (ONE || a.phase == 0) set_up<OP, ONE>(a, h);
  int taken = 0;
  if (OP == kFork && (ONE || a.phase == 1)) {
    taken = plan_children(a, c, sums);
    if (!ONE && blockIdx.x == 0 && threadIdx.x == 0) a.tile_counts[kTiles] = taken;
  }
  if (OP == kFork && !ONE && a.phase == 2) taken = a.tile_counts[kTiles];
  if (ONE) __syncthreads();
  if (!ONE && a.phase == 1) {
    if (threadIdx.x < kTiles) tiles[threadIdx.x] = 0;
    __syncthreads();
  }
  if (ONE || a.phase == 1) count_holders<OP, ONE>(a, c, h);
  if (ONE || a.phase == 1) __syncthreads();
  if (!ONE && a.phase == 1 && threadIdx.x < kTiles && tiles[threadIdx.x] != 0)
    atomicAdd(a.tile_counts + threadIdx.x, tiles[threadIdx.x]);
  if constexpr (OP == kCompact) {
    if (ONE || a.phase == 2) write_moves<ONE>(a, h, map, sums);
    if (ONE) __syncthreads();
    if (ONE || a.phase == 3) renumber<ONE>(a, h, map);
  } else {
    if (ONE || a.phase == 2) write_free<OP, ONE>(a, h, free_of(a) - taken, sums);
  }
}

template <Op OP>
cudaError_t run(PagesArgs a, cudaStream_t stream) {
  const size_t children = OP == kFork ? sizeof(int) * (2 * (size_t)a.requests + a.children) : 0;
  const size_t all = children + sizeof(int) * (size_t)a.num_blocks * (OP == kCompact ? 2 : 1);
  // the limit is the kernel's, not the call's: the same one from every host thread
  constexpr size_t kMost = 226 * 1024, kPlain = 40 * 1024;
  const auto limit = [&](auto kernel, size_t smem) {
    return smem > kPlain ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost)
                         : cudaSuccess;
  };
  const int64_t entries = (int64_t)(a.requests + a.children) * a.width + a.num_blocks;
  a.row_lanes = 1;
  while (a.row_lanes < 32 && a.row_lanes * kEach < a.width) a.row_lanes *= 2;
  a.row_parts = std::max(1, (a.width + a.row_lanes * kEach - 1) / (a.row_lanes * kEach));
  if (entries <= kFewEntries && all <= kMost) {
    const cudaError_t e = limit(pages_kernel<OP, true>, all);
    return e ? e : launch_after_previous(pages_kernel<OP, true>, 1, kThreads, all, a, stream);
  }
  cudaError_t e = limit(pages_kernel<OP, false>, children);
  const int grid = (int)std::min<int64_t>(kTiles, (entries + kThreads - 1) / kThreads);
  for (a.phase = 0; !e && a.phase < (OP == kCompact ? 4 : 3); ++a.phase)
    e = launch_after_previous(pages_kernel<OP, false>, grid, kThreads, a.phase == 1 ? children : 0, a, stream);
  return e;
}

// ------------------------------------------------------------------ copying

constexpr int kCopyThreads = 128;
constexpr int kCopyPiece = 16384;  // bytes that a CTA copies at a time
constexpr int kCopyCaches = 64;    // to a launch

struct CopyArgs {
  struct Cache {
    char* data;
    int64_t stride, bytes;  // between blocks; of a block
    int pieces_before;      // in the caches before it
  } caches[kCopyCaches];
  const int32_t *sources, *destinations;
  int64_t pairs;
  int num_blocks, num_caches, pieces;  // pieces of a pair over all caches
  int groups, parts;                   // pairs p with p % groups == g in turn, the pieces of each over `parts` CTAs
};

// Pairs that are none cost a look each: a CTA looks at 128 of its pairs at a
// time and copies the blocks of those that are.  Bound by memory: 5923 blocks
// of 32 KB in four caches 263 us, 5.9 TB/s (90 % of the copy rate), 596 of 16
// KB 14 us, 5.6 TB/s.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyArgs a) {
  __shared__ int2 pairs[kCopyThreads];
  __shared__ int found;
  dev::wait_for_previous();
  const int g = blockIdx.x % a.groups, part = blockIdx.x / a.groups;
  for (int64_t p0 = 0; p0 * a.groups < a.pairs; p0 += kCopyThreads) {
    const int64_t p = (p0 + threadIdx.x) * a.groups + g;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    if (p < a.pairs) {
      const int from = a.sources[p], to = a.destinations[p];
      if (from >= 0 && from < a.num_blocks && to >= 0 && to < a.num_blocks && from != to)
        pairs[atomicAdd(&found, 1)] = make_int2(from, to);
    }
    __syncthreads();
    for (int i = 0; i < found; ++i) {
      const int2 pair = pairs[i];
      int cache = 0;
      for (int piece = part; piece < a.pieces; piece += a.parts) {
        while (cache + 1 < a.num_caches && piece >= a.caches[cache + 1].pieces_before) ++cache;
        const CopyArgs::Cache& c = a.caches[cache];
        const int64_t begin = (int64_t)(piece - c.pieces_before) * kCopyPiece;
        const int n = (int)(min((int64_t)kCopyPiece, c.bytes - begin) / (int64_t)sizeof(V));
        const V* from = reinterpret_cast<const V*>(c.data + pair.x * c.stride + begin);
        V* to = reinterpret_cast<V*>(c.data + pair.y * c.stride + begin);
        constexpr int U = 8;
        for (int j0 = threadIdx.x; j0 < n; j0 += kCopyThreads * U) {
          V v[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (j0 + u * kCopyThreads < n) v[u] = from[j0 + u * kCopyThreads];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (j0 + u * kCopyThreads < n) to[j0 + u * kCopyThreads] = v[u];
        }
      }
    }
    __syncthreads();
  }
}

bool pool_ok(int num_requests, int block_size, int64_t table_stride, int table_width, int num_blocks) {
  return num_requests >= 0 && num_requests <= kMaxRequests && block_size >= 1 && block_size <= (1 << 20) &&
         table_width >= 0 && table_width <= kMaxWidth && table_stride >= table_width && num_blocks >= 0 &&
         num_blocks <= (1 << 30);
}

// The two-phase protocol's answer: true where the call ends with *e.
bool temp_done(void* temp, size_t* bytes, size_t need, cudaError_t* e) {
  if (bytes == nullptr) {
    *e = cudaErrorInvalidValue;
    return true;
  }
  if (temp == nullptr) {
    *bytes = need;
    *e = cudaSuccess;
    return true;
  }
  *e = *bytes < need || (reinterpret_cast<uintptr_t>(temp) & 15) != 0 ? cudaErrorInvalidValue : cudaSuccess;
  return *e != cudaSuccess;
}

constexpr size_t kCountBytes = ((kTiles + 1) * sizeof(int32_t) + 15) / 16 * 16;

}  // namespace

extern "C" cudaError_t cusort_page_fork(void* d_temp_storage, size_t* temp_storage_bytes,
                                        const int32_t* d_block_tables, int64_t table_stride, int table_width,
                                        const int32_t* d_lens, int num_requests, const int32_t* d_parents,
                                        int num_children, int block_size, const int32_t* d_free_blocks,
                                        const int32_t* d_num_free, const int32_t* d_shares, int num_blocks,
                                        int32_t* d_block_tables_out, int32_t* d_lens_out, int32_t* d_sources,
                                        int32_t* d_destinations, uint8_t* d_served, int32_t* d_shares_out,
                                        int32_t* d_free_blocks_out, int32_t* d_num_free_out, cudaStream_t stream) {
  cudaError_t e;
  if (!pool_ok(num_requests, block_size, table_stride, table_width, num_blocks) || num_children < 0 ||
      num_children > kMaxRequests)
    return cudaErrorInvalidValue;
  if (temp_done(d_temp_storage, temp_storage_bytes, kCountBytes, &e)) return e;
  const bool tables = num_requests > 0 && table_width > 0;
  if ((tables && d_block_tables == nullptr) || (num_requests > 0 && d_lens == nullptr) ||
      (num_children > 0 && (d_parents == nullptr || d_lens_out == nullptr || d_sources == nullptr ||
                            d_destinations == nullptr || d_served == nullptr ||
                            (table_width > 0 && d_block_tables_out == nullptr))) ||
      (num_blocks > 0 && (d_free_blocks == nullptr || d_shares == nullptr || d_shares_out == nullptr ||
                          d_free_blocks_out == nullptr)) ||
      d_num_free == nullptr || d_num_free_out == nullptr)
    return cudaErrorInvalidValue;
  // what is read by every CTA, whenever it comes to run, must not be written meanwhile
  if (d_num_free == d_num_free_out ||
      (num_blocks > 0 && (d_free_blocks == d_free_blocks_out || d_shares == d_shares_out)) ||
      (tables && d_block_tables == d_block_tables_out) ||
      (num_children > 0 && num_requests > 0 && d_lens == d_lens_out))
    return cudaErrorInvalidValue;
  PagesArgs a{};
  a.tables = d_block_tables;
  a.table_stride = table_stride;
  a.width = table_width;
  a.requests = num_requests;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.lens = d_lens;
  a.parents = d_parents;
  a.children = num_children;
  a.free_blocks = d_free_blocks;
  a.num_free = d_num_free;
  a.shares = d_shares;
  a.tables_out = d_block_tables_out;
  a.lens_out = d_lens_out;
  a.sources = d_sources;
  a.destinations = d_destinations;
  a.served = d_served;
  a.shares_out = d_shares_out;
  a.free_out = d_free_blocks_out;
  a.num_free_out = d_num_free_out;
  a.tile_counts = static_cast<int32_t*>(d_temp_storage);
  return run<kFork>(a, stream);
}

extern "C" cudaError_t cusort_page_free(void* d_temp_storage, size_t* temp_storage_bytes,
                                        const int32_t* d_block_tables, int64_t table_stride, int table_width,
                                        const int32_t* d_lens, const int32_t* d_keep_lens, int num_requests,
                                        int block_size, const int32_t* d_free_blocks, const int32_t* d_num_free,
                                        const int32_t* d_shares, int num_blocks, int32_t* d_shares_out,
                                        int32_t* d_free_blocks_out, int32_t* d_num_free_out, cudaStream_t stream) {
  cudaError_t e;
  if (!pool_ok(num_requests, block_size, table_stride, table_width, num_blocks)) return cudaErrorInvalidValue;
  if (temp_done(d_temp_storage, temp_storage_bytes, kCountBytes, &e)) return e;
  if ((num_requests > 0 && ((table_width > 0 && d_block_tables == nullptr) || d_lens == nullptr ||
                            d_keep_lens == nullptr)) ||
      (num_blocks > 0 && (d_free_blocks == nullptr || d_shares == nullptr || d_shares_out == nullptr ||
                          d_free_blocks_out == nullptr)) ||
      d_num_free == nullptr || d_num_free_out == nullptr || d_num_free == d_num_free_out ||
      (num_blocks > 0 && (d_free_blocks == d_free_blocks_out || d_shares == d_shares_out)))
    return cudaErrorInvalidValue;
  PagesArgs a{};
  a.tables = d_block_tables;
  a.table_stride = table_stride;
  a.width = table_width;
  a.requests = num_requests;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.lens = d_lens;
  a.keep = d_keep_lens;
  a.free_blocks = d_free_blocks;
  a.num_free = d_num_free;
  a.shares = d_shares;
  a.shares_out = d_shares_out;
  a.free_out = d_free_blocks_out;
  a.num_free_out = d_num_free_out;
  a.tile_counts = static_cast<int32_t*>(d_temp_storage);
  return run<kFree>(a, stream);
}

extern "C" cudaError_t cusort_page_compact(void* d_temp_storage, size_t* temp_storage_bytes,
                                           const int32_t* d_block_tables, int64_t table_stride, int table_width,
                                           const int32_t* d_lens, int num_requests, int block_size, int num_blocks,
                                           int32_t* d_block_tables_out, int32_t* d_sources, int32_t* d_destinations,
                                           int32_t* d_shares_out, int32_t* d_free_blocks_out,
                                           int32_t* d_num_free_out, cudaStream_t stream) {
  cudaError_t e;
  if (!pool_ok(num_requests, block_size, table_stride, table_width, num_blocks)) return cudaErrorInvalidValue;
  if (temp_done(d_temp_storage, temp_storage_bytes, kCountBytes + 8 * (size_t)num_blocks, &e)) return e;
  if ((num_requests > 0 && (d_lens == nullptr || (table_width > 0 && (d_block_tables == nullptr ||
                                                                     d_block_tables_out == nullptr ||
                                                                     d_block_tables == d_block_tables_out)))) ||
      (num_blocks > 1 && (d_sources == nullptr || d_destinations == nullptr)) ||
      (num_blocks > 0 && (d_shares_out == nullptr || d_free_blocks_out == nullptr)) || d_num_free_out == nullptr)
    return cudaErrorInvalidValue;
  PagesArgs a{};
  a.tables = d_block_tables;
  a.table_stride = table_stride;
  a.width = table_width;
  a.requests = num_requests;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.lens = d_lens;
  a.tables_out = d_block_tables_out;
  a.sources = d_sources;
  a.destinations = d_destinations;
  a.shares_out = d_shares_out;
  a.free_out = d_free_blocks_out;
  a.num_free_out = d_num_free_out;
  a.tile_counts = static_cast<int32_t*>(d_temp_storage);
  a.holders = reinterpret_cast<int32_t*>(static_cast<char*>(d_temp_storage) + kCountBytes);
  a.map = a.holders + num_blocks;
  return run<kCompact>(a, stream);
}

extern "C" cudaError_t cusort_page_copy(void* const* d_caches, const int64_t* block_strides, const size_t* block_bytes,
                                        int num_caches, int num_blocks, const int32_t* d_sources,
                                        const int32_t* d_destinations, int64_t num_pairs, cudaStream_t stream) {
  if (num_caches < 0 || num_blocks < 0 || num_pairs < 0 || num_pairs > INT32_MAX ||
      (num_caches > 0 && (d_caches == nullptr || block_strides == nullptr || block_bytes == nullptr)) ||
      (num_pairs > 0 && (d_sources == nullptr || d_destinations == nullptr)))
    return cudaErrorInvalidValue;
  for (int c = 0; c < num_caches; ++c)
    if ((block_bytes[c] > 0 && num_blocks > 0 && d_caches[c] == nullptr) || block_bytes[c] > (size_t)1 << 40 ||
        (num_blocks > 1 && block_strides[c] < (int64_t)block_bytes[c]))
      return cudaErrorInvalidValue;
  if (num_pairs == 0 || num_blocks < 2) return cudaSuccess;
  for (int c = 0; c < num_caches;) {
    CopyArgs a{};
    a.sources = d_sources;
    a.destinations = d_destinations;
    a.pairs = num_pairs;
    a.num_blocks = num_blocks;
    uintptr_t bits = 0;
    int64_t pieces = 0;
    for (; c < num_caches && a.num_caches < kCopyCaches; ++c) {
      if (block_bytes[c] == 0) continue;
      const int64_t of = ((int64_t)block_bytes[c] + kCopyPiece - 1) / kCopyPiece;
      if (pieces + of > INT32_MAX) {
        if (pieces == 0) return cudaErrorInvalidValue;
        break;
      }
      a.caches[a.num_caches++] = {static_cast<char*>(d_caches[c]), block_strides[c], (int64_t)block_bytes[c],
                                  (int)pieces};
      pieces += of;
      bits |= reinterpret_cast<uintptr_t>(d_caches[c]) | (uintptr_t)block_strides[c] | (uintptr_t)block_bytes[c];
    }
    if (pieces == 0) continue;
    a.pieces = (int)pieces;
    // every pair has its CTAs where there are few, every CTA several pairs where there are many
    constexpr int64_t kCtas = kSms * 12;
    a.groups = (int)std::min<int64_t>(num_pairs, kCtas);
    a.parts = (int)std::min<int64_t>(pieces, std::max<int64_t>(1, kCtas / a.groups));
    const int64_t grid = (int64_t)a.groups * a.parts;
    const auto copy = [&](auto kernel) { return launch_after_previous(kernel, grid, kCopyThreads, 0, a, stream); };
    const cudaError_t e = (bits & 15) == 0  ? copy(copy_kernel<uint4>)
                          : (bits & 7) == 0 ? copy(copy_kernel<uint2>)
                          : (bits & 3) == 0 ? copy(copy_kernel<uint32_t>)
                          : (bits & 1) == 0 ? copy(copy_kernel<uint16_t>)
                                            : copy(copy_kernel<uint8_t>);
    if (e) return e;
  }
  return cudaSuccess;
}
