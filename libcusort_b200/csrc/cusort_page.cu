// cusort_page.cu -- one serving step's placement in a paged cache, from the
// requests' lengths: new blocks from the free list, block tables, and a slot
// and position for every new token.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"
#include "cusort_overlap.cuh"

namespace {

constexpr int kFewRequests = 512;
constexpr int64_t kFewTokens = 148 * 1024;
constexpr int kMaxRequests = 16384;  // two 32-bit scans of them fit in shared memory
constexpr uint32_t kAll = 0xffffffffu;
constexpr uint32_t kMost = 0x7fffffffu;

struct PageArgs {
  const int32_t *cached, *fresh;  // tokens in the cache, tokens of this step
  int num_requests, block_size, num_blocks;  // num_blocks: length of the free list
  unsigned long long inverse;                // of the block size, see blocks_of
  bool whole_lengths;                        // the lengths can be read four at a time
  int64_t num_tokens;
  int32_t* tables;
  int64_t table_stride;
  int table_width;
  const int32_t *free_blocks, *num_free;  // num_free null: the tables hold every block already
  int64_t* slots;
  int32_t *positions, *starts;
  uint8_t* served;
  int32_t* num_free_out;
};

// Sums stop at 2^31 - 1, so that lengths of any size keep their order.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kMost); }

// n / a.block_size for n < 2^32: the high word of n * (2^64 / size rounded up), which errs by less than n * size / 2^64.
__device__ __forceinline__ uint32_t blocks_of(const PageArgs& a, uint32_t n) {
  return a.block_size == 1 ? n : (uint32_t)__umul64hi(n, a.inverse);
}

// The sum of 32 lanes' values, each at most 2^31 - 1, up to that.
__device__ __forceinline__ uint32_t sum_sat(uint32_t v) {
  const uint64_t high = __reduce_add_sync(kAll, v >> 16), low = __reduce_add_sync(kAll, v & 0xffffu);
  return (uint32_t)min((high << 16) + low, (uint64_t)kMost);
}

struct Request {
  uint32_t cached, fresh, held, need;  // held: blocks before this step; need: blocks to be taken from the free list
  bool fits;
};

__device__ __forceinline__ Request request_of(const PageArgs& a, int32_t cached, int32_t fresh) {
  Request q;
  q.cached = (uint32_t)max(cached, 0);
  q.fresh = (uint32_t)max(fresh, 0);
  const uint32_t up = a.block_size - 1;
  q.held = blocks_of(a, q.cached + up);
  const uint32_t end = blocks_of(a, q.cached + q.fresh + up);  // of no use beyond 2^31, where the request does not fit
  q.fits = q.cached + q.fresh <= kMost && end <= (uint32_t)a.table_width;
  q.need = q.fits && a.num_free != nullptr ? end - q.held : 0;
  return q;
}
__device__ __forceinline__ Request request_of(const PageArgs& a, int r) {
  return request_of(a, a.cached[r], a.fresh[r]);
}

// The last of starts[0 .. n) that is at most i (starts[0] is), found by the
// whole warp.
__device__ __forceinline__ int warp_search(const uint32_t* starts, int n, uint32_t i, int lane) {
  int at = 0;
  while (n > 1) {
    const int step = (n + 31) >> 5, probe = lane * step;
    const int below = __popc(__ballot_sync(kAll, probe < n && starts[at + (probe < n ? probe : 0)] <= i));
    at += (below - 1) * step;
    n = min(step, n - (below - 1) * step);
  }
  return at;
}

// Every CTA scans all requests (they are few), then takes its share of the
// tokens, N consecutive ones to a thread: a search for the first one's request
// and a walk from there, the blocks from the table or, for blocks of this
// step, straight from the free list, so that no CTA waits for another's table
// entries.  A block's first token writes its entry.
//
// Bound by latency where there are few tokens (256 requests of one: 3.3 us),
// by instruction issue where there are many (1.05M tokens of 4096 requests:
// 10.6 us; 3.5 us of it are the launch and the scan; 51 % of the issue slots).
template <int THREADS, int N>
__global__ void __launch_bounds__(THREADS) page_plan_kernel(PageArgs a) {
  constexpr int W = THREADS / 32;
  extern __shared__ uint32_t s_scan[];  // [R + 1] token starts, [R + 1] blocks taken before
  __shared__ uint32_t s_sums[2][W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = a.num_requests;
  uint32_t *s_start = s_scan, *s_taken = s_scan + R + 1;
  cusort_b200::dev::wait_for_previous();
  uint32_t sum_t = 0, sum_b = 0;  // of the requests so far
  for (int base = 0; base < R; base += THREADS * 4) {
    const int r0 = base + threadIdx.x * 4;
    int32_t cached[4], fresh[4];
    if (a.whole_lengths && r0 + 4 <= R) {
      *reinterpret_cast<int4*>(cached) = *reinterpret_cast<const int4*>(a.cached + r0);
      *reinterpret_cast<int4*>(fresh) = *reinterpret_cast<const int4*>(a.fresh + r0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cached[j] = r0 + j < R ? a.cached[r0 + j] : 0;
        fresh[j] = r0 + j < R ? a.fresh[r0 + j] : 0;
      }
    }
    uint32_t tokens[4], blocks[4], in_t = 0, in_b = 0;  // before each of the four, then of all
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Request q = request_of(a, cached[j], fresh[j]);
      tokens[j] = in_t;
      blocks[j] = in_b;
      in_t = add_sat(in_t, q.fresh);
      in_b = add_sat(in_b, q.need);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t t = __shfl_up_sync(kAll, in_t, d), b = __shfl_up_sync(kAll, in_b, d);
      if (lane >= d) in_t = add_sat(in_t, t), in_b = add_sat(in_b, b);
    }
    if (lane == 31) s_sums[0][warp] = in_t, s_sums[1][warp] = in_b;
    uint32_t before_t = __shfl_up_sync(kAll, in_t, 1), before_b = __shfl_up_sync(kAll, in_b, 1);
    if (lane == 0) before_t = before_b = 0;
    __syncthreads();
    const uint32_t warp_t = lane < W ? s_sums[0][lane] : 0, warp_b = lane < W ? s_sums[1][lane] : 0;
    before_t = add_sat(add_sat(before_t, sum_t), sum_sat(lane < warp ? warp_t : 0));
    before_b = add_sat(add_sat(before_b, sum_b), sum_sat(lane < warp ? warp_b : 0));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r0 + j < R) {
        s_start[r0 + j] = add_sat(before_t, tokens[j]);
        s_taken[r0 + j] = add_sat(before_b, blocks[j]);
      }
    }
    sum_t = add_sat(sum_t, sum_sat(warp_t));
    sum_b = add_sat(sum_b, sum_sat(warp_b));
    __syncthreads();
  }
  if (threadIdx.x == 0) s_start[R] = sum_t, s_taken[R] = sum_b;
  __syncthreads();
  const uint32_t left = a.num_free == nullptr ? 0u : (uint32_t)min(max(*a.num_free, 0), a.num_blocks);
  const uint32_t room = (uint32_t)a.num_tokens;  // below 2^31, and a step of the grid fits beside it
  for (int r = blockIdx.x * THREADS + threadIdx.x; r <= R; r += gridDim.x * THREADS) {
    a.starts[r] = (int32_t)s_start[r];
    const uint32_t taken = s_taken[r];
    // the requests before r got their blocks, and r is the first that did not
    if (a.num_free_out != nullptr && taken <= left && (r == R || s_taken[r + 1] > left))
      *a.num_free_out = (int32_t)(left - taken);
    if (r < R) {
      const Request q = request_of(a, r);
      const bool served = q.fits && (q.need == 0 || s_taken[r + 1] <= left);
      a.served[r] = served;
      // blocks whose first token lies beyond the slot map, where no token's thread comes by
      if (served && s_start[r + 1] > room) {
        for (uint32_t n = 0; n < q.need; ++n)
          if (s_start[r] + ((q.held + n) * a.block_size - q.cached) >= room)
            a.tables[r * a.table_stride + q.held + n] = a.free_blocks[left - 1 - (taken + n)];
      }
    }
  }
  const uint32_t total = s_start[R];
  const uint32_t size = a.block_size;
  for (uint32_t w0 = (blockIdx.x * THREADS + warp * 32) * N; w0 < room; w0 += gridDim.x * THREADS * N) {
    const uint32_t i0 = w0 + lane * N;
    int64_t slot[N];
    int32_t position[N];
    // the last request that starts at or before i0: the warp's first one by all of its lanes, then each lane from
    // there to the warp's last one
    int r = 0;
    if (w0 < total) {
      r = warp_search(s_start, R, w0, lane);
      int hi = r + 1 + warp_search(s_start + r, R - r, min(w0 + 32 * N, total) - 1, lane);
      while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (s_start[mid] <= i0) r = mid; else hi = mid;
      }
    }
    uint32_t next = 0, pos = 0, page = 0, in = 0, held = 0, taken = 0;
    int32_t* table = nullptr;
    int32_t id = -1;
    bool served = false, fetch = true;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t i = i0 + n;
      slot[n] = position[n] = -1;
      if (i >= total) continue;
      if (n == 0 || i >= next) {
        while (n > 0 && s_start[r + 1] <= i) ++r;
        const Request q = request_of(a, r);
        next = s_start[r + 1];
        taken = s_taken[r];
        pos = min(q.cached + (i - s_start[r]), kMost);
        page = blocks_of(a, pos);
        in = pos - page * size;
        held = a.num_free != nullptr ? q.held : (uint32_t)a.table_width;
        served = q.fits && (q.need == 0 || s_taken[r + 1] <= left);
        table = a.tables + r * a.table_stride;
        fetch = true;
      } else {
        pos = min(pos + 1, kMost);
        if (++in == size) in = 0, ++page, fetch = true;
      }
      position[n] = (int32_t)pos;
      if (!served) continue;
      if (fetch) {
        id = page < held ? table[page] : a.free_blocks[left - 1 - (taken + page - held)];
        if (page >= held && in == 0) table[page] = id;
        fetch = false;
      }
      if (id >= 0) slot[n] = (int64_t)id * size + in;
    }
    if (N == 4 && i0 + N <= room) {
      longlong2* out = reinterpret_cast<longlong2*>(a.slots + i0);
      out[0] = make_longlong2(slot[0], slot[1 % N]);
      out[1] = make_longlong2(slot[2 % N], slot[3 % N]);
      *reinterpret_cast<int4*>(a.positions + i0) =
          make_int4(position[0], position[1 % N], position[2 % N], position[3 % N]);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (i0 + n < room) {
          a.slots[i0 + n] = slot[n];
          a.positions[i0 + n] = position[n];
        }
      }
    }
  }
}

template <int THREADS, int N>
cudaError_t run(const PageArgs& a, cudaStream_t stream) {
  const size_t smem = sizeof(uint32_t) * 2 * (a.num_requests + 1), most = sizeof(uint32_t) * 2 * (kMaxRequests + 1);
  if (smem > 47 * 1024) {  // beside the sums
    // the limit is the kernel's, not the call's: the same one from every host thread
    const cudaError_t e = cudaFuncSetAttribute(page_plan_kernel<THREADS, N>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e) return e;
  }
  const int64_t per_cta = THREADS * N;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(148, (a.num_tokens + per_cta - 1) / per_cta));
  return cusort_b200::launch_after_previous(page_plan_kernel<THREADS, N>, grid, THREADS, smem, a, stream);
}

}  // namespace

extern "C" cudaError_t cusort_page_plan(const int32_t* d_cached_lens, const int32_t* d_new_lens, int num_requests,
                                        int block_size, int32_t* d_block_tables, int64_t table_stride,
                                        int table_width, const int32_t* d_free_blocks, int num_blocks,
                                        const int32_t* d_num_free, int64_t num_tokens, int64_t* d_slots,
                                        int32_t* d_positions, int32_t* d_starts, uint8_t* d_served,
                                        int32_t* d_num_free_out, cudaStream_t stream) {
  if (num_requests < 0 || num_requests > kMaxRequests || block_size < 1 || block_size > (1 << 20) ||
      table_width < 0 || table_stride < table_width || num_blocks < 0 || num_blocks > (1 << 30) || num_tokens < 0 || num_tokens > INT32_MAX)
    return cudaErrorInvalidValue;
  if ((d_num_free == nullptr ? d_free_blocks != nullptr
                             : d_num_free_out == nullptr || (num_blocks > 0 && d_free_blocks == nullptr)) ||
      d_starts == nullptr ||
      (num_requests > 0 && (d_cached_lens == nullptr || d_new_lens == nullptr || d_served == nullptr ||
                            (table_width > 0 && d_block_tables == nullptr))) ||
      (num_tokens > 0 && (d_slots == nullptr || d_positions == nullptr)))
    return cudaErrorInvalidValue;
  // every CTA reads the count, whenever it comes to run, and one writes what is left
  if (d_num_free != nullptr && d_num_free == d_num_free_out) return cudaErrorInvalidValue;
  const bool whole =
      ((reinterpret_cast<uintptr_t>(d_cached_lens) | reinterpret_cast<uintptr_t>(d_new_lens)) & 15) == 0;
  const unsigned long long inverse = block_size == 1 ? 0 : ~0ull / block_size + 1;
  const PageArgs a{d_cached_lens, d_new_lens, num_requests, block_size, num_blocks, inverse, whole, num_tokens, d_block_tables,
                   table_stride, table_width, d_free_blocks, d_num_free, d_slots, d_positions, d_starts, d_served,
                   d_num_free_out};
  // Four tokens to a thread need one search instead of four and whole-vector stores, but a longer chain; a large CTA
  // scans many requests faster.
  const bool aligned = ((reinterpret_cast<uintptr_t>(d_slots) | reinterpret_cast<uintptr_t>(d_positions)) & 15) == 0;
  if (num_tokens > kFewTokens && aligned) return run<1024, 4>(a, stream);
  return num_requests > kFewRequests ? run<1024, 1>(a, stream) : run<256, 1>(a, stream);
}
