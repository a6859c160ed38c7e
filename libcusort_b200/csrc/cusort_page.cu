// cusort_page.cu -- one serving step's placement in a paged cache, from the
// requests' lengths: new blocks from the free list, block tables, and a slot
// and position for every new token.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/cusort_b200.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 16384;  // two 32-bit scans of them fit in shared memory
constexpr uint32_t kAll = 0xffffffffu;
constexpr uint32_t kMost = 0x7fffffffu;

struct PageArgs {
  const int32_t *cached, *fresh;  // tokens in the cache, tokens of this step
  int num_requests, block_size, num_blocks;  // num_blocks: length of the free list
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

struct Request {
  uint32_t cached, fresh, need;  // need: blocks to be taken from the free list
  bool fits;
};

__device__ __forceinline__ Request request_of(const PageArgs& a, int r) {
  Request q;
  q.cached = (uint32_t)max(a.cached[r], 0);
  q.fresh = (uint32_t)max(a.fresh[r], 0);
  const uint32_t b = a.block_size, held = (q.cached + b - 1) / b, end = (q.cached + q.fresh + b - 1) / b;
  q.fits = q.cached + q.fresh <= kMost && end <= (uint32_t)a.table_width;
  q.need = q.fits && a.num_free != nullptr ? end - held : 0;
  return q;
}

// Every CTA scans all requests (they are few), then takes its share of the
// tokens: a search for the token's request, and its block from the table or,
// for a block of this step, straight from the free list, so that no CTA waits
// for another's table entries.  A block's first token writes its entry.
__global__ void __launch_bounds__(kThreads) page_plan_kernel(PageArgs a) {
  extern __shared__ uint32_t s_scan[];  // [R + 1] token starts, [R + 1] blocks taken before
  __shared__ uint32_t s_sums[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = a.num_requests;
  uint32_t *s_start = s_scan, *s_taken = s_scan + R + 1;
  const int each = (R + kThreads - 1) / kThreads, r0 = threadIdx.x * each, r1 = min(r0 + each, R);
  uint32_t tokens = 0, blocks = 0;
  for (int r = r0; r < r1; ++r) {
    const Request q = request_of(a, r);
    s_start[r] = tokens;
    s_taken[r] = blocks;
    tokens = add_sat(tokens, q.fresh);
    blocks = add_sat(blocks, q.need);
  }
  uint32_t in_t = tokens, in_b = blocks;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t t = __shfl_up_sync(kAll, in_t, d), b = __shfl_up_sync(kAll, in_b, d);
    if (lane >= d) in_t = add_sat(in_t, t), in_b = add_sat(in_b, b);
  }
  uint32_t before_t = __shfl_up_sync(kAll, in_t, 1), before_b = __shfl_up_sync(kAll, in_b, 1);
  if (lane == 0) before_t = before_b = 0;
  if (lane == 31) s_sums[0][warp] = in_t, s_sums[1][warp] = in_b;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before_t = add_sat(before_t, s_sums[0][w]), before_b = add_sat(before_b, s_sums[1][w]);
  for (int r = r0; r < r1; ++r) {
    s_start[r] = add_sat(s_start[r], before_t);
    s_taken[r] = add_sat(s_taken[r], before_b);
  }
  if (threadIdx.x == kThreads - 1) {
    s_start[R] = add_sat(before_t, tokens);
    s_taken[R] = add_sat(before_b, blocks);
  }
  __syncthreads();
  const uint32_t left = a.num_free == nullptr ? 0u : (uint32_t)min(max(*a.num_free, 0), a.num_blocks);
  if (blockIdx.x == 0) {
    uint32_t used = 0;
    for (int r = threadIdx.x; r < R; r += kThreads) {
      const Request q = request_of(a, r);
      const uint32_t upto = s_taken[r + 1];
      a.served[r] = q.fits && (q.need == 0 || upto <= left);
      if (upto <= left) used = max(used, upto);
    }
    for (int r = threadIdx.x; r <= R; r += kThreads) a.starts[r] = (int32_t)s_start[r];
    used = __reduce_max_sync(kAll, used);
    __syncthreads();
    if (lane == 0) s_sums[0][warp] = used;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kThreads / 32; ++w) used = max(used, s_sums[0][w]);
      if (a.num_free_out != nullptr) *a.num_free_out = (int32_t)(left - used);
    }
  }
  const int64_t total = s_start[R], most = max(total, a.num_tokens);
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < most; i += (int64_t)gridDim.x * kThreads) {
    int64_t slot = -1;
    int32_t position = -1;
    if (i < total) {
      int lo = 0, hi = R;  // the last request that starts at or before i
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= i) lo = mid; else hi = mid;
      }
      const Request q = request_of(a, lo);
      const uint32_t pos = min(q.cached + (uint32_t)(i - s_start[lo]), kMost);
      position = (int32_t)pos;
      if (q.fits && (q.need == 0 || s_taken[lo + 1] <= left)) {
        const uint32_t b = a.block_size, page = pos / b, in = pos - page * b, held = (q.cached + b - 1) / b;
        int32_t* entry = a.tables + lo * a.table_stride + page;
        int32_t id;
        if (a.num_free != nullptr && page >= held) {
          id = a.free_blocks[left - 1 - (s_taken[lo] + page - held)];
          if (in == 0) *entry = id;
        } else {
          id = *entry;
        }
        if (id >= 0) slot = (int64_t)id * b + in;
      }
    }
    if (i < a.num_tokens) {
      a.slots[i] = slot;
      a.positions[i] = position;
    }
  }
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
  const PageArgs a{d_cached_lens, d_new_lens, num_requests, block_size, num_blocks, num_tokens, d_block_tables,
                   table_stride, table_width, d_free_blocks, d_num_free, d_slots, d_positions, d_starts, d_served,
                   d_num_free_out};
  const size_t smem = sizeof(uint32_t) * 2 * (num_requests + 1);
  if (smem > 48 * 1024 - 1024) {
    const cudaError_t e = cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(sizeof(uint32_t) * 2 * (kMaxRequests + 1)));
    if (e) return e;
  }
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(148, (num_tokens + kThreads - 1) / kThreads));
  page_plan_kernel<<<grid, kThreads, smem, stream>>>(a);
  return cudaGetLastError();
}
