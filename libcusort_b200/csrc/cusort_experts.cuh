// cusort_experts.cuh -- what the experts' products of 16-bit and of 32-bit
// operands share: the segments of a plan, and rows of none.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cusort_b200 {

constexpr int kMaxExperts = 1024;

// The products of 16-bit operands.
constexpr int kBlockK = 64;   // contracted elements to a step: one swizzle row
constexpr int kTileM = 128;   // lanes of a CTA's tensor memory
constexpr int kSumLoad = 32;  // columns of a sum that a warp reads at a time

// PAIR: tiles of 256 columns of the result, 128 in each of two CTAs, and half of the rows in each.  COLUMNS: 128, or 64
// (not by pairs): the other 64 lanes of tensor memory get products of what lies behind in shared memory, and nobody
// looks at them.
template <int BN, int COLUMNS, int STAGES, int SUB, bool PAIR> struct ProductShape {
  static_assert(COLUMNS == 128 || (COLUMNS == 64 && !PAIR), "");
  static constexpr int kRows = BN, kWeightColumns = COLUMNS, kStages = STAGES, kSub = SUB;
  static constexpr bool kPair = PAIR;
  static constexpr int kCtas = PAIR ? 2 : 1, kTile = COLUMNS * kCtas;
  static constexpr uint32_t kBytesA = COLUMNS * kBlockK * 2;
  static constexpr int kRowStep = 16 * kCtas;       // the instruction's width comes in such steps
  // A stage holds SUB steps of kBlockK, each the weights' part and then the rows'.
  static constexpr uint32_t kBytesB = BN / kCtas * kBlockK * 2, kStep = kBytesA + kBytesB, kStage = SUB * kStep;
  // Each of the two sums has the columns that are read of it, which in the form for the fewest rows are more than it
  // has rows: one that is read has no columns of the other, which grows meanwhile, nor any that were not allocated.
  static constexpr uint32_t kSumColumns = (BN + kSumLoad - 1) / kSumLoad * kSumLoad, kColumns = 2 * kSumColumns;
  static constexpr uint32_t kStaging = 4 * 2048;  // 32 x 32 16-bit elements for each storing warp
};

// Rows of a tile where no expert can have more, where experts have few on
// average, and where they have many (by pairs of CTAs).  64 experts, 2048 ->
// 1536, by the second and the third: 8 rows each 65 and 69 us, 64 71 and 75, 80
// 84 and 76, 128 89 and 80.  The rule goes by averages, since the counts stay
// on the device, and these are of experts with equal counts: a batch whose rows
// nearly all go to one expert takes tiles that are smaller than they could be.
constexpr int kProductFewestRows = 16, kProductFewRows = 64, kProductManyRows = 256;
using ProductFewestNarrow = ProductShape<kProductFewestRows, 64, 9, 2, false>;
using ProductFewest = ProductShape<kProductFewestRows, 128, 5, 2, false>;
using ProductFew = ProductShape<kProductFewRows, 128, 4, 2, false>;
using ProductMany = ProductShape<kProductManyRows, 128, 6, 1, true>;

// Expert segments as the CTA keeps them in shared memory.
struct Segments {
  int32_t* first;  // [experts] rows: clamped into [0, capacity]
  int32_t* count;
  int32_t* tiles;  // [experts + 1] sums of the tiles before each expert
};

struct SegmentArgs {
  const int32_t *counts, *offsets;
  int experts, capacity;
};

// First row and number of rows of an expert's segment, within the rows there are.
__host__ __device__ inline int2 segment(const SegmentArgs& a, int e) {
  const int offset = a.offsets[e], first = min(max(offset, 0), a.capacity);
  const int64_t end = min((int64_t)offset + a.counts[e], (int64_t)a.capacity);
  return make_int2(first, (int)max(end - first, (int64_t)0));
}

// Sums of tiles stop at 2^30, more than there are of any plan's.
__device__ __forceinline__ uint32_t add_tiles(uint32_t a, uint32_t b) { return min(a + b, 1u << 30); }

// All threads: fills s; tiles(count) is the number of tiles of an expert with
// that many rows.  Segments that do not overlap have `most` tiles at most; of
// others those that go beyond it are left out, and all after them.
template <int THREADS, typename F>
__device__ __forceinline__ void load_segments(const SegmentArgs& a, const Segments& s, uint32_t* sums, uint32_t most,
                                              F&& tiles) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kEach = (kMaxExperts + THREADS - 1) / THREADS;
  const int per = (a.experts + THREADS - 1) / THREADS;  // consecutive experts to a thread
  uint32_t mine[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x * per + i;
    mine[i] = 0;
    if (i < per && e < a.experts) {
      const int2 seg = segment(a, e);
      s.first[e] = seg.x;
      s.count[e] = seg.y;
      mine[i] = tiles(seg.y);
    }
    sum = add_tiles(sum, mine[i]);
  }
  uint32_t scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t v = __shfl_up_sync(kAll, scan, d);
    if (lane >= d) scan = add_tiles(scan, v);
  }
  if (lane == 31) sums[warp] = scan;
  if (threadIdx.x == 0) s.tiles[a.experts] = 0;
  uint32_t before = __shfl_up_sync(kAll, scan, 1);
  if (lane == 0) before = 0;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before = add_tiles(before, sums[w]);
  const uint32_t begin = before;
  uint32_t last = 0;  // the end of the last one that stays
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    before = add_tiles(before, mine[i]);
    if (before <= most) last = before;
  }
  atomicMax(s.tiles + a.experts, (int)last);
  __syncthreads();
  const uint32_t end = s.tiles[a.experts];
  before = begin;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x * per + i;
    if (i < per && e < a.experts) {
      s.tiles[e] = (int)min(before, end);
      before = add_tiles(before, mine[i]);
      if (before > end) s.count[e] = 0;
    }
  }
  __syncthreads();
}

// The expert whose tiles hold tile t.
__device__ __forceinline__ int find(const int32_t* tiles, int experts, int t) {
  int low = 0, high = experts;  // tiles[low] <= t < tiles[high]
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (tiles[mid] <= t) low = mid;
    else high = mid;
  }
  return low;
}

__device__ __forceinline__ uint32_t align_up(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// Zeros in 16-bit elements [begin, end) of x, by `threads` threads.
__device__ __forceinline__ void clear(uint16_t* x, int64_t begin, int64_t end, int thread, int threads) {
  if (begin >= end) return;
  const int64_t head = min(end, begin + (int64_t)((16 - (reinterpret_cast<uintptr_t>(x + begin) & 15)) % 16) / 2);
  const int64_t words = (end - head) / 8;
  uint4* body = reinterpret_cast<uint4*>(x + head);
  if (begin + thread < head) x[begin + thread] = 0;
#pragma unroll 4
  for (int64_t i = thread; i < words; i += threads) body[i] = make_uint4(0, 0, 0, 0);
  if (head + words * 8 + thread < end) x[head + words * 8 + thread] = 0;
}

// Where rows of no segment that begin at row r end, by experts e0, e0 + step and
// so on: at the segment that begins next, the capacity where none does, r itself
// where a segment covers it.
__host__ __device__ inline int no_segment_until(const Segments& s, int experts, int capacity, int r, int e0, int step) {
  int until = capacity;
  for (int e = e0; e < experts; e += step)
    if (s.count[e] > 0 && s.first[e] + s.count[e] > r) {
      const int begin = s.first[e] > r ? s.first[e] : r;
      until = begin < until ? begin : until;
    }
  return until;
}
// Where the last segment ends, by the same experts.
__host__ __device__ inline int segments_end(const Segments& s, int experts, int e0, int step) {
  int end = 0;
  for (int e = e0; e < experts; e += step)
    if (s.count[e] > 0 && s.first[e] + s.count[e] > end) end = s.first[e] + s.count[e];
  return end;
}

// f(begin, end) for part `me` of `all` of the rows that belong to no segment:
// those behind a segment by its expert, whatever the segments' order, those
// behind the last one in equal parts.  Each of the lanes of a warp looks at its
// share of the experts for what comes next.
#pragma nv_exec_check_disable
template <typename Lanes, typename F>
__host__ __device__ inline void other_rows(const Segments& s, int experts, int capacity, int me, int all,
                                           const Lanes& lanes, F&& f) {
  const int end = lanes.highest(segments_end(s, experts, lanes.lane, lanes.count));
  for (int e = me; e <= experts; e += all) {  // the last: before the first segment
    if (e < experts && s.count[e] == 0) continue;
    const int r = e < experts ? s.first[e] + s.count[e] : 0;
    if (r < end) f(r, lanes.lowest(no_segment_until(s, experts, capacity, r, lanes.lane, lanes.count)));
  }
  const int64_t left = capacity - end, per = (left + all - 1) / all, part = me * per;
  if (part < left) f((int)(end + part), (int)(part + per < left ? end + part + per : capacity));
}

struct WarpLanes {
  int lane, count = 32;
  __device__ __forceinline__ int highest(int v) const { return __reduce_max_sync(0xffffffffu, v); }
  __device__ __forceinline__ int lowest(int v) const { return __reduce_min_sync(0xffffffffu, v); }
};

// One warp's part in clearing the rows that belong to no segment (16-bit
// elements, `width` to a row; warp `me` of `all`).
__device__ __forceinline__ void clear_other_rows(uint16_t* out, int64_t width, const SegmentArgs& a, const Segments& s,
                                                 int me, int all) {
  const WarpLanes lanes{(int)(threadIdx.x & 31)};
  other_rows(s, a.experts, a.capacity, me, all, lanes,
             [&](int begin, int end) { clear(out, begin * width, end * width, lanes.lane, 32); });
}

// The products of 32-bit operands (cusort_experts_f32.cu).
// out[r] = rows[r] x weights[e], element (i, o) of them i * in_stride + o * out_stride behind their start.
cudaError_t float_products(const float* rows, int64_t row_stride, const float* weights, int64_t expert_stride,
                           int64_t in_stride, int64_t out_stride, const SegmentArgs& segments, float* out, int in,
                           int width, cudaStream_t stream);
// grad[e] = slow_e^T x fast_e, [experts][slow_width][fast_width].
cudaError_t float_products_grad(const float* slow, int64_t slow_stride, const float* fast, int64_t fast_stride,
                                const SegmentArgs& segments, float* grad, int slow_width, int fast_width,
                                cudaStream_t stream);

}  // namespace cusort_b200
