// cusort_experts.cu -- the experts' matrix products: every row of a segment
// times its expert's weights, and the gradient of the weights.  (The gradient
// of the rows is the product with the weights' other order.)  16-bit operands
// here, on the tensor cores; 32-bit ones in cusort_experts_f32.cu.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <type_traits>
#include <utility>

#include "../../include/cusort_b200.h"
#include "cusort_dispatch.h"
#include "cusort_experts.cuh"
#include "cusort_float.cuh"
#include "cusort_overlap.cuh"
#include "cusort_tensor.cuh"

namespace cusort_b200 {

cudaError_t encode_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                       const uint32_t* box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};
  Encode encode = known.load();
  if (encode == nullptr) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || f == nullptr)
      return e != cudaSuccess ? e : cudaErrorNotSupported;
    known = encode = reinterpret_cast<Encode>(f);
  }
  cuuint64_t d[3], s[2];
  cuuint32_t b[3], one[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = dims[i], b[i] = box[i];
  for (int i = 0; i + 1 < rank; ++i) s[i] = strides[i];
  // both types have 16 bits, and nothing but zeros outside depends on which it is
  const auto call = [&] {
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), d, s, b, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE,
                  box[0] == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = call();
  if (r != CUDA_SUCCESS) {
    // a host thread that has made no call of the runtime yet (as one that runs a backward pass) has no context
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (!e) e = cudaSetDevice(device);
    if (e) return e;
    r = call();
  }
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace cusort_b200

namespace {

using namespace cusort_b200;

constexpr int kThreads = 320;  // warps 0, 2, 8 and 9 bring operands, 1 multiplies, 3 clears rows, 4 to 7 store
constexpr int kSms = 148;
constexpr uint32_t kBoxBytes = kBlockK * dev::kBoxRowBytes;  // 64 rows of 64 elements
constexpr uint32_t kAll = 0xffffffffu;

// CTAs that gave up waiting (a bounded wait ran out), and how many of them were
// told: what comes between a reader's look and its answer stays for the next one.
__device__ uint32_t g_lost[2];

constexpr int kEnds = 4;  // buffers for the ends of segments, in the gradient of the weights

// Barriers and flags of one CTA.  PAIR: two CTAs work on one tile, each with
// half of either operand; the first one multiplies.
template <int STAGES, bool PAIR> struct Pipe {
  uint64_t full[STAGES];   // a stage's copies are there; those of both CTAs count on the first one's barrier
  uint64_t empty[STAGES];  // a stage was multiplied
  // the same of the buffers for the ends of segments, of this CTA alone; in the first of two CTAs: both have cleared
  // what lies behind the end; multiplied
  uint64_t end_full[kEnds], end_cleared[kEnds], end_empty[kEnds];
  uint64_t sum_full[2], sum_empty[2];
  uint32_t tmem, gave_up, sums[kThreads / 32];
};

// The barriers' addresses.
template <int STAGES, bool PAIR> struct PipeAt {
  using P = Pipe<STAGES, PAIR>;
  uint32_t base;
  __device__ __forceinline__ explicit PipeAt(const P& p) : base(dev::smem_u32(&p)) {}
  __device__ __forceinline__ uint32_t full(int i) const { return base + offsetof(P, full) + 8 * i; }
  __device__ __forceinline__ uint32_t empty(int i) const { return base + offsetof(P, empty) + 8 * i; }
  __device__ __forceinline__ uint32_t end_full(int i) const { return base + offsetof(P, end_full) + 8 * i; }
  __device__ __forceinline__ uint32_t end_cleared(int i) const { return base + offsetof(P, end_cleared) + 8 * i; }
  __device__ __forceinline__ uint32_t end_empty(int i) const { return base + offsetof(P, end_empty) + 8 * i; }
  __device__ __forceinline__ uint32_t sum_full(int i) const { return base + offsetof(P, sum_full) + 8 * i; }
  __device__ __forceinline__ uint32_t sum_empty(int i) const { return base + offsetof(P, sum_empty) + 8 * i; }
  // The storing warps have read a sum: one lane says so.
  __device__ __forceinline__ void release_sum(int i) const {
    if (PAIR) dev::arrive_first(sum_empty(i));
    else dev::arrive(sum_empty(i));
  }
};

template <int STAGES, bool PAIR>
__device__ __forceinline__ void init_pipe(Pipe<STAGES, PAIR>& p, uint32_t columns) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      dev::mbar_init(&p.full[i], 1);
      dev::mbar_init(&p.empty[i], 1);
    }
    for (int i = 0; i < kEnds; ++i) {
      dev::mbar_init(&p.end_full[i], 1);
      dev::mbar_init(&p.end_cleared[i], 2);
      dev::mbar_init(&p.end_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) dev::mbar_init(&p.sum_full[i], 1), dev::mbar_init(&p.sum_empty[i], PAIR ? 8 : 4);
    p.gave_up = 0;
    dev::fence_mbar_init();
  }
  __syncwarp();
  if (threadIdx.x / 32 == 1) dev::tmem_alloc<PAIR>(&p.tmem, columns);
  dev::tmem_fence_before();
  if (PAIR) dev::cluster_sync();
  else __syncthreads();
  dev::tmem_fence_after();
}

// The producer's place in the ring of stages.
template <int STAGES> struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++stage == STAGES) stage = 0, parity ^= 1;
  }
};

// The end of every warp's work: tensor memory is given back.  Where a wait ran
// out, whoever's it was, copies and products may be under way that nobody waited
// for; they take microseconds and are given a millisecond.  (Where none ran out
// in one CTA of a pair, its sums were whole, so that the other one's products
// are done too.)
template <int STAGES, bool PAIR>
__device__ __forceinline__ void close_pipe(Pipe<STAGES, PAIR>& p, uint32_t columns) {
  dev::tmem_fence_before();
  __syncthreads();
  if (p.gave_up) {
    if (threadIdx.x == 0) atomicAdd(&g_lost[0], 1u);
    const uint64_t t0 = dev::globaltimer_ns();
    while (dev::globaltimer_ns() - t0 < 1000000) __nanosleep(1000);
  }
  if (PAIR) dev::cluster_sync();
  if (threadIdx.x / 32 == 1) {
    dev::tmem_fence_after();
    dev::tmem_free<PAIR>(p.tmem, columns);
  }
}

// What stands in the results in the place of two sums that a wait in vain has
// cost: NaN, in either type.  A role whose wait ran out waits and hands on no
// more, so that nobody takes a barrier's phase for another one or arrives twice
// in one: no stages are filled or multiplied any more.  Those who wait for them
// run out in turn, at once in this CTA, after their own limit in the other of a
// pair; the storing warps go on to the end.  (The roles' loops run on with
// nothing to do: left early they made a call of 8.2 us one of 8.4.)
constexpr uint32_t kLost = 0x7fff7fffu;

// A wait of a whole warp, by one lane: 32 of them keep shared memory busy.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const dev::WaitLimit& limit) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = dev::wait_for(bar, parity, limit);
  __syncwarp();
  return __shfl_sync(kAll, ok, 0);
}

// The warps that bring operands: 0 and 2 one of them, 8 and 9 the other, each
// every second step.  A thread takes some 200 cycles to issue a tiled copy,
// whatever its size: with one warp for all of them the products ran at half
// the rate, with one for each operand a step took 350 cycles.
__device__ __forceinline__ bool brings(int warp) { return warp == 0 || warp == 2 || warp >= 8; }

// ---------------------------------------------------------------- the products

struct ProductArgs {
  CUtensorMap weights, rows[3];  // the rows by boxes of 64, 32 and 16
  SegmentArgs segments;
  void* out;
  int in, width;      // of a row, and of a row of the result
  int width_tiles;    // tiles of the result's width
  uint32_t most;      // tiles of rows
  uint64_t limit_ns;  // bound on every wait
  int64_t skip;       // for tests: every CTA's step that is never brought; -1: none
};

template <typename Shape> size_t product_bytes(int experts) {
  return 1024 + Shape::kStages * Shape::kStage + Shape::kStaging + sizeof(Pipe<Shape::kStages, Shape::kPair>) +
         4 * (3 * (size_t)experts + 1);
}

struct ProductTile {
  int expert, row, rows, column;  // first row and number of rows; first column of the result
};

template <typename Shape>
__device__ __forceinline__ ProductTile product_tile(const ProductArgs& a, const Segments& s, uint32_t t) {
  ProductTile p;
  p.expert = find(s.tiles, a.segments.experts, t / a.width_tiles);
  const uint32_t before = s.tiles[p.expert], tiles = s.tiles[p.expert + 1] - before;
  const uint32_t local = t - before * a.width_tiles, count = s.count[p.expert];
  // the rows in equal tiles, whole steps of the instruction's width
  const uint32_t per = align_up((count + tiles - 1) / tiles, Shape::kRowStep), tile = local % tiles;
  p.row = s.first[p.expert] + tile * per;
  p.rows = min(per, count - tile * per);
  p.column = local / tiles * Shape::kTile;
  return p;
}

// out^T = weights^T x rows^T by tiles of 128 (PAIR: 256) of the result's
// columns (the lanes of tensor memory) and up to BN rows of one segment.  So
// the instruction's width is the number of rows, in steps of 16 (PAIR: 32): an
// expert with three rows costs a width of 16, and its weights stream through
// the lanes.  Two sums in tensor memory: one is stored while the next grows.
//
// Many rows an expert, a pair of CTAs to a tile, so that each takes in half of
// either operand: bound by what an SM takes in from L2 (32 KB to a step of 512
// cycles of the tensor cores: 51 to 57 bytes a cycle) and by the power cap.
// One expert of 8192 rows, 4096 -> 4096: 188 us, 1.46 PFLOP/s (the library's
// batched product: 184); 64 experts of 700, 2048 -> 1408: 216 us (215); of
// about 400, whose tiles are no wider than 224 rows, 129 (115).  With a CTA to
// each 128 x 256 tile: 354 us for the first.
// Few rows, a CTA to a tile, two steps of 64 to a stage: bound by memory (128
// experts with 4 rows each, 2048 -> 1536: 118 us, 6.8 TB/s), below that by how
// much of the weights each of the few CTAs has under way.  So where no expert
// can have more than 16 rows their part of a stage is small and there are five
// stages, not four, and tiles of 64 columns where that still leaves no more
// than one to an SM (six rows of six experts, 2048 -> 1024, from memory: 10.5
// us with four stages, 9.4 with five, 8.9 with half the columns; 4096 -> 1024
// 17.3, 14.7, 12.6; 4.2 us are there without any contraction).  Splitting the
// contraction over clusters of two or three CTAs took as long or longer (11.4 us
// for the first): their barriers and the joining cost what the shorter loops
// gained.
//
// The tensor cores cut what an addition leaves beyond 32 bits instead of
// rounding it: of 2048 to 4096 products' sums 0.1 to 0.2 % come to the
// neighbour of the 16-bit number nearest to the exact sum, 0.01 to 0.04 % where
// every addition is rounded; the distance from the exact sums, which that one
// rounding makes, is the same in five digits (1.65e-3 of them in bfloat16).
template <typename T, typename Shape, bool IN_ORDER>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ ProductArgs a) {
  constexpr int BN = Shape::kRows, COLUMNS = Shape::kWeightColumns, STAGES = Shape::kStages, SUB = Shape::kSub;
  constexpr bool PAIR = Shape::kPair;
  constexpr uint32_t kBytesA = Shape::kBytesA;
  extern __shared__ uint8_t raw[];
  uint8_t* base = raw + (align_up(dev::smem_u32(raw), 1024) - dev::smem_u32(raw));
  uint8_t* staging = base + STAGES * Shape::kStage;
  Pipe<STAGES, PAIR>& p = *reinterpret_cast<Pipe<STAGES, PAIR>*>(staging + Shape::kStaging);
  const int experts = a.segments.experts;
  Segments s;
  s.first = reinterpret_cast<int32_t*>(&p + 1);
  s.count = s.first + experts;
  s.tiles = s.count + experts;

  const PipeAt<STAGES, PAIR> at(p);
  const dev::WaitLimit limit{&p.gave_up, a.limit_ns};

  init_pipe(p, Shape::kColumns);
  dev::wait_for_previous();
  load_segments<kThreads>(a.segments, s, p.sums, a.most, [](int count) { return (count + BN - 1) / BN; });
  const uint32_t tiles = (uint32_t)s.tiles[experts] * a.width_tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = PAIR ? dev::cluster_rank() : 0;
  const int steps = (a.in + SUB * kBlockK - 1) / (SUB * kBlockK);
  const uint32_t t0 = blockIdx.x / Shape::kCtas, t_step = gridDim.x / Shape::kCtas;
  const uint32_t stages = dev::smem_u32(base);

  if (brings(warp)) {
    if (dev::elect_one()) {
      Ring<STAGES> ring;
      uint32_t turn = (warp == 2 || warp == 9);  // whether it takes the odd steps
      int64_t step_of_cta = -1;
      bool lost = false;
      for (uint32_t t = t0; t < tiles; t += t_step) {
        const ProductTile tile = product_tile<Shape>(a, s, t);
        const int column = tile.column + rank * kTileM;
        const int mine = align_up(tile.rows, Shape::kRowStep) / Shape::kCtas, row = tile.row + rank * mine;
        const uint32_t bytes = SUB * Shape::kCtas * (kBytesA + mine * dev::kBoxRowBytes);
        for (int k = 0; k < steps; ++k, ring.next()) {
          ++step_of_cta;
          if ((turn ^= 1) == 0 || lost) continue;
          lost = !dev::wait_for(at.empty(ring.stage), ring.parity ^ 1, limit);
          if (lost || step_of_cta == a.skip) continue;
          const uint32_t to = stages + ring.stage * Shape::kStage, own = at.full(ring.stage);
          const uint32_t bar = PAIR ? dev::in_first(own) : own;
          // the first CTA's barrier counts the copies of both
          if (warp < 8 && rank == 0) dev::arrive_expect(own, bytes);
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            const int x = (k * SUB + u) * kBlockK;
            const uint32_t step = to + u * Shape::kStep;
            if (warp >= 8) {
              // no more rows than are multiplied: what an SM takes in is what bounds the products
              int r = 0;
              for (; mine - r >= 64; r += 64)
                dev::tma_load_2d<PAIR>(step + kBytesA + r * dev::kBoxRowBytes, &a.rows[0], bar, x, row + r);
              if (mine & 32) {
                dev::tma_load_2d<PAIR>(step + kBytesA + r * dev::kBoxRowBytes, &a.rows[1], bar, x, row + r);
                r += 32;
              }
              if (mine & 16)
                dev::tma_load_2d<PAIR>(step + kBytesA + r * dev::kBoxRowBytes, &a.rows[2], bar, x, row + r);
            } else if (IN_ORDER) {
              dev::tma_load_3d<PAIR>(step, &a.weights, bar, x, column, tile.expert);
            } else {
              dev::tma_load_3d<PAIR>(step, &a.weights, bar, column, x, tile.expert);
              if (COLUMNS == 128)
                dev::tma_load_3d<PAIR>(step + kBytesA / 2, &a.weights, bar, column + kBlockK, x, tile.expert);
            }
          }
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    if (dev::elect_one()) {
      Ring<STAGES> ring;
      Ring<2> sums;
      const uint64_t first_a = dev::operand_descriptor(stages, IN_ORDER ? 16 : kBoxBytes, 1024);
      const uint64_t first_b = dev::operand_descriptor(stages + kBytesA, 16, 1024);
      bool lost = false;
      for (uint32_t t = t0; t < tiles; t += t_step, sums.next()) {
        const ProductTile tile = product_tile<Shape>(a, s, t);
        const uint32_t instruction = dev::mma_instruction(std::is_same_v<T, __nv_bfloat16>, !IN_ORDER, false,
                                                          kTileM * Shape::kCtas, align_up(tile.rows, Shape::kRowStep));
        const uint32_t sum = p.tmem + sums.stage * Shape::kSumColumns;
        lost = lost || !dev::wait_for<PAIR>(at.sum_empty(sums.stage), sums.parity ^ 1, limit);
        dev::tmem_fence_after();
        for (int k = 0; k < steps; ++k, ring.next()) {
          lost = lost || !dev::wait_for(at.full(ring.stage), ring.parity, limit);
          if (lost) continue;
          dev::tmem_fence_after();
          const uint32_t stage = ring.stage * (Shape::kStage / 16);
#pragma unroll
          for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < kBlockK / 16; ++i)
              dev::mma_issue<PAIR>(sum, first_a + stage + (u * Shape::kStep + i * (IN_ORDER ? 32 : 2048)) / 16,
                                   first_b + stage + (u * Shape::kStep + i * 32) / 16, instruction, k + u + i > 0);
          dev::mma_commit<PAIR>(at.empty(ring.stage));
        }
        if (!lost) dev::mma_commit<PAIR>(at.sum_full(sums.stage));
      }
    }
  } else if (warp == 3) {
    clear_other_rows(static_cast<uint16_t*>(a.out), a.width, a.segments, s, blockIdx.x, gridDim.x);
  } else if (warp >= 4 && warp < 8) {
    // the sums to 16 bits, through shared memory from a column of the result to a lane to a row's piece to a lane
    Ring<2> sums;
    const int quarter = warp & 3;
    uint8_t* mine = staging + quarter * 2048;
    T* out = static_cast<T*>(a.out);
    const bool whole = a.width % 8 == 0;  // the result's first byte lies on a 16-byte boundary
    bool lost = false;
    for (uint32_t t = t0; t < tiles; t += t_step, sums.next()) {
      const ProductTile tile = product_tile<Shape>(a, s, t);
      lost = lost || !warp_wait(at.sum_full(sums.stage), sums.parity, limit);
      dev::tmem_fence_after();
      const int column = tile.column + rank * kTileM + quarter * 32;
      for (int c = 0; c < tile.rows && quarter * 32 < COLUMNS; c += 32) {
        uint32_t v[32];
        dev::tmem_load32(p.tmem + sums.stage * Shape::kSumColumns + c + ((uint32_t)quarter << 21), v);
        dev::tmem_load_wait(v);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t both =
              dev::from_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]), T{}) | (lost ? kLost : 0);
          const uint32_t other = __shfl_xor_sync(kAll, both, 1);
          // even lanes: row 2j, odd ones: row 2j + 1, each of this column and its neighbour
          const uint32_t word = lane & 1 ? __byte_perm(other, both, 0x7632) : __byte_perm(both, other, 0x5410);
          *reinterpret_cast<uint32_t*>(mine + (2 * j + (lane & 1)) * 64 + (lane >> 1) * 4) = word;
        }
        __syncwarp();
        const int rows = min(32, tile.rows - c);
        const int64_t first = (int64_t)(tile.row + c);
        if (whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + lane / 4, x = column + lane % 4 * 8;
            if (row < rows && x < a.width)
              *reinterpret_cast<uint4*>(out + (first + row) * a.width + x) =
                  *reinterpret_cast<const uint4*>(mine + row * 64 + lane % 4 * 16);
          }
        } else {
          T x[32];
#pragma unroll
          for (int row = 0; row < 32; ++row) x[row] = *reinterpret_cast<const T*>(mine + row * 64 + lane * 2);
          T* to = out + first * a.width + column + lane;
          const int there = column + lane < a.width ? rows : 0;
#pragma unroll
          for (int row = 0; row < 32; ++row, to += a.width)
            if (row < there) *to = x[row];
        }
        __syncwarp();
      }
      dev::tmem_fence_before();
      __syncwarp();
      if (lane == 0 && !lost) at.release_sum(sums.stage);
    }
  }
  __syncwarp();
  close_pipe(p, Shape::kColumns);
}

// ---------------------------------------------------- the gradient of the weights

struct GradArgs {
  CUtensorMap out;         // where its rows lie on 16-byte boundaries
  // the rows whose width is the gradient's slower dimension, and those of the contiguous one; by boxes of 16 for ends
  CUtensorMap slow, fast, slow_end, fast_end;
  SegmentArgs segments;
  void* result;  // [experts][slow_width][fast_width]
  int slow_width, fast_width, slow_tiles, fast_tiles;
  uint64_t limit_ns;
  int64_t skip;
};

constexpr int kGradN = 256;
constexpr int kGradStages = 5;
constexpr uint32_t kGradStage = 4 * kBoxBytes;
constexpr uint32_t kStoreBox = 32 * 64;              // 32 rows of 32 elements, stored as one box
constexpr int kStoreBoxes = 3;                       // for each storing warp: one is filled, others are being stored
constexpr uint32_t kGradStaging = 4 * kStoreBoxes * kStoreBox;
constexpr int kChunkBytes = kBoxBytes;    // 64 contracted rows of 64 elements
constexpr int kEndRows = 16;              // contracted by one instruction
constexpr int kEndChunk = kEndRows * 128, kEndBytes = 4 * kEndChunk;

size_t grad_bytes(int experts) {
  return 1024 + kGradStages * kGradStage + kEnds * kEndBytes + kGradStaging + sizeof(Pipe<kGradStages, true>) +
         8 * (size_t)experts;
}

struct GradTile {
  int expert, slow, fast, chunks;  // first elements; 64-element chunks of the contiguous dimension in each of the CTAs
  int2 segment;
  // The segment's rows in whole instructions, by steps of kBlockK; its end, fewer than kEndRows, is one by itself.
  __device__ __forceinline__ int whole() const { return segment.y / kEndRows * kEndRows; }
  __device__ __forceinline__ int steps() const { return (whole() + kBlockK - 1) / kBlockK; }
  __device__ __forceinline__ int end() const { return segment.y % kEndRows; }
};

__device__ __forceinline__ GradTile grad_tile(const GradArgs& a, const int2* segments, uint32_t t) {
  const uint32_t per_expert = (uint32_t)a.slow_tiles * a.fast_tiles, local = t % per_expert;
  GradTile g;
  g.expert = t / per_expert;
  g.slow = local % a.slow_tiles * (2 * kTileM);
  g.fast = local / a.slow_tiles * kGradN;
  g.chunks = min(kGradN / 2, (a.fast_width - g.fast + 1) / 2 + kBlockK - 1) / kBlockK;
  g.segment = segments[g.expert];
  return g;
}

// gradient[e] = slow_e^T x fast_e, contracted over the rows of e's segment: both operands lie with the contracted
// dimension across.  Rows behind a segment's end are another expert's, or anything at all: the last fewer than 16 rows
// come by themselves, and what comes with them is cleared in shared memory.
//
// Always by pairs of CTAs.  Many rows: bound as the products are (8192 rows, 4096 x 4096: 192 us, 1.43 PFLOP/s; 32
// experts of 1024, 2048 x 4096: 395 to 400 us).  Few (128 experts of 128 rows, 2048 x 1024): 183 to 199 us, 2.7 to 2.9
// TB/s written, of which 120 are left without the stores, while a plain fill of as many bytes takes 78 to 96.  So neither
// memory nor the tensor cores (16 % busy) bound it: a sum of 256 columns a CTA is there after two steps, and then four
// warps have to read, round and stage it.  Stored by tiled copies of 64-byte rows: whole sectors straight from
// registers took 194 us where these took 181, and 271 instead of 233 where rows are 2800 bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    grad_weights_kernel(const __grid_constant__ GradArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* base = raw + (align_up(dev::smem_u32(raw), 1024) - dev::smem_u32(raw));
  uint8_t* ends = base + kGradStages * kGradStage;
  uint8_t* staging = ends + kEnds * kEndBytes;
  Pipe<kGradStages, true>& p = *reinterpret_cast<Pipe<kGradStages, true>*>(staging + kGradStaging);

  int2* segments = reinterpret_cast<int2*>(&p + 1);

  const PipeAt<kGradStages, true> at(p);
  const dev::WaitLimit limit{&p.gave_up, a.limit_ns};

  init_pipe(p, 512);
  dev::wait_for_previous();
  for (int e = threadIdx.x; e < a.segments.experts; e += kThreads) segments[e] = segment(a.segments, e);
  __syncthreads();
  const uint32_t tiles = (uint32_t)a.slow_tiles * a.fast_tiles * a.segments.experts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = dev::cluster_rank();
  const uint32_t t0 = blockIdx.x / 2, t_step = gridDim.x / 2;
  const uint32_t stages = dev::smem_u32(base);

  if (brings(warp)) {
    if (dev::elect_one()) {
      Ring<kGradStages> ring;
      Ring<kEnds> end;
      uint32_t turn = (warp == 2 || warp == 9);  // whether it takes the odd steps
      int64_t step_of_cta = -1;
      bool lost = false;
      for (uint32_t t = t0; t < tiles; t += t_step) {
        const GradTile g = grad_tile(a, segments, t);
        const int slow = g.slow + rank * kTileM, fast = g.fast + rank * g.chunks * kBlockK;
        const uint32_t bytes = (2 + g.chunks) * kChunkBytes;
        const int steps = g.steps();
        if (g.end()) {
          // ahead of the steps, into a buffer of its own, so that it is there and cleared when they are done
          if (warp == 2 || warp == 9) lost = lost || !dev::wait_for(at.end_empty(end.stage), end.parity ^ 1, limit);
          if ((warp == 2 || warp == 9) && !lost) {
            const uint32_t to = dev::smem_u32(ends) + end.stage * kEndBytes, bar = at.end_full(end.stage);
            const int row = g.segment.x + g.whole();
            if (warp < 8) {
              dev::arrive_expect(bar, (2 + g.chunks) * kEndChunk);
              for (int c = 0; c < 2; ++c)
                dev::tma_load_2d(to + c * kEndChunk, &a.slow_end, bar, slow + c * kBlockK, row);
            } else {
              for (int c = 0; c < g.chunks; ++c)
                dev::tma_load_2d(to + (2 + c) * kEndChunk, &a.fast_end, bar, fast + c * kBlockK, row);
            }
          }
          end.next();
        }
        for (int k = 0; k < steps; ++k, ring.next()) {
          ++step_of_cta;
          if ((turn ^= 1) == 0 || lost) continue;
          lost = !dev::wait_for(at.empty(ring.stage), ring.parity ^ 1, limit);
          if (lost || step_of_cta == a.skip) continue;
          const uint32_t to = stages + ring.stage * kGradStage, bar = dev::in_first(at.full(ring.stage));
          const int row = g.segment.x + k * kBlockK;
          if (warp < 8) {
            if (rank == 0) dev::arrive_expect(at.full(ring.stage), 2 * bytes);
            dev::tma_load_2d<true>(to, &a.slow, bar, slow, row);
            dev::tma_load_2d<true>(to + kChunkBytes, &a.slow, bar, slow + kBlockK, row);
          } else {
            for (int c = 0; c < g.chunks; ++c)
              dev::tma_load_2d<true>(to + (2 + c) * kChunkBytes, &a.fast, bar, fast + c * kBlockK, row);
          }
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    if (dev::elect_one()) {
      Ring<kGradStages> ring;
      Ring<2> sums;
      const uint64_t first_a = dev::operand_descriptor(stages, kChunkBytes, 1024);
      const uint64_t first_b = dev::operand_descriptor(stages + 2 * kChunkBytes, kChunkBytes, 1024);
      Ring<kEnds> end;
      const uint64_t end_a = dev::operand_descriptor(dev::smem_u32(ends), kEndChunk, 1024);
      const uint64_t end_b = dev::operand_descriptor(dev::smem_u32(ends) + 2 * kEndChunk, kEndChunk, 1024);
      bool lost = false;
      for (uint32_t t = t0; t < tiles; t += t_step) {
        const GradTile g = grad_tile(a, segments, t);
        if (g.segment.y == 0) continue;
        const uint32_t instruction = dev::mma_instruction(std::is_same_v<T, __nv_bfloat16>, true, true, 2 * kTileM,
                                                          2 * g.chunks * kBlockK);
        const uint32_t sum = p.tmem + sums.stage * kGradN;
        const int whole = g.whole(), steps = g.steps();
        lost = lost || !dev::wait_for<true>(at.sum_empty(sums.stage), sums.parity ^ 1, limit);
        for (int k = 0; k < steps; ++k, ring.next()) {
          lost = lost || !dev::wait_for(at.full(ring.stage), ring.parity, limit);
          if (lost) continue;
          dev::tmem_fence_after();
          const uint32_t stage = ring.stage * (kGradStage / 16);
          const int depth = min(kBlockK, whole - k * kBlockK) / 16;
#pragma unroll
          for (int i = 0; i < kBlockK / 16; ++i)
            if (i < depth)
              dev::mma_issue<true>(sum, first_a + stage + i * 2048 / 16, first_b + stage + i * 2048 / 16, instruction,
                                   k + i > 0);
          dev::mma_commit<true>(at.empty(ring.stage));
        }
        if (g.end()) {
          lost = lost || !dev::wait_for<true>(at.end_cleared(end.stage), end.parity, limit);
          if (!lost) {
            dev::tmem_fence_after();
            const uint32_t buffer = end.stage * (kEndBytes / 16);
            dev::mma_issue<true>(sum, end_a + buffer, end_b + buffer, instruction, steps > 0);
            dev::mma_commit<true>(at.end_empty(end.stage));
          }
          end.next();
        }
        if (!lost) dev::mma_commit<true>(at.sum_full(sums.stage));
        sums.next();
      }
    }
  } else if (warp == 3) {
    // What came with the ends of segments is cleared.  With the ends in the stages, among the steps, this took about a
    // microsecond that nothing hid (32 experts of 1023 rows, 2048 x 4096: 457 us where this way took 414; 399 to 408 in
    // later runs, 396 to 400 of 1024 rows); done by the multiplying warp, 685.
    Ring<kEnds> end;
    for (uint32_t t = t0; t < tiles; t += t_step) {
      const GradTile g = grad_tile(a, segments, t);
      if (!g.end()) continue;
      if (!warp_wait(at.end_full(end.stage), end.parity, limit)) break;  // every later one is lost too
      uint8_t* chunk = ends + end.stage * kEndBytes + lane * 16;  // 8 lanes to a row
      for (int c = 0; c < 2 + g.chunks; ++c, chunk += kEndChunk)
        for (int row = g.end(); row < kEndRows; row += 4)
          if (row + lane / 8 < kEndRows)
            *reinterpret_cast<uint4*>(chunk + row * dev::kBoxRowBytes) = make_uint4(0, 0, 0, 0);
      dev::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) dev::arrive_first(at.end_cleared(end.stage));
      end.next();
    }
  } else if (warp >= 4 && warp < 8) {
    Ring<2> sums;
    const int quarter = warp & 3;
    uint8_t* mine = staging + quarter * kStoreBoxes * kStoreBox;
    const bool whole = a.fast_width % 8 == 0;
    int filled = 0;
    bool lost = false;
    for (uint32_t t = t0; t < tiles; t += t_step) {
      const GradTile g = grad_tile(a, segments, t);
      const int m = g.slow + rank * kTileM + quarter * 32;
      const int columns = min(2 * g.chunks * kBlockK, a.fast_width - g.fast), rows = min(32, a.slow_width - m);
      const bool empty = g.segment.y == 0;
      if (!empty) {
        lost = lost || !warp_wait(at.sum_full(sums.stage), sums.parity, limit);
        dev::tmem_fence_after();
      }
      const uint32_t gone = lost && !empty ? kLost : 0;
      for (int c = 0; c < columns; c += 32) {
        uint32_t v[32];
        if (empty) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        } else {
          dev::tmem_load32(p.tmem + sums.stage * kGradN + c + ((uint32_t)quarter << 21), v);
          dev::tmem_load_wait(v);
        }
        if (rows <= 0) continue;
        // 16-byte pieces in the order of the tiled copies of 64-byte rows: the piece's number xor that of the row pair
        uint8_t* box = mine + filled * kStoreBox;
        dev::store_wait<kStoreBoxes - 1>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t* x = v + j * 8;
          uint4 w;
          w.x = dev::from_float2(__uint_as_float(x[0]), __uint_as_float(x[1]), T{}) | gone;
          w.y = dev::from_float2(__uint_as_float(x[2]), __uint_as_float(x[3]), T{}) | gone;
          w.z = dev::from_float2(__uint_as_float(x[4]), __uint_as_float(x[5]), T{}) | gone;
          w.w = dev::from_float2(__uint_as_float(x[6]), __uint_as_float(x[7]), T{}) | gone;
          *reinterpret_cast<uint4*>(box + lane * 64 + ((j ^ (lane >> 1 & 3)) * 16)) = w;
        }
        if (whole) {
          dev::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) dev::tma_store_3d(&a.out, dev::smem_u32(box), g.fast + c, m, g.expert);
        } else {
          __syncwarp();
          T* out = static_cast<T*>(a.result) + ((int64_t)g.expert * a.slow_width + m) * a.fast_width + g.fast + c;
          T x[32];
#pragma unroll
          for (int row = 0; row < 32; ++row)
            x[row] = *reinterpret_cast<const T*>(box + row * 64 + ((lane / 8 ^ (row >> 1 & 3)) * 16) + lane % 8 * 2);
          out += lane;
          const int there = c + lane < columns ? rows : 0;
#pragma unroll
          for (int row = 0; row < 32; ++row, out += a.fast_width)
            if (row < there) *out = x[row];
          __syncwarp();
        }
        filled = (filled + 1) % kStoreBoxes;
      }
      if (!empty) {
        dev::tmem_fence_before();
        __syncwarp();
        if (lane == 0 && !lost) at.release_sum(sums.stage);
        sums.next();
      }
    }
    dev::store_wait<0>();
  }
  __syncwarp();
  close_pipe(p, 512);
}

// --------------------------------------------------------- operands laid out anew

struct RepackArgs {
  const uint16_t *x, *x_end;  // x_end: behind the last element of all
  uint16_t* y;
  int64_t outer_stride, row_stride, pitch;  // elements
  int64_t rows;                             // of all outer parts together
  int per_outer, width;
  const int32_t* counts;  // where it is given: outer parts with none are left out
};

// The 16-byte word at `word`, of which the elements in [x, end) are read.
__device__ __forceinline__ uint4 load_word(const uint4* word, const uint16_t* x, const uint16_t* end) {
  const uint16_t* e = reinterpret_cast<const uint16_t*>(word);
  if (e >= x && e + 8 <= end) return *word;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t low = e + 2 * i >= x && e + 2 * i < end ? e[2 * i] : 0;
    const uint32_t high = e + 2 * i + 1 >= x && e + 2 * i + 1 < end ? e[2 * i + 1] : 0;
    w[i] = low | high << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes from byte `shift` (even, below 16) of two words on.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int shift) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t v[5];
  switch (shift >> 2) {  // the same in the whole warp
#define TAKE(q) \
  case q: \
    _Pragma("unroll") for (int i = 0; i < 5; ++i) v[i] = w[q + i < 8 ? q + i : 7]; \
    break;
    TAKE(0) TAKE(1) TAKE(2) TAKE(3)
#undef TAKE
  }
  const uint32_t order = shift & 2 ? 0x5432 : 0x3210;
  return make_uint4(__byte_perm(v[0], v[1], order), __byte_perm(v[1], v[2], order), __byte_perm(v[2], v[3], order),
                    __byte_perm(v[3], v[4], order));
}

// Rows of a width or at an address that the tiled copies do not take (they want 16-byte steps), copied to where they
// do: y[r] = x's row r, `pitch` elements apart, whole 16-byte words of it (what lies behind the row's end is anything).
// One warp to a row, two aligned words shifted together for each one stored; bound by memory.
__global__ void __launch_bounds__(256) repack_kernel(const __grid_constant__ RepackArgs a) {
  dev::wait_for_previous();
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, words = (a.width + 7) / 8;
  for (int64_t r = blockIdx.x * 8ll + (threadIdx.x >> 5); r < a.rows; r += gridDim.x * 8ll) {
    const int64_t outer = r / a.per_outer;
    if (a.counts != nullptr && a.counts[outer] <= 0) continue;
    const uint16_t* x = a.x + outer * a.outer_stride + (r - outer * a.per_outer) * a.row_stride;
    const int shift = reinterpret_cast<uintptr_t>(x) & 15;
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x) - shift);
    const uint16_t* row_end = x + a.width;
    uint4* to = reinterpret_cast<uint4*>(a.y + r * a.pitch);
    for (int i0 = lane; i0 < words; i0 += 32 * U) {
      uint4 w[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + 32 * u;
        w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
        if (i < words) {
          w[u][0] = load_word(from + i, a.x, a.x_end);
          if (shift && reinterpret_cast<const uint16_t*>(from + i + 1) < row_end)
            w[u][1] = load_word(from + i + 1, a.x, a.x_end);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + 32 * u < words) to[i0 + 32 * u] = shifted(w[u][0], w[u][1], shift);
    }
  }
}

// ------------------------------------------------------------------- the host side

// An operand: `outer` matrices of `rows` rows of `width` contiguous elements.
struct Operand {
  const void* data;
  int64_t outer, rows, width, outer_stride, row_stride;

  bool ready() const {
    return ((reinterpret_cast<uintptr_t>(data) | (uintptr_t)(rows > 1 ? row_stride * 2 : 0) |
             (uintptr_t)(outer > 1 ? outer_stride * 2 : 0)) & 15) == 0 &&
           (rows <= 1 || row_stride >= width) && (outer <= 1 || outer_stride > 0);
  }
  int64_t pitch() const { return (width + 7) / 8 * 8; }
  size_t bytes() const { return ready() ? 0 : ((size_t)(outer * rows * pitch()) * 2 + 255) / 256 * 256; }

  // Copies it to `temp`, if need be.
  cudaError_t prepare(uint8_t*& temp, const int32_t* counts, cudaStream_t stream) {
    if (ready()) return cudaSuccess;
    const size_t size = bytes();
    const uint16_t* x = static_cast<const uint16_t*>(data);
    RepackArgs a{x, x + (outer - 1) * outer_stride + (rows - 1) * row_stride + width, reinterpret_cast<uint16_t*>(temp),
                 outer_stride, row_stride, pitch(), outer * rows, (int)rows, (int)width, counts};
    data = temp;
    row_stride = pitch();
    outer_stride = rows * pitch();
    temp += size;
    return launch_after_previous(repack_kernel, std::min<int64_t>(kSms * 8, (a.rows + 7) / 8), 256, 0, a, stream);
  }

  cudaError_t map(CUtensorMap* m, bool matrix, uint32_t box_rows, uint32_t box_width = kBlockK) const {
    // strides of dimensions of one element are never used, but have to be in order
    const uint64_t row = (uint64_t)(rows > 1 ? row_stride : pitch()) * 2;
    const uint64_t dims[3] = {(uint64_t)width, (uint64_t)rows, (uint64_t)outer};
    const uint64_t strides[2] = {row, outer > 1 ? (uint64_t)outer_stride * 2 : row * rows};
    const uint32_t box[3] = {box_width, box_rows, 1};
    return encode_map(m, data, matrix ? 2 : 3, dims, strides, box);
  }
};

// Over `ctas` CTAs to a tile, a cluster.
template <typename Kernel, typename Args>
cudaError_t run(Kernel kernel, const Args& a, int64_t tiles, int ctas, size_t smem, cudaStream_t stream) {
  // the limit is the kernel's, not the call's: the same one from every host thread
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e) return e;
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(kSms / ctas, tiles)) * ctas;
  return launch_after_previous(kernel, grid, kThreads, smem, a, stream, ctas);
}

template <typename T, typename Shape>
cudaError_t product(ProductArgs& a, Operand weights, Operand rows, bool in_order, int64_t row_tiles,
                    cudaStream_t stream) {
  a.width_tiles = (a.width + Shape::kTile - 1) / Shape::kTile;
  a.most = (uint32_t)row_tiles;
  cudaError_t e = weights.map(&a.weights, false, in_order ? Shape::kWeightColumns : kBlockK);
  for (int i = 0; !e && i < 3; ++i) e = rows.map(&a.rows[i], true, 64 >> i);
  if (e) return e;
  const size_t smem = product_bytes<Shape>(a.segments.experts);
  const int64_t tiles = row_tiles * a.width_tiles;
  return in_order ? run(product_kernel<T, Shape, true>, a, tiles, Shape::kCtas, smem, stream)
                  : run(product_kernel<T, Shape, false>, a, tiles, Shape::kCtas, smem, stream);
}

// Tiles begin before this many rows and end within 32 bits.
constexpr int64_t kMaxRows = INT32_MAX - 1024;

bool sizes_fit(int64_t capacity, int64_t in, int64_t out, int experts) {
  return capacity >= 0 && capacity <= kMaxRows && in >= 1 && in <= (1 << 20) && out >= 1 && out <= (1 << 20) &&
         experts >= 1 && experts <= kMaxExperts;
}

// Whether elements of the type can be loaded from these addresses.
bool on_elements(cusort_float_type type, const void* x, const void* y) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
  return (bits & (uintptr_t)(float_type_bytes(type) - 1)) == 0;
}

}  // namespace

extern "C" cudaError_t cusort_expert_products(void* d_temp_storage, size_t* temp_storage_bytes, cusort_float_type type,
                                              const void* d_rows, int64_t row_stride, const void* d_weights,
                                              int64_t expert_stride, int64_t in_stride, int64_t out_stride,
                                              const int32_t* d_counts, const int32_t* d_offsets, void* d_out,
                                              int64_t capacity, int64_t in, int64_t out, int num_experts,
                                              cudaStream_t stream) {
  if (temp_storage_bytes == nullptr || float_type_bytes(type) == 0 || !sizes_fit(capacity, in, out, num_experts) ||
      row_stride < 0 || expert_stride < 0 || in_stride < 0 || out_stride < 0 || !on_elements(type, d_rows, d_weights))
    return cudaErrorInvalidValue;
  const bool in_order = !(out_stride == 1 || out == 1);
  if (in_order && in_stride != 1 && in != 1) return cudaErrorInvalidValue;
  const bool whole = type == CUSORT_FLOAT_F32;  // its loads take any address and stride
  Operand rows{d_rows, 1, capacity, in, 0, row_stride};
  Operand weights{d_weights, num_experts, in_order ? out : in, in_order ? in : out, expert_stride,
                  in_order ? out_stride : in_stride};
  const size_t need = std::max<size_t>(1, capacity == 0 || whole ? 0 : rows.bytes() + weights.bytes());
  if (d_temp_storage == nullptr) {
    *temp_storage_bytes = need;
    return cudaSuccess;
  }
  if (*temp_storage_bytes < need) return cudaErrorInvalidValue;
  if (capacity == 0) return cudaSuccess;
  if (d_rows == nullptr || d_weights == nullptr || d_counts == nullptr || d_offsets == nullptr || d_out == nullptr ||
      (reinterpret_cast<uintptr_t>(d_out) & 15) != 0 ||
      (need > 1 && (reinterpret_cast<uintptr_t>(d_temp_storage) & 15) != 0))
    return cudaErrorInvalidValue;
  const SegmentArgs segments{d_counts, d_offsets, num_experts, (int)capacity};
  if (whole)
    return float_products(static_cast<const float*>(d_rows), row_stride, static_cast<const float*>(d_weights),
                          expert_stride, in_stride, out_stride, segments, static_cast<float*>(d_out), (int)in, (int)out,
                          stream);
  const bool few = capacity <= (int64_t)kProductFewRows * num_experts;
  ProductArgs a;
  a.segments = segments;
  a.out = d_out;
  a.in = (int)in;
  a.width = (int)out;
  a.limit_ns = wait_limit_ns();
  a.skip = debug_skip_tile();
  // at most one part-filled tile to an expert, and no expert without a row
  const int rows_of_tile =
      capacity <= kProductFewestRows ? kProductFewestRows : few ? kProductFewRows : kProductManyRows;
  const int64_t tiles = capacity / rows_of_tile + std::min<int64_t>(num_experts, capacity);
  if (tiles * ((out + kTileM - 1) / kTileM) > 1 << 30) return cudaErrorInvalidValue;
  uint8_t* temp = static_cast<uint8_t*>(d_temp_storage);
  cudaError_t e = rows.prepare(temp, nullptr, stream);
  if (!e) e = weights.prepare(temp, d_counts, stream);
  if (e) return e;
  const auto go = [&](auto t) {
    using T = decltype(t);
    if (capacity <= kProductFewestRows)
      return tiles * ((out + kTileM - 1) / kTileM) <= kSms / 2
                 ? product<T, ProductFewestNarrow>(a, weights, rows, in_order, tiles, stream)
                 : product<T, ProductFewest>(a, weights, rows, in_order, tiles, stream);
    return few ? product<T, ProductFew>(a, weights, rows, in_order, tiles, stream)
               : product<T, ProductMany>(a, weights, rows, in_order, tiles, stream);
  };
  return type == CUSORT_FLOAT_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

extern "C" cudaError_t cusort_expert_products_grad_weights(
    void* d_temp_storage, size_t* temp_storage_bytes, cusort_float_type type, const void* d_rows, int64_t row_stride,
    const void* d_grad_out, int64_t grad_stride, const int32_t* d_counts, const int32_t* d_offsets,
    void* d_grad_weights, int in_contiguous, int64_t capacity, int64_t in, int64_t out, int num_experts,
    cudaStream_t stream) {
  if (temp_storage_bytes == nullptr || float_type_bytes(type) == 0 || !sizes_fit(capacity, in, out, num_experts) ||
      row_stride < 0 || grad_stride < 0 || !on_elements(type, d_rows, d_grad_out))
    return cudaErrorInvalidValue;
  Operand slow{d_rows, 1, capacity, in, 0, row_stride}, fast{d_grad_out, 1, capacity, out, 0, grad_stride};
  if (in_contiguous) std::swap(slow, fast);
  const bool whole = type == CUSORT_FLOAT_F32;
  const size_t need = std::max<size_t>(1, capacity == 0 || whole ? 0 : slow.bytes() + fast.bytes());
  if (d_temp_storage == nullptr) {
    *temp_storage_bytes = need;
    return cudaSuccess;
  }
  if (*temp_storage_bytes < need) return cudaErrorInvalidValue;
  if (d_grad_weights == nullptr || (reinterpret_cast<uintptr_t>(d_grad_weights) & 15) != 0)
    return cudaErrorInvalidValue;
  if (capacity == 0)
    return cudaMemsetAsync(d_grad_weights, 0, (size_t)num_experts * in * out * float_type_bytes(type), stream);
  if (d_rows == nullptr || d_grad_out == nullptr || d_counts == nullptr || d_offsets == nullptr ||
      (need > 1 && (reinterpret_cast<uintptr_t>(d_temp_storage) & 15) != 0))
    return cudaErrorInvalidValue;
  const SegmentArgs segments{d_counts, d_offsets, num_experts, (int)capacity};
  if (whole)
    return float_products_grad(static_cast<const float*>(slow.data), slow.row_stride,
                               static_cast<const float*>(fast.data), fast.row_stride, segments,
                               static_cast<float*>(d_grad_weights), (int)slow.width, (int)fast.width, stream);
  GradArgs a;
  a.segments = segments;
  a.result = d_grad_weights;
  a.slow_width = (int)slow.width;
  a.fast_width = (int)fast.width;
  a.slow_tiles = (int)((slow.width + 2 * kTileM - 1) / (2 * kTileM));
  a.fast_tiles = (int)((fast.width + kGradN - 1) / kGradN);
  a.limit_ns = wait_limit_ns();
  a.skip = debug_skip_tile();
  const int64_t tiles = (int64_t)a.slow_tiles * a.fast_tiles * num_experts;
  if (tiles > INT32_MAX) return cudaErrorInvalidValue;
  uint8_t* temp = static_cast<uint8_t*>(d_temp_storage);
  cudaError_t e = slow.prepare(temp, nullptr, stream);
  if (!e) e = fast.prepare(temp, nullptr, stream);
  if (!e) e = slow.map(&a.slow, true, kBlockK);
  if (!e) e = fast.map(&a.fast, true, kBlockK);
  if (!e) e = slow.map(&a.slow_end, true, kEndRows);
  if (!e) e = fast.map(&a.fast_end, true, kEndRows);
  if (!e && fast.width % 8 == 0) {
    const Operand out{d_grad_weights, num_experts, slow.width, fast.width, slow.width * fast.width, fast.width};
    e = out.map(&a.out, false, 32, 32);
  }
  if (e) return e;
  const size_t smem = grad_bytes(num_experts);
  return type == CUSORT_FLOAT_F16 ? run(grad_weights_kernel<__half>, a, tiles, 2, smem, stream)
                                  : run(grad_weights_kernel<__nv_bfloat16>, a, tiles, 2, smem, stream);
}

extern "C" cudaError_t cusort_read_product_status(uint32_t* status, cudaStream_t stream) {
  if (status == nullptr) return cudaErrorInvalidValue;
  void* words = nullptr;
  uint32_t lost[2] = {};
  cudaError_t e = cudaGetSymbolAddress(&words, g_lost);
  if (!e) e = cudaMemcpyAsync(lost, words, sizeof(lost), cudaMemcpyDeviceToHost, stream);
  if (!e) e = cudaStreamSynchronize(stream);
  if (e) return e;
  *status = lost[0] != lost[1];
  if (*status == 0) return cudaSuccess;
  e = cudaMemcpyAsync(static_cast<uint32_t*>(words) + 1, lost, sizeof(uint32_t), cudaMemcpyHostToDevice, stream);
  return e ? e : cudaStreamSynchronize(stream);
}
