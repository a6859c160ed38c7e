// cusort_tensor.cuh -- what the matrix products need of the tensor cores and
// of the tiled copies: bounded barrier waits, tensor maps, shared-memory and
// instruction descriptors, accumulators in tensor memory.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cusort_device.cuh"

namespace cusort_b200 {
namespace dev {

// 64 16-bit elements along the contiguous dimension: the width of every box
// that the tiled copies load, whose 16-byte pieces they permute within each 8
// rows (128-byte swizzle).  Boxes that are stored are half as wide, with the
// 64-byte swizzle.
constexpr int kBoxRowBytes = 128;

// A box into this CTA's shared memory, counted on the barrier `bar` (PAIR: of either CTA of a cluster of two).
template <bool PAIR = false>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
template <bool PAIR = false>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// A box from shared memory, what lies outside the tensor left out; a group of
// one.  All of the thread's groups but the last N have been read when
// store_wait returns.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
               "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void store_wait() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// Shared-memory matrix descriptor of a 128-byte-swizzled operand.  `leading`
// and `stride` in bytes:
//   contracted dimension contiguous: `stride` from one group of 8 rows to the
//   next (1024), `leading` unused; 16 elements on: 32 bytes on;
//   other dimension contiguous: `leading` from one 64-element column of boxes
//   to the next, `stride` from one group of 8 contracted rows to the next
//   (1024); 16 contracted elements on: 2048 bytes on.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t address, uint32_t leading, uint32_t stride) {
  return (uint64_t)((address & 0x3ffff) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Instruction descriptor: 16-bit operands of one type, 32-bit sums.
__host__ __device__ constexpr uint32_t mma_instruction(bool bf16, bool a_transposed, bool b_transposed, int m, int n) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_transposed ? 1u << 15 : 0u) | (b_transposed ? 1u << 16 : 0u) |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// One thread: accumulator (at the tensor-memory address) (+)= A x B.  PAIR:
// over a cluster of two CTAs, issued by the first; A and the accumulator lie
// half their rows in each, B half its columns in each, all at the same
// addresses.
template <bool PAIR>
__device__ __forceinline__ void mma_issue(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t instruction,
                                          bool add) {
  if constexpr (PAIR)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(accumulator),
        "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(accumulator),
        "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
        : "memory");
}
// The barrier (PAIR: the one at this address in both CTAs) gets one arrival when the products issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t address, uint32_t columns) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes of tensor memory: v[i] = column i of this thread's lane, after
// tmem_load_wait.
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(address));
}
// v is there when this returns, and is not looked at before.
__device__ __forceinline__ void tmem_load_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                 "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]),
                 "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                 "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                 "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]),
                 "+r"(v[31])
               :
               : "memory");
}

// One thread of a whole warp, the same one each time.  Where copies and
// products are issued under it, the compiler knows that a single thread does.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

// Number of this CTA in its cluster.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// This shared-memory address in the cluster's first CTA.
__device__ __forceinline__ uint32_t in_first(uint32_t address) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(address));
  return r;
}
// All threads of the cluster.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Barriers by their shared-memory addresses.
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// At the barrier at this address of the cluster's first CTA.
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first(bar)) : "memory");
}
// Whether a phase is over.  CLUSTER: of a barrier at which other CTAs of the cluster arrive.
template <bool CLUSTER>
__device__ __forceinline__ bool is_over(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if constexpr (CLUSTER)
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  return ok != 0;
}

// What ends a CTA's waits: a time, and a word in shared memory that says that
// one of them ran out.  From then on they all return false at once.
struct WaitLimit {
  volatile uint32_t* gave_up;
  uint64_t ns;
};

// The rest of wait_for, for a phase that was not over yet.  Not inlined: with
// this loop in the loops that bring and multiply tiles a wait cost 380 cycles
// even where the phase was over.
template <bool CLUSTER>
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, WaitLimit limit) {
  uint64_t t0 = 0;
  for (;;) {
    // the clock is looked at now and then: reading it takes longer than most waits
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (is_over<CLUSTER>(bar, parity)) return true;
    if (*limit.gave_up) return false;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > limit.ns) {
      *limit.gave_up = 1;
      return false;
    }
  }
}

// Waits for a phase of a barrier; false: in vain.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, WaitLimit limit) {
  return is_over<CLUSTER>(bar, parity) || wait_long<CLUSTER>(bar, parity, limit);
}

}  // namespace dev

// Tensor map of 16-bit elements, zeros outside.  dims and box from the
// contiguous dimension on; strides in bytes, of the dimensions after it.  The
// box's rows are 128 or 64 bytes, whose swizzle it has.
cudaError_t encode_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                       const uint32_t* box);

}  // namespace cusort_b200
