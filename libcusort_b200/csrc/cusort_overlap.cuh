// cusort_overlap.cuh -- launches whose own time overlaps the end of the kernel
// before them in the stream (programmatic dependent launch).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cusort_device.cuh"

namespace cusort_b200 {
namespace dev {

// The first thing that every thread of such a kernel does: it waits until the
// kernel before is done and its writes are seen.  Nothing is read or written
// before, so the stream's order holds for any kernels around; what is gained
// is most of the time from the end of one kernel to the work of the next
// (dispatch, combine and their gradients, 4 MB to 120 MB each: 2 us a kernel).
//
// No kernel lets the next one come earlier than at its own end.  Put beside
// the CTAs of a kernel that still runs, the next one's end up on some SMs in
// numbers: a step of 1024 tokens (route to combine) took 23.5 us that way and
// 18.2 this way, routing with its gradient over 32768 tokens 19.7 and 12.1.
__device__ __forceinline__ void wait_for_previous() { pdl_wait(); }

}  // namespace dev

// Launches a kernel that begins with wait_for_previous(), over clusters of
// `cluster` CTAs.
template <typename Args>
cudaError_t launch_after_previous(void (*kernel)(Args), int64_t grid, int threads, size_t smem, const Args& args,
                                  cudaStream_t stream, int cluster = 1) {
  if (grid < 1 || grid > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args);
}

}  // namespace cusort_b200
