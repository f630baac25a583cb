// A kernel that follows another on the stream and is set up while that one still runs (programmatic dependent launch).
//
// The kernel before calls allow_dependents() in every thread block; the one that follows calls wait_for_previous() before it
// touches anything that earlier work on the stream writes or reads: the wait ends when the kernel before has ended and its
// writes can be seen, and since that kernel has waited in its turn, everything before it has ended as well.
#pragma once

#include <cuda_runtime.h>

namespace nb200 {

#ifdef __CUDACC__
__device__ __forceinline__ void allow_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace nb200
