// rt_chain.cuh — kernels of one call that follow one another: the next one's
// blocks are put on the SMs while the last of the one before still run, and
// wait there (in hardware) until it has completed and its writes are visible.
#pragma once
#include <cuda_runtime.h>

namespace rt {

// Device: blocks until every kernel this one was launched behind with
// launch_after has completed.  Nothing those kernels write may be read, and
// nothing they read may be written, before it.
__device__ __forceinline__ void wait_for_previous_kernel() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// Device: the next kernel's blocks may be scheduled once every block of this
// one has come here or ended.
__device__ __forceinline__ void let_next_kernel_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Host: launches `kernel`, which calls wait_for_previous_kernel(), behind the
// previous kernel of the stream.
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem,
                         cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

}  // namespace rt
