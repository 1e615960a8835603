// Launches that overlap the end of the kernel before them in the stream.
#pragma once
#include <cuda_runtime.h>

#include "hb_status.h"

namespace hb {

// Launch a kernel that may begin once every CTA of the one before it has started and allowed it
// (griddepcontrol.launch_dependents), or else when that one is done: its setup then costs no time of its own. A kernel
// launched so reads and writes nothing but its parameters before griddepcontrol.wait, which returns when the one
// before is complete with its memory visible, and allows the next one only after that; or it reads nothing that the
// one before writes, was let in by a kernel that had waited itself, and waits before it ends. What other kernels may have
// written is read with ordinary loads or asynchronous copies, never with __ldg: that asks for memory that nothing writes
// while the kernel lives, and the kernel lives before they are done.
template <class... P, class... A>
int launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                 const A&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? HB_OK : HB_ERR_LAUNCH;
}

__device__ __forceinline__ void wait_for_kernel_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace hb
