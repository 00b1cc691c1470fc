// Programmatic dependent launch: the order of this library's kernels in a stream.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace hc {

// A kernel launched with the stream-serialization attribute may start while its predecessor in the
// stream is still draining.  `pdl_release` lets the successor be scheduled as soon as every CTA of this
// grid has issued it (or exited); `pdl_wait` blocks until the predecessor has completed and its memory is
// visible.  Both are no-ops for an ordinary launch.  Everything before pdl_wait must touch no global
// memory that an earlier kernel may write.  Behind it, loads go by the coherent path: the non-coherent one
// (the read-only cache) is for memory that does not change while the kernel runs, and the kernel may have
// started while its predecessor was still writing.  Both cost the same here.
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches `fn` so that it may start (up to its pdl_wait) under its predecessor's tail.
inline cudaError_t launch_behind(const void* fn, void** args, dim3 grid, dim3 block, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace hc
