// Launches of the 8-bit operators' kernels.
//
// Each is a programmatic dependent launch: it may become resident while the
// kernel before it on the stream drains, waits for that kernel's completion
// (wait_previous_launch, first thing, before any access to memory another
// kernel may write or read) and then lets the next one come up the same way.
// A chain of short kernels so loses most of its launch gaps. Because a kernel
// signals only after its own wait, whatever ran two launches back is complete
// when its successor starts. (A product after its own quantisation signals at
// once and waits later; what follows it waits for it as for any other.)
#pragma once

#include <cuda_runtime.h>

namespace rns8cuda {

__device__ __forceinline__ void wait_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, unsigned cluster,
                           cudaStream_t stream, const Args&... args) {
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace rns8cuda
