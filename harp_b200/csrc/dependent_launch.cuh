// Programmatic dependent launch: a kernel launched so may start (set up barriers,
// tensor memory, shared memory) while the kernel before it on the stream still
// runs, and reads or writes global memory only after dependency_wait(), which
// returns once that kernel has completed and its writes are visible.  A kernel
// allows the next one to start with dependency_release(): the next one's blocks
// then take the SMs that this one's blocks leave.  A kernel launched in the
// ordinary way waits for the whole of the one before it, as ever.
//
// Every thread of a kernel launched so calls dependency_wait() before its first
// access to global memory, also when it has nothing to do.
#pragma once

#include <c10/cuda/CUDAException.h>
#include <cuda_runtime.h>

#include <utility>

namespace harp {

__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependency_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launch `kern`, in clusters of `cluster` blocks along x if that is more than one.
template <typename... P, typename... A>
void launch_dependent(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int cluster,
                      A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...));
}

}  // namespace harp
