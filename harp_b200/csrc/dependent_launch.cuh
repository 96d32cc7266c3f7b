// Programmatic dependent launch: a kernel launched so may start (set up barriers,
// tensor memory, shared memory) while the kernel before it on the stream still
// runs, and reads or writes global memory only after dependency_wait(), which
// returns once that kernel has completed and its writes are visible.  A kernel
// allows the next one to start before its own end with dependency_release(): the
// next one's blocks then take the SMs that this one's blocks leave.  A kernel
// launched in the ordinary way waits for the whole of the one before it, as ever.
//
// The int8 GEMMs release at their start (back to back on B200: 4 x 6912 x 1152 in 4.2
// us, 4.9 without the release; 4352 x 1152 x 1152 9.1 and 10.1).  The quantisers do
// not: blocks of the next kernel that wait beside theirs cost more than they save
// (fp32 norm of 1061 x 1155 and its dequantisation 10.8 us with, 8.5 without).
//
// Every thread of a kernel launched so calls dependency_wait() before its first
// access to global memory, also when it has nothing to do.
//
// What it then reads may have been written while it was already running, so it reads
// with ordinary (coherent) loads, never through the read-only path, which wants data
// that do not change during the kernel (and which the compiler may move ahead of the
// wait): no read-only or cache-hint load intrinsics, no pointer parameters that promise
// not to alias; loads in assembly are volatile.
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
