// Launches of the dense and norm kernels as programmatic dependents: a kernel
// may start while the one before it in the stream still runs, sets itself up,
// and waits (pdl_wait) for its end before it touches any memory that others
// write.  Saves about 2 us between two calls of few rows.  Every kernel here
// calls pdl_begin first and pdl_wait in every thread before its first access, and
// reads with ordinary loads: the read-only path (__ldg, ld.global.nc) is for
// memory that nobody writes while the kernel lives, and these live while the
// kernel in front still writes what they read, weights (an optimizer's step,
// quantize_rows) like activations.
#pragma once
#include <cuda_runtime.h>

namespace ngl {
namespace dev {

// The next kernel of the stream may start as soon as all CTAs are here.
__device__ __forceinline__ void pdl_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Until the kernel before this one has ended and its writes are seen.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_dependent(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t s,
                             A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, P(args)...);
}

}  // namespace dev
}  // namespace ngl
