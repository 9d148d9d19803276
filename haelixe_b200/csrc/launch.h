// Launches that may overlap the end of the kernel before them on the stream
// (programmatic dependent launch): the kernel calls after_prior_kernels()
// before its first access to global memory, which waits until all of them
// are complete and their writes visible, and may_start_next() once, so that the
// next such kernel's launch is under way by then. In a decode step, a row of
// kernels of a few microseconds, this hides most of a launch.
#pragma once

#include <cuda_runtime.h>

#include "hx_internal.h"

namespace hx {

__device__ __forceinline__ void after_prior_kernels() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void may_start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// cluster: CTAs of a cluster along x, 0 for none.
template <typename... P, typename... A>
cudaError_t launch_overlapped(cudaStream_t st, void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster,
                              A&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e == cudaSuccess) note_launch();
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace hx
