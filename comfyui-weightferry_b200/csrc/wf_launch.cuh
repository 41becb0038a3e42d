// Kernel launches as programmatic dependents of the previous kernel of the stream. Internal linkage.
#pragma once

#include <cuda_runtime.h>

#include <utility>

#include "wf_common.cuh"

namespace wf {
namespace {

// Programmatic dependent launch: the kernel is launched while the previous kernel of the stream may still run, so its
// set-up (barriers, tensor memory, cluster sync) overlaps that kernel's tail; every thread waits here for the previous
// grid's completion and memory before it touches global memory. Without a programmatic launch this returns at once.
__device__ __forceinline__ void wait_prior_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// WEIGHTFERRY_PDL=0 launches plain kernels instead of programmatic dependents
inline bool use_pdl() {
    static const bool pdl = env_digit("WEIGHTFERRY_PDL", 1) != 0;
    return pdl;
}

// a launch of clusters of `cluster` CTAs (0: the kernel's own cluster shape) as a programmatic dependent
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent_clusters(void (*kern)(KArgs...), dim3 grid, int cluster, int threads, size_t smem,
                                      cudaStream_t stream, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = 0;
    if (use_pdl()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 0) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                             Args &&...args) {
    return launch_dependent_clusters(kern, grid, 0, threads, smem, stream, std::forward<Args>(args)...);
}

}  // namespace
}  // namespace wf
