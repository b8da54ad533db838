// launch.cuh -- kernel launch with optional programmatic dependent launch.
#pragma once
#include <cuda_runtime.h>
#include <utility>
#include "kernels.h"

namespace gncx {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" :::); }

// Launch `k` on `st`; when programmatic dependent launch is enabled the kernel
// may begin before its predecessor on the stream completes, and must call
// pdl_wait() before it touches anything that predecessor writes or reads.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_k(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                            Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...);
}

// Launch `k` with programmatic dependent launch whatever gncx_set_weight_prefetch
// says: it may be set up while its predecessor on the stream still runs, and
// calls pdl_wait() before it touches any memory that a predecessor may read or
// write.  cluster > 1: clusters of that many CTAs along x.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_early(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster,
                                Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...);
}
template <typename... KArgs, typename... Args>
inline cudaError_t launch_after(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                Args&&... args) {
    return launch_early(k, grid, block, smem, st, 1, std::forward<Args>(args)...);
}

}  // namespace gncx
