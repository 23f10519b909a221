// Kernels that begin while the one in front of them in the stream ends, and wait for its end themselves: what they do before that overlaps with it, and so does their launch.
#pragma once
#include <cuda_runtime.h>

namespace attn {

// Everything that kernels in front have written can be read behind this, and what they read can be written.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The kernel behind this one may begin (it waits for the end of this one all the same).
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The kernel has to wait_for_previous_kernel before it touches memory.  `cluster` CTAs in a row, of grid.x, share their shared memory.
template <typename... P, typename... A>
cudaError_t launch_early_in_clusters(unsigned cluster, void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const A &...args) {
    return launch_early_in_clusters(1, kernel, grid, threads, smem, stream, args...);
}

}  // namespace attn
