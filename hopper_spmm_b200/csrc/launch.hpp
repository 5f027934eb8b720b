// How the kernels of a product are launched.
#pragma once

#include <atomic>
#include <cuda_runtime.h>

#include "common.hpp"

namespace b200spmm {

// Launches a kernel of a product: it may start when the last block of the kernel before it in the stream has ended, and
// waits itself for that one's results (ptx::wait_for_grids_before).  What a launch costs on the GPU between two others - the
// results' way, the blocks' start, what they set up - overlaps: 4.1 -> 2.8 us a call for 1003 x 997 at 2 %, 32 columns,
// 8.2 -> 6.2 for 4096 x 4096 at 1 %, 128 columns.  The kernels do not let the next one in any earlier: its blocks would take
// the places that become free, unevenly (the same 4096 x 4096: 8.8 us).
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// How many clusters of two CTAs of a kernel the current device runs at once; `known` keeps the answer.
template <typename... P>
int max_pairs(void (*kernel)(P...), unsigned threads, size_t smem, std::atomic<uint32_t> &known, uint32_t *out) {
    *out = known.load(std::memory_order_relaxed);
    if (*out) return B200SPMM_OK;
    B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * 148);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    B200_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n < 1) return B200SPMM_ERR_UNSUPPORTED;
    *out = (uint32_t)n;
    known.store(*out, std::memory_order_relaxed);
    return B200SPMM_OK;
}

}  // namespace b200spmm
