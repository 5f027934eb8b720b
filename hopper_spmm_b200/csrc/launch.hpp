// How the kernels of a product are launched.
#pragma once

#include <cuda_runtime.h>

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

}  // namespace b200spmm
