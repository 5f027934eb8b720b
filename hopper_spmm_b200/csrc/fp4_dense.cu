// Product of a 4-bit matrix with a 16-bit dense one.
#include <algorithm>

#include "common.hpp"
#include "fp4.hpp"
#include "fp4_dense_narrow.cuh"
#include "launch.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

template <typename T, bool kMx, int kNB, int kU, bool kTokens>
int launch_narrow(const DenseParams &prm, int device, cudaStream_t stream) {
    using Cfg = NarrowCfg<kNB, kU>;
    auto kernel = fp4_narrow_kernel<T, kMx, kNB, kU, kTokens>;
    static thread_local int configured = -1;
    if (configured != device) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmemBytes));
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        configured = device;
    }
    const dim3 grid((prm.m + 127u) / 128u * (4 / kU), (prm.n + 8 * kNB - 1) / (8 * kNB));
    if (grid.y > 65535u) return B200SPMM_ERR_UNSUPPORTED;
    B200_CUDA_TRY(launch_after(kernel, grid, 32 * kNarrowWarps, Cfg::kSmemBytes, 1, stream, prm));
    return B200SPMM_OK;
}

template <typename T, bool kMx, bool kTokens>
int launch_narrow_rows(const DenseParams &prm, int device, cudaStream_t stream) {
    // A block of threads reads all of B: as many rows a block as leave a block for every SM
    const uint32_t blocks = (prm.m + 127u) / 128u, sms = (uint32_t)sm_count();
    if (prm.n <= 8) {
        if (blocks >= sms) return launch_narrow<T, kMx, 1, 4, kTokens>(prm, device, stream);
        if (blocks * 2 >= sms) return launch_narrow<T, kMx, 1, 2, kTokens>(prm, device, stream);
        return launch_narrow<T, kMx, 1, 1, kTokens>(prm, device, stream);
    }
    if (blocks * 2 >= sms) return launch_narrow<T, kMx, 2, 2, kTokens>(prm, device, stream);
    return launch_narrow<T, kMx, 2, 1, kTokens>(prm, device, stream);
}

}  // namespace

int launch_dense_product(const b200spmm_fp4_t *a, const void *b, int64_t ldb, int64_t n, int b_dtype, bool b_transposed, void *c, int64_t ldc, int c_dtype,
                         bool c_transposed, cudaStream_t stream) {
    const Layout l = layout_of(a->rows, a->cols, a->format);
    DenseParams prm{};
    prm.values = static_cast<const uint8_t *>(a->values);
    prm.scales = static_cast<const uint8_t *>(a->scales);
    prm.whole = a->tensor_scale;
    prm.m = (uint32_t)a->rows;
    prm.k = (uint32_t)a->cols;
    prm.pitch = l.pitch;
    prm.groups = l.groups;
    prm.b = static_cast<const uint8_t *>(b);
    prm.ldb = ldb;
    prm.n = (uint32_t)n;
    prm.b_wide = reinterpret_cast<uintptr_t>(b) % 16u == 0 && ldb % 8 == 0;
    prm.c = target_of(c, ldc, c_dtype, c_transposed);
    if (a->format == B200SPMM_MXFP4)
        return b_transposed ? launch_narrow_rows<__nv_bfloat16, true, true>(prm, a->device, stream) : launch_narrow_rows<__nv_bfloat16, true, false>(prm, a->device, stream);
    if (b_dtype == B200SPMM_T_F16)
        return b_transposed ? launch_narrow_rows<__half, false, true>(prm, a->device, stream) : launch_narrow_rows<__half, false, false>(prm, a->device, stream);
    return b_transposed ? launch_narrow_rows<__nv_bfloat16, false, true>(prm, a->device, stream) : launch_narrow_rows<__nv_bfloat16, false, false>(prm, a->device, stream);
}

}  // namespace fp4
}  // namespace b200spmm
