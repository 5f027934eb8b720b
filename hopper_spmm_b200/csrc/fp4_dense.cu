// Product of a 4-bit matrix with a 16-bit dense one.
#include <algorithm>
#include <atomic>

#include "../../include/b200_spmm_kat.h"
#include "common.hpp"
#include "fp4.hpp"
#include "fp4_dense_narrow.cuh"
#include "fp4_dense_wide.cuh"
#include "launch.hpp"
#include "tensormap.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

template <typename T, bool kMx, int kNB, bool kTokens, bool kExact>
int launch_narrow(const b200spmm_fp4_t *a, const DenseParams &d, cudaStream_t stream) {
    constexpr uint32_t kMostBytes = 226u * 1024u;
    auto kernel = fp4_narrow_kernel<T, kMx, kNB, kTokens, kExact>;
    static thread_local int configured = -1;
    if (configured != a->device) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostBytes));
        configured = a->device;
    }
    const uint32_t passes = (d.n + 8 * kNB - 1) / (8 * kNB);
    if (passes > 65535u) return B200SPMM_ERR_UNSUPPORTED;
    NarrowParams prm{};
    prm.d = d;
    prm.tiles = (d.m + 15u) / 16u;
    const NarrowShare share = narrow_share(prm.tiles, d.k, (uint32_t)sm_count());
    prm.at_once = share.at_once;
    prm.slices = share.slices;
    prm.row_blocks = (prm.at_once * 16u + 126u) / 128u + 1u;
    const uint32_t stage = narrow_stage(kMx, prm.at_once, prm.row_blocks, kNB).bytes(), warps = prm.at_once * prm.slices;
    const uint32_t sums = prm.slices > 1 ? warps * 16u * 8u * kNB * (uint32_t)sizeof(float) : 0u;
    prm.stages = std::min({kNarrowMaxStages, (kMostBytes - 1280u - sums) / stage, std::max<uint32_t>(2, (d.k + kNarrowStage - 1) / kNarrowStage)});
    B200_CUDA_TRY(status_of_launch(stream, &prm.status));
    prm.wait_limit_ns = wait_limit_ns();
    CUtensorMap ma;
    if (!encode_2d(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->values, d.pitch, d.m, d.pitch, kNarrowStage / 2, rows_of_box(0, prm.at_once * 16u), CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) {
        set_last_error_static("a tensor map of a 4-bit matrix could not be made");
        return B200SPMM_ERR_CUDA;
    }
    B200_CUDA_TRY(launch_after(kernel, dim3(share.blocks, passes), 32 * (warps + kNarrowLoaders), 1280u + prm.stages * stage + sums, 1, stream, ma, prm));
    return B200SPMM_OK;
}

template <typename T, bool kMx, bool kTokens>
int launch_narrow_columns(const b200spmm_fp4_t *a, const DenseParams &d, cudaStream_t stream) {
    if (d.c.type == B200SPMM_T_F32) return d.n <= 8 ? launch_narrow<T, kMx, 1, kTokens, true>(a, d, stream) : launch_narrow<T, kMx, 2, kTokens, true>(a, d, stream);
    return d.n <= 8 ? launch_narrow<T, kMx, 1, kTokens, false>(a, d, stream) : launch_narrow<T, kMx, 2, kTokens, false>(a, d, stream);
}

// Columns shared out evenly over as few tiles as there can be, 64 at least (fewer take longer: 24 with 28672 x 8192 88 us as 32, 66 as 64); a
// part has at least four steps, 512 values of k: shorter ones are not worth their sums' way through memory.  A step of tiles that fill the GPU (18,944
// rows, 12,288 values of k less 4,096) measured 0.34 us with 64 columns, 0.43 with 128, 0.62 with 192 and 0.74 with 256 in 16 bits, 0.53 to 0.66 for an
// fp32 C; the estimates are up to a quarter below that, so that tiles are cut a little later than they might.
Split wide_split(uint32_t m, uint32_t n, uint32_t k, bool exact, uint32_t pairs) {
    const uint32_t most = exact ? WideCfg::kExactCols : kPairCols4, tiles_n = (n + most - 1) / most, cols = std::max(64u, ((n + tiles_n - 1) / tiles_n + 31u) / 32u * 32u);
    return make_split(m, n, cols, (k + kWideK - 1) / kWideK, 4, 0.55, exact ? 0.6 : cols <= WideCfg::kTwoCols ? 0.33 : 0.5, 256 * kWideK * 2, pairs);
}

// Pairs of CTAs of the wide kernel that the current device runs at once (its instances take the same room).
int wide_pairs(int device, uint32_t *out) {
    static std::atomic<uint32_t> known[kMaxDevices];
    return max_pairs(fp4_wide_kernel<__half, false, true, false>, WideCfg::kThreads, WideCfg::kSmemBytes, known[device], out);
}

template <typename T, bool kMx, bool kTokens, bool kExact>
int launch_wide(const b200spmm_fp4_t *a, const DenseParams &d, float *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
    uint32_t pairs = 0;
    const int st = wide_pairs(a->device, &pairs);
    if (st != B200SPMM_OK) return st;
    auto kernel = fp4_wide_kernel<T, kMx, kTokens, kExact>;
    static thread_local int configured = -1;
    if (configured != a->device) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WideCfg::kSmemBytes));
        configured = a->device;
    }
    WideParams prm{};
    prm.d = d;
    prm.split = wide_split(d.m, d.n, d.k, kExact, pairs);
    if (prm.split.parts > 1 && (!workspace || workspace_bytes < split_workspace(prm.split))) prm.split = wide_split(d.m, d.n, d.k, kExact, 1);
    prm.row_blocks = (d.m + 127u) / 128u;
    prm.stages_a = WideCfg::stages_a(kTokens, kExact, prm.split.cols);
    prm.stages_b = WideCfg::stages_b(kTokens, kExact, prm.split.cols);
    prm.partial = workspace;
    B200_CUDA_TRY(status_of_launch(stream, &prm.status));
    prm.wait_limit_ns = wait_limit_ns();
    CUtensorMap ma, mb;
    const auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t pitch_b = (d.n > 1 || !kTokens) && (d.k > 1 || kTokens) ? (uint64_t)d.ldb * 2u : ((uint64_t)(kTokens ? d.k : d.n) * 2u + 15u) / 16u * 16u;
    if (!encode_2d(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->values, d.pitch, d.m, d.pitch, kWideK / 2, rows_of_box(0, 128), CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
        !encode_2d(&mb, type, d.b, kTokens ? d.k : d.n, kTokens ? d.n : d.k, pitch_b, 64, rows_of_box(1, kTokens ? prm.split.cols / 2u : kWideK), CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) {
        set_last_error_static("a tensor map of a product with a 4-bit matrix could not be made");
        return B200SPMM_ERR_CUDA;
    }
    B200_CUDA_TRY(launch_after(kernel, dim3(2 * std::min(pairs, prm.split.items)), WideCfg::kThreads, WideCfg::smem_bytes(kTokens, kExact, prm.split.cols), 2, stream, ma, mb, prm));
    if (prm.split.parts > 1)
        B200_CUDA_TRY(launch_after(fp4_join_kernel, dim3((prm.split.items - prm.split.whole) / prm.split.parts, prm.split.cols / kJoinCols), kPairRows4, 0, 1, stream, prm.split,
                                   (const float *)workspace, d.m, d.n, kMx ? (const float *)nullptr : d.whole, (const float *)nullptr, Widen<T, kMx>::kLeft, d.c));
    return B200SPMM_OK;
}

// B, whose rows start anywhere, with rows that start on 16 bytes.
__global__ void __launch_bounds__(256) fp4_align_kernel(const uint16_t *src, int64_t ld, uint32_t rows, uint32_t cols, uint4 *dst, uint32_t pieces) {
    ptx::wait_for_grids_before();
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < (uint64_t)rows * pieces; i += (uint64_t)gridDim.x * 256u) {
        const uint32_t row = (uint32_t)(i / pieces), col = (uint32_t)(i % pieces) * 8u;
        const uint16_t *from = src + (int64_t)row * ld + col;
        alignas(16) uint16_t v[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = col + e < cols ? from[e] : (uint16_t)0;
        dst[i] = *reinterpret_cast<const uint4 *>(v);
    }
}

// Up to 16 columns go to the narrow kernel (9 to 16 take either one 44 to 48 us with 28672 x 8192 in fp16), which reads any B, though rows that
// start anywhere element by element.  From some 16,000 elements on, those that a block then reads one by one (8 a row of few columns), a
// copy pays: 28672 x 8192 x 9 columns 88 -> 48 us, 4096 x 2048 x 3 11.1 -> 9.1, but 3 tokens there 7.1 -> 8.2.
constexpr uint32_t kNarrowColumns = 16;
constexpr uint64_t kCopyFrom = 16384;
// Whether B's rows, as they lie, start on 16 bytes; a single column's neighbours are one row.
bool rows_aligned(const void *b, int64_t ldb, int64_t n, bool b_transposed) { return reinterpret_cast<uintptr_t>(b) % 16u == 0 && (ldb % 8 == 0 || (n == 1 && b_transposed)); }
void one_column(int64_t n, int64_t *ldb, bool *b_transposed, uint32_t k) {
    if (n != 1 || *b_transposed || *ldb != 1) return;
    *b_transposed = true;
    *ldb = k;
}
// Pieces of 16 bytes of a row of the copy: whole lines of 128, of which boxes then touch no more than they have to, and single ones for the narrow kernel.
uint64_t aligned_pieces(uint64_t cols) { return cols <= kNarrowColumns ? (cols + 7u) / 8u : (cols + 63u) / 64u * 8u; }
uint64_t aligned_bytes(uint64_t rows, uint64_t cols) { return rows * aligned_pieces(cols) * 16u; }

template <typename T, bool kMx, bool kTokens>
int launch_dense(const b200spmm_fp4_t *a, const DenseParams &d, uint8_t *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
    const uint64_t rows = kTokens ? d.n : d.k, cols = kTokens ? d.k : d.n, need = aligned_bytes(rows, cols);
    const bool copy = !d.b_wide && workspace && workspace_bytes >= need && (d.n > kNarrowColumns || (uint64_t)d.k * (kTokens ? d.n : 8u) >= kCopyFrom);
    if (!copy && (d.n <= kNarrowColumns || !d.b_wide)) return launch_narrow_columns<T, kMx, kTokens>(a, d, stream);
    auto wide = [&](const DenseParams &with, uint8_t *ws, uint64_t bytes) {
        return with.c.type == B200SPMM_T_F32 ? launch_wide<T, kMx, kTokens, true>(a, with, reinterpret_cast<float *>(ws), bytes, stream)
                                             : launch_wide<T, kMx, kTokens, false>(a, with, reinterpret_cast<float *>(ws), bytes, stream);
    };
    if (!copy) return wide(d, workspace, workspace_bytes);
    // no tensor map describes B: a copy that one does goes first into the workspace
    const uint32_t pieces = (uint32_t)aligned_pieces(cols);
    B200_CUDA_TRY(launch_after(fp4_align_kernel, dim3((unsigned)std::min<uint64_t>((rows * pieces + 255u) / 256u, (uint64_t)sm_count() * 8u)), 256, 0, 1, stream,
                               reinterpret_cast<const uint16_t *>(d.b), d.ldb, (uint32_t)rows, (uint32_t)cols, reinterpret_cast<uint4 *>(workspace), pieces));
    DenseParams with = d;
    with.b = workspace;
    with.ldb = (int64_t)pieces * 8;
    with.b_wide = true;
    if (d.n <= kNarrowColumns) return launch_narrow_columns<T, kMx, kTokens>(a, with, stream);
    return wide(with, workspace + need, workspace_bytes - need);
}

}  // namespace

int dense_product_workspace(const b200spmm_fp4_t *a, const void *b, int64_t ldb, int64_t n, bool b_transposed, uint64_t *bytes) {
    *bytes = 0;
    const uint32_t m = (uint32_t)a->rows, k = (uint32_t)a->cols;
    if (n > kNarrowColumns) {
        uint32_t pairs = 0;
        const int st = wide_pairs(a->device, &pairs);
        if (st != B200SPMM_OK) return st;
        *bytes = std::max(split_workspace(wide_split(m, (uint32_t)n, k, false, pairs)), split_workspace(wide_split(m, (uint32_t)n, k, true, pairs)));
    }
    one_column(n, &ldb, &b_transposed, k);
    if (!rows_aligned(b, ldb, n, b_transposed)) *bytes += aligned_bytes(b_transposed ? (uint64_t)n : a->cols, b_transposed ? a->cols : (uint64_t)n);
    return B200SPMM_OK;
}

int launch_dense_product(const b200spmm_fp4_t *a, const void *b, int64_t ldb, int64_t n, int b_dtype, bool b_transposed, void *c, int64_t ldc, int c_dtype,
                         bool c_transposed, uint8_t *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
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
    one_column(n, &ldb, &b_transposed, prm.k);
    prm.ldb = ldb;
    prm.n = (uint32_t)n;
    prm.b_wide = rows_aligned(b, ldb, n, b_transposed);
    prm.c = target_of(c, ldc, c_dtype, c_transposed);
    auto run = [&](auto type, auto mx) {
        using T = decltype(type);
        constexpr bool kMx = decltype(mx)::value;
        return b_transposed ? launch_dense<T, kMx, true>(a, prm, workspace, workspace_bytes, stream)
                            : launch_dense<T, kMx, false>(a, prm, workspace, workspace_bytes, stream);
    };
    if (a->format == B200SPMM_MXFP4) return run(__nv_bfloat16(), std::true_type());
    return b_dtype == B200SPMM_T_F16 ? run(__half(), std::false_type()) : run(__nv_bfloat16(), std::false_type());
}

}  // namespace fp4
}  // namespace b200spmm

/* Declared in b200_spmm_kat.h: how a product with few 16-bit columns is shared out. */
extern "C" int b200spmm_kat_fp4_narrow_share(uint64_t rows, uint64_t cols, uint32_t sms, uint32_t *blocks, uint32_t *rounds, uint32_t *at_once, uint32_t *slices) {
    using namespace b200spmm::fp4;
    if (!rows || !cols || rows > 0x7FFFFFFFull - 128 || cols > 0x7FFFFFFFull - 256 || !sms || !blocks || !rounds || !at_once || !slices) return B200SPMM_ERR_INVALID_ARG;
    const NarrowShare s = narrow_share((uint32_t)((rows + 15) / 16), (uint32_t)cols, sms);
    *blocks = s.blocks;
    *rounds = s.rounds;
    *at_once = s.at_once;
    *slices = s.slices;
    return B200SPMM_OK;
}
