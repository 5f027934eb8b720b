// Product of two 4-bit matrices on the block-scaled tensor core (layout: fp4.hpp).
//
//     C[m, n] = s_A s_B  sum over k  (a[m, k] sa[m, k / block]) (b[n, k] sb[n, k / block])
//
// tcgen05.mma takes 128 rows of A, up to 256 of B and 64 values of k a call and applies the scales itself.  A block of
// threads makes a tile of C: one thread brings stages of 256 values of k (128 bytes of a row: one swizzled TMA box an operand,
// and the scales, which lie as they are needed, by bulk copies), one thread copies the scales to tensor memory and issues the
// MMAs, four warps take the finished accumulator to C.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "fp4.hpp"
#include "fp4_convert.cuh"
#include "fp4_store.cuh"
#include "launch.hpp"
#include "tensormap.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

constexpr uint32_t kTileM = 128, kStageK = 256, kMmaK = 64;
constexpr unsigned long long kLingerNs = 20000000ull;  // after a wait that ran out: what was under way to shared memory arrives

struct ProductParams {
    const uint8_t *a_scales, *b_scales;
    const float *a_whole, *b_whole;
    uint32_t m, n, k, groups;
    Target c;
    uint32_t *status;
    unsigned long long wait_limit_ns;
};

template <bool kMx, int kN>
struct ProductCfg {
    static constexpr uint32_t kGroupsPerStage = kMx ? 2 : 4;                   // scale groups of a stage
    static constexpr uint32_t kBlocksB = (kN + 127) / 128;                     // 128-row blocks of B's scales
    static constexpr uint32_t kBytesA = kTileM * kStageK / 2, kBytesB = kN * kStageK / 2;
    static constexpr uint32_t kScaleBytesA = kGroupsPerStage * 512, kScaleBytesB = kBlocksB * kScaleBytesA;
    static constexpr uint32_t kStageBytes = kBytesA + kBytesB + kScaleBytesA + kScaleBytesB;
    static constexpr uint32_t kPerSm = kN <= 64 ? 2 : 1;                       // resident blocks
    static constexpr uint32_t kStages = (kPerSm == 2 ? 110u * 1024u : 220u * 1024u) / kStageBytes < 6 ? (kPerSm == 2 ? 110u * 1024u : 220u * 1024u) / kStageBytes : 6;
    static constexpr uint32_t kScaleCols = kGroupsPerStage * 4 * (1 + kBlocksB);  // tensor memory columns of a stage's scales
    static constexpr uint32_t kNeedCols = kN + kStages * kScaleCols;
    static constexpr uint32_t kTmemCols = kNeedCols <= 64 ? 64 : kNeedCols <= 128 ? 128 : kNeedCols <= 256 ? 256 : 512;
    static_assert(kNeedCols <= 512 && kTmemCols * kPerSm <= 512 && kStages >= 3, "tensor memory of an SM");
    static constexpr int kThreads = 192;  // warps 0-3: epilogue, 4: loads, 5: MMAs
    static constexpr size_t kSmemBytes = 1024 + (size_t)kStages * kStageBytes + (2 * kStages + 1) * 8 + 16;
};

template <bool kMx, int kN>
__global__ void __launch_bounds__((ProductCfg<kMx, kN>::kThreads), (ProductCfg<kMx, kN>::kPerSm))
fp4_product_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const ProductParams p) {
    using Cfg = ProductCfg<kMx, kN>;
    constexpr uint32_t kStages = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t *base = smem_raw + pad;
    const uint32_t a_addr = raw_addr + pad, b_addr = a_addr + kStages * Cfg::kBytesA, sa_addr = b_addr + kStages * Cfg::kBytesB,
                   sb_addr = sa_addr + kStages * Cfg::kScaleBytesA;
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + (size_t)kStages * Cfg::kStageBytes);
    const uint32_t bars_addr = ptx::smem_u32(bars);
    auto full_bar = [&](uint32_t s) { return bars_addr + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bars_addr + 8u * (kStages + s); };
    const uint32_t done_bar = bars_addr + 8u * 2u * kStages;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(bars + 2 * kStages + 1);
    uint32_t *tmem_slot = const_cast<uint32_t *>(abort_flag) + 1;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint64_t limit = p.wait_limit_ns;
    const uint32_t n0 = blockIdx.x * kN, m0 = blockIdx.y * kTileM;
    const uint32_t n_stages = (p.k + kStageK - 1) / kStageK;

    if (tid == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(done_bar, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
    }
    if (warp == 5) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), Cfg::kTmemCols);
        ptx::tmem_relinquish_alloc_permit();
    }
    ptx::wait_for_grids_before();
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot, tmem_scales = tmem + kN;

    if (warp == 4) {
        if (lane == 0) {
            for (uint32_t it = 0; it < n_stages; ++it) {
                const uint32_t s = it % kStages;
                if (!ptx::mbar_wait(empty_bar(s), (it / kStages & 1u) ^ 1u, abort_flag, limit)) break;
                const uint32_t g0 = it * Cfg::kGroupsPerStage, bytes = min(Cfg::kGroupsPerStage, p.groups - g0) * 512u;
                uint32_t n_blocks = 0;
#pragma unroll
                for (uint32_t j = 0; j < Cfg::kBlocksB; ++j) n_blocks += n0 + j * 128u < p.n ? 1u : 0u;
                ptx::mbar_arrive_expect_tx(full_bar(s), Cfg::kBytesA + Cfg::kBytesB + bytes * (1u + n_blocks));
                ptx::tma_load_2d(a_addr + s * Cfg::kBytesA, &tmap_a, (int32_t)(it * (kStageK / 2)), (int32_t)m0, full_bar(s));
                ptx::tma_load_2d(b_addr + s * Cfg::kBytesB, &tmap_b, (int32_t)(it * (kStageK / 2)), (int32_t)n0, full_bar(s));
                ptx::bulk_load(sa_addr + s * Cfg::kScaleBytesA, p.a_scales + ((uint64_t)(m0 / 128u) * p.groups + g0) * 512u, bytes, full_bar(s));
                for (uint32_t j = 0; j < n_blocks; ++j)
                    ptx::bulk_load(sb_addr + s * Cfg::kScaleBytesB + j * Cfg::kScaleBytesA, p.b_scales + ((uint64_t)(n0 / 128u + j) * p.groups + g0) * 512u, bytes, full_bar(s));
            }
        }
    } else if (warp == 5) {
        if (lane == 0) {
            const uint64_t a_desc0 = ptx::make_smem_desc(a_addr, 16, 1024, ptx::kSwizzle128B), b_desc0 = ptx::make_smem_desc(b_addr, 16, 1024, ptx::kSwizzle128B);
            const uint64_t sa_desc0 = ptx::make_smem_desc(sa_addr, 0, 128, ptx::kSwizzleNone), sb_desc0 = ptx::make_smem_desc(sb_addr, 0, 128, ptx::kSwizzleNone);
            bool alive = true;
            for (uint32_t it = 0; it < n_stages; ++it) {
                const uint32_t s = it % kStages;
                alive = ptx::mbar_wait(full_bar(s), it / kStages & 1u, abort_flag, limit);
                if (!alive) break;
                ptx::tcgen05_fence_after_sync();
                const uint32_t steps = min(kStageK / kMmaK, (p.k - it * kStageK + kMmaK - 1) / kMmaK);
                const uint32_t n_groups = min(Cfg::kGroupsPerStage, p.groups - it * Cfg::kGroupsPerStage);
                // A stage's scales have columns of their own: they are overwritten when the stage is, after its MMAs
                const uint32_t sa = tmem_scales + s * Cfg::kScaleCols, sb = sa + Cfg::kGroupsPerStage * 4u;
                for (uint32_t g = 0; g < n_groups; ++g) {
                    ptx::tmem_copy_scales(sa + g * 4u, sa_desc0 + ((s * Cfg::kScaleBytesA + g * 512u) >> 4));
#pragma unroll
                    for (uint32_t j = 0; j < Cfg::kBlocksB; ++j)
                        ptx::tmem_copy_scales(sb + (g * Cfg::kBlocksB + j) * 4u, sb_desc0 + ((s * Cfg::kScaleBytesB + j * Cfg::kScaleBytesA + g * 512u) >> 4));
                }
                for (uint32_t i = 0; i < steps; ++i) {
                    const uint32_t g = kMx ? i / 2 : i, id = kMx ? (i & 1u) * 2u : 0u;
                    ptx::umma_fp4_ss<kMx>(tmem, a_desc0 + ((s * Cfg::kBytesA + i * 32u) >> 4), b_desc0 + ((s * Cfg::kBytesB + i * 32u) >> 4),
                                          ptx::make_fp4_instr_desc(kMx, kTileM, kN, id), sa + g * 4u, sb + g * Cfg::kBlocksB * 4u, (it | i) ? 1u : 0u);
                }
                ptx::umma_commit(empty_bar(s));
            }
            ptx::umma_commit(done_bar);
            if (!alive) ptx::mbar_wait_bounded(done_bar, 0, limit);
        }
    } else {
        const Factor f(*reinterpret_cast<const volatile float *>(p.a_whole), *reinterpret_cast<const volatile float *>(p.b_whole));
        uint32_t ok = 1;
        if (lane == 0) ok = ptx::mbar_wait(done_bar, 0, abort_flag, limit) ? 1u : 0u;
        ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
        if (ok && !*abort_flag) {
            ptx::tcgen05_fence_after_sync();
            const uint32_t row = m0 + (uint32_t)warp * 32u + (uint32_t)lane;
            constexpr uint32_t kCols = kN < 32 ? 16 : 32;
#pragma unroll 1
            for (uint32_t c = 0; c < (uint32_t)kN && n0 + c < p.n; c += kCols) {
                uint32_t r[kCols];
                if constexpr (kCols == 16) ptx::tmem_ld_32x32b_x16(tmem + (((uint32_t)warp * 32u) << 16) + c, r);
                else ptx::tmem_ld_32x32b_x32(tmem + (((uint32_t)warp * 32u) << 16) + c, r);
                ptx::tmem_ld_wait();
                float v[kCols];
#pragma unroll
                for (uint32_t i = 0; i < kCols; ++i) v[i] = f.apply(__uint_as_float(r[i]));
                if (row < p.m) store_row(p.c, row, n0 + c, p.n, v);
            }
        }
    }
    __syncwarp();
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = ptx::global_timer_ns();
        while (ptx::global_timer_ns() - t0 < kLingerNs) __nanosleep(1000);
        if (tid == 0) atomicOr(p.status, kDevStatusTimeout);
        __syncthreads();
    }
    if (warp == 5) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

// Values as bytes, boxes of 128 of a row: what lies past the matrix arrives as zeros.
bool encode_values(CUtensorMap *map, const b200spmm_fp4_t *x, const Layout &l, uint32_t box_rows) {
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, x->values, l.pitch, x->rows, l.pitch, kStageK / 2, box_rows, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

template <bool kMx, int kN>
int launch_width(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, const ProductParams &prm, cudaStream_t stream) {
    using Cfg = ProductCfg<kMx, kN>;
    auto kernel = fp4_product_kernel<kMx, kN>;
    static thread_local int configured = -1;
    if (configured != a->device) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmemBytes));
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        configured = a->device;
    }
    CUtensorMap ma, mb;
    if (!encode_values(&ma, a, layout_of(a->rows, a->cols, a->format), kTileM) || !encode_values(&mb, b, layout_of(b->rows, b->cols, b->format), kN)) {
        set_last_error_static("a tensor map of a 4-bit matrix could not be made");
        return B200SPMM_ERR_CUDA;
    }
    const dim3 grid((prm.n + kN - 1) / kN, (prm.m + kTileM - 1) / kTileM);
    if (grid.y > 65535u) return B200SPMM_ERR_UNSUPPORTED;
    B200_CUDA_TRY(launch_after(kernel, grid, Cfg::kThreads, Cfg::kSmemBytes, 1, stream, ma, mb, prm));
    return B200SPMM_OK;
}

template <bool kMx>
int launch_format(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, const ProductParams &prm, cudaStream_t stream) {
    if (prm.n <= 16) return launch_width<kMx, 16>(a, b, prm, stream);
    if (prm.n <= 32) return launch_width<kMx, 32>(a, b, prm, stream);
    if (prm.n <= 64) return launch_width<kMx, 64>(a, b, prm, stream);
    if (prm.n <= 128) return launch_width<kMx, 128>(a, b, prm, stream);
    return launch_width<kMx, 256>(a, b, prm, stream);
}

}  // namespace

int launch_product(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, void *c, int64_t ldc, int c_dtype, bool c_transposed, cudaStream_t stream) {
    // C^T = B A^T: the longer side of C goes to the 128 rows of the MMA, the shorter one to its columns, which may be few
    if (a->rows < b->rows) {
        std::swap(a, b);
        c_transposed = !c_transposed;
    }
    ProductParams prm{};
    prm.a_scales = static_cast<const uint8_t *>(a->scales);
    prm.b_scales = static_cast<const uint8_t *>(b->scales);
    prm.a_whole = a->tensor_scale;
    prm.b_whole = b->tensor_scale;
    prm.m = (uint32_t)a->rows;
    prm.n = (uint32_t)b->rows;
    prm.k = (uint32_t)a->cols;
    prm.groups = layout_of(a->rows, a->cols, a->format).groups;
    prm.c = target_of(c, ldc, c_dtype, c_transposed);
    B200_CUDA_TRY(status_word(&prm.status));
    prm.wait_limit_ns = kDeviceWaitLimitNs;
    return a->format == B200SPMM_MXFP4 ? launch_format<true>(a, b, prm, stream) : launch_format<false>(a, b, prm, stream);
}

}  // namespace fp4
}  // namespace b200spmm
