// Product of two 4-bit matrices on the block-scaled tensor core (layout: fp4.hpp).
//
//     C[m, n] = s_A s_B  sum over k  (a[m, k] sa[m, k / block]) (b[n, k] sb[n, k / block])
//
// Two kernels.  Few columns (up to 64, decoding): blocks of threads of their own, below; bound by one read of the longer operand (28672 x 8192
// nvfp4 x 8 columns 24 us, 5.6 TB/s).
// More: pairs of CTAs (fp4_product_pair.cuh).
//
// tcgen05.mma takes 128 rows of A, up to 256 of B and 64 values of k a call and applies the scales itself.  A block of
// threads makes a tile of C: one thread brings stages of 256 values of k (128 bytes of a row: one swizzled TMA box an operand,
// and the scales, which lie as they are needed, by bulk copies), four warps bring the scales to tensor memory and at the end
// the accumulator to C, one thread issues the MMAs.
#include <algorithm>
#include <atomic>

#include "common.hpp"
#include "fp4.hpp"
#include "fp4_convert.cuh"
#include "fp4_product_pair.cuh"
#include "launch.hpp"
#include "tensormap.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

constexpr uint32_t kTileM = 128;

template <bool kMx, int kN>
struct ProductCfg {
    static_assert(kN <= 64, "wider ones are made by pairs");
    static constexpr uint32_t kGroupsPerStage = kMx ? 2 : 4;                   // scale groups of a stage
    static constexpr uint32_t kBytesA = kTileM * kStageK / 2, kBytesB = kN * kStageK / 2;
    static constexpr uint32_t kScaleBytesA = kGroupsPerStage * 512, kScaleBytesB = kScaleBytesA;
    static constexpr uint32_t kStageBytes = kBytesA + kBytesB + kScaleBytesA + kScaleBytesB;
    static constexpr uint32_t kPerSm = 2;                                      // resident blocks
    static constexpr uint32_t kStages = 110u * 1024u / kStageBytes < 6 ? 110u * 1024u / kStageBytes : 6;
    static constexpr uint32_t kScaleCols = kGroupsPerStage * 8;  // tensor memory columns of a stage's scales
    static constexpr uint32_t kNeedCols = kN + kStages * kScaleCols;
    static constexpr uint32_t kTmemCols = kNeedCols <= 64 ? 64 : kNeedCols <= 128 ? 128 : kNeedCols <= 256 ? 256 : 512;
    static_assert(kNeedCols <= 512 && kTmemCols * kPerSm <= 512 && kStages >= 3, "tensor memory of an SM");
    static constexpr int kThreads = 192;  // warps 0-3: epilogue, 4: loads, 5: MMAs
    static constexpr size_t kSmemBytes = 1024 + (size_t)kStages * kStageBytes + (3 * kStages + 1) * 8 + 16;
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
    auto ready_bar = [&](uint32_t s) { return bars_addr + 8u * (2 * kStages + s); };
    const uint32_t done_bar = bars_addr + 8u * 3u * kStages;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(bars + 3 * kStages + 1);
    uint32_t *tmem_slot = const_cast<uint32_t *>(abort_flag) + 1;

    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;  // (the shuffle: a warp is known to be one)
    const uint64_t limit = p.wait_limit_ns;
    const uint32_t m0 = blockIdx.x * kTileM;
    const uint32_t n_stages = (p.k + kStageK - 1) / kStageK;

    if (tid == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
            ptx::mbar_init(ready_bar(s), 4);
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
        const uint32_t on = lane == 0 ? 1u : 0u;
        const uint8_t *scales = p.a_scales + (uint64_t)(m0 / 128u) * p.groups * 512u;
        uint32_t s = 0, phase = 1;
        for (uint32_t it = 0; it < n_stages; ++it) {
            if (!__all_sync(0xFFFFFFFFu, ptx::mbar_wait(empty_bar(s), phase, abort_flag, limit))) break;
            const uint32_t g0 = it * Cfg::kGroupsPerStage, bytes = min(Cfg::kGroupsPerStage, p.groups - g0) * 512u;
            ptx::mbar_arrive_expect_tx_if(on, full_bar(s), Cfg::kBytesA + Cfg::kBytesB + bytes * 2u);
            ptx::tma_load_2d_if(on, a_addr + s * Cfg::kBytesA, &tmap_a, (int32_t)(it * (kStageK / 2)), (int32_t)m0, full_bar(s));
            ptx::bulk_load_if(on, sa_addr + s * Cfg::kScaleBytesA, scales + (uint64_t)g0 * 512u, bytes, full_bar(s));
            ptx::tma_load_2d_if(on, b_addr + s * Cfg::kBytesB, &tmap_b, (int32_t)(it * (kStageK / 2)), 0, full_bar(s));
            ptx::bulk_load_if(on, sb_addr + s * Cfg::kScaleBytesB, p.b_scales + (uint64_t)g0 * 512u, bytes, full_bar(s));
            s = s + 1 == kStages ? 0u : s + 1;
            phase ^= s == 0 ? 1u : 0u;
        }
    } else if (warp == 5) {
        const uint32_t on = lane == 0 ? 1u : 0u;
        const uint64_t a_desc = ptx::make_smem_desc(a_addr, 16, 1024, ptx::kSwizzle128B), b_desc = ptx::make_smem_desc(b_addr, 16, 1024, ptx::kSwizzle128B);
        const uint32_t a_lo = (uint32_t)a_desc, a_hi = (uint32_t)(a_desc >> 32), b_lo = (uint32_t)b_desc, b_hi = (uint32_t)(b_desc >> 32);
        bool alive = true;
        uint32_t s = 0, phase = 0, left = p.k;
        for (uint32_t it = 0; it < n_stages; ++it) {
            alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait(ready_bar(s), phase, abort_flag, limit));
            if (!alive) break;
            ptx::tcgen05_fence_after_sync();
            const uint32_t sa = tmem_scales + s * Cfg::kScaleCols, sb = sa + Cfg::kGroupsPerStage * 4u;
            const uint32_t a = a_lo + s * (Cfg::kBytesA >> 4), b = b_lo + s * (Cfg::kBytesB >> 4);
            constexpr uint32_t idesc = ptx::make_fp4_instr_desc(kMx, kTileM, kN, 0);
            if (left >= kStageK) {
                ptx::umma_fp4_ss_x4_if<kMx, 1>(on, tmem, a, a_hi, b, b_hi, idesc, sa, sb, 4, it ? 1u : 0u);
            } else {
                for (uint32_t i = 0; i * kMmaK < left; ++i) {
                    const uint32_t g = kMx ? i / 2 : i;
                    ptx::umma_fp4_ss_if<kMx, 1>(on, tmem, a + i * 2u, a_hi, b + i * 2u, b_hi, kMx && i % 2 ? idesc | ptx::kSecondScales : idesc, sa + g * 4u, sb + g * 4u, (it | i) ? 1u : 0u);
                }
            }
            ptx::umma_commit_if(on, empty_bar(s));
            left -= kStageK;
            s = s + 1 == kStages ? 0u : s + 1;
            phase ^= s == 0 ? 1u : 0u;
        }
        ptx::umma_commit_if(on, done_bar);
        if (!alive && on) ptx::mbar_wait_bounded(done_bar, 0, limit);
    } else {
        const uint32_t lanes = ((uint32_t)warp * 32u) << 16;
        for (uint32_t it = 0; it < n_stages; ++it) {
            const uint32_t s = it % kStages;
            uint32_t ok = 1;
            if (lane == 0) ok = ptx::mbar_wait(full_bar(s), it / kStages & 1u, abort_flag, limit) ? 1u : 0u;
            if (!__shfl_sync(0xFFFFFFFFu, ok, 0)) break;
            // A stage's scales have columns of their own: they are overwritten when the stage is, after its MMAs
            uint4 a[Cfg::kGroupsPerStage], b[Cfg::kGroupsPerStage];
#pragma unroll
            for (uint32_t g = 0; g < Cfg::kGroupsPerStage; ++g) {
                a[g] = ptx::ld_shared_v4(sa_addr + s * Cfg::kScaleBytesA + g * 512u + (uint32_t)lane * 16u);
                b[g] = ptx::ld_shared_v4(sb_addr + s * Cfg::kScaleBytesB + g * 512u + (uint32_t)lane * 16u);
            }
            ptx::tcgen05_fence_after_sync();
            ptx::tmem_st_v4(tmem_scales + lanes + s * Cfg::kScaleCols, a);
            ptx::tmem_st_v4(tmem_scales + lanes + s * Cfg::kScaleCols + Cfg::kGroupsPerStage * 4u, b);
            ptx::tmem_st_wait();
            ptx::tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ready_bar(s));
        }
        const Factor f(p.a_whole ? *reinterpret_cast<const volatile float *>(p.a_whole) : 1.f, p.b_whole ? *reinterpret_cast<const volatile float *>(p.b_whole) : 1.f);
        uint32_t ok = 1;
        if (lane == 0) ok = ptx::mbar_wait(done_bar, 0, abort_flag, limit) ? 1u : 0u;
        ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
        if (ok && !*abort_flag) {
            ptx::tcgen05_fence_after_sync();
            const uint32_t row = m0 + (uint32_t)warp * 32u + (uint32_t)lane;
            constexpr uint32_t kCols = kN < 32 ? 16 : 32;
#pragma unroll 1
            for (uint32_t c = 0; c < (uint32_t)kN && c < p.n; c += kCols) {
                uint32_t r[kCols];
                if constexpr (kCols == 16) ptx::tmem_ld_32x32b_x16(tmem + (((uint32_t)warp * 32u) << 16) + c, r);
                else ptx::tmem_ld_32x32b_x32(tmem + (((uint32_t)warp * 32u) << 16) + c, r);
                ptx::tmem_ld_wait();
                float v[kCols];
#pragma unroll
                for (uint32_t i = 0; i < kCols; ++i) v[i] = f.apply(__uint_as_float(r[i]));
                if (row < p.m) store_row(p.c, row, c, p.n, v);
            }
        }
    }
    __syncwarp();
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = ptx::global_timer_ns();
        while (ptx::global_timer_ns() - t0 < kLingerNs) __nanosleep(1000);
        if (tid == 0) atomicAdd(p.status, 1u);
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
    if (!encode_values(&ma, a, layout_of(a->rows, a->cols, a->format), rows_of_box(0, kTileM)) || !encode_values(&mb, b, layout_of(b->rows, b->cols, b->format), rows_of_box(1, kN))) {
        set_last_error_static("a tensor map of a 4-bit matrix could not be made");
        return B200SPMM_ERR_CUDA;
    }
    B200_CUDA_TRY(launch_after(kernel, dim3((prm.m + kTileM - 1) / kTileM), Cfg::kThreads, Cfg::kSmemBytes, 1, stream, ma, mb, prm));
    return B200SPMM_OK;
}

// Tiles of 128 or 256 columns, the scales' blocks being 128 rows long, with fewer columns past the end; a single tile as wide as it has to be.
// A step of 256 values of k of tiles that fill the GPU (18,944 rows) measured 0.56 us with 96 columns and 0.63 with 256 in nvfp4, 0.53 and 0.60 in mxfp4;
// the estimates are a third below that, so that tiles are cut a little later than they might; a part has at least 512 values of k.
Split pair_split(uint32_t m, uint32_t n, uint32_t k, uint32_t pairs) {
    const uint32_t cols = n <= kPairCols4 ? (n + 31u) / 32u * 32u : (n + 127u) / 128u * 128u < (n + 255u) / 256u * 256u ? 128u : 256u;
    return make_split(m, n, cols, (k + kStageK - 1) / kStageK, 2, 0.45, 0.35, 256 * kStageK * 9 / 16, pairs);
}

int product_pairs(int device, uint32_t *out) {
    static std::atomic<uint32_t> known[kMaxDevices];
    return max_pairs(fp4_product_pair_kernel<false>, PairCfg4<false>::kThreads, PairCfg4<false>::kSmemBytes, known[device], out);
}

template <bool kMx>
int launch_pairs(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, const ProductParams &from, float *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
    using Cfg = PairCfg4<kMx>;
    uint32_t pairs = 0;
    const int st = product_pairs(a->device, &pairs);
    if (st != B200SPMM_OK) return st;
    auto kernel = fp4_product_pair_kernel<kMx>;
    static thread_local int configured = -1;
    if (configured != a->device) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmemBytes));
        configured = a->device;
    }
    ProductParams prm = from;
    prm.split = pair_split(prm.m, prm.n, prm.k, pairs);
    if (prm.split.parts > 1 && (!workspace || workspace_bytes < split_workspace(prm.split))) prm.split = pair_split(prm.m, prm.n, prm.k, 1);
    prm.partial = workspace;
    CUtensorMap ma, mb;
    if (!encode_values(&ma, a, layout_of(a->rows, a->cols, a->format), rows_of_box(0, 128)) || !encode_values(&mb, b, layout_of(b->rows, b->cols, b->format), rows_of_box(1, prm.split.cols / 2u))) {
        set_last_error_static("a tensor map of a 4-bit matrix could not be made");
        return B200SPMM_ERR_CUDA;
    }
    B200_CUDA_TRY(launch_after(kernel, dim3(2 * std::min(pairs, prm.split.items)), Cfg::kThreads, Cfg::kSmemBytes, 2, stream, ma, mb, prm));
    if (prm.split.parts > 1)
        B200_CUDA_TRY(launch_after(fp4_join_kernel, dim3((prm.split.items - prm.split.whole) / prm.split.parts, prm.split.cols / kJoinCols), kPairRows4, 0, 1, stream, prm.split,
                                   (const float *)workspace, prm.m, prm.n, prm.a_whole, prm.b_whole, 1.f, prm.c));
    return B200SPMM_OK;
}

template <bool kMx>
int launch_format(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, const ProductParams &prm, float *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
    if (prm.n <= 16) return launch_width<kMx, 16>(a, b, prm, stream);
    if (prm.n <= 32) return launch_width<kMx, 32>(a, b, prm, stream);
    if (prm.n <= 64) return launch_width<kMx, 64>(a, b, prm, stream);
    return launch_pairs<kMx>(a, b, prm, workspace, workspace_bytes, stream);
}

// Which operand gives the rows of the MMA, true: b.  C^T = B A^T, so either may.  Up to 64 columns have to be columns.  Else the rows are those
// that are neighbours in C: a warp's lanes hold them, and write 64 or 128 bytes in a row, where row by row every lane
// would write to a line of its own.
bool rows_from_b(uint64_t a_rows, uint64_t b_rows, bool c_transposed) {
    if (std::min(a_rows, b_rows) <= 64) return a_rows < b_rows;
    return !c_transposed;
}

}  // namespace

int product_workspace(const b200spmm_fp4_t *a, int64_t n, uint64_t *bytes) {
    *bytes = 0;
    if (std::min<uint64_t>(a->rows, (uint64_t)n) <= 64) return B200SPMM_OK;
    uint32_t pairs = 0;
    const int st = product_pairs(a->device, &pairs);
    if (st != B200SPMM_OK) return st;
    const uint32_t m = (uint32_t)a->rows, k = (uint32_t)a->cols;
    *bytes = std::max(split_workspace(pair_split(m, (uint32_t)n, k, pairs)), split_workspace(pair_split((uint32_t)n, m, k, pairs)));
    return B200SPMM_OK;
}

int launch_product(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, void *c, int64_t ldc, int c_dtype, bool c_transposed, float *workspace,
                   uint64_t workspace_bytes, cudaStream_t stream) {
    if (rows_from_b(a->rows, b->rows, c_transposed)) {
        std::swap(a, b);
        c_transposed = !c_transposed;
    }
    ProductParams prm{};
    prm.a_scales = static_cast<const uint8_t *>(a->scales);
    prm.b_scales = static_cast<const uint8_t *>(b->scales);
    if (a->format == B200SPMM_NVFP4) {  // (mxfp4 has no scale of the tensor)
        prm.a_whole = a->tensor_scale;
        prm.b_whole = b->tensor_scale;
    }
    prm.m = (uint32_t)a->rows;
    prm.n = (uint32_t)b->rows;
    prm.k = (uint32_t)a->cols;
    prm.groups = layout_of(a->rows, a->cols, a->format).groups;
    prm.c = target_of(c, ldc, c_dtype, c_transposed);
    B200_CUDA_TRY(status_of_launch(stream, &prm.status));
    prm.wait_limit_ns = wait_limit_ns();
    return a->format == B200SPMM_MXFP4 ? launch_format<true>(a, b, prm, workspace, workspace_bytes, stream)
                                         : launch_format<false>(a, b, prm, workspace, workspace_bytes, stream);
}

}  // namespace fp4
}  // namespace b200spmm
