// Product of two 4-bit matrices, tiles of 256 rows x up to 256 columns by pairs of CTAs (tcgen05.mma.cta_group::2).
//
// Bound: the tensor core's 4-bit rate, four times that of 16 bits, which is more than L2 feeds: a pair's tile brings 72 KB
// for 512 clocks of it, 70 bytes a clock and SM where some 51 come: 28672 x 8192 x 2,048 nvfp4 197 us (4.9 PFLOP/s), mxfp4, with half
// the scales, 186; one of 4096 in each direction 36.  The pair shares B: each CTA brings 128 rows of A, half of B's rows and all the scales of
// either.
// C lies column by column (the operands are exchanged where it does not), so that lanes, which hold rows, write neighbours.
// Warps 0-7 take accumulators to C, warps 8-15 bring scales to tensor memory (four of them a stage, each its quarter of the lanes;
// tcgen05.cp does the same, but in line with the MMAs: 110 clocks a copy of 512 bytes, twelve a stage, doubled the time),
// warp 16 of the even CTA issues the MMAs, warps 17 and 18 load.
//
//   full[s]   stage s has landed (TMA bytes, each CTA its own): the scales' warps wait for it
//   ready[s]  ... and its scales are in tensor memory, in both CTAs (eight warps arrive at the even CTA)
//   empty[s]  its MMAs are done (commit, in both CTAs)
//   done, taken  the accumulator of an item is complete (commit, in both CTAs), and has been read (16 warps arrive at the even CTA)
#pragma once

#include "fp4_split.cuh"

namespace b200spmm {
namespace fp4 {

constexpr uint32_t kStageK = 256, kMmaK = 64;
constexpr unsigned long long kLingerNs = 20000000ull;  // after a wait that ran out: what was under way to shared memory arrives

struct ProductParams {
    const uint8_t *a_scales, *b_scales;
    const float *a_whole, *b_whole;
    uint32_t m, n, k, groups;
    Target c;
    Split split;
    float *partial;
    uint32_t *status;
    unsigned long long wait_limit_ns;
};

template <bool kMx>
struct PairCfg4 {
    static constexpr uint32_t kGroups = kMx ? 2 : 4;  // of scales in a stage
    static constexpr uint32_t kBytesA = 128 * kStageK / 2, kBytesB = kPairCols4 / 2 * kStageK / 2;
    static constexpr uint32_t kScaleBytesA = kGroups * 512, kScaleBytesB = 2 * kScaleBytesA;
    static constexpr uint32_t kStageBytes = kBytesA + kBytesB + kScaleBytesA + kScaleBytesB;
    static constexpr uint32_t kStages = 5;
    static constexpr uint32_t kScaleCols = kGroups * 12;  // of tensor memory: four for A, eight for B's 256 rows, a group
    static constexpr uint32_t kTmemCols = 512;
    static constexpr int kEpilogueWarps = 8, kScaleWarps = 8, kMmaWarp = kEpilogueWarps + kScaleWarps, kThreads = 32 * (kMmaWarp + 3);
    static constexpr uint32_t kBarriers = 3 * kStages + 3;
    static constexpr size_t kSmemBytes = 1024 + (size_t)kStages * kStageBytes + kBarriers * 8 + 16;
    static_assert(kPairCols4 + kStages * kScaleCols <= kTmemCols && kSmemBytes <= 227 * 1024, "memory of an SM");
};

template <bool kMx>
__global__ void __launch_bounds__(PairCfg4<kMx>::kThreads, 1)
fp4_product_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const ProductParams p) {
    using Cfg = PairCfg4<kMx>;
    constexpr uint32_t kStages = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    // the same offsets in both CTAs: descriptors and multicast commits rely on it
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
    const uint32_t done_bar = bars_addr + 8u * 3u * kStages, taken_bar = done_bar + 8u, drain_bar = done_bar + 16u;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(bars + Cfg::kBarriers);
    uint32_t *tmem_slot = const_cast<uint32_t *>(abort_flag) + 1;

    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31u;  // (the shuffle: a warp is known to be one)
    const uint64_t limit = p.wait_limit_ns;
    const uint32_t rank = ptx::cluster_cta_rank(), pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

    if (tid == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            ptx::mbar_init(full_bar(s), 2);
            ptx::mbar_init(ready_bar(s), 8);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(done_bar, 1);
        ptx::mbar_init(taken_bar, 2 * Cfg::kEpilogueWarps);
        ptx::mbar_init(drain_bar, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
    }
    if (warp == Cfg::kMmaWarp) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), Cfg::kTmemCols);
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    ptx::wait_for_grids_before();
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive();  // the other CTA's barriers exist before anything arrives on them
    ptx::cluster_wait();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot, tmem_scales = tmem + kPairCols4;

    if (warp > Cfg::kMmaWarp) {
        // =========================================================== loads
        // One warp A and its scales, one B: an instruction holds its warp for some 130 clocks, and a stage has five.
        const uint32_t on = lane == 0 ? 1u : 0u;
        const bool is_a = warp == Cfg::kMmaWarp + 1;
        uint32_t s = 0, phase = 1;
        bool alive = true;
        for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
            const Item w = split_item(p.split, item);
            const uint32_t row_block = is_a ? w.m0 / 128u + rank : w.n0 / 128u;
            const uint32_t rows = is_a ? p.m : p.n;
            const uint32_t half = p.split.cols / 2u;
            // blocks of scales: one of A, B's all, in as far as they exist
            const uint32_t blocks = (row_block * 128u < rows ? 1u : 0u) + (!is_a && p.split.cols > 128u && (row_block + 1u) * 128u < rows ? 1u : 0u);
            const int32_t y = (int32_t)(is_a ? w.m0 + rank * 128u : w.n0 + rank * half);
            const uint32_t tile_bytes = is_a ? Cfg::kBytesA : half * 128u;
            const uint32_t dst = is_a ? a_addr : b_addr, dst_scales = is_a ? sa_addr : sb_addr;
            const uint32_t stage = is_a ? Cfg::kBytesA : Cfg::kBytesB, stage_scales = is_a ? Cfg::kScaleBytesA : Cfg::kScaleBytesB;
            const void *map = is_a ? &tmap_a : &tmap_b;
            const uint8_t *scales = (is_a ? p.a_scales : p.b_scales) + (uint64_t)row_block * p.groups * 512u;
            for (uint32_t step = w.first; step < w.last; ++step) {
                alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait(empty_bar(s), phase, abort_flag, limit));
                if (!alive) break;
                const uint32_t g0 = step * Cfg::kGroups, bytes = min(Cfg::kGroups, p.groups - g0) * 512u;
                ptx::mbar_arrive_expect_tx_if(on, full_bar(s), tile_bytes + bytes * blocks);
                ptx::tma_load_2d_if(on, dst + s * stage, map, (int32_t)(step * (kStageK / 2)), y, full_bar(s));
                ptx::bulk_load_if(on & (blocks > 0 ? 1u : 0u), dst_scales + s * stage_scales, scales + (uint64_t)g0 * 512u, bytes, full_bar(s));
                if (!is_a) ptx::bulk_load_if(on & (blocks > 1 ? 1u : 0u), dst_scales + s * stage_scales + Cfg::kScaleBytesA, scales + (uint64_t)(p.groups + g0) * 512u, bytes, full_bar(s));
                s = s + 1 == kStages ? 0u : s + 1;
                phase ^= s == 0 ? 1u : 0u;
            }
        }
    } else if (warp == Cfg::kMmaWarp) {
        // =========================================================== MMAs (even CTA)
        if (rank == 0) {
            const uint32_t on = lane == 0 ? 1u : 0u;
            const uint64_t a_desc = ptx::make_smem_desc(a_addr, 16, 1024, ptx::kSwizzle128B), b_desc = ptx::make_smem_desc(b_addr, 16, 1024, ptx::kSwizzle128B);
            const uint32_t a_lo = (uint32_t)a_desc, a_hi = (uint32_t)(a_desc >> 32), b_lo = (uint32_t)b_desc, b_hi = (uint32_t)(b_desc >> 32);
            const uint32_t idesc = ptx::make_fp4_instr_desc(kMx, kPairRows4, p.split.cols, 0);
            uint32_t s = 0, phase = 0, round = 0;
            bool alive = true;
            for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs, ++round) {
                const Item w = split_item(p.split, item);
                if (round) alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait_cluster(taken_bar, (round - 1u) & 1u, abort_flag, limit));
                uint32_t accumulate = 0, left = p.k - w.first * kStageK;  // values of k from this step on
                for (uint32_t step = w.first; alive && step < w.last; ++step) {
                    alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait_cluster(ready_bar(s), phase, abort_flag, limit));
                    if (!alive) break;
                    ptx::tcgen05_fence_after_sync();
                    const uint32_t sa = tmem_scales + s * Cfg::kScaleCols, sb = sa + Cfg::kGroups * 4u;
                    const uint32_t a = a_lo + s * (Cfg::kBytesA >> 4), b = b_lo + s * (Cfg::kBytesB >> 4);
                    if (left >= kStageK) {
                        ptx::umma_fp4_ss_x4_if<kMx, 2>(on, tmem, a, a_hi, b, b_hi, idesc, sa, sb, 8, accumulate);
                    } else {
                        for (uint32_t i = 0; i * kMmaK < left; ++i) {
                            const uint32_t g = kMx ? i / 2 : i;
                            ptx::umma_fp4_ss_if<kMx, 2>(on, tmem, a + i * 2u, a_hi, b + i * 2u, b_hi, kMx && i % 2 ? idesc | ptx::kSecondScales : idesc, sa + g * 4u, sb + g * 8u,
                                                        i ? 1u : accumulate);
                        }
                    }
                    ptx::umma_commit_pair_if(on, empty_bar(s));
                    accumulate = 1;
                    left -= kStageK;
                    s = s + 1 == kStages ? 0u : s + 1;
                    phase ^= s == 0 ? 1u : 0u;
                }
                if (alive) ptx::umma_commit_pair_if(on, done_bar);
            }
            if (!alive && on) {
                ptx::umma_commit_pair_local(drain_bar);
                ptx::mbar_wait_bounded(drain_bar, 0, limit);
            }
        }
    } else if (warp >= Cfg::kEpilogueWarps) {
        // =========================================================== scales to tensor memory
        const uint32_t lanes = ((warp & 3u) * 32u) << 16, mine = (warp - Cfg::kEpilogueWarps) >> 2;
        const bool two_blocks = p.split.cols > 128u;
        uint32_t it = 0;
        bool alive = true;
        for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
            const Item w = split_item(p.split, item);
            for (uint32_t step = w.first; step < w.last; ++step, ++it) {
                if ((it & 1u) != mine) continue;
                const uint32_t s = it % kStages;
                // The stage's last step was the other four warps', so that this warp may be two phases of `full` behind, which a parity does not
                // tell apart: it waits for that step's MMAs first, as the load did.
                const uint32_t phase = it / kStages & 1u;
                uint32_t ok = 1;
                if (lane == 0) ok = (it < kStages || ptx::mbar_wait(empty_bar(s), phase ^ 1u, abort_flag, limit)) && ptx::mbar_wait(full_bar(s), phase, abort_flag, limit) ? 1u : 0u;
                alive = __shfl_sync(0xFFFFFFFFu, ok, 0) != 0u;
                if (!alive) break;
                // A stage's scales have columns of their own: they are overwritten when the stage is, after its MMAs.  (Groups that were
                // not loaded, at the end of k, have no MMAs; what they hold goes nowhere.)
                uint4 a[Cfg::kGroups], b[2 * Cfg::kGroups];
                const uint32_t src_a = sa_addr + s * Cfg::kScaleBytesA + lane * 16u, src_b = sb_addr + s * Cfg::kScaleBytesB + lane * 16u;
#pragma unroll
                for (uint32_t g = 0; g < Cfg::kGroups; ++g) {
                    a[g] = ptx::ld_shared_v4(src_a + g * 512u);
                    b[2 * g] = ptx::ld_shared_v4(src_b + g * 512u);
                    b[2 * g + 1] = two_blocks ? ptx::ld_shared_v4(src_b + Cfg::kScaleBytesA + g * 512u) : make_uint4(0u, 0u, 0u, 0u);
                }
                ptx::tcgen05_fence_after_sync();
                const uint32_t dst = tmem_scales + lanes + s * Cfg::kScaleCols;
                ptx::tmem_st_v4(dst, a);
                if constexpr (kMx) {
                    ptx::tmem_st_v4(dst + Cfg::kGroups * 4u, b);
                } else {
                    ptx::tmem_st_v4(dst + Cfg::kGroups * 4u, *reinterpret_cast<const uint4(*)[4]>(b));
                    ptx::tmem_st_v4(dst + Cfg::kGroups * 4u + 16u, *reinterpret_cast<const uint4(*)[4]>(b + 4));
                }
                ptx::tmem_st_wait();
                ptx::tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) ptx::mbar_arrive(ready_bar(s));
                    else ptx::mbar_arrive_cluster_relaxed(ptx::map_to_cta(ready_bar(s), 0));
                }
            }
        }
    } else {
        // =========================================================== C
        const uint32_t q = warp & 3u, half = warp >> 2, row = q * 32u + lane, lanes = (q * 32u) << 16;
        const Factor f(p.a_whole ? *reinterpret_cast<const volatile float *>(p.a_whole) : 1.f, p.b_whole ? *reinterpret_cast<const volatile float *>(p.b_whole) : 1.f);
        const uint32_t taken = rank == 0 ? taken_bar : ptx::map_to_cta(taken_bar, 0);
        uint32_t round = 0;
        for (uint32_t item = pair; item < p.split.items; item += n_pairs, ++round) {
            const Item w = split_item(p.split, item);
            uint32_t ok = 1;
            if (lane == 0) ok = ptx::mbar_wait(done_bar, round & 1u, abort_flag, limit) ? 1u : 0u;
            if (!__shfl_sync(0xFFFFFFFFu, ok, 0)) break;
            ptx::tcgen05_fence_after_sync();
            const uint32_t c_row = w.m0 + rank * 128u + row;
            auto free_accumulator = [&]() {
                ptx::tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) ptx::mbar_arrive(taken);
                    else ptx::mbar_arrive_cluster_relaxed(taken);
                }
            };
            if (w.slot == ~0u && p.c.type != B200SPMM_T_F32) {
                // the accumulator as 16-bit numbers to registers first: the next item's MMAs run while they are written
                uint32_t packed[4][16];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t c = half * 32u + j * 64u;
                    if (c >= p.split.cols) break;
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        uint32_t r[16];
                        ptx::tmem_ld_32x32b_x16(tmem + lanes + c + h * 16u, r);
                        ptx::tmem_ld_wait();
                        float v[16];
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) v[i] = f.apply(__uint_as_float(r[i]));
                        pack_row(p.c.type, v, packed[j] + h * 8u);
                    }
                }
                free_accumulator();
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t c = half * 32u + j * 64u;
                    if (c < p.split.cols && c_row < p.m && w.n0 + c < p.n) store_packed_column(p.c, c_row, w.n0 + c, p.n, packed[j]);
                }
                continue;
            }
#pragma unroll 1
            for (uint32_t c = half * 32u; c < p.split.cols; c += 64u) {
                uint32_t r[32];
                ptx::tmem_ld_32x32b_x32(tmem + lanes + c, r);
                ptx::tmem_ld_wait();
                if (w.slot != ~0u) {  // column by column: neighbouring lanes write neighbours
                    float *dst = p.partial + ((uint64_t)w.slot * p.split.cols + c) * kPairRows4 + rank * 128u + row;
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) dst[i * kPairRows4] = __uint_as_float(r[i]);
                } else if (c_row < p.m && w.n0 + c < p.n) {
                    float v[32];
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) v[i] = f.apply(__uint_as_float(r[i]));
                    store_row(p.c, c_row, w.n0 + c, p.n, v);
                }
            }
            free_accumulator();
        }
    }
    __syncwarp();
    // ---- teardown: every role ends up here, on success and on timeout alike
    if (*abort_flag) {  // loads may still be on their way into shared memory
        const uint64_t t0 = ptx::global_timer_ns();
        while (ptx::global_timer_ns() - t0 < kLingerNs) __nanosleep(1000);
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive();  // neither CTA lets go of what the other's MMAs, commits or arrives may still reach
    ptx::cluster_wait();
    if (warp == Cfg::kMmaWarp) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem, Cfg::kTmemCols);
    }
    if (tid == 0 && *abort_flag) atomicAdd(p.status, 1u);
}

}  // namespace fp4
}  // namespace b200spmm
