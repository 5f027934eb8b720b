// Product of a 4-bit matrix with many 16-bit columns: batches and prompts.
//
//     C[m, n] = s_A  sum over k  (a[m, k] sa[m, k / block]) B[k, n]
//
// Bound: the tensor core's 16-bit rate, and below a hundred columns or so one read of A.  Two CTAs on neighbouring SMs share MMAs
// of 256 rows x up to 256 columns (tcgen05.mma.cta_group::2): each brings half of B's columns, so that an SM fetches
// 40 bytes a clock from L2 at the full rate where a CTA alone would need 72, more than that path gives (about 51).
// A arrives packed, is widened by eight warps (exactly, see Widen) and goes through registers into tensor memory, from where the
// MMA takes it: shared memory, which B keeps busy, sees its 4 bits only once.
//
// A step is 128 values of k.  Warps 0-7 of a CTA widen: lane = row of the warp's quarter of tensor memory, warps w and w + 4
// take a half of the step each; after an item's last step they take the accumulator to C.  Warp 8 of the even CTA issues the
// MMAs, warp 9 loads.
//
//   full[s]   stage s has landed (TMA bytes, each CTA its own): the widening warps wait for it, with B's part of it
//   ready[b]  buffer b of widened A is written in both CTAs (16 warps arrive at the even CTA)
//   empty[s]  the MMAs of the step in stage s are done (commit, in both CTAs): the stage and its buffer of widened A are free
//   done      the accumulator of an item is complete (commit, in both CTAs).  The widening warps read it before they write the next item's
//             first buffer, so ready[] also says that the accumulator is free.
//
// Items are tiles of C.  Those of the last, incomplete round are cut along k into parts, so that every pair has something to
// do; their sums go to the workspace and a second kernel adds them up in order.
#pragma once

#include "fp4_widen.cuh"

namespace b200spmm {
namespace fp4 {

constexpr uint32_t kWideK = 128, kWideRows = 256, kWideCols = 256;

// How C is shared out over `pairs` pairs: tiles of 256 rows x `cols` columns, row blocks of them one after the other.
struct WideSplit {
    uint32_t cols;        // of a tile, a multiple of 32
    uint32_t tiles_n;     // tiles side by side
    uint32_t whole;       // tiles that one pair makes alone
    uint32_t parts;       // of the others
    uint32_t items;
    uint32_t steps;       // of k
};

inline WideSplit wide_split(uint32_t m, uint32_t n, uint32_t k, uint32_t pairs) {
    WideSplit s{};
    s.tiles_n = (n + kWideCols - 1) / kWideCols;
    s.cols = ((n + s.tiles_n - 1) / s.tiles_n + 31u) / 32u * 32u;
    s.steps = (k + kWideK - 1) / kWideK;
    const uint32_t tiles = (m + kWideRows - 1) / kWideRows * s.tiles_n, rest = tiles % pairs;
    // a part has at least four steps: shorter ones are not worth their sums' way through memory
    s.parts = rest ? std::min(pairs / rest, s.steps / 4) : 1;
    if (s.parts < 2) s.parts = 1;
    s.whole = s.parts > 1 ? tiles - rest : tiles;
    s.items = s.whole + (tiles - s.whole) * s.parts;
    return s;
}
inline uint64_t wide_workspace(const WideSplit &s) { return (uint64_t)(s.items - s.whole) * kWideRows * s.cols * sizeof(float); }

struct WideCfg {
    static constexpr uint32_t kBytesA = 128 * kWideK / 2, kBytesScales = 1024, kBoxBytes = 64 * 2 * 128, kBytesB = 2 * kBoxBytes;
    static constexpr uint32_t kStageBytes = kBytesA + kBytesScales + kBytesB, kStages = 5;
    static constexpr uint32_t kBuffers = 4, kBufferCols = kWideK / 2;  // of widened A, in tensor memory behind the accumulator
    static constexpr int kWarps = 10, kThreads = 32 * kWarps;
    static constexpr uint32_t kTmemCols = 512;
    static constexpr uint32_t kBarriers = 2 * kStages + kBuffers + 2;
    static constexpr size_t kSmemBytes = 1024 + (size_t)kStages * kStageBytes + kBarriers * 8 + 16;
    static_assert(kWideCols + kBuffers * kBufferCols <= kTmemCols && kSmemBytes <= 227 * 1024, "memory of an SM");
};

struct WideParams {
    DenseParams d;
    WideSplit split;
    uint32_t row_blocks;
    float *partial;
    uint32_t *status;
    unsigned long long wait_limit_ns;
};

struct WideItem {
    uint32_t m0, n0, first, last;  // steps [first, last)
    uint32_t slot;                 // of a part, else ~0
};
B200_DEVICE WideItem wide_item(const WideSplit &s, uint32_t i) {
    uint32_t tile = i, part = 0, parts = 1, slot = ~0u;
    if (i >= s.whole) {
        slot = i - s.whole;
        tile = s.whole + slot / s.parts;
        part = slot % s.parts;
        parts = s.parts;
    }
    if (parts == 1) slot = ~0u;
    return {tile / s.tiles_n * kWideRows, tile % s.tiles_n * s.cols, part * s.steps / parts, (part + 1) * s.steps / parts, slot};
}

template <typename T, bool kMx, bool kTokens>
__global__ void __launch_bounds__(WideCfg::kThreads, 1)
fp4_wide_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const WideParams p) {
    using Cfg = WideCfg;
    using W = Widen<T, kMx>;
    constexpr uint32_t kStages = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    // the same offsets in both CTAs: descriptors and multicast commits rely on it
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t *base = smem_raw + pad;
    const uint32_t b_addr = raw_addr + pad, a_addr = b_addr + kStages * Cfg::kBytesB, s_addr = a_addr + kStages * Cfg::kBytesA;
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + (size_t)kStages * Cfg::kStageBytes);
    const uint32_t bars_addr = ptx::smem_u32(bars);
    auto full_bar = [&](uint32_t s) { return bars_addr + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bars_addr + 8u * (kStages + s); };
    auto ready_bar = [&](uint32_t b) { return bars_addr + 8u * (2 * kStages + b); };
    const uint32_t done_bar = bars_addr + 8u * (2 * kStages + Cfg::kBuffers), drain_bar = done_bar + 8u;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(bars + Cfg::kBarriers);
    uint32_t *tmem_slot = const_cast<uint32_t *>(abort_flag) + 1;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint64_t limit = p.wait_limit_ns;
    const uint32_t rank = ptx::cluster_cta_rank(), pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t cols_half = p.split.cols / 2u;  // of B, this CTA's

    if (tid == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (uint32_t b = 0; b < Cfg::kBuffers; ++b) ptx::mbar_init(ready_bar(b), 16);
        ptx::mbar_init(done_bar, 1);
        ptx::mbar_init(drain_bar, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
    }
    if (warp == 8) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), Cfg::kTmemCols);
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    ptx::wait_for_grids_before();
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive();  // the other CTA's barriers exist before anything arrives on them
    ptx::cluster_wait();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 9) {
        // =========================================================== loads
        uint32_t it = 0;
        bool alive = lane == 0;
        for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
            const WideItem w = wide_item(p.split, item);
            const uint32_t row_block = w.m0 / 128u + rank;
            const uint32_t n0 = w.n0 + rank * cols_half;
            const uint32_t boxes = kTokens ? 2u : (cols_half + 63u) / 64u;
            const uint32_t box_bytes = kTokens ? cols_half * 128u : Cfg::kBoxBytes;
            for (uint32_t step = w.first; step < w.last; ++step, ++it) {
                const uint32_t s = it % kStages;
                alive = ptx::mbar_wait(empty_bar(s), (it / kStages & 1u) ^ 1u, abort_flag, limit);
                if (!alive) break;
                constexpr uint32_t kGroups = kMx ? 1 : 2;
                const uint32_t g0 = step * kGroups, scale_bytes = row_block < p.row_blocks ? min(kGroups, p.d.groups - g0) * 512u : 0u;
                ptx::mbar_arrive_expect_tx(full_bar(s), Cfg::kBytesA + scale_bytes + boxes * box_bytes);
                ptx::tma_load_2d(a_addr + s * Cfg::kBytesA, &tmap_a, (int32_t)(step * (kWideK / 2)), (int32_t)(w.m0 + rank * 128u), full_bar(s));
                if (scale_bytes) ptx::bulk_load(s_addr + s * Cfg::kBytesScales, p.d.scales + ((uint64_t)row_block * p.d.groups + g0) * 512u, scale_bytes, full_bar(s));
                for (uint32_t i = 0; i < boxes; ++i) {
                    if constexpr (kTokens) ptx::tma_load_2d(b_addr + s * Cfg::kBytesB + i * Cfg::kBoxBytes, &tmap_b, (int32_t)(step * kWideK + i * 64u), (int32_t)n0, full_bar(s));
                    else ptx::tma_load_2d(b_addr + s * Cfg::kBytesB + i * Cfg::kBoxBytes, &tmap_b, (int32_t)(n0 + i * 64u), (int32_t)(step * kWideK), full_bar(s));
                }
            }
        }
    } else if (warp == 8) {
        // =========================================================== MMAs (even CTA)
        if (rank == 0 && lane == 0) {
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? ptx::kFmtF16 : ptx::kFmtBF16;
            const uint32_t idesc = ptx::make_instr_desc(fmt, kWideRows, p.split.cols, false, !kTokens);
            // B [n][k]: 64 values of k a row of the swizzle, eight rows 1024 bytes.  [k][n]: 64 columns a row, eight k 1024 bytes, the next 64
            // columns a box away.
            const uint64_t b_desc0 = ptx::make_smem_desc(b_addr, kTokens ? 16u : Cfg::kBoxBytes, 1024, ptx::kSwizzle128B);
            uint32_t it = 0;
            bool alive = true;
            for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
                const WideItem w = wide_item(p.split, item);
                for (uint32_t step = w.first; step < w.last; ++step, ++it) {
                    const uint32_t s = it % kStages, b = it % Cfg::kBuffers;
                    alive = ptx::mbar_wait_cluster(ready_bar(b), it / Cfg::kBuffers & 1u, abort_flag, limit);
                    if (!alive) break;
                    ptx::tcgen05_fence_after_sync();
                    const uint32_t n_mma = min(kWideK / 16u, (p.d.k - step * kWideK + 15u) / 16u);
                    const uint32_t a = tmem + kWideCols + b * Cfg::kBufferCols;
                    for (uint32_t i = 0; i < n_mma; ++i) {
                        const uint32_t at = s * Cfg::kBytesB + (kTokens ? i / 4u * Cfg::kBoxBytes + i % 4u * 32u : i * 2048u);
                        ptx::umma_pair_f16_ts(tmem, a + i * 8u, b_desc0 + (at >> 4), idesc, step > w.first || i ? 1u : 0u);
                    }
                    ptx::umma_commit_pair(empty_bar(s));
                }
                if (alive) ptx::umma_commit_pair(done_bar);
            }
            if (!alive) {
                ptx::umma_commit_pair_local(drain_bar);
                ptx::mbar_wait_bounded(drain_bar, 0, limit);
            }
        }
    } else {
        // =========================================================== widening, and C
        const uint32_t q = warp & 3u, half = warp >> 2, row = q * 32u + lane;
        const uint32_t lanes = (q * 32u) << 16;
        const float whole = (kMx ? 1.f : *reinterpret_cast<const volatile float *>(p.d.whole));
        uint32_t it = 0, round = 0;
        bool alive = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            uint32_t ok = 1;
            if (lane == 0) ok = ptx::mbar_wait(bar, parity, abort_flag, limit) ? 1u : 0u;
            return __shfl_sync(0xFFFFFFFFu, ok, 0) != 0u;
        };
        for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs, ++round) {
            const WideItem w = wide_item(p.split, item);
            for (uint32_t step = w.first; step < w.last; ++step, ++it) {
                const uint32_t s = it % kStages, b = it % Cfg::kBuffers;
                alive = wait(full_bar(s), it / kStages & 1u);
                if (alive && it >= Cfg::kBuffers) {
                    const uint32_t old = it - Cfg::kBuffers;
                    alive = wait(empty_bar(old % kStages), old / kStages & 1u);
                }
                if (!alive) break;
                // 64 values: bytes 32 half .. + 31 of the row's 64, pieces of 16 bytes in the order of the 64-byte swizzle
                const uint32_t src = a_addr + s * Cfg::kBytesA + row * 64u, turn = row >> 1 & 3u;
                uint32_t codes[8];
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const uint4 v = ptx::ld_shared_v4(src + ((half * 2u + i) ^ turn) * 16u);
                    codes[4 * i] = v.x; codes[4 * i + 1] = v.y; codes[4 * i + 2] = v.z; codes[4 * i + 3] = v.w;
                }
                const uint32_t group = kMx ? 0u : half;
                uint32_t four = 0;  // scales of what lies past the last column: zeros (there is no group that was not loaded)
                if (step * kWideK + half * 64u < p.d.k)
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(four) : "r"(s_addr + s * Cfg::kBytesScales + group * 512u + lane * 16u + q * 4u) : "memory");
                uint32_t out[32];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {  // eight values each
                    const uint32_t sc = kMx ? W::scale(four >> (half * 16u + i / 4u * 8u) & 0xFFu) : W::scale(four >> (i / 2u * 8u) & 0xFFu);
                    const uint32_t p0 = W::template pair<12>(codes[i], sc), p1 = W::template pair<8>(codes[i], sc);
                    const uint32_t p2 = W::template pair<4>(codes[i], sc), p3 = W::template pair<0>(codes[i], sc);
                    out[4 * i] = __byte_perm(p0, p1, 0x5410);  // (0, 4) and (1, 5) to (0, 1) and (4, 5)
                    out[4 * i + 1] = __byte_perm(p2, p3, 0x5410);
                    out[4 * i + 2] = __byte_perm(p0, p1, 0x7632);
                    out[4 * i + 3] = __byte_perm(p2, p3, 0x7632);
                }
                ptx::tcgen05_fence_after_sync();
                ptx::tmem_st_32x32b_x32(tmem + lanes + kWideCols + b * Cfg::kBufferCols + half * 32u, out);
                ptx::tmem_st_wait();
                ptx::tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) ptx::mbar_arrive(ready_bar(b));
                    else ptx::mbar_arrive_cluster_relaxed(ptx::map_to_cta(ready_bar(b), 0));
                }
            }
            if (!alive) break;
            alive = wait(done_bar, round & 1u);
            if (!alive) break;
            ptx::tcgen05_fence_after_sync();
            const uint32_t c_row = w.m0 + rank * 128u + row;
#pragma unroll 1
            for (uint32_t c = half * 32u; c < p.split.cols; c += 64u) {
                uint32_t r[32];
                ptx::tmem_ld_32x32b_x32(tmem + lanes + c, r);
                ptx::tmem_ld_wait();
                if (w.slot != ~0u) {  // column by column: neighbouring lanes write neighbours
                    float *dst = p.partial + ((uint64_t)w.slot * p.split.cols + c) * kWideRows + rank * 128u + row;
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) dst[i * kWideRows] = __uint_as_float(r[i]);
                } else if (c_row < p.d.m && w.n0 + c < p.d.n) {
                    float v[32];
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * W::kLeft * whole;
                    store_row(p.d.c, c_row, w.n0 + c, p.d.n, v);
                }
            }
            ptx::tcgen05_fence_before_sync();
        }
    }
    __syncwarp();
    // ---- teardown: every role ends up here, on success and on timeout alike
    if (*abort_flag) {  // loads may still be on their way into shared memory
        const uint64_t t0 = ptx::global_timer_ns();
        while (ptx::global_timer_ns() - t0 < 20000000ull) __nanosleep(1000);
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_arrive();  // neither CTA lets go of what the other's MMAs, commits or arrives may still reach
    ptx::cluster_wait();
    if (warp == 8) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem, Cfg::kTmemCols);
    }
    if (tid == 0 && *abort_flag) atomicOr(p.status, kDevStatusTimeout);
}

// C of the tiles that were cut: the parts' sums in order.  A thread a row and 32 columns.
__global__ void __launch_bounds__(kWideRows) fp4_join_kernel(const WideSplit s, const float *__restrict__ partial, uint32_t m, uint32_t n, float left,
                                                             const float *__restrict__ whole, const Target c) {
    ptx::wait_for_grids_before();
    const float f = left * (whole ? *reinterpret_cast<const volatile float *>(whole) : 1.f);
    const uint32_t tile = s.whole + blockIdx.x, col = blockIdx.y * 32u;
    const uint32_t row = tile / s.tiles_n * kWideRows + threadIdx.x, n0 = tile % s.tiles_n * s.cols + col;
    if (row >= m || n0 >= n) return;
    float v[32] = {};
    for (uint32_t part = 0; part < s.parts; ++part) {
        const float *src = partial + ((uint64_t)(blockIdx.x * s.parts + part) * s.cols + col) * kWideRows + threadIdx.x;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) v[i] += src[i * kWideRows];
    }
#pragma unroll
    for (uint32_t i = 0; i < 32; ++i) v[i] *= f;
    store_row(c, row, n0, n, v);
}

}  // namespace fp4
}  // namespace b200spmm
