// Product of a 4-bit matrix with many 16-bit columns: batches and prompts.
//
//     C[m, n] = s_A  sum over k  (a[m, k] sa[m, k / block]) B[k, n]
//
// Bound: the tensor core's 16-bit rate, and below a hundred columns or so one read of A.  Two CTAs on neighbouring SMs share MMAs
// of 256 rows x up to 256 columns (tcgen05.mma.cta_group::2): each brings half of B's columns, so that an SM fetches
// 40 bytes a clock from L2 at the full rate where a CTA alone would need 72, more than that path gives (about 51).
// 28672 x 8192 nvfp4 x fp16: 2,048 columns 616 us (1,560 TFLOP/s), 192 77 (112 tiles for 74 pairs, two rounds where 1.5 would do), 64 48.
// A arrives packed, is widened by sixteen warps (exactly, see Widen) and goes through registers into tensor memory, from where the
// MMA takes it: shared memory, which B keeps busy, sees its 4 bits only once.
//
// A step is 128 values of k.  Warps 0-15 of a CTA widen: lane = row of the warp's quarter of tensor memory, warps 4 g .. 4 g + 3
// every fourth step, so that what a step has to wait for (its stage, its way to tensor memory) overlaps with three others;
// after an item's last step they take the accumulator to C.  Warp 16 of the even CTA issues the MMAs, warps 17 and 18 load.  Up to 128
// columns, where issuing a step's MMAs takes longer than they do, warp 19 issues those of every second step, to an accumulator of its own.
//
// A and B have stages of their own: those of A, which comes from memory, are free again as soon as they have been read.
//
//   full a, full b   a stage has landed (TMA bytes, each CTA its own): the widening warps wait for both
//   empty a   the four warps that widen it have read it
//   ready[g]  group g's buffer of widened A is written in both CTAs, and B's stage is there (eight warps arrive at the even CTA)
//   empty b   the MMAs of the step are done (commit, in both CTAs): the stage of B and the buffer of widened A are free
//   done      the accumulators of an item are complete (commits, in both CTAs)
//   taken     all 32 warps have read it (they arrive at the even CTA)
//
// The tensor core cuts what it adds to an accumulator off to fp32, which over 512 MMAs (8,192 values of k) leaves sums off by 4e-6 of their
// size.  That is nothing beside the rounding of a 16-bit C; for an fp32 one (kExact) the accumulator, of up to 128 columns, is emptied
// every four steps into rounded fp32 sums in shared memory, 3e-7, while a second one fills: 192 columns 124 us, 2,048 1,020.
#pragma once

#include "fp4_split.cuh"
#include "fp4_widen.cuh"

namespace b200spmm {
namespace fp4 {

constexpr uint32_t kWideK = 128;  // of a step

struct WideCfg {
    static constexpr uint32_t kBytesA = 128 * kWideK / 2, kBytesScales = 1024;
    static constexpr uint32_t kStageA = kBytesA + kBytesScales, kMinA = 6, kMaxA = 12, kMaxB = 8;  // stages
    static constexpr uint32_t kBuffers = 4, kBufferCols = kWideK / 2;  // of widened A, in tensor memory behind the accumulator
    static constexpr uint32_t kWideners = 16;
    static_assert(kBuffers == kWideners / 4 && kBuffers < kMinA, "a group of four warps has a buffer of its own");
    static constexpr int kSecondMma = kWideners + 3, kWarps = kWideners + 4, kThreads = 32 * kWarps;
    static constexpr uint32_t kTwoCols = 128;  // up to which two warps issue MMAs
    static constexpr uint32_t kTmemCols = 512;
    static constexpr uint32_t kBarriers = 2 * kMaxA + 2 * kMaxB + kBuffers + 6;
    static constexpr uint32_t kExactCols = 128, kExactBytes = kExactCols * 128 * 4, kRun = 4;  // kExact: columns, their sums, steps of an accumulator
    static constexpr uint32_t kOtherBytes = 1024 + kBarriers * 8 + 16;
    static constexpr size_t kSmemBytes = 227 * 1024;  // at most
    static_assert(kPairCols4 + kBuffers * kBufferCols <= kTmemCols, "tensor memory of an SM");
    // A box of B, 128 bytes wide, and the boxes of a stage: [n][k] two of 64 values of k for each of a CTA's columns, [k][n] 64 columns each.
    __host__ __device__ static constexpr uint32_t box_bytes(bool tokens, uint32_t cols) { return tokens ? cols / 2u * 128u : kWideK * 128u; }
    __host__ __device__ static constexpr uint32_t boxes(bool tokens, uint32_t cols) { return tokens ? 2u : (cols / 2u + 63u) / 64u; }
    __host__ __device__ static constexpr uint32_t b_bytes(bool tokens, uint32_t cols) { return box_bytes(tokens, cols) * boxes(tokens, cols); }
    // Few columns leave room for more stages.
    static constexpr uint32_t room(bool exact) { return (uint32_t)kSmemBytes - kOtherBytes - (exact ? kExactBytes : 0u); }
    static uint32_t stages_b(bool tokens, bool exact, uint32_t cols) { return std::min<uint32_t>(kMaxB, (room(exact) - kMinA * kStageA) / b_bytes(tokens, cols)); }
    static uint32_t stages_a(bool tokens, bool exact, uint32_t cols) {
        return std::min<uint32_t>(kMaxA, (room(exact) - stages_b(tokens, exact, cols) * b_bytes(tokens, cols)) / kStageA);
    }
    static size_t smem_bytes(bool tokens, bool exact, uint32_t cols) {
        return kOtherBytes + (exact ? kExactBytes : 0u) + (size_t)stages_a(tokens, exact, cols) * kStageA + (size_t)stages_b(tokens, exact, cols) * b_bytes(tokens, cols);
    }
};
static_assert((WideCfg::room(true) - WideCfg::kMinA * WideCfg::kStageA) / WideCfg::b_bytes(false, WideCfg::kExactCols) >= 5, "shared memory");
static_assert((WideCfg::room(false) - WideCfg::kMinA * WideCfg::kStageA) / WideCfg::b_bytes(false, 256) >= 5, "shared memory");
static_assert((WideCfg::room(false) - WideCfg::kMinA * WideCfg::kStageA) / WideCfg::b_bytes(false, WideCfg::kTwoCols) >= WideCfg::kMaxB && WideCfg::kMaxB % 2 == 0,
              "where two warps issue MMAs, a stage of B always belongs to the same one");

struct WideParams {
    DenseParams d;
    Split split;
    uint32_t row_blocks;
    uint32_t stages_a, stages_b;
    float *partial;
    uint32_t *status;
    unsigned long long wait_limit_ns;
};

template <typename T, bool kMx, bool kTokens, bool kExact>
__global__ void __launch_bounds__(WideCfg::kThreads, 1)
fp4_wide_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const WideParams p) {
    using Cfg = WideCfg;
    using W = Widen<T, kMx>;
    const uint32_t stages_a = p.stages_a, stages_b = p.stages_b, box_bytes = Cfg::box_bytes(kTokens, p.split.cols), boxes = Cfg::boxes(kTokens, p.split.cols), bytes_b = box_bytes * boxes;
    extern __shared__ uint8_t smem_raw[];
    // the same offsets in both CTAs: descriptors and multicast commits rely on it
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t *base = smem_raw + pad;
    const uint32_t b_addr = raw_addr + pad, a_addr = b_addr + stages_b * bytes_b, s_addr = a_addr + stages_a * Cfg::kBytesA;
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + (size_t)stages_b * bytes_b + (size_t)stages_a * Cfg::kStageA);
    const uint32_t bars_addr = ptx::smem_u32(bars);
    auto full_b = [&](uint32_t s) { return bars_addr + 8u * s; };
    auto empty_b = [&](uint32_t s) { return bars_addr + 8u * (Cfg::kMaxB + s); };
    auto full_a = [&](uint32_t s) { return bars_addr + 8u * (2 * Cfg::kMaxB + s); };
    auto empty_a = [&](uint32_t s) { return bars_addr + 8u * (2 * Cfg::kMaxB + Cfg::kMaxA + s); };
    auto ready_bar = [&](uint32_t b) { return bars_addr + 8u * (2 * Cfg::kMaxB + 2 * Cfg::kMaxA + b); };
    const uint32_t done_bar = bars_addr + 8u * (2 * Cfg::kMaxB + 2 * Cfg::kMaxA + Cfg::kBuffers), taken_bar = done_bar + 16u, drain_bar = done_bar + 32u;  // done and taken: two, of which kExact uses the second, too
    float *exact_sums = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(bars) + Cfg::kBarriers * 8 + 16);  // kExact: [column][row]
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(bars + Cfg::kBarriers);
    uint32_t *tmem_slot = const_cast<uint32_t *>(abort_flag) + 1;

    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31u;  // (the shuffle: a warp is known to be one)
    const uint64_t limit = p.wait_limit_ns;
    const uint32_t rank = ptx::cluster_cta_rank(), pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t cols_half = p.split.cols / 2u;  // of B, this CTA's
    const bool two_mma = !kExact && p.split.cols <= Cfg::kTwoCols;

    if (tid == 0) {
        for (uint32_t s = 0; s < stages_a; ++s) {
            ptx::mbar_init(full_a(s), 1);
            ptx::mbar_init(empty_a(s), 4);
        }
        for (uint32_t s = 0; s < stages_b; ++s) {
            ptx::mbar_init(full_b(s), 1);
            ptx::mbar_init(empty_b(s), 1);
        }
        for (uint32_t b = 0; b < Cfg::kBuffers; ++b) ptx::mbar_init(ready_bar(b), 8);
        for (uint32_t d = 0; d < 2; ++d) {
            ptx::mbar_init(done_bar + 8u * d, two_mma ? 2u : 1u);
            ptx::mbar_init(taken_bar + 8u * d, 2 * Cfg::kWideners);
        }
        for (uint32_t d = 0; d < 2; ++d) ptx::mbar_init(drain_bar + 8u * d, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
    }
    if (warp == Cfg::kWideners) {
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

    if (warp == Cfg::kWideners + 1 || warp == Cfg::kWideners + 2) {
        // =========================================================== loads
        // One warp A and its scales, one B: an instruction holds its warp for some 130 clocks.
        const uint32_t on = lane == 0 ? 1u : 0u;
        const bool is_a = warp == Cfg::kWideners + 1;
        constexpr uint32_t kGroups = kMx ? 1 : 2;
        const uint32_t stages = is_a ? stages_a : stages_b;
        uint32_t s = 0, phase = 1;
        bool alive = true;
        for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
            const Item w = split_item(p.split, item);
            const uint32_t row_block = w.m0 / 128u + rank;
            const uint32_t n0 = w.n0 + rank * cols_half;
            const bool has_scales = row_block < p.row_blocks;
            const uint8_t *scales = p.d.scales + (uint64_t)row_block * p.d.groups * 512u;
            for (uint32_t step = w.first; step < w.last; ++step) {
                alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait(is_a ? empty_a(s) : empty_b(s), phase, abort_flag, limit));
                if (!alive) break;
                if (is_a) {
                    const uint32_t g0 = step * kGroups, scale_bytes = has_scales ? min(kGroups, p.d.groups - g0) * 512u : 0u;
                    ptx::mbar_arrive_expect_tx_if(on, full_a(s), Cfg::kBytesA + scale_bytes);
                    ptx::tma_load_2d_if(on, a_addr + s * Cfg::kBytesA, &tmap_a, (int32_t)(step * (kWideK / 2)), (int32_t)(w.m0 + rank * 128u), full_a(s));
                    ptx::bulk_load_if(on & (has_scales ? 1u : 0u), s_addr + s * Cfg::kBytesScales, scales + (uint64_t)g0 * 512u, scale_bytes, full_a(s));
                } else {
                    ptx::mbar_arrive_expect_tx_if(on, full_b(s), boxes * box_bytes);
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const uint32_t there = on & (i < boxes ? 1u : 0u);
                        if constexpr (kTokens) ptx::tma_load_2d_if(there, b_addr + s * bytes_b + i * box_bytes, &tmap_b, (int32_t)(step * kWideK + i * 64u), (int32_t)n0, full_b(s));
                        else ptx::tma_load_2d_if(there, b_addr + s * bytes_b + i * box_bytes, &tmap_b, (int32_t)(n0 + i * 64u), (int32_t)(step * kWideK), full_b(s));
                    }
                }
                s = s + 1 == stages ? 0u : s + 1;
                phase ^= s == 0 ? 1u : 0u;
            }
        }
    } else if (warp >= Cfg::kWideners) {
        // =========================================================== MMAs (even CTA): every step, or every second one each
        const uint32_t which_warp = warp == Cfg::kWideners ? 0u : 1u;
        if (rank == 0 && (which_warp == 0 || two_mma)) {
            const uint32_t on = lane == 0 ? 1u : 0u;
            constexpr uint32_t fmt = std::is_same<T, __half>::value ? ptx::kFmtF16 : ptx::kFmtBF16;
            const uint32_t idesc = ptx::make_instr_desc(fmt, kPairRows4, p.split.cols, false, !kTokens);
            // B [n][k]: 64 values of k a row of the swizzle, eight rows 1024 bytes.  [k][n]: 64 columns a row, eight k 1024 bytes, the next 64
            // columns a box away.
            const uint64_t b_desc = ptx::make_smem_desc(b_addr, kTokens ? 16u : box_bytes, 1024, ptx::kSwizzle128B);
            const uint32_t b_lo = (uint32_t)b_desc, b_hi = (uint32_t)(b_desc >> 32), by = two_mma ? 2u : 1u;
            uint32_t s = which_warp, buffer = which_warp, phase = 0, round = 0;  // rounds: items, or with kExact runs of four steps
            uint32_t before = 0;                                                 // steps of the items before
            bool alive = true;
            for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
                const Item w = split_item(p.split, item);
                uint32_t step = w.first + (two_mma ? (which_warp ^ before) & 1u : 0u);
                before += w.last - w.first;
                do {
                    const uint32_t end = kExact ? min(step + Cfg::kRun, w.last) : w.last, which = kExact ? round & 1u : which_warp, d = tmem + which * Cfg::kExactCols;
                    const uint32_t bar = kExact ? 8u * which : 0u;
                    if (kExact ? round >= 2 : round >= 1)
                        alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait_cluster(taken_bar + bar, (kExact ? (round >> 1) - 1u : round - 1u) & 1u, abort_flag, limit));
                    uint32_t accumulate = 0;
                    for (; alive && step < end; step += by) {
                        alive = __all_sync(0xFFFFFFFFu, ptx::mbar_wait_cluster(ready_bar(buffer), phase, abort_flag, limit));
                        if (!alive) break;
                        ptx::tcgen05_fence_after_sync();
                        const uint32_t a = tmem + kPairCols4 + buffer * Cfg::kBufferCols, b = b_lo + s * (bytes_b >> 4);
                        const uint32_t left = p.d.k - step * kWideK;  // values of k from this step on
                        if (left >= kWideK) {
                            constexpr uint32_t kNext = kTokens ? 2u : 128u;
                            ptx::umma_pair_f16_ts_x4_if<kNext>(on, d, a, b, b_hi, idesc, accumulate);
                            ptx::umma_pair_f16_ts_x4_if<kNext>(on, d, a + 32u, b + (kTokens ? box_bytes >> 4 : 512u), b_hi, idesc, 1u);
                        } else {
                            for (uint32_t i = 0; i * 16u < left; ++i)
                                ptx::umma_pair_f16_ts_if(on, d, a + i * 8u, b + ((kTokens ? i / 4u * box_bytes + i % 4u * 32u : i * 2048u) >> 4), b_hi, idesc, i ? 1u : accumulate);
                        }
                        ptx::umma_commit_pair_if(on, empty_b(s));
                        accumulate = 1;
                        s += by;
                        if (s >= stages_b) s -= stages_b;
                        buffer += by;
                        if (buffer >= Cfg::kBuffers) {
                            buffer -= Cfg::kBuffers;
                            phase ^= 1u;
                        }
                    }
                    if (alive) ptx::umma_commit_pair_if(on, done_bar + bar);
                    ++round;
                } while (alive && step < w.last);
            }
            if (!alive && on) {
                ptx::umma_commit_pair_local(drain_bar + 8u * which_warp);
                ptx::mbar_wait_bounded(drain_bar + 8u * which_warp, 0, limit);
            }
        }
    } else {
        // =========================================================== widening, and C
        const uint32_t q = warp & 3u, mine = warp >> 2, row = q * 32u + lane;
        const uint32_t lanes = (q * 32u) << 16;
        const LeftOver rest(W::kLeft, kMx ? 1.f : *reinterpret_cast<const volatile float *>(p.d.whole));
        const uint32_t ready = rank == 0 ? ready_bar(mine) : ptx::map_to_cta(ready_bar(mine), 0);
        const uint32_t taken = rank == 0 ? taken_bar : ptx::map_to_cta(taken_bar, 0);
        const uint32_t buffer = tmem + lanes + kPairCols4 + mine * Cfg::kBufferCols;
        // its next step's stages and phases, and whether there was one before
        uint32_t s = mine, phase = 0, sb = mine, phase_b = 0, round = 0;
        bool alive = true, again = false;
        auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, ptx::mbar_wait(bar, parity, abort_flag, limit)) != 0; };
        auto widen_step = [&](uint32_t step) {
            // The stage's last step was other warps', so that this one might be two phases of `full a` behind, which a parity does not tell
            // apart: that step's warps have read it first, as for the load.
            alive = wait(empty_a(s), phase ^ 1u) && wait(full_a(s), phase);
            if (!alive) return;
            // the row's 64 bytes, pieces of 16 in the order of the 64-byte swizzle, and its words of scales
            const uint32_t src = a_addr + s * Cfg::kBytesA + row * 64u, turn = row >> 1 & 3u;
            uint32_t four[2] = {0u, 0u};  // scales of what lies past the last column: zeros (there is no group that was not loaded)
#pragma unroll
            for (uint32_t g = 0; g < (kMx ? 1u : 2u); ++g)
                if (step * kWideK + g * 64u < p.d.k)
                    four[g] = ptx::ld_shared_u32(s_addr + s * Cfg::kBytesScales + g * 512u + lane * 16u + q * 4u);
            const bool two = W::needs_two(four[0]) || W::needs_two(four[1]);
            const bool any_two = kMx && __any_sync(0xFFFFFFFFu, two);
            uint32_t out[32];
            auto widen = [&](auto twice, uint32_t h) {
                const uint4 lo = ptx::ld_shared_v4(src + ((2u * h) ^ turn) * 16u), hi = ptx::ld_shared_v4(src + ((2u * h + 1u) ^ turn) * 16u);
                if (h == 1) {
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(empty_a(s));
                }
                const uint32_t codes[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {  // eight values each
                    const uint32_t c = codes[i];
                    const uint32_t sc = W::template scale<decltype(twice)::value>(kMx ? four[0] >> (h * 16u + i / 4u * 8u) & 0xFFu : four[h] >> (i / 2u * 8u) & 0xFFu);
                    W::template eight<decltype(twice)::value>(c, sc, out + 4 * i);
                }
            };
            // half of it before the buffer is free
            if (any_two) widen(std::true_type(), 0);
            else widen(std::false_type(), 0);
            if (again) {  // the MMAs of the step four before leave the buffer
                const bool wrapped = sb < Cfg::kBuffers;  // (B's stage of that step)
                alive = wait(empty_b(wrapped ? sb + stages_b - Cfg::kBuffers : sb - Cfg::kBuffers), wrapped ? phase_b ^ 1u : phase_b);
                if (!alive) return;
            }
            ptx::tcgen05_fence_after_sync();
            ptx::tmem_st_32x32b_x32(buffer, out);
            if (any_two) widen(std::true_type(), 1);
            else widen(std::false_type(), 1);
            ptx::tmem_st_32x32b_x32(buffer + 32u, out);
            // (B's stage was last that of a step that is done by now, at least as old as the one waited for)
            alive = wait(full_b(sb), phase_b);
            ptx::tmem_st_wait();  // (tensor memory is let go of after a wait that ran out, too)
            if (!alive) return;
            ptx::tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) ptx::mbar_arrive(ready);
                else ptx::mbar_arrive_cluster_relaxed(ready);
            }
            again = true;
            s += Cfg::kBuffers;
            if (s >= stages_a) {
                s -= stages_a;
                phase ^= 1u;
            }
            sb += Cfg::kBuffers;
            if (sb >= stages_b) {
                sb -= stages_b;
                phase_b ^= 1u;
            }
        };
        // The sum's 16 columns from c on, of the first accumulator, the second or both.
        auto columns = [&](uint32_t c, bool first, bool second, float (&v)[16]) {
            uint32_t r[16];
            ptx::tmem_ld_32x32b_x16(tmem + lanes + (first ? 0u : Cfg::kExactCols) + c, r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
            if (!(first && second)) return;
            ptx::tmem_ld_32x32b_x16(tmem + lanes + Cfg::kExactCols + c, r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) v[i] += __uint_as_float(r[i]);
        };
        auto free_accumulator = [&](uint32_t which) {
            ptx::tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) ptx::mbar_arrive(taken + 8u * which);
                else ptx::mbar_arrive_cluster_relaxed(taken + 8u * which);
            }
        };
        auto store_part = [&](const Item &w, uint32_t c, const float (&v)[16]) {  // column by column: neighbouring lanes write neighbours
            float *dst = p.partial + ((uint64_t)w.slot * p.split.cols + c) * kPairRows4 + rank * 128u + row;
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) dst[i * kPairRows4] = v[i];
        };
        uint32_t before = 0;  // steps of the items before
        for (uint32_t item = pair; alive && item < p.split.items; item += n_pairs) {
            const Item w = split_item(p.split, item);
            const uint32_t c_row0 = w.m0 + rank * 128u + q * 32u, steps = w.last - w.first;
            if constexpr (kExact) {
                // a step of each run is this warp's; a run's sums are taken when its step of the next one is under way
                const uint32_t runs = (steps + Cfg::kRun - 1) / Cfg::kRun;
                for (uint32_t run = 0; run <= runs; ++run) {
                    const uint32_t step = run * Cfg::kRun + ((mine - before) & (Cfg::kRun - 1u));
                    if (run < runs && step < steps) widen_step(w.first + step);
                    if (!alive) break;
                    if (run == 0) continue;
                    alive = wait(done_bar + 8u * (round & 1u), round >> 1 & 1u);
                    if (!alive) break;
                    ptx::tcgen05_fence_after_sync();
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t c = mine * 32u + j * 8u;
                        if (c >= p.split.cols) break;
                        uint32_t r[8];
                        ptx::tmem_ld_32x32b_x8(tmem + lanes + (round & 1u) * Cfg::kExactCols + c, r);
                        ptx::tmem_ld_wait();
                        float *sum = exact_sums + c * 128u + row;
#pragma unroll
                        for (uint32_t i = 0; i < 8; ++i) sum[i * 128u] = run > 1 ? sum[i * 128u] + __uint_as_float(r[i]) : __uint_as_float(r[i]);
                    }
                    free_accumulator(round & 1u);
                    ++round;
                }
                if (!alive) break;
#pragma unroll 1
                for (uint32_t c = mine * 32u; c < min(mine * 32u + 32u, p.split.cols); c += 16u) {
                    float v[16];
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i) v[i] = exact_sums[(c + i) * 128u + row];
                    if (w.slot != ~0u) {
                        store_part(w, c, v);
                    } else if (w.n0 + c < p.d.n) {
                        uint32_t words[16];
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) words[i] = __float_as_uint(rest.apply(v[i]));
                        store_words(p.d.c, c_row0, p.d.m, w.n0 + c, p.d.n, words);
                    }
                }
            } else {
                for (uint32_t step = (mine - before) & (Cfg::kBuffers - 1u); alive && step < steps; step += Cfg::kBuffers) widen_step(w.first + step);
                if (!alive) break;
                const bool first = !two_mma || steps > 1u || (before & 1u) == 0u, second = two_mma && (steps > 1u || (before & 1u) != 0u);
                alive = wait(done_bar, round & 1u);
                if (!alive) break;
                ptx::tcgen05_fence_after_sync();
                if (w.slot == ~0u) {
                    // the accumulator as 16-bit numbers to registers first: the next item's MMAs run while they are written
                    uint32_t packed[2][16];
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t c = mine * 32u + j / 2u * 128u;
                        if (c >= p.split.cols) break;
                        float v[16];
                        columns(c + j % 2u * 16u, first, second, v);
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) v[i] = rest.apply(v[i]);
                        pack_row(p.d.c.type, v, packed[j / 2u] + j % 2u * 8u);
                    }
                    free_accumulator(0);
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j) {
                        const uint32_t c = mine * 32u + j * 128u;
                        if (c < p.split.cols && w.n0 + c < p.d.n) store_words(p.d.c, c_row0, p.d.m, w.n0 + c, p.d.n, packed[j]);
                    }
                } else {
#pragma unroll 1
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t c = mine * 32u + j / 2u * 128u + j % 2u * 16u;
                        if (c >= p.split.cols) break;
                        float v[16];
                        columns(c, first, second, v);
                        store_part(w, c, v);
                    }
                    free_accumulator(0);
                }
                ++round;
            }
            before += steps;
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
    if (warp == Cfg::kWideners) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem, Cfg::kTmemCols);
    }
    if (tid == 0 && *abort_flag) atomicAdd(p.status, 1u);
}

}  // namespace fp4
}  // namespace b200spmm
