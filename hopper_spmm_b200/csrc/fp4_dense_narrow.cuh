// Product of a 4-bit matrix with a few columns of 16-bit values: decoding.
//
//     C[m, 0..n) = s_A  sum over k  (a[m, k] sa[m, k / block]) B[k, 0..n)
//
// Bound: one read of A; what it waits for is latency.  The widening of its codes, a dozen operations for eight values whatever n is, fills half of the
// issue slots (52 % with 8 columns of fp16) while memory gives 61 % of its rate: a warp has one step between two waits for a stage that all of them
// share.  Codes become 16-bit numbers in registers and meet eight columns of B at a time there (mma.sync, 16 rows x 8 columns x 16 values of k;
// at this width a product is a small part of the work, and for tcgen05 the numbers would have to go through shared or tensor memory).
//
// Tiles of 16 rows are shared out evenly over the SMs, one block of threads each, which goes through k with up to 14 of them at a time: one warp
// brings stages of 256 values of k of all their rows, two take turns with the same of B, put in the order of the MMAs' operands (one
// alone kept the others waiting, 5 us for 8,192 values of k), and up to 28 multiply, a tile or, k being sliced, a part of one each.  The slices' sums meet in shared memory, in order, at the end.  (Row blocks of
// 128 whose eight warps sliced k and fetched for themselves came to 38 us for 28672 x 8192 times one column: 224 blocks on 148 SMs, and 18
// operations for eight values.)  28672 x 8192 nvfp4, whose 132 MB take 20 us to read: one column in fp16 33 us, 8 34, 16 47; in bf16, which takes
// twice the operations to widen, 50, 48 and 57.
//
// Lane 4 g + t takes 16 bytes of values, 32 codes, of rows r(g) and r(g) + 8 of its tile from k = 32 t of a step of 128 on; r puts rows that are
// four apart side by side, whose pieces of a step lie in different halves of the swizzled 128 bytes.  Which k an operand
// position of the MMA stands for is free as long as both operands agree: lane t's positions of MMA j are pairs 2 (j % 2) and
// 2 (j % 2) + 1 of word j / 2 of its four, as Widen makes them.
#pragma once

#include <algorithm>
#include <cuda.h>
#include <type_traits>

#include "fp4_widen.cuh"
#include "warp_mma.cuh"

namespace b200spmm {
namespace fp4 {

constexpr uint32_t kNarrowStep = 128, kNarrowStage = 256;  // values of k
constexpr uint32_t kNarrowTiles = 14;                      // of 16 rows at a time, at most: two warps for each, and those that load, are a block's 32
constexpr uint32_t kNarrowWarps = 2 * kNarrowTiles, kNarrowLoaders = 3;  // that multiply, at most, and load
static_assert(kNarrowWarps + kNarrowLoaders <= 32 && 2 * (kNarrowTiles + 1) + kNarrowLoaders > 32 && 16 * kNarrowTiles <= 256, "a block's warps, a box's rows");
constexpr uint32_t kNarrowMaxStages = 8;
constexpr uint32_t kNarrowRun = 4;                         // steps of a warp between two roundings of its sums, for an fp32 C

struct NarrowParams {
    DenseParams d;
    uint32_t tiles;       // of the matrix
    uint32_t at_once;     // ... of a block, side by side
    uint32_t slices;      // of k: warps of a tile
    uint32_t stages;
    uint32_t row_blocks;  // whose scales a stage has room for
    uint32_t* status;
    unsigned long long wait_limit_ns;
};

// How a block's tiles are gone through: as many at a time in every round (x 8192 times one fp16 column: 32,000 rows as 13 tiles and 1 of 14 took 59 us, as
// 14 35; 66,304 as 13, 13 and 2 86, as 14 and 14 62), each sliced as far as there are steps and warps: two for a tile, or 26 in all.  (28 in all: 2048
// rows 11.8 us for 11.3, 14336 times 16 columns 32.3 for 30.8; 4096 times 16 24.4 for 25.1.)
struct NarrowShare {
    uint32_t blocks, rounds, at_once, slices;
};
inline NarrowShare narrow_share(uint32_t tiles, uint32_t k, uint32_t sms) {
    NarrowShare s{};
    s.blocks = std::min(tiles, sms);
    const uint32_t of_block = (tiles + s.blocks - 1) / s.blocks;
    s.rounds = (of_block + kNarrowTiles - 1) / kNarrowTiles;
    s.at_once = (of_block + s.rounds - 1) / s.rounds;
    s.slices = std::max<uint32_t>(1, std::min(std::max(2u, 26u / s.at_once), (k + kNarrowStep - 1) / kNarrowStep));
    return s;
}

// Bytes of a stage: values, scales, B.
struct NarrowStage {
    uint32_t values, scales, b;
    __host__ __device__ uint32_t bytes() const { return (values + scales + b + 1023u) / 1024u * 1024u; }  // (the swizzle's period)
};
__host__ __device__ inline NarrowStage narrow_stage(bool mx, uint32_t at_once, uint32_t row_blocks, uint32_t nb) {
    return {at_once * 16u * (kNarrowStage / 2), row_blocks * (mx ? 2u : 4u) * 512u, nb * kNarrowStage * 16u};
}

B200_DEVICE void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// kNB: columns / 8.  kTokens: B lies [n][k], else [k][n].  kExact: an fp32 C.  mma.sync cuts its sums off as tcgen05.mma does (fp4_dense_wide.cuh):
// the 4,096 values of k that a warp has of 28672 x 8192 left them off by 3.5e-6 of their size.  They are therefore added, rounded, to others every
// 512: 3e-7, for 0 to 2.6 us of 33 to 58.
template <typename T, bool kMx, int kNB, bool kTokens, bool kExact>
__global__ void __launch_bounds__(32 * (kNarrowWarps + kNarrowLoaders), 1) fp4_narrow_kernel(const __grid_constant__ CUtensorMap tmap_a, const NarrowParams p) {
    using W = Widen<T, kMx>;
    constexpr uint32_t kGroups = kMx ? 2 : 4, kCols = 8 * kNB, kStepB = kNB * kNarrowStep * 16u;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw), pad = (1024u - (raw_addr & 1023u)) & 1023u, base = raw_addr + pad;
    uint8_t *smem = smem_raw + pad;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const NarrowStage size = narrow_stage(kMx, p.at_once, p.row_blocks, kNB);
    const uint32_t stage_bytes = size.bytes(), consumers = p.at_once * p.slices;
    const uint32_t bars = base + p.stages * stage_bytes, full = bars, empty = bars + 8u * kNarrowMaxStages, first_stage = base;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + (size_t)p.stages * stage_bytes + 16 * kNarrowMaxStages);
    float *sums = reinterpret_cast<float *>(smem + (size_t)p.stages * stage_bytes + 256);
    const uint32_t n0 = blockIdx.y * kCols;
    const uint32_t tile_begin = (uint32_t)((uint64_t)p.tiles * blockIdx.x / gridDim.x), tile_end = (uint32_t)((uint64_t)p.tiles * (blockIdx.x + 1u) / gridDim.x);
    const uint32_t k_stages = (p.d.k + kNarrowStage - 1) / kNarrowStage;

    if (tid == 0) {
        for (uint32_t s = 0; s < p.stages; ++s) {
            ptx::mbar_init(full + 8u * s, 1 + 32);  // the copies of A, and B's warp
            ptx::mbar_init(empty + 8u * s, consumers);
        }
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_a);
    }
    // columns past the end stay zeros, as far as B's warps do not come to them
    for (uint32_t i = tid; i < p.stages * (size.b / 16u); i += blockDim.x)
        ptx::st_shared_v4(first_stage + i / (size.b / 16u) * stage_bytes + size.values + size.scales + i % (size.b / 16u) * 16u, make_uint4(0u, 0u, 0u, 0u));
    ptx::wait_for_grids_before();
    __syncthreads();
    uint32_t s = 0, phase = 0;
    bool alive = true;
    auto step_on = [&]() {
        s = s + 1 == p.stages ? 0u : s + 1;
        phase ^= s == 0 ? 1u : 0u;
    };
    auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, ptx::mbar_wait(bar, parity, abort_flag, p.wait_limit_ns)) != 0; };

    if (warp == consumers) {
        // =========================================================== A: values in one box, 128 bytes a row, scales by row blocks
        const uint32_t on = lane == 0 ? 1u : 0u;
        for (uint32_t tile0 = tile_begin; alive && tile0 < tile_end; tile0 += p.at_once) {
            const uint32_t m0 = tile0 * 16u, rows = min(min(p.at_once, tile_end - tile0) * 16u, p.d.m - m0);
            const uint32_t block0 = m0 / 128u, blocks = (m0 + rows - 1u) / 128u - block0 + 1u;
            const uint8_t *scales = p.d.scales + (uint64_t)block0 * p.d.groups * 512u;
            for (uint32_t ks = 0; ks < k_stages; ++ks) {
                alive = wait(empty + 8u * s, phase ^ 1u);
                if (!alive) break;
                const uint32_t at = first_stage + s * stage_bytes, g0 = ks * kGroups, bytes = min(kGroups, p.d.groups - g0) * 512u;
                ptx::mbar_arrive_expect_tx_if(on, full + 8u * s, size.values + blocks * bytes);
                ptx::tma_load_2d_if(on, at, &tmap_a, (int32_t)(ks * (kNarrowStage / 2)), (int32_t)m0, full + 8u * s);
                for (uint32_t b = 0; b < blocks; ++b)
                    ptx::bulk_load_if(on, at + size.values + b * (kGroups * 512u), scales + ((uint64_t)b * p.d.groups + g0) * 512u, bytes, full + 8u * s);
                step_on();
            }
        }
    } else if (warp > consumers) {
        // =========================================================== B.  [n][k]: 16 bytes of a column for each lane and word of codes;
        // [k][n]: rows of 8 columns, in the order that puts the eight which one operand needs side by side
        const T *b = reinterpret_cast<const T *>(p.d.b);
        const uint32_t loads = kTokens ? min((uint32_t)kCols, p.d.n - n0) : kNB * 8u;
        bool mine = warp == consumers + 1u;
        for (uint32_t tile0 = tile_begin; alive && tile0 < tile_end; tile0 += p.at_once) {
            for (uint32_t ks = 0; ks < k_stages; ++ks, mine = !mine) {
                if (!mine) {
                    step_on();
                    continue;
                }
                alive = wait(empty + 8u * s, phase ^ 1u);
                if (!alive) break;
                const uint32_t to = first_stage + s * stage_bytes + size.values + size.scales;
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)kNB * 8u; ++i) {
                    if (i >= loads) break;
                    uint32_t at, left;
                    const T *src;
                    if constexpr (kTokens) {  // lane: which 16 bytes of a column's 512
                        const uint32_t k = ks * kNarrowStage + lane * 8u, step = lane / 16u, tt = lane / 4u % 4u, w = lane % 4u;
                        at = step * kStepB + ((i / 8u * 4u + w) * 32u + i % 8u * 4u + tt) * 16u;
                        left = k < p.d.k ? min(8u, p.d.k - k) : 0u;
                        src = b + (int64_t)(n0 + i) * p.d.ldb + k;
                    } else {
                        const uint32_t nb = i / 8u, kk = i % 4u * 32u + lane, k = ks * kNarrowStage + i % 8u * 32u + lane, col = n0 + nb * 8u;
                        const uint32_t order = W::kNeighbours ? lane : (lane & ~7u) | (lane & 3u) << 1 | (lane >> 2 & 1u);
                        at = i % 8u / 4u * kStepB + nb * (kNarrowStep * 16u) + ((order << 2) + (kk >> 5)) * 16u;
                        left = k < p.d.k && col < p.d.n ? min(8u, p.d.n - col) : 0u;
                        src = b + (int64_t)k * p.d.ldb + col;
                    }
                    if (p.d.b_wide) {
                        ptx::cp_async_16(to + at, left ? src : b, left * 2u);
                    } else {
                        alignas(16) T v[8];
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) v[e] = e < left ? src[e] : Elem<T>::from_float(0.f);
                        ptx::st_shared_v4(to + at, *reinterpret_cast<const uint4 *>(v));
                    }
                }
                if (p.d.b_wide) ptx::cp_async_arrive(full + 8u * s);
                else ptx::mbar_arrive(full + 8u * s);
                step_on();
            }
        }
        ptx::cp_async_commit();
        ptx::cp_async_wait_group<0>();
    } else if (warp < consumers) {
        const uint32_t mine = warp / p.slices, slice = warp % p.slices, r_of_g = (g >> 1) | (g & 1u) << 2;
        const LeftOver rest(W::kLeft, kMx ? 1.f : *reinterpret_cast<const volatile float *>(p.d.whole));
        for (uint32_t tile0 = tile_begin; alive && tile0 < tile_end; tile0 += p.at_once) {
            const uint32_t m0 = tile0 * 16u, row = m0 + mine * 16u + r_of_g;
            const bool busy = tile0 + mine < tile_end;
            const uint32_t values_at = (mine * 16u + r_of_g) * 128u;
            // the words of scales of rows `row` and `row` + 8; those of a tile past the end may be anywhere in the stage
            auto scale_at = [&](uint32_t r) { return size.values + (busy ? r / 128u - m0 / 128u : 0u) * (kGroups * 512u) + (r & 31u) * 16u + (r >> 5 & 3u) * 4u; };
            const uint32_t lo_at = scale_at(row), hi_at = scale_at(row + 8u);
            float acc[kNB][4] = {}, sum[kNB][4] = {};
            uint32_t turn = slice;  // steps until this warp's next one
            uint32_t taken = 0;     // steps that are in `acc`
            for (uint32_t ks = 0; ks < k_stages; ++ks) {
                alive = wait(full + 8u * s, phase);
                if (!alive) break;
#pragma unroll
                for (uint32_t step = 0; step < kNarrowStage / kNarrowStep; ++step) {
                    if (turn != 0) {
                        --turn;
                        continue;
                    }
                    turn = p.slices - 1u;
                    const uint32_t at = first_stage + s * stage_bytes, b_at = at + size.values + size.scales + step * kStepB;
                    const uint32_t piece = at + values_at + ((step * 4u + t) ^ r_of_g) * 16u;
                    const uint4 lo = ptx::ld_shared_v4(piece), hi = ptx::ld_shared_v4(piece + 8u * 128u);
                    const uint32_t group = kMx ? step : step * 2u + (t >> 1);
                    uint32_t f_lo = ptx::ld_shared_u32(at + lo_at + group * 512u), f_hi = ptx::ld_shared_u32(at + hi_at + group * 512u);
                    if (ks * kGroups + group >= p.d.groups) f_lo = f_hi = 0u;  // (not loaded)
                    auto multiply = [&](auto twice) {
                        constexpr bool kTwice = decltype(twice)::value;
                        uint32_t sl[2], sh[2];
                        if constexpr (kMx) {
                            sl[0] = sl[1] = W::template scale<kTwice>(f_lo >> t * 8u & 0xFFu);
                            sh[0] = sh[1] = W::template scale<kTwice>(f_hi >> t * 8u & 0xFFu);
                        } else {
                            W::two_scales(f_lo >> (t & 1u) * 16u, sl);
                            W::two_scales(f_hi >> (t & 1u) * 16u, sh);
                        }
#pragma unroll
                        for (uint32_t w = 0; w < 4; ++w) {
                            uint32_t pl[4], ph[4];
                            W::template pairs<kTwice>(w == 0 ? lo.x : w == 1 ? lo.y : w == 2 ? lo.z : lo.w, sl[w >> 1], pl);
                            W::template pairs<kTwice>(w == 0 ? hi.x : w == 1 ? hi.y : w == 2 ? hi.z : hi.w, sh[w >> 1], ph);
#pragma unroll
                            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                                uint32_t bf[4];  // operands of two MMAs: b0, b1 of either
                                if constexpr (kTokens) {
                                    const uint4 v = ptx::ld_shared_v4(b_at + (nb * 4u + w) * 512u + lane * 16u);
                                    bf[0] = W::kNeighbours ? v.x : __byte_perm(v.x, v.z, 0x5410);  // k 0, 1 or 0, 4
                                    bf[1] = W::kNeighbours ? v.y : __byte_perm(v.x, v.z, 0x7632);  // 2, 3 or 1, 5
                                    bf[2] = W::kNeighbours ? v.z : __byte_perm(v.y, v.w, 0x5410);  // 4, 5 or 2, 6
                                    bf[3] = W::kNeighbours ? v.w : __byte_perm(v.y, v.w, 0x7632);  // 6, 7 or 3, 7
                                } else {
                                    // matrix m holds the values of k of pair m of the word of the four lanes' ranges, its row r at slot 4 (8 w + 2 m + r % 2) + r / 2
                                    const uint32_t mat = lane >> 3, r = lane & 7u;
                                    ldmatrix_x4_trans(b_at + nb * (kNarrowStep * 16u) + (((w * 8u + mat * 2u + (r & 1u)) << 2) + (r >> 1)) * 16u, bf);
                                }
                                mma_16x8x16<T>(acc[nb], pl[0], ph[0], pl[1], ph[1], bf[0], bf[1]);
                                mma_16x8x16<T>(acc[nb], pl[2], ph[2], pl[3], ph[3], bf[2], bf[3]);
                            }
                        }
                    };
                    if (kMx && __any_sync(0xFFFFFFFFu, W::needs_two(f_lo) || W::needs_two(f_hi))) multiply(std::true_type());
                    else multiply(std::false_type());
                    if (kExact && ++taken == kNarrowRun) {
                        taken = 0;
#pragma unroll
                        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) {
                                sum[nb][e] += acc[nb][e];
                                acc[nb][e] = 0.f;
                            }
                    }
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(empty + 8u * s);
                step_on();
            }
            if constexpr (kExact) {
#pragma unroll
                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) acc[nb][e] += sum[nb][e];
            }
            // ---- to C, over shared memory where k was sliced: [warp][column][row].  A warp whose wait gave up comes to the barrier as well: the
            // others, whose waits may have ended in time, count on it there, and no wait of theirs would end it.  All leave then.
            if (p.slices > 1) {
#pragma unroll
                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) sums[(warp * kCols + nb * 8u + t * 2u + (e & 1u)) * 16u + (e >> 1) * 8u + r_of_g] = acc[nb][e];
                if (ptx::bar_or(1, consumers * 32u, !alive)) break;
                for (uint32_t i = tid; i < p.at_once * 16u * kCols; i += consumers * 32u) {
                    const uint32_t r = i % 16u, col = i / 16u % kCols, tile = i / (16u * kCols);
                    float v[1] = {0.f};
                    for (uint32_t z = 0; z < p.slices; ++z) v[0] += sums[((tile * p.slices + z) * kCols + col) * 16u + r];
                    v[0] = rest.apply(v[0]);
                    const uint32_t c_row = m0 + tile * 16u + r;
                    if (tile0 + tile < tile_end && c_row < p.d.m && n0 + col < p.d.n) store_row(p.d.c, c_row, n0 + col, p.d.n, v);
                }
                asm volatile("bar.sync 1, %0;" ::"r"(consumers * 32u) : "memory");  // (the next tiles' sums go there)
            } else if (busy && alive) {
#pragma unroll
                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t col = n0 + nb * 8u + t * 2u + (e & 1u), c_row = row + (e >> 1) * 8u;
                        float v[1] = {rest.apply(acc[nb][e])};
                        if (c_row < p.d.m && col < p.d.n) store_row(p.d.c, c_row, col, p.d.n, v);
                    }
            }
        }
    }
    __syncwarp();
    if (*abort_flag) {
        const uint64_t t0 = ptx::global_timer_ns();
        while (ptx::global_timer_ns() - t0 < 20000000ull) __nanosleep(1000);  // what is under way to shared memory arrives
        if (lane == 0) atomicAdd(p.status, 1u);
    }
}

}  // namespace fp4
}  // namespace b200spmm
