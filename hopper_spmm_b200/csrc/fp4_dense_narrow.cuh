// Product of a 4-bit matrix with a few columns of 16-bit values: decoding.
//
//     C[m, 0..n) = s_A  sum over k  (a[m, k] sa[m, k / block]) B[k, 0..n)
//
// Bound: one read of A.  The matrix goes from memory through registers: a warp widens its codes to 16 bits, exactly (an e2m1
// number times an e4m3 scale has six significant bits), and multiplies them with eight columns of B at a time (mma.sync, 16 rows x
// 8 columns x 16 values of k; at this width a product is a small part of what the reading takes, and the matrix would have
// to go through shared or tensor memory for tcgen05).
//
// A warp takes steps of 32 rows x 128 values of k.  The rows are i, i + 32, i + 64, i + 96 of a block of 128 for eight neighbouring i:
// their scales are whole 16-byte pieces.  Lane 4 g + t reads 16 bytes of values, 32 codes, of each of its four rows i0 + g + 32 q from k = 32 t on, and
// one piece with the scales.  Which k an operand position of the MMA stands for is free as long as both operands agree: lane t's
// positions of MMA j are pairs 2 (j % 2) and 2 (j % 2) + 1 of word j / 2 of its four, as Widen makes them.
// The eight warps of a block share out k, 128 values at a time, and their sums meet in shared memory in a fixed order.
#pragma once

#include <type_traits>

#include "fp4_widen.cuh"

namespace b200spmm {
namespace fp4 {

constexpr int kNarrowWarps = 8, kNarrowAhead = 4;  // steps of A under way
constexpr uint32_t kNarrowK = 128;

template <int kNB, int kU>
struct NarrowCfg {
    static constexpr uint32_t kStepBytes = 5 * 32 * 16;           // of a warp: four pieces of values, one of scales, a lane
    static constexpr uint32_t kRingBytes = kNarrowWarps * kNarrowAhead * kStepBytes;
    static constexpr uint32_t kBBytes = kNarrowK * kNB * 16;      // of a warp's 128 values of k
    static constexpr uint32_t kBRingBytes = kNarrowWarps * 2 * kBBytes;
    static constexpr uint32_t kRows = 32 * kU;
    static constexpr uint32_t kSumBytes = kNarrowWarps * kRows * kNB * 8 * 4;
    static constexpr size_t kSmemBytes = kRingBytes + kBRingBytes > kSumBytes ? kRingBytes + kBRingBytes : kSumBytes;
};

template <typename T>
B200_DEVICE void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

B200_DEVICE void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// kNB: columns / 8.  kU: steps of 32 rows of a block.  kTokens: B lies [n][k], else [k][n].
template <typename T, bool kMx, int kNB, int kU, bool kTokens>
__global__ void __launch_bounds__(32 * kNarrowWarps, 2) fp4_narrow_kernel(const DenseParams p) {
    using Cfg = NarrowCfg<kNB, kU>;
    using W = Widen<T, kMx>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t ring = ptx::smem_u32(smem) + warp * kNarrowAhead * Cfg::kStepBytes + lane * 16u;
    const uint32_t b_ring = ptx::smem_u32(smem) + Cfg::kRingBytes + warp * 2 * Cfg::kBBytes;
    uint8_t *b_smem = smem + Cfg::kRingBytes + warp * 2 * Cfg::kBBytes;
    const uint32_t row_block = blockIdx.x / (4 / kU), u0 = blockIdx.x % (4 / kU) * kU;
    const uint32_t n0 = blockIdx.y * (8 * kNB);
    const uint32_t chunks = (p.k + kNarrowK - 1) / kNarrowK;
    const uint32_t mine = chunks > warp ? (chunks - warp + kNarrowWarps - 1) / kNarrowWarps : 0;  // of this warp

    ptx::wait_for_grids_before();

    // ---- A: step i of this warp is 32 rows of its chunk i / kU
    auto fetch_a = [&](uint32_t i) {
        if (i < mine * kU) {
            const uint32_t chunk = warp + i / kU * kNarrowWarps, u = u0 + i % kU;
            const uint32_t row = row_block * 128u + u * 8u + g, at = chunk * (kNarrowK / 2) + t * 16u;
            const uint32_t dst = ring + i % kNarrowAhead * Cfg::kStepBytes;
            const bool in = at < p.pitch;
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                const bool there = in && row + q * 32u < p.m;
                ptx::cp_async_16(dst + q * 512u, there ? p.values + (uint64_t)(row + q * 32u) * p.pitch + at : p.values, there ? 16u : 0u);
            }
            const uint32_t group = kMx ? chunk : chunk * 2u + (t >> 1);
            const bool there = group < p.groups;
            ptx::cp_async_16(dst + 4u * 512u, there ? p.scales + scale_word(row_block * 128u + u * 8u + g, group, p.groups) : p.scales, there ? 16u : 0u);
        }
    };
    // ---- B: 128 values of k of all columns.  [n][k]: what the lane's operands are made of, piece by piece.  [k][n]: rows of 8
    // columns, in the order that puts the eight which one operand needs side by side.
    auto fetch_b = [&](uint32_t i) {
        if (i >= mine) return;
        const uint32_t k0 = (warp + i * kNarrowWarps) * kNarrowK, buf = i & 1u;
        const T *b = reinterpret_cast<const T *>(p.b);
        if constexpr (kTokens) {
#pragma unroll
            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                const uint32_t col = n0 + nb * 8u + g;
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) {
                    const uint32_t k = k0 + t * 32u + w * 8u, at = buf * Cfg::kBBytes + (nb * 4u + w) * 512u + lane * 16u;
                    const uint32_t left = col < p.n && k < p.k ? min(8u, p.k - k) : 0u;
                    const T *src = b + (int64_t)col * p.ldb + k;
                    if (p.b_wide) {
                        ptx::cp_async_16(b_ring + at, left ? src : b, left * 2u);
                    } else {
                        T v[8];
#pragma unroll
                        for (uint32_t j = 0; j < 8; ++j) v[j] = j < left ? src[j] : Elem<T>::from_float(0.f);
                        *reinterpret_cast<uint4 *>(b_smem + at) = *reinterpret_cast<const uint4 *>(v);
                    }
                }
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t kk = j * 32u + lane, k = k0 + kk;
                const uint32_t in_lane = kk & 31u, 
                               order = W::kNeighbours ? in_lane : (in_lane & ~7u) | (in_lane & 3u) << 1 | (in_lane >> 2 & 1u), slot = (order << 2) + (kk >> 5);
#pragma unroll
                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                    const uint32_t col = n0 + nb * 8u, at = buf * Cfg::kBBytes + nb * (kNarrowK * 16u) + slot * 16u;
                    const uint32_t left = k < p.k && col < p.n ? min(8u, p.n - col) : 0u;
                    const T *src = b + (int64_t)k * p.ldb + col;
                    if (p.b_wide) {
                        ptx::cp_async_16(b_ring + at, left ? src : b, left * 2u);
                    } else {
                        T v[8];
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) v[e] = e < left ? src[e] : Elem<T>::from_float(0.f);
                        *reinterpret_cast<uint4 *>(b_smem + at) = *reinterpret_cast<const uint4 *>(v);
                    }
                }
            }
        }
    };

    float acc[kU][2][kNB][4] = {};
    // One group of copies a step.  B of a chunk comes with the first step of the chunk before it.
    fetch_b(0);
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)kNarrowAhead - 1; ++i) {
        fetch_a(i);
        ptx::cp_async_commit();
    }
    for (uint32_t chunk = 0; chunk < mine; ++chunk) {
        uint32_t bf[kNB][4][4];  // operands of the eight MMAs: b0, b1 of two of them for each word of codes
#pragma unroll
        for (uint32_t u = 0; u < (uint32_t)kU; ++u) {
            const uint32_t i = chunk * kU + u;
            if (u == 0) {
                // B of this chunk has been under way since the first step of the last one: all but the kNarrowAhead - 2 youngest groups
                // are waited for below, and it is older than those if a chunk has that many steps; else everything is
                if constexpr (kU >= kNarrowAhead - 1) ptx::cp_async_wait_group<kNarrowAhead - 2>();
                else ptx::cp_async_wait_group<0>();
                __syncwarp();
                const uint32_t buf = b_ring + (chunk & 1u) * Cfg::kBBytes;
#pragma unroll
                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        if constexpr (kTokens) {
                            const uint4 v = ptx::ld_shared_v4(buf + (nb * 4u + w) * 512u + lane * 16u);
                            bf[nb][w][0] = W::kNeighbours ? v.x : __byte_perm(v.x, v.z, 0x5410);  // k 0, 1 or 0, 4
                            bf[nb][w][1] = W::kNeighbours ? v.y : __byte_perm(v.x, v.z, 0x7632);  // 2, 3 or 1, 5
                            bf[nb][w][2] = W::kNeighbours ? v.z : __byte_perm(v.y, v.w, 0x5410);  // 4, 5 or 2, 6
                            bf[nb][w][3] = W::kNeighbours ? v.w : __byte_perm(v.y, v.w, 0x7632);  // 6, 7 or 3, 7
                        } else {
                            // matrix i holds the values of k of pair i of word w of the four lanes' ranges, its row r at slot 4 (8 w + 2 i + r % 2) + r / 2
                            const uint32_t mat = lane >> 3, r = lane & 7u;
                            ldmatrix_x4_trans(buf + nb * (kNarrowK * 16u) + (((w * 8u + mat * 2u + (r & 1u)) << 2) + (r >> 1)) * 16u, bf[nb][w]);
                        }
                    }
                __syncwarp();
                fetch_b(chunk + 1);  // (goes into the buffer of the chunk before this one, which every lane has read)
            } else {
                ptx::cp_async_wait_group<kNarrowAhead - 2>();
            }
            fetch_a(i + kNarrowAhead - 1);  // (into the place of step i - 1, which this lane alone reads)
            ptx::cp_async_commit();
            const uint32_t at = ring + i % kNarrowAhead * Cfg::kStepBytes;
            const uint4 sc = ptx::ld_shared_v4(at + 4u * 512u);
            auto multiply = [&](auto twice, uint32_t tile) {
                constexpr bool kTwice = decltype(twice)::value;
                const uint4 lo = ptx::ld_shared_v4(at + tile * 1024u), hi = ptx::ld_shared_v4(at + tile * 1024u + 512u);
                const uint32_t s_lo = tile ? sc.z : sc.x, s_hi = tile ? sc.w : sc.y;
                uint32_t sl[2], sh[2];
                if constexpr (kMx) {
                    sl[0] = sl[1] = W::template scale<kTwice>(s_lo >> t * 8u & 0xFFu);
                    sh[0] = sh[1] = W::template scale<kTwice>(s_hi >> t * 8u & 0xFFu);
                } else {
                    const uint32_t at_byte = (t & 1u) * 16u;
                    sl[0] = W::template scale<kTwice>(s_lo >> at_byte & 0xFFu);
                    sl[1] = W::template scale<kTwice>(s_lo >> (at_byte + 8u) & 0xFFu);
                    sh[0] = W::template scale<kTwice>(s_hi >> at_byte & 0xFFu);
                    sh[1] = W::template scale<kTwice>(s_hi >> (at_byte + 8u) & 0xFFu);
                }
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) {
                    uint32_t pl[4], ph[4];
                    W::template pairs<kTwice>(wl[w], sl[w >> 1], pl);
                    W::template pairs<kTwice>(wh[w], sh[w >> 1], ph);
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
                            mma_16x8x16<T>(acc[u][tile][nb], pl[2 * j], ph[2 * j], pl[2 * j + 1], ph[2 * j + 1], bf[nb][w][2 * j], bf[nb][w][2 * j + 1]);
                }
            };
            if (kMx && __any_sync(0xFFFFFFFFu, W::needs_two(sc.x) || W::needs_two(sc.y) || W::needs_two(sc.z) || W::needs_two(sc.w))) {
                multiply(std::true_type(), 0);
                multiply(std::true_type(), 1);
            } else {
                multiply(std::false_type(), 0);
                multiply(std::false_type(), 1);
            }
        }
    }
    ptx::cp_async_wait_group<0>();
    __syncthreads();

    // ---- the warps' sums meet: [warp][column][row], rows in order
    float *sums = reinterpret_cast<float *>(smem);
    constexpr uint32_t kRows = Cfg::kRows, kCols = 8 * kNB;
#pragma unroll
    for (uint32_t u = 0; u < (uint32_t)kU; ++u)
#pragma unroll
        for (uint32_t tile = 0; tile < 2; ++tile)
#pragma unroll
            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t q = tile * 2u + (e >> 1), col = nb * 8u + t * 2u + (e & 1u);
                    sums[(warp * kCols + col) * kRows + q * (8u * kU) + u * 8u + g] = acc[u][tile][nb][e];
                }
    __syncthreads();
    const float whole = (kMx ? 1.f : *reinterpret_cast<const volatile float *>(p.whole)) * 1.f;
    for (uint32_t i = tid; i < kRows * kCols; i += 32 * kNarrowWarps) {
        // neighbouring lanes write neighbours: rows where C lies column by column, else columns
        const uint32_t r = p.c.transposed ? i % kRows : i / kCols, col = p.c.transposed ? i / kRows : i % kCols;
        const uint32_t row = row_block * 128u + r / (8u * kU) * 32u + u0 * 8u + r % (8u * kU);
        float v[1] = {0.f};
#pragma unroll
        for (uint32_t w = 0; w < (uint32_t)kNarrowWarps; ++w) v[0] += sums[(w * kCols + col) * kRows + r];
        v[0] = v[0] * W::kLeft * whole;
        if (row < p.m && n0 + col < p.n) store_row(p.c, row, n0 + col, p.n, v);
    }
}

}  // namespace fp4
}  // namespace b200spmm
