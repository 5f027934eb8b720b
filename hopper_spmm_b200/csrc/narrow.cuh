// A few columns times rows of a weight matrix that is read once: what a block of threads does.
//
// Bound: one read of the matrix.  Each warp copies its own rows to a ring of its own in shared memory (cp.async, 16 bytes a lane), so no warp waits for
// another while k goes by, and a wait is one for the lane's own copies.  A warp has a tile of 16 rows, or of every `slices`-th step of 128 bytes of those rows; the
// columns lie in shared memory for all warps, as a whole where there is room, else piece by piece.  16 rows x 8 columns x 16 values of k meet in mma.sync: at
// this width a product is a small part of the work, and for tcgen05 widened weights would have to go through shared or tensor memory.
//
// Lane 4 g + t of a warp holds rows g and g + 8 of the tile.  Which values of k an operand position of the MMA stands for is free as long as both operands
// agree, so a lane takes neighbours of its rows: of 4-bit integers kSpan / 4 of every kSpan, the widest span that has one scale (and one of the columns'
// scales), whose sum is multiplied by them in fp32; of 16-bit values 8 of every 32.  Columns are stored in units of 16 bytes, 8 values of k, in the order in which lanes
// t = 0..3 read them side by side, each unit in the order of the pairs that a mask takes out of a word of eight codes: 0 4, 1 5, 2 6, 3 7.
#pragma once

#include <algorithm>

#include "fp4_convert.cuh"
#include "mma_16x8x16.cuh"

namespace b200spmm {
namespace narrow {

constexpr uint32_t kTileRows = 16, kStepBytes = 128, kStageBytes = kTileRows * kStepBytes;
constexpr uint32_t kMaxSmem = 227 * 1024;

// Rows of weights: 4-bit integers or 16-bit values.
struct Matrix {
    const uint8_t *values;
    uint64_t pitch;      // bytes between rows
    uint32_t row_bytes;  // of a row
    uint32_t groups, shift;  // of a row that have a scale, each of 2^shift columns
    uint32_t rows;       // between the scales of two groups
    const uint16_t *scales;
    const uint8_t *zeros;  // anything where there are none
    uint32_t zero_mask, zero_else;
    bool bf16_scales;
};

// T: the type of both operands of the MMA.  kSpan: columns of 4-bit integers that share their scales, 32, 64 or 128; 0: the weights are T themselves.
template <typename T_, int kSpan_>
struct Weights {
    using T = T_;
    static constexpr int kSpan = kSpan_;
    static constexpr bool kCodes = kSpan > 0;
    static constexpr uint32_t kStep = kCodes ? 2 * kStepBytes : kStepBytes / 2;  // values of k
    static constexpr uint32_t kUnits = kStep / 8;                                // of a column
    static constexpr uint32_t kBlocks = kCodes ? kStep / (kCodes ? kSpan : 1) : 2;  // of a step, with a scale each; halves
    static constexpr uint32_t kWords = kCodes ? 8 / kBlocks : 1;                 // of a lane in a block: units of 8 values
    static constexpr uint32_t kEntries = kBlocks / 2;                            // scales that a lane fetches for its warp
};

// Where unit `u` (8 values of k from 8 u on) of a column lies.
template <class W>
B200_DEVICE uint32_t unit_place(uint32_t u) {
    if constexpr (W::kCodes) {
        constexpr uint32_t n = W::kSpan / 8;
        return u / n * n + u % (n / 4) * 4 + u % n / (n / 4);
    } else {
        return u;
    }
}

// The eight values of a unit in the order of its MMAs' operands.
template <class W>
B200_DEVICE uint4 unit_order(uint4 v) {
    if constexpr (W::kCodes)
        return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
    else
        return v;
}

B200_DEVICE uint32_t shared_swizzle(uint32_t row) { return (row & 1u) << 2 | (row & 2u) | (row >> 2 & 1u); }  // of a row's eight pieces: no two lanes of a load meet in a bank

// Eight codes less their zero, exactly: pairs 0 4, 1 5, 2 6, 3 7.  A code under the exponent of 1024 (or, four bits up, of 64 times 16; bf16: of 128) is that number and the
// code; `minus` takes the number and the zero away.
template <typename T> struct Widen;
// (w & mask) | bits in one instruction: with both as constants the compiler makes two of it.
template <uint32_t kMask>
B200_DEVICE uint32_t masked(uint32_t w, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(kMask), "r"(bits));
    return r;
}
B200_DEVICE uint32_t in_register(uint32_t constant) {
    uint32_t r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(constant));
    return r;
}
template <>
struct Widen<__half> {
    uint32_t low, high;  // -(1024 + zero), -(64 + zero), twice
    B200_DEVICE explicit Widen(uint32_t zero) : low(0xE400E400u | zero * 0x00010001u), high(0xD400D400u | zero * 0x00100010u) {}
    static constexpr uint32_t kBits = 0x64006400u;
    B200_DEVICE void operator()(uint32_t w, uint32_t bits, uint32_t (&out)[4]) const {
        const __half2 sixteenth = __half2half2(__ushort_as_half((unsigned short)0x2C00u));
#pragma unroll
        for (int i = 0; i < 4; i += 2, w >>= 8) {
            const uint32_t a = masked<0x000F000Fu>(w, bits), b = masked<0x00F000F0u>(w, bits);
            const __half2 x = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&low));
            const __half2 y = __hfma2(*reinterpret_cast<const __half2 *>(&b), sixteenth, *reinterpret_cast<const __half2 *>(&high));
            out[i] = *reinterpret_cast<const uint32_t *>(&x);
            out[i + 1] = *reinterpret_cast<const uint32_t *>(&y);
        }
    }
};
template <>
struct Widen<__nv_bfloat16> {
    uint32_t minus;
    B200_DEVICE explicit Widen(uint32_t zero) : minus(0xC300C300u | zero * 0x00010001u) {}
    static constexpr uint32_t kBits = 0x43004300u;
    B200_DEVICE void operator()(uint32_t w, uint32_t bits, uint32_t (&out)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i, w >>= 4) {
            const uint32_t a = masked<0x000F000Fu>(w, bits);
            const __nv_bfloat162 x = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&minus));
            out[i] = *reinterpret_cast<const uint32_t *>(&x);
        }
    }
};

// The columns in shared memory: column j at base + j * pitch (and `plane` further on its second part, where it is the sum of two), and their scales, column by column.
struct Columns {
    uint32_t base, pitch, plane;
    uint32_t scales, groups, shift;
    uint32_t steps;  // that have room
};

template <int kBytes>
B200_DEVICE void ld_shared(uint32_t addr, uint32_t *v) {
    if constexpr (kBytes == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
    else if constexpr (kBytes == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(addr) : "memory");
}

// What a warp does in a round of tiles.
struct Share {
    uint64_t row_lo, row_hi;  // of the matrix: rows g and g + 8 of the tile, as far as they exist
    uint32_t slice, slices;   // steps slice, slice + slices, ...
    uint32_t steps;           // of a whole row
    uint32_t ring;            // shared memory
    bool busy;
};

// sums[nb][e] += the products of the warp's steps: rows g (e < 2) and g + 8, columns 8 nb + 2 t + e % 2.  All threads of the block come here alike:
// stage(step, count) brings these steps of the columns to shared memory; `staged` says that they are there as a whole.
template <class W, int kNB, int kPlanes, bool kScaled, int kStages, class Stage>
B200_DEVICE void accumulate(const Matrix &m, const Share &s, const Columns &c, uint32_t n, bool staged, Stage &&stage, float (&sums)[kNB][4]) {
    using T = typename W::T;
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    // Copies run kStages steps ahead: rows g and g + 8, pieces t and t + 4.
    const uint32_t own = g * kStepBytes + (t ^ shared_swizzle(g)) * 16u, ahead = s.slices * kStepBytes;
    uint32_t copied = s.slice * kStepBytes + t * 16u;  // bytes of a row up to the next copy
    const uint8_t *lo = m.values + s.row_lo * m.pitch + copied, *hi = m.values + s.row_hi * m.pitch + copied;
    const uint32_t row_bytes = s.busy ? m.row_bytes : 0u;
    auto issue = [&](uint32_t at) {
        if constexpr (W::kCodes) {
            // (codes behind a row's end meet zeros, whatever they are)
            if (copied < row_bytes) {
                ptx::cp_async_16(at + own, lo);
                ptx::cp_async_16(at + own + 8u * kStepBytes, hi);
            }
            if (copied + 64u < row_bytes) {
                ptx::cp_async_16(at + (own ^ 64u), lo + 64);
                ptx::cp_async_16(at + (own ^ 64u) + 8u * kStepBytes, hi + 64);
            }
        } else {
            if (copied - t * 16u < row_bytes) {
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {  // zeros behind a row's end
                    const uint32_t place = copied + i * 64u, left = place < row_bytes ? min(16u, row_bytes - place) : 0u, back = left ? i * 64u : 0u - copied;
                    ptx::cp_async_16(at + (own ^ i * 64u), lo + (int32_t)back, left);
                    ptx::cp_async_16(at + (own ^ i * 64u) + 8u * kStepBytes, hi + (int32_t)back, left);
                }
            }
        }
        ptx::cp_async_commit();
        copied += ahead;
        lo += ahead;
        hi += ahead;
    };
    // Scales and zeros come by ordinary loads a step ahead, each to one lane of the four that need it: of row g (even t) or g + 8, blocks t / 2 + 2 i.
    constexpr uint32_t kEntries = W::kCodes ? W::kEntries : 1u;
    const uint32_t entry_row = (uint32_t)(t & 1u ? s.row_hi : s.row_lo);
    uint32_t scale_next[kEntries], zero_next[kEntries], entry_k = s.slice * W::kStep + (t >> 1) * (uint32_t)W::kSpan;
    auto fetch = [&]() {
        if constexpr (W::kCodes) {
#pragma unroll
            for (uint32_t i = 0; i < kEntries; ++i) {  // (behind a row's end the last one again)
                const uint32_t at = min((entry_k + 2u * i * (uint32_t)W::kSpan) >> m.shift, m.groups - 1u) * m.rows + entry_row;
                scale_next[i] = m.scales[at];
                zero_next[i] = m.zeros[at];
            }
            entry_k += s.slices * W::kStep;
        }
    };
    if (s.busy) {
#pragma unroll
        for (uint32_t i = 0; i < kStages; ++i) issue(s.ring + i * kStageBytes);
        fetch();
    }
    uint32_t column[kNB];  // this lane's, for the second operand; those behind the last are any of the others: nobody looks at their sums
#pragma unroll
    for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) column[nb] = c.base + min(nb * 8u + g, n - 1u) * c.pitch + t * 16u;
    uint32_t step = s.slice, at = s.ring;
    const uint32_t bits = W::kCodes ? in_register(Widen<T>::kBits) : 0u;
    for (uint32_t first = 0; first < s.steps; first += c.steps) {
        const uint32_t end = min(s.steps, first + c.steps);
        if (!staged) {
            if (first) __syncthreads();  // (nobody reads what was there any more)
            stage(first, end - first);
            __syncthreads();
        }
        for (; s.busy && step < end; step += s.slices) {
            uint32_t entries[kEntries];  // a scale's bits in fp32, the zero in the lowest four (a scale has 11 digits at most)
            if constexpr (W::kCodes) {
#pragma unroll
                for (uint32_t i = 0; i < kEntries; ++i) {
                    const float v = m.bf16_scales ? __uint_as_float(scale_next[i] << 16) : __half2float(__ushort_as_half((unsigned short)scale_next[i]));
                    entries[i] = (__float_as_uint(v) & ~15u) | (zero_next[i] & m.zero_mask) | m.zero_else;
                }
                fetch();
            }
            ptx::cp_async_wait_group<kStages - 1>();
            __syncwarp();
            const uint32_t x_at = (step - first) * (W::kUnits * 16u);
#pragma unroll
            for (uint32_t b = 0; b < W::kBlocks; ++b) {
                constexpr uint32_t kRegs = W::kCodes ? W::kWords : 4u;
                uint32_t w_lo[kRegs], w_hi[kRegs];
                const uint32_t piece = W::kBlocks == 2 ? 4u * b + t : W::kBlocks == 4 ? 2u * b + (t >> 1) : b, rest = W::kBlocks == 2 ? 0u : W::kBlocks == 4 ? (t & 1u) * 8u : t * 4u;
                const uint32_t from = at + g * kStepBytes + (piece ^ shared_swizzle(g)) * 16u + rest;
                ld_shared<4 * kRegs>(from, w_lo);
                ld_shared<4 * kRegs>(from + 8u * kStepBytes, w_hi);
                if (b + 1 == W::kBlocks) {  // the stage is read: what comes kStages steps later may be copied there
                    __syncwarp();
                    issue(at);
                    at = at + kStageBytes == s.ring + kStages * kStageBytes ? s.ring : at + kStageBytes;
                }
                if constexpr (!W::kCodes) {
#pragma unroll
                    for (int plane = 0; plane < kPlanes; ++plane)
#pragma unroll
                        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                            const uint4 x = ptx::ld_shared_v4(column[nb] + x_at + b * 64u + plane * c.plane);
                            fp4::mma_16x8x16<T>(sums[nb], w_lo[0], w_hi[0], w_lo[1], w_hi[1], x.x, x.y);
                            fp4::mma_16x8x16<T>(sums[nb], w_lo[2], w_hi[2], w_lo[3], w_hi[3], x.z, x.w);
                        }
                } else {
                    const uint32_t source = (lane & ~3u) | (b & 1u) << 1;
                    const uint32_t e_lo = __shfl_sync(0xFFFFFFFFu, entries[b >> 1], source), e_hi = __shfl_sync(0xFFFFFFFFu, entries[b >> 1], source | 1u);
                    const Widen<T> widen_lo(e_lo & 15u), widen_hi(e_hi & 15u);
                    float part[kNB][4];
#pragma unroll
                    for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) part[nb][0] = part[nb][1] = part[nb][2] = part[nb][3] = 0.f;
#pragma unroll
                    for (uint32_t w = 0; w < W::kWords; ++w) {
                        uint32_t a_lo[4], a_hi[4];
                        widen_lo(w_lo[w], bits, a_lo);
                        widen_hi(w_hi[w], bits, a_hi);
#pragma unroll
                        for (int plane = 0; plane < kPlanes; ++plane)
#pragma unroll
                            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                                const uint4 x = ptx::ld_shared_v4(column[nb] + x_at + (b * W::kWords + w) * 64u + plane * c.plane);
                                fp4::mma_16x8x16<T>(part[nb], a_lo[0], a_hi[0], a_lo[1], a_hi[1], x.x, x.y);
                                fp4::mma_16x8x16<T>(part[nb], a_lo[2], a_hi[2], a_lo[3], a_hi[3], x.z, x.w);
                            }
                    }
                    const float s_lo = __uint_as_float(e_lo & ~15u), s_hi = __uint_as_float(e_hi & ~15u);
#pragma unroll
                    for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                        float x0 = 1.f, x1 = 1.f;
                        if constexpr (kScaled) {
                            const uint32_t group = min((step * W::kStep + b * (uint32_t)W::kSpan) >> c.shift, c.groups - 1u), j = nb * 8u + t * 2u;
                            x0 = __uint_as_float(ptx::ld_shared_u32(c.scales + (min(j, n - 1u) * c.groups + group) * 4u));
                            x1 = __uint_as_float(ptx::ld_shared_u32(c.scales + (min(j + 1u, n - 1u) * c.groups + group) * 4u));
                        }
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) sums[nb][e] = fmaf(kScaled ? part[nb][e] * (e & 1u ? x1 : x0) : part[nb][e], e < 2 ? s_lo : s_hi, sums[nb][e]);
                    }
                }
            }
        }
    }
    __syncwarp();
}

// A warp's sums to its ring, [column][row], and one of a tile's from those of its slices, in order.
template <int kNB>
B200_DEVICE void leave_sums(float *ring, const float (&sums)[kNB][4]) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
#pragma unroll
    for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) ring[(nb * 8u + t * 2u + (e & 1u)) * kTileRows + (e >> 1) * 8u + g] = sums[nb][e];
}
B200_DEVICE float joined(const float *rings, uint32_t ring_floats, uint32_t first_warp, uint32_t slices, uint32_t column, uint32_t row) {
    float v = 0.f;
    for (uint32_t z = 0; z < slices; ++z) v += rings[(first_warp + z) * ring_floats + column * kTileRows + row];
    return v;
}

// How a block goes through `tiles` of its own with up to `warps` warps: as many tiles at a time in every round, each cut along k as far as there are warps and steps.
struct Split {
    uint32_t at_once, slices, rounds;
    __host__ __device__ Split(uint32_t tiles, uint32_t steps, uint32_t warps) {
        rounds = (tiles + warps - 1) / warps;
        at_once = (tiles + rounds - 1) / rounds;
        slices = warps / at_once;
        if (slices > steps) slices = steps;
        if (slices < 1) slices = 1;
    }
};

// Sources of columns: eight values of k, from 8 u on, of column j as a unit.
template <typename T>
struct Plain {  // 16-bit values `along` elements apart along k, `across` between columns
    const T *x;
    int64_t along, across;
    bool wide;  // neighbours along k, and every column starts on 16 bytes
    uint32_t k;
    B200_DEVICE uint4 operator()(uint32_t j, uint32_t u) const {
        const T *p = x + (int64_t)j * across + (int64_t)u * 8 * along;
        const uint32_t left = u * 8u < k ? k - u * 8u : 0u;
        if (wide && left >= 8u) return *reinterpret_cast<const uint4 *>(p);
        alignas(16) T v[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = e < left ? p[(int64_t)e * along] : fp4::Elem<T>::from_float(0.f);
        return *reinterpret_cast<const uint4 *>(v);
    }
};
struct Eights {  // e4m3, as fp16
    const uint8_t *x;
    int64_t across;
    bool wide;  // every column starts on 8 bytes
    uint32_t k;
    B200_DEVICE uint4 operator()(uint32_t j, uint32_t u) const {
        const uint8_t *p = x + (int64_t)j * across + (int64_t)u * 8;
        const uint32_t left = u * 8u < k ? k - u * 8u : 0u;
        alignas(8) uint16_t v[4];
        if (wide && left >= 8u) {
            *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = (uint16_t)((2 * e < left ? p[2 * e] : 0u) | (2 * e + 1 < left ? p[2 * e + 1] : 0u) << 8);
        }
        uint32_t h[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[e]) : "h"(v[e]));
        return make_uint4(h[0], h[1], h[2], h[3]);
    }
};

// `count` steps of n columns from step `first` on to shared memory, by all threads.  A warp takes 32 neighbouring units of a column, or, where neighbours lie across
// the columns, up to 32 columns of a unit.
template <class W, class Source>
B200_DEVICE void stage_columns(const Source &from, const Columns &c, uint32_t first, uint32_t count, uint32_t n, bool across) {
    const uint32_t units = count * W::kUnits, u0 = first * W::kUnits, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31u;
    auto put = [&](uint32_t j, uint32_t u, uint4 v) { ptx::st_shared_v4(c.base + j * c.pitch + unit_place<W>(u) * 16u, unit_order<W>(v)); };
    if (across) {
        for (uint32_t u = warp; u < units; u += warps)
            if (lane < n) put(lane, u, from(lane, u0 + u));
        return;
    }
    // pieces of 32 units, all columns of one after the other; four at a time
    constexpr uint32_t kBatch = 4;
    uint32_t j = 0, u = warp * 32u + lane;
    while (true) {
        uint4 v[kBatch];
        uint32_t js[kBatch], us[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            while (u >= units && j < n) {
                u -= units;
                ++j;
            }
            js[b] = j;
            us[b] = u;
            if (j < n) v[b] = from(j, u0 + u);
            u += warps * 32u;
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b)
            if (js[b] < n) put(js[b], us[b], v[b]);
        if (js[kBatch - 1] >= n) return;
    }
}

// Bytes between columns with room for `steps`: lanes of two neighbouring columns read from different halves of 128 bytes.
template <class W>
__host__ __device__ constexpr uint32_t column_pitch(uint32_t steps) { return (steps * W::kUnits * 16u + 127u) / 128u * 128u + 64u; }

}  // namespace narrow
}  // namespace b200spmm
