// A few columns times rows of a weight matrix that is read once: what a block of threads does.
//
// Bound: one read of the matrix.  Each warp copies its own rows to a ring of its own in shared memory (cp.async, 16 bytes a lane), so no warp waits for
// another while k goes by, and a wait is one for the warp's own copies.  A warp has a tile of 16 rows at a time, or every `slices`-th step of
// those rows; its copies run ahead into its next tile.  The columns lie in shared memory for all warps, as a whole where there is room, else piece by piece.  16 rows x 8
// columns meet in mma.sync: at this width a product is a small part of the work, and for tcgen05 widened weights would have to go through shared or tensor memory.
//
// Lane 4 g + t of a warp holds rows g and g + 8 of the tile.  Which values of k an operand position of the MMA stands for is free as long as both operands
// agree, so a lane takes neighbours of its rows: of 4-bit integers kSpan / 4 of every kSpan, the widest span that has one scale (and one of the columns'
// scales), whose sum is multiplied by them in fp32; of 16-bit values 8 of every 32, and
// the sum over a step's 64 goes to one in fp32: the MMA cuts off what it adds up, a row of 24,000 in one accumulator was 2e-4 off.  Columns are stored in units of 8 values of k, in the order in which lanes
// t = 0..3 read them side by side, each unit as the pairs that a mask takes out of a word of eight codes: 0 4, 1 5, 2 6, 3 7.
//
// What it spends its time on is instructions, not bytes: the same copies with nothing else take 19.7 us for 28672 x 8192 codes, 120 MB.
#pragma once

#include <algorithm>
#include <type_traits>

#include "fp4_convert.cuh"
#include "warp_mma.cuh"

namespace b200spmm {
namespace narrow {

constexpr uint32_t kTileRows = 16, kStepBytes = 128;  // of a row, in a step
constexpr uint32_t kMaxSmem = 227 * 1024;
constexpr uint32_t kWholeGroup = 31;  // a shift that leaves one group, however long a row is

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

// T: the type of the MMA's operands.  kSpan: columns of 4-bit integers that share their scales, 32, 64 or 128; 0: the weights are T themselves.  kPiece: bytes of a row in a
// stage of the ring: 128 neighbouring bytes go to shared memory in one access where 64 and 64 take two; with 64 a lane of codes in spans of 128 reads what it copied itself and
// waits for nobody before it does.  (Experts in 16 bits, one token 37.4 us with 64, 36.7 with 128; in 4 bits, 8 tokens 149 and 155.)
template <typename T_, int kSpan_>
struct Weights {
    using T = T_;
    static constexpr int kSpan = kSpan_;
    static constexpr bool kCodes = kSpan > 0;
    static constexpr uint32_t kPiece = kCodes ? 64 : 128, kPieces = kStepBytes / kPiece, kStageBytes = kTileRows * kPiece;
    static constexpr uint32_t kStep = kCodes ? 2 * kStepBytes : kStepBytes / 2;  // values of k
    static constexpr uint32_t kUnits = kStep / 8;                                // of a column, in a step
    static constexpr uint32_t kBlocks = kCodes ? kStep / (kCodes ? kSpan : 1) : 2;  // of a step, with a scale each; halves
    static constexpr uint32_t kOfStage = kBlocks / kPieces;                      // blocks of a stage
    static constexpr uint32_t kWords = kCodes ? kSpan / 32 : 1;                  // of a lane in a block: units of 8 values
    static constexpr uint32_t kEntries = kCodes ? kBlocks / 2 : 1;               // scales that a lane fetches for its warp
};

// Where unit `u` (8 values of k from 8 u on) of a column lies, in bytes.
template <class W>
B200_DEVICE uint32_t unit_place(uint32_t u) {
    if constexpr (W::kCodes) {
        constexpr uint32_t n = W::kSpan / 8, words = n / 4;
        return (u / n * n + u % words * 4u + u % n / words) * 16u;
    } else {
        return u * 16u;
    }
}

// The eight 16-bit values of a unit in the order of their MMAs' operands.
template <class W>
B200_DEVICE uint4 unit_order(uint4 v) {
    if constexpr (W::kCodes)
        return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
    else
        return v;
}

// Where piece `p` of 16 bytes of row r lies in a stage: no two lanes of a load meet in a bank.
template <class W>
B200_DEVICE uint32_t stage_place(uint32_t r, uint32_t p) {
    const uint32_t swap = W::kPiece == 128 ? (r & 1u) << 2 | (r & 2u) | (r >> 2 & 1u) : (r & 2u) | (r >> 2 & 1u);
    return r * W::kPiece + (p ^ swap) * 16u;
}

// (w & mask) | bits in one instruction: with both as constants the compiler makes two of it (28672 x 8192 times one column: 38 us for 33).
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

// Eight codes less their zero, exactly: pairs 0 4, 1 5, 2 6, 3 7.  A code under the exponent of 1024 (or, four bits up, of 64 times 16; bf16: of 128) is that number and the
// code; what is added takes the number and the zero away.  (The way of Y. J. Kim et al., "Who Says Elephants Can't Run", arXiv:2211.10017, with the zero in what is added.)  Nine operations a word
// of eight for fp16: four masks, a shift, four additions; eleven for bf16.
template <typename T> struct Widen;
template <>
struct Widen<__half> {
    static constexpr uint32_t kBits = 0x64006400u;
    B200_DEVICE static uint32_t minus(uint32_t zero) { return 0xE400E400u + zero * 0x00010001u; }
    uint32_t low, high;  // -(1024 + zero), -(64 + zero), twice
    B200_DEVICE explicit Widen(uint32_t minus) : low(minus), high(minus * 16u + (0xD400D400u - 0xE400E400u * 16u)) {}
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
    static constexpr uint32_t kBits = 0x43004300u;
    B200_DEVICE static uint32_t minus(uint32_t zero) { return 0xC300C300u + zero * 0x00010001u; }
    uint32_t low;  // -(128 + zero), twice
    B200_DEVICE explicit Widen(uint32_t minus) : low(minus) {}
    B200_DEVICE void operator()(uint32_t w, uint32_t bits, uint32_t (&out)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i, w >>= 4) {
            const uint32_t a = masked<0x000F000Fu>(w, bits);
            const __nv_bfloat162 x = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&low));
            out[i] = *reinterpret_cast<const uint32_t *>(&x);
        }
    }
};

// The columns of a tile in shared memory: column j at base + j * pitch (and `plane` further on its second part, where it is the sum of two), and their scales, `groups` of each: of the
// steps that are there, which begin with a group.
struct Columns {
    uint32_t base, pitch, plane, n;
    uint32_t scales, groups, shift;
    const uint16_t *order;  // column j of a tile is order[j] / each of those in shared memory; null: j
    uint32_t each;
    B200_DEVICE uint32_t address(uint32_t j) const { return base + (order ? order[j] / each : j) * pitch; }
};

// A unit of a lane's column, by lanes that have one; the others' registers hold what they held, and so do the sums of columns that nobody looks at.  (A load
// takes four accesses with all lanes, one with those of a single column.  Registers that are written under a condition live on: the same few are used again.)
B200_DEVICE void column_unit(bool has, uint32_t addr, uint4 &v) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %5, 0;\n@q ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n}\n"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "r"(addr), "r"((uint32_t)has) : "memory");
}

template <int kBytes>
B200_DEVICE void ld_shared(uint32_t addr, uint32_t *v) {
    if constexpr (kBytes == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
    else if constexpr (kBytes == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(addr) : "memory");
}

// How a block goes through `tiles` of its own with up to `warps` warps: as many tiles at a time in every round, each cut along k as far as there are warps and steps.  More
// than one round means whole tiles.
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

// The warp's number, by an operation whose result the compiler knows to be one for all lanes: what follows from it takes no lane's registers.
B200_DEVICE uint32_t warp_index() { return __reduce_max_sync(0xFFFFFFFFu, threadIdx.x >> 5); }

// Bytes of a warp's ring, where its sums go in the end.
template <class W, int kNB, int kStages>
constexpr uint32_t kRingOf = kStages * W::kStageBytes > kNB * 512u ? kStages * W::kStageBytes : kNB * 512u;

// What a warp does: tiles first, first + at_once ... below `end` (none, where it is beyond `at_once` or `end`), of each the steps slice, slice + slices ...
struct Share {
    uint32_t first, end;
    uint32_t slice, slices, at_once, rounds;
    uint32_t steps;   // of a whole row
    uint32_t window;  // steps that the columns have room for
    uint32_t ring;    // shared memory
    B200_DEVICE Share(const Split &split, uint32_t begin, uint32_t end_, uint32_t warp, uint32_t steps_, uint32_t window_, uint32_t ring_)
        : first(begin + warp / split.slices), end(end_), slice(warp % split.slices), slices(split.slices), at_once(split.at_once), rounds(split.rounds), steps(steps_), window(window_), ring(ring_) {
        if (warp / split.slices >= split.at_once) first = end_;
    }
};

// All threads of a block come here alike.  place_of(tile) is what the others are told of a tile (a number's quotients, say, that they would all take); rows_of(place, r) row r
// (0 to 15) of it in the matrix, columns_of(place) what it is multiplied with.  stage(first step, steps) brings columns to shared memory, all of them before the first tile, or
// (window < steps) window by window in every round.  done(place, sums) gets a tile's sums in one warp: rows g (e < 2) and g + 8, columns 8 nb + 2 t + e % 2.
template <class W, int kNB, int kPlanes, bool kScaled, int kStages, class PlaceOf, class RowsOf, class ColumnsOf, class Stage, class Done>
B200_DEVICE void multiply(const Matrix &m, const Share &s, PlaceOf &&place_of, RowsOf &&rows_of, ColumnsOf &&columns_of, Stage &&stage, Done &&done) {
    using T = typename W::T;
    static_assert(kStages == W::kPieces || kStages == 2 * W::kPieces, "a ring of one step or two");
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    // Copies run kStages stages ahead.  A lane copies 16 bytes of rows r, r + 8 and, with 128 bytes of a row, r + 4, r + 12.
    constexpr uint32_t kLanes = W::kPiece / 16;  // of a row
    const uint32_t copy_row = lane / kLanes, copy_piece = lane % kLanes, own = stage_place<W>(copy_row, copy_piece), last_copy = s.steps * kStepBytes;
    uint32_t copy_tile = s.first, copied = 0, lo_4 = 0, hi_4 = 0;  // the next copy's tile, and bytes of a row up to it; from a row to the fourth after it
    const uint8_t *lo = nullptr, *hi = nullptr;
    auto copy_from = [&]() {
        copied = s.slice * kStepBytes + copy_piece * 16u;
        const auto place = place_of(copy_tile);
        const uint64_t row_lo = rows_of(place, copy_row), row_hi = rows_of(place, copy_row + 8u);
        lo = m.values + row_lo * m.pitch + copied;
        hi = m.values + row_hi * m.pitch + copied;
        if (W::kPiece == 128) {
            lo_4 = (uint32_t)((rows_of(place, copy_row + 4u) - row_lo) * m.pitch);
            hi_4 = (uint32_t)((rows_of(place, copy_row + 12u) - row_hi) * m.pitch);
        }
    };
    auto issue = [&](uint32_t at, uint32_t piece) {  // of the next step
        const uint32_t place = copied + piece * W::kPiece;
        if constexpr (W::kCodes) {
            const bool there = copy_tile < s.end && place < m.row_bytes;  // (codes behind a row's end meet zeros, whatever they are)
            ptx::cp_async_16_if(there, at + own, lo + piece * W::kPiece);
            ptx::cp_async_16_if(there, at + own + 8u * W::kPiece, hi + piece * W::kPiece);
            if (W::kPiece == 128) {  // (the place of a row's piece is another four rows further on: their lowest bit of three)
                ptx::cp_async_16_if(there, at + (own ^ 16u) + 4u * W::kPiece, lo + lo_4);
                ptx::cp_async_16_if(there, at + (own ^ 16u) + 12u * W::kPiece, hi + hi_4);
            }
        } else if (copy_tile < s.end) {  // zeros behind a row's end
            const uint32_t left = place < m.row_bytes ? min(16u, m.row_bytes - place) : 0u, back = left ? piece * W::kPiece : 0u - copied;
            ptx::cp_async_16(at + own, lo + (int32_t)back, left);
            ptx::cp_async_16(at + own + 8u * W::kPiece, hi + (int32_t)back, left);
            if (W::kPiece == 128) {
                ptx::cp_async_16(at + (own ^ 16u) + 4u * W::kPiece, lo + lo_4 + (int32_t)back, left);
                ptx::cp_async_16(at + (own ^ 16u) + 12u * W::kPiece, hi + hi_4 + (int32_t)back, left);
            }
        }
        if (piece + 1u == W::kPieces) {
            const uint32_t ahead = s.slices * kStepBytes;
            copied += ahead;
            lo += ahead;
            hi += ahead;
            if (copied >= last_copy) {
                copy_tile += s.at_once;
                if (copy_tile < s.end) copy_from();
                else copied = 0;
            }
        }
        ptx::cp_async_commit();
    };
    // Scales and zeros come by ordinary loads a step ahead, each to one lane of the four that need it: of row g (even t) or g + 8, blocks t / 2 + 2 i.
    constexpr uint32_t kEntries = W::kEntries;
    uint32_t scale_next[kEntries], zero_next[kEntries], entry_tile = s.first, entry_row = 0, entry_k = 0;
    const uint32_t entry_first = s.slice * W::kStep + (t >> 1) * (uint32_t)W::kSpan, entry_end = s.steps * W::kStep;
    auto entries_from = [&]() {
        entry_k = entry_first;
        entry_row = (uint32_t)rows_of(place_of(entry_tile), g + (t & 1u) * 8u);
    };
    auto fetch = [&]() {
        if constexpr (W::kCodes) {
#pragma unroll
            for (uint32_t i = 0; i < kEntries; ++i) {  // (behind a row's end the last one again)
                const uint32_t at = min((entry_k + 2u * i * (uint32_t)W::kSpan) >> m.shift, m.groups - 1u) * m.rows + entry_row;
                scale_next[i] = m.scales[at];
                zero_next[i] = m.zeros[at];
            }
            entry_k += s.slices * W::kStep;
            if (entry_k >= entry_end) {
                entry_tile += s.at_once;
                if (entry_tile < s.end) entries_from();
            }
        }
    };
    if (s.first < s.end) {
        copy_from();
#pragma unroll 1
        for (uint32_t i = 0; i < kStages; ++i) issue(s.ring + i * W::kStageBytes, i % W::kPieces);
        if constexpr (W::kCodes) {
            entries_from();
            fetch();
        }
    }
    const bool whole = s.window >= s.steps;
    if (whole) {
        stage(0u, s.steps);
        __syncthreads();
    }
    const uint32_t bits = W::kCodes ? in_register(Widen<T>::kBits) : 0u;
    uint32_t here = s.ring, tile = s.first;  // a step's stages
    uint4 xs[2] = {};
    float sums[kNB][4];
    for (uint32_t round = 0; round < s.rounds; ++round, tile += s.at_once) {
        const bool busy = tile < s.end;
        const Columns c = busy ? columns_of(place_of(tile)) : Columns{};
        uint32_t column[kNB];  // this lane's, for the second operand, where it has one
        bool has[kNB];
#pragma unroll
        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
            has[nb] = nb * 8u + g < c.n;
            column[nb] = (has[nb] ? c.address(nb * 8u + g) : c.base) + t * 16u;
            sums[nb][0] = sums[nb][1] = sums[nb][2] = sums[nb][3] = 0.f;
        }
        uint32_t step = s.slice;
        for (uint32_t first = 0; first < s.steps; first += s.window) {
            const uint32_t end = min(s.steps, first + s.window);
            if (!whole) {
                __syncthreads();  // (nobody reads what was there any more)
                stage(first, end - first);
                __syncthreads();
            }
            for (; busy && step < end; step += s.slices) {
                float scale[kEntries];
                uint32_t minus[kEntries];
                if constexpr (W::kCodes) {
#pragma unroll
                    for (uint32_t i = 0; i < kEntries; ++i) {
                        scale[i] = m.bf16_scales ? __uint_as_float(scale_next[i] << 16) : __half2float(__ushort_as_half((unsigned short)scale_next[i]));
                        minus[i] = Widen<T>::minus((zero_next[i] & m.zero_mask) | m.zero_else);
                    }
                    fetch();
                }
                const uint32_t x_at = (step - first) * (W::kUnits * 16u);
                float part[kNB][4];  // of a block of codes, or of a step of 16-bit weights
#pragma unroll
                for (uint32_t b = 0; b < W::kBlocks; ++b) {
                    constexpr uint32_t kRegs = W::kCodes ? W::kWords : 4u;
                    const uint32_t at = here + b / W::kOfStage * W::kStageBytes, in = b % W::kOfStage;
                    constexpr bool kOwn = W::kPiece == 64 && W::kOfStage == 1;  // a lane reads what it copied itself
                    if (in == 0u) {
                        ptx::cp_async_wait_group<kStages - 1>();
                        if (!kOwn) __syncwarp();
                    }
                    uint32_t w_lo[kRegs], w_hi[kRegs];
                    const uint32_t piece = !W::kCodes || W::kSpan == 128 ? 4u * in + t : W::kSpan == 64 ? 2u * in + (t >> 1) : in;
                    const uint32_t from = at + stage_place<W>(g, piece) + (!W::kCodes || W::kSpan == 128 ? 0u : W::kSpan == 64 ? (t & 1u) * 8u : t * 4u);
                    ld_shared<4 * kRegs>(from, w_lo);
                    ld_shared<4 * kRegs>(from + 8u * W::kPiece, w_hi);
                    if (in + 1u == W::kOfStage) {  // the stage is read: what comes kStages later may be copied there
                        __syncwarp();  // (where a lane read what it copied itself too: nothing else orders its loads before the bytes of a copy that it asks for next)
                        issue(at, b / W::kOfStage);
                        if (kStages != W::kPieces && b + 1 == W::kBlocks) here = 2u * s.ring + W::kPieces * W::kStageBytes - here;  // (the other step's)
                    }
                    if (W::kCodes || b == 0) {
#pragma unroll
                        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) part[nb][0] = part[nb][1] = part[nb][2] = part[nb][3] = 0.f;
                    }
                    if constexpr (!W::kCodes) {
#pragma unroll
                        for (int plane = 0; plane < kPlanes; ++plane)
#pragma unroll
                            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                                uint4 &x = xs[(b + nb + plane) % 2u];
                                column_unit(has[nb], column[nb] + x_at + b * 64u + plane * c.plane, x);
                                fp4::mma_16x8x16<T>(part[nb], w_lo[0], w_hi[0], w_lo[1], w_hi[1], x.x, x.y);
                                fp4::mma_16x8x16<T>(part[nb], w_lo[2], w_hi[2], w_lo[3], w_hi[3], x.z, x.w);
                            }
                        if (b + 1u == W::kBlocks) {  // (the MMA cuts off what it adds up: a row's sum is rounded here instead)
#pragma unroll
                            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                                for (uint32_t e = 0; e < 4; ++e) sums[nb][e] += part[nb][e];
                        }
                    } else {
                        const uint32_t source = (lane & ~3u) | (b & 1u) << 1;
                        const float s_lo = __shfl_sync(0xFFFFFFFFu, scale[b >> 1], source), s_hi = __shfl_sync(0xFFFFFFFFu, scale[b >> 1], source | 1u);
                        const Widen<T> widen_lo(__shfl_sync(0xFFFFFFFFu, minus[b >> 1], source)), widen_hi(__shfl_sync(0xFFFFFFFFu, minus[b >> 1], source | 1u));
#pragma unroll
                        for (uint32_t w = 0; w < W::kWords; ++w) {
                            uint32_t a_lo[4], a_hi[4];
                            widen_lo(w_lo[w], bits, a_lo);
                            widen_hi(w_hi[w], bits, a_hi);
#pragma unroll
                            for (int plane = 0; plane < kPlanes; ++plane)
#pragma unroll
                                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                                    uint4 &x = xs[(w + nb + plane) % 2u];
                                    column_unit(has[nb], column[nb] + x_at + (b * W::kWords + w) * 64u + plane * c.plane, x);
                                    fp4::mma_16x8x16<T>(part[nb], a_lo[0], a_hi[0], a_lo[1], a_hi[1], x.x, x.y);
                                    fp4::mma_16x8x16<T>(part[nb], a_lo[2], a_hi[2], a_lo[3], a_hi[3], x.z, x.w);
                                }
                        }
#pragma unroll
                        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                            float x0 = 1.f, x1 = 1.f;
                            if constexpr (kScaled) {
                                const uint32_t group = ((step - first) * W::kStep + b * (uint32_t)W::kSpan) >> c.shift, j = nb * 8u + t * 2u;
                                x0 = __uint_as_float(ptx::ld_shared_u32(c.scales + (min(j, c.n - 1u) * c.groups + group) * 4u));
                                x1 = __uint_as_float(ptx::ld_shared_u32(c.scales + (min(j + 1u, c.n - 1u) * c.groups + group) * 4u));
                            }
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) sums[nb][e] = fmaf(kScaled ? part[nb][e] * (e & 1u ? x1 : x0) : part[nb][e], e < 2 ? s_lo : s_hi, sums[nb][e]);
                        }
                    }
                }
            }
        }
        if (s.slices == 1 && busy) done(place_of(tile), sums);
    }
    if (s.slices > 1) {  // (one round) the slices' sums meet in the first one's warp, in order
        __syncwarp();
        const bool busy = s.first < s.end;
#pragma unroll
        for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
            if (busy && s.slice) ptx::st_shared_v4(s.ring + (nb * 32u + lane) * 16u, *reinterpret_cast<const uint4 *>(sums[nb]));
        __syncthreads();
        if (busy && s.slice == 0) {
            for (uint32_t z = 1; z < s.slices; ++z)
#pragma unroll
                for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb) {
                    const uint4 v = ptx::ld_shared_v4(s.ring + z * kRingOf<W, kNB, kStages> + (nb * 32u + lane) * 16u);
                    sums[nb][0] += __uint_as_float(v.x);
                    sums[nb][1] += __uint_as_float(v.y);
                    sums[nb][2] += __uint_as_float(v.z);
                    sums[nb][3] += __uint_as_float(v.w);
                }
            done(place_of(s.first), sums);
        }
    }
}

// Sources of columns: eight values of k, from 8 u on, of column j as a unit.
template <typename T>
struct Plain {  // 16-bit values `along` elements apart along k, `across` between columns
    const T *x;
    int64_t along, across;
    bool wide;  // neighbours along k, and every column starts on 16 bytes
    bool even;  // ... on 4
    uint32_t k;
    B200_DEVICE uint4 operator()(uint32_t j, uint32_t u) const {
        const T *p = x + (int64_t)j * across + (int64_t)u * 8 * along;
        const uint32_t left = u * 8u < k ? k - u * 8u : 0u;
        if (wide && left >= 8u) return *reinterpret_cast<const uint4 *>(p);
        if (even && left >= 8u) {
            const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
            return make_uint4(q[0], q[1], q[2], q[3]);
        }
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
        uint32_t v[2] = {0u, 0u};
        if (wide && left >= 8u) {
            const uint2 both = *reinterpret_cast<const uint2 *>(p);
            v[0] = both.x;
            v[1] = both.y;
        } else {
#pragma unroll 1
            for (uint32_t e = 0; e < 8u; ++e) {
                v[0] = v[0] >> 8 | v[1] << 24;
                v[1] = v[1] >> 8 | (e < left ? (uint32_t)p[e] : 0u) << 24;
            }
        }
        uint32_t h[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[e]) : "h"((uint16_t)(v[e / 2] >> e % 2 * 16)));
        return make_uint4(h[0], h[1], h[2], h[3]);
    }
};

// `count` steps of n columns from step `first` on to shared memory, by all threads.  A warp takes 32 neighbouring units of a column, or, where neighbours lie across
// the columns, up to 32 columns of a unit.
template <class W, class Source>
B200_DEVICE void stage_columns(const Source &from, uint32_t base, uint32_t pitch, uint32_t first, uint32_t count, uint32_t n, bool across) {
    const uint32_t units = count * W::kUnits, u0 = first * W::kUnits, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31u;
    auto put = [&](uint32_t j, uint32_t u, uint4 v) { ptx::st_shared_v4(base + j * pitch + unit_place<W>(u), unit_order<W>(v)); };
    if (across) {
        for (uint32_t u = warp; u < units; u += warps)
            for (uint32_t j = lane; j < n; j += 32u) put(j, u, from(j, u0 + u));
        return;
    }
    // pieces of 32 units, all columns of one after the other, four at a time
    constexpr uint32_t kBatch = 4;
    uint32_t j = 0, u = warp * 32u + lane, js[kBatch], us[kBatch];
    uint4 v[kBatch];
    auto ask = [&]() {
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
    };
    ask();
    while (true) {
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b)
            if (js[b] < n) put(js[b], us[b], v[b]);
        if (js[kBatch - 1] >= n) return;
        ask();
    }
}

// Bytes between columns with room for `steps`: lanes of two neighbouring columns read from different halves of 128 bytes.
template <class W>
__host__ __device__ constexpr uint32_t column_pitch(uint32_t steps) { return (steps * W::kUnits * 16u + 127u) / 128u * 128u + 64u; }

}  // namespace narrow
}  // namespace b200spmm
