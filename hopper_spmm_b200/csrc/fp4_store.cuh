// From accumulators to C: the tensors' scales, the element type, either order of C.
#pragma once

#include "fp4.hpp"
#include "fp4_convert.cuh"

namespace b200spmm {
namespace fp4 {

// The product of two tensors' scales, applied in steps none of which leaves fp32's range unless the result does: the mantissa (1 for
// powers of two), then both halves of the exponent.
struct Factor {
    float mantissa, half0, half1;
    B200_DEVICE Factor(float a, float b) {
        const double ab = (double)a * (double)b;
        const int64_t bits = __double_as_longlong(ab);
        const int e = (int)(bits >> 52 & 0x7FF) - 1023;  // (a product of two fp32 numbers is never subnormal in 64 bits)
        if (e == 1024 || e == -1023) {  // NaN, infinity or zero
            mantissa = (float)ab;
            half0 = half1 = 1.f;
            return;
        }
        mantissa = (float)__longlong_as_double((bits & ~(0x7FFll << 52)) | (1023ll << 52));
        const int e0 = e / 2, e1 = e - e0;
        half0 = ldexpf(1.f, e0);
        half1 = ldexpf(1.f, e1);
    }
    B200_DEVICE float apply(float v) const { return v * mantissa * half0 * half1; }
};

struct Target {
    uint8_t *ptr;
    int64_t ldc;  // elements
    int type;     // B200SPMM_T_*
    bool transposed;  // element (row, col) at [col * ldc + row]
    bool wide;    // rows start on 16 bytes
};

inline Target target_of(void *c, int64_t ldc, int type, bool transposed) {
    const int64_t esz = type == B200SPMM_T_F32 ? 4 : 2;
    return {static_cast<uint8_t *>(c), ldc, type, transposed, reinterpret_cast<uintptr_t>(c) % 16u == 0 && ldc * esz % 16 == 0};
}

template <typename T, int N>
B200_DEVICE void store_row_as(const Target &c, uint32_t row, uint32_t col, uint32_t n, const float (&v)[N]) {
    T *out = reinterpret_cast<T *>(c.ptr);
    if (c.transposed) {  // lanes hold neighbouring rows: every store is one run
        T *dst = out + (int64_t)col * c.ldc + row;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < n) dst[(int64_t)i * c.ldc] = Elem<T>::from_float(v[i]);
        return;
    }
    T *dst = out + (int64_t)row * c.ldc + col;
    constexpr int kPer = 16 / sizeof(T);
    if (N % kPer == 0 && c.wide && n - col >= (uint32_t)N) {
#pragma unroll
        for (int i = 0; i < N / kPer; ++i) {
            uint4 four;
            T *e = reinterpret_cast<T *>(&four);
#pragma unroll
            for (int j = 0; j < kPer; ++j) e[j] = Elem<T>::from_float(v[i * kPer + j]);
            reinterpret_cast<uint4 *>(dst)[i] = four;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < n) dst[i] = Elem<T>::from_float(v[i]);
    }
}

// N neighbours of a row, from column `col` (a multiple of N) on; those at `n` and behind do not exist.
template <int N>
B200_DEVICE void store_row(const Target &c, uint32_t row, uint32_t col, uint32_t n, const float (&v)[N]) {
    if (c.type == B200SPMM_T_F32) store_row_as<float>(c, row, col, n, v);
    else if (c.type == B200SPMM_T_F16) store_row_as<__half>(c, row, col, n, v);
    else store_row_as<__nv_bfloat16>(c, row, col, n, v);
}

// The same in two steps, for sums that have to leave their place before they are written: 16 of them as 16-bit numbers, and 32 of those to C.
B200_DEVICE void pack_row(int type, const float (&v)[16], uint32_t *out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (type == B200SPMM_T_F16) {
            const __half2 two = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            out[i] = *reinterpret_cast<const uint32_t *>(&two);
        } else {
            const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            out[i] = *reinterpret_cast<const uint32_t *>(&two);
        }
    }
}
// 32 16-bit numbers of a row as 16 words, to a C that lies column by column: lanes hold neighbouring rows.
B200_DEVICE void store_packed_column(const Target &c, uint32_t row, uint32_t col, uint32_t n, const uint32_t (&v)[16]) {
    uint16_t *dst = reinterpret_cast<uint16_t *>(c.ptr) + (int64_t)col * c.ldc + row;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (col + i < n) dst[(int64_t)i * c.ldc] = (uint16_t)(v[i / 2] >> (i & 1) * 16);
}
// 16 words of each lane, transposed between the 16 lanes of either half of the warp: word i of lane l goes to word l % 16 of lane i (of its half).
B200_DEVICE void transpose_16(uint32_t (&v)[16], uint32_t lane) {
#pragma unroll
    for (uint32_t d = 1; d < 16; d <<= 1)
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)
            if (!(i & d)) {
                const bool upper = (lane & d) != 0;
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, upper ? v[i] : v[i | d], d);
                if (upper) v[i] = got;
                else v[i | d] = got;
            }
}
// A warp's 32 rows of C from `row0` on, 16 words of each (32 16-bit numbers, or 16 fp32 ones) from column `col` on; words[] is lost.  Row by
// row the words change places first, so that 16 lanes write 64 neighbouring bytes of a row.  All lanes take part.
B200_DEVICE void store_words(const Target &c, uint32_t row0, uint32_t rows, uint32_t col, uint32_t n, uint32_t (&v)[16]) {
    const uint32_t lane = threadIdx.x & 31u;
    const bool half = c.type != B200SPMM_T_F32;
    if (c.transposed) {  // lanes hold neighbouring rows
        const uint32_t row = row0 + lane;
        if (row >= rows) return;
        if (half) {
            store_packed_column(c, row, col, n, v);
        } else {
            uint32_t *dst = reinterpret_cast<uint32_t *>(c.ptr) + (int64_t)col * c.ldc + row;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (col + i < n) dst[(int64_t)i * c.ldc] = v[i];
        }
        return;
    }
    transpose_16(v, lane);
    const uint32_t first = row0 + (lane & 16u), at = col + (lane & 15u) * (half ? 2u : 1u);
    if (half) {
        uint16_t *dst = reinterpret_cast<uint16_t *>(c.ptr) + (int64_t)first * c.ldc + at;
        const bool pairs = reinterpret_cast<uintptr_t>(c.ptr) % 4u == 0 && c.ldc % 2 == 0;  // (columns come in pairs, too)
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i, dst += c.ldc) {
            if (first + i >= rows) break;
            if (pairs && at + 1u < n) {
                *reinterpret_cast<uint32_t *>(dst) = v[i];
            } else {
                if (at < n) dst[0] = (uint16_t)v[i];
                if (at + 1u < n) dst[1] = (uint16_t)(v[i] >> 16);
            }
        }
    } else {
        uint32_t *dst = reinterpret_cast<uint32_t *>(c.ptr) + (int64_t)first * c.ldc + at;
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i, dst += c.ldc)
            if (first + i < rows && at < n) *dst = v[i];
    }
}

}  // namespace fp4
}  // namespace b200spmm
