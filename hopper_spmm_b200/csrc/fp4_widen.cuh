// What the two kernels for 16-bit operands share: their parameters, and the way from 4 bits to 16.
#pragma once

#include "fp4_store.cuh"

namespace b200spmm {
namespace fp4 {

struct DenseParams {
    const uint8_t *values, *scales;
    const float *whole;
    uint32_t m, k, pitch, groups;
    const uint8_t *b;  // 16-bit
    int64_t ldb;       // elements
    uint32_t n;
    bool b_wide;       // B's rows (as they lie) start on 16 bytes
    Target c;
};

template <typename T> B200_DEVICE uint32_t mul2(uint32_t a, uint32_t b);
template <> B200_DEVICE uint32_t mul2<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <> B200_DEVICE uint32_t mul2<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Codes are widened by placing their bits as the sign, the low exponent bits and the top mantissa bit of the 16-bit type: 2^-14 (fp16)
// or 2^-126 (bf16) of their value, subnormal ones included.  The multiplication with the block's scale takes most of that back; what is
// left of it, a power of two, waits for the end of the sum.
//   fp16, nvfp4: scale * 2^7, the product 2^-7 of its value: 21 at most, and at least 2^-17 with all its bits
//   bf16, nvfp4: scale * 2^118, the product 2^-8 of its value
//   bf16, mxfp4: 2^126, then the scale: the range is the whole of bf16's
template <typename T, bool kMx> struct Widen;
template <> struct Widen<__half, false> {
    static constexpr float kLeft = 128.f;
    B200_DEVICE static uint32_t scale(uint32_t byte) {  // of a block, twice
        uint32_t r;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(byte | byte << 8)));
        return mul2<__half>(r, 0x58005800u);  // 2^7
    }
    template <int kShift> B200_DEVICE static uint32_t pair(uint32_t w, uint32_t s) {
        const uint32_t x = w << kShift;  // (two codes at the top of the halves)
        return mul2<__half>((x & 0x80008000u) | (x >> 3 & 0x0E000E00u), s);
    }
};
template <> struct Widen<__nv_bfloat16, false> {
    static constexpr float kLeft = 256.f;
    B200_DEVICE static uint32_t scale(uint32_t byte) {
        const float f = from_e4m3(byte) * 0x1p118f;
        return (__float_as_uint(f) >> 16) * 0x10001u;  // (exact: four bits, or NaN)
    }
    template <int kShift> B200_DEVICE static uint32_t pair(uint32_t w, uint32_t s) {
        const uint32_t x = w << kShift;
        return mul2<__nv_bfloat16>((x & 0x80008000u) | (x >> 6 & 0x01C001C0u), s);
    }
};
template <> struct Widen<__nv_bfloat16, true> {
    static constexpr float kLeft = 1.f;
    B200_DEVICE static uint32_t scale(uint32_t byte) { return (__float_as_uint(from_e8m0(byte)) >> 16) * 0x10001u; }
    template <int kShift> B200_DEVICE static uint32_t pair(uint32_t w, uint32_t s) {
        const uint32_t x = w << kShift;
        return mul2<__nv_bfloat16>(mul2<__nv_bfloat16>((x & 0x80008000u) | (x >> 6 & 0x01C001C0u), 0x7E807E80u), s);
    }
};

}  // namespace fp4
}  // namespace b200spmm
