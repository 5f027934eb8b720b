// What the two kernels for 16-bit operands share: their parameters, and the way from 4 bits to 16.
#pragma once

#include <type_traits>

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
//   bf16, mxfp4: scale * 2^126, for scales up to 2.  Larger ones (kTwice) take two multiplications, as does NaN: the range is the whole of
//   bf16's.
// Two codes that are four apart in a word are widened together, by a shift and two masks; eight are then put in order.
template <typename T, int kShift>
B200_DEVICE uint32_t place(uint32_t w) {
    const uint32_t x = w << kShift;  // (the codes at the top of the halves)
    if constexpr (std::is_same<T, __half>::value) return (x & 0x80008000u) | (x >> 3 & 0x0E000E00u);
    else return (x & 0x80008000u) | (x >> 6 & 0x01C001C0u);
}

template <typename T, bool kMx> struct Widen {
    static_assert(!kMx || std::is_same<T, __nv_bfloat16>::value, "the scales of mxfp4 go beyond fp16");
    static constexpr float kLeft = kMx ? 1.f : std::is_same<T, __half>::value ? 128.f : 256.f;
    // Whether one of a word's four scales is larger than 2, a byte of 129 or more.
    B200_DEVICE static bool needs_two(uint32_t four) { return kMx && __vcmpgtu4(four, 0x80808080u) != 0u; }
    // The scale `byte` twice.
    template <bool kTwice> B200_DEVICE static uint32_t scale(uint32_t byte) {
        if constexpr (kMx) {
            return kTwice ? (__float_as_uint(from_e8m0(byte)) >> 16) * 0x10001u : (byte + 126u) * 0x00800080u;
        } else if constexpr (std::is_same<T, __half>::value) {
            uint32_t r;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(byte | byte << 8)));
            return mul2<__half>(r, 0x58005800u);  // 2^7
        } else {
            return (__float_as_uint(from_e4m3(byte) * 0x1p118f) >> 16) * 0x10001u;  // (exact: four bits, or NaN)
        }
    }
    // Codes kAt and kAt + 4 of a word.
    template <bool kTwice, int kAt> B200_DEVICE static uint32_t pair(uint32_t w, uint32_t s) {
        uint32_t x = place<T, 12 - 4 * kAt>(w);
        if constexpr (kTwice && kMx) x = mul2<T>(x, 0x7E807E80u);  // 2^126
        return mul2<T>(x, s);
    }
    template <bool kTwice> B200_DEVICE static void eight(uint32_t w, uint32_t s, uint32_t *out) {
        const uint32_t p0 = pair<kTwice, 0>(w, s), p1 = pair<kTwice, 1>(w, s), p2 = pair<kTwice, 2>(w, s), p3 = pair<kTwice, 3>(w, s);
        out[0] = __byte_perm(p0, p1, 0x5410);  // (0, 4) and (1, 5) to (0, 1) and (4, 5)
        out[1] = __byte_perm(p2, p3, 0x5410);
        out[2] = __byte_perm(p0, p1, 0x7632);
        out[3] = __byte_perm(p2, p3, 0x7632);
    }
};

}  // namespace fp4
}  // namespace b200spmm
