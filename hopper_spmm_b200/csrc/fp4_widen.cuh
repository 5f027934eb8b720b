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

// From codes to 16 bits, all exact.  What is left of a power of two waits for the end of the sum (kLeft).
//   fp16, nvfp4: the conversion's own instruction, two neighbouring codes at a time, times the scale (2,688 at most, 2^-10 at least)
//   bf16: the code's bits become the sign, the low exponent bits and the top mantissa bit of a bf16 number, 2^-126 of its value (subnormal
//   ones included), by a multiplication that puts them in both places and a mask; two codes that are four apart in their word at a time.
//     nvfp4: times scale * 2^118, which leaves 2^-8
//     mxfp4: times scale * 2^126, for scales up to 2.  Larger ones (kTwice) take two multiplications, as does NaN: the range is the
//     whole of bf16's.
// (Shifts, masks, byte moves and conversions run at 64 lanes a clock and SM, multiplications of either kind at another 64; with shifts
// and masks alone for fp16, too, widening took 23 operations for eight values, here 8 and 17.)
template <typename T, bool kMx> struct Widen {
    static_assert(!kMx || std::is_same<T, __nv_bfloat16>::value, "the scales of mxfp4 go beyond fp16");
    static constexpr bool kHalf = std::is_same<T, __half>::value;
    static constexpr float kLeft = kMx || kHalf ? 1.f : 256.f;
    static constexpr bool kNeighbours = kHalf;  // pair i of a word: codes 2 i and 2 i + 1, else i and i + 4
    // Whether one of a word's four scales is larger than 2, a byte of 129 or more.
    B200_DEVICE static bool needs_two(uint32_t four) { return kMx && __vcmpgtu4(four, 0x80808080u) != 0u; }
    // The scale `byte` twice.
    template <bool kTwice> B200_DEVICE static uint32_t scale(uint32_t byte) {
        if constexpr (kMx) {
            return kTwice ? (__float_as_uint(from_e8m0(byte)) >> 16) * 0x10001u : (byte + 126u) * 0x00800080u;
        } else if constexpr (std::is_same<T, __half>::value) {
            uint32_t r;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(byte | byte << 8)));
            return r;
        } else {
            return (__float_as_uint(from_e4m3(byte) * 0x1p118f) >> 16) * 0x10001u;  // (exact: four bits, or NaN)
        }
    }
    // The scales in the two low bytes of `word`.
    B200_DEVICE static void two_scales(uint32_t word, uint32_t (&out)[2]) {
        if constexpr (kHalf) {
            uint32_t r;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)word));
            out[0] = __byte_perm(r, r, 0x1010);
            out[1] = __byte_perm(r, r, 0x3232);
        } else {
            out[0] = scale<false>(word & 0xFFu);
            out[1] = scale<false>(word >> 8 & 0xFFu);
        }
    }
    // The four pairs of a word.
    template <bool kTwice> B200_DEVICE static void pairs(uint32_t w, uint32_t s, uint32_t (&out)[4]) {
        if constexpr (kHalf) {
            asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
                "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\ncvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}\n"
                : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3]) : "r"(w));
        } else {
            const uint32_t v = w >> 8;
            out[0] = (w & 0x000F000Fu) * 0x1040u & 0x81C081C0u;  // bits 3..0 to 15..12 and 9..6
            out[1] = (w & 0x00F000F0u) * 0x0104u & 0x81C081C0u;
            out[2] = (v & 0x000F000Fu) * 0x1040u & 0x81C081C0u;
            out[3] = (v & 0x00F000F0u) * 0x0104u & 0x81C081C0u;
            if constexpr (kTwice && kMx) {
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = mul2<T>(out[i], 0x7E807E80u);  // 2^126
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = mul2<T>(out[i], s);
    }
    // ... in the order of the codes.
    template <bool kTwice> B200_DEVICE static void eight(uint32_t w, uint32_t s, uint32_t *out) {
        uint32_t p[4];
        pairs<kTwice>(w, s, p);
        out[0] = kNeighbours ? p[0] : __byte_perm(p[0], p[1], 0x5410);  // (0, 4) and (1, 5) to (0, 1) and (4, 5)
        out[1] = kNeighbours ? p[1] : __byte_perm(p[2], p[3], 0x5410);
        out[2] = kNeighbours ? p[2] : __byte_perm(p[0], p[1], 0x7632);
        out[3] = kNeighbours ? p[3] : __byte_perm(p[2], p[3], 0x7632);
    }
};

// What a sum still lacks: the power of two that Widen left, 1 at least, and the tensor's scale.  In this order no step leaves fp32's range unless
// the result does.
struct LeftOver {
    float first, second;
    B200_DEVICE LeftOver(float left, float whole) : first(whole < 1.f ? whole * left : left), second(whole < 1.f ? 1.f : whole) {}
    B200_DEVICE float apply(float v) const { return v * first * second; }
};

}  // namespace fp4
}  // namespace b200spmm
