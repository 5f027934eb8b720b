// Conversions between fp32 and the few-bit types of 4-bit matrices, one element or block at a time.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx_sm100.cuh"

namespace b200spmm {
namespace fp4 {

// Eight values to eight e2m1 codes, the first in the lowest bits; ties to even, at most 6.
B200_DEVICE uint32_t to_e2m1x8(const float *v) {
    uint32_t r;
    asm("{\n.reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n}\n"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Two of them back, from the low byte of `byte`: the first in the low half.
B200_DEVICE __half2 from_e2m1x2(uint32_t byte) {
    uint32_t r;
    asm("{\n.reg .b8 b, x, y, z;\nmov.b32 {b, x, y, z}, %1;\ncvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(r) : "r"(byte));
    return *reinterpret_cast<__half2 *>(&r);
}

// The nearest e4m3 number (ties to even, at most 448) to v >= 0.
B200_DEVICE uint32_t to_e4m3(float v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
    return r & 0xFFu;
}
B200_DEVICE float from_e4m3(uint32_t byte) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(byte & 0xFFu)));
    return __half2float(__ushort_as_half((unsigned short)(r & 0xFFFFu)));
}
// 2^(byte - 127); 255 is NaN.
B200_DEVICE float from_e8m0(uint32_t byte) {
    return __uint_as_float(byte == 0xFFu ? 0x7FFFFFFFu : byte == 0u ? 0x00400000u : byte << 23);
}

constexpr uint32_t kInfBits = 0x7F800000u;

// 2^k for k in [-126, 127].
B200_DEVICE float exp2_int(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// The exponent of a tensor's scale: the smallest k for which its largest block's scale, amax / 6 / 2^k, is at most 448, that is
// ceil(log2(amax / 2688)), 2688 = 1.3125 * 2^11; 0 for a tensor of zeros.
B200_DEVICE int tensor_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax) & 0x7FFFFFFFu;
    if (bits == 0u) return 0;
    const int k = (int)(bits >> 23) - 127 - 11 + ((bits & 0x7FFFFFu) > 0x280000u ? 1 : 0);
    return max(-126, min(127, k));  // (a subnormal amax ends at -126 either way)
}
// The exponent of a given scale, rounded up to a power of two.
B200_DEVICE int exponent_above(float scale) {
    const uint32_t bits = __float_as_uint(scale) & 0x7FFFFFFFu;
    const int k = (int)(bits >> 23) - 127 + ((bits & 0x7FFFFFu) ? 1 : 0);
    return max(-126, min(127, k));
}

// One block of an nvfp4 matrix: scale byte and codes of 16 values whose largest magnitude has the bits `top`.
//
// scale = e4m3(amax / 6 / 2^k), codes e2m1(x / scale / 2^k).  Both quotients have to be rounded as real numbers are, or values next
// to a border between two codes - many, where x has few digits - would fall on the wrong side.  A rounded fp32 quotient does that:
// the borders have at most seven bits after multiplication by the divisor, so an fp32 dividend that is not on one is far enough from
// it for its rounded quotient not to be on one either.  x / (scale 2^k) is rounded by Markstein's method (multiply by the rounded
// reciprocal, add the remainder times it), three operations for an element instead of a division.  The remainder is exact; it is
// rounded down only so that it is -0 where it vanishes, which leaves the quotient of -0 its sign.
//
// The rounded reciprocal of an e4m3 number: one step of Newton's method from the hardware's approximation leaves an error of some 2^-46,
// and the reciprocals of 8 ... 15, times powers of two, are no nearer than 2^-29 to the middle between two fp32 numbers.
B200_DEVICE float reciprocal_e4m3(float s) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return __fmaf_rn(r, __fmaf_rn(-s, r, 1.f), r);
}
struct TensorScale {
    float up, down;  // 2^k, 2^-k
    bool plain;      // neither block scales nor their reciprocals leave fp32's normal range with it
    B200_DEVICE explicit TensorScale(int k) {
        up = exp2_int(k);
        down = k == 127 ? __uint_as_float(0x00400000u) : exp2_int(-k);
        plain = k > -100 && k < 100;
    }
};
B200_DEVICE uint32_t quantize_block_nv(const float (&v)[16], uint32_t top, const TensorScale &tensor, uint2 &codes) {
    if (top >= kInfBits) {  // infinity or NaN: the block is NaN
        codes = make_uint2(0u, 0u);
        return 0x7Fu;
    }
    const float amax = __uint_as_float(top), scaled = fminf(amax * tensor.down, 1e30f);
    const float sixth = scaled * (1.f / 6.f);
    const uint32_t byte = to_e4m3(__fmaf_rn(__fmaf_rd(sixth, -6.f, scaled), 1.f / 6.f, sixth));
    const float s = from_e4m3(byte);
    const float r = byte ? reciprocal_e4m3(s) : 0.f;
    float q[16];
    if (tensor.plain && scaled < 1e30f) {
        const float rs = r * tensor.down, ss = -s * tensor.up;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float q0 = v[i] * rs;
            q[i] = __fmaf_rn(__fmaf_rd(q0, ss, v[i]), rs, q0);
        }
    } else {
        // 2^-k first, which changes no digits of what matters; a given tensor scale far too small leaves numbers that are all beyond 6
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = fminf(fmaxf(v[i] * tensor.down, -1e30f), 1e30f), q0 = x * r;
            q[i] = __fmaf_rn(__fmaf_rd(q0, -s, x), r, q0);
        }
    }
    codes = make_uint2(to_e2m1x8(q), to_e2m1x8(q + 8));
    return byte;
}

// The scale byte of a block of an mxfp4 matrix, 2^(floor(log2(amax)) - 2), and what its values are multiplied with: exactly, but
// for values far below the smallest code.
B200_DEVICE uint32_t block_scale_mx(uint32_t top, float &factor) {
    if (top >= kInfBits) {
        factor = 0.f;
        return 0xFFu;
    }
    const uint32_t e = top >> 23, byte = e > 2u ? e - 2u : 0u;
    factor = __uint_as_float((254u - byte) << 23);
    return byte;
}

// Where the four scales `group` of row `row` lie.
B200_DEVICE uint64_t scale_word(uint32_t row, uint32_t group, uint32_t groups) {
    return ((uint64_t)(row >> 7) * groups + group) * 512u + (row & 31u) * 16u + ((row >> 5) & 3u) * 4u;
}

template <typename T> struct Elem;
template <> struct Elem<float> {
    B200_DEVICE static float to_float(float v) { return v; }
    B200_DEVICE static float from_float(float v) { return v; }
};
template <> struct Elem<__half> {
    B200_DEVICE static float to_float(__half v) { return __half2float(v); }
    B200_DEVICE static __half from_float(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
    B200_DEVICE static float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    B200_DEVICE static __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};

}  // namespace fp4
}  // namespace b200spmm
