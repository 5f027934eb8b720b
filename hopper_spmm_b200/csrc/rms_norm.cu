// The residual's addition, the RMS norm and the rounding to few bits in one pass over a row.
//
//     h = x + r,  y = (h w) / sqrt(mean(h^2) + eps),  scale = max |y| / 448,  value = y / scale
//
// Bound: HBM; for a few rows the latency of one read, one reduction and one write.  A row stays in registers, eight neighbours a thread and up to four times
// that, while its sum of squares and, for a scale of the whole row, its max |h w| are reduced together: y is the product of h w with one positive number,
// so the largest |y| is the largest |h w| times it, and one reduction serves both.  Scales of groups of 32, 64 and 128 come from 4, 8 or 16 neighbouring lanes.
// Rows longer than a block's registers (32,768 columns) are read a second time.
//
// 8192 x 8192 bf16 with a bf16 residual, to e4m3 with scales of 128: 81 us, 5.8 TB/s, 89 % of a copy's rate (104 before kernels were made for the weight's and the
// result's type, 170 before all loads of a row came before the first use of one).  5001 x 4090, whose rows start on 4 bytes, with an fp32 residual and scales of 32: 60 us, 3.8 TB/s, issue: two
// values an access, and a scale's arithmetic for each two of a lane.  8 x 8192: 3.0 us in a captured loop, a launch and one reduction (a call from
// Python takes the host 5 us or more).
#include <type_traits>

#include "entry.hpp"
#include "fp4_convert.cuh"
#include "launch.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

constexpr float kTop = 448.f;  // the largest number of e4m3
constexpr uint32_t kPer = 8;   // values of a row that a thread has at a time, so that a warp has 256 neighbours
constexpr uint32_t kSpan = 32 * kPer;
constexpr uint32_t kTiny = 0x0D800000u;  // the bits of 2^-100

struct NormParams {
    const void *x, *r, *w;
    void *sum, *out;
    float *scales;
    int64_t ldx, ldr, lds, ldo;
    uint64_t rows;
    uint32_t cols, groups;
    int w_type, out_type;
    uint32_t group, group_shift;  // columns that share a scale, a power of two; 0: the row does
    float eps;
};

// What a kernel is made for: any weight and result, or a weight of X's type and e4m3 with a scale of the row, of groups, or a result of X's type.  (Asked while it runs, that
// takes 26 branches for 8 values.)
enum : int { kAny, kRow, kGroups, kSame };

template <int kBytes> struct Access;
template <> struct Access<1> { using Type = uint8_t; };
template <> struct Access<2> { using Type = uint16_t; };
template <> struct Access<4> { using Type = uint32_t; };
template <> struct Access<8> { using Type = uint2; };
template <> struct Access<16> { using Type = uint4; };
template <> struct Access<32> { using Type = uint4; };  // two of them

// kE neighbours of T at once, where `on`; else zeros.
template <typename T, int kE>
struct Raw {
    using U = typename Access<kE * sizeof(T)>::Type;
    static constexpr int kN = kE * sizeof(T) / sizeof(U);
    U u[kN];
    B200_DEVICE void load(const T *p, bool on) {
#pragma unroll
        for (int i = 0; i < kN; ++i) u[i] = on ? reinterpret_cast<const U *>(p)[i] : U{};
    }
    B200_DEVICE void store(T *p) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) reinterpret_cast<U *>(p)[i] = u[i];
    }
    B200_DEVICE float operator[](int i) const { return Elem<T>::to_float(reinterpret_cast<const T *>(u)[i]); }
    B200_DEVICE void set(int i, T v) { reinterpret_cast<T *>(u)[i] = v; }
};

template <typename T, int kE>
B200_DEVICE void store_as(void *p, int64_t at, const float *v) {
    Raw<T, kE> raw;
#pragma unroll
    for (int i = 0; i < kE; ++i) raw.set(i, Elem<T>::from_float(v[i]));
    raw.store(static_cast<T *>(p) + at);
}

// v[j * kE + e] *= w[column of it]
template <typename T, int kE>
B200_DEVICE void times_weight_as(const void *w, uint32_t cols, uint32_t col, float (&v)[kPer]) {
    Raw<T, kE> raw[kPer / kE];
#pragma unroll
    for (uint32_t j = 0; j < kPer / kE; ++j) raw[j].load(static_cast<const T *>(w) + col + j * 32u * kE, col + j * 32u * kE < cols);
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) v[i] *= raw[i / kE][i % kE];
}
template <typename X, int kE, int kKind>
B200_DEVICE void times_weight(const NormParams &p, uint32_t col, float (&v)[kPer]) {
    if constexpr (kKind != kAny) return times_weight_as<X, kE>(p.w, p.cols, col, v);
    if (!p.w) return;
    if (p.w_type == B200SPMM_T_F32) times_weight_as<float, kE>(p.w, p.cols, col, v);
    else if (p.w_type == B200SPMM_T_F16) times_weight_as<__half, kE>(p.w, p.cols, col, v);
    else times_weight_as<__nv_bfloat16, kE>(p.w, p.cols, col, v);
}

// The row's sum and its largest bits, in every thread that has part of it: a warp, or the block.
struct Both {
    float sum;
    uint32_t top;  // of |.|, as bits: NaN is above infinity
};
B200_DEVICE Both reduce(Both b, bool whole_block, Both *shared) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        b.sum += __shfl_xor_sync(0xFFFFFFFFu, b.sum, d);
        b.top = max(b.top, __shfl_xor_sync(0xFFFFFFFFu, b.top, d));
    }
    if (!whole_block) return b;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, warps = blockDim.x >> 5;
    __syncthreads();  // (what is there may still be read)
    if (lane == 0) shared[warp] = b;
    __syncthreads();
    b = lane < warps ? shared[lane] : Both{0.f, 0u};
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        b.sum += __shfl_xor_sync(0xFFFFFFFFu, b.sum, d);
        b.top = max(b.top, __shfl_xor_sync(0xFFFFFFFFu, b.top, d));
    }
    return b;
}

// Two products in one instruction.
B200_DEVICE void times_two(float &a, float &b, float by) {
    asm("{\n.reg .b64 v, w;\nmov.b64 v, {%0, %1};\nmov.b64 w, {%2, %2};\nmul.rn.f32x2 v, v, w;\nmov.b64 {%0, %1}, v;\n}\n" : "+f"(a), "+f"(b) : "f"(by));
}

B200_DEVICE uint32_t bits_of(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// R: the residual's type, void for none.  kV: times eight values of a row that a thread keeps; 0: none, the row is read again.  kE: neighbours that are read
// and written at once, on whose size all rows start and end; lane l's are kE from kE l on in each 32 kE columns.
template <typename X, typename R, int kV, int kE, int kKind>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormParams p) {
    constexpr bool kKeep = kV > 0, kAdds = !std::is_void<R>::value;
    constexpr int kKept = kKeep ? kV : 1;
    constexpr uint32_t kJ = kPer / kE;
    using RT = std::conditional_t<kAdds, R, float>;
    __shared__ Both shared[32];
    ptx::wait_for_grids_before();
    const bool whole_block = blockDim.y == 1;  // else each warp has a row
    const uint64_t row = (uint64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // (a warp as a whole)
    const uint32_t lane = threadIdx.x & 31u, first = (threadIdx.x >> 5) * kSpan + lane * kE, step = blockDim.x * kPer;
    const X *x = static_cast<const X *>(p.x) + (int64_t)row * p.ldx;
    const RT *r = kAdds ? static_cast<const RT *>(p.r) + (int64_t)row * p.ldr : nullptr;
    // Raw values of all that a thread keeps are asked for before the first is used.
    auto load = [&](uint32_t col, float (&h)[kKept][kPer]) {
        Raw<X, kE> a[kKept][kJ];
        Raw<RT, kE> b[kKept][kJ];
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)kKept; ++i)
#pragma unroll
            for (uint32_t j = 0; j < kJ; ++j) {
                const uint32_t at = col + i * step + j * 32u * kE;
                a[i][j].load(x + at, at < p.cols);
                if constexpr (kAdds) b[i][j].load(r + at, at < p.cols);
            }
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)kKept; ++i)
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) {
                h[i][e] = a[i][e / kE][e % kE];
                if constexpr (kAdds) h[i][e] += b[i][e / kE][e % kE];
            }
    };
    float h[kKept][kPer], down = 1.f;  // h times `down`, a power of two
    auto each = [&](auto &&fn) {  // fn(first column, values) for all that this thread has
        if constexpr (kKeep) {
#pragma unroll
            for (uint32_t i = 0; i < (uint32_t)kV; ++i) fn(first + i * step, h[i]);
        } else {
            for (uint32_t at = 0; at < p.cols; at += step) {  // (every lane as often: groups are reduced inside)
                load(at + first, h);
#pragma unroll
                for (uint32_t e = 0; e < kPer; ++e) h[0][e] *= down;
                fn(at + first, h[0]);
            }
        }
    };
    if constexpr (kKeep) load(first, h);
    const bool eights = kKind == kAny ? p.out_type == B200SPMM_T_E4M3 : kKind != kSame, of_row = kKind == kAny ? eights && p.group == 0 : kKind == kRow;
    auto sums = [&]() {
        Both b{0.f, 0u};
        each([&](uint32_t col, float (&v)[kPer]) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) b.sum = fmaf(v[e], v[e], b.sum);
            if (of_row) {
                float y[kPer];
#pragma unroll
                for (uint32_t e = 0; e < kPer; ++e) y[e] = v[e];
                times_weight<X, kE, kKind>(p, col, y);
#pragma unroll
                for (uint32_t e = 0; e < kPer; ++e) b.top = max(b.top, bits_of(y[e]));
            }
        });
        return reduce(b, whole_block, shared);
    };
    // the sum is kept before anything is scaled
    auto keep_sum = [&](uint32_t col, const float (&v)[kPer]) {
        if constexpr (kAdds) {
            if (p.sum)
#pragma unroll
                for (uint32_t j = 0; j < kJ; ++j)
                    if (col + j * 32u * kE < p.cols) store_as<RT, kE>(p.sum, (int64_t)row * p.lds + col + j * 32u * kE, v + j * kE);
        }
    };
    if constexpr (kKeep) each([&](uint32_t col, float (&v)[kPer]) { keep_sum(col, v); });
    Both all = sums();
    float factor = 1.f / sqrtf(all.sum / (float)p.cols + p.eps);
    if (!(all.sum <= 1e37f) || all.sum < 1e-28f || (of_row && (all.top >= kInfBits || (all.top < kTiny && all.top != 0u)))) {
        // squares beyond fp32's range, or h w where the norm would not be, or zeros: from values that are scaled so that the largest lies in [1, 2)
        Both most{0.f, 0u};
        each([&](uint32_t, float (&v)[kPer]) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) most.top = max(most.top, bits_of(v[e]));
        });
        most = reduce(most, whole_block, shared);
        if (most.top != 0u && most.top < kInfBits) {
            const int k = max(-126, min(126, ilogbf(__uint_as_float(most.top))));
            down = ldexpf(1.f, -k);
            if constexpr (kKeep) each([&](uint32_t, float (&v)[kPer]) {
#pragma unroll
                for (uint32_t e = 0; e < kPer; ++e) v[e] *= down;
            });
            all = sums();
            // h factor = (h down) (factor / down)
            factor = (float)(ldexp(1.0, k) / sqrt((double)(all.sum / (float)p.cols) * ldexp(1.0, 2 * k) + (double)p.eps));
        }
    }
    // Values are quotients of h w and its largest: the norm cancels, and fewer roundings stand between a value and its type's border.
    // A scale, and what brings |h w| to values; from the largest |h w|, as bits.  Below 2^-100 the latter is for |h w| times 2^100, and 0 where the values are to be zeros.
    auto scales_of = [&](uint32_t top, float *scale, float *inverse) {
        const float y = __uint_as_float(top) * factor;
        *scale = y < __uint_as_float(kInfBits) ? y * (1.f / kTop) : __uint_as_float(0x7FFFFFFFu);
        *inverse = *scale > 0.f ? __frcp_rn(__uint_as_float(top) * (top < kTiny ? 0x1p100f : 1.f) * (1.f / kTop)) : 0.f;
    };
    float inverse = 0.f;
    if (of_row) {
        float scale;
        scales_of(all.top, &scale, &inverse);
        if (threadIdx.x == 0) p.scales[row] = scale;
    }
    // What h is multiplied by before w, which may lie as far from 1 as h: y / w, or, for scales of groups, the power of two next below the norm's reciprocal, which leaves the quotients as they are.
    const uint32_t power = __float_as_uint(factor) & kInfBits;
    const bool in_two = eights && !of_row && down == 1.f && power != 0u && power != kInfBits;
    const float first_by = !eights ? factor : in_two ? __uint_as_float(power) : 1.f;
    if (in_two) factor = __uint_as_float((__float_as_uint(factor) & ~kInfBits) | 0x3F800000u);
    const uint32_t lanes = min(32u, p.group / kE), together = max(1u, p.group / (32u * kE));  // of a group: lanes, and times 32 kE columns of a thread
    each([&](uint32_t col, float (&v)[kPer]) {
        if constexpr (!kKeep) {
            if (kAdds && p.sum) {  // (h as it is, of which `v` may be a scaled copy: from the inputs, which may lie where the sum goes)
                float whole[1][kPer];
                load(col, whole);
                keep_sum(col, whole[0]);
            }
        }
        if (kKind != kRow)
#pragma unroll
            for (uint32_t e = 0; e < kPer; e += 2) times_two(v[e], v[e + 1], first_by);
        times_weight<X, kE, kKind>(p, col, v);
        uint32_t tops[kJ];
        float inverses[kJ];
        if (eights && !of_row) {
#pragma unroll
            for (uint32_t j = 0; j < kJ; ++j) {
                tops[j] = 0u;
#pragma unroll
                for (uint32_t e = 0; e < (uint32_t)kE; ++e) tops[j] = max(tops[j], bits_of(v[j * kE + e]));
            }
            if constexpr (kJ > 1) {
                if (together >= 2)
#pragma unroll
                    for (uint32_t j = 0; j < kJ; j += 2) tops[j] = tops[j + 1] = max(tops[j], tops[j + 1]);
                if (together >= 4)
#pragma unroll
                    for (uint32_t j = 0; j < kJ; j += 4) tops[j] = tops[j + 1] = tops[j + 2] = tops[j + 3] = max(tops[j], tops[j + 2]);
            }
#pragma unroll
            for (uint32_t j = 0; j < kJ; ++j) {
#pragma unroll
                for (uint32_t d = 1; d < 32u; d *= 2u)
                    if (d < lanes) tops[j] = max(tops[j], __shfl_xor_sync(0xFFFFFFFFu, tops[j], d));
                const uint32_t at = col + j * 32u * kE;
                float scale;
                scales_of(tops[j], &scale, inverses + j);
                if (at < p.cols && (at & (p.group - 1u)) == 0) p.scales[row * p.groups + (at >> p.group_shift)] = scale;
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kJ; ++j) {
            const uint32_t at = col + j * 32u * kE;
            const bool there = at < p.cols;
            if (eights) {
                const uint32_t top = of_row ? all.top : tops[j];
                const float by = of_row ? inverse : inverses[j];
                if (top < kTiny || by == 0.f)
#pragma unroll
                    for (uint32_t e = 0; e < (uint32_t)kE; ++e) v[j * kE + e] = by == 0.f ? 0.f : v[j * kE + e] * 0x1p100f;
                Raw<uint8_t, kE> q;
#pragma unroll
                for (uint32_t e = 0; e < (uint32_t)kE; e += 2) {
                    uint16_t two;
                    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(kE > 1 ? v[j * kE + (kE > 1 ? e + 1 : e)] * by : 0.f), "f"(v[j * kE + e] * by));
                    if constexpr (kE > 1) reinterpret_cast<uint16_t *>(q.u)[e / 2] = two;
                    else reinterpret_cast<uint8_t *>(q.u)[0] = (uint8_t)two;
                }
                if (there) q.store(static_cast<uint8_t *>(p.out) + (int64_t)row * p.ldo + at);
            } else if (there) {
                const float *y = v + j * kE;
                const int64_t to = (int64_t)row * p.ldo + at;
                if constexpr (kKind != kAny) store_as<X, kE>(p.out, to, y);
                else if (p.out_type == B200SPMM_T_F32) store_as<float, kE>(p.out, to, y);
                else if (p.out_type == B200SPMM_T_F16) store_as<__half, kE>(p.out, to, y);
                else store_as<__nv_bfloat16, kE>(p.out, to, y);
            }
        }
    });
}

// Whether all rows start and end on `e` elements of their types.
bool goes_by(const b200spmm_rms_norm_t *a, uint32_t e) {
    auto fits = [&](const void *p, int64_t ld, int type) { return !p || (aligned(p, std::min<uintptr_t>(16, e * size_of(type))) && (a->rows <= 1 || ld % e == 0)); };
    return a->cols % e == 0 && fits(a->x, a->ldx, a->x_dtype) && fits(a->residual, a->ldr, a->r_dtype) && fits(a->sum, a->lds, a->r_dtype) &&
           fits(a->out, a->ldo, a->out_dtype) && fits(a->weight, e, a->w_dtype);
}

template <typename X, typename R, int kV, int kE, int kKind>
int launch_kernel(const NormParams &p, uint64_t blocks, dim3 threads, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = threads;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, rms_norm_kernel<X, R, kV, kE, kKind>, NormParams(p)));
    return B200SPMM_OK;
}

template <typename X, typename R>
int launch(const NormParams &p, uint32_t e, int kind, cudaStream_t stream) {
    const uint32_t spans = (p.cols + kSpan - 1) / kSpan;
    uint32_t warps = 1, rows_of_block = 4;
    const bool few = p.rows <= 2ull * sm_count();
    if (spans > 4 || (few && spans > 1)) {  // else a warp a row.  Few rows: as many threads as there are values; many: four times eight of them a thread
        rows_of_block = 1;
        warps = std::min(32u, few ? spans : (spans + 3) / 4);
    }
    const uint32_t per = (spans + warps - 1) / warps;
    const uint64_t blocks = (p.rows + rows_of_block - 1) / rows_of_block;
    if (blocks > 0x7FFFFFFFull) return B200SPMM_ERR_UNSUPPORTED;
    const dim3 threads(32 * warps, rows_of_block);
    // kernels of their own for what many rows of ordinary sizes are; else one that asks while it runs
    auto of = [&](auto v, auto n, auto k) { return launch_kernel<X, R, decltype(v)::value, decltype(n)::value, decltype(k)::value>(p, blocks, threads, stream); };
    auto kinds = [&](auto n) {
        using V = std::integral_constant<int, 4>;
        if (kind == kRow) return of(V(), n, std::integral_constant<int, kRow>());
        if (kind == kGroups) return of(V(), n, std::integral_constant<int, kGroups>());
        return of(V(), n, std::integral_constant<int, kSame>());
    };
    auto any = [&](auto n) {
        using A = std::integral_constant<int, kAny>;
        return per <= 1 ? of(std::integral_constant<int, 1>(), n, A()) : per <= 4 ? of(std::integral_constant<int, 4>(), n, A()) : of(std::integral_constant<int, 0>(), n, A());
    };
    if (per > 1 && per <= 4 && kind != kAny && e > 1) return e == 8 ? kinds(std::integral_constant<int, 8>()) : kinds(std::integral_constant<int, 2>());
    return e == 8 ? any(std::integral_constant<int, 8>()) : any(std::integral_constant<int, 1>());
}

template <typename X>
int launch_for(const NormParams &p, int r_type, uint32_t e, int kind, cudaStream_t stream) {
    if (!p.r) return launch<X, void>(p, e, kind, stream);
    if (r_type == B200SPMM_T_F32) return launch<X, float>(p, e, kind, stream);
    return launch<X, X>(p, e, kind, stream);
}

}  // namespace
}  // namespace fp4
}  // namespace b200spmm

using namespace b200spmm;
using namespace b200spmm::fp4;

extern "C" int b200spmm_rms_norm(const b200spmm_rms_norm_t *a, void *stream) {
    if (!a || !is_type(a->x_dtype) || (a->out_dtype != B200SPMM_T_E4M3 && !is_type(a->out_dtype))) return B200SPMM_ERR_INVALID_ARG;
    if (a->residual && a->r_dtype != a->x_dtype && a->r_dtype != B200SPMM_T_F32) return B200SPMM_ERR_INVALID_ARG;
    if ((a->weight && !is_type(a->w_dtype)) || (a->sum && !a->residual) || !(a->eps >= 0.f)) return B200SPMM_ERR_INVALID_ARG;
    if (a->group != 0 && ((a->group != 32 && a->group != 64 && a->group != 128) || a->out_dtype != B200SPMM_T_E4M3)) return B200SPMM_ERR_INVALID_ARG;
    if (a->cols > 0x7FFFFFFFull - 65536) return B200SPMM_ERR_UNSUPPORTED;
    const bool e4m3 = a->out_dtype == B200SPMM_T_E4M3;
    int st = check_dense(a->x, a->x_dtype, a->rows, a->cols, a->ldx);
    if (st == B200SPMM_OK && a->residual) st = check_dense(a->residual, a->r_dtype, a->rows, a->cols, a->ldr);
    if (st == B200SPMM_OK && a->sum) st = check_dense(a->sum, a->r_dtype, a->rows, a->cols, a->lds);
    if (st == B200SPMM_OK && !e4m3) st = check_dense(a->out, a->out_dtype, a->rows, a->cols, a->ldo);
    if (st != B200SPMM_OK) return st;
    const bool empty = a->rows == 0 || a->cols == 0;
    if (!empty && (!a->out || (a->rows > 1 && a->ldo < (int64_t)a->cols))) return B200SPMM_ERR_INVALID_ARG;
    if (a->weight && !aligned(a->weight, size_of(a->w_dtype))) return B200SPMM_ERR_INVALID_ARG;
    if (e4m3 && !empty && (!a->scales || !aligned(a->scales, 4))) return B200SPMM_ERR_INVALID_ARG;
    return on_device(a->device, [&]() -> int {
        if (empty) {
            // (a row without columns has one scale all the same)
            if (e4m3 && a->group == 0 && a->rows && a->scales) B200_CUDA_TRY(cudaMemsetAsync(a->scales, 0, a->rows * 4, static_cast<cudaStream_t>(stream)));
            return B200SPMM_OK;
        }
        NormParams p{a->x, a->residual, a->weight, a->sum, a->out, a->scales, a->ldx, a->ldr, a->lds, a->ldo, a->rows, (uint32_t)a->cols};
        p.groups = a->group ? ((uint32_t)a->cols + a->group - 1) / a->group : 1;
        p.w_type = a->w_dtype;
        p.out_type = a->out_dtype;
        p.group = (uint32_t)a->group;
        p.group_shift = a->group == 128 ? 7 : a->group == 64 ? 6 : 5;
        p.eps = a->eps;
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const uint32_t e = goes_by(a, 8) ? 8 : goes_by(a, 2) ? 2 : 1;
        const bool same = a->weight && a->w_dtype == a->x_dtype && (e4m3 || a->out_dtype == a->x_dtype);
        const int kind = !same ? kAny : !e4m3 ? kSame : a->group ? kGroups : kRow;
        if (a->x_dtype == B200SPMM_T_F32) return launch_for<float>(p, a->r_dtype, e, kind, s);
        if (a->x_dtype == B200SPMM_T_F16) return launch_for<__half>(p, a->r_dtype, e, kind, s);
        return launch_for<__nv_bfloat16>(p, a->r_dtype, e, kind, s);
    });
}
