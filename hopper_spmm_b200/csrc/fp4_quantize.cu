// Dense matrices to 4 bits and back (layout: fp4.hpp).
#include <algorithm>

#include "common.hpp"
#include "fp4.hpp"
#include "fp4_convert.cuh"
#include "launch.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

constexpr int kThreads = 256;

// Where one matrix goes.
struct Dest {
    uint8_t *values, *scales;
    float *tensor_scale;
    uint32_t rows, cols;  // of the 4-bit matrix
    uint32_t pitch, groups;
};

// 16 neighbours of a row as fp32, zeros behind `count`.  kWide: the address is a multiple of 16 bytes.
template <typename T>
B200_DEVICE void load16(const T *src, uint32_t count, bool wide, float (&v)[16]) {
    if (wide && count >= 16u) {
        constexpr int kVecs = 16 * sizeof(T) / 16;
        uint4 raw[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) raw[i] = ptx::ld_global_v4(reinterpret_cast<const uint4 *>(src) + i);
        const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = Elem<T>::to_float(e[i]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) v[i] = i < count ? Elem<T>::to_float(src[i]) : 0.f;
    }
}

// The bits of the largest magnitude (NaN above infinity above all numbers).
template <int N>
B200_DEVICE uint32_t top_bits(const float (&v)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// (row, unit) of a walk over rows of `units` units each, `step` units at a time.
struct Walk {
    uint32_t row, unit, row_step, unit_step, units;
    B200_DEVICE Walk(uint32_t units_, uint64_t first, uint64_t step) : units(max(units_, 1u)) {
        row = (uint32_t)(first / units);
        unit = (uint32_t)(first % units);
        row_step = (uint32_t)(step / units);
        unit_step = (uint32_t)(step % units);
    }
    B200_DEVICE void next() {
        row += row_step;
        unit += unit_step;
        if (unit >= units) {
            unit -= units;
            ++row;
        }
    }
};

B200_DEVICE uint32_t block_max(uint32_t m, uint32_t *shared) {
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if ((threadIdx.x & 31u) == 0) shared[threadIdx.x >> 5] = m;
    __syncthreads();
    m = 0;
    for (uint32_t i = 0; i < blockDim.x / 32u; ++i) m = max(m, shared[i]);
    __syncthreads();
    return m;
}

// partial[block] = the largest finite magnitude that the block has seen.  Bound: one read of the matrix.
template <typename T>
__global__ void __launch_bounds__(kThreads) amax_kernel(const T *__restrict__ x, int64_t ldx, uint32_t rows, uint32_t cols, bool wide,
                                                        float *__restrict__ partial) {
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    uint32_t m = 0;
    for (Walk w((cols + 15u) / 16u, (uint64_t)blockIdx.x * kThreads + threadIdx.x, (uint64_t)gridDim.x * kThreads); w.row < rows; w.next()) {
        float v[16];
        load16(x + (int64_t)w.row * ldx + w.unit * 16u, cols - w.unit * 16u, wide, v);
        uint32_t t = top_bits(v);
        if (t >= kInfBits) {  // only what is finite counts
            t = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
                t = max(t, b < kInfBits ? b : 0u);
            }
        }
        m = max(m, t);
    }
    m = block_max(m, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = __uint_as_float(m);
}

// The exponent of the tensor's scale, for every thread: from the partial maxima, or from a given scale.
B200_DEVICE int find_exponent(const float *partial, uint32_t n_partial, const float *given, uint32_t *shared) {
    if (given) return exponent_above(*reinterpret_cast<const volatile float *>(given));
    uint32_t m = 0;
    for (uint32_t i = threadIdx.x; i < n_partial; i += blockDim.x) m = max(m, __float_as_uint(*reinterpret_cast<const volatile float *>(partial + i)));
    return tensor_exponent(__uint_as_float(block_max(m, shared)));
}

// Blocks along the rows of x.  A thread takes 16 neighbours; four (nvfp4) or eight (mxfp4) lanes together hold the four scales
// that lie in one word.  Rows end with units that hold nothing: the scales behind the last column, which the products read, are zeros.
template <typename T, bool kMx>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, bool wide, const float *partial, uint32_t n_partial,
                                                                 const float *given, const Dest d) {
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    float inv_tensor = 1.f;
    if constexpr (!kMx) {
        const int k = find_exponent(partial, n_partial, given, shared);
        if (blockIdx.x == 0 && threadIdx.x == 0) *d.tensor_scale = exp2_int(k);
        inv_tensor = k == 127 ? __uint_as_float(0x00400000u) : exp2_int(-k);
    } else if (blockIdx.x == 0 && threadIdx.x == 0) {
        *d.tensor_scale = 1.f;
    }
    constexpr uint32_t kLanes = kMx ? 8 : 4;  // of a word of scales
    const uint32_t lane = threadIdx.x & 31u;
    for (Walk w(d.groups * kLanes, (uint64_t)blockIdx.x * kThreads + threadIdx.x, (uint64_t)gridDim.x * kThreads);
         __any_sync(0xFFFFFFFFu, w.row < d.rows); w.next()) {
        const bool here = w.row < d.rows;
        const uint32_t col = w.unit * 16u;
        float v[16];
        load16(x + (int64_t)w.row * ldx + col, here && col < d.cols ? d.cols - col : 0u, wide, v);
        uint32_t top = top_bits(v), byte;
        uint2 codes;
        if constexpr (kMx) {
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            float factor;
            byte = block_scale_mx(top, factor);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = byte == 0xFFu ? 0.f : v[i] * factor;
            codes = make_uint2(to_e2m1x8(v), to_e2m1x8(v + 8));
            byte <<= (lane >> 1 & 3u) * 8u;
            byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
            byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 4);
        } else {
            byte = quantize_block_nv(v, top, inv_tensor, codes) << (lane & 3u) * 8u;
            byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 1);
            byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
        }
        if (!here) continue;  // (no lane leaves the loop alone: the condition is the warp's)
        if (col / 2u < d.pitch) *reinterpret_cast<uint2 *>(d.values + (uint64_t)w.row * d.pitch + col / 2u) = codes;
        if (lane % kLanes == 0) *reinterpret_cast<uint32_t *>(d.scales + scale_word(w.row, w.unit / kLanes, d.groups)) = byte;
    }
}

// Blocks along the columns of x (kCols: the 4-bit matrix is the transpose), along the rows, or both from one read.  A block of
// threads takes 128 x 64 of x through shared memory, which is read once along either axis; what goes to the transpose is put
// together there as well, so that 64 neighbouring bytes are written.
constexpr uint32_t kTileR = 128, kTileC = 64, kOutPitch = kTileR / 2 + 16;

template <typename T, bool kMx, bool kRows, bool kCols>
__global__ void __launch_bounds__(kThreads) quantize_tiles_kernel(const T *__restrict__ x, int64_t ldx, uint32_t x_rows, uint32_t x_cols, bool wide,
                                                                  const float *partial, uint32_t n_partial, const float *given, const Dest by_rows,
                                                                  const Dest by_cols, uint32_t tiles_c, uint64_t tiles) {
    constexpr uint32_t kPitch = kTileC + 16 / sizeof(T);  // elements: 16 bytes more than a row, so that neither way of reading collides
    __shared__ __align__(16) T tile[kTileR * kPitch];
    __shared__ __align__(16) uint8_t out[kTileC * kOutPitch];
    __shared__ __align__(16) uint8_t out_scale[kTileC * 8];
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    const uint32_t tid = threadIdx.x;
    float inv_tensor = 1.f;
    if constexpr (!kMx) {
        const int k = find_exponent(partial, n_partial, given, shared);
        inv_tensor = k == 127 ? __uint_as_float(0x00400000u) : exp2_int(-k);
        if (blockIdx.x == 0 && tid == 0) {
            if (kRows) *by_rows.tensor_scale = exp2_int(k);
            if (kCols) *by_cols.tensor_scale = exp2_int(k);
        }
    } else if (blockIdx.x == 0 && tid == 0) {
        if (kRows) *by_rows.tensor_scale = 1.f;
        if (kCols) *by_cols.tensor_scale = 1.f;
    }
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t r0 = (uint32_t)(t / tiles_c) * kTileR, c0 = (uint32_t)(t % tiles_c) * kTileC;
        if (wide) {
            constexpr uint32_t kPer = 16 / sizeof(T), kVecs = kTileC / kPer;
            for (uint32_t i = tid; i < kTileR * kVecs; i += kThreads) {
                const uint32_t r = i / kVecs, c = i % kVecs * kPer;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (r0 + r < x_rows) {
                    const T *src = x + (int64_t)(r0 + r) * ldx + c0 + c;
                    if (c0 + c + kPer <= x_cols) {
                        v = ptx::ld_global_v4(src);
                    } else {
                        T *e = reinterpret_cast<T *>(&v);
                        for (uint32_t j = 0; j < kPer; ++j)
                            if (c0 + c + j < x_cols) e[j] = src[j];
                    }
                }
                *reinterpret_cast<uint4 *>(tile + r * kPitch + c) = v;
            }
        } else {
            for (uint32_t i = tid; i < kTileR * kTileC; i += kThreads) {
                const uint32_t r = i / kTileC, c = i % kTileC;
                tile[r * kPitch + c] = r0 + r < x_rows && c0 + c < x_cols ? x[(int64_t)(r0 + r) * ldx + c0 + c] : Elem<T>::from_float(0.f);
            }
        }
        __syncthreads();
        if constexpr (kRows) {
            for (uint32_t i = tid; i < kTileR * (kTileC / 16); i += kThreads) {
                const uint32_t r = i / 4, u = i % 4, row = r0 + r, col = c0 + u * 16;
                float v[16];
                const T *src = tile + r * kPitch + u * 16;
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = Elem<T>::to_float(src[j]);
                uint32_t top = top_bits(v), byte;
                uint2 codes;
                if constexpr (kMx) {
                    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    float factor;
                    byte = block_scale_mx(top, factor);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = byte == 0xFFu ? 0.f : v[j] * factor;
                    codes = make_uint2(to_e2m1x8(v), to_e2m1x8(v + 8));
                    byte <<= (u >> 1) * 8u;
                    byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
                } else {
                    byte = quantize_block_nv(v, top, inv_tensor, codes) << u * 8u;
                    byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 1);
                    byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
                }
                if (row < by_rows.rows) {
                    if (col / 2u < by_rows.pitch) *reinterpret_cast<uint2 *>(by_rows.values + (uint64_t)row * by_rows.pitch + col / 2u) = codes;
                    if (u == 0) {
                        if constexpr (kMx) {  // a tile is half a word of scales wide
                            if (c0 / 128u < by_rows.groups)
                                *reinterpret_cast<uint16_t *>(by_rows.scales + scale_word(row, c0 / 128u, by_rows.groups) + (c0 / 64u & 1u) * 2u) = (uint16_t)byte;
                        } else if (c0 / 64u < by_rows.groups) {
                            *reinterpret_cast<uint32_t *>(by_rows.scales + scale_word(row, c0 / 64u, by_rows.groups)) = byte;
                        }
                    }
                }
            }
        }
        if constexpr (kCols) {
            constexpr uint32_t kBlk = kMx ? 32 : 16;
            for (uint32_t i = tid; i < kTileC * (kTileR / kBlk); i += kThreads) {
                const uint32_t c = i % kTileC, b = i / kTileC;
                float v[kBlk];
#pragma unroll
                for (uint32_t j = 0; j < kBlk; ++j) v[j] = Elem<T>::to_float(tile[(b * kBlk + j) * kPitch + c]);
                const uint32_t top = top_bits(v);
                if constexpr (kMx) {
                    float factor;
                    const uint32_t byte = block_scale_mx(top, factor);
#pragma unroll
                    for (uint32_t j = 0; j < kBlk; ++j) v[j] = byte == 0xFFu ? 0.f : v[j] * factor;
                    *reinterpret_cast<uint4 *>(out + c * kOutPitch + b * 16u) =
                        make_uint4(to_e2m1x8(v), to_e2m1x8(v + 8), to_e2m1x8(v + 16), to_e2m1x8(v + 24));
                    out_scale[c * 8u + b] = (uint8_t)byte;
                } else {
                    uint2 codes;
                    out_scale[c * 8u + b] = (uint8_t)quantize_block_nv(v, top, inv_tensor, codes);
                    *reinterpret_cast<uint2 *>(out + c * kOutPitch + b * 8u) = codes;
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < kTileC * 4u; i += kThreads) {
                const uint32_t c = i / 4, q = i % 4, row = c0 + c, at = r0 / 2u + q * 16u;
                if (row < by_cols.rows && at < by_cols.pitch)
                    *reinterpret_cast<uint4 *>(by_cols.values + (uint64_t)row * by_cols.pitch + at) = *reinterpret_cast<const uint4 *>(out + c * kOutPitch + q * 16u);
            }
            constexpr uint32_t kWords = kMx ? 1 : 2;  // of scales for a column of the tile
            for (uint32_t i = tid; i < kTileC * kWords; i += kThreads) {
                const uint32_t c = i / kWords, w = i % kWords, row = c0 + c, group = r0 / kTileR * kWords + w;
                if (row < by_cols.rows && group < by_cols.groups)
                    *reinterpret_cast<uint32_t *>(by_cols.scales + scale_word(row, group, by_cols.groups)) = *reinterpret_cast<const uint32_t *>(out_scale + c * 8u + w * 4u);
            }
        }
        __syncthreads();  // the next tile overwrites what this one reads
    }
}

// A thread takes 16 values and their scale.  Bound: reading the matrix and writing x once.
template <typename T, bool kMx>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t *__restrict__ values, const uint8_t *__restrict__ scales,
                                                              const float *__restrict__ tensor_scale, uint32_t rows, uint32_t cols, uint32_t pitch,
                                                              uint32_t groups, T *__restrict__ x, int64_t ldx, bool wide) {
    ptx::wait_for_grids_before();
    const float whole = kMx ? 1.f : *reinterpret_cast<const volatile float *>(tensor_scale);
    for (Walk w((cols + 15u) / 16u, (uint64_t)blockIdx.x * kThreads + threadIdx.x, (uint64_t)gridDim.x * kThreads); w.row < rows; w.next()) {
        const uint2 codes = *reinterpret_cast<const uint2 *>(values + (uint64_t)w.row * pitch + w.unit * 8u);
        const uint32_t block = kMx ? w.unit / 2u : w.unit;
        const uint32_t byte = scales[scale_word(w.row, block / 4u, groups) + block % 4u];
        const float s = kMx ? from_e8m0(byte) : from_e4m3(byte);
        T out[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 two = __half22float2(from_e2m1x2((i < 4 ? codes.x : codes.y) >> (i & 3) * 8));
            out[2 * i] = Elem<T>::from_float(two.x * s * whole);  // code times scale is exact: one rounding, and one to T
            out[2 * i + 1] = Elem<T>::from_float(two.y * s * whole);
        }
        T *dst = x + (int64_t)w.row * ldx + w.unit * 16u;
        if (wide && cols - w.unit * 16u >= 16u) {
#pragma unroll
            for (uint32_t i = 0; i < 16 * sizeof(T) / 16; ++i) reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(out)[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i)
                if (w.unit * 16u + i < cols) dst[i] = out[i];
        }
    }
}

Dest dest_of(const b200spmm_fp4_t *m) {
    const Layout l = layout_of(m->rows, m->cols, m->format);
    const uint32_t rows = m->cols ? (uint32_t)m->rows : 0u;  // (rows of no columns have nothing to write)
    return {static_cast<uint8_t *>(m->values), static_cast<uint8_t *>(m->scales), m->tensor_scale, rows, (uint32_t)m->cols, l.pitch, l.groups};
}

// Blocks for `work` blocks' worth of units: up to eight of 256 threads a multiprocessor.
unsigned grid_for(uint64_t work) { return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>(work, (uint64_t)sm_count() * 8u)); }

template <typename T, bool kMx>
int quantize_typed(const T *x, int64_t ldx, uint32_t x_rows, uint32_t x_cols, const float *given, const b200spmm_fp4_t *by_rows,
                   const b200spmm_fp4_t *by_cols, float *workspace, cudaStream_t stream) {
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16u == 0 && ldx * (int64_t)sizeof(T) % 16 == 0;
    uint32_t n_partial = 0;
    if (!kMx && !given) {
        const uint64_t units = (uint64_t)x_rows * ((x_cols + 15u) / 16u);
        n_partial = std::min(kAmaxBlocks, grid_for((units + kThreads - 1) / kThreads));
        B200_CUDA_TRY(launch_after(amax_kernel<T>, dim3(n_partial), kThreads, 0, 1, stream, x, ldx, x_rows, x_cols, wide, workspace));
    }
    if (!by_cols) {
        const Dest d = dest_of(by_rows);
        const uint64_t units = (uint64_t)d.rows * d.groups * (kMx ? 8u : 4u);
        B200_CUDA_TRY(launch_after(quantize_rows_kernel<T, kMx>, dim3(grid_for((units + kThreads - 1) / kThreads)), kThreads, 0, 1, stream, x, ldx, wide,
                                   (const float *)workspace, n_partial, given, d));
        return B200SPMM_OK;
    }
    const Dest rows = by_rows ? dest_of(by_rows) : Dest{}, cols = dest_of(by_cols);
    // the tiles cover the padded scales of either matrix, too
    const uint32_t tiles_c = std::max<uint32_t>((x_cols + kTileC - 1) / kTileC, rows.groups * (kMx ? 2u : 1u));
    const uint64_t tiles = (uint64_t)tiles_c * ((x_rows + kTileR - 1) / kTileR);
    auto kernel = by_rows ? quantize_tiles_kernel<T, kMx, true, true> : quantize_tiles_kernel<T, kMx, false, true>;
    B200_CUDA_TRY(launch_after(kernel, dim3(grid_for(tiles)), kThreads, 0, 1, stream, x, ldx, x_rows, x_cols, wide, (const float *)workspace, n_partial,
                               given, rows, cols, tiles_c, tiles));
    return B200SPMM_OK;
}

template <typename T>
int dequantize_typed(const b200spmm_fp4_t *a, T *x, int64_t ldx, cudaStream_t stream) {
    const Dest d = dest_of(a);
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16u == 0 && ldx * (int64_t)sizeof(T) % 16 == 0;
    const uint64_t units = (uint64_t)d.rows * ((d.cols + 15u) / 16u);
    auto kernel = a->format == B200SPMM_MXFP4 ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
    B200_CUDA_TRY(launch_after(kernel, dim3(grid_for((units + kThreads - 1) / kThreads)), kThreads, 0, 1, stream, (const uint8_t *)d.values,
                               (const uint8_t *)d.scales, (const float *)d.tensor_scale, d.rows, d.cols, d.pitch, d.groups, x, ldx, wide));
    return B200SPMM_OK;
}

}  // namespace

int launch_quantize(const void *x, int64_t ldx, int x_dtype, uint64_t x_rows, uint64_t x_cols, const float *given, const b200spmm_fp4_t *by_rows,
                    const b200spmm_fp4_t *by_cols, float *workspace, cudaStream_t stream) {
    const bool mx = (by_rows ? by_rows : by_cols)->format == B200SPMM_MXFP4;
    const uint32_t r = (uint32_t)x_rows, c = (uint32_t)x_cols;
    auto run = [&](auto type) {
        using T = decltype(type);
        const T *p = static_cast<const T *>(x);
        return mx ? quantize_typed<T, true>(p, ldx, r, c, given, by_rows, by_cols, workspace, stream)
                  : quantize_typed<T, false>(p, ldx, r, c, given, by_rows, by_cols, workspace, stream);
    };
    return x_dtype == B200SPMM_T_F32 ? run(float()) : x_dtype == B200SPMM_T_F16 ? run(__half()) : run(__nv_bfloat16());
}

int launch_dequantize(const b200spmm_fp4_t *a, void *x, int64_t ldx, int x_dtype, cudaStream_t stream) {
    return x_dtype == B200SPMM_T_F32   ? dequantize_typed(a, static_cast<float *>(x), ldx, stream)
           : x_dtype == B200SPMM_T_F16 ? dequantize_typed(a, static_cast<__half *>(x), ldx, stream)
                                       : dequantize_typed(a, static_cast<__nv_bfloat16 *>(x), ldx, stream);
}

}  // namespace fp4
}  // namespace b200spmm
