// Dense matrices to 4 bits and back (layout: fp4.hpp).
#include <algorithm>
#include <type_traits>

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

// The bits of the largest magnitude (NaN above infinity above all numbers).
template <int N>
B200_DEVICE uint32_t top_bits(const float (&v)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// (row, unit) of a walk over rows of `units` units each, `step` units at a time.  Rows are counted from the last one on where a pass follows
// another over the same matrix: what that one read last is still in L2.
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

// 16 neighbours as they are, zeros behind `count`.  `align`: what all rows' starts are multiples of, 8 bytes or 16.
template <typename T>
struct Raw16 {
    uint4 v[sizeof(T)];
    B200_DEVICE void load(const T *src, uint32_t count, uint32_t align) {
        if (align >= 16u && count >= 16u) {
#pragma unroll
            for (uint32_t i = 0; i < sizeof(T); ++i) v[i] = ptx::ld_global_v4(reinterpret_cast<const uint4 *>(src) + i);
        } else if (align >= 8u && count >= 16u) {
#pragma unroll
            for (uint32_t i = 0; i < 2 * sizeof(T); ++i) reinterpret_cast<uint2 *>(v)[i] = reinterpret_cast<const uint2 *>(src)[i];
        } else {
            T *e = reinterpret_cast<T *>(v);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) e[i] = i < count ? src[i] : Elem<T>::from_float(0.f);
        }
    }
    // The bits of the largest magnitude, as those of an fp32 number; 16-bit types two at a time.
    B200_DEVICE uint32_t top() const {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 *h = reinterpret_cast<const __half2 *>(v);
                __half2 most = __habs2(h[0]);
#pragma unroll
                for (int i = 1; i < 8; ++i) most = __hmax2_nan(most, __habs2(h[i]));
                m = *reinterpret_cast<const uint32_t *>(&most);
            } else {
                const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(v);
                __nv_bfloat162 most = __habs2(h[0]);
#pragma unroll
                for (int i = 1; i < 8; ++i) most = __hmax2_nan(most, __habs2(h[i]));
                m = *reinterpret_cast<const uint32_t *>(&most);
            }
            const uint16_t one = (uint16_t)max(m & 0xFFFFu, m >> 16);
            return __float_as_uint(Elem<T>::to_float(*reinterpret_cast<const T *>(&one)));
        }
    }
    B200_DEVICE void floats(float (&f)[16]) const {
        const T *e = reinterpret_cast<const T *>(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = Elem<T>::to_float(e[i]);
    }
    // ... of those that are finite.
    B200_DEVICE uint32_t finite_top() const {
        const uint32_t t = top();
        if (t < kInfBits) return t;
        float f[16];
        floats(f);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t b = __float_as_uint(f[i]) & 0x7FFFFFFFu;
            m = max(m, b < kInfBits ? b : 0u);
        }
        return m;
    }
};

// partial[block] = the largest finite magnitude that the block has seen.  Bound: one read of the matrix; 64 bytes a thread are under way.
template <typename T>
__global__ void __launch_bounds__(kThreads) amax_kernel(const T *x, int64_t ldx, uint32_t rows, uint32_t cols, uint32_t align,
                                                        float *partial) {
    constexpr int kAhead = sizeof(T) == 4 ? 1 : 2;
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    uint32_t m = 0;
    for (Walk w((cols + 15u) / 16u, (uint64_t)blockIdx.x * kThreads + threadIdx.x, (uint64_t)gridDim.x * kThreads); w.row < rows;) {
        Raw16<T> v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            v[i].load(x + (int64_t)w.row * ldx + w.unit * 16u, w.row < rows ? cols - w.unit * 16u : 0u, align);
            w.next();
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) m = max(m, v[i].finite_top());
    }
    m = block_max(m, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = __uint_as_float(m);
}

// The same of rows that start on less than 8 bytes: a warp takes 512 of a row, lanes neighbours (28672 x 8191 fp16 quantised in 409 us, 535 with
// 16 neighbours a lane).
template <typename T>
__global__ void __launch_bounds__(kThreads) amax_any_kernel(const T *x, int64_t ldx, uint32_t rows, uint32_t cols, float *partial) {
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t m = 0;
    for (Walk w((cols + 511u) / 512u, ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / 32u, (uint64_t)gridDim.x * (kThreads / 32u)); w.row < rows; w.next()) {
        const T *src = x + (int64_t)w.row * ldx + w.unit * 512u;
        const uint32_t count = cols - w.unit * 512u;
        Raw16<T> v;
        T *e = reinterpret_cast<T *>(v.v);
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) e[i] = i * 32u + lane < count ? src[i * 32u + lane] : Elem<T>::from_float(0.f);
        m = max(m, v.finite_top());
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

// One unit of 16 neighbours of a row, `raw`, to codes and scales.  Four (nvfp4) or eight (mxfp4) lanes together hold the four scales that lie
// in one word; all lanes of a warp take part.
template <typename T, bool kMx>
B200_DEVICE void quantize_unit(const Raw16<T> &raw, const TensorScale &tensor, bool here, uint32_t row, uint32_t unit, const Dest &d) {
    constexpr uint32_t kLanes = kMx ? 8 : 4;
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t top = raw.top(), byte;
    float v[16];
    raw.floats(v);
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
        byte = quantize_block_nv(v, top, tensor, codes) << (lane & 3u) * 8u;
        byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 1);
        byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
    }
    if (!here) return;
    if (unit * 8u < d.pitch) *reinterpret_cast<uint2 *>(d.values + (uint64_t)row * d.pitch + unit * 8u) = codes;
    if (lane % kLanes == 0) *reinterpret_cast<uint32_t *>(d.scales + scale_word(row, unit / kLanes, d.groups)) = byte;
}

// Blocks along the rows of x, a unit a thread.  Rows end with units that hold nothing: the scales behind the last column, which the
// products read, are zeros.  Bound: reading x once (after amax_kernel, which leaves its last rows in L2: they come first) and writing the
// codes: 28672 x 8192 fp16 91 us in mxfp4, 6.5 TB/s; with the pass before it, 181 in nvfp4.
template <typename T, bool kMx>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T *x, int64_t ldx, const float *partial, uint32_t n_partial, const float *given,
                                                                 const Dest d) {
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    const TensorScale tensor(kMx ? 0 : find_exponent(partial, n_partial, given, shared));
    if (blockIdx.x == 0 && threadIdx.x == 0) *d.tensor_scale = tensor.up;
    for (Walk w(d.groups * (kMx ? 8u : 4u), (uint64_t)blockIdx.x * kThreads + threadIdx.x, (uint64_t)gridDim.x * kThreads);
         __any_sync(0xFFFFFFFFu, w.row < d.rows); w.next()) {
        const bool here = w.row < d.rows;
        const uint32_t col = w.unit * 16u, row = d.rows - 1u - w.row;
        Raw16<T> raw;
        raw.load(x + (int64_t)row * ldx + col, here && col < d.cols ? d.cols - col : 0u, 16u);
        quantize_unit<T, kMx>(raw, tensor, here, row, w.unit, d);
    }
}

// A small matrix in nvfp4, a unit for every thread of one cluster: its largest value is found and used in the same launch.  Bound: latency
// (8 x 8192, the activations of eight tokens: 10 us a call, most of it the host's).
constexpr unsigned kClusterCtas = 8, kClusterThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kClusterThreads) quantize_cluster_kernel(const T *x, int64_t ldx, const Dest d) {
    __shared__ uint32_t shared[kClusterThreads / 32], all[kClusterCtas];
    ptx::cluster_arrive();  // no CTA writes to another one's shared memory before that one runs
    ptx::cluster_wait();
    ptx::wait_for_grids_before();
    const uint32_t units = max(d.groups * 4u, 1u), at = blockIdx.x * blockDim.x + threadIdx.x, row = at / units, unit = at % units;
    const bool here = row < d.rows;
    Raw16<T> raw;
    raw.load(x + (int64_t)row * ldx + unit * 16u, here && unit * 16u < d.cols ? d.cols - unit * 16u : 0u, 16u);
    uint32_t m = __reduce_max_sync(0xFFFFFFFFu, raw.finite_top());
    if ((threadIdx.x & 31u) == 0) shared[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x < 32u) {
        m = __reduce_max_sync(0xFFFFFFFFu, threadIdx.x < blockDim.x / 32u ? shared[threadIdx.x] : 0u);
        // to every CTA of the cluster, each its own place
        if (threadIdx.x < gridDim.x) ptx::st_cluster_u32(ptx::map_to_cta(ptx::smem_u32(all + blockIdx.x), threadIdx.x), m);
    }
    ptx::cluster_arrive();
    ptx::cluster_wait();
    m = 0;
    for (uint32_t i = 0; i < gridDim.x; ++i) m = max(m, all[i]);
    const TensorScale tensor(tensor_exponent(__uint_as_float(m)));
    if (at == 0) *d.tensor_scale = tensor.up;
    quantize_unit<T, false>(raw, tensor, here, row, unit, d);
}

// Blocks along the columns of x (kCols: the 4-bit matrix is the transpose), along the rows, or both from one read; also rows that start on
// any element.  A block of threads takes 128 x 64 of x through shared memory, where it is read along either axis: columns two at a time and 16
// rows a thread, the other 16 of an mxfp4 block being 16 lanes away.  Rows lie in shared memory with their halves exchanged
// where bit 4 of their number is set, so that those lanes do not collide.  What goes to the transpose is put together there as
// well, and leaves 64 neighbouring bytes at a time.  Bound: shared memory and issue: 28672 x 8192 fp16 to the transpose 134 us in mxfp4, of
// which one read and the writing would be 91; both ways with the largest value's pass 307 in nvfp4, of which two reads and the writing would be 184.
constexpr uint32_t kTileR = 128, kTileC = 64, kOutPitch = kTileR / 2 + 16;

template <typename T, bool kMx, bool kRows, bool kCols>
__global__ void __launch_bounds__(kThreads, 4) quantize_tiles_kernel(const T *x, int64_t ldx, uint32_t x_rows, uint32_t x_cols, uint32_t align,
                                                                  const float *partial, uint32_t n_partial, const float *given, const Dest by_rows,
                                                                  const Dest by_cols, uint32_t tiles_c, uint64_t tiles) {
    constexpr uint32_t kPer = 16 / sizeof(T), kVecs = kTileC / kPer;  // elements of a piece, pieces of a row
    __shared__ __align__(16) uint4 tile[kTileR * kVecs];
    __shared__ __align__(16) uint8_t out[kCols ? kTileC * kOutPitch : 16];
    __shared__ __align__(16) uint8_t out_scale[kCols ? kTileC * 8 : 16];
    __shared__ uint32_t shared[kThreads / 32];
    ptx::wait_for_grids_before();
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    const TensorScale tensor(kMx ? 0 : find_exponent(partial, n_partial, given, shared));
    if (blockIdx.x == 0 && tid == 0) {
        if (kRows) *by_rows.tensor_scale = tensor.up;
        if (kCols) *by_cols.tensor_scale = tensor.up;
    }
    auto piece = [&](uint32_t r, uint32_t p) { return r * kVecs + (p ^ ((r >> 4 & 1u) * (kVecs / 2u))); };
    // A tile whose rows start on 8 or 4 bytes, in pieces of as many.
    auto load_tile = [&](auto bytes, uint32_t r0, uint32_t c0) {
        using V = std::conditional_t<decltype(bytes)::value == 8, uint2, uint32_t>;
        constexpr uint32_t kIn = sizeof(V) / sizeof(T), kRow = kTileC / kIn, kLoads = kTileR * kRow / kThreads;
        V v[kLoads];
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t r = (i * kThreads + tid) / kRow, c = (i * kThreads + tid) % kRow * kIn;
            v[i] = V();
            if (r0 + r < x_rows) v[i] = *reinterpret_cast<const V *>(x + (int64_t)(r0 + r) * ldx + c0 + c);
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t r = (i * kThreads + tid) / kRow, c = (i * kThreads + tid) % kRow * kIn;
            *reinterpret_cast<V *>(reinterpret_cast<T *>(tile + piece(r, c / kPer)) + c % kPer) = v[i];
        }
    };
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint64_t u = tiles - 1u - t;  // from the end on, see Walk
        const uint32_t r0 = (uint32_t)(u / tiles_c) * kTileR, c0 = (uint32_t)(u % tiles_c) * kTileC;
        if (align >= 16u && c0 + kTileC <= x_cols) {
            uint4 v[kTileR * kVecs / kThreads];
#pragma unroll
            for (uint32_t i = 0; i < kTileR * kVecs / kThreads; ++i) {
                const uint32_t r = (i * kThreads + tid) / kVecs, p = (i * kThreads + tid) % kVecs;
                v[i] = r0 + r < x_rows ? ptx::ld_global_v4(x + (int64_t)(r0 + r) * ldx + c0 + p * kPer) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (uint32_t i = 0; i < kTileR * kVecs / kThreads; ++i) tile[piece((i * kThreads + tid) / kVecs, (i * kThreads + tid) % kVecs)] = v[i];
        } else if (align >= 8u && c0 + kTileC <= x_cols) {
            load_tile(std::integral_constant<uint32_t, 8>(), r0, c0);
        } else if (sizeof(T) < 4 && align >= 4u && c0 + kTileC <= x_cols) {
            load_tile(std::integral_constant<uint32_t, sizeof(T) < 4 ? 4 : 8>(), r0, c0);
        } else {
#pragma unroll 8
            for (uint32_t i = tid; i < kTileR * kTileC; i += kThreads) {
                const uint32_t r = i / kTileC, c = i % kTileC;
                reinterpret_cast<T *>(tile + piece(r, c / kPer))[c % kPer] =
                    r0 + r < x_rows && c0 + c < x_cols ? x[(int64_t)(r0 + r) * ldx + c0 + c] : Elem<T>::from_float(0.f);
            }
        }
        __syncthreads();
        if constexpr (kRows) {
#pragma unroll 1
            for (uint32_t i = tid; i < kTileR * (kTileC / 16); i += kThreads) {
                const uint32_t r = i / 4, q = i % 4, row = r0 + r, col = c0 + q * 16;
                Raw16<T> raw;
#pragma unroll
                for (uint32_t j = 0; j < sizeof(T); ++j) raw.v[j] = tile[piece(r, q * sizeof(T) + j)];
                uint32_t top = raw.top(), byte;
                float v[16];
                raw.floats(v);
                uint2 codes;
                if constexpr (kMx) {
                    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    float factor;
                    byte = block_scale_mx(top, factor);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = byte == 0xFFu ? 0.f : v[j] * factor;
                    codes = make_uint2(to_e2m1x8(v), to_e2m1x8(v + 8));
                    byte <<= (q >> 1) * 8u;
                    byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
                } else {
                    byte = quantize_block_nv(v, top, tensor, codes) << q * 8u;
                    byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 1);
                    byte |= __shfl_xor_sync(0xFFFFFFFFu, byte, 2);
                }
                if (row < by_rows.rows) {
                    if (col / 2u < by_rows.pitch) *reinterpret_cast<uint2 *>(by_rows.values + (uint64_t)row * by_rows.pitch + col / 2u) = codes;
                    if (q == 0) {
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
            // lanes 0-15 and 16-31: 16 rows each, of columns 2 (lane % 16) and + 1 of a half of the tile
            const uint32_t b = (tid >> 6) * 2u + (lane >> 4), c = ((tid >> 5 & 1u) * 16u + (lane & 15u)) * 2u;
            float v[2][16];
            uint32_t top[2] = {0u, 0u};
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) {
                const T *e = reinterpret_cast<const T *>(tile + piece(b * 16u + j, c / kPer)) + c % kPer;
                struct alignas(2 * sizeof(T)) Two { T a, b; };
                const Two two = *reinterpret_cast<const Two *>(e);
                v[0][j] = Elem<T>::to_float(two.a);
                v[1][j] = Elem<T>::to_float(two.b);
            }
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
                top[k] = top_bits(v[k]);
                uint2 codes;
                if constexpr (kMx) {
                    const uint32_t both = max(top[k], __shfl_xor_sync(0xFFFFFFFFu, top[k], 16));
                    float factor;
                    const uint32_t byte = block_scale_mx(both, factor);
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) v[k][j] = byte == 0xFFu ? 0.f : v[k][j] * factor;
                    codes = make_uint2(to_e2m1x8(v[k]), to_e2m1x8(v[k] + 8));
                    if (lane < 16u) out_scale[(c + k) * 8u + b / 2u] = (uint8_t)byte;
                } else {
                    out_scale[(c + k) * 8u + b] = (uint8_t)quantize_block_nv(v[k], top[k], tensor, codes);
                }
                *reinterpret_cast<uint2 *>(out + (c + k) * kOutPitch + b * 8u) = codes;
            }
            __syncthreads();
            for (uint32_t i = tid; i < kTileC * 4u; i += kThreads) {
                const uint32_t col = i / 4, q = i % 4, row = c0 + col, at = r0 / 2u + q * 16u;
                if (row < by_cols.rows && at < by_cols.pitch)
                    *reinterpret_cast<uint4 *>(by_cols.values + (uint64_t)row * by_cols.pitch + at) = *reinterpret_cast<const uint4 *>(out + col * kOutPitch + q * 16u);
            }
            constexpr uint32_t kWords = kMx ? 1 : 2;  // of scales for a column of the tile
            for (uint32_t i = tid; i < kTileC * kWords; i += kThreads) {
                const uint32_t col = i / kWords, w = i % kWords, row = c0 + col, group = r0 / kTileR * kWords + w;
                if (row < by_cols.rows && group < by_cols.groups)
                    *reinterpret_cast<uint32_t *>(by_cols.scales + scale_word(row, group, by_cols.groups)) = *reinterpret_cast<const uint32_t *>(out_scale + col * 8u + w * 4u);
            }
        }
        __syncthreads();  // the next tile overwrites what this one reads
    }
}

// A thread takes eight values, a word of codes, and writes them in one piece; where rows start anywhere, a warp's 256 values go through
// shuffles and leave 32 neighbours at a time.  Bound: reading the matrix and writing x once:
// 28672 x 8192 nvfp4 117 us to fp16, 187 to fp32, 5.1 and 5.7 TB/s; to fp32 rows that start anywhere, 4090 x 5001
// mxfp4, 31, where its bytes are 14: the shuffles.
template <typename T, bool kMx, bool kWide>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t *values, const uint8_t *scales,
                                                              const float *tensor_scale, uint32_t rows, uint32_t cols, uint32_t pitch,
                                                              uint32_t groups, T *x, int64_t ldx) {
    constexpr uint32_t kAhead = 4;
    ptx::wait_for_grids_before();
    const uint32_t lane = threadIdx.x & 31u;
    const float whole = kMx ? 1.f : *reinterpret_cast<const volatile float *>(tensor_scale);
    // a warp's unit: 256 columns of a row
    for (Walk w((cols + 255u) / 256u, ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / 32u, (uint64_t)gridDim.x * (kThreads / 32u)); w.row < rows;) {
        uint32_t codes[kAhead], row[kAhead], col[kAhead], bytes[kAhead];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            row[a] = w.row;
            col[a] = w.unit * 256u + lane * 8u;
            const uint32_t block = col[a] / (kMx ? 32u : 16u);
            codes[a] = bytes[a] = 0u;
            if (w.row < rows && col[a] < cols) {
                codes[a] = *reinterpret_cast<const uint32_t *>(values + (uint64_t)row[a] * pitch + col[a] / 2u);
                bytes[a] = scales[scale_word(row[a], block / 4u, groups) + block % 4u];
            }
            w.next();
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            if (row[a] >= rows) break;  // (the warp's)
            const float s = kMx ? from_e8m0(bytes[a]) : from_e4m3(bytes[a]);
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 two = __half22float2(from_e2m1x2(codes[a] >> i * 8));
                v[2 * i] = kMx ? two.x * s : two.x * s * whole;  // code times scale is exact: one rounding, and one to T
                v[2 * i + 1] = kMx ? two.y * s : two.y * s * whole;
            }
            T *dst = x + (int64_t)row[a] * ldx + col[a];
            if constexpr (kWide) {
                if (col[a] + 8u <= cols) {
                    uint4 out[sizeof(T) / 2];
                    T *e = reinterpret_cast<T *>(out);
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_float(v[i]);
                    if constexpr (sizeof(T) == 4) ptx::st_global_v8(dst, reinterpret_cast<const uint32_t *>(out));
                    else *reinterpret_cast<uint4 *>(dst) = out[0];
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        if (col[a] + i < cols) dst[i] = Elem<T>::from_float(v[i]);
                }
            } else {
                const uint32_t first = col[a] - lane * 8u;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {  // value 32 i + lane of the warp's: lane 4 i + lane / 8 has it, as its value lane % 8
                    float mine = 0.f;
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const float f = __shfl_sync(0xFFFFFFFFu, v[j], (int)(i * 4u + lane / 8u));
                        if (lane % 8u == j) mine = f;
                    }
                    const uint32_t c = first + i * 32u + lane;
                    if (c < cols) x[(int64_t)row[a] * ldx + c] = Elem<T>::from_float(mine);
                }
            }
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
    // what all rows start on, in bytes: 16 or less
    const uint64_t starts = reinterpret_cast<uintptr_t>(x) | (x_rows > 1 ? (uint64_t)ldx * sizeof(T) : 0u) | 16u;
    const uint32_t align = (uint32_t)(starts & (~starts + 1u));
    const bool wide = align == 16u;
    uint32_t n_partial = 0;
    const uint64_t row_units = by_rows ? (uint64_t)dest_of(by_rows).rows * dest_of(by_rows).groups * (kMx ? 8u : 4u) : 0;
    if (!kMx && !given && !by_cols && wide && row_units <= kClusterCtas * kClusterThreads) {
        const unsigned ctas = (unsigned)std::max<uint64_t>(1, (row_units + kClusterThreads - 1) / kClusterThreads);
        B200_CUDA_TRY(launch_after(quantize_cluster_kernel<T>, dim3(ctas), kClusterThreads, 0, ctas, stream, x, ldx, dest_of(by_rows)));
        return B200SPMM_OK;
    }
    if (!kMx && !given) {
        const uint64_t units = (uint64_t)x_rows * ((x_cols + 15u) / 16u);
        n_partial = std::min(kAmaxBlocks, grid_for((units + kThreads - 1) / kThreads));
        if (align >= 8u) B200_CUDA_TRY(launch_after(amax_kernel<T>, dim3(n_partial), kThreads, 0, 1, stream, x, ldx, x_rows, x_cols, align, workspace));
        else B200_CUDA_TRY(launch_after(amax_any_kernel<T>, dim3(n_partial), kThreads, 0, 1, stream, x, ldx, x_rows, x_cols, workspace));
    }
    if (!by_cols && wide) {
        B200_CUDA_TRY(launch_after(quantize_rows_kernel<T, kMx>, dim3(grid_for((row_units + kThreads - 1) / kThreads)), kThreads, 0, 1, stream, x, ldx,
                                   (const float *)workspace, n_partial, given, dest_of(by_rows)));
        return B200SPMM_OK;
    }
    const Dest rows = by_rows ? dest_of(by_rows) : Dest{}, cols = by_cols ? dest_of(by_cols) : Dest{};
    // the tiles cover the padded scales of either matrix, too
    const uint32_t tiles_c = std::max<uint32_t>((x_cols + kTileC - 1) / kTileC, rows.groups * (kMx ? 2u : 1u));
    const uint64_t tiles = (uint64_t)tiles_c * ((x_rows + kTileR - 1) / kTileR);
    auto kernel = !by_cols ? quantize_tiles_kernel<T, kMx, true, false> : by_rows ? quantize_tiles_kernel<T, kMx, true, true> : quantize_tiles_kernel<T, kMx, false, true>;
    B200_CUDA_TRY(launch_after(kernel, dim3(grid_for(tiles)), kThreads, 0, 1, stream, x, ldx, x_rows, x_cols, align, (const float *)workspace, n_partial,
                               given, rows, cols, tiles_c, tiles));
    return B200SPMM_OK;
}

template <typename T>
int dequantize_typed(const b200spmm_fp4_t *a, T *x, int64_t ldx, cudaStream_t stream) {
    const Dest d = dest_of(a);
    const bool wide = reinterpret_cast<uintptr_t>(x) % (8 * sizeof(T)) == 0 && ldx % 8 == 0, mx = a->format == B200SPMM_MXFP4;
    const uint64_t warps = ((uint64_t)d.rows * ((d.cols + 255u) / 256u) + 3u) / 4u;  // with four units each
    auto kernel = mx ? (wide ? dequantize_kernel<T, true, true> : dequantize_kernel<T, true, false>)
                     : (wide ? dequantize_kernel<T, false, true> : dequantize_kernel<T, false, false>);
    B200_CUDA_TRY(launch_after(kernel, dim3(grid_for((warps + kThreads / 32u - 1) / (kThreads / 32u))), kThreads, 0, 1, stream, (const uint8_t *)d.values,
                               (const uint8_t *)d.scales, (const float *)d.tensor_scale, d.rows, d.cols, d.pitch, d.groups, x, ldx));
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
