// Product of a matrix of 4-bit integers with a few columns.
//
//     C[m, j] = sum over groups g of k  scale[g, m] (sum over k in g  (code[m, k] - zero[g, m]) B[k, j])
//
// The inner sums are of exact products (a code less its zero is a small whole number, columns have 16 bits, or 8 with scales of their own), 128 values of k at most, the
// outer one is rounded in fp32 for each: what the MMA cuts off never grows with k.  How it is done: narrow.cuh.
//
// 28672 x 8192 in groups of 128 with zeros, 123 MB, 18.8 us at a copy's rate: one fp16 column 29.6 us, 8 in e4m3 36.  Of the 29.6 multiplying takes 21 (5.5 TB/s: 320 instructions
// for a step of 16 rows x 256 codes fill what issue slots there are), from 3.2 us on, when the columns are there; 1,792 tiles are 12 for 132 blocks and 13 for 16, which end 2 to 4 us
// after the others.  (Times of a captured loop; a call from Python takes the host 5 us or more.)  One column in bf16 31.5, 8 in fp16 30.7 and in bf16 32.5.  8 columns of 8,192 take half of the shared memory and 3 us longer to come.  14331 x 4090 in groups of 64 times 33 columns: 41 us, five MMAs for
// each operand and columns that start on 4 bytes (49 where they came value by value, 61 in two reads of the matrix).
#include "entry.hpp"
#include "fp4_store.cuh"
#include "launch.hpp"
#include "int4.hpp"

namespace b200spmm {
namespace narrow {
namespace {

using fp4::Target;

struct Int4Params {
    Matrix m;
    uint32_t rows, k, n;
    const void *x;
    int64_t along, across;
    bool wide, even;
    const float *x_scales;
    uint32_t x_groups, x_shift;
    Target c;
    uint32_t tiles, warps, steps, window, cols;  // of all blocks together; of a block; of a row; that the columns have room for; of a pass, at most
    uint32_t scales;  // of a column, in a window
};

template <int kNB>
constexpr uint32_t kMaxWarps = kNB <= 1 ? 28 : kNB <= 2 ? 24 : kNB <= 3 ? 20 : 16;

// A lane's sums to C.
template <typename T, int kNB>
B200_DEVICE void store_sums(const Target &c, uint32_t row, uint32_t rows, uint32_t j0, uint32_t n, const float (&sums)[kNB][4]) {
    const int64_t along = c.transposed ? 1 : c.ldc, across = c.transposed ? c.ldc : 1;
    const uint32_t t = threadIdx.x & 3u;
    T *out = reinterpret_cast<T *>(c.ptr);
#pragma unroll
    for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t j = nb * 8u + t * 2u + (e & 1u), r = row + (e >> 1) * 8u;
            if (j < n && r < rows) out[(int64_t)r * along + (int64_t)(j0 + j) * across] = fp4::Elem<T>::from_float(sums[nb][e]);
        }
}

// kScaled: columns in e4m3 with scales.
template <typename T, int kSpan, int kNB, bool kScaled, int kRing>
__global__ void __launch_bounds__(32 * kMaxWarps<kNB>, 1) int4_kernel(const Int4Params p) {
    using W = Weights<T, kSpan>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t base = ptx::smem_u32(smem), warp = warp_index(), g = (threadIdx.x & 31u) >> 2;
    constexpr uint32_t ring_bytes = kRingOf<W, kNB, kRing>;
    const uint32_t j0 = blockIdx.y * (8u * kNB);
    Columns c{};
    c.base = base + p.warps * ring_bytes;
    c.pitch = column_pitch<W>(p.window);
    c.plane = 0;
    c.n = min(8u * kNB, p.n - j0);
    c.scales = c.base + p.cols * c.pitch;
    c.groups = p.scales;
    c.shift = p.x_shift;
    const uint32_t begin = (uint32_t)((uint64_t)p.tiles * blockIdx.x / gridDim.x), end = (uint32_t)((uint64_t)p.tiles * (blockIdx.x + 1u) / gridDim.x);
    const Split split(end - begin, p.steps, p.warps);
    const Share s(split, begin, end, warp, p.steps, p.window, base + warp * ring_bytes);
    ptx::wait_for_grids_before();
    multiply<W, kNB, 1, kScaled, kRing>(
        p.m, s, [](uint32_t tile) { return tile; }, [&](uint32_t tile, uint32_t r) { return (uint64_t)min(tile * kTileRows + r, p.rows - 1u); }, [&](uint32_t) { return c; },
        [&](uint32_t first, uint32_t count) {
            if constexpr (kScaled) {
                // a warp takes a column's; behind a row's end the last one again
                float *to = reinterpret_cast<float *>(smem + (c.scales - base));
                const uint32_t group = (uint32_t)((uint64_t)first * W::kStep >> p.x_shift);
                for (uint32_t j = threadIdx.x >> 5; j < c.n; j += blockDim.x >> 5)
                    for (uint32_t i = threadIdx.x & 31u; i < p.scales; i += 32u) to[j * p.scales + i] = p.x_scales[(uint64_t)(j0 + j) * p.x_groups + min(group + i, p.x_groups - 1u)];
                stage_columns<W>(Eights{static_cast<const uint8_t *>(p.x) + (int64_t)j0 * p.across, p.across, p.wide, p.k}, c.base, c.pitch, first, count, c.n, false);
            } else
                stage_columns<W>(Plain<T>{static_cast<const T *>(p.x) + (int64_t)j0 * p.across, p.along, p.across, p.wide, p.even, p.k}, c.base, c.pitch, first, count, c.n, p.along != 1);
        },
        [&](uint32_t tile, const float(&sums)[kNB][4]) {
            const uint32_t row = tile * kTileRows + g;
            if (p.c.type == B200SPMM_T_F32) store_sums<float, kNB>(p.c, row, p.rows, j0, c.n, sums);
            else if (p.c.type == B200SPMM_T_F16) store_sums<__half, kNB>(p.c, row, p.rows, j0, c.n, sums);
            else store_sums<__nv_bfloat16, kNB>(p.c, row, p.rows, j0, c.n, sums);
        });
}

template <typename T, int kSpan, int kNB, bool kScaled, int kRing>
int launch(Int4Params p, cudaStream_t stream) {
    using W = Weights<T, kSpan>;
    auto kernel = int4_kernel<T, kSpan, kNB, kScaled, kRing>;
    const uint32_t blocks = std::min<uint32_t>(p.tiles, fp4::sm_count()), passes = (p.n + 8 * kNB - 1) / (8 * kNB);
    p.steps = (p.k + W::kStep - 1) / W::kStep;
    p.cols = std::min<uint32_t>(8 * kNB, p.n);
    const Split split((p.tiles + blocks - 1) / blocks, p.steps, kMaxWarps<kNB>);
    p.warps = split.at_once * split.slices;
    // the columns as a whole, or as much of them as there is room for, with their scales: one of a column, or of every group
    const bool of_column = p.x_shift == kWholeGroup;
    const uint32_t ring = p.warps * kRingOf<W, kNB, kRing>, of_step = kScaled && !of_column ? W::kStep >> p.x_shift : 0u;
    p.window = steps_that_fit<W>(p.steps, p.cols, of_step * 4u, ring + (kScaled && of_column ? p.cols * 4u : 0u));
    if (kRing == 4 && p.window < p.steps) return launch<T, kSpan, kNB, kScaled, 2>(p, stream);  // (half the ring, more room)
    if (p.window == 0) return B200SPMM_ERR_UNSUPPORTED;
    p.scales = of_column ? 1u : of_step * p.window;
    const uint32_t bytes = ring + p.cols * (column_pitch<W>(p.window) + (kScaled ? p.scales * 4u : 0u));
    static std::atomic<uint64_t> allowed{0};
    B200_CUDA_TRY(allow_smem(kernel, allowed));
    B200_CUDA_TRY(launch_after(kernel, dim3(blocks, passes), 32u * p.warps, bytes, 1, stream, p));
    return B200SPMM_OK;
}

template <typename T, int kSpan, bool kScaled>
int launch_width(const Int4Params &p, cudaStream_t stream) {
    // as few reads of the matrix as go with 40 columns at once, and as many columns in each
    const uint32_t passes = (p.n + 39) / 40, eights = ((p.n + passes - 1) / passes + 7) / 8;
    if (eights <= 1) return launch<T, kSpan, 1, kScaled, 4>(p, stream);
    if (eights == 2) return launch<T, kSpan, 2, kScaled, 4>(p, stream);
    if (eights == 3) return launch<T, kSpan, 3, kScaled, 4>(p, stream);
    if (eights == 4) return launch<T, kSpan, 4, kScaled, 4>(p, stream);
    return launch<T, kSpan, 5, kScaled, 4>(p, stream);
}
template <typename T, bool kScaled>
int launch_span(const Int4Params &p, uint32_t span, cudaStream_t stream) {
    if (span == 32) return launch_width<T, 32, kScaled>(p, stream);
    if (span == 64) return launch_width<T, 64, kScaled>(p, stream);
    return launch_width<T, 128, kScaled>(p, stream);
}

}  // namespace
}  // namespace narrow
}  // namespace b200spmm

using namespace b200spmm;
using namespace b200spmm::fp4;

extern "C" int b200spmm_int4_product(const b200spmm_int4_t *a, const void *d_B, int64_t ldb, int64_t n, int b_dtype, int b_transposed, const float *d_b_scales, int b_group,
                                     void *d_C, int64_t ldc, int c_dtype, int c_transposed, void *stream) {
    int st = narrow::check_int4(a);
    if (st != B200SPMM_OK) return st;
    if (n < 0) return B200SPMM_ERR_INVALID_ARG;
    if (n > 65535) return B200SPMM_ERR_UNSUPPORTED;
    const bool eights = b_dtype == B200SPMM_T_E4M3;
    if (eights) {
        if (!b_transposed || (b_group != 0 && b_group != 32 && b_group != 64 && b_group != 128)) return B200SPMM_ERR_INVALID_ARG;
        if (n > 0 && a->cols > 0 && (!d_B || (n > 1 && ldb < (int64_t)a->cols) || !d_b_scales || !aligned(d_b_scales, 4))) return B200SPMM_ERR_INVALID_ARG;
    } else {
        st = check_dense(d_B, b_dtype, b_transposed ? (uint64_t)n : a->cols, b_transposed ? a->cols : (uint64_t)n, ldb);
        if (st != B200SPMM_OK) return st;
        if (d_b_scales || b_group) return B200SPMM_ERR_INVALID_ARG;
        if (b_dtype == B200SPMM_T_F32) return B200SPMM_ERR_UNSUPPORTED;
    }
    const uint64_t rows = c_transposed ? (uint64_t)n : a->rows, cols = c_transposed ? a->rows : (uint64_t)n;
    st = check_dense(d_C, c_dtype, rows, cols, ldc);
    if (st != B200SPMM_OK) return st;
    return on_device(a->device, [&]() -> int {
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (rows == 0 || cols == 0) return B200SPMM_OK;
        if (a->cols == 0) return zero_output(d_C, ldc, c_dtype, rows, cols, s);
        narrow::Int4Params p{};
        p.m = narrow::matrix_of(a);
        p.rows = (uint32_t)a->rows;
        p.k = (uint32_t)a->cols;
        p.n = (uint32_t)n;
        p.x = d_B;
        p.along = b_transposed ? 1 : ldb;
        p.across = b_transposed ? ldb : 1;
        const uint32_t unit = eights ? 8 : 16;
        p.wide = p.along == 1 && aligned(d_B, unit) && (n == 1 || p.across * (eights ? 1 : 2) % unit == 0);
        p.even = !eights && p.along == 1 && aligned(d_B, 4) && (n == 1 || p.across % 2 == 0);
        p.x_scales = d_b_scales;
        p.x_groups = b_group ? (p.k + b_group - 1) / b_group : 1;
        p.x_shift = narrow::shift_of(b_group);
        p.c = target_of(d_C, ldc, c_dtype, c_transposed != 0);
        p.tiles = (p.rows + narrow::kTileRows - 1) / narrow::kTileRows;
        uint32_t span = narrow::span_of(a);
        if (eights) {
            if (b_group) span = std::min<uint32_t>(span, b_group);
            return narrow::launch_span<__half, true>(p, span, s);
        }
        if (b_dtype == B200SPMM_T_F16) return narrow::launch_span<__half, false>(p, span, s);
        return narrow::launch_span<__nv_bfloat16, false>(p, span, s);
    });
}
