// How a product is shared out over pairs of CTAs that make tiles of 256 rows x up to 256 columns.
//
// Items are tiles of C.  Those of the last, incomplete round are cut along k into parts, so that every pair has something to
// do; their sums go to the workspace and a second kernel adds them up in order.
#pragma once

#include <algorithm>

#include "fp4_store.cuh"

namespace b200spmm {
namespace fp4 {

constexpr uint32_t kPairRows4 = 256, kPairCols4 = 256;

// Tiles of 256 rows x `cols` columns.  The side with fewer tiles is gone through in groups that L2 holds while the other one streams
// by: 28672 x 8192 nvfp4 times 2,048 columns, the long side in the columns, took 267 us side by side and 220 the other way round.
struct Split {
    uint32_t cols;              // of a tile, a multiple of 32
    uint32_t inner, outer;      // tiles of either side
    uint32_t group;             // inner tiles at a time
    bool inner_rows;            // the inner side is the rows'
    uint32_t whole;             // tiles that one pair makes alone
    uint32_t parts;             // of the others
    uint32_t items;
    uint32_t steps;             // of k
};

// `step_us`: what a step of a tile of 256 columns takes, `least_us` one of few; `step_bytes`: of 256 rows or columns of either operand in a step, the larger.
inline Split make_split(uint32_t m, uint32_t n, uint32_t cols, uint32_t steps, uint32_t min_steps, double step_us, double least_us, uint32_t step_bytes, uint32_t pairs) {
    Split s{};
    s.cols = cols;
    s.steps = steps;
    const uint32_t tiles_m = (m + kPairRows4 - 1) / kPairRows4, tiles_n = (n + cols - 1) / cols, tiles = tiles_m * tiles_n, rest = tiles % pairs;
    s.inner_rows = tiles_m < tiles_n;
    s.inner = std::min(tiles_m, tiles_n);
    s.outer = std::max(tiles_m, tiles_n);
    const uint32_t fit = (uint32_t)std::max<uint64_t>(4, (48ull << 20) / ((uint64_t)step_bytes * steps));  // of the 126 MB of L2
    const uint32_t groups = (s.inner + fit - 1) / fit;
    s.group = (s.inner + groups - 1) / groups;
    // Parts of the last round's tiles: as many as make it shortest, their sums' way through memory and the second launch, some 8 us, counted
    const double tile_us = std::max(least_us, step_us * cols / kPairCols4) * steps, sums_us = (double)rest * kPairRows4 * cols * 8. / 5e6;
    s.parts = 1;
    double best = tile_us;
    for (uint32_t parts = 2; rest && parts <= 32 && parts * min_steps <= steps; ++parts) {
        const double time = tile_us * ((rest * parts + pairs - 1) / pairs) / parts + sums_us * parts + 8.;
        if (time < best) {
            best = time;
            s.parts = parts;
        }
    }
    s.whole = s.parts > 1 ? tiles - rest : tiles;
    s.items = s.whole + (tiles - s.whole) * s.parts;
    return s;
}
inline uint64_t split_workspace(const Split &s) { return (uint64_t)(s.items - s.whole) * kPairRows4 * s.cols * sizeof(float); }

struct Item {
    uint32_t m0, n0, first, last;  // steps [first, last)
    uint32_t slot;                 // of a part, else ~0
};
B200_DEVICE void split_tile(const Split &s, uint32_t tile, uint32_t &m0, uint32_t &n0) {
    const uint32_t of_group = s.group * s.outer, first = tile / of_group * s.group, in_group = tile % of_group, size = min(s.group, s.inner - first);
    const uint32_t inner = first + in_group % size, outer = in_group / size;
    m0 = (s.inner_rows ? inner : outer) * kPairRows4;
    n0 = (s.inner_rows ? outer : inner) * s.cols;
}
B200_DEVICE Item split_item(const Split &s, uint32_t i) {
    Item w{0, 0, 0, s.steps, ~0u};
    uint32_t tile = i;
    if (i >= s.whole) {
        w.slot = i - s.whole;
        tile = s.whole + w.slot / s.parts;
        const uint32_t part = w.slot % s.parts;
        w.first = part * s.steps / s.parts;
        w.last = (part + 1) * s.steps / s.parts;
    }
    split_tile(s, tile, w.m0, w.n0);
    return w;
}

constexpr uint32_t kJoinCols = 8;
// C of the tiles that were cut: the parts' sums in order.  A thread a row and 8 columns: few loads are under way
// in all, and with 32 they were behind one another.
static __global__ void __launch_bounds__(kPairRows4) fp4_join_kernel(const Split s, const float *partial, uint32_t m, uint32_t n, const float *a_whole,
                                                             const float *b_whole, float left, const Target c) {
    ptx::wait_for_grids_before();
    const Factor f(a_whole ? *reinterpret_cast<const volatile float *>(a_whole) : 1.f, b_whole ? *reinterpret_cast<const volatile float *>(b_whole) : left);
    const uint32_t col = blockIdx.y * kJoinCols;
    uint32_t row, n0;
    split_tile(s, s.whole + blockIdx.x, row, n0);
    row += threadIdx.x;
    n0 += col;
    if (row >= m || n0 >= n) return;
    float v[kJoinCols] = {};
    for (uint32_t part = 0; part < s.parts; ++part) {
        const float *src = partial + ((uint64_t)(blockIdx.x * s.parts + part) * s.cols + col) * kPairRows4 + threadIdx.x;
#pragma unroll
        for (uint32_t i = 0; i < kJoinCols; ++i) v[i] += src[i * kPairRows4];
    }
#pragma unroll
    for (uint32_t i = 0; i < kJoinCols; ++i) v[i] = f.apply(v[i]);
    store_row(c, row, n0, n, v);
}

}  // namespace fp4
}  // namespace b200spmm
