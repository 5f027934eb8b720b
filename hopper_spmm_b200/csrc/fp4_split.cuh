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

// Tiles of 256 rows x `cols` columns, side by side before one below the other.
struct Split {
    uint32_t cols;        // of a tile, a multiple of 32
    uint32_t tiles_n;     // tiles side by side
    uint32_t whole;       // tiles that one pair makes alone
    uint32_t parts;       // of the others
    uint32_t items;
    uint32_t steps;       // of k
};

inline Split make_split(uint32_t m, uint32_t n, uint32_t cols, uint32_t steps, uint32_t min_steps, uint32_t pairs) {
    Split s{};
    s.cols = cols;
    s.tiles_n = (n + cols - 1) / cols;
    s.steps = steps;
    const uint32_t tiles = (m + kPairRows4 - 1) / kPairRows4 * s.tiles_n, rest = tiles % pairs;
    s.parts = rest ? std::min(pairs / rest, steps / min_steps) : 1;
    if (s.parts < 2) s.parts = 1;
    s.whole = s.parts > 1 ? tiles - rest : tiles;
    s.items = s.whole + (tiles - s.whole) * s.parts;
    return s;
}
inline uint64_t split_workspace(const Split &s) { return (uint64_t)(s.items - s.whole) * kPairRows4 * s.cols * sizeof(float); }

struct Item {
    uint32_t m0, n0, first, last;  // steps [first, last)
    uint32_t slot;                 // of a part, else ~0
};
B200_DEVICE Item split_item(const Split &s, uint32_t i) {
    uint32_t tile = i, part = 0, parts = 1, slot = ~0u;
    if (i >= s.whole) {
        slot = i - s.whole;
        tile = s.whole + slot / s.parts;
        part = slot % s.parts;
        parts = s.parts;
    }
    if (parts == 1) slot = ~0u;
    return {tile / s.tiles_n * kPairRows4, tile % s.tiles_n * s.cols, part * s.steps / parts, (part + 1) * s.steps / parts, slot};
}

// C of the tiles that were cut: the parts' sums in order.  A thread a row and 32 columns.
static __global__ void __launch_bounds__(kPairRows4) fp4_join_kernel(const Split s, const float *__restrict__ partial, uint32_t m, uint32_t n, const float *__restrict__ a_whole,
                                                             const float *__restrict__ b_whole, float left, const Target c) {
    ptx::wait_for_grids_before();
    const Factor f(a_whole ? *reinterpret_cast<const volatile float *>(a_whole) : 1.f, b_whole ? *reinterpret_cast<const volatile float *>(b_whole) : left);
    const uint32_t tile = s.whole + blockIdx.x, col = blockIdx.y * 32u;
    const uint32_t row = tile / s.tiles_n * kPairRows4 + threadIdx.x, n0 = tile % s.tiles_n * s.cols + col;
    if (row >= m || n0 >= n) return;
    float v[32] = {};
    for (uint32_t part = 0; part < s.parts; ++part) {
        const float *src = partial + ((uint64_t)(blockIdx.x * s.parts + part) * s.cols + col) * kPairRows4 + threadIdx.x;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) v[i] += src[i * kPairRows4];
    }
#pragma unroll
    for (uint32_t i = 0; i < 32; ++i) v[i] = f.apply(v[i]);
    store_row(c, row, n0, n, v);
}

}  // namespace fp4
}  // namespace b200spmm
