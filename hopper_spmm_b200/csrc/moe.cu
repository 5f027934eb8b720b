// A mixture-of-experts layer for a few tokens, in three kernels: logits; routing, gate, up and SiLU; down and the weighted sum.
//
//     y_t = sum over chosen experts e of  share_te  D_e (silu(G_e x_t) * (U_e x_t))
//
// Bound: one read of every chosen expert.  Work is counted in tiles of the chosen experts, one expert's after the other's, and shared out evenly over the SMs, whose blocks multiply
// each tile with all tokens of its expert (narrow.cuh).  A tile of the first product is 8 rows of the gate and the same 8 of up: both values of an inner value
// lie in one warp, and SiLU is taken where the sums are joined.  The second product's results are left for each token and expert; who comes last to 16 rows of
// y adds them up in the order of the token's choices, so that the result is the same whoever that is.  Nobody waits for anybody.
// The routing is cheap and needed by every block: each finds the chosen experts for itself, from the logits, before its first tile.
#include <type_traits>

#include "entry.hpp"
#include "int4.hpp"
#include "launch.hpp"

namespace b200spmm {
namespace narrow {
namespace {

constexpr uint32_t kWarps = 24, kThreads = 32 * kWarps;
constexpr int kRing = 2;
constexpr uint32_t kRingBytes = kRing * kStageBytes, kRingFloats = kRingBytes / 4;
constexpr uint32_t kMaxTokens = 256, kMaxExperts = 1024, kMaxTop = 32;
constexpr uint32_t kMoeSmem = kMaxSmem - 1024;  // beside a few numbers of a block's own
constexpr uint32_t kLogitTokens = 8, kLogitThreads = 128;

struct MoeParams {
    Matrix gate_up, down;
    uint32_t experts, hidden, inner, top, tokens, pairs;
    bool renormalize;
    const void *x, *router;
    int64_t ldx, ld_router, ldy;
    bool x_wide, router_wide;
    void *y;
    bool y_f16;  // else bf16
    const double *logits;  // null: ids are given
    const void *ids_in;
    int id_bytes;
    int32_t *ids;          // [pairs], as used: -1 for none
    float *shares;
    uint32_t *arrived;     // for every 16 rows of y
    float *h;              // [pairs][h_ld]
    uint32_t h_ld;
    float *parts;          // [pairs][hidden]
};

// ------------------------------------------------------------------ logits, in 64 bits: products of 16-bit numbers are exact in fp32, eight of them are added there

template <typename T>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const MoeParams p, double *logits) {
    __shared__ double shared[kLogitThreads / 32][kLogitTokens];
    ptx::wait_for_grids_before();
    const uint32_t e = blockIdx.x, t0 = blockIdx.y * kLogitTokens, n = min(kLogitTokens, p.tokens - t0), lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const Plain<T> w{static_cast<const T *>(p.router) + (int64_t)e * p.ld_router, 1, 0, p.router_wide, p.hidden};
    const Plain<T> x{static_cast<const T *>(p.x) + (int64_t)t0 * p.ldx, 1, p.ldx, p.x_wide, p.hidden};
    double sum[kLogitTokens] = {};
    for (uint32_t u = threadIdx.x; u * 8u < p.hidden; u += kLogitThreads) {
        const uint4 a = w(0, u);
        uint4 b[kLogitTokens];
#pragma unroll
        for (uint32_t j = 0; j < kLogitTokens; ++j)
            if (j < n) b[j] = x(j, u);
#pragma unroll
        for (uint32_t j = 0; j < kLogitTokens; ++j) {
            if (j >= n) break;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(fp4::Elem<T>::to_float(reinterpret_cast<const T *>(&a)[i]), fp4::Elem<T>::to_float(reinterpret_cast<const T *>(&b[j])[i]), s);
            sum[j] += (double)s;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < kLogitTokens; ++j) {
        if (j >= n) break;
        for (int d = 16; d > 0; d >>= 1) sum[j] += __shfl_xor_sync(0xFFFFFFFFu, sum[j], d);
        if (lane == 0) shared[warp][j] = sum[j];
    }
    __syncthreads();
    if (threadIdx.x < n) {
        double s = 0.0;
        for (uint32_t i = 0; i < kLogitThreads / 32; ++i) s += shared[i][threadIdx.x];
        logits[(uint64_t)(t0 + threadIdx.x) * p.experts + e] = s;
    }
}

// ------------------------------------------------------------------ routing

// Larger numbers have larger keys; NaN the largest, and both zeros one.
B200_DEVICE uint64_t key_of(double v) {
    if (v != v) return ~0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// A block's view of the routing, in shared memory.
struct Routing {
    int32_t *ids;       // [pairs]
    uint16_t *active;   // the chosen experts, ascending
    uint16_t *counts;   // of their pairs
    uint16_t *pairs;    // of the expert at hand, ascending
    uint32_t *n_active;
    uint8_t *flags;     // tiles of a round that a block has completed
};
__host__ __device__ inline uint32_t routing_bytes(uint32_t pairs, uint32_t experts) { return (4u * pairs + 4u * experts + 2u * pairs + 16u + 32u + 127u) / 128u * 128u; }
B200_DEVICE Routing routing_at(uint8_t *at, uint32_t pairs, uint32_t experts) {
    Routing r;
    r.ids = reinterpret_cast<int32_t *>(at);
    r.n_active = reinterpret_cast<uint32_t *>(at + 4u * pairs);
    r.flags = at + 4u * pairs + 16u;
    r.active = reinterpret_cast<uint16_t *>(at + 4u * pairs + 48u);
    r.counts = r.active + experts;
    r.pairs = r.counts + experts;
    return r;
}

// One warp: the `top` largest logits of token t, in order; lane j's share of choice j.
B200_DEVICE void choose(const MoeParams &p, uint32_t t, int32_t *ids, bool write) {
    const double *l = p.logits + (uint64_t)t * p.experts;
    const uint32_t lane = threadIdx.x & 31u;
    uint64_t last = 0;
    uint32_t last_at = 0, mine = 0;
    for (uint32_t j = 0; j < p.top; ++j) {
        uint64_t best = 0;
        uint32_t best_at = 0xFFFFFFFFu;
        for (uint32_t e = lane; e < p.experts; e += 32u) {  // the first of the largest that come after the last choice
            const uint64_t k = key_of(l[e]);
            if ((j == 0 || k < last || (k == last && e > last_at)) && (best_at == 0xFFFFFFFFu || k > best)) {
                best = k;
                best_at = e;
            }
        }
        const bool any = best_at != 0xFFFFFFFFu;
        const uint32_t high = __reduce_max_sync(0xFFFFFFFFu, any ? (uint32_t)(best >> 32) : 0u);
        const bool in = any && (uint32_t)(best >> 32) == high;
        const uint32_t low = __reduce_max_sync(0xFFFFFFFFu, in ? (uint32_t)best : 0u);
        last = (uint64_t)high << 32 | low;
        last_at = __reduce_min_sync(0xFFFFFFFFu, in && (uint32_t)best == low ? best_at : 0xFFFFFFFFu);
        if (lane == j) mine = last_at;
    }
    const uint32_t first = __shfl_sync(0xFFFFFFFFu, mine, 0);
    const double most = l[first];
    const bool chosen = lane < p.top;
    const float e = chosen ? expf((float)(l[mine] - most)) : 0.f;
    float sum = e;
    if (!p.renormalize) {
        sum = 0.f;
        for (uint32_t i = lane; i < p.experts; i += 32u) sum += expf((float)(l[i] - most));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (chosen) {
        ids[t * p.top + lane] = (int32_t)mine;
        if (write) {
            p.ids[t * p.top + lane] = (int32_t)mine;
            p.shares[t * p.top + lane] = e / sum;
        }
    }
}

// The chosen experts and how many pairs each has, from the ids in shared memory, by all threads.
B200_DEVICE void find_active(const MoeParams &p, const Routing &r) {
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) {
        uint32_t n = 0;
        for (uint32_t i = 0; i < p.pairs; ++i) n += r.ids[i] == (int32_t)e ? 1u : 0u;
        r.counts[e] = (uint16_t)n;
    }
    __syncthreads();
    if (threadIdx.x < 32u) {
        uint32_t n = 0;
        for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
            const uint32_t e = e0 + threadIdx.x;
            const bool on = e < p.experts && r.counts[e] != 0;
            const uint32_t all = __ballot_sync(0xFFFFFFFFu, on);
            if (on) r.active[n + __popc(all & ((1u << threadIdx.x) - 1u))] = (uint16_t)e;
            n += __popc(all);
        }
        if (threadIdx.x == 0) *r.n_active = n;
    }
    __syncthreads();
}

// The pairs of an expert, ascending, by the first warp; the others wait.
B200_DEVICE void list_pairs(const MoeParams &p, const Routing &r, uint32_t expert) {
    __syncthreads();
    if (threadIdx.x < 32u) {
        uint32_t n = 0;
        for (uint32_t i0 = 0; i0 < p.pairs; i0 += 32u) {
            const uint32_t i = i0 + threadIdx.x;
            const bool on = i < p.pairs && r.ids[i] == (int32_t)expert;
            const uint32_t all = __ballot_sync(0xFFFFFFFFu, on);
            if (on) r.pairs[n + __popc(all & ((1u << threadIdx.x) - 1u))] = (uint16_t)i;
            n += __popc(all);
        }
    }
    __syncthreads();
}

// Tokens of an expert as columns.
template <typename T>
struct Gathered {
    Plain<T> x;
    const uint16_t *pairs;
    uint32_t top;
    B200_DEVICE uint4 operator()(uint32_t j, uint32_t u) const { return x(pairs[j] / top, u); }
};

// A part of a block's work: tiles of one expert.
struct Segment {
    uint32_t expert, n, tile, tiles;
};

// ------------------------------------------------------------------ gate, up, SiLU

template <class W, int kNB>
B200_DEVICE void gate_up_pass(const MoeParams &p, const Segment &g, const Routing &r, uint8_t *smem, uint32_t columns_at, uint32_t columns_bytes, uint32_t j0, uint32_t n) {
    using T = typename W::T;
    const uint32_t base = ptx::smem_u32(smem), warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), row = (threadIdx.x & 31u) >> 2;
    const uint32_t steps = (p.hidden + W::kStep - 1) / W::kStep;
    Columns c{};
    c.base = base + columns_at;
    c.steps = min(steps, (columns_bytes / n - 64u) / 128u * 128u / (W::kUnits * 16u));
    c.pitch = column_pitch<W>(c.steps);
    const Split split(g.tiles, steps, kWarps);
    auto stage = [&](uint32_t first, uint32_t count) {
        stage_columns<W>(Gathered<T>{Plain<T>{static_cast<const T *>(p.x), 1, p.ldx, p.x_wide, p.hidden}, r.pairs + j0, p.top}, c, first, count, n, false);
    };
    bool staged = false;
    for (uint32_t tile0 = 0; tile0 < g.tiles; tile0 += split.at_once) {
        const uint32_t tiles = min(split.at_once, g.tiles - tile0), mine = warp / split.slices;
        const uint32_t i = min((g.tile + tile0 + mine) * 8u + row, p.inner - 1u);
        Share s;
        s.slice = warp % split.slices;
        s.slices = split.slices;
        s.steps = steps;
        s.ring = base + warp * kRingBytes;
        s.busy = mine < tiles;
        s.row_lo = (uint64_t)g.expert * 2u * p.inner + i;
        s.row_hi = s.row_lo + p.inner;
        float sums[kNB][4] = {};
        accumulate<W, kNB, 1, false, kRing>(p.gate_up, s, c, n, staged, stage, sums);
        staged = c.steps >= steps;
        if (s.busy) leave_sums<kNB>(reinterpret_cast<float *>(smem + warp * kRingBytes), sums);
        __syncthreads();
        for (uint32_t k = threadIdx.x; k < tiles * 8u * n; k += kThreads) {
            const uint32_t q = k % 8u, j = k / 8u % n, of = k / (8u * n), at = (g.tile + tile0 + of) * 8u + q;
            const float a = joined(reinterpret_cast<const float *>(smem), kRingFloats, of * split.slices, split.slices, j, q);
            const float b = joined(reinterpret_cast<const float *>(smem), kRingFloats, of * split.slices, split.slices, j, q + 8u);
            if (at < p.inner) p.h[(uint64_t)r.pairs[j0 + j] * p.h_ld + at] = a / (1.f + expf(-a)) * b;
        }
        __syncthreads();
    }
}

template <class W>
__global__ void __launch_bounds__(kThreads, 1) gate_up_kernel(const MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const Routing r = routing_at(smem + kWarps * kRingBytes, p.pairs, p.experts);
    const uint32_t columns_at = kWarps * kRingBytes + routing_bytes(p.pairs, p.experts), columns_bytes = kMoeSmem - columns_at;
    ptx::wait_for_grids_before();
    const bool write = blockIdx.x == 0;
    if (p.logits) {
        for (uint32_t t = threadIdx.x >> 5; t < p.tokens; t += kWarps) choose(p, t, r.ids, write);
    } else {
        for (uint32_t i = threadIdx.x; i < p.pairs; i += kThreads) {
            const int64_t e = p.id_bytes == 8 ? static_cast<const int64_t *>(p.ids_in)[i] : static_cast<const int32_t *>(p.ids_in)[i];
            const int32_t id = e >= 0 && e < (int64_t)p.experts ? (int32_t)e : -1;
            r.ids[i] = id;
            if (write) p.ids[i] = id;
        }
    }
    if (write)
        for (uint32_t i = threadIdx.x; i < (p.hidden + kTileRows - 1u) / kTileRows; i += kThreads) p.arrived[i] = 0;
    find_active(p, r);
    const uint32_t of_expert = (p.inner + 7u) / 8u, all = *r.n_active * of_expert;
    const uint32_t end = (uint32_t)((uint64_t)all * (blockIdx.x + 1u) / gridDim.x);
    for (uint32_t at = (uint32_t)((uint64_t)all * blockIdx.x / gridDim.x); at < end;) {
        Segment g;
        g.expert = r.active[at / of_expert];
        g.n = r.counts[g.expert];
        g.tile = at % of_expert;
        g.tiles = min(end - at, of_expert - g.tile);
        list_pairs(p, r, g.expert);
        for (uint32_t j0 = 0; j0 < g.n; j0 += 16u) {
            const uint32_t n = min(16u, g.n - j0);
            if (n <= 8u) gate_up_pass<W, 1>(p, g, r, smem, columns_at, columns_bytes, j0, n);
            else gate_up_pass<W, 2>(p, g, r, smem, columns_at, columns_bytes, j0, n);
        }
        at += g.tiles;
    }
}

// ------------------------------------------------------------------ down and the sum

// Inner values as a sum of two 16-bit numbers, the second what the first leaves over: fp16 has 22 digits that way, bf16 16.  fp16 gets them scaled by a power of two that takes
// the pair's largest to [2^14, 2^15).
template <typename T>
struct Halves {
    const float *h;
    const uint16_t *pairs;
    const float *scale;  // of column j; null: 1
    uint32_t ld, k;
    B200_DEVICE void operator()(uint32_t j, uint32_t u, uint4 *high, uint4 *low) const {
        const float *from = h + (uint64_t)pairs[j] * ld + u * 8u, by = scale ? scale[j] : 1.f;
        alignas(16) float v[8];
        reinterpret_cast<float4 *>(v)[0] = reinterpret_cast<const float4 *>(from)[0];
        reinterpret_cast<float4 *>(v)[1] = reinterpret_cast<const float4 *>(from)[1];
        alignas(16) T a[8], b[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const float x = u * 8u + e < k ? v[e] * by : 0.f;
            a[e] = fp4::Elem<T>::from_float(x);
            const float rest = x - fp4::Elem<T>::to_float(a[e]);
            b[e] = fp4::Elem<T>::from_float(fabsf(rest) <= 3.0e38f ? rest : 0.f);  // (an infinity or NaN is the first number's)
        }
        *high = *reinterpret_cast<const uint4 *>(a);
        *low = *reinterpret_cast<const uint4 *>(b);
    }
};

template <class W, int kNB>
B200_DEVICE void down_pass(const MoeParams &p, const Segment &g, const Routing &r, uint8_t *smem, uint32_t columns_at, uint32_t columns_bytes, float *scales, uint32_t j0, uint32_t n, bool last) {
    using T = typename W::T;
    constexpr bool kScale = std::is_same<T, __half>::value;
    const uint32_t base = ptx::smem_u32(smem), warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u, row = lane >> 2;
    const uint32_t steps = (p.inner + W::kStep - 1) / W::kStep;
    Columns c{};
    c.base = base + columns_at;
    c.steps = min(steps, (columns_bytes / (2u * n) - 64u) / 128u * 128u / (W::kUnits * 16u));
    c.pitch = column_pitch<W>(c.steps);
    c.plane = n * c.pitch;
    if constexpr (kScale) {
        for (uint32_t j = warp; j < n; j += kWarps) {
            const float *h = p.h + (uint64_t)r.pairs[j0 + j] * p.h_ld;
            uint32_t top = 0;
            for (uint32_t i = lane; i < p.inner; i += 32u) {
                const uint32_t b = __float_as_uint(h[i]) & 0x7FFFFFFFu;
                if (b < fp4::kInfBits) top = max(top, b);
            }
            top = __reduce_max_sync(0xFFFFFFFFu, top);
            if (lane == 0) scales[j] = fp4::exp2_int(max(-126, min(126, 14 - ((int)(top >> 23) - 127))));
        }
        __syncthreads();
    }
    const Split split(g.tiles, steps, kWarps);
    auto stage = [&](uint32_t first, uint32_t count) {
        const Halves<T> from{p.h, r.pairs + j0, kScale ? scales : nullptr, p.h_ld, p.inner};
        const uint32_t units = count * W::kUnits, have = (p.inner + 7u) / 8u, u0 = first * W::kUnits;
        for (uint32_t i = threadIdx.x; i < n * units; i += kThreads) {
            const uint32_t j = i / units, u = i - j * units, to = c.base + j * c.pitch + unit_place<W>(u) * 16u;
            uint4 high = make_uint4(0u, 0u, 0u, 0u), low = high;
            if (u0 + u < have) from(j, u0 + u, &high, &low);
            ptx::st_shared_v4(to, unit_order<W>(high));
            ptx::st_shared_v4(to + c.plane, unit_order<W>(low));
        }
    };
    bool staged = false;
    for (uint32_t tile0 = 0; tile0 < g.tiles; tile0 += split.at_once) {
        const uint32_t tiles = min(split.at_once, g.tiles - tile0), mine = warp / split.slices;
        Share s;
        s.slice = warp % split.slices;
        s.slices = split.slices;
        s.steps = steps;
        s.ring = base + warp * kRingBytes;
        s.busy = mine < tiles;
        s.row_lo = (uint64_t)g.expert * p.hidden + min((g.tile + tile0 + mine) * kTileRows + row, p.hidden - 1u);
        s.row_hi = (uint64_t)g.expert * p.hidden + min((g.tile + tile0 + mine) * kTileRows + row + 8u, p.hidden - 1u);
        float sums[kNB][4] = {};
        accumulate<W, kNB, 2, false, kRing>(p.down, s, c, n, staged, stage, sums);
        staged = c.steps >= steps;
        if (s.busy) leave_sums<kNB>(reinterpret_cast<float *>(smem + warp * kRingBytes), sums);
        __syncthreads();
        for (uint32_t k = threadIdx.x; k < tiles * kTileRows * n; k += kThreads) {
            const uint32_t q = k % kTileRows, j = k / kTileRows % n, of = k / (kTileRows * n), at = (g.tile + tile0 + of) * kTileRows + q;
            float v = joined(reinterpret_cast<const float *>(smem), kRingFloats, of * split.slices, split.slices, j, q);
            if constexpr (kScale) v = v / scales[j];
            if (at < p.hidden) p.parts[(uint64_t)r.pairs[j0 + j] * p.hidden + at] = v;
        }
        if (!last) {
            __syncthreads();
            continue;
        }
        // What this block left of these rows is there before its arrival is; who sees all the others' adds up.
        __threadfence();
        __syncthreads();
        if (threadIdx.x < tiles) r.flags[threadIdx.x] = atomicAdd(p.arrived + g.tile + tile0 + threadIdx.x, 1u) + 1u == *r.n_active;
        __threadfence();
        __syncthreads();
        for (uint32_t of = 0; of < tiles; ++of) {
            if (!r.flags[of]) continue;
            for (uint32_t k = threadIdx.x; k < kTileRows * p.tokens; k += kThreads) {
                const uint32_t at = (g.tile + tile0 + of) * kTileRows + k % kTileRows, t = k / kTileRows;
                if (at >= p.hidden) continue;
                float v = 0.f;
                for (uint32_t i = t * p.top; i < (t + 1u) * p.top; ++i)
                    if (r.ids[i] >= 0) v = fmaf(p.shares[i], __ldcg(p.parts + (uint64_t)i * p.hidden + at), v);
                static_cast<uint16_t *>(p.y)[(int64_t)t * p.ldy + at] = p.y_f16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
            }
        }
        __syncthreads();
    }
}

template <class W>
__global__ void __launch_bounds__(kThreads, 1) down_kernel(const MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float scales[16];
    const Routing r = routing_at(smem + kWarps * kRingBytes, p.pairs, p.experts);
    const uint32_t columns_at = kWarps * kRingBytes + routing_bytes(p.pairs, p.experts), columns_bytes = kMoeSmem - columns_at;
    ptx::wait_for_grids_before();
    for (uint32_t i = threadIdx.x; i < p.pairs; i += kThreads) r.ids[i] = p.ids[i];
    find_active(p, r);
    const uint32_t of_expert = (p.hidden + kTileRows - 1u) / kTileRows, all = *r.n_active * of_expert;
    if (all == 0) {  // nobody was chosen
        for (uint32_t t = blockIdx.x; t < p.tokens; t += gridDim.x)
            for (uint32_t i = threadIdx.x; i < p.hidden; i += kThreads) static_cast<uint16_t *>(p.y)[(int64_t)t * p.ldy + i] = 0;
        return;
    }
    const uint32_t end = (uint32_t)((uint64_t)all * (blockIdx.x + 1u) / gridDim.x);
    for (uint32_t at = (uint32_t)((uint64_t)all * blockIdx.x / gridDim.x); at < end;) {
        Segment g;
        g.expert = r.active[at / of_expert];
        g.n = r.counts[g.expert];
        g.tile = at % of_expert;
        g.tiles = min(end - at, of_expert - g.tile);
        list_pairs(p, r, g.expert);
        for (uint32_t j0 = 0; j0 < g.n; j0 += 16u) {
            const uint32_t n = min(16u, g.n - j0);
            if (n <= 8u) down_pass<W, 1>(p, g, r, smem, columns_at, columns_bytes, scales, j0, n, j0 + n == g.n);
            else down_pass<W, 2>(p, g, r, smem, columns_at, columns_bytes, scales, j0, n, j0 + n == g.n);
        }
        at += g.tiles;
    }
}

// ------------------------------------------------------------------ launches

// Where the parts of the workspace begin.
struct Layout {
    uint64_t logits, ids, shares, arrived, h, parts, bytes;
    uint32_t h_ld;
};
Layout layout_of(const b200spmm_moe_t *m, uint64_t tokens) {
    Layout l{};
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at = (at + bytes + 255) / 256 * 256;
        return here;
    };
    const uint64_t pairs = tokens * (uint64_t)m->top_k;
    l.h_ld = (uint32_t)((m->inner + 7) / 8 * 8);
    l.logits = take(tokens * m->experts * 8);
    l.ids = take(pairs * 4);
    l.shares = take(pairs * 4);
    l.arrived = take((m->hidden + kTileRows - 1) / kTileRows * 4);
    l.h = take(pairs * l.h_ld * 4);
    l.parts = take(pairs * m->hidden * 4);
    l.bytes = at;
    return l;
}

int check_moe(const b200spmm_moe_t *m) {
    if (!m || (m->dtype != B200SPMM_T_F16 && m->dtype != B200SPMM_T_BF16)) return B200SPMM_ERR_INVALID_ARG;
    if (m->experts == 0 || m->hidden == 0 || m->inner == 0 || m->top_k < 1) return B200SPMM_ERR_INVALID_ARG;
    if (m->experts > kMaxExperts || m->top_k > (int32_t)kMaxTop || m->hidden > 0x1000000ull || m->inner > 0x1000000ull) return B200SPMM_ERR_UNSUPPORTED;
    const uint64_t rows[2] = {m->experts * 2 * m->inner, m->experts * m->hidden}, cols[2] = {m->hidden, m->inner};
    const b200spmm_int4_t *codes[2] = {m->gate_up, m->down};
    const void *plain[2] = {m->gate_up_16, m->down_16};
    const int64_t ld[2] = {m->ld_gate_up, m->ld_down};
    if ((codes[0] != nullptr) != (codes[1] != nullptr)) return B200SPMM_ERR_INVALID_ARG;
    for (int i = 0; i < 2; ++i) {
        if ((codes[i] != nullptr) == (plain[i] != nullptr)) return B200SPMM_ERR_INVALID_ARG;
        if (codes[i]) {
            const int st = check_int4(codes[i]);
            if (st != B200SPMM_OK) return st;
            if (codes[i]->rows != rows[i] || codes[i]->cols != cols[i] || codes[i]->device != m->device) return B200SPMM_ERR_INVALID_ARG;
        } else {
            if (ld[i] < (int64_t)cols[i]) return B200SPMM_ERR_INVALID_ARG;
            if (ld[i] % 8 != 0 || !fp4::aligned(plain[i], 16)) return B200SPMM_ERR_UNSUPPORTED;
        }
    }
    return B200SPMM_OK;
}

Matrix plain_matrix(const void *values, int64_t ld, uint64_t cols) {
    Matrix out{};
    out.values = static_cast<const uint8_t *>(values);
    out.pitch = (uint64_t)ld * 2;
    out.row_bytes = (uint32_t)cols * 2u;
    return out;
}

template <class W>
int launch_gate_up(const MoeParams &p, uint32_t blocks, cudaStream_t stream) {
    static std::atomic<uint64_t> allowed{0};
    B200_CUDA_TRY(allow_smem(gate_up_kernel<W>, allowed, kMoeSmem));
    B200_CUDA_TRY(launch_after(gate_up_kernel<W>, dim3(blocks), kThreads, kMoeSmem, 1, stream, p));
    return B200SPMM_OK;
}
template <class W>
int launch_down(const MoeParams &p, uint32_t blocks, cudaStream_t stream) {
    static std::atomic<uint64_t> allowed{0};
    B200_CUDA_TRY(allow_smem(down_kernel<W>, allowed, kMoeSmem));
    B200_CUDA_TRY(launch_after(down_kernel<W>, dim3(blocks), kThreads, kMoeSmem, 1, stream, p));
    return B200SPMM_OK;
}

template <typename T>
int launch_moe(const b200spmm_moe_t *m, const MoeParams &p, double *logits, cudaStream_t stream) {
    if (logits) {
        B200_CUDA_TRY(launch_after(logits_kernel<T>, dim3(p.experts, (p.tokens + kLogitTokens - 1) / kLogitTokens), kLogitThreads, 0, 1, stream, p, logits));
    }
    const uint64_t most = std::min<uint64_t>(p.experts, p.pairs);  // experts that may be chosen
    auto blocks = [&](uint32_t tiles) { return (uint32_t)std::min<uint64_t>(fp4::sm_count(), most * tiles); };
    const uint32_t up = blocks((p.inner + 7) / 8), down = blocks((p.hidden + kTileRows - 1) / kTileRows);
    int st;
    if (m->gate_up) {
        const uint32_t a = span_of(m->gate_up), b = span_of(m->down);
        st = a == 32 ? launch_gate_up<Weights<T, 32>>(p, up, stream) : a == 64 ? launch_gate_up<Weights<T, 64>>(p, up, stream) : launch_gate_up<Weights<T, 128>>(p, up, stream);
        if (st != B200SPMM_OK) return st;
        // bf16 for its range: inner values are as large as they are, and codes are exact in either type
        using B = __nv_bfloat16;
        return b == 32 ? launch_down<Weights<B, 32>>(p, down, stream) : b == 64 ? launch_down<Weights<B, 64>>(p, down, stream) : launch_down<Weights<B, 128>>(p, down, stream);
    }
    st = launch_gate_up<Weights<T, 0>>(p, up, stream);
    return st != B200SPMM_OK ? st : launch_down<Weights<T, 0>>(p, down, stream);
}

// ids null: they are found from the logits, and left, with the shares, at out_ids and out_shares where those are wanted.
int run_moe(const b200spmm_moe_t *m, const void *x, int64_t ldx, int64_t tokens, const void *ids, int id_bytes, const float *shares, void *y, int64_t ldy, int32_t *out_ids,
            float *out_shares, void *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
    const Layout l = layout_of(m, (uint64_t)tokens);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    MoeParams p{};
    p.gate_up = m->gate_up ? matrix_of(m->gate_up) : plain_matrix(m->gate_up_16, m->ld_gate_up, m->hidden);
    p.down = m->down ? matrix_of(m->down) : plain_matrix(m->down_16, m->ld_down, m->inner);
    p.experts = (uint32_t)m->experts;
    p.hidden = (uint32_t)m->hidden;
    p.inner = (uint32_t)m->inner;
    p.top = (uint32_t)m->top_k;
    p.tokens = (uint32_t)tokens;
    p.pairs = p.tokens * p.top;
    p.renormalize = m->renormalize != 0;
    p.x = x;
    p.ldx = ldx;
    p.x_wide = fp4::aligned(x, 16) && (tokens == 1 || ldx % 8 == 0);
    p.router = m->router;
    p.ld_router = m->ld_router;
    p.router_wide = fp4::aligned(m->router, 16) && (m->experts == 1 || m->ld_router % 8 == 0);
    p.y = y;
    p.ldy = ldy;
    p.y_f16 = m->dtype == B200SPMM_T_F16;
    double *logits = ids ? nullptr : reinterpret_cast<double *>(ws + l.logits);
    p.logits = logits;
    p.ids_in = ids;
    p.id_bytes = id_bytes;
    p.ids = out_ids ? out_ids : reinterpret_cast<int32_t *>(ws + l.ids);
    p.shares = shares ? const_cast<float *>(shares) : out_shares ? out_shares : reinterpret_cast<float *>(ws + l.shares);  // (given ones are only read)
    p.arrived = reinterpret_cast<uint32_t *>(ws + l.arrived);
    p.h = reinterpret_cast<float *>(ws + l.h);
    p.h_ld = l.h_ld;
    p.parts = reinterpret_cast<float *>(ws + l.parts);
    return m->dtype == B200SPMM_T_F16 ? launch_moe<__half>(m, p, logits, stream) : launch_moe<__nv_bfloat16>(m, p, logits, stream);
}

// Checks that both calls make.
int check_call(const b200spmm_moe_t *m, const void *x, int64_t ldx, int64_t tokens, void *y, int64_t ldy, const void *workspace, uint64_t workspace_bytes) {
    int st = check_moe(m);
    if (st != B200SPMM_OK) return st;
    if (tokens < 0) return B200SPMM_ERR_INVALID_ARG;
    if (tokens > kMaxTokens) return B200SPMM_ERR_UNSUPPORTED;
    st = fp4::check_dense(x, m->dtype, (uint64_t)tokens, m->hidden, ldx);
    if (st == B200SPMM_OK) st = fp4::check_dense(y, m->dtype, (uint64_t)tokens, m->hidden, ldy);
    if (st != B200SPMM_OK) return st;
    if (tokens > 0 && (!workspace || !fp4::aligned(workspace, 16) || workspace_bytes < layout_of(m, (uint64_t)tokens).bytes)) return B200SPMM_ERR_INVALID_ARG;
    return B200SPMM_OK;
}

}  // namespace
}  // namespace narrow
}  // namespace b200spmm

using namespace b200spmm;

extern "C" {

int b200spmm_moe_workspace(const b200spmm_moe_t *m, int64_t tokens, uint64_t *bytes) {
    if (!bytes || tokens < 0) return B200SPMM_ERR_INVALID_ARG;
    *bytes = 0;
    const int st = narrow::check_moe(m);
    if (st != B200SPMM_OK) return st;
    if (tokens > narrow::kMaxTokens) return B200SPMM_ERR_UNSUPPORTED;
    *bytes = narrow::layout_of(m, (uint64_t)tokens).bytes;
    return B200SPMM_OK;
}

int b200spmm_moe(const b200spmm_moe_t *m, const void *d_x, int64_t ldx, int64_t tokens, void *d_y, int64_t ldy, int32_t *d_ids, float *d_shares, void *workspace,
                 uint64_t workspace_bytes, void *stream) {
    const int st = narrow::check_call(m, d_x, ldx, tokens, d_y, ldy, workspace, workspace_bytes);
    if (st != B200SPMM_OK) return st;
    if (!m->router || !fp4::aligned(m->router, 2) || m->ld_router < (int64_t)m->hidden || m->top_k > (int64_t)m->experts) return B200SPMM_ERR_INVALID_ARG;
    if (!fp4::aligned(d_ids, 4) || !fp4::aligned(d_shares, 4)) return B200SPMM_ERR_INVALID_ARG;
    return fp4::on_device(m->device, [&]() -> int {
        if (tokens == 0) return B200SPMM_OK;
        return narrow::run_moe(m, d_x, ldx, tokens, nullptr, 0, nullptr, d_y, ldy, d_ids, d_shares, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
    });
}

int b200spmm_moe_experts(const b200spmm_moe_t *m, const void *d_x, int64_t ldx, int64_t tokens, const void *d_ids, int id_bytes, const float *d_shares, void *d_y,
                         int64_t ldy, void *workspace, uint64_t workspace_bytes, void *stream) {
    const int st = narrow::check_call(m, d_x, ldx, tokens, d_y, ldy, workspace, workspace_bytes);
    if (st != B200SPMM_OK) return st;
    if (id_bytes != 4 && id_bytes != 8) return B200SPMM_ERR_INVALID_ARG;
    if (tokens > 0 && (!d_ids || !d_shares || !fp4::aligned(d_ids, id_bytes) || !fp4::aligned(d_shares, 4))) return B200SPMM_ERR_INVALID_ARG;
    return fp4::on_device(m->device, [&]() -> int {
        if (tokens == 0) return B200SPMM_OK;
        return narrow::run_moe(m, d_x, ldx, tokens, d_ids, id_bytes, d_shares, d_y, ldy, nullptr, nullptr, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
