// A mixture-of-experts layer for a few tokens: logits; routing, gate, up and SiLU; down; the weighted sum.
//
//     y_t = sum over chosen experts e of  share_te  D_e (silu(G_e x_t) * (U_e x_t))
//
// Bound: one read of every chosen expert.  The pairs of a token and a choice, sorted by expert and cut into runs of up to 16, are what an expert's tiles are multiplied with; the
// tiles of all runs, one run's after the other's, are shared out evenly over the SMs, whose warps take a tile each, or a part of one, and run ahead into the next
// (narrow.cuh).  A tile of the first product is 8 rows of the gate and the same 8 of up: both values of an inner value lie in one lane.  The second product's results are
// left for each pair; a last kernel adds them up in the order of the token's choices.
// The routing is cheap and needed by every block: each finds the runs for itself, from the logits, before its first tile.
//
// One token, 8 of 64 experts of 2048 x 1024 in bf16, 101 MB: 37 us for 15.4 at a copy's rate.  The experts' bytes come at 6.5 to 7 TB/s; the rest is what stands before them: four
// launches, logits 3 us, the choice and its runs 5, the first copies 2 to 4.  Much of that is waiting for instructions that are run once and that the weights have pushed out of L2.
// 8 tokens through 64 experts of 4096 x 2048 in 4 bits, 554 MB: 157 us for 85; 32 through 128, 1.1 GB: 305 for 172: the instructions that a step of codes takes, as in int4.cu, and
// in the second product two numbers for each inner value (with one of 11 digits, 146 us for the 157).  Times of a captured loop; a call from Python takes the host 5 us or more.
#include <type_traits>

#include "entry.hpp"
#include "int4.hpp"
#include "launch.hpp"

namespace b200spmm {
namespace narrow {
namespace {

// With 16, 20 and 24 warps: one token in bf16 36.9, 36.9 and 37.8 us, 16 of them 147, 144 and 148; 8 with experts in 4 bits 160, 157 and 161, 32 through 128 experts 297, 305 and 315.
constexpr uint32_t kWarps = 20, kThreads = 32 * kWarps;
constexpr uint32_t kRun = 16;  // columns that a tile meets at once, at most
template <class W>
constexpr int kRing = 2 * W::kPieces;  // stages of a warp: two steps
template <class W>
constexpr uint32_t kRingBytes = kRingOf<W, 2, kRing<W>>;
constexpr int kHalves = 2;  // numbers that an inner value is the sum of
constexpr uint32_t kMaxTokens = 256, kMaxExperts = 1024, kMaxTop = 32;
constexpr uint32_t kLogitTokens = 4, kLogitThreads = 256;

struct MoeParams {
    Matrix gate_up, down;
    uint32_t experts, hidden, inner, top, tokens, pairs;
    bool all_tokens;  // are columns of the first product, in all blocks
    uint32_t run, up_columns, down_columns;  // columns of a run, and that a block has room for as a whole, in either product
    uint4 *routing;  // as the first blocks found it
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
    float *h;              // [pairs][h_ld]
    uint32_t h_ld;
    float *parts;          // [pairs][hidden]
};

// ------------------------------------------------------------------ logits, in 64 bits: products of 16-bit numbers are exact there, and beyond fp32's range (in fp32, eight at a time, a small
// term beside two large ones that cancel was lost, and the experts whose logits it told apart were exchanged; bf16's largest products were infinite)

template <typename T>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const MoeParams p, double *logits) {
    __shared__ double shared[kLogitThreads / 32][kLogitTokens];
    ptx::wait_for_grids_before();
    const uint32_t e = blockIdx.x, t0 = blockIdx.y * kLogitTokens, n = min(kLogitTokens, p.tokens - t0), lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const Plain<T> w{static_cast<const T *>(p.router) + (int64_t)e * p.ld_router, 1, 0, p.router_wide, false, p.hidden};
    const Plain<T> x{static_cast<const T *>(p.x) + (int64_t)t0 * p.ldx, 1, p.ldx, p.x_wide, false, p.hidden};
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
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[j] = fma((double)fp4::Elem<T>::to_float(reinterpret_cast<const T *>(&a)[i]), (double)fp4::Elem<T>::to_float(reinterpret_cast<const T *>(&b[j])[i]), sum[j]);
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
    uint16_t *pairs;    // [pairs] by expert, ascending
    uint16_t *starts;   // [experts + 1]: of an expert's pairs
    uint16_t *ranks;    // [pairs] among its expert's
    uint32_t *runs;     // expert << 16 | first of its pairs
    uint32_t *n_runs;
};
// (an expert with n pairs has at most n runs)
__host__ __device__ constexpr uint32_t routing_bytes(uint32_t pairs, uint32_t experts) { return (12u * pairs + 2u * experts + 2u + 16u + 127u) / 128u * 128u; }
B200_DEVICE Routing routing_at(uint8_t *at, uint32_t pairs, uint32_t experts) {
    Routing r;
    r.n_runs = reinterpret_cast<uint32_t *>(at);
    r.ids = reinterpret_cast<int32_t *>(at + 16u);
    r.runs = reinterpret_cast<uint32_t *>(r.ids + pairs);
    r.pairs = reinterpret_cast<uint16_t *>(r.runs + pairs);
    r.ranks = r.pairs + pairs;
    r.starts = r.ranks + pairs;
    return r;
}

B200_DEVICE double value_of(uint64_t key) { return __longlong_as_double((long long)(key >> 63 ? key ^ 1ull << 63 : ~key)); }

// One warp: the `top` largest logits of token t, in order; lane j's share of choice j.  Up to 32 kKeys experts, whose keys a lane keeps (0: none, or taken).
template <int kKeys>
B200_DEVICE void choose_of(const MoeParams &p, uint32_t t, int32_t *ids, bool write) {
    const double *l = p.logits + (uint64_t)t * p.experts;
    const uint32_t lane = threadIdx.x & 31u;
    uint64_t keys[kKeys], mine = 0, most = 0;
    uint32_t mine_at = 0;
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)kKeys; ++i) keys[i] = lane + 32u * i < p.experts ? key_of(l[lane + 32u * i]) : 0ull;
    float sum = 0.f;
    for (uint32_t j = 0; j < p.top; ++j) {
        uint64_t best = 0;
        uint32_t best_at = lane;
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)kKeys; ++i)
            if (keys[i] > best) {
                best = keys[i];
                best_at = lane + 32u * i;
            }
        const uint32_t high = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(best >> 32));
        const uint32_t low = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(best >> 32) == high ? (uint32_t)best : 0u);
        const uint64_t key = (uint64_t)high << 32 | low;
        const uint32_t at = __reduce_min_sync(0xFFFFFFFFu, best == key ? best_at : 0xFFFFFFFFu);  // (of equal ones the first)
        if (j == 0) {
            most = key;
            if (!p.renormalize)
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)kKeys; ++i)
                    if (keys[i]) sum += expf((float)(value_of(keys[i]) - value_of(most)));
        }
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)kKeys; ++i)
            if (at == lane + 32u * i) keys[i] = 0;
        if (lane == j) {
            mine = key;
            mine_at = at;
        }
    }
    const bool chosen = lane < p.top;
    const float e = chosen ? expf((float)(value_of(mine) - value_of(most))) : 0.f;
    if (p.renormalize) sum = e;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (chosen) {
        ids[t * p.top + lane] = (int32_t)mine_at;
        if (write) {
            p.ids[t * p.top + lane] = (int32_t)mine_at;
            p.shares[t * p.top + lane] = e / sum;
        }
    }
}
// The same for up to 128 experts, from how many keys are before each: all compared with all, without a round that waits for the last.  `keys`: shared memory of the warp.
template <int kKeys>
B200_DEVICE void choose_by_rank(const MoeParams &p, uint32_t t, int32_t *ids, bool write, uint64_t *keys) {
    const double *l = p.logits + (uint64_t)t * p.experts;
    const uint32_t lane = threadIdx.x & 31u;
    uint64_t mine[kKeys], most = 0;
    uint32_t rank[kKeys] = {};
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)kKeys; ++i) {
        mine[i] = lane + 32u * i < p.experts ? key_of(l[lane + 32u * i]) : 0ull;
        if (lane + 32u * i < p.experts) keys[lane + 32u * i] = mine[i];
    }
    __syncwarp();
#pragma unroll 4
    for (uint32_t e = 0; e < p.experts; ++e) {
        const uint64_t k = keys[e];
        most = k > most ? k : most;
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)kKeys; ++i) rank[i] += k > mine[i] || (k == mine[i] && e < lane + 32u * i) ? 1u : 0u;
    }
    float part[kKeys], sum = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)kKeys; ++i) {
        const bool chosen = mine[i] && rank[i] < p.top;
        part[i] = mine[i] && (chosen || !p.renormalize) ? expf((float)(value_of(mine[i]) - value_of(most))) : 0.f;
        sum += part[i];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)kKeys; ++i) {
        if (!mine[i] || rank[i] >= p.top) continue;
        ids[t * p.top + rank[i]] = (int32_t)(lane + 32u * i);
        if (write) {
            p.ids[t * p.top + rank[i]] = (int32_t)(lane + 32u * i);
            p.shares[t * p.top + rank[i]] = part[i] / sum;
        }
    }
    __syncwarp();
}
B200_DEVICE void choose(const MoeParams &p, uint32_t t, int32_t *ids, bool write, uint64_t *keys) {
    if (p.experts <= 64u) choose_by_rank<2>(p, t, ids, write, keys);
    else if (p.experts <= 128u) choose_by_rank<4>(p, t, ids, write, keys);
    else if (p.experts <= 256u) choose_of<8>(p, t, ids, write);
    else choose_of<32>(p, t, ids, write);
}

// The runs, of up to `most` pairs, from the ids in shared memory, by all threads.
B200_DEVICE void find_runs(const MoeParams &p, const Routing &r, uint32_t most) {
    for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) r.starts[e] = 0;
    __syncthreads();
    if (threadIdx.x < 32u) {
        const uint32_t lane = threadIdx.x;
        // how many pairs of its expert come before each, 32 pairs at a time, and so how many each expert has
        for (uint32_t i0 = 0; i0 < p.pairs; i0 += 32u) {
            const int32_t id = i0 + lane < p.pairs ? r.ids[i0 + lane] : -1;
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, id), before = __popc(same & ((1u << lane) - 1u));
            const uint32_t n = id >= 0 ? r.starts[id] : 0u;
            __syncwarp();
            if (id >= 0) {
                r.ranks[i0 + lane] = (uint16_t)(n + before);
                if (before == 0) r.starts[id] = (uint16_t)(n + __popc(same));
            }
            __syncwarp();
        }
        // the starts in place of the numbers, and the runs
        uint32_t pairs = 0, runs = 0;
        for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
            const uint32_t e = e0 + lane, n = e < p.experts ? r.starts[e] : 0u, m = (n + most - 1u) / most;
            uint32_t both_to = n << 16 | m;  // up to this one (at most 8,192 of either)
#pragma unroll 1
            for (uint32_t d = 1; d < 32u; d *= 2u) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, both_to, d);
                if (lane >= d) both_to += v;
            }
            const uint32_t start = pairs + (both_to >> 16) - n, run = runs + (both_to & 0xFFFFu) - m;
            if (e < p.experts) r.starts[e] = (uint16_t)start;
            for (uint32_t i = 0; i < m; ++i) r.runs[run + i] = e << 16 | (start + i * most);
            const uint32_t all = __shfl_sync(0xFFFFFFFFu, both_to, 31);
            pairs += all >> 16;
            runs += all & 0xFFFFu;
        }
        if (lane == 0) {
            r.starts[p.experts] = (uint16_t)pairs;
            *r.n_runs = runs;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.pairs; i += kThreads)
        if (r.ids[i] >= 0) r.pairs[r.starts[r.ids[i]] + r.ranks[i]] = (uint16_t)i;
    __syncthreads();
}
B200_DEVICE uint32_t run_expert(const Routing &r, uint32_t run) { return r.runs[run] >> 16; }
B200_DEVICE uint32_t run_start(const Routing &r, uint32_t run) { return r.runs[run] & 0xFFFFu; }
B200_DEVICE uint32_t run_end(const Routing &r, uint32_t run) {  // (the last one ends with its expert's pairs)
    return run + 1u < *r.n_runs ? run_start(r, run + 1u) : r.starts[run_expert(r, run) + 1u];
}

// A block's share of `of_run` tiles of every run, in parts whose columns have room, or of a single run: part(first, end, first run's pairs, how many, the longest run's).
template <class Part>
B200_DEVICE void each_part(const Routing &r, uint32_t of_run, uint32_t room, Part &&part) {
    const uint32_t all = *r.n_runs * of_run, end = (uint32_t)((uint64_t)all * (blockIdx.x + 1u) / gridDim.x);
    for (uint32_t at = (uint32_t)((uint64_t)all * blockIdx.x / gridDim.x); at < end;) {
        const uint32_t run0 = at / of_run, pair0 = run_start(r, run0);
        uint32_t run = run0, longest = 0;
        while (run * of_run < end && run < *r.n_runs && (run == run0 || run_end(r, run) - pair0 <= room)) {
            longest = max(longest, run_end(r, run) - run_start(r, run));
            ++run;
        }
        const uint32_t to = min(end, run * of_run);
        part(at, to, pair0, run_end(r, run - 1u) - pair0, longest);
        at = to;
        __syncthreads();  // (the columns and the rings are free again)
    }
}

// What a tile of a run is.
struct Place {
    uint32_t tile, expert, start, n;  // of the run; its expert and pairs
};
B200_DEVICE Place place_in(const Routing &r, uint32_t of_run, uint32_t tile) {
    const uint32_t run = tile / of_run, start = run_start(r, run);
    return {tile - run * of_run, run_expert(r, run), start, run_end(r, run) - start};
}

// Tokens of pairs as columns.
template <typename T>
struct Gathered {
    Plain<T> x;
    const uint16_t *pairs;
    uint32_t top;
    B200_DEVICE uint4 operator()(uint32_t j, uint32_t u) const { return x(pairs[j] / top, u); }
};

// Columns that become fp16 are scaled by a power of two that takes their largest number to [2^14, 2^15): what lies more than 2^31 below it loses digits.
B200_DEVICE int power_of(uint32_t top) { return max(-126, min(126, 14 - ((int)(top >> 23) - 127))); }

// The largest finite |.| of n columns, as fp32's bits, by all threads: top_of(j, u) is that of unit u of column j.  32 divides `units`.
// (Calls of their own, as all that brings columns: inlined, they take registers from the loops that follow.)
template <class TopOf>
B200_DEVICE void find_tops(uint32_t *tops, uint32_t n, uint32_t units, TopOf top_of) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) tops[i] = 0u;
    __syncthreads();
    const uint32_t lane = threadIdx.x & 31u, pieces = units / 32u;
    constexpr uint32_t kBatch = 4;
    for (uint32_t q = threadIdx.x >> 5; q < n * pieces; q += kBatch * kWarps) {
        uint32_t top[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t at = q + b * kWarps;
            top[b] = at < n * pieces ? top_of(at / pieces, at % pieces * 32u + lane) : 0u;
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t at = q + b * kWarps, most = __reduce_max_sync(0xFFFFFFFFu, top[b]);
            if (lane == 0 && at < n * pieces) atomicMax(tops + at / pieces, most);
        }
    }
    __syncthreads();
}

// Columns of fp16 from those of bf16.
template <class From>
struct Converted {
    From from;
    const uint32_t *tops;
    B200_DEVICE uint32_t top_of(uint32_t j, uint32_t u) const {
        const uint4 v = from(j, u);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w, a = w << 16 & 0x7FFF0000u, b = w & 0x7FFF0000u;
            top = max(top, max(a < fp4::kInfBits ? a : 0u, b < fp4::kInfBits ? b : 0u));
        }
        return top;
    }
    B200_DEVICE uint4 operator()(uint32_t j, uint32_t u) const {
        const uint4 v = from(j, u);
        const float by = fp4::exp2_int(power_of(tops[j]));
        auto two = [&](uint32_t w) {
            const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xFFFF0000u) * by);
            return *reinterpret_cast<const uint32_t *>(&h);
        };
        return make_uint4(two(v.x), two(v.y), two(v.z), two(v.w));
    }
};

// ------------------------------------------------------------------ gate, up, SiLU

// X: x's type.  Codes are widened to fp16 either way, which takes nine operations a word of eight where bf16 takes eleven: bf16 columns are brought to fp16.
template <class W, typename X, int kNB>
B200_DEVICE void gate_up_part(const MoeParams &p, const Routing &r, uint8_t *smem, uint32_t columns_at, uint32_t begin, uint32_t end, uint32_t pair0, uint32_t n) {
    constexpr bool kConvert = !std::is_same<typename W::T, X>::value;
    const uint32_t base = ptx::smem_u32(smem), warp = warp_index(), lane = threadIdx.x & 31u;
    const uint32_t steps = (p.hidden + W::kStep - 1) / W::kStep, of_run = (p.inner + 7u) / 8u, pitch = column_pitch<W>(steps);
    uint32_t *tops = reinterpret_cast<uint32_t *>(smem + columns_at + p.up_columns * pitch);
    const Split split(end - begin, steps, kWarps);
    const Share s(split, begin, end, warp, steps, steps, base + warp * kRingBytes<W>);
    multiply<W, kNB, 1, false, kRing<W>>(
        p.gate_up, s,
        [&](uint32_t tile) { return place_in(r, of_run, tile); },
        [&](const Place &at, uint32_t row) { return ((uint64_t)at.expert * 2u + row / 8u) * p.inner + min(at.tile * 8u + row % 8u, p.inner - 1u); },
        [&](const Place &at) {
            if (p.all_tokens) return Columns{base + columns_at, pitch, 0, at.n, 0, 0, 0, r.pairs + at.start, p.top};
            return Columns{base + columns_at + (at.start - pair0) * pitch, pitch, 0, at.n, 0, 0, 0, nullptr, 1};
        },
        [&](uint32_t first, uint32_t count) {
            if (p.all_tokens) return;
            const Gathered<X> from{Plain<X>{static_cast<const X *>(p.x), 1, p.ldx, p.x_wide, false, p.hidden}, r.pairs + pair0, p.top};
            if constexpr (kConvert) {
                const Converted<Gathered<X>> to{from, tops};
                find_tops(tops, n, count * W::kUnits, [&](uint32_t j, uint32_t u) { return to.top_of(j, u); });
                stage_columns<W>(to, base + columns_at, pitch, first, count, n, false);
            } else {
                stage_columns<W>(from, base + columns_at, pitch, first, count, n, false);
            }
        },
        [&](const Place &at, const float(&sums)[kNB][4]) {
            const uint32_t i = at.tile * 8u + (lane >> 2);
#pragma unroll
            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e) {
                    const uint32_t j = nb * 8u + (lane & 3u) * 2u + e;
                    if (j >= at.n || i >= p.inner) continue;
                    const uint32_t pair = r.pairs[at.start + j];
                    const float back = kConvert ? fp4::exp2_int(-power_of(tops[p.all_tokens ? pair / p.top : at.start + j - pair0])) : 1.f, gate = sums[nb][e] * back;
                    p.h[(uint64_t)pair * p.h_ld + i] = gate / (1.f + expf(-gate)) * (sums[nb][e + 2] * back);
                }
        });
}

// All tokens as columns, where there is room for them: they need no routing.
template <class W, typename X>
B200_DEVICE void stage_tokens(const MoeParams &p, uint8_t *smem, uint32_t columns_at) {
    const uint32_t steps = (p.hidden + W::kStep - 1) / W::kStep, pitch = column_pitch<W>(steps), at = ptx::smem_u32(smem) + columns_at;
    uint32_t *tops = reinterpret_cast<uint32_t *>(smem + columns_at + p.up_columns * pitch);
    const Plain<X> from{static_cast<const X *>(p.x), 1, p.ldx, p.x_wide, false, p.hidden};
    if constexpr (!std::is_same<typename W::T, X>::value) {
        const Converted<Plain<X>> to{from, tops};
        find_tops(tops, p.tokens, steps * W::kUnits, [&](uint32_t j, uint32_t u) { return to.top_of(j, u); });
        stage_columns<W>(to, at, pitch, 0, steps, p.tokens, false);
    } else {
        stage_columns<W>(from, at, pitch, 0, steps, p.tokens, false);
    }
}

template <class W, typename X>
__global__ void __launch_bounds__(kThreads, 1) gate_up_kernel(const MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const Routing r = routing_at(smem + kWarps * kRingBytes<W>, p.pairs, p.experts);
    const uint32_t columns_at = kWarps * kRingBytes<W> + routing_bytes(p.pairs, p.experts);
    ptx::wait_for_grids_before();
    const bool write = blockIdx.x == 0;
    if (p.all_tokens) stage_tokens<W, X>(p, smem, columns_at);
    if (p.logits) {
        for (uint32_t t = threadIdx.x >> 5; t < p.tokens; t += kWarps)
            choose(p, t, r.ids, write, reinterpret_cast<uint64_t *>(smem + (threadIdx.x >> 5) * kRingBytes<W>));
    } else {
        for (uint32_t i = threadIdx.x; i < p.pairs; i += kThreads) {
            const int64_t e = p.id_bytes == 8 ? static_cast<const int64_t *>(p.ids_in)[i] : static_cast<const int32_t *>(p.ids_in)[i];
            const int32_t id = e >= 0 && e < (int64_t)p.experts ? (int32_t)e : -1;
            r.ids[i] = id;
            if (write) p.ids[i] = id;
        }
    }
    __syncthreads();
    find_runs(p, r, p.run);
    if (write)
        for (uint32_t i = threadIdx.x; i < routing_bytes(p.pairs, p.experts) / 16u; i += kThreads) p.routing[i] = reinterpret_cast<const uint4 *>(smem + kWarps * kRingBytes<W>)[i];
    each_part(r, (p.inner + 7u) / 8u, p.all_tokens ? p.pairs : p.up_columns, [&](uint32_t begin, uint32_t end, uint32_t pair0, uint32_t n, uint32_t longest) {
        if (longest <= 8u) gate_up_part<W, X, 1>(p, r, smem, columns_at, begin, end, pair0, n);
        else gate_up_part<W, X, 2>(p, r, smem, columns_at, begin, end, pair0, n);
    });
}

// ------------------------------------------------------------------ down

// Inner values as the sum of two 16-bit numbers, the second what the first leaves over: fp16 has 22 digits that way, bf16 16.
template <typename T>
B200_DEVICE void split_unit(const float4 (&from)[2], uint32_t left, float by, uint4 *high, uint4 *low) {
    const float v[8] = {from[0].x, from[0].y, from[0].z, from[0].w, from[1].x, from[1].y, from[1].z, from[1].w};
    alignas(16) T a[8], b[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        const float x = e < left ? v[e] * by : 0.f;
        a[e] = fp4::Elem<T>::from_float(x);
        const float rest = x - fp4::Elem<T>::to_float(a[e]);
        b[e] = fp4::Elem<T>::from_float(fabsf(rest) <= 3.0e38f ? rest : 0.f);  // (an infinity or NaN is the first number's)
    }
    *high = *reinterpret_cast<const uint4 *>(a);
    *low = *reinterpret_cast<const uint4 *>(b);
}

// Inner values of n pairs as columns, by all threads; kPieces: `count` steps from step `first` on, and `anew` where their largest ones are not known yet, else all steps.
template <class W, bool kPieces>
__device__ __noinline__ void stage_inner(const float *h, uint32_t h_ld, uint32_t inner, const uint16_t *pairs, uint32_t n, uint32_t base, uint32_t pitch, uint32_t plane, uint32_t *tops,
                                         uint32_t first, uint32_t count, bool anew) {
    using T = typename W::T;
    constexpr bool kScale = std::is_same<T, __half>::value;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    // (a row of h has room for whole units; what lies behind its end does not count)
    auto load = [&](uint32_t j, uint32_t u, float4(&v)[2]) {
        const float4 *from = reinterpret_cast<const float4 *>(h + (uint64_t)pairs[j] * h_ld + u * 8u);
        v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u * 8u < inner) {
            v[0] = from[0];
            v[1] = from[1];
        }
    };
    const uint32_t u0 = kPieces ? first * W::kUnits : 0u, room = (kPieces ? count : (inner + W::kStep - 1) / W::kStep) * W::kUnits, pieces = (room + 31u) / 32u;
    if (kScale && (!kPieces || anew))
        find_tops(tops, n, (inner + 255u) / 256u * 32u, [&](uint32_t j, uint32_t u) {
            float4 v[2];
            load(j, u, v);
            const float w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
            uint32_t top = 0;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const uint32_t b = __float_as_uint(w[e]) & 0x7FFFFFFFu;
                if (u * 8u + e < inner && b < fp4::kInfBits) top = max(top, b);
            }
            return top;
        });
    constexpr uint32_t kBatch = 3;
    for (uint32_t q = warp; q < n * pieces; q += kBatch * kWarps) {
        float4 v[kBatch][2];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t at = q + b * kWarps;
            if (at < n * pieces) load(at / pieces, u0 + at % pieces * 32u + lane, v[b]);
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t at = q + b * kWarps, j = at / pieces, u = at % pieces * 32u + lane;
            if (at >= n * pieces || u >= room) continue;
            uint4 high, low;
            split_unit<T>(v[b], (u0 + u) * 8u < inner ? inner - (u0 + u) * 8u : 0u, kScale ? fp4::exp2_int(power_of(tops[j])) : 1.f, &high, &low);
            const uint32_t to = base + j * pitch + unit_place<W>(u);
            ptx::st_shared_v4(to, unit_order<W>(high));
            ptx::st_shared_v4(to + plane, unit_order<W>(low));
        }
    }
}

// kPieces: a part may be one run whose columns have no room as a whole.
template <class W, int kNB, bool kPieces>
B200_DEVICE void down_part(const MoeParams &p, const Routing &r, uint8_t *smem, uint32_t columns_at, uint32_t begin, uint32_t end, uint32_t pair0, uint32_t n) {
    constexpr bool kScale = std::is_same<typename W::T, __half>::value;
    const uint32_t base = ptx::smem_u32(smem), warp = warp_index(), lane = threadIdx.x & 31u;
    const uint32_t steps = (p.inner + W::kStep - 1) / W::kStep, of_run = (p.hidden + kTileRows - 1u) / kTileRows;
    const uint32_t window = !kPieces || n <= p.down_columns ? steps : (((kMaxSmem - columns_at) / n - 4u) / kHalves - column_pitch<W>(0)) / (W::kUnits * 16u);
    const uint32_t pitch = column_pitch<W>(window), plane = (kPieces ? n : p.down_columns) * pitch;
    bool anew = true;
    uint32_t *tops = reinterpret_cast<uint32_t *>(smem + columns_at + kHalves * plane);
    const Split split(end - begin, steps, kWarps);
    const Share s(split, begin, end, warp, steps, window, base + warp * kRingBytes<W>);
    multiply<W, kNB, kHalves, false, kRing<W>>(
        p.down, s,
        [&](uint32_t tile) { return place_in(r, of_run, tile); },
        [&](const Place &at, uint32_t row) { return (uint64_t)at.expert * p.hidden + min(at.tile * kTileRows + row, p.hidden - 1u); },
        [&](const Place &at) { return Columns{base + columns_at + (at.start - pair0) * pitch, pitch, plane, at.n, 0, 0, 0, nullptr, 1}; },
        [&](uint32_t first, uint32_t count) {
            stage_inner<W, kPieces>(p.h, p.h_ld, p.inner, r.pairs + pair0, n, base + columns_at, pitch, plane, tops, first, count, anew);
            if (kPieces) anew = false;
        },
        [&](const Place &at, const float(&sums)[kNB][4]) {
#pragma unroll
            for (uint32_t nb = 0; nb < (uint32_t)kNB; ++nb)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t j = nb * 8u + (lane & 3u) * 2u + (e & 1u), row = at.tile * kTileRows + (lane >> 2) + (e >> 1) * 8u;
                    if (j < at.n && row < p.hidden)
                        p.parts[(uint64_t)r.pairs[at.start + j] * p.hidden + row] = kScale ? sums[nb][e] * fp4::exp2_int(-power_of(tops[at.start + j - pair0])) : sums[nb][e];
                }
        });
}

template <class W, bool kPieces>
__global__ void __launch_bounds__(kThreads, 1) down_kernel(const MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const Routing r = routing_at(smem + kWarps * kRingBytes<W>, p.pairs, p.experts);
    const uint32_t columns_at = kWarps * kRingBytes<W> + routing_bytes(p.pairs, p.experts);
    ptx::wait_for_grids_before();
    for (uint32_t i = threadIdx.x; i < routing_bytes(p.pairs, p.experts) / 16u; i += kThreads) reinterpret_cast<uint4 *>(smem + kWarps * kRingBytes<W>)[i] = p.routing[i];
    __syncthreads();
    each_part(r, (p.hidden + kTileRows - 1u) / kTileRows, p.down_columns, [&](uint32_t begin, uint32_t end, uint32_t pair0, uint32_t n, uint32_t longest) {
        if (longest <= 8u) down_part<W, 1, kPieces>(p, r, smem, columns_at, begin, end, pair0, n);
        else down_part<W, 2, kPieces>(p, r, smem, columns_at, begin, end, pair0, n);
    });
}

// ------------------------------------------------------------------ the weighted sum, in the order of the choices

constexpr uint32_t kSumThreads = 128;

__global__ void __launch_bounds__(kSumThreads) sum_kernel(const MoeParams p) {
    ptx::wait_for_grids_before();
    const uint32_t at = blockIdx.x * kSumThreads + threadIdx.x, t = blockIdx.y;
    if (at >= p.hidden) return;
    float v = 0.f;
#pragma unroll 8
    for (uint32_t i = t * p.top; i < (t + 1u) * p.top; ++i)
        if (p.ids[i] >= 0) v = fmaf(p.shares[i], p.parts[(uint64_t)i * p.hidden + at], v);
    static_cast<uint16_t *>(p.y)[(int64_t)t * p.ldy + at] = p.y_f16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// ------------------------------------------------------------------ launches

// Where the parts of the workspace begin.
struct Layout {
    uint64_t logits, ids, shares, routing, h, parts, bytes;
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
    l.routing = take(routing_bytes((uint32_t)pairs, (uint32_t)m->experts));
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
            if (ld[i] % 8 != 0 || ld[i] > 1 << 28 || !fp4::aligned(plain[i], 16)) return B200SPMM_ERR_UNSUPPORTED;
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

// Columns that a block has room for, in `planes` parts.
template <class W>
uint32_t room_for(const MoeParams &p, uint32_t k, uint32_t planes) {
    static_assert(kWarps * kRingBytes<W> + routing_bytes(kMaxTokens * kMaxTop, kMaxExperts) < kMaxSmem, "the largest routing has room beside the rings");
    const uint32_t taken = kWarps * kRingBytes<W> + routing_bytes(p.pairs, p.experts), steps = (k + W::kStep - 1) / W::kStep;
    const uint64_t each = (uint64_t)planes * ((uint64_t)steps * W::kUnits * 16u + 192u) + 4u;
    return (uint32_t)std::min<uint64_t>(p.pairs, (kMaxSmem - taken) / each);  // (as many as there are pairs at most)
}
template <class Up, typename X, class Down>
int launch_all(MoeParams p, double *logits, cudaStream_t stream) {
    static std::atomic<uint64_t> up_allowed{0}, down_allowed[2] = {};
    p.up_columns = room_for<Up>(p, p.hidden, 1);
    p.down_columns = room_for<Down>(p, p.inner, kHalves);
    // Columns of all tokens are there before the routing is, those of a block's own pairs are fewer.  With all and with its own: 1, 2, 4, 8 and 16 tokens in
    // bf16 36.9 and 38.6 us, 55.1 and 56.8, 83.8 and 85.4, 108.7 and 109.9, 143.9 and 144.5; with experts in 4 bits 53.3 and 56.9, 81.2 and 83.9, 120.8 and 121.6, 159.8 and 157.5, 214.5 and 209.1.
    p.all_tokens = p.tokens <= std::min(4u, p.up_columns);
    // Inner values of a run come in pieces where it has no room for them as a whole: 32 tokens, 2 of 8 experts of 4096 x 14336 each in codes for fp16 375 us, in bf16 522, where shorter
    // runs that read an expert again and again take 720 and 1,795; with a kernel for both, 8 tokens through 64 experts of 4096 x 2048 take 168 us for 157.
    // (As many of them as a column of either half has room for with codes, of both with 16-bit experts: beyond that, a call is refused.)
    p.run = std::min(kRun, p.up_columns);
    if (p.run == 0 || room_for<Down>(p, p.inner, Down::kCodes ? 1 : kHalves) == 0) return B200SPMM_ERR_UNSUPPORTED;
    // (there are as many runs as pairs, or fewer)
    auto blocks = [&](uint32_t tiles) { return (uint32_t)std::min<uint64_t>(fp4::sm_count(), (uint64_t)p.pairs * tiles); };
    B200_CUDA_TRY(allow_smem(gate_up_kernel<Up, X>, up_allowed));
    const bool pieces = p.run > p.down_columns;
    const auto down = pieces ? down_kernel<Down, true> : down_kernel<Down, false>;
    B200_CUDA_TRY(allow_smem(down, down_allowed[pieces]));
    if (logits) B200_CUDA_TRY(launch_after(logits_kernel<X>, dim3(p.experts, (p.tokens + kLogitTokens - 1) / kLogitTokens), kLogitThreads, 0, 1, stream, p, logits));
    B200_CUDA_TRY(launch_after(gate_up_kernel<Up, X>, dim3(blocks((p.inner + 7) / 8)), kThreads, kMaxSmem, 1, stream, p));
    B200_CUDA_TRY(launch_after(down, dim3(blocks((p.hidden + kTileRows - 1) / kTileRows)), kThreads, kMaxSmem, 1, stream, p));
    B200_CUDA_TRY(launch_after(sum_kernel, dim3((p.hidden + kSumThreads - 1) / kSumThreads, p.tokens), kSumThreads, 0, 1, stream, p));
    return B200SPMM_OK;
}
// Inner values beside codes have 22 digits, for bf16 too: with 11 they are the largest error of a layer before its result is rounded.
template <int kUp, typename X>
int launch_codes(const MoeParams &p, uint32_t span, double *logits, cudaStream_t stream) {
    using Up = Weights<__half, kUp>;
    return span == 32   ? launch_all<Up, X, Weights<__half, 32>>(p, logits, stream)
           : span == 64 ? launch_all<Up, X, Weights<__half, 64>>(p, logits, stream)
                        : launch_all<Up, X, Weights<__half, 128>>(p, logits, stream);
}

template <typename T>
int launch_moe(const b200spmm_moe_t *m, const MoeParams &p, double *logits, cudaStream_t stream) {
    if (!m->gate_up) return launch_all<Weights<T, 0>, T, Weights<T, 0>>(p, logits, stream);
    const uint32_t a = span_of(m->gate_up), b = span_of(m->down);
    return a == 32 ? launch_codes<32, T>(p, b, logits, stream) : a == 64 ? launch_codes<64, T>(p, b, logits, stream) : launch_codes<128, T>(p, b, logits, stream);
}

// ids null: they are found from the logits, and left, with the shares, at out_ids and out_shares where those are wanted.
int run_moe(const b200spmm_moe_t *m, const void *x, int64_t ldx, int64_t tokens, const void *ids, int id_bytes, const float *shares, void *y, int64_t ldy, int32_t *out_ids,
            float *out_shares, void *workspace, cudaStream_t stream) {
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
    p.routing = reinterpret_cast<uint4 *>(ws + l.routing);
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
        return narrow::run_moe(m, d_x, ldx, tokens, nullptr, 0, nullptr, d_y, ldy, d_ids, d_shares, workspace, static_cast<cudaStream_t>(stream));
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
        return narrow::run_moe(m, d_x, ldx, tokens, d_ids, id_bytes, d_shares, d_y, ldy, nullptr, nullptr, workspace, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
