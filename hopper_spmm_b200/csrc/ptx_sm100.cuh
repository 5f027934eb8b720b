// Inline-PTX layer for sm_100a: mbarrier (bounded waits), TMA tiled / gather4 loads,
// cp.async row gathers, tcgen05 (TMEM allocation, MMA, commit, load) and the shared-memory /
// instruction descriptors they consume.  Takes the place of the reference's sm_90a wrappers
// (src/ptx/barrier.h, src/ptx/tma.h, src/ptx/wgmma.h, src/ptx/ptx_utils.h).
//
// Unlike the reference's mbarrier_wait (src/ptx/barrier.h:29-41), every wait here gives up
// after a time limit and reports it, so a broken pipeline ends the kernel instead of hanging
// the device.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace b200spmm {
namespace ptx {

#define B200_DEVICE __device__ __forceinline__

B200_DEVICE uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

B200_DEVICE uint64_t global_timer_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// The kernels of a product are launched with programmatic stream serialization (launch_after in capi.cu): a grid may
// start once every block of the grid before it in the stream has ended, while that one's results are still on their way.
// From this wait on they are visible.  Before it a kernel may read what the plan holds - made, and waited for, when
// the plan was - and nothing else; and it writes nothing.  Every thread waits, so that a grid that has ended means that those
// before it have too.
B200_DEVICE void wait_for_grids_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A load that may not go through the read-only path: what it reads may have been written since this grid started.
B200_DEVICE uint4 ld_global_v4(const void *p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

// 32 bytes, 32-byte aligned.
B200_DEVICE void ld_global_v8(const void *p, uint32_t *v) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p) : "memory");
}

// 32 bytes, 32-byte aligned.
B200_DEVICE void st_global_v8(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// A load of a stream that nothing writes: what is not in L2 comes with the 256 bytes around it, the next of the stream.  (The
// entries of row units, of which a lane group has one batch under way: 300,000 nodes, 64 / 128 features 77.6 / 141 -> 73.4 / 136
// us, 2^20 nodes, 64 features 230 -> 220; an instruction of its own that fetches ahead costs 5 to 20 % instead.)
B200_DEVICE uint4 ld_global_nc_v4_ahead(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// ------------------------------------------------------------------ mbarrier

B200_DEVICE void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

B200_DEVICE void fence_mbar_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }

B200_DEVICE void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Adds `bytes` to the transaction count the current phase waits for, without arriving.
B200_DEVICE void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

B200_DEVICE void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

B200_DEVICE bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

// Wait for the phase with the given parity to complete.  Returns false when `*abort_flag`
// (shared memory) is raised by another role or when `limit_ns` elapses, in which case this
// thread raises the flag itself.  The caller must then leave its loop.
B200_DEVICE bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 0) {
            if (*abort_flag) return false;
            if (global_timer_ns() - t0 > limit_ns) {
                *abort_flag = 1;
                return false;
            }
        }
    }
}

// The same wait without an abort flag: for the teardown after a failure, where the flag is already
// up and the waiter only wants its own outstanding work to finish (or the time to run out).
B200_DEVICE bool mbar_wait_bounded(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 0 && global_timer_ns() - t0 > limit_ns) return false;
    }
}

// Waits at barrier `id` for `threads` threads, whole warps, and tells all of them alike whether one of them brought `mine`.
B200_DEVICE bool bar_or(uint32_t id, uint32_t threads, bool mine) {
    uint32_t any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 q, %3, 0;\nbar.red.or.pred p, %1, %2, q;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(any) : "r"(id), "r"(threads), "r"(mine ? 1u : 0u) : "memory");
    return any != 0;
}

// ------------------------------------------------------------------ proxies and fences

// Orders this thread's generic-proxy shared-memory accesses with async-proxy accesses
// (TMA, tcgen05.mma operand reads).
B200_DEVICE void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

B200_DEVICE void tcgen05_fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
B200_DEVICE void tcgen05_fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }


// ------------------------------------------------------------------ TMA loads (own HBM only)

B200_DEVICE void prefetch_tensormap(const void *tmap) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(tmap) : "memory");
}

// 2-D tiled load: box at (x, y) -> smem, completion as bytes on `bar`.
// x * element size must be a multiple of 16 bytes.
B200_DEVICE void tma_load_2d(uint32_t dst, const void *tmap, int32_t x, int32_t y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// Plain bulk copy global -> shared of `bytes` contiguous bytes (a multiple of 16, both addresses
// 16-byte aligned), completion counted in bytes on `bar`.  One request whatever the size, where a
// tiled load of narrow rows costs the TMA unit one request per row.
B200_DEVICE void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Gather of four rows y0..y3 of a 2-D tensor, box width taken from the tensor map, starting at
// column x.  The four rows land one after another in shared memory.
B200_DEVICE void tma_gather4_2d(uint32_t dst, const void *tmap, int32_t x, int32_t y0, int32_t y1, int32_t y2,
                                int32_t y3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4, %5, %6}], [%7];"
        ::"r"(dst), "l"(tmap), "r"(x), "r"(y0), "r"(y1), "r"(y2), "r"(y3), "r"(bar)
        : "memory");
}

// The same for a warp that goes through its loop as one, with `on` set in a single lane (see umma_pair_f16_ts_if).
B200_DEVICE void mbar_arrive_expect_tx_if(uint32_t on, uint32_t bar, uint32_t bytes) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %2, 0;\n@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(bar), "r"(bytes), "r"(on) : "memory");
}
B200_DEVICE void tma_load_2d_if(uint32_t on, uint32_t dst, const void *tmap, int32_t x, int32_t y, uint32_t bar) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %5, 0;\n"
                 "@q cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}\n"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(bar), "r"(on) : "memory");
}
B200_DEVICE void bulk_load_if(uint32_t on, uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %4, 0;\n"
                 "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n}\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "r"(on) : "memory");
}

B200_DEVICE uint4 ld_shared_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
B200_DEVICE uint32_t ld_shared_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
B200_DEVICE void st_shared_v4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
B200_DEVICE void st_shared_u16(uint32_t addr, uint16_t v) {
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}

// ------------------------------------------------------------------ cp.async (16-byte gathers)

// Copies 16 bytes global -> shared, bypassing L1; src_bytes < 16 zero-fills the rest
// (src_bytes == 0 reads nothing and writes 16 zero bytes).
B200_DEVICE void cp_async_16(uint32_t dst, const void *src, uint32_t src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
// Copies 4 bytes global -> shared (cached in L1: neighbouring words are fetched next).
B200_DEVICE void cp_async_4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
B200_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// One arrival on `bar` when the copies that this thread has issued so far have landed.
B200_DEVICE void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
template <int N>
B200_DEVICE void cp_async_wait_group() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------ tensor memory

// Whole-warp calls.  `n_cols` is a power of two in [32, 512]; the base address is written to
// shared memory at `dst_smem`.
B200_DEVICE void tmem_alloc(uint32_t dst_smem, uint32_t n_cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(n_cols)
                 : "memory");
}
B200_DEVICE void tmem_relinquish_alloc_permit() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
B200_DEVICE void tmem_dealloc(uint32_t taddr, uint32_t n_cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(n_cols) : "memory");
}

// 32 lanes x 8 consecutive 32-bit columns.
B200_DEVICE void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns: thread i of the warp receives lane
// (taddr.lane + i), columns taddr.col .. +15.  A warp may only touch the 32 lanes of its own
// quarter: lanes 32*(warp_id % 4) .. +31.
B200_DEVICE void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// 32 lanes x 32 consecutive 32-bit columns: thread i receives lane (taddr.lane + i), columns
// taddr.col .. +31, i.e. 128 contiguous bytes of one accumulator row.
B200_DEVICE void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// The other way: thread i's 32 words to lane taddr.lane + i.
B200_DEVICE void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
          "r"(r[30]), "r"(r[31])
        : "memory");
}
B200_DEVICE void tmem_st_32x32b_x32(uint32_t taddr, const float (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
          "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]), "f"(r[19]),
          "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]), "f"(r[28]), "f"(r[29]),
          "f"(r[30]), "f"(r[31])
        : "memory");
}
B200_DEVICE void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
B200_DEVICE void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------------ CTA pairs (cta_group::2)
// A cluster of two CTAs on neighbouring SMs can run ONE tcgen05.mma of M = 256: CTA r holds rows
// 128 r .. of A and of the accumulator and columns (N / 2) r .. of B in its own shared / tensor memory, at
// the same offsets in both CTAs; the even CTA (rank 0) issues.  Every byte of B is then fetched from L2
// by one of the two SMs only.

B200_DEVICE uint32_t cluster_cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
B200_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
B200_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of `local_smem_addr` in the shared memory of CTA `rank` of this cluster.
B200_DEVICE uint32_t map_to_cta(uint32_t local_smem_addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local_smem_addr), "r"(rank));
    return r;
}
// One arrival on a barrier that may live in the other CTA of the cluster (address from map_to_cta).
B200_DEVICE void mbar_arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// The same without ordering of this thread's earlier memory operations (for data that another proxy wrote
// and whose completion this thread has already observed).
B200_DEVICE void mbar_arrive_cluster_relaxed(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
B200_DEVICE void tmem_alloc_pair(uint32_t dst_smem, uint32_t n_cols) {  // whole warp, the same warp in both CTAs
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(n_cols) : "memory");
}
B200_DEVICE void tmem_relinquish_alloc_permit_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
B200_DEVICE void tmem_dealloc_pair(uint32_t taddr, uint32_t n_cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(n_cols) : "memory");
}
// D (+)= A * B over the pair; issued by ONE thread of the even CTA.  `on` == 0 skips it.
B200_DEVICE void umma_pair_ss_lohi_if(bool tf32, uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                      uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    if (tf32)
        asm volatile(
            "{\n.reg .pred p, q;\n.reg .b64 da, db;\nmov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
            "setp.ne.b32 p, %6, 0;\nsetp.ne.b32 q, %7, 0;\n"
            "@q tcgen05.mma.cta_group::2.kind::tf32 [%0], da, db, %5, p;\n}\n"
            ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(on) : "memory");
    else
        asm volatile(
            "{\n.reg .pred p, q;\n.reg .b64 da, db;\nmov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
            "setp.ne.b32 p, %6, 0;\nsetp.ne.b32 q, %7, 0;\n"
            "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n}\n"
            ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(on) : "memory");
}
// The same with a 2:4 sparse A: K is twice as large, and tensor memory column `meta` (an even one; the descriptor's lowest bit
// adds one) says in both CTAs which two of four columns A's values belong to.
enum : uint32_t { kSparseA = 1u << 2 };  // of the instruction descriptor
B200_DEVICE void umma_pair_sparse_f16_if(uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t meta,
                                         uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 da, db;\nmov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
        "setp.ne.b32 p, %7, 0;\nsetp.ne.b32 q, %8, 0;\n"
        "@q tcgen05.mma.sp.cta_group::2.kind::f16 [%0], da, db, [%5], %6, p;\n}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(meta), "r"(idesc), "r"(accumulate), "r"(on) : "memory");
}
// 128 lanes x 16 bytes from shared memory (core matrices of eight lanes) to four columns of tensor memory, in both CTAs; runs in
// order with the MMAs that the thread issues.
B200_DEVICE void tmem_copy_pair_128x128b(uint32_t taddr, uint64_t smem_desc) {
    asm volatile("tcgen05.cp.cta_group::2.128x128b [%0], %1;" ::"r"(taddr), "l"(smem_desc) : "memory");
}
// Forms for a warp that goes through its loop as one, with `on` set in a single lane: addresses and descriptors then stay in uniform
// registers, which is where these instructions want them.  A lone lane moves each there: 90 clocks an MMA, and the tensor pipe waits.
// A in tensor memory (row = lane, two 16-bit values of k a column) in both CTAs, each with its own 128 rows.
B200_DEVICE void umma_pair_f16_ts_if(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 db;\nmov.b64 db, {%2, %3};\nsetp.ne.b32 p, %5, 0;\nsetp.ne.b32 q, %6, 0;\n"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], db, %4, p;\n}\n"
                 ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(on) : "memory");
}
// Four in a row: 64 values of k, eight columns of A further each time and `kNext` units of 16 bytes of B.
template <uint32_t kNext>
B200_DEVICE void umma_pair_f16_ts_x4_if(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, q, t;\n.reg .b64 db;\n.reg .b32 la, lb;\nsetp.ne.b32 p, %5, 0;\nsetp.ne.b32 q, %6, 0;\nsetp.eq.b32 t, %0, %0;\n"
                 "mov.b64 db, {%2, %3};\n@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], db, %4, p;\n"
                 "add.u32 la, %1, 8;\nadd.u32 lb, %2, %7;\nmov.b64 db, {lb, %3};\n@q tcgen05.mma.cta_group::2.kind::f16 [%0], [la], db, %4, t;\n"
                 "add.u32 la, %1, 16;\nadd.u32 lb, %2, %8;\nmov.b64 db, {lb, %3};\n@q tcgen05.mma.cta_group::2.kind::f16 [%0], [la], db, %4, t;\n"
                 "add.u32 la, %1, 24;\nadd.u32 lb, %2, %9;\nmov.b64 db, {lb, %3};\n@q tcgen05.mma.cta_group::2.kind::f16 [%0], [la], db, %4, t;\n}\n"
                 ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(on), "n"(kNext), "n"(2 * kNext), "n"(3 * kNext) : "memory");
}
B200_DEVICE void umma_commit_pair_if(uint32_t on, uint32_t bar) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %2, 0;\n"
                 "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n"
                 ::"r"(bar), "h"((uint16_t)3), "r"(on) : "memory");
}
B200_DEVICE void umma_commit_if(uint32_t on, uint32_t bar) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(on) : "memory");
}
// One arrival on the barrier at offset `bar` in BOTH CTAs of the pair (mask 0b11) when every MMA this
// thread issued so far has finished.
B200_DEVICE void umma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// The same, arriving on the issuing CTA's barrier only.
B200_DEVICE void umma_commit_pair_local(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
B200_DEVICE void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// mbar_wait for a barrier on which the other CTA of the cluster arrives: acquire at cluster scope.
B200_DEVICE bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
B200_DEVICE bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, uint64_t limit_ns) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait_cluster(bar, parity)) return true;
        if ((it & 63u) == 0) {
            if (*abort_flag) return false;
            if (global_timer_ns() - t0 > limit_ns) {
                *abort_flag = 1;
                return false;
            }
        }
    }
}

// ------------------------------------------------------------------ tcgen05.mma

// Shared-memory matrix descriptor (64 bit):
//   [0,14)  start address >> 4          [16,30) leading-dimension byte offset >> 4
//   [32,46) stride-dimension byte offset >> 4     [46,48) version = 1
//   [49,52) base offset = 0             [61,64) swizzle: 0 none, 1 128B over 32-byte units,
//                                               2 128B, 4 64B, 6 32B (16-byte units)
enum : uint32_t { kSwizzleNone = 0, kSwizzle128BBase32B = 1, kSwizzle128B = 2, kSwizzle64B = 4, kSwizzle32B = 6 };

B200_DEVICE uint64_t make_smem_desc(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes, uint32_t swizzle) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
    d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)((sbo_bytes >> 4) & 0x3FFFu) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)(swizzle & 7u) << 61;
    return d;
}

// Instruction descriptor for kind::f16 / kind::tf32 with fp32 accumulation:
//   [4,6) D format (1 = f32)   [7,10) A format   [10,13) B format  (0 f16, 1 bf16, 2 tf32)
//   [15] A is MN-major   [16] B is MN-major   [17,23) N >> 3   [24,29) M >> 4
enum : uint32_t { kFmtF16 = 0, kFmtBF16 = 1, kFmtTF32 = 2 };

__host__ __device__ constexpr uint32_t make_instr_desc(uint32_t fmt, uint32_t m, uint32_t n, bool a_mn_major,
                                                       bool b_mn_major) {
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) |
           ((n >> 3) << 17) | ((m >> 4) << 24);
}

// D[tmem] (+)= A[smem] * B[smem]; issued by ONE thread.  accumulate == 0 overwrites D.
B200_DEVICE void umma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
B200_DEVICE void umma_tf32_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptors given as 32-bit halves (the high words are loop constants, the low words change by
// one add per tile).
B200_DEVICE void umma_f16_ss_lohi(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                 uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        ".reg .b64 da, db;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Same, issued only when `on` is non-zero (predicated, no branch).
B200_DEVICE void umma_f16_ss_lohi_if(uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                    uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        ".reg .b64 da, db;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "setp.ne.b32 p, %6, 0;\n"
        "setp.ne.b32 q, %7, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(on)
        : "memory");
}
// Descriptors given as 32-bit halves (the high words are loop constants, the low words change by
// one add per tile).
B200_DEVICE void umma_tf32_ss_lohi(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                 uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        ".reg .b64 da, db;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], da, db, %5, p;\n"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Same, issued only when `on` is non-zero (predicated, no branch).
B200_DEVICE void umma_tf32_ss_lohi_if(uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                    uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        ".reg .b64 da, db;\n"
        "mov.b64 da, {%1, %2};\n"
        "mov.b64 db, {%3, %4};\n"
        "setp.ne.b32 p, %6, 0;\n"
        "setp.ne.b32 q, %7, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], da, db, %5, p;\n"
        "}\n"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(on)
        : "memory");
}

// ------------------------------------------------------------------ block-scaled 4-bit MMA
// D (+)= (scaled A) * (scaled B): e2m1 operands, K-major, 64 values a call, whose scales lie in tensor memory: row r of a 128-row block
// in lane r % 32 (the same in each quarter of the lanes), column r / 32, four scales to a 32-bit word.  Instruction descriptor:
//   [4,6) which scale of B's words   [7,10) A format, [10,12) B format (1 = e2m1)   [17,23) N >> 3
//   [23] scales are e8m0 (0: e4m3)   [27,29) M >> 7   [29,31) which scale of A's words
// kCtas 2: shared by a pair, 256 rows, the scales of A each CTA's own, those of B in both.  `on` set in a single lane, see above.
// nvfp4 takes all four scales of a word (16 values each), mxfp4 two of them (32 values each): 0 or 2 in the descriptor.
__host__ __device__ constexpr uint32_t make_fp4_instr_desc(bool e8m0, uint32_t m, uint32_t n, uint32_t scale_id) {
    return (scale_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((e8m0 ? 1u : 0u) << 23) | ((m >> 7) << 27) | (scale_id << 29);
}
template <bool kMx, int kCtas>
B200_DEVICE void umma_fp4_ss_if(uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t a_scales,
                                uint32_t b_scales, uint32_t accumulate) {
#define B200_FP4_MMA(ctas, kind)                                                                                              \
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 da, db;\nmov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"                     \
                 "setp.ne.b32 p, %8, 0;\nsetp.ne.b32 q, %9, 0;\n"                                                              \
                 "@q tcgen05.mma.cta_group::" ctas ".kind::" kind " [%0], da, db, %5, [%6], [%7], p;\n}\n"                       \
                 ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate), "r"(on) : "memory")
    if constexpr (kMx && kCtas == 1) B200_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
    else if constexpr (kMx) B200_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
    else if constexpr (kCtas == 1) B200_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    else B200_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
#undef B200_FP4_MMA
}
constexpr uint32_t kSecondScales = make_fp4_instr_desc(false, 0, 0, 2) ^ make_fp4_instr_desc(false, 0, 0, 0);  // the second pair of a word's scales
// Four in a row, 256 values of k: 32 bytes further in either operand, the scales' words `next_b` (B) and four (A) columns on - for mxfp4
// the second and the fourth take the second pair of a word.
template <bool kMx, int kCtas>
B200_DEVICE void umma_fp4_ss_x4_if(uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t a_scales,
                                   uint32_t b_scales, uint32_t next_b, uint32_t accumulate) {
    const uint32_t idesc1 = kMx ? idesc | kSecondScales : idesc;
    const uint32_t a1 = a_scales + (kMx ? 0u : 4u), a2 = a_scales + (kMx ? 4u : 8u), a3 = a_scales + (kMx ? 4u : 12u);
    const uint32_t b1 = b_scales + (kMx ? 0u : next_b), b2 = b_scales + (kMx ? 1u : 2u) * next_b, b3 = b_scales + (kMx ? 1u : 3u) * next_b;
#define B200_FP4_MMA4(ctas, kind)                                                                                                          \
    asm volatile("{\n.reg .pred p, q, t;\n.reg .b64 da, db;\n.reg .b32 la, lb;\nsetp.ne.b32 p, %14, 0;\nsetp.ne.b32 q, %15, 0;\nsetp.eq.b32 t, %0, %0;\n" \
                 "mov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"                                                                           \
                 "@q tcgen05.mma.cta_group::" ctas ".kind::" kind " [%0], da, db, %5, [%6], [%10], p;\n"                                      \
                 "add.u32 la, %1, 2;\nadd.u32 lb, %3, 2;\nmov.b64 da, {la, %2};\nmov.b64 db, {lb, %4};\n"                                    \
                 "@q tcgen05.mma.cta_group::" ctas ".kind::" kind " [%0], da, db, %16, [%7], [%11], t;\n"                                     \
                 "add.u32 la, %1, 4;\nadd.u32 lb, %3, 4;\nmov.b64 da, {la, %2};\nmov.b64 db, {lb, %4};\n"                                    \
                 "@q tcgen05.mma.cta_group::" ctas ".kind::" kind " [%0], da, db, %5, [%8], [%12], t;\n"                                      \
                 "add.u32 la, %1, 6;\nadd.u32 lb, %3, 6;\nmov.b64 da, {la, %2};\nmov.b64 db, {lb, %4};\n"                                    \
                 "@q tcgen05.mma.cta_group::" ctas ".kind::" kind " [%0], da, db, %16, [%9], [%13], t;\n}\n"                                  \
                 ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(a_scales), "r"(a1), "r"(a2), "r"(a3), "r"(b_scales), "r"(b1),   \
                   "r"(b2), "r"(b3), "r"(accumulate), "r"(on), "r"(idesc1) : "memory")
    if constexpr (kMx && kCtas == 1) B200_FP4_MMA4("1", "mxf4.block_scale.scale_vec::2X");
    else if constexpr (kMx) B200_FP4_MMA4("2", "mxf4.block_scale.scale_vec::2X");
    else if constexpr (kCtas == 1) B200_FP4_MMA4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    else B200_FP4_MMA4("2", "mxf4nvf4.block_scale.scale_vec::4X");
#undef B200_FP4_MMA4
}

// 16 bytes of shared memory a lane to four columns of the warp's quarter of tensor memory, for kN addresses one after the other.
template <int kN>
B200_DEVICE void tmem_st_v4(uint32_t taddr, const uint4 (&v)[kN]) {
    static_assert(kN == 2 || kN == 4, "columns of one store");
    if constexpr (kN == 2)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"r"(taddr), "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w) : "memory");
    else
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                     ::"r"(taddr), "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w),
                       "r"(v[2].x), "r"(v[2].y), "r"(v[2].z), "r"(v[2].w), "r"(v[3].x), "r"(v[3].y), "r"(v[3].z), "r"(v[3].w) : "memory");
}

// Makes `bar` receive one arrival when every tcgen05.mma this thread issued so far has
// finished (implies tcgen05.fence::before_thread_sync).
B200_DEVICE void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace ptx
}  // namespace b200spmm
