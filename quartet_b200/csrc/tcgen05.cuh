// tcgen05 (5th-generation tensor core) wrappers: tensor-memory allocation, fences, commit, accumulator loads /
// stores, the shared-memory matrix descriptor of a K-major, 128-byte-swizzled operand, and what the GEMM kernels
// share: the bounded pipeline wait, the CTA-pair (cta_group::2) forms and the tile order.
#pragma once
#include "common.cuh"

namespace quartet {

__device__ __forceinline__ void tmem_alloc(uint32_t* dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// registers -> 4 / 8 consecutive TMEM columns of this warp's 32 lanes (one value per lane and column)
__device__ __forceinline__ void tc_st4(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, K-major operand, 128-byte swizzle: rows are 128 B apart,
// groups of 8 rows 1024 B apart.
__device__ __forceinline__ uint64_t make_desc_sw128(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);       // start address
    d |= (uint64_t)(1024 >> 4) << 32;                // stride byte offset (leading offset unused here)
    d |= (uint64_t)1 << 46;                          // descriptor version (sm_100)
    d |= (uint64_t)2 << 61;                          // SWIZZLE_128B
    return d;
}

// Bounded wait on wall-clock time (2 s), for the pipeline barriers.
__device__ __forceinline__ bool gemm_wait(uint64_t* bar, uint32_t parity, int32_t who, volatile int* dead) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*dead) return false;
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u) {
            uint64_t now;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
            if (t0 == 0) t0 = now;
            if (now - t0 > 2000000000ull || *dead) break;
        }
    }
    atomicOr(&g_status, who | 0x100);
    *dead = 1;
    return false;
}

// The same for a whole warp: its lanes poll for themselves, so they may leave the wait apart, and one may give up as another sees the
// barrier complete.  They go on together and with one answer, as warp-wide instructions (tcgen05.ld / st, elect.sync) and the warp's own
// barriers need it.
__device__ __forceinline__ bool gemm_wait_warp(uint64_t* bar, uint32_t parity, int32_t who, volatile int* dead) {
    return __all_sync(0xFFFFFFFFu, gemm_wait(bar, parity, who, dead));
}

// One lane of a fully converged warp (elect.sync): the issuing warp runs its loop on all 32 lanes so
// that ring indices, descriptors and addresses stay warp-uniform, and only the tcgen05 instructions
// themselves are predicated on the elected lane.
__device__ __forceinline__ bool elect_one() {
    uint32_t pred = 0;
    asm volatile(
        "{\n\t.reg .b32 rx;\n\t.reg .pred px;\n\t"
        "elect.sync rx|px, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, px;\n\t}"
        : "=r"(pred));
    return pred != 0;
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t mapa_u32(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    // default semantics (as the pipelines of CUTLASS use for consumer -> producer signalling across
    // CTAs); an explicit .release.cluster here costs ~1500 cycles per arrive
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_alloc2(uint32_t* dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish2() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// arrive, once all MMAs issued so far are done, on the barrier at this shared-memory offset in BOTH CTAs of the pair (one
// instruction instead of two commits; only the completion signal is multicast, no data copy)
__device__ __forceinline__ void tc_commit2_pair(uint32_t own_addr) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     own_addr),
                 "h"((uint16_t)3)
                 : "memory");
}
// Tile order of the persistent two-CTA kernel.  Tiles that run at the same time (consecutive
// indices) form a compact block of RASTER_BAND row pairs by as many column tiles, so that the rows of A
// and B a wave reads are few and each is shared by many CTAs while it is hot in the L2 of their die.
constexpr int RASTER_BAND = 8;
__device__ __forceinline__ void tile_coords(int tile, int m_pairs, int n_tiles, int& m_pair, int& n_blk) {
    const int per_band = RASTER_BAND * n_tiles;
    const int band = tile / per_band, within = tile - band * per_band;
    const int rows = min(RASTER_BAND, m_pairs - band * RASTER_BAND);
    n_blk = within / rows;
    m_pair = band * RASTER_BAND + (within - n_blk * rows);
}

}  // namespace quartet
