// 8-bit block-scaled product for sm_100a:  D[M, N] = alpha * A[M, K] . B[N, K]^T
//
//   A, B     e4m3 or e5m2 codes, K-major, row pitch K bytes (K a multiple of 128: the quantizer pads with zeros)
//   SFA/SFB  E8M0 scales, one byte per 32 values, in 512-byte blocks of 128 rows x 4 scales
//   D        bf16 or fp32, row pitch ldd elements
//
// tcgen05.mma.kind::mxf8f6f4.block_scale multiplies by the scales inside the tensor core, so a scale for each block of 128
// costs nothing beyond its bytes: the same byte stands for the four groups of 32.
//
// gemm_fp8_split_kernel: few rows of A, or a small result.  The roles are swapped -- 128 rows of B are the instruction's M
// and up to 256 rows of A its N -- so that a single token still feeds every row of the tensor core with one weight row, and
// the contraction is split over the CTAs of a cluster, which add their fp32 partial results in rank order through
// distributed shared memory: no workspace, no atomics, the same bits every time.  (Up to eight rows go to gemv_fp8.cu.)
#include "common.cuh"
#include "gemm_fp8.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>

#include <algorithm>

namespace quartet {

// Instruction descriptor, kind::mxf8f6f4, UE8M0 scales, both operands K-major.
__device__ __forceinline__ uint32_t make_idesc_fp8(int m, int n, int a_e5m2, int b_e5m2, uint32_t sf_id) {
    uint32_t d = 0;
    d |= sf_id << 4;                    // B scale id: byte of the 32-bit scale column
    d |= (uint32_t)a_e5m2 << 7;         // A format: 0 e4m3, 1 e5m2
    d |= (uint32_t)b_e5m2 << 10;        // B format
    d |= (uint32_t)(n >> 3) << 17;
    d |= 1u << 23;                      // scale format UE8M0
    d |= (uint32_t)(m >> 4) << 24;
    d |= sf_id << 29;                   // A scale id
    return d;
}
__device__ __forceinline__ void tc_mma_mxf8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        :
        : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
        : "memory");
}

// ---------------------------------------------------------------------------
// swapped roles, contraction split over a cluster
// ---------------------------------------------------------------------------
template <int BT, int CTAS>  // rows of A (tokens) a CTA takes; CTAs on an SM
struct SplitCfg {
    static constexpr int W_BYTES = 128 * 128;
    static constexpr int X_BYTES = BT * 128;
    static constexpr int X_BLOCKS = BT == 256 ? 2 : 1;                // scale blocks of 128 rows
    static constexpr int SF_BYTES = 512 * (1 + X_BLOCKS), SF_COLS = 4 * (1 + X_BLOCKS);
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + SF_BYTES;
    static constexpr int STAGES_FIT = (CTAS == 2 ? 112 : 226) * 1024 / STAGE_BYTES, STAGES = CTAS == 1 || STAGES_FIT < 5 ? STAGES_FIT : 5;
    static constexpr int SF_COL0 = BT;
    static constexpr int TMEM_COLS = BT == 256 ? 512 : BT == 128 ? 256 : 128;  // BT accumulator columns and the scales' of each stage
    static constexpr int SMEM = STAGES * STAGE_BYTES + 512;
    static_assert(SF_COL0 + STAGES * SF_COLS <= TMEM_COLS, "tensor memory capacity");
    static_assert(STAGES * (W_BYTES + X_BYTES) >= BT * 128 * 4, "the partial result reuses the operand stages");
    static_assert(SMEM <= (CTAS == 2 ? 113 : 227) * 1024, "CTAs of an SM");
};

constexpr int SPLIT_THREADS = 256, SPLIT_MAX = 8;  // warps 0, 2, 3 issue copies (weight, A, scales), 1 the MMAs; 4-7 feed scales, then drain

// The sum of the cluster's partial results, in rank order.  The tokens' results, four side by side, are dealt out over the threads of the whole
// cluster; a thread has eight reads on their way at a time (200 rows, K and N 4096: 12.7 us, 13.6 with one position at a time).
template <int S>
__device__ __forceinline__ void split_finish(uint32_t red_addr, const Fp8GemmParams& p, int rank, int64_t t0, int tokens, int64_t n_first) {
    constexpr int U = SPLIT_MAX / S, STEP = S * SPLIT_THREADS;
    const int64_t n0 = n_first + (threadIdx.x & 31) * 4;
    if (n0 >= p.N) return;
    for (int i0 = rank * SPLIT_THREADS + threadIdx.x; i0 < tokens * 32; i0 += U * STEP) {
        float4 q[U][S];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (i0 + u * STEP < tokens * 32) {
                    const uint32_t at = red_addr + (i0 + u * STEP) * 16;
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(q[u][s].x), "=f"(q[u][s].y), "=f"(q[u][s].z), "=f"(q[u][s].w)
                                 : "r"(S == 1 ? at : mapa_u32(at, s))
                                 : "memory");
                }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * STEP;
            if (i >= tokens * 32) break;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) v[0] += q[u][s].x, v[1] += q[u][s].y, v[2] += q[u][s].z, v[3] += q[u][s].w;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] *= p.alpha;
            const int64_t at = (t0 + (i >> 5)) * p.ldd + n0;
            if (p.d_f32) {
                float* d = static_cast<float*>(p.d) + at;
                if (n0 + 4 <= p.N)
                    *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
                else
                    for (int k = 0; k < 4 && n0 + k < p.N; ++k) d[k] = v[k];
            } else {
                __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.d) + at;
                if (n0 + 4 <= p.N) {
                    __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
                    *reinterpret_cast<uint2*>(d) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
                } else {
                    for (int k = 0; k < 4 && n0 + k < p.N; ++k) d[k] = __float2bfloat16_rn(v[k]);
                }
            }
        }
    }
}

template <int BT, int CTAS>
__global__ void __launch_bounds__(SPLIT_THREADS, CTAS) gemm_fp8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                         const Fp8GemmParams p, const int splits) {
    using C = SplitCfg<BT, CTAS>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        // uniform over the grid: no CTA of the cluster gets further
        if (threadIdx.x == 0) atomicOr(&g_status, WAIT_GEMM_ALIGN | 0x100);
        return;
    }
    uint8_t* s_w = smem;
    uint8_t* s_x = s_w + C::STAGES * C::W_BYTES;
    uint8_t* s_sf = s_x + C::STAGES * C::X_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_sf + C::STAGES * C::SF_BYTES);
    uint64_t* empty = full + C::STAGES;
    uint64_t* sf_land = empty + C::STAGES;
    uint64_t* sf_full = sf_land + C::STAGES;
    uint64_t* acc_full = sf_full + C::STAGES;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(acc_full + 1);
    volatile int* dead = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % splits;          // the cluster spans the split axis
    const int n_blk = (int)blockIdx.x / splits, t_blk = blockIdx.y, x_blocks = (int)((p.M + 127) / 128);
    const int c0 = (int)((int64_t)p.k_chunks * rank / splits), c1 = (int)((int64_t)p.k_chunks * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 2);
            mbar_init(&empty[i], 1);
            mbar_init(&sf_land[i], 1);
            mbar_init(&sf_full[i], 4);
        }
        mbar_init(acc_full, 1);
        *dead = 0;
        fence_mbar_init();
        prefetch_tmap(&tm_w);
        prefetch_tmap(&tm_x);
    }
    if (warp == 1) {
        tmem_alloc(s_tmem, C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    if (warp == 1) {
        // the loop runs on all lanes and only the instructions themselves on an elected one: addresses and descriptors then stay in
        // uniform registers (590 cycles a chunk on one lane alone, 545 so: the four MMAs' own pace, whatever their N up to 64)
        const uint32_t w_base = smem_u32(s_w), x_base = smem_u32(s_x);
        const uint32_t id0 = make_idesc_fp8(128, BT, p.b_e5m2, p.a_e5m2, 0), id1 = make_idesc_fp8(128, BT, p.b_e5m2, p.a_e5m2, 1);
        const uint32_t id2 = make_idesc_fp8(128, BT, p.b_e5m2, p.a_e5m2, 2), id3 = make_idesc_fp8(128, BT, p.b_e5m2, p.a_e5m2, 3);
        uint32_t s = 0, ph = 0;
        for (int c = c0; c < c1; ++c) {
            if (!gemm_wait(&sf_full[s], ph, WAIT_GEMM_SF, dead)) break;
            if (!gemm_wait(&full[s], ph, WAIT_GEMM_FULL, dead)) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t sf = tmem + C::SF_COL0 + s * C::SF_COLS;
                const uint64_t wd = make_desc_sw128(w_base + s * C::W_BYTES), xd = make_desc_sw128(x_base + s * C::X_BYTES);
                tc_mma_mxf8(tmem, wd, xd, id0, sf, sf + 4, c != c0);  // 32 values a step, one scale byte each
                tc_mma_mxf8(tmem, wd + 2, xd + 2, id1, sf | (1u << 30), (sf + 4) | (1u << 30), 1);
                tc_mma_mxf8(tmem, wd + 4, xd + 4, id2, sf | (2u << 30), (sf + 4) | (2u << 30), 1);
                tc_mma_mxf8(tmem, wd + 6, xd + 6, id3, sf | (3u << 30), (sf + 4) | (3u << 30), 1);
                tc_commit(&empty[s]);
            }
            __syncwarp();
            if (++s == C::STAGES) s = 0, ph ^= 1;
        }
        if (elect_one()) tc_commit(acc_full);
        __syncwarp();
    } else if (warp < 4) {
        // three threads in three warps: one thread starts a copy only every few hundred cycles
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (int c = c0; c < c1; ++c) {
                if (!gemm_wait(&empty[s], ph ^ 1, WAIT_GEMM_EMPTY, dead)) break;
                if (warp == 0) {
                    mbar_arrive_expect_tx(&full[s], C::W_BYTES);
                    tma_load_2d(s_w + s * C::W_BYTES, &tm_w, c * 128, n_blk * 128, &full[s]);
                } else if (warp == 2) {
                    mbar_arrive_expect_tx(&full[s], C::X_BYTES);
                    tma_load_2d(s_x + s * C::X_BYTES, &tm_x, c * 128, t_blk * BT, &full[s]);
                } else {
                    uint8_t* dst = s_sf + s * C::SF_BYTES;
                    mbar_arrive_expect_tx(&sf_land[s], C::SF_BYTES);
                    bulk_load(dst, p.b_sf + ((int64_t)n_blk * p.k_chunks + c) * 512, 512, &sf_land[s]);
                    bulk_load(dst + 512, p.a_sf + ((int64_t)(t_blk * BT / 128) * p.k_chunks + c) * 512, 512, &sf_land[s]);
                    // rows past the last block are zeros; its scales stand in for theirs, there being none
                    if (C::X_BLOCKS == 2) bulk_load(dst + 1024, p.a_sf + ((int64_t)min(t_blk * 2 + 1, x_blocks - 1) * p.k_chunks + c) * 512, 512, &sf_land[s]);
                }
                if (++s == C::STAGES) s = 0, ph ^= 1;
            }
        }
    } else {
        // Scales go to tensor memory through registers, a warp per lane quadrant.  (A copy issued among the MMAs orders itself with them:
        // the chain copy -> MMA -> copy took 745 cycles a stage, whatever the number of stages or of issuing threads.)
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t s = 0, ph = 0;
        for (int c = c0; c < c1; ++c) {
            if (!gemm_wait(&sf_land[s], ph, WAIT_GEMM_FULL, dead)) break;
            const uint4* sf = reinterpret_cast<const uint4*>(s_sf + s * C::SF_BYTES) + lane;
            const uint4 w4 = sf[0], x4 = sf[32];
            const uint32_t v[8] = {w4.x, w4.y, w4.z, w4.w, x4.x, x4.y, x4.z, x4.w};
            __syncwarp();  // (a wait's lanes may leave it apart; tensor-memory instructions are the warp's)
            tc_st8(tmem + lane_base + C::SF_COL0 + s * C::SF_COLS, v);
            if constexpr (C::X_BLOCKS == 2) {
                const uint4 z4 = sf[64];
                const uint32_t z[8] = {z4.x, z4.y, z4.z, z4.w, 0, 0, 0, 0};
                tc_st4(tmem + lane_base + C::SF_COL0 + s * C::SF_COLS + 8, z);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sf_full[s]);
            if (++s == C::STAGES) s = 0, ph ^= 1;
        }
    }
    __syncwarp();
    // ---- partial results [token][weight row] in fp32 over the operand stages: all copies have landed and been read ----
    const bool ok = gemm_wait_warp(acc_full, 0, WAIT_GEMM_ACC_FULL, dead);
    tc_fence_after();
    float* red = reinterpret_cast<float*>(smem);
    const int row = (warp & 3) * 32 + lane;
    const int64_t t0 = (int64_t)t_blk * BT;
    const int tokens = (int)(p.M - t0 < BT ? p.M - t0 : BT);
    __syncthreads();
    if (ok) {
        // two warps per lane quadrant take turns
#pragma unroll 1
        for (int cb = (warp >> 2) * 32; cb < tokens; cb += 64) {
            uint32_t r[32];
            tc_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + cb, r);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (cb + i < tokens) red[(cb + i) * 128 + row] = __uint_as_float(r[i]);
        }
    }
    tc_fence_before();
    if (splits > 1)
        cluster_sync_all();
    else
        __syncthreads();
    if (ok) {
        const uint32_t red_addr = smem_u32(red);
        const int64_t n0 = (int64_t)n_blk * 128;
        if (splits == 1) split_finish<1>(red_addr, p, rank, t0, tokens, n0);
        else if (splits == 2) split_finish<2>(red_addr, p, rank, t0, tokens, n0);
        else if (splits == 4) split_finish<4>(red_addr, p, rank, t0, tokens, n0);
        else split_finish<8>(red_addr, p, rank, t0, tokens, n0);
    }
    if (splits > 1) cluster_sync_all();  // no CTA leaves while a peer may still read its partial results
    __syncthreads();
    if (*dead)
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies still in flight land before shared memory is released
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

template <int BT, int CTAS>
static int launch_split(const uint8_t* a, const uint8_t* b, int64_t K, const Fp8GemmParams& p, int splits, cudaStream_t stream) {
    using C = SplitCfg<BT, CTAS>;
    CUtensorMap tm_w, tm_x;
    int rc = make_tmap_2d(&tm_w, b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.N, K, 128, 128, 3);
    if (rc) return rc;
    if ((rc = make_tmap_2d(&tm_x, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.M, K, 128, BT, 3))) return rc;
    auto kern = gemm_fp8_split_kernel<BT, CTAS>;
    static thread_local int smem_set = -1;
    if ((rc = set_max_smem_once(kern, C::SMEM, smem_set))) return rc;
    const int64_t n_tiles = (p.N + 127) / 128, t_tiles = (p.M + BT - 1) / BT;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_tiles * splits), (unsigned)t_tiles);
    cfg.blockDim = dim3(SPLIT_THREADS), cfg.dynamicSmemBytes = C::SMEM, cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)splits, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    return check_cuda(cudaLaunchKernelEx(&cfg, kern, tm_w, tm_x, p, splits), "gemm_fp8 launch");
}

// ---------------------------------------------------------------------------
// CTA pairs (cta_group::2): 256 x 256 results a pair, persistent
//
// Narrower tiles would fill the last wave better where N is a small multiple of 64 or 32, but a product of 160 columns takes 0.83 of the time of one
// of 256: 8192 x 8192 x 4096 in 198 us, 227 with 192 columns, 263 with 160; 4096 x 640 x 32000 in 86, 89 and 92.
// ---------------------------------------------------------------------------
struct PairCfg {
    static constexpr int BN = 256;
    static constexpr int A_BYTES = 128 * 128;                // this CTA's rows of A, 128 values
    static constexpr int B_BYTES = 128 * 128;                // this CTA's half of B's rows
    static constexpr int SFA_BYTES = 512, SFB_BYTES = 1024;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
    static constexpr int STG_BYTES = 8 * 4096;               // a staging buffer for each epilogue warp
    static constexpr int STAGES = (232448 - STG_BYTES - 512) / STAGE_BYTES;
    static constexpr int SMEM = STAGES * STAGE_BYTES + STG_BYTES + 512;
    // Consecutive tiles accumulate in columns [0, 256) and [128, 384): the 128 they share are drained into registers first, so
    // that the next tile's products start while the rest of the epilogue still runs.
    static constexpr int ACC_SHIFT = 128;
    static constexpr int SF_COL0 = 384, SF_COLS = 12, SF_SLOTS = 4;
    static_assert(SF_COL0 + SF_SLOTS * SF_COLS <= 512, "tensor memory capacity");
    static_assert(SF_SLOTS < STAGES, "scale slots are recycled through the stage barriers");
};
constexpr int PAIR_THREADS = 512;  // warps 0, 10, 15 issue copies (A, B, scales), 1 the MMAs, 6-9 feed scales, 2-5 and 11-14 drain

__device__ __forceinline__ void tc_mma2_mxf8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        :
        : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
        : "memory");
}

// 32 rows x 64 columns of results, one row per thread, through 4 KB of swizzled staging to global memory: one tensor store of 64 bf16
// columns or two of 32 fp32 columns, 128 bytes a row.  A tensor store clips only to whole 16-byte units of a row (measured: the rest of the last
// unit is written as zeros), so the tensor map ends with the last whole unit, at n_whole, and the few columns behind it are written value by value.
__device__ __forceinline__ void store_block64(const uint32_t (&r0)[32], const uint32_t (&r1)[32], const Fp8GemmParams& p, const CUtensorMap* tm_d, int row0,
                                              int col, uint8_t* stg, int lane) {
    const int n_whole = (int)p.N & (p.d_f32 ? ~3 : ~7);
    if (n_whole < p.N && col + 64 > n_whole) {
        const int64_t row = (int64_t)row0 + lane;
        if (row < p.M) {
#pragma unroll
            for (int i = 0; i < 64; ++i) {
                if (col + i < n_whole || col + i >= p.N) continue;
                const float v = __uint_as_float(i < 32 ? r0[i & 31] : r1[i & 31]) * p.alpha;
                if (p.d_f32)
                    static_cast<float*>(p.d)[row * p.ldd + col + i] = v;
                else
                    static_cast<__nv_bfloat16*>(p.d)[row * p.ldd + col + i] = __float2bfloat16_rn(v);
            }
        }
    }
    if (col >= n_whole) return;
    auto staging_free = [&]() {  // the store before has been read from it
        if (lane == 0) bulk_wait_read0();
        __syncwarp();
    };
    auto send = [&](int c) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(tm_d, c, row0, stg);
            bulk_commit();
        }
    };
    if (p.d_f32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (col + 32 * h >= n_whole) break;
            staging_free();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(h ? r1[4 * j + k] : r0[4 * j + k]) * p.alpha;
                *reinterpret_cast<float4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
            }
            send(col + 32 * h);
        }
    } else {
        staging_free();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = (8 * j + 2 * k) & 31;
                const __nv_bfloat162 t = __floats2bfloat162_rn(__uint_as_float(j < 4 ? r0[i] : r1[i]) * p.alpha, __uint_as_float(j < 4 ? r0[i + 1] : r1[i + 1]) * p.alpha);
                w[k] = *reinterpret_cast<const uint32_t*>(&t);
            }
            *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        send(col);
    }
}

// One product, or two that do not depend on one another: the second one's tiles fill the pairs that the first one's last round leaves idle.
struct PairMaps {
    CUtensorMap a, b, d, sfb;
};
struct PairSecond {
    PairMaps tm;
    Fp8GemmParams g;
    int extra;  // how many of its tiles take as long as one of the first product's
};
__device__ __forceinline__ int pair_rows(const Fp8GemmParams& p) { return (int)((p.M + 255) / 256); }
__device__ __forceinline__ int pair_cols(const Fp8GemmParams& p) { return (int)((p.N + 255) / 256); }

// The tiles of a pair of CTAs.  The first product's are dealt out in rounds; of the second one's, the pairs that the last of these rounds left out
// take `extra` each, and all take the rest in rounds that begin with them.
template <bool TWO>
struct PairTiles {
    int n, tiles0, tiles1, first1, step1, end1, first2, at, stage = 0;
    __device__ __forceinline__ PairTiles(int t0, int t1, int extra, int pair, int n_pairs) : n(n_pairs), tiles0(t0), tiles1(t1), at(pair) {
        if (!TWO) return;
        const int busy = tiles0 % n;                 // pairs that the last round takes; 0: all
        step1 = n - busy;
        end1 = busy ? min(tiles1, step1 * extra) : 0;
        first1 = pair >= busy ? pair - busy : end1;
        first2 = end1 + (pair >= busy ? pair - busy : pair + step1);
    }
    __device__ __forceinline__ bool next(int& product, int& tile) {
        if (!TWO) {
            product = 0, tile = at, at += n;
            return tile < tiles0;
        }
        if (stage == 0 && at >= tiles0) stage = 1, at = first1;
        if (stage == 1 && at >= end1) stage = 2, at = first2;
        product = stage > 0, tile = at;
        at += stage == 1 ? step1 : n;
        return stage < 2 || tile < tiles1;
    }
};

template <bool TWO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_d,
                         const __grid_constant__ CUtensorMap tm_sfb, const Fp8GemmParams p0, const __grid_constant__ PairSecond p1) {
    using C = PairCfg;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(&g_status, WAIT_GEMM_ALIGN | 0x100);
        return;
    }
    uint8_t* s_a = smem;
    uint8_t* s_b = s_a + C::STAGES * C::A_BYTES;
    uint8_t* s_stg = s_b + C::STAGES * C::B_BYTES;
    uint8_t* s_sfb = s_stg + C::STG_BYTES;
    uint8_t* s_sfa = s_sfb + C::STAGES * C::SFB_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_sfa + C::STAGES * C::SFA_BYTES);
    uint64_t* full = bars;                       // local: this CTA's copies of a stage have landed
    uint64_t* empty = full + C::STAGES;          // local: the pair's MMAs are done with the stage
    uint64_t* sf_full = empty + C::STAGES;       // leader: 8 feeder warps (both CTAs) have fed the stage
    uint64_t* sf_land = sf_full + C::STAGES;     // local: the stage's scale blocks have landed
    uint64_t* sf_free = sf_land + C::STAGES;     // local: the 4 feeder warps have the stage's scales in tensor memory
    uint64_t* acc_full = sf_free + C::STAGES;    // local: accumulator complete
    uint64_t* acc_empty = acc_full + 1;          // leader: 16 epilogue warps (both CTAs) have drained the shared columns
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(acc_empty + 1);
    volatile int* dead = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 2);
            mbar_init(&empty[i], 1);
            mbar_init(&sf_full[i], 8);
            mbar_init(&sf_land[i], 1);
            mbar_init(&sf_free[i], 4);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);
        *dead = 0;
        fence_mbar_init();
        prefetch_tmap(&tm_a);
        prefetch_tmap(&tm_b);
        prefetch_tmap(&tm_d);
        prefetch_tmap(&tm_sfb);
    }
    __syncthreads();
    if (warp == 1) {
        tmem_alloc2(s_tmem, 512);
        tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    const int m_pairs0 = pair_rows(p0), n_tiles0 = pair_cols(p0), k_stages0 = p0.k_chunks;
    PairTiles<TWO> tiles(m_pairs0 * n_tiles0, TWO ? pair_rows(p1.g) * pair_cols(p1.g) : 0, TWO ? p1.extra : 0, blockIdx.x >> 1, gridDim.x >> 1);
    int product, tile, m_pair, n_blk;
    auto second = [&]() { return TWO && product; };
    auto coords = [&]() { tile_coords(tile, second() ? pair_rows(p1.g) : m_pairs0, second() ? pair_cols(p1.g) : n_tiles0, m_pair, n_blk); };

    if (warp == 0 || warp == 10 || warp == 15) {
        if (lane == 0) {
            const int role = warp == 0 ? 0 : (warp == 10 ? 1 : 2);
            const uint64_t keep = l2_policy_evict_last();
            uint32_t s = 0, ph = 0;
            while (!*dead && tiles.next(product, tile)) {
                const Fp8GemmParams& p = second() ? p1.g : p0;
                const int k_stages = second() ? p1.g.k_chunks : k_stages0;
                coords();
                const int m_blocks = (int)((p.M + 127) / 128);
                const int m_blk = m_pair * 2 + (int)rank;
                const int n0 = n_blk * C::BN;
                // a second row block past the last one reads zero rows; its scales are the last block's, there being none of its own
                const uint8_t* sfa_src = p.a_sf + (int64_t)min(m_blk, m_blocks - 1) * p.k_chunks * 512;
                for (int ks = 0; ks < k_stages; ++ks) {
                    if (!gemm_wait(role == 2 ? &sf_free[s] : &empty[s], ph ^ 1, WAIT_GEMM_EMPTY, dead)) break;
                    if (role == 0) {
                        mbar_arrive_expect_tx(&full[s], C::A_BYTES);
                        tma_load_2d_hint(s_a + s * C::A_BYTES, second() ? &p1.tm.a : &tm_a, ks * 128, m_blk * 128, &full[s], keep);
                    } else if (role == 1) {
                        mbar_arrive_expect_tx(&full[s], C::B_BYTES);
                        tma_load_2d_hint(s_b + s * C::B_BYTES, second() ? &p1.tm.b : &tm_b, ks * 128, n0 + (int)rank * 128, &full[s], keep);
                    } else {
                        mbar_arrive_expect_tx(&sf_land[s], C::SFA_BYTES + C::SFB_BYTES);
                        bulk_load_hint(s_sfa + s * C::SFA_BYTES, sfa_src + (int64_t)ks * 512, C::SFA_BYTES, &sf_land[s], keep);
                        tma_load_2d_hint(s_sfb + s * C::SFB_BYTES, second() ? &p1.tm.sfb : &tm_sfb, ks * 128, n0 / 128, &sf_land[s], keep);
                    }
                    if (++s == C::STAGES) s = 0, ph ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (leader) {
            uint32_t s = 0, ph = 0, slot = 0, aph = 0, acc_it = 0;
            const uint32_t a_base = smem_u32(s_a), b_base = smem_u32(s_b);
            const uint32_t empty_own = smem_u32(&empty[0]), accf_own = smem_u32(acc_full);
            while (!*dead && tiles.next(product, tile)) {
                const Fp8GemmParams& p = second() ? p1.g : p0;
                const int k_stages = second() ? p1.g.k_chunks : k_stages0;
                const uint32_t id0 = make_idesc_fp8(256, C::BN, p.a_e5m2, p.b_e5m2, 0), id1 = make_idesc_fp8(256, C::BN, p.a_e5m2, p.b_e5m2, 1);
                const uint32_t id2 = make_idesc_fp8(256, C::BN, p.a_e5m2, p.b_e5m2, 2), id3 = make_idesc_fp8(256, C::BN, p.a_e5m2, p.b_e5m2, 3);
                if (!gemm_wait(acc_empty, aph ^ 1, WAIT_GEMM_ACC_EMPTY, dead)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (acc_it & 1) * C::ACC_SHIFT;
                ++acc_it;
                for (int ks = 0; ks < k_stages; ++ks) {
                    if (!gemm_wait(&sf_full[s], ph, WAIT_GEMM_SF, dead)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t sf = tmem_base + C::SF_COL0 + slot * C::SF_COLS;
                        const uint64_t ad = make_desc_sw128(a_base + s * C::A_BYTES), bd = make_desc_sw128(b_base + s * C::B_BYTES);
                        tc_mma2_mxf8(d_tmem, ad, bd, id0, sf, sf + 4, ks != 0);
                        tc_mma2_mxf8(d_tmem, ad + 2, bd + 2, id1, sf | (1u << 30), (sf + 4) | (1u << 30), 1);
                        tc_mma2_mxf8(d_tmem, ad + 4, bd + 4, id2, sf | (2u << 30), (sf + 4) | (2u << 30), 1);
                        tc_mma2_mxf8(d_tmem, ad + 6, bd + 6, id3, sf | (3u << 30), (sf + 4) | (3u << 30), 1);
                        tc_commit2_pair(empty_own + s * 8);
                    }
                    __syncwarp();
                    if (++s == C::STAGES) s = 0, ph ^= 1;
                    if (++slot == C::SF_SLOTS) slot = 0;
                }
                if (elect_one()) tc_commit2_pair(accf_own);
                __syncwarp();
                aph ^= 1;
            }
        }
    } else if (warp >= 6 && warp <= 9) {
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t it = 0;
        while (!*dead && tiles.next(product, tile)) {
            const int k_stages = second() ? p1.g.k_chunks : k_stages0;
            for (int ks = 0; ks < k_stages; ++ks, ++it) {
                const int s = it % C::STAGES;
                const uint32_t ph = (it / C::STAGES) & 1;
                if (!gemm_wait(&sf_land[s], ph, WAIT_GEMM_FULL, dead)) break;
                const uint32_t sf = tmem_base + lane_base + C::SF_COL0 + (it % C::SF_SLOTS) * C::SF_COLS;
                const uint4 va = *reinterpret_cast<const uint4*>(s_sfa + s * C::SFA_BYTES + lane * 16);
                const uint4 v0 = *reinterpret_cast<const uint4*>(s_sfb + s * C::SFB_BYTES + lane * 16);
                const uint4 v1 = *reinterpret_cast<const uint4*>(s_sfb + s * C::SFB_BYTES + 512 + lane * 16);
                const uint32_t ra[8] = {va.x, va.y, va.z, va.w, 0, 0, 0, 0}, rb[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                if (it >= (uint32_t)C::SF_SLOTS) {
                    const uint32_t pit = it - C::SF_SLOTS;
                    if (!gemm_wait(&empty[pit % C::STAGES], (pit / C::STAGES) & 1, WAIT_GEMM_EMPTY, dead)) break;
                    tc_fence_after();
                }
                __syncwarp();  // (a wait's lanes may leave it apart; tensor-memory instructions are the warp's)
                tc_st4(sf, ra);
                tc_st8(sf + 4, rb);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                // Only now is the buffer given back, when the scales have left it for certain.  An arrive behind the loads alone let the copy of five
                // chunks later overtake them where operands were late: scales of chunk c + 5 on chunk c in one of some 200 products from cold memory.
                if (lane == 0) mbar_arrive(&sf_free[s]);
                if (!gemm_wait(&full[s], ph, WAIT_GEMM_FULL, dead)) break;
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&sf_full[s]), 0));
            }
        }
    } else {
        // two warps per lane quadrant; each takes one 64-column block of the shared half of the accumulator, then one of the other half
        const int q = warp & 3, par = warp >= 11 ? 1 : 0;
        uint8_t* stg = s_stg + (par * 4 + q) * 4096;
        uint32_t acc_it = 0;
        for (; !*dead && tiles.next(product, tile); ++acc_it) {
            const Fp8GemmParams& p = second() ? p1.g : p0;
            const CUtensorMap* d_map = second() ? &p1.tm.d : &tm_d;
            coords();
            const int n0 = n_blk * C::BN;
            const int row0 = (m_pair * 2 + (int)rank) * 128 + q * 32;
            if (!gemm_wait_warp(acc_full, acc_it & 1, WAIT_GEMM_ACC_FULL, dead)) break;
            tc_fence_after();
            const uint32_t t0 = tmem_base + ((uint32_t)(q * 32) << 16) + (acc_it & 1) * C::ACC_SHIFT;
            const int first = (acc_it & 1) ? 0 : 128;         // the half that the next tile's accumulator overlaps
            const int c0 = first + par * 64, c1 = (first ^ 128) + par * 64;
            uint32_t r0[32], r1[32];
            tc_ld32(t0 + c0, r0);
            tc_ld32(t0 + c0 + 32, r1);
            tc_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(acc_empty), 0));
            const bool rows = row0 < p.M;
            if (rows && n0 + c0 < p.N) store_block64(r0, r1, p, d_map, row0, n0 + c0, stg, lane);
            tc_ld32(t0 + c1, r0);
            tc_ld32(t0 + c1 + 32, r1);
            tc_wait_ld();
            if (rows && n0 + c1 < p.N) store_block64(r0, r1, p, d_map, row0, n0 + c1, stg, lane);
            tc_fence_before();  // all of this tile's tensor-memory reads are complete before the warp's next arrive
        }
        if (lane == 0) bulk_wait0();
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*dead)
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc2(tmem_base, 512);
    }
}

static int pair_maps(PairMaps* m, const Fp8Product& x) {
    const Fp8GemmParams& p = x.g;
    const int64_t K = (int64_t)p.k_chunks * 128;
    int rc = make_tmap_2d(&m->a, x.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.M, K, 128, 128, 3);
    if (rc) return rc;
    if ((rc = make_tmap_2d(&m->b, x.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.N, K, 128, 128, 3))) return rc;
    if (p.d_f32)
        rc = make_tmap_2d(&m->d, p.d, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.N & ~(int64_t)3, p.M, (uint64_t)p.ldd * 4, 32, 32, 3);
    else
        rc = make_tmap_2d(&m->d, p.d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.N & ~(int64_t)7, p.M, (uint64_t)p.ldd * 2, 64, 32, 3);
    if (rc) return rc;
    // B's scales as 32-bit words: a row for each 128-row block, 128 words a chunk; a stage takes one chunk of two row blocks
    return make_tmap_2d(&m->sfb, p.b_sf, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, (uint64_t)p.k_chunks * 128, (uint64_t)((p.N + 127) / 128), (uint64_t)p.k_chunks * 512, 128,
                        2, 0);
}

// One product, or two of which the first has the longer contraction.
template <bool TWO>
static int launch_pair(const Fp8Product* x, cudaStream_t stream) {
    using C = PairCfg;
    PairMaps first;
    PairSecond second{};
    int64_t tiles = 0;
    int rc = pair_maps(&first, x[0]);
    if (rc || (TWO && (rc = pair_maps(&second.tm, x[1])))) return rc;
    for (int i = 0; i < (TWO ? 2 : 1); ++i) tiles += ((x[i].g.M + 255) / 256) * ((x[i].g.N + 255) / 256);
    if (TWO) second.g = x[1].g, second.extra = x[0].g.k_chunks / x[1].g.k_chunks;
    auto kern = gemm_fp8_pair_kernel<TWO>;
    static thread_local int smem_set = -1;
    if ((rc = set_max_smem_once(kern, C::SMEM, smem_set))) return rc;
    int dev = 0, sms = 0;
    if ((rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice"))) return rc;
    if ((rc = device_sm_count(&sms))) return rc;
    // a persistent kernel launches no more clusters than can be resident at once
    static thread_local int cached_dev = -1, cached_clusters = 0;
    if (cached_dev != dev) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)sms), cfg.blockDim = dim3(PAIR_THREADS), cfg.dynamicSmemBytes = C::SMEM;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
        cfg.attrs = &attr, cfg.numAttrs = 1;
        int n = 0;
        if ((rc = check_cuda(cudaOccupancyMaxActiveClusters(&n, kern, &cfg), "cudaOccupancyMaxActiveClusters"))) return rc;
        if (n < 1) return fail(QUARTET_E_CUDA, "no CTA pair can be resident");
        cached_dev = dev, cached_clusters = n;
    }
    const int clusters = (int)(tiles < cached_clusters ? tiles : cached_clusters);
    return check_cuda(launch_pdl(kern, dim3(clusters * 2), dim3(PAIR_THREADS), C::SMEM, stream, first.a, first.b, first.d, first.sfb, x[0].g, second), "gemm_fp8 launch");
}

QUARTET_DEFINE_STATUS_READER(status_gemm_fp8)

// How many clusters of 1, 2, 4 and 8 CTAs can be resident at one CTA to an SM (148, 74, 33 and 15 here: clusters do not cross a group of SMs).
static int resident_clusters(const int (**out)[4]) {
    static thread_local int cached_dev = -1, cached[4];
    int dev = 0, rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc) return rc;
    if (cached_dev != dev) {
        using C = SplitCfg<128, 1>;
        auto kern = gemm_fp8_split_kernel<128, 1>;
        static thread_local int smem_set = -1;
        if ((rc = set_max_smem_once(kern, C::SMEM, smem_set))) return rc;
        for (int i = 0; i < 4; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(8), cfg.blockDim = dim3(SPLIT_THREADS), cfg.dynamicSmemBytes = C::SMEM;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 1u << i, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
            cfg.attrs = &attr, cfg.numAttrs = 1;
            if ((rc = check_cuda(cudaOccupancyMaxActiveClusters(&cached[i], kern, &cfg), "cudaOccupancyMaxActiveClusters"))) return rc;
            if (i == 0 && cached[i] < 1) return fail(QUARTET_E_CUDA, "no CTA can be resident");
        }
        cached_dev = dev;
    }
    *out = &cached;
    return QUARTET_OK;
}

// Which kernel, and how many ways the contraction is split.  Up to eight rows: the stream over B (both sides' times are in gemv_fp8.cu).  Else the way that takes the least by a model in
// units of 40 ns: a round of resident tiles takes `chunk` for every 128 values of its part of the contraction and `start` for its beginning and end, of
// which a persistent kernel pays `again` in its later rounds, and a cluster that adds partial results takes `join` more.
// Over 84 shapes (M 9 to 32000, N 100 to 32000, K 128 to 32000) the way taken is 2 % behind the best one on average, 19 % at most.
//     us, best split of each            pairs    256 rows   128 rows   128 rows, two CTAs on an SM
//     200 x 640, K 4096                  14.3      10.0        7.7         8.4
//     256 x 4096, K 11008                32.1      18.9       21.0        19.8
//     300 x 11000, K 640                 10.1      10.6       11.3         7.9
//     512 x 4096, K 640                   7.1       7.9        6.3         7.2
//     8000 x 640, K 4096                 27.4      35.2       42.9        32.3
constexpr struct { int chunk, start, again; } COST_PAIR{6, 115, 35};
constexpr struct { int chunk, start, join; } COST_256{6, 140, 30}, COST_128{5, 105, 30}, COST_128_TWO{5, 150, 30}, COST_FEW{5, 150, 8};

enum class Way {
    FEW_TOKENS = QUARTET_FP8_STREAM,
    PAIR = QUARTET_FP8_PAIRS,
    ROWS_256 = QUARTET_FP8_ROWS_256,
    ROWS_128 = QUARTET_FP8_ROWS_128,
    ROWS_128_TWO = QUARTET_FP8_ROWS_128_TWO,
    ROWS_FEW = QUARTET_FP8_ROWS_FEW
};

static int pick_way(const Fp8GemmParams& p, Way* way, int* splits, int64_t* cost) {
    *way = Way::FEW_TOKENS, *splits = 1, *cost = 0;
    if (gemv_fits(p.M, (int64_t)p.k_chunks * 128)) return QUARTET_OK;
    const int (*resident)[4] = nullptr;
    int rc = resident_clusters(&resident);
    if (rc) return rc;
    auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    *cost = INT64_MAX;
    auto consider = [&](Way w, int sp, int64_t c) {
        if (c < *cost) *cost = c, *way = w, *splits = sp;
    };
    const int64_t n_tiles = ceil_div(p.N, 128);
    if (p.M > 64 && p.N >= 64) {
        const int64_t rounds = ceil_div(ceil_div(p.M, 256) * ceil_div(p.N, 256), (*resident)[1]);
        consider(Way::PAIR, 1, rounds * COST_PAIR.chunk * p.k_chunks + COST_PAIR.start + (rounds - 1) * COST_PAIR.again);
    }
    for (int i = 0; i < 4 && (1 << i) <= p.k_chunks && (*resident)[i] > 0; ++i) {
        const int sp = 1 << i;
        const int64_t chunks = ceil_div(p.k_chunks, sp), slots = (*resident)[i];
        auto start = [&](const auto& c) { return c.start + (sp > 1 ? c.join : 0); };
        if (p.M > 64) {
            const int64_t rounds = ceil_div(n_tiles * ceil_div(p.M, 128), slots), rounds_256 = ceil_div(n_tiles * ceil_div(p.M, 256), slots);
            if (p.M > 128 && sp < 8) consider(Way::ROWS_256, sp, rounds_256 * (COST_256.chunk * chunks + start(COST_256)));
            consider(Way::ROWS_128, sp, rounds * (COST_128.chunk * chunks + start(COST_128)));
            // two CTAs on an SM share its tensor core, but the beginning and end of one run under the other's products
            consider(Way::ROWS_128_TWO, sp, rounds * COST_128_TWO.chunk * chunks + (rounds + 1) / 2 * start(COST_128_TWO));
        } else {
            // with few rows the second one costs three quarters of a round: they wait for memory more than for the tensor core
            const int64_t rounds = ceil_div(n_tiles * ceil_div(p.M, p.M > 32 ? 64 : 32), slots);
            consider(Way::ROWS_FEW, sp, (rounds / 2 * 7 + rounds % 2 * 4) * COST_FEW.chunk * chunks / 4 + (rounds + 1) / 2 * start(COST_FEW));
        }
    }
    return QUARTET_OK;
}

static int run_way(const Fp8Product& x, Way way, int splits, cudaStream_t s) {
    const int64_t K = (int64_t)x.g.k_chunks * 128;
    switch (way) {
        case Way::FEW_TOKENS: return gemv_fp8_codes(x.a, x.b, x.g, s);
        case Way::PAIR: return launch_pair<false>(&x, s);
        case Way::ROWS_256: return launch_split<256, 1>(x.a, x.b, K, x.g, splits, s);
        case Way::ROWS_128: return launch_split<128, 1>(x.a, x.b, K, x.g, splits, s);
        case Way::ROWS_128_TWO: return launch_split<128, 2>(x.a, x.b, K, x.g, splits, s);
        default: return x.g.M > 32 ? launch_split<64, 2>(x.a, x.b, K, x.g, splits, s) : launch_split<32, 2>(x.a, x.b, K, x.g, splits, s);
    }
}

static int product(const Fp8Product& x, cudaStream_t s) {
    Way way;
    int64_t cost;
    int splits = 1, rc = pick_way(x.g, &way, &splits, &cost);
    return rc ? rc : run_way(x, way, splits, s);
}

// Two products that do not depend on one another: in one launch of CTA pairs where by the model that takes 11/12 of the two at most, as the second one
// then fills what the first one's last round leaves idle.  us of a whole backward pass, two launches / one: 4096 x 32000, K 640 263 / 249; 8192 x 5120,
// K 1024 112-145 / 95-117; 1000 x 3000, K 2000 31-42 / 23-32; 300 x 2600, K 2600 23-31 / 23-25.  Where it would save 5 % of the chunks (8187 x 11008,
// K 4096) the busier chip runs slower by as much, 578 / 582.
int product_two(const Fp8Product& x, const Fp8Product& y, cudaStream_t s) {
    Way wx, wy;
    int64_t cost_x, cost_y;
    int sx = 1, sy = 1, rc = pick_way(x.g, &wx, &sx, &cost_x);
    if (rc || (rc = pick_way(y.g, &wy, &sy, &cost_y))) return rc;
    auto for_pairs = [](const Fp8GemmParams& g) { return g.M > 64 && g.N >= 64; };
    if (wx != Way::FEW_TOKENS && wy != Way::FEW_TOKENS && for_pairs(x.g) && for_pairs(y.g)) {
        const int (*resident)[4] = nullptr;
        if ((rc = resident_clusters(&resident))) return rc;
        const int64_t n = (*resident)[1], cx = x.g.k_chunks, cy = y.g.k_chunks;
        auto tiles = [](const Fp8GemmParams& g) { return ((g.M + 255) / 256) * ((g.N + 255) / 256); };
        const int64_t tx = tiles(x.g), ty = tiles(y.g), rounds = (tx + ty + n - 1) / n;
        const int64_t chunks = std::max((tx * cx + ty * cy + n - 1) / n, std::max(cx, cy));
        const int64_t joined = COST_PAIR.chunk * chunks + COST_PAIR.start + (rounds - 1) * COST_PAIR.again;
        if (12 * joined <= 11 * (cost_x + cost_y)) {
            const Fp8Product both[2] = {cx >= cy ? x : y, cx >= cy ? y : x};
            return launch_pair<true>(both, s);
        }
    }
    rc = run_way(x, wx, sx, s);
    return rc ? rc : run_way(y, wy, sy, s);
}

static int check_extents(int64_t M, int64_t N, int64_t K) {
    if (M < 1 || N < 1 || K < 128 || K % 128 || M > 8388480 || N > 8388480 || K > (1 << 30))
        return fail(QUARTET_E_SHAPE, "need 1 <= M, N <= 8388480 and K a multiple of 128 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    return QUARTET_OK;
}

}  // namespace quartet

using namespace quartet;

extern "C" __attribute__((visibility("default"))) int quartet_gemm_fp8_form(int64_t M, int64_t N, int64_t K, int32_t* form, int32_t* splits) {
    if (!form || !splits) return fail(QUARTET_E_NULL, "form and splits must be non-NULL");
    int rc = check_extents(M, N, K);
    if (rc) return rc;
    if ((rc = check_device())) return rc;
    Fp8GemmParams p{};
    p.M = M, p.N = N, p.k_chunks = (int)(K / 128);
    Way way;
    int64_t cost;
    int s = 1;
    if ((rc = pick_way(p, &way, &s, &cost))) return rc;
    *form = (int32_t)way, *splits = s;
    return QUARTET_OK;
}

extern "C" __attribute__((visibility("default"))) int quartet_gemm_fp8_tn(const uint8_t* a, const uint8_t* a_sf, int a_fmt, const uint8_t* b,
                                                                          const uint8_t* b_sf, int b_fmt, int64_t M, int64_t N, int64_t K, float alpha,
                                                                          void* d, int d_dtype, int64_t ldd, quartet_stream_t stream) {
    if (!a || !a_sf || !b || !b_sf || !d) return fail(QUARTET_E_NULL, "a, a_sf, b, b_sf and d must be non-NULL");
    if ((a_fmt != QUARTET_E4M3 && a_fmt != QUARTET_E5M2) || (b_fmt != QUARTET_E4M3 && b_fmt != QUARTET_E5M2))
        return fail(QUARTET_E_ARG, "a_fmt and b_fmt must be 0 (e4m3) or 1 (e5m2)");
    if (d_dtype != QUARTET_BF16 && d_dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "d_dtype must be 0 or 1");
    int rc = check_extents(M, N, K);
    if (rc) return rc;
    if (ldd < N || ldd % (d_dtype == QUARTET_F32 ? 4 : 8)) return fail(QUARTET_E_SHAPE, "rows of d must start on 16-byte boundaries and hold N results");
    if (!aligned16(a) || !aligned16(b) || !aligned16(a_sf) || !aligned16(b_sf) || !aligned16(d)) return fail(QUARTET_E_ALIGN, "operands must be 16-byte aligned");
    if ((rc = bind_context_of(a))) return rc;
    if ((rc = check_device())) return rc;
    Fp8GemmParams p{};
    p.a_sf = a_sf, p.b_sf = b_sf;
    p.M = M, p.N = N, p.ldd = ldd;
    p.k_chunks = (int)(K / 128);
    p.a_e5m2 = a_fmt, p.b_e5m2 = b_fmt;
    p.alpha = alpha, p.d = d, p.d_f32 = d_dtype == QUARTET_F32;
    return product(Fp8Product{a, b, p}, static_cast<cudaStream_t>(stream));
}

extern "C" __attribute__((visibility("default"))) int64_t quartet_linear_fp8_workspace_bytes(int64_t M, int64_t K) {
    const int64_t pk = (K + 127) / 128 * 128;
    if (K < 1 || gemv_fits(M, pk)) return 0;
    return M * pk + quartet_sf_bytes(M, pk);
}

extern "C" __attribute__((visibility("default"))) int quartet_linear_fp8(const void* x, int x_dtype, int64_t M, int64_t K, const uint8_t* w, const uint8_t* w_sf,
                                                                         int w_fmt, int64_t N, float alpha, uint8_t* workspace, void* y, int y_dtype, int64_t ldy,
                                                                         quartet_stream_t stream) {
    if (!x || !w || !w_sf || !y) return fail(QUARTET_E_NULL, "x, w, w_sf and y must be non-NULL");
    if (M < 1 || N < 1 || K < 1 || M > 8388480 || N > 8388480 || K > (1 << 30))
        return fail(QUARTET_E_SHAPE, "need 1 <= M, N <= 8388480 and K >= 1 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    // everything is checked before the first of the two steps is launched
    if (x_dtype != QUARTET_BF16 && x_dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "x_dtype must be 0 (bf16) or 1 (f32)");
    if (w_fmt != QUARTET_E4M3 && w_fmt != QUARTET_E5M2) return fail(QUARTET_E_ARG, "w_fmt must be 0 (e4m3) or 1 (e5m2)");
    if (y_dtype != QUARTET_BF16 && y_dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "y_dtype must be 0 or 1");
    const bool f32 = x_dtype == QUARTET_F32;
    if (ldy < N || ldy % (y_dtype == QUARTET_F32 ? 4 : 8)) return fail(QUARTET_E_SHAPE, "rows of y must start on 16-byte boundaries and hold N results");
    if (reinterpret_cast<uintptr_t>(x) & (f32 ? 3u : 1u)) return fail(QUARTET_E_ALIGN, "x must be aligned to its type");
    if (!aligned16(w) || !aligned16(w_sf) || !aligned16(y) || !aligned16(workspace)) return fail(QUARTET_E_ALIGN, "w, w_sf, y and workspace must be 16-byte aligned");
    const int64_t pk = (K + 127) / 128 * 128;
    if (!gemv_fits(M, pk)) {
        if (!workspace) return fail(QUARTET_E_NULL, "workspace must be non-NULL for %lld rows", (long long)M);
        uint8_t* sf = workspace + M * pk;  // pk is a multiple of 128, so the scales are aligned like the codes
        const int rc = quartet_quant_fp8(x, x_dtype, M, K, QUARTET_E4M3, 0, workspace, sf, nullptr, nullptr, stream);
        return rc ? rc : quartet_gemm_fp8_tn(workspace, sf, QUARTET_E4M3, w, w_sf, w_fmt, M, N, pk, alpha, y, y_dtype, ldy, stream);
    }
    int rc = bind_context_of(w);
    if (rc) return rc;
    if ((rc = check_device())) return rc;
    Fp8GemmParams p{};
    p.b_sf = w_sf;
    p.M = M, p.N = N, p.ldd = ldy;
    p.k_chunks = (int)(pk / 128);
    p.b_e5m2 = w_fmt;
    p.alpha = alpha, p.d = y, p.d_f32 = y_dtype == QUARTET_F32;
    return gemv_fp8_values(x, f32, K, w, p, static_cast<cudaStream_t>(stream));
}
