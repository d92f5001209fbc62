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
// and up to 128 rows of A its N -- so that a single token still feeds every row of the tensor core with one weight row, and
// the contraction is split over the CTAs of a cluster, which add their fp32 partial results in rank order through
// distributed shared memory: no workspace, no atomics, the same bits every time.
#include "common.cuh"
#include "tcgen05.cuh"

#include <cuda_bf16.h>

namespace quartet {

struct Fp8GemmParams {
    const uint8_t* a_sf;
    const uint8_t* b_sf;
    int64_t M, N;
    int64_t ldd;
    int k_chunks;        // K / 128
    int a_e5m2, b_e5m2;
    float alpha;
    void* d;
    int d_f32;
};

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
// One 512-byte scale block from shared memory to four tensor-memory columns, replicated into the four lane quadrants.  Ordered
// with the MMAs the same thread issues.
__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(128 >> 4) << 32;    // eight 16-byte rows to the next
    d |= (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// ---------------------------------------------------------------------------
// swapped roles, contraction split over a cluster
// ---------------------------------------------------------------------------
template <int BT>  // rows of A (tokens) a CTA takes
struct SplitCfg {
    static constexpr int W_BYTES = 128 * 128;
    static constexpr int X_BYTES = BT * 128;
    static constexpr int STAGES = BT == 128 ? 6 : 8;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + 1024;
    static constexpr int SF_COL0 = BT;
    static constexpr int TMEM_COLS = BT == 128 ? 256 : 128;   // BT accumulator columns and eight scale columns a stage
    static constexpr int SMEM = STAGES * STAGE_BYTES + 256;
    static_assert(SF_COL0 + STAGES * 8 <= TMEM_COLS, "tensor memory capacity");
    static_assert(STAGES * (W_BYTES + X_BYTES) >= BT * 128 * 4, "the partial result reuses the operand stages");
    static_assert(SMEM <= 232448, "shared memory capacity");
};

constexpr int SPLIT_THREADS = 128;

template <int BT>
__global__ void __launch_bounds__(SPLIT_THREADS, 1) gemm_fp8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                         const Fp8GemmParams p, const int splits) {
    using C = SplitCfg<BT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        // uniform over the grid: no CTA of the cluster gets further
        if (threadIdx.x == 0) atomicOr(&g_status, WAIT_GEMM_ALIGN | 0x100);
        return;
    }
    uint8_t* s_w = smem;
    uint8_t* s_x = s_w + C::STAGES * C::W_BYTES;
    uint8_t* s_sf = s_x + C::STAGES * C::X_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_sf + C::STAGES * 1024);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(acc_full + 1);
    volatile int* dead = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % splits;          // the cluster spans the split axis
    const int n_blk = (int)blockIdx.x / splits, t_blk = blockIdx.y;
    const int c0 = (int)((int64_t)p.k_chunks * rank / splits), c1 = (int)((int64_t)p.k_chunks * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
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

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (int c = c0; c < c1; ++c) {
                if (!gemm_wait(&empty[s], ph ^ 1, WAIT_GEMM_EMPTY, dead)) break;
                mbar_arrive_expect_tx(&full[s], C::STAGE_BYTES);
                tma_load_2d(s_w + s * C::W_BYTES, &tm_w, c * 128, n_blk * 128, &full[s]);
                tma_load_2d(s_x + s * C::X_BYTES, &tm_x, c * 128, t_blk * BT, &full[s]);
                bulk_load(s_sf + s * 1024, p.b_sf + ((int64_t)n_blk * p.k_chunks + c) * 512, 512, &full[s]);
                bulk_load(s_sf + s * 1024 + 512, p.a_sf + ((int64_t)(t_blk * BT / 128) * p.k_chunks + c) * 512, 512, &full[s]);
                if (++s == C::STAGES) s = 0, ph ^= 1;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (int c = c0; c < c1; ++c) {
                if (!gemm_wait(&full[s], ph, WAIT_GEMM_FULL, dead)) break;
                tc_fence_after();
                const uint32_t sf = tmem + C::SF_COL0 + s * 8;
                tc_cp_scales(sf, smem_u32(s_sf + s * 1024));
                tc_cp_scales(sf + 4, smem_u32(s_sf + s * 1024 + 512));
                const uint64_t wd = make_desc_sw128(smem_u32(s_w + s * C::W_BYTES)), xd = make_desc_sw128(smem_u32(s_x + s * C::X_BYTES));
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)  // 32 values a step, one scale byte each
                    tc_mma_mxf8(tmem, wd + 2 * j, xd + 2 * j, make_idesc_fp8(128, BT, p.b_e5m2, p.a_e5m2, j), sf | (j << 30), (sf + 4) | (j << 30),
                                (c != c0) | j);
                tc_commit(&empty[s]);
                if (++s == C::STAGES) s = 0, ph ^= 1;
            }
            tc_commit(acc_full);
        }
    }
    __syncwarp();
    // ---- partial results [token][weight row] in fp32 over the operand stages: all copies have landed and been read ----
    const bool ok = gemm_wait(acc_full, 0, WAIT_GEMM_ACC_FULL, dead);
    tc_fence_after();
    float* red = reinterpret_cast<float*>(smem);
    const int row = warp * 32 + lane;
    __syncthreads();
    if (ok) {
#pragma unroll 1
        for (int cb = 0; cb < BT; cb += 32) {
            uint32_t r[32];
            tc_ld32(tmem + ((uint32_t)(warp * 32) << 16) + cb, r);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) red[(cb + i) * 128 + row] = __uint_as_float(r[i]);
        }
    }
    tc_fence_before();
    if (splits > 1)
        cluster_sync_all();
    else
        __syncthreads();
    if (ok) {
        // this CTA adds the partial results of tokens rank, rank + splits, ...; 32 threads a token, four results each
        const int64_t t0 = (int64_t)t_blk * BT;
        const int tokens = (int)(p.M - t0 < BT ? p.M - t0 : BT);
        const int64_t n0 = (int64_t)n_blk * 128 + lane * 4;
        const uint32_t red_addr = smem_u32(red) + lane * 16;
        for (int t = rank + warp * splits; t < tokens; t += 4 * splits) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < splits; ++s) {
                const uint32_t at = red_addr + t * 512;
                float4 q;
                const uint32_t peer = splits > 1 ? mapa_u32(at, s) : at;
                if (splits > 1)
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(q.x), "=f"(q.y), "=f"(q.z), "=f"(q.w) : "r"(peer) : "memory");
                else
                    q = *reinterpret_cast<const float4*>(red + t * 128 + lane * 4);
                v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] *= p.alpha;
            const int64_t at = (t0 + t) * p.ldd + n0;
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
    if (splits > 1) cluster_sync_all();  // no CTA leaves while a peer may still read its partial results
    __syncthreads();
    if (*dead)
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies still in flight land before shared memory is released
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

template <int BT>
static int launch_split(const uint8_t* a, const uint8_t* b, int64_t K, const Fp8GemmParams& p, int splits, cudaStream_t stream) {
    using C = SplitCfg<BT>;
    CUtensorMap tm_w, tm_x;
    int rc = make_tmap_2d(&tm_w, b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.N, K, 128, 128, 3);
    if (rc) return rc;
    if ((rc = make_tmap_2d(&tm_x, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.M, K, 128, BT, 3))) return rc;
    auto kern = gemm_fp8_split_kernel<BT>;
    static thread_local int smem_set = -1;
    if ((rc = set_max_smem_once(kern, C::SMEM, smem_set))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.N + 127) / 128 * splits), (unsigned)((p.M + BT - 1) / BT));
    cfg.blockDim = dim3(SPLIT_THREADS), cfg.dynamicSmemBytes = C::SMEM, cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)splits, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    return check_cuda(cudaLaunchKernelEx(&cfg, kern, tm_w, tm_x, p, splits), "gemm_fp8 launch");
}

QUARTET_DEFINE_STATUS_READER(status_gemm_fp8)

}  // namespace quartet

using namespace quartet;

extern "C" __attribute__((visibility("default"))) int quartet_gemm_fp8_tn(const uint8_t* a, const uint8_t* a_sf, int a_fmt, const uint8_t* b,
                                                                          const uint8_t* b_sf, int b_fmt, int64_t M, int64_t N, int64_t K, float alpha,
                                                                          void* d, int d_dtype, int64_t ldd, quartet_stream_t stream) {
    if (!a || !a_sf || !b || !b_sf || !d) return fail(QUARTET_E_NULL, "a, a_sf, b, b_sf and d must be non-NULL");
    if ((a_fmt != QUARTET_E4M3 && a_fmt != QUARTET_E5M2) || (b_fmt != QUARTET_E4M3 && b_fmt != QUARTET_E5M2))
        return fail(QUARTET_E_ARG, "a_fmt and b_fmt must be 0 (e4m3) or 1 (e5m2)");
    if (d_dtype != QUARTET_BF16 && d_dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "d_dtype must be 0 or 1");
    if (M < 1 || N < 1 || K < 128 || K % 128 || M > 8388480 || N > 8388480 || K > (1 << 30))
        return fail(QUARTET_E_SHAPE, "need 1 <= M, N <= 8388480 and K a multiple of 128 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    if (ldd < N || ldd % (d_dtype == QUARTET_F32 ? 4 : 8)) return fail(QUARTET_E_SHAPE, "rows of d must start on 16-byte boundaries and hold N results");
    if (!aligned16(a) || !aligned16(b) || !aligned16(a_sf) || !aligned16(b_sf) || !aligned16(d)) return fail(QUARTET_E_ALIGN, "operands must be 16-byte aligned");
    int rc = bind_context_of(a);
    if (rc) return rc;
    if ((rc = check_device())) return rc;
    Fp8GemmParams p{};
    p.a_sf = a_sf, p.b_sf = b_sf;
    p.M = M, p.N = N, p.ldd = ldd;
    p.k_chunks = (int)(K / 128);
    p.a_e5m2 = a_fmt, p.b_e5m2 = b_fmt;
    p.alpha = alpha, p.d = d, p.d_f32 = d_dtype == QUARTET_F32;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch_split<128>(a, b, K, p, 1, s);
}
