// 8-bit block-scaled product for up to eight rows of A (tokens being generated):  D[M, N] = alpha * A[M, K] . B[N, K]^T
//
// Every byte of the weight B is used for at most eight results, so the kernel is a stream over B: N K (1 + 1/32) bytes at the memory's rate
// is its floor.  A CTA of sixteen warps visits blocks of 16 RW rows of B; RW groups of KW = 16 / RW warps each take 16 rows, the
// warps of a group a share of the contraction each.  A warp owns a ring of tensor copies (16 rows x 128 values and their scales) that
// runs on into its next block while the present one is reduced, so the stream never pauses, and there is nothing to set up per
// block: no tensor memory, no cluster.  All SMs take part evenly, which the memory's rate needs: one SM draws at most about 24 bytes a clock from
// it, however many copies are under way.
// The products are m16n8k16 in fp16, which holds every 8-bit code: 16 rows of B, converted as they come from shared memory, and the
// (up to) eight rows of A, converted once.  Sums over the 128 values of a chunk (over 32, where the scales differ inside it) are scaled in fp32 and
// added to fp32 sums, which the warps of a group join in a fixed order in shared memory.  (The 8-bit form of the instruction converts both
// operands inside: 30 us at N 12288, K 4096, one row, where this takes 14.)
// Bound by the latency of a warp's chain from a chunk's copy over its conversions and products to the sum, which four warps a scheduler cover in
// part: at N 12288, K 4096 and one row 6.8 M warp instructions fill 49 % of the issue slots and the memory is 36 % busy, 4 us of the launch
// among them.  Eight warps instead of sixteen took half as long again; 32 warps or deeper rings gain nothing.
// us, quantizer included, weights from memory, 1 / 4 / 8 rows here | tensor-memory kernel behind its quantizer:
//     N  1920, K   640     3.8   4.0   4.1  |   5.2   5.4   5.6
//     N  4096, K  4096     6.7   7.1   8.4  |   8.4   8.6   8.7
//     N 32000, K   640     7.4   7.8   8.5  |   7.9   7.9   8.1
//     N  4096, K 11008    11.8  14.1  13.6  |  13.2  13.4  13.6
//     N 12288, K  4096    13.5  13.9  15.2  |  13.9  14.2  13.7
//     N 32000, K  4096    26.4  27.3  29.0  |  24.8  24.9  25.1
// So eight rows as the limit whatever the size gains up to a quarter on small weights and loses up to a sixth on the largest.  It stays a rule
// on M and K alone because it also decides whether a call needs a workspace, whose size is asked for without N.
// A comes as codes and scales, or as values that the CTA quantizes into shared memory while its first copies are under way.
#include "common.cuh"
#include "gemm_fp8.cuh"
#include "quant_fp8.cuh"

namespace quartet {

constexpr int GEMV_WARPS = 16, GEMV_THREADS = 32 * GEMV_WARPS, GEMV_STAGES = 3;
constexpr int GEMV_W_BYTES = 16 * 128, GEMV_SF_BYTES = 256, GEMV_STAGE_BYTES = GEMV_W_BYTES + GEMV_SF_BYTES;
constexpr int GEMV_RING = GEMV_WARPS * GEMV_STAGES * GEMV_STAGE_BYTES;
constexpr int GEMV_FIXED = GEMV_RING + 2 * GEMV_WARPS * 128 * 4 + GEMV_WARPS * GEMV_STAGES * 8;

enum { A_CODES = 0, A_BF16 = 1, A_F32 = 2 };

// rows of A in shared memory, in fp16: 32 bytes more than the values, so that four rows' eight-byte reads lie in different banks
static inline int64_t gemv_pitch(int64_t pk) { return 2 * pk + 32; }
bool gemv_fits(int64_t M, int64_t pk) { return M <= 8 && M * (gemv_pitch(pk) + pk / 32) <= 96 * 1024; }

// acc + v 2^(w - 127) 2^(x - 127), NaN for a byte of 255.  The summed exponent is halved into two factors on the same side of one: what
// lies between leaves fp32 only where the product does (below 2^-149 both are lost).
__device__ __forceinline__ float scaled_add(float v, uint32_t w, uint32_t x, float acc) {
    const uint32_t e = w + x, h = e >> 1, r = e - h;  // 0 .. 254 each: 2^(h - 127), 2^(r - 127), the least of them subnormal
    const float a = __uint_as_float(max(w, x) == 255u ? 0x7FC00000u : max(h << 23, 0x00400000u)), b = __uint_as_float(max(r << 23, 0x00400000u));
    return fmaf(v * a, b, acc);
}

template <bool E5M2>
__device__ __forceinline__ uint32_t f16x2_of(uint32_t two) {  // two codes in the low bytes
    uint32_t h;
    if constexpr (E5M2)
        asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    else
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

struct GemvParams {
    Fp8GemmParams g;
    const uint8_t* a;       // codes (A_CODES) or values
    int64_t a_cols;         // values in a row (A_BF16, A_F32)
    int a_vec;
    int kw;                 // warps that share a row group's contraction
    int blocks;             // blocks of 16 * GEMV_WARPS / kw rows
};

template <int AMODE, bool B_E5M2, bool A_E5M2>
__global__ void __launch_bounds__(GEMV_THREADS) gemv_fp8_kernel(const __grid_constant__ CUtensorMap tm_w, const GemvParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(&g_status, WAIT_GEMM_ALIGN | 0x100);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* s_w = smem + warp * (GEMV_STAGES * GEMV_W_BYTES);
    uint8_t* s_sf = smem + GEMV_WARPS * GEMV_STAGES * GEMV_W_BYTES + warp * (GEMV_STAGES * GEMV_SF_BYTES);
    float* s_part = reinterpret_cast<float*>(smem + GEMV_RING);                 // [2][warp][16 rows x 8 tokens]
    uint64_t* full = reinterpret_cast<uint64_t*>(s_part + 2 * GEMV_WARPS * 128) + warp * GEMV_STAGES;
    uint8_t* s_a = smem + GEMV_FIXED;
    const int chunks = p.g.k_chunks, M = (int)p.g.M;
    const int pitch = chunks * 256 + 32;
    uint32_t* s_asf = reinterpret_cast<uint32_t*>(s_a + M * pitch);             // [token][chunk], four scale bytes
    const int kw = p.kw, rw = GEMV_WARPS / kw, kpart = warp % kw, group = warp / kw;
    const int c0 = chunks * kpart / kw, mine = chunks * (kpart + 1) / kw - c0;

    if (lane == 0) {
        for (int i = 0; i < GEMV_STAGES; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
        prefetch_tmap(&tm_w);
    }
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();

    // The ring's position in this warp's sequence of (block, chunk): coordinates and the scales' address move on by addition.  Blocks whose
    // group lies past the last row are the last ones, and are left out.
    const int blocks_mine = (int)((p.g.N - (int64_t)group * 16 + rw * 16 - 1) / (rw * 16));     // blocks whose rows of this group exist
    int blk = blockIdx.x, ck = 0, row0 = 0;
    const uint8_t* sf_src = nullptr;
    auto at_block = [&]() {
        row0 = (blk * rw + group) * 16;
        sf_src = p.g.b_sf + ((int64_t)(row0 >> 7) * chunks + c0) * 512 + (row0 & 31) * 16;
    };
    at_block();
    int ahead = 0;  // copies issued and not yet consumed
    auto fill = [&](int s) {
        if (blk >= blocks_mine || mine == 0) return;
        if (lane == 0) {
            mbar_arrive_expect_tx(&full[s], GEMV_STAGE_BYTES);
            tma_load_2d(s_w + s * GEMV_W_BYTES, &tm_w, (c0 + ck) * 128, row0, &full[s]);
            bulk_load(s_sf + s * GEMV_SF_BYTES, sf_src, GEMV_SF_BYTES, &full[s]);
        }
        ++ahead;
        sf_src += 512;
        if (++ck == mine) {
            ck = 0, blk += gridDim.x;
            at_block();
        }
    };
    for (int s = 0; s < GEMV_STAGES; ++s) fill(s);

    // A into shared memory
    if constexpr (AMODE == A_CODES) {
        for (int i = tid; i < M * chunks * 8; i += GEMV_THREADS) {
            const int r = i / (chunks * 8), c = i - r * (chunks * 8);
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.a + (int64_t)r * chunks * 128) + c);
            uint4* dst = reinterpret_cast<uint4*>(s_a + r * pitch + c * 32);
            dst[0] = make_uint4(f16x2_of<A_E5M2>(v.x), f16x2_of<A_E5M2>(v.x >> 16), f16x2_of<A_E5M2>(v.y), f16x2_of<A_E5M2>(v.y >> 16));
            dst[1] = make_uint4(f16x2_of<A_E5M2>(v.z), f16x2_of<A_E5M2>(v.z >> 16), f16x2_of<A_E5M2>(v.w), f16x2_of<A_E5M2>(v.w >> 16));
        }
        for (int i = tid; i < M * chunks; i += GEMV_THREADS) {
            const int r = i / chunks, c = i - r * chunks;
            s_asf[i] = __ldg(reinterpret_cast<const uint32_t*>(p.g.a_sf + (int64_t)c * 512 + r * 16));
        }
    } else {
        using R = RowPart<AMODE == A_F32>;
        const int j = tid & 7, n = M * chunks;
        for (int i0 = 0; i0 < n; i0 += 2 * GEMV_THREADS / 8) {   // two row parts a thread in flight
            R part[2];
            int at[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                at[u] = i0 + u * (GEMV_THREADS / 8) + (tid >> 3);
                const int r = at[u] / chunks;
                part[u].load(p.a, at[u] < n ? M : 0, p.a_cols, p.a_vec, r, (int64_t)(at[u] - r * chunks) * 128, j);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t sb = fp8_scale_byte(mag_over_8<AMODE == A_F32>(part[u].mag()), 8);
                if (at[u] >= n) continue;
                const int r = at[u] / chunks, c = at[u] - r * chunks;
#pragma unroll
                for (int q = 0; q < R::N; ++q) {
                    uint32_t w[R::PER / 4];
                    part[u].template codes<false>(w, q, fp8_inv_scale(sb));
                    uint2* dst = reinterpret_cast<uint2*>(s_a + r * pitch + c * 256 + (j + 8 * q) * R::PER * 2);
#pragma unroll
                    for (int k = 0; k < R::PER / 4; ++k) dst[k] = make_uint2(f16x2_of<false>(w[k]), f16x2_of<false>(w[k] >> 16));
                }
                if (j == 0) s_asf[at[u]] = sb * 0x01010101u;
            }
        }
    }
    __syncthreads();

    const int g = lane >> 2, q = lane & 3;     // accumulator: rows g, g + 8 of B, tokens 2 q, 2 q + 1
    // (rows of A past the last one: the first row's values, whose results nobody reads)
    const uint8_t* a_row = s_a + (g < M ? g : 0) * pitch + c0 * 256 + q * 8;
    const uint32_t* asf0 = s_asf + (2 * q < M ? 2 * q : 0) * chunks + c0;
    const uint32_t* asf1 = s_asf + (2 * q + 1 < M ? 2 * q + 1 : 0) * chunks + c0;
    // ldmatrix: lanes 0-7 rows 0-7, 8-15 rows 8-15 of the first 16 bytes, 16-31 the same of the second; 128-byte swizzle
    uint32_t m_off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) m_off[k] = (lane & 15) * 128 + (((2 * k + (lane >> 4)) ^ (lane & 7)) << 4);
    const uint32_t w_base = smem_u32(s_w);
    uint32_t s = 0, ph = 0, buf = 0;
    bool dead = false;                         // a wait gave up: this warp only keeps the barriers
    for (int b = blockIdx.x; b < p.blocks; b += gridDim.x, buf ^= 1) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        if (!dead && b < blocks_mine) {
            const int seg = ((b * rw + group) >> 1) & 3;  // 32-row segment of the rows in their block of 128
            for (int c = 0; c < mine; ++c) {
                if (!mbar_wait(&full[s], ph, WAIT_GEMM_FULL)) {
                    dead = true;
                    break;
                }
                __syncwarp();  // (the wait's lanes may leave it apart; ldmatrix and the products are the warp's)
                --ahead;
                const uint8_t* sfw = s_sf + s * GEMV_SF_BYTES + seg * 4 + g * 16;
                const uint32_t w0 = *reinterpret_cast<const uint32_t*>(sfw), w1 = *reinterpret_cast<const uint32_t*>(sfw + 128);
                const uint32_t x0 = asf0[c], x1 = asf1[c];
                const uint32_t base = w_base + s * GEMV_W_BYTES;
                const uint8_t* av = a_row + c * 256;
                float cc[4][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t f[4];
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
                                 : "r"(base + m_off[k])
                                 : "memory");
                    // a thread's four neighbouring values of a row stand for the instruction's columns 2 q, 2 q + 1, 2 q + 8, 2 q + 9, and so do A's
                    const uint2 xa = *reinterpret_cast<const uint2*>(av + k * 64), xb = *reinterpret_cast<const uint2*>(av + k * 64 + 32);
                    mma_f16_first(cc[k], f16x2_of<B_E5M2>(f[0]), f16x2_of<B_E5M2>(f[1]), f16x2_of<B_E5M2>(f[0] >> 16), f16x2_of<B_E5M2>(f[1] >> 16), xa.x, xa.y);
                    mma_f16(cc[k], f16x2_of<B_E5M2>(f[2]), f16x2_of<B_E5M2>(f[3]), f16x2_of<B_E5M2>(f[2] >> 16), f16x2_of<B_E5M2>(f[3] >> 16), xb.x, xb.y);
                }
                // Two factors 2^(b - 127) make one, 2^(w + x - 254), taken as a whole: either by itself may lead out of fp32 where the product is well
                // inside.  One scale for the whole chunk, as this library's quantizers write them, and bytes of 64 .. 190, whose sums leave a normal factor:
                const bool block = w0 == __byte_perm(w0, 0, 0) && w1 == __byte_perm(w1, 0, 0) && x0 == __byte_perm(x0, 0, 0) && x1 == __byte_perm(x1, 0, 0);
                constexpr uint32_t LOW = 64u << 24, SPAN = 127u << 24, ONE = 127u << 23;
                const bool plain = __all_sync(0xFFFFFFFFu, block && max(max(w0 - LOW, w1 - LOW), max(x0 - LOW, x1 - LOW)) < SPAN);
                __syncwarp();
                fill((int)s);  // the stage has been read, its scales by the vote above: its next copy may start
                if (++s == GEMV_STAGES) s = 0, ph ^= 1;
                if (plain) {
                    const uint32_t f0 = (w0 >> 1) & 0x7F800000u, f1 = (w1 >> 1) & 0x7F800000u, g0 = (x0 >> 1) & 0x7F800000u, g1 = (x1 >> 1) & 0x7F800000u;
                    const float s00 = __uint_as_float(f0 + g0 - ONE), s01 = __uint_as_float(f0 + g1 - ONE);
                    const float s10 = __uint_as_float(f1 + g0 - ONE), s11 = __uint_as_float(f1 + g1 - ONE);
                    acc[0] = fmaf((cc[0][0] + cc[1][0]) + (cc[2][0] + cc[3][0]), s00, acc[0]);
                    acc[1] = fmaf((cc[0][1] + cc[1][1]) + (cc[2][1] + cc[3][1]), s01, acc[1]);
                    acc[2] = fmaf((cc[0][2] + cc[1][2]) + (cc[2][2] + cc[3][2]), s10, acc[2]);
                    acc[3] = fmaf((cc[0][3] + cc[1][3]) + (cc[2][3] + cc[3][3]), s11, acc[3]);
                } else {
                    // Rows of zeros (byte 0) come here too: a chunk under one scale then takes one step, not four.
                    const bool whole = __all_sync(0xFFFFFFFFu, block);
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) cc[0][i] = (cc[0][i] + cc[1][i]) + (cc[2][i] + cc[3][i]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (k > 0 && whole) break;
                        const uint32_t wb0 = (w0 >> (8 * k)) & 255u, wb1 = (w1 >> (8 * k)) & 255u, xb0 = (x0 >> (8 * k)) & 255u, xb1 = (x1 >> (8 * k)) & 255u;
                        acc[0] = scaled_add(cc[k][0], wb0, xb0, acc[0]);
                        acc[1] = scaled_add(cc[k][1], wb0, xb1, acc[1]);
                        acc[2] = scaled_add(cc[k][2], wb1, xb0, acc[2]);
                        acc[3] = scaled_add(cc[k][3], wb1, xb1, acc[3]);
                    }
                }
            }
        }
        float* part = s_part + (buf * GEMV_WARPS + warp) * 128;   // [token][row]
        part[(2 * q) * 16 + g] = acc[0], part[(2 * q + 1) * 16 + g] = acc[1];
        part[(2 * q) * 16 + g + 8] = acc[2], part[(2 * q + 1) * 16 + g + 8] = acc[3];
        __syncthreads();  // one barrier a block: the partial sums alternate between two buffers
        for (int i = tid; i < rw * 16 * M; i += GEMV_THREADS) {
            const int row = i % (rw * 16), tok = i / (rw * 16), gr = row >> 4;
            const int64_t n = (int64_t)b * rw * 16 + row;
            float v = 0.f;
            for (int k = 0; k < kw; ++k) v += s_part[(buf * GEMV_WARPS + gr * kw + k) * 128 + tok * 16 + (row & 15)];
            v *= p.g.alpha;
            if (n < p.g.N) {
                if (p.g.d_f32)
                    static_cast<float*>(p.g.d)[tok * p.g.ldd + n] = v;
                else
                    static_cast<__nv_bfloat16*>(p.g.d)[tok * p.g.ldd + n] = __float2bfloat16_rn(v);
            }
        }
    }
    // after a wait that gave up, copies may still be in flight: they land before shared memory is released
    for (int i = 0; i < GEMV_STAGES && ahead > 0; ++i, --ahead) {
        mbar_wait(&full[s], ph, WAIT_GEMM_FULL);
        if (++s == GEMV_STAGES) s = 0, ph ^= 1;
    }
}

// KW, the warps that share a row's contraction: the number for which the SM with the most blocks has the least to do, a block's reduction
// counted as one more chunk.
static int gemv_pick_kw(int64_t N, int chunks, int sms) {
    int best = 1;
    int64_t cost = INT64_MAX;
    for (int kw = 1; kw <= GEMV_WARPS && kw <= chunks; kw *= 2) {
        const int64_t rows = 16 * (GEMV_WARPS / kw), blocks = (N + rows - 1) / rows;
        const int64_t c = ((blocks + sms - 1) / sms) * ((chunks + kw - 1) / kw + 1);
        if (c <= cost) cost = c, best = kw;
    }
    return best;
}

template <int AMODE, bool B_E5M2, bool A_E5M2>
static int launch_gemv(const uint8_t* b, GemvParams p, cudaStream_t stream) {
    const int64_t K = (int64_t)p.g.k_chunks * 128;
    CUtensorMap tm_w;
    int rc = make_tmap_2d(&tm_w, b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, p.g.N, K, 128, 16, 3);
    if (rc) return rc;
    int sms = 0;
    if ((rc = device_sm_count(&sms))) return rc;
    p.kw = gemv_pick_kw(p.g.N, p.g.k_chunks, sms);
    const int rows = 16 * (GEMV_WARPS / p.kw);
    p.blocks = (int)((p.g.N + rows - 1) / rows);
    const int smem = GEMV_FIXED + (int)(p.g.M * (gemv_pitch(K) + K / 32));
    auto kern = gemv_fp8_kernel<AMODE, B_E5M2, A_E5M2>;
    static thread_local int smem_set = -1;
    if ((rc = set_max_smem_once(kern, GEMV_FIXED + 96 * 1024, smem_set))) return rc;
    const int grid = p.blocks < sms ? p.blocks : sms;
    return check_cuda(launch_pdl(kern, dim3((unsigned)grid), dim3(GEMV_THREADS), smem, stream, tm_w, p), "gemv_fp8 launch");
}

int gemv_fp8_codes(const uint8_t* a, const uint8_t* b, const Fp8GemmParams& g, cudaStream_t s) {
    GemvParams p{};
    p.g = g, p.a = a;
    if (g.b_e5m2) return g.a_e5m2 ? launch_gemv<A_CODES, true, true>(b, p, s) : launch_gemv<A_CODES, true, false>(b, p, s);
    return g.a_e5m2 ? launch_gemv<A_CODES, false, true>(b, p, s) : launch_gemv<A_CODES, false, false>(b, p, s);
}
int gemv_fp8_values(const void* x, bool f32, int64_t cols, const uint8_t* b, const Fp8GemmParams& g, cudaStream_t s) {
    GemvParams p{};
    p.g = g, p.a = static_cast<const uint8_t*>(x), p.a_cols = cols;
    p.a_vec = aligned16(x) && cols % (f32 ? 4 : 8) == 0;
    if (f32) return g.b_e5m2 ? launch_gemv<A_F32, true, false>(b, p, s) : launch_gemv<A_F32, false, false>(b, p, s);
    return g.b_e5m2 ? launch_gemv<A_BF16, true, false>(b, p, s) : launch_gemv<A_BF16, false, false>(b, p, s);
}

QUARTET_DEFINE_STATUS_READER(status_gemv_fp8)

}  // namespace quartet
