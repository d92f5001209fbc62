// 8-bit quantizers of the block-scaled linear layer.
//
//   scale of a block   2^e, e the least integer with amax <= MAX * 2^e   (MAX = 448 for e4m3, 57344 for e5m2; both are 1.75 * 2^top)
//   code               x * 2^-e rounded to the format, nearest, ties to the even one
//
// A block is 1 x 128 values along the contraction (activations, gradients) or 128 x 128 (weights, whose transpose then
// has the same codes).  The scale byte is E8M0, repeated four times, because the tensor core takes one byte per 32 values:
// the layout (and the 512-byte blocks of 128 rows) is the one the 4-bit kernels of this library use.  Codes are padded
// with zeros to a multiple of 128 columns, so that the product's contraction never ends inside a block.
// A power of two as scale makes x * 2^-e exact, so the only rounding is the code's own.  A block that holds an infinity or
// a NaN gets scale byte 255 and NaN codes: it is NaN as a whole, which a product carries into every result it touches.
//
// One CTA takes 128 rows x 128 columns; eight threads share a row (16-byte loads, 128 bytes a row and load).  Bytes
// per value: the input's 2 or 4, and 1 + 1/32 for each orientation written.
#include "common.cuh"
#include "quant_fp8.cuh"

namespace quartet {

constexpr int F8_TILE = 128, F8_THREADS = 256;

struct Fp8QuantParams {
    const uint8_t* x;
    int64_t rows, cols;
    int64_t pitch, pitch_t;          // of the codes: cols / rows padded to 128
    uint8_t *codes, *sf, *codes_t, *sf_t;
    int top;                         // exponent of MAX: 8 (e4m3) or 15 (e5m2)
    int vec;                         // rows of x start on 16-byte boundaries
};

template <bool F32, bool SQUARE, bool ROWS, bool TRANS>
constexpr int fp8_quant_smem() { return TRANS ? F8_TILE * F8_TILE * (F32 ? 4 : 2) + F8_TILE * F8_TILE + 8 * F8_TILE * 4 : 0; }

template <bool F32, bool SQUARE, bool ROWS, bool TRANS>
__global__ void __launch_bounds__(F8_THREADS) quant_fp8_kernel(const Fp8QuantParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t s_red[8];
    constexpr int EB = F32 ? 4 : 2;
    const int tid = threadIdx.x, j = tid & 7, r0 = tid >> 3;
    const int64_t col0 = (int64_t)blockIdx.x * F8_TILE, row0 = (int64_t)blockIdx.y * F8_TILE;
    const bool e5m2 = p.top == 15;
    pdl_launch_dependents();
    pdl_wait();

    RowPart<F32> part[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) part[s].load(p.x, p.rows, p.cols, p.vec, row0 + r0 + 32 * s, col0, j);

    uint32_t tile_byte = 0;
    if constexpr (SQUARE) {
        uint32_t m = 0u;
#pragma unroll
        for (int s = 0; s < 4; ++s) m = max(m, part[s].amax());
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if ((tid & 31) == 0) s_red[tid >> 5] = m;
        __syncthreads();
        m = s_red[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = max(m, s_red[w]);
        tile_byte = fp8_scale_byte(m, p.top);
    }
    if constexpr (ROWS) {
        uint8_t* sf = p.sf + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 512;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int r = r0 + 32 * s;
            const uint32_t sb = SQUARE ? tile_byte : fp8_scale_byte(max_over_8(part[s].amax()), p.top);
            if (row0 + r < p.rows) {
                uint8_t* dst = p.codes + (row0 + r) * p.pitch + col0;
#pragma unroll
                for (int i = 0; i < RowPart<F32>::N; ++i) part[s].store_codes(dst + (j + 8 * i) * RowPart<F32>::PER, i, sb, e5m2);
            }
            if (j == 0) *reinterpret_cast<uint32_t*>(sf + (r & 31) * 16 + (r >> 5) * 4) = row0 + r < p.rows ? sb * 0x01010101u : 0u;
        }
    }
    if constexpr (TRANS) {
        // The raw tile through shared memory; warp w then owns rows 16 w .. 16 w + 15 and a lane the column pairs lane
        // and lane + 32 (bf16) or the columns lane + 32 i (fp32): every read is one conflict-free row segment.
        uint8_t* s_x = smem;
        uint8_t* s_t = smem + F8_TILE * F8_TILE * EB;
        uint32_t* s_max = reinterpret_cast<uint32_t*>(s_t + F8_TILE * F8_TILE);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < RowPart<F32>::N; ++i)
                *reinterpret_cast<uint4*>(s_x + (r0 + 32 * s) * (F8_TILE * EB) + (j + 8 * i) * 16) = part[s].q[i];
        __syncthreads();
        const int w = tid >> 5, lane = tid & 31;
        constexpr int SETS = F32 ? 4 : 2;
#pragma unroll 1
        for (int set = 0; set < SETS && !SQUARE; ++set) {
            uint32_t m0 = 0u, m1 = 0u;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(s_x + (16 * w + i) * (F8_TILE * EB) + (lane + 32 * set) * 4);
                if (F32) {
                    m0 = max(m0, v & 0x7FFFFFFFu);
                } else {
                    m0 = max(m0, (v << 16) & 0x7FFFFFFFu);
                    m1 = max(m1, v & 0x7FFF0000u);
                }
            }
            if (F32) {
                s_max[w * F8_TILE + lane + 32 * set] = m0;
            } else {
                s_max[w * F8_TILE + 2 * (lane + 32 * set)] = m0;
                s_max[w * F8_TILE + 2 * (lane + 32 * set) + 1] = m1;
            }
        }
        __syncthreads();
        constexpr int PER = F32 ? 1 : 2;
#pragma unroll 1
        for (int set = 0; set < SETS; ++set) {
            uint32_t raw[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[i] = *reinterpret_cast<const uint32_t*>(s_x + (16 * w + i) * (F8_TILE * EB) + (lane + 32 * set) * 4);
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                const int col = PER * (lane + 32 * set) + c;
                uint32_t sb = tile_byte;
                if (!SQUARE) {
                    uint32_t m = 0u;
#pragma unroll
                    for (int k = 0; k < 8; ++k) m = max(m, s_max[k * F8_TILE + col]);
                    sb = fp8_scale_byte(m, p.top);
                }
                const float inv = fp8_inv_scale(sb == 255u ? 127u : sb);
                uint32_t out[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t x = raw[4 * k + t];
                        v[t] = __uint_as_float(F32 ? x : (c ? x & 0xFFFF0000u : x << 16)) * inv;
                    }
                    out[k] = sb == 255u ? 0x7F7F7F7Fu : cvt_fp8x4(v[0], v[1], v[2], v[3], e5m2);
                }
                *reinterpret_cast<uint4*>(s_t + col * F8_TILE + ((w ^ (col & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
                if (w == 0) {
                    uint8_t* sf = p.sf_t + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * 512;
                    *reinterpret_cast<uint32_t*>(sf + (col & 31) * 16 + (col >> 5) * 4) = col0 + col < p.cols ? sb * 0x01010101u : 0u;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int col = r0 + 32 * s;
            if (col0 + col < p.cols)
                *reinterpret_cast<uint4*>(p.codes_t + (col0 + col) * p.pitch_t + row0 + j * 16) =
                    *reinterpret_cast<const uint4*>(s_t + col * F8_TILE + ((j ^ (col & 7)) << 4));
        }
    }
}

// codes + scales -> values, out = code * 2^(sf - 127) * scale: four values a thread
template <bool F32OUT>
__global__ void __launch_bounds__(256) dequant_fp8_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ sf, int64_t rows,
                                                          int64_t cols, int64_t pitch, int e5m2, float scale, void* __restrict__ out) {
    const int64_t per_row = (cols + 3) >> 2, total = rows * per_row, stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
        const int64_t row = i / per_row, c = (i - row * per_row) * 4;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(codes + row * pitch + c));
        const int64_t r = row & 127;
        const uint32_t b = __ldg(sf + ((row >> 7) * (pitch >> 7) + (c >> 7)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + ((c >> 5) & 3));
        const float s = (b == 255u ? __uint_as_float(0x7FC00000u) : b == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(b << 23)) * scale;
        for (int k = 0; k < 4 && c + k < cols; ++k) {
            uint32_t h;
            const uint16_t two = (uint16_t)((w >> (8 * k)) & 0xFFu);
            if (e5m2)
                asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(two));
            else
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
            const float v = __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu))) * s;
            if (F32OUT)
                static_cast<float*>(out)[row * cols + c + k] = v;
            else
                static_cast<__nv_bfloat16*>(out)[row * cols + c + k] = __float2bfloat16_rn(v);
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <bool F32, bool SQUARE, bool ROWS, bool TRANS>
static int launch_quant_fp8(const Fp8QuantParams& p, cudaStream_t s) {
    auto kern = quant_fp8_kernel<F32, SQUARE, ROWS, TRANS>;
    constexpr int smem = fp8_quant_smem<F32, SQUARE, ROWS, TRANS>();
    static thread_local int smem_set = -1;
    int rc = set_max_smem_once(kern, smem, smem_set);
    if (rc) return rc;
    const dim3 grid((unsigned)((p.cols + 127) / 128), (unsigned)((p.rows + 127) / 128));
    return check_cuda(launch_pdl(kern, grid, dim3(F8_THREADS), smem, s, p), "quant_fp8 launch");
}
template <bool F32, bool SQUARE>
static int pick_quant_fp8(const Fp8QuantParams& p, cudaStream_t s) {
    if (p.codes && p.codes_t) return launch_quant_fp8<F32, SQUARE, true, true>(p, s);
    return p.codes ? launch_quant_fp8<F32, SQUARE, true, false>(p, s) : launch_quant_fp8<F32, SQUARE, false, true>(p, s);
}

}  // namespace quartet

using namespace quartet;

extern "C" __attribute__((visibility("default"))) int quartet_quant_fp8(const void* x, int x_dtype, int64_t rows, int64_t cols, int fmt, int square,
                                                                        uint8_t* codes, uint8_t* sf, uint8_t* codes_t, uint8_t* sf_t,
                                                                        quartet_stream_t stream) {
    if (!x) return fail(QUARTET_E_NULL, "x must be non-NULL");
    if ((!codes && !codes_t) || (codes && !sf) || (codes_t && !sf_t))
        return fail(QUARTET_E_NULL, "need codes with sf, codes_t with sf_t, or both pairs");
    if (x_dtype != QUARTET_BF16 && x_dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "x_dtype must be 0 (bf16) or 1 (f32)");
    if (fmt != QUARTET_E4M3 && fmt != QUARTET_E5M2) return fail(QUARTET_E_ARG, "fmt must be 0 (e4m3) or 1 (e5m2)");
    if (square != 0 && square != 1) return fail(QUARTET_E_ARG, "square must be 0 (blocks of 1 x 128) or 1 (128 x 128)");
    if (rows < 1 || cols < 1 || rows > 8388480 || cols > 0x3FFFFFFF)
        return fail(QUARTET_E_SHAPE, "need 1 <= rows <= 8388480 and cols >= 1 (got %lld x %lld)", (long long)rows, (long long)cols);
    if (reinterpret_cast<uintptr_t>(x) & (x_dtype == QUARTET_F32 ? 3u : 1u)) return fail(QUARTET_E_ALIGN, "x must be aligned to its type");
    if (!aligned16(codes) || !aligned16(sf) || !aligned16(codes_t) || !aligned16(sf_t)) return fail(QUARTET_E_ALIGN, "outputs must be 16-byte aligned");
    int rc = bind_context_of(x);
    if (rc) return rc;
    if ((rc = check_device())) return rc;
    const bool f32 = x_dtype == QUARTET_F32;
    Fp8QuantParams p{};
    p.x = static_cast<const uint8_t*>(x);
    p.rows = rows, p.cols = cols;
    p.pitch = (cols + 127) / 128 * 128, p.pitch_t = (rows + 127) / 128 * 128;
    p.codes = codes, p.sf = sf, p.codes_t = codes_t, p.sf_t = sf_t;
    p.top = fmt == QUARTET_E4M3 ? 8 : 15;
    p.vec = aligned16(x) && cols % (f32 ? 4 : 8) == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (f32) return square ? pick_quant_fp8<true, true>(p, s) : pick_quant_fp8<true, false>(p, s);
    return square ? pick_quant_fp8<false, true>(p, s) : pick_quant_fp8<false, false>(p, s);
}

extern "C" __attribute__((visibility("default"))) int quartet_dequant_fp8(const uint8_t* codes, const uint8_t* sf, int64_t rows, int64_t cols, int fmt,
                                                                          float scale, void* out, int out_dtype, quartet_stream_t stream) {
    if (!codes || !sf || !out) return fail(QUARTET_E_NULL, "codes, sf and out must be non-NULL");
    if (fmt != QUARTET_E4M3 && fmt != QUARTET_E5M2) return fail(QUARTET_E_ARG, "fmt must be 0 (e4m3) or 1 (e5m2)");
    if (out_dtype != QUARTET_BF16 && out_dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "out_dtype must be 0 or 1");
    if (rows < 1 || cols < 1 || rows > 0x7FFFFFFF || cols > 0x3FFFFFFF)
        return fail(QUARTET_E_SHAPE, "need rows, cols >= 1 (got %lld x %lld)", (long long)rows, (long long)cols);
    if (!aligned16(codes) || !aligned16(out)) return fail(QUARTET_E_ALIGN, "codes and out must be 16-byte aligned");
    int rc = bind_context_of(codes);
    if (rc) return rc;
    if ((rc = check_device())) return rc;
    const int64_t total = rows * ((cols + 3) / 4), pitch = (cols + 127) / 128 * 128;
    const unsigned grid = (unsigned)((total + 255) / 256 < 148 * 16 ? (total + 255) / 256 : 148 * 16);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_dtype == QUARTET_F32)
        dequant_fp8_kernel<true><<<grid, 256, 0, s>>>(codes, sf, rows, cols, pitch, fmt, scale, out);
    else
        dequant_fp8_kernel<false><<<grid, 256, 0, s>>>(codes, sf, rows, cols, pitch, fmt, scale, out);
    return check_cuda(cudaGetLastError(), "dequant_fp8 launch");
}
