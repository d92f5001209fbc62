// Arithmetic of the 8-bit quantizers: the scale byte of a block, the conversion to codes, and sixteen values of a row as one thread holds them.
#pragma once
#include "common.cuh"
#include "quant_math.cuh"

namespace quartet {

__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits, int top) {
    if (amax_bits >= 0x7F800000u) return 255u;
    const int b = (int)(amax_bits >> 23) - top + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0u : (uint32_t)b;
}
// 2^(127 - b); b <= 247 here, so the exponent field stays positive
__device__ __forceinline__ float fp8_inv_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }

__device__ __forceinline__ uint32_t cvt_fp8x4(float a, float b, float c, float d, bool e5m2) {
    uint16_t lo, hi;
    if (e5m2) {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    } else {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    }
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Sixteen values of a row as 16-byte chunks j, j + 8 (bf16) or j, j + 8, j + 16, j + 24 (fp32) of the 128 columns; zeros
// outside the tensor.
template <bool F32>
struct RowPart {
    static constexpr int N = F32 ? 4 : 2, PER = F32 ? 4 : 8;
    uint4 q[N];
    __device__ __forceinline__ void load(const uint8_t* x, int64_t rows, int64_t cols, int vec, int64_t row, int64_t col0, int j) {
        constexpr int EB = F32 ? 4 : 2;
        const uint8_t* base = x + row * cols * EB;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t c = col0 + (j + 8 * i) * PER;
            q[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row >= rows) continue;
            if (vec) {  // cols is a multiple of PER: a chunk is inside or outside as a whole
                if (c < cols) q[i] = __ldg(reinterpret_cast<const uint4*>(base + c * EB));
            } else {
                uint32_t w[4] = {0u, 0u, 0u, 0u};
                for (int k = 0; k < PER; ++k) {
                    if (c + k >= cols) break;
                    if (F32)
                        w[k & 3] = __ldg(reinterpret_cast<const uint32_t*>(base) + c + k);
                    else
                        w[k >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(base) + c + k) << (16 * (k & 1));
                }
                q[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    __device__ __forceinline__ void chunk(int i, float (&v)[PER]) const {
        if constexpr (F32) {
            v[0] = __uint_as_float(q[i].x), v[1] = __uint_as_float(q[i].y), v[2] = __uint_as_float(q[i].z), v[3] = __uint_as_float(q[i].w);
        } else {
            unpack_bf16x8(q[i], v);
        }
    }
    // bits of the largest magnitude: integer order is the order of magnitudes, infinities and NaN on top
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[PER];
            chunk(i, v);
#pragma unroll
            for (int k = 0; k < PER; ++k) m = max(m, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        }
        return m;
    }
    // the PER codes of chunk i, four to a word
    __device__ __forceinline__ void codes(uint32_t (&w)[PER / 4], int i, uint32_t sb, bool e5m2) const {
        const float inv = fp8_inv_scale(sb == 255u ? 127u : sb);
        float v[PER];
        chunk(i, v);
#pragma unroll
        for (int k = 0; k < PER / 4; ++k) {
            w[k] = cvt_fp8x4(v[4 * k] * inv, v[4 * k + 1] * inv, v[4 * k + 2] * inv, v[4 * k + 3] * inv, e5m2);
            if (sb == 255u) w[k] = 0x7F7F7F7Fu;
        }
    }
    __device__ __forceinline__ void store_codes(uint8_t* dst, int i, uint32_t sb, bool e5m2) const {
        uint32_t w[PER / 4];
        codes(w, i, sb, e5m2);
        if constexpr (F32)
            *reinterpret_cast<uint32_t*>(dst) = w[0];
        else
            *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    }
};

__device__ __forceinline__ uint32_t max_over_8(uint32_t m) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    return m;
}

}  // namespace quartet
