// Arithmetic of the 8-bit quantizers: the scale byte of a block, the conversion to codes, and sixteen values of a row as one thread holds them.
// The quantizers are bound by instruction issue before they are bound by memory, so magnitudes of bf16 values are compared two
// at a time as packed 16-bit integers and products are taken in packed fp32 pairs.
#pragma once
#include "common.cuh"
#include "quant_math.cuh"

namespace quartet {

// Bits of an fp32 magnitude -> scale byte: the least e with amax <= 1.75 * 2^(top + e), or 255 for an infinity or a NaN.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits, int top) {
    if (amax_bits >= 0x7F800000u) return 255u;
    const int b = (int)(amax_bits >> 23) - top + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0u : (uint32_t)b;
}
// 2^(127 - b); b <= 247 for finite blocks, so the exponent field stays positive.  NaN for byte 255: every code of the block becomes NaN.
__device__ __forceinline__ float fp8_inv_scale(uint32_t b) { return __uint_as_float(b == 255u ? 0x7FC00000u : (254u - b) << 23); }

template <bool E5M2>
__device__ __forceinline__ uint32_t cvt_fp8x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    if constexpr (E5M2) {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    } else {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    }
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// The largest magnitude of words of values, as bits: the order of the integers is that of the magnitudes, infinities and NaN on top.  fp32: the
// larger of two magnitudes, NaN first.  bf16 pairs: as 16-bit integers, negative values too order by magnitude among themselves, both
// signed and unsigned; the signed maximum finds the largest positive value, the unsigned one the largest negative value if there is
// one, so that no sign has to be cleared word by word.  Words are taken in pairs: both have three-operand instructions.
template <bool F32>
struct Mag;
template <>
struct Mag<true> {
    float m = 0.f;
    __device__ __forceinline__ void take(uint32_t a, uint32_t b) {
        asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(fabsf(__uint_as_float(a))), "f"(fabsf(__uint_as_float(b))));
    }
    __device__ __forceinline__ uint32_t packed() const { return __float_as_uint(m); }
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t bits(uint32_t m) { return m; }
};
template <>
struct Mag<false> {
    uint32_t s = 0u, u = 0u;
    __device__ __forceinline__ void take(uint32_t a, uint32_t b) {
        s = __vimax3_s16x2(s, a, b);
        u = __vimax3_u16x2(u, a, b);
    }
    __device__ __forceinline__ uint32_t packed() const { return __vmaxu2(s, u & 0x7FFF7FFFu); }  // of the low and of the high halves
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
    static __device__ __forceinline__ uint32_t bits(uint32_t m) { return max(m << 16, m & 0xFFFF0000u); }  // as an fp32 value's
};

// Sixteen values of a row as 16-byte chunks j, j + 8 (bf16) or j, j + 8, j + 16, j + 24 (fp32) of 128 columns; zeros outside the tensor.
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
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    if (c + k < cols) {
                        if (F32)
                            w[k & 3] = __ldg(reinterpret_cast<const uint32_t*>(base) + c + k);
                        else
                            w[k >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(base) + c + k) << (16 * (k & 1));
                    }
                }
                q[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    __device__ __forceinline__ uint32_t mag() const {  // packed
        Mag<F32> m;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            m.take(q[i].x, q[i].y);
            m.take(q[i].z, q[i].w);
        }
        return m.packed();
    }
    // the PER codes of chunk i, four to a word
    template <bool E5M2>
    __device__ __forceinline__ void codes(uint32_t (&w)[PER / 4], int i, float inv) const {
        const uint32_t r[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
        const f32x2_t s = pack2(inv, inv);
#pragma unroll
        for (int k = 0; k < PER / 4; ++k) {
            float a, b, c, d;
            if constexpr (F32) {
                unpack2(mul2(pack2(__uint_as_float(r[0]), __uint_as_float(r[1])), s), a, b);
                unpack2(mul2(pack2(__uint_as_float(r[2]), __uint_as_float(r[3])), s), c, d);
            } else {
                unpack2(mul2(pack2(__uint_as_float(r[2 * k] << 16), __uint_as_float(r[2 * k] & 0xFFFF0000u)), s), a, b);
                unpack2(mul2(pack2(__uint_as_float(r[2 * k + 1] << 16), __uint_as_float(r[2 * k + 1] & 0xFFFF0000u)), s), c, d);
            }
            w[k] = cvt_fp8x4<E5M2>(a, b, c, d);
        }
    }
    template <bool E5M2>
    __device__ __forceinline__ void store_codes(uint8_t* dst, int i, float inv) const {
        uint32_t w[PER / 4];
        codes<E5M2>(w, i, inv);
        if constexpr (F32)
            *reinterpret_cast<uint32_t*>(dst) = w[0];
        else
            *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    }
};

// over the eight threads of a row
template <bool F32>
__device__ __forceinline__ uint32_t mag_over_8(uint32_t m) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = Mag<F32>::join(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    return Mag<F32>::bits(m);
}

}  // namespace quartet
