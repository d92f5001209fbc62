// Rotary positions: in every head the pairs (x1, x2) of the first `rot` values turn by the angle pos * inv_freq[i],
//
//   y1 = s (x1 cos a - x2 sin a)      y2 = s (x1 sin a + x2 cos a)        (inverse: -a)
//
// with the pairs side by side (interleaved: 2 i, 2 i + 1) or half the rotated part apart (i, i + rot / 2); values past `rot` are
// copied.  Up to three segments (q, k, v) share one launch, each with its own strides for batch, token and head, so that
// the split of a packed projection into heads -- and, backward, its join -- is the same pass over memory as the rotation.
//
// Angles: the turn pos * inv_freq / 2 pi is taken in 64 bits and reduced there, because in 32 bits a position of 2^17 leaves an angle
// 2^-7 wrong; its fraction goes to sincospif, with the part that 32 bits lose put back to first order.  A CTA computes the
// rot / 2 pairs of its token once, in shared memory, and every head uses them: the angles cost no memory traffic.
// Bound by memory: each value is read and written once.
#include "common.cuh"
#include "quant_math.cuh"

namespace quartet {

constexpr int ROT_THREADS = 128, ROT_MAX_PAIRS = 256, ROT_MAX_SEGS = 3;

struct RotSeg {
    const void* src;
    void* dst;
    int64_t s_b, s_t, s_h, d_b, d_t, d_h;  // strides in elements; values of a head are adjacent
    int heads, rotate;
};
struct RotParams {
    RotSeg seg[ROT_MAX_SEGS];
    int n_seg, d, rot;
    int64_t T;
    const void* pos;        // NULL: token t is at offset + t
    int pos_i64;
    int64_t pos_b, pos_t, offset;
    const double* inv_freq;
    float scale;
    int inverse;
};

// Values one thread moves at a time: 16 bytes where every row allows it, single values otherwise.
template <bool F32, bool VEC>
struct RotVec {
    static constexpr int N = VEC ? (F32 ? 4 : 8) : 1;
    float v[N];
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        if constexpr (VEC && F32) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
        } else if constexpr (VEC) {
            unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i)), v);
        } else if constexpr (F32) {
            v[0] = __ldg(static_cast<const float*>(p) + i);
        } else {
            v[0] = __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t*>(p) + i) << 16);
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t i) const {
        if constexpr (VEC && F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
        } else if constexpr (VEC) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t*>(&t);
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if constexpr (F32) {
            static_cast<float*>(p)[i] = v[0];
        } else {
            static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v[0]);
        }
    }
};

template <bool F32, bool INTERLEAVED, bool VEC>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const RotParams p) {
    __shared__ __align__(16) float s_cos[ROT_MAX_PAIRS], s_sin[ROT_MAX_PAIRS];
    using V = RotVec<F32, VEC>;
    const int pairs = p.rot >> 1;
    const int64_t token = blockIdx.x, b = token / p.T, t = token - b * p.T;
    pdl_launch_dependents();
    pdl_wait();
    int64_t pos = p.offset + t;
    if (p.pos) {
        const int64_t at = b * p.pos_b + t * p.pos_t;
        pos = p.pos_i64 ? (int64_t)__ldg(static_cast<const long long*>(p.pos) + at) : (int64_t)__ldg(static_cast<const int*>(p.pos) + at);
    }
    for (int i = threadIdx.x; i < pairs; i += ROT_THREADS) {
        double turn = (double)pos * (p.inv_freq[i] * 0.15915494309189533577);
        turn = 2.0 * (turn - rint(turn));  // half turns, in [-1, 1]
        const float hi = (float)turn, lo = (float)(turn - (double)hi) * 3.14159265f;
        float s, c;
        sincospif(hi, &s, &c);
        const float c2 = c - s * lo, s2 = s + c * lo;
        s_cos[i] = c2 * p.scale;
        s_sin[i] = (p.inverse ? -s2 : s2) * p.scale;
    }
    __syncthreads();
    // a unit is what a thread moves at once: one vector of side-by-side pairs, two vectors half a rotated part apart, or
    // one vector that is only copied
    constexpr int RU = INTERLEAVED ? (VEC ? V::N : 2) : 2 * V::N;  // values of a rotated unit
#pragma unroll 1
    for (int g = 0; g < p.n_seg; ++g) {
        const RotSeg& sg = p.seg[g];
        const int turned = sg.rotate ? p.rot : 0;
        const int ru = turned / RU, units = ru + (p.d - turned) / V::N, total = units * sg.heads;
        const int64_t so = b * sg.s_b + t * sg.s_t, to = b * sg.d_b + t * sg.d_t;
        for (int u = threadIdx.x; u < total; u += ROT_THREADS) {
            const int h = u / units, i = u - h * units;
            const int64_t sh = so + h * sg.s_h, dh = to + h * sg.d_h;
            if (i >= ru) {
                V x;
                const int at = turned + (i - ru) * V::N;
                x.load(sg.src, sh + at);
                x.store(sg.dst, dh + at);
            } else if constexpr (INTERLEAVED && VEC) {
                V x, y;
                x.load(sg.src, sh + i * RU);
#pragma unroll
                for (int k = 0; k < V::N / 2; ++k) {
                    const float c = s_cos[i * (RU / 2) + k], s = s_sin[i * (RU / 2) + k];
                    y.v[2 * k] = x.v[2 * k] * c - x.v[2 * k + 1] * s;
                    y.v[2 * k + 1] = x.v[2 * k] * s + x.v[2 * k + 1] * c;
                }
                y.store(sg.dst, dh + i * RU);
            } else {
                const int a1 = INTERLEAVED ? 2 * i : i * V::N, a2 = INTERLEAVED ? 2 * i + 1 : pairs + i * V::N;
                V x1, x2, y1, y2;
                x1.load(sg.src, sh + a1);
                x2.load(sg.src, sh + a2);
#pragma unroll
                for (int k = 0; k < V::N; ++k) {
                    const float c = s_cos[i * V::N + k], s = s_sin[i * V::N + k];
                    y1.v[k] = x1.v[k] * c - x2.v[k] * s;
                    y2.v[k] = x1.v[k] * s + x2.v[k] * c;
                }
                y1.store(sg.dst, dh + a1);
                y2.store(sg.dst, dh + a2);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <bool F32>
static int launch_rotary(const RotParams& p, int64_t tokens, bool interleaved, bool vec, cudaStream_t s) {
    void (*kern)(const RotParams) = interleaved ? (vec ? rotary_kernel<F32, true, true> : rotary_kernel<F32, true, false>)
                                                : (vec ? rotary_kernel<F32, false, true> : rotary_kernel<F32, false, false>);
    return check_cuda(launch_pdl(kern, dim3((unsigned)tokens), dim3(ROT_THREADS), 0, s, p), "rotary launch");
}

}  // namespace quartet

using namespace quartet;

extern "C" __attribute__((visibility("default"))) int quartet_rotary(int n_seg, const void* const* src, void* const* dst, const int64_t* strides6,
                                                                     const int32_t* heads, const int32_t* rotate, int dtype, int64_t batch, int64_t tokens,
                                                                     int64_t d, int64_t rot, int interleaved, const void* pos, int pos_i64, int64_t pos_stride_b,
                                                                     int64_t pos_stride_t, int64_t offset, const double* inv_freq, float scale, int inverse,
                                                                     quartet_stream_t stream) {
    if (n_seg < 1 || n_seg > ROT_MAX_SEGS) return fail(QUARTET_E_ARG, "n_seg must be 1..%d (got %d)", ROT_MAX_SEGS, n_seg);
    if (!src || !dst || !strides6 || !heads || !rotate || !inv_freq) return fail(QUARTET_E_NULL, "src, dst, strides6, heads, rotate and inv_freq must be non-NULL");
    if (dtype != QUARTET_BF16 && dtype != QUARTET_F32) return fail(QUARTET_E_ARG, "dtype must be 0 (bf16) or 1 (f32)");
    if (batch < 1 || tokens < 1 || batch > 0x7FFFFFFF || tokens > 0x7FFFFFFF || batch * tokens > 0x7FFFFFFF)
        return fail(QUARTET_E_SHAPE, "need 1 <= batch * tokens < 2^31 (got %lld x %lld)", (long long)batch, (long long)tokens);
    if (d < 2 || d > 65536 || rot < 2 || rot % 2 || rot > d || rot > 2 * ROT_MAX_PAIRS)
        return fail(QUARTET_E_SHAPE, "need an even rot, 2 <= rot <= min(d, %d) (got rot %lld, d %lld)", 2 * ROT_MAX_PAIRS, (long long)rot, (long long)d);
    const bool f32 = dtype == QUARTET_F32;
    const int eb = f32 ? 4 : 2, per = 16 / eb;
    RotParams p{};
    bool vec = d % per == 0 && (interleaved ? rot : rot / 2) % per == 0;
    for (int g = 0; g < n_seg; ++g) {
        const int64_t* st = strides6 + 6 * g;
        if (!src[g] || !dst[g]) return fail(QUARTET_E_NULL, "segment %d has a NULL pointer", g);
        if (heads[g] < 1 || heads[g] > 65536) return fail(QUARTET_E_SHAPE, "segment %d: need 1 <= heads <= 65536", g);
        if ((reinterpret_cast<uintptr_t>(src[g]) | reinterpret_cast<uintptr_t>(dst[g])) & (uintptr_t)(eb - 1))
            return fail(QUARTET_E_ALIGN, "segment %d is not aligned to its type", g);
        vec = vec && aligned16(src[g]) && aligned16(dst[g]);
        for (int k = 0; k < 6; ++k) vec = vec && st[k] % per == 0;
        p.seg[g] = RotSeg{src[g], dst[g], st[0], st[1], st[2], st[3], st[4], st[5], heads[g], rotate[g] != 0};
    }
    if (reinterpret_cast<uintptr_t>(inv_freq) & 7u) return fail(QUARTET_E_ALIGN, "inv_freq must be 8-byte aligned");
    if (pos && (reinterpret_cast<uintptr_t>(pos) & (pos_i64 ? 7u : 3u))) return fail(QUARTET_E_ALIGN, "pos must be aligned to its type");
    int rc = bind_context_of(src[0]);
    if (rc) return rc;
    if ((rc = check_device())) return rc;
    p.n_seg = n_seg, p.d = (int)d, p.rot = (int)rot, p.T = tokens;
    p.pos = pos, p.pos_i64 = pos_i64, p.pos_b = pos_stride_b, p.pos_t = pos_stride_t, p.offset = offset;
    p.inv_freq = inv_freq, p.scale = scale, p.inverse = inverse != 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return f32 ? launch_rotary<true>(p, batch * tokens, interleaved != 0, vec, s) : launch_rotary<false>(p, batch * tokens, interleaved != 0, vec, s);
}
