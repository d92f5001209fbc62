// Norm over many tensors at once, and clipping by it.
//
//   n = sqrt(sum over all tensors of g^2)   (or the largest |g|)      c = min(1, max_norm / (n + 1e-6))      g <- g c
//
// Two launches whatever the number of tensors: the first leaves one partial sum per CTA, the second adds the partials in a fixed
// order in every CTA for itself (so no counter, no atomics and no third launch) and scales.  The list of tensors travels in the
// kernel's parameters: nothing is copied to the device, so a call can be captured into a graph.
// Squares of fp32 values are taken and added in 64 bits: gradients whose squares leave the range of 32 bits (above 1.8e19, below 1e-19) keep their
// norm.  A sum of n of them has n / (8192 * 888) * 8 additions in a row and some 30 joins, 2^-53 each: 2^-46 for 71 M values, 2^-41 for 2^31, far below
// the result's own rounding.  bf16 values, twice as many a byte, would be bound by their conversion to 64 bits; their squares are exact in 32, and where
// they lie well inside the range four are added there before the conversion, two roundings of 2^-24 on the sum of squares, 2^-24 on the norm at
// the very most.  That is done where the tensor starts on a 16-byte boundary and not in its last values: the same bf16 values at
// another alignment may give a norm that differs by as much.
// Bound by memory: all gradients are read once for the norm; read again (as far as they have left the 126 MB L2) and written to be scaled.
// 71 M fp32 elements into another buffer 139 us, 0.94 of two reads and a write at the measured rate; the norm of 202 M bf16 elements 61 us, 6600 GB/s.
// (Walking backwards in the second pass, from what the first read last, costs more than it saves: 237 us against 164 for 405 MB of bf16 in place.)
#include <algorithm>
#include <cstdlib>

#include "common.cuh"
#include "quant_math.cuh"

namespace quartet {

constexpr int NORM_THREADS = 256, NORM_MAX_GRID = 148 * 6;  // six CTAs an SM: bf16 at 6600 GB/s, with four 5400
static_assert(NORM_MAX_GRID <= QUARTET_NORM_PARTIALS, "workspace");
constexpr int NORM_CHUNK = 8192;  // elements a CTA takes at a time

template <int CAP>
struct TensorList {
    const void* src[CAP];
    void* dst[CAP];
    int64_t numel[CAP];
    uint32_t first[CAP];   // index of a tensor's first chunk
    uint8_t flags[CAP];    // 1: src fp32, 2: dst fp32, 4: both 16-byte aligned
    int n;
    uint32_t chunks;
};

template <int CAP>
__device__ __forceinline__ int tensor_of(const TensorList<CAP>& l, uint32_t chunk) {
    int lo = 0, hi = l.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// What a thread gathers of its elements.  KIND 0: sum of squares.
template <int KIND>
struct Gather {
    double a[4] = {0.0, 0.0, 0.0, 0.0};
    __device__ __forceinline__ void one(float v, int k = 0) { a[k] = fma((double)v, (double)v, a[k]); }
    __device__ __forceinline__ void f32x4(const float4& v) { one(v.x, 0), one(v.y, 1), one(v.z, 2), one(v.w, 3); }
    __device__ __forceinline__ void bf16x8(const uint4& q) {
        float v[8];
        unpack_bf16x8(q, v);
        const float s0 = fmaf(v[0], v[0], v[1] * v[1]), s1 = fmaf(v[2], v[2], v[3] * v[3]);
        const float s2 = fmaf(v[4], v[4], v[5] * v[5]), s3 = fmaf(v[6], v[6], v[7] * v[7]);
        const float t0 = s0 + s1, t1 = s2 + s3;
        // below 2^-60 a square may have lost bits, above 2^120 a sum may overflow next time; a NaN fails both tests
        if (t0 > 0x1p-60f && t1 > 0x1p-60f && t0 < 0x1p120f && t1 < 0x1p120f) {
            a[0] += (double)t0, a[1] += (double)t1;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) one(v[k], k & 3);
        }
    }
    __device__ __forceinline__ double value() const { return (a[0] + a[1]) + (a[2] + a[3]); }
};
// KIND 1: the largest magnitude, as bits: their integers are ordered like the magnitudes, infinities and NaN on top.
template <>
struct Gather<1> {
    uint32_t m = 0u;
    __device__ __forceinline__ void one(float v, int = 0) { m = max(m, __float_as_uint(v) & 0x7FFFFFFFu); }
    __device__ __forceinline__ void f32x4(const float4& v) { one(v.x), one(v.y), one(v.z), one(v.w); }
    __device__ __forceinline__ void bf16x8(const uint4& q) {
        uint32_t k = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu), __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
        m = max(m, max(k << 16, k & 0xFFFF0000u));
    }
    __device__ __forceinline__ double value() const { return (double)__uint_as_float(m); }
};
template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
    if (KIND == 0) return a + b;
    return (b > a || b != b) ? b : a;
}
// Sum (or maximum) over the CTA, in a fixed order, in every thread.
template <int KIND>
__device__ __forceinline__ double block_join(double v, double* s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join<KIND>(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int w = 1; w < NORM_THREADS / 32; ++w) v = join<KIND>(v, s[w]);
    return v;
}

template <int CAP, int KIND>
__global__ void __launch_bounds__(NORM_THREADS) norm_partials_kernel(const __grid_constant__ TensorList<CAP> l, double* __restrict__ partials, int accumulate) {
    __shared__ double s_red[NORM_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    Gather<KIND> acc;
    for (uint32_t c = blockIdx.x; c < l.chunks; c += gridDim.x) {
        const int i = tensor_of(l, c);
        const int64_t at = (int64_t)(c - l.first[i]) * NORM_CHUNK, left = l.numel[i] - at;
        const int count = left < NORM_CHUNK ? (int)left : NORM_CHUNK;
        int done = 0;
        if (l.flags[i] & 4) {
            if (l.flags[i] & 1) {
                const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(l.src[i]) + at);
                const int n4 = count >> 2;
                done = n4 << 2;
                for (int k = threadIdx.x; k < n4; k += 4 * NORM_THREADS) {
                    float4 v[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = k + u * NORM_THREADS < n4 ? __ldg(q + k + u * NORM_THREADS) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int u = 0; u < 4; ++u) acc.f32x4(v[u]);
                }
            } else {
                const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(l.src[i]) + at);
                const int n8 = count >> 3;
                done = n8 << 3;
                for (int k = threadIdx.x; k < n8; k += 4 * NORM_THREADS) {
                    uint4 v[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = k + u * NORM_THREADS < n8 ? __ldg(q + k + u * NORM_THREADS) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                    for (int u = 0; u < 4; ++u) acc.bf16x8(v[u]);
                }
            }
        }
        for (int k = done + threadIdx.x; k < count; k += NORM_THREADS)
            acc.one((l.flags[i] & 1) ? __ldg(static_cast<const float*>(l.src[i]) + at + k)
                                     : __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t*>(l.src[i]) + at + k) << 16));
    }
    double v = acc.value();
    v = block_join<KIND>(v, s_red);
    if (threadIdx.x == 0) partials[blockIdx.x] = accumulate ? join<KIND>(partials[blockIdx.x], v) : v;
}

// The norm's square (or the norm, KIND 1) from the partials, in every thread.
template <int KIND>
__device__ __forceinline__ double join_partials(const double* __restrict__ partials, int n, double* s) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += NORM_THREADS) v = join<KIND>(v, partials[i]);
    return block_join<KIND>(v, s);
}

template <int KIND>
__global__ void __launch_bounds__(NORM_THREADS) norm_finish_kernel(const double* __restrict__ partials, int n, double* __restrict__ total, float* __restrict__ norm) {
    __shared__ double s_red[NORM_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const double v = join_partials<KIND>(partials, n, s_red);
    if (threadIdx.x == 0) {
        if (total) *total = v;
        if (norm) *norm = (float)(KIND == 0 ? sqrt(v) : v);
    }
}

__device__ __forceinline__ void store_scaled(void* dst, int64_t i, float v, bool f32) {
    if (f32)
        static_cast<float*>(dst)[i] = v;
    else
        static_cast<__nv_bfloat16*>(dst)[i] = __float2bfloat16_rn(v);
}

template <int CAP, int KIND>
__global__ void __launch_bounds__(NORM_THREADS) clip_kernel(const __grid_constant__ TensorList<CAP> l, const double* __restrict__ partials, int n_partials,
                                                           double max_norm, float* __restrict__ norm) {
    __shared__ double s_red[NORM_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const double total = join_partials<KIND>(partials, n_partials, s_red);
    const double nrm = KIND == 0 ? sqrt(total) : total;
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nrm;
    const double ratio = max_norm / (nrm + 1e-6);
    const float coef = ratio >= 1.0 ? 1.0f : (float)ratio;  // a NaN norm makes every gradient NaN
    for (uint32_t c = blockIdx.x; c < l.chunks; c += gridDim.x) {
        const int i = tensor_of(l, c);
        const void* src = l.src[i];
        void* dst = l.dst[i];
        if (coef == 1.0f && src == dst) continue;
        const bool sf = l.flags[i] & 1, df = l.flags[i] & 2;
        const int64_t at = (int64_t)(c - l.first[i]) * NORM_CHUNK, left = l.numel[i] - at;
        const int count = left < NORM_CHUNK ? (int)left : NORM_CHUNK;
        int done = 0;
        if (l.flags[i] & 4) {
            // four loads of 16 bytes under way before the first is used
            if (sf) {
                const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(src) + at);
                const int n4 = count >> 2;
                done = n4 << 2;
                for (int k0 = threadIdx.x; k0 < n4; k0 += 4 * NORM_THREADS) {
                    float4 v[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (k0 + u * NORM_THREADS < n4) v[u] = q[k0 + u * NORM_THREADS];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int k = k0 + u * NORM_THREADS;
                        if (k >= n4) break;
                        const float4 o = make_float4(v[u].x * coef, v[u].y * coef, v[u].z * coef, v[u].w * coef);
                        if (df) {
                            reinterpret_cast<float4*>(static_cast<float*>(dst) + at)[k] = o;
                        } else {
                            const __nv_bfloat162 a = __floats2bfloat162_rn(o.x, o.y), b = __floats2bfloat162_rn(o.z, o.w);
                            reinterpret_cast<uint2*>(static_cast<uint16_t*>(dst) + at)[k] =
                                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                        }
                    }
                }
            } else if (df) {
                // eight bytes in, sixteen out: neighbouring lanes write neighbouring units (two stores of a lane side by side cost a third more)
                const uint2* q = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(src) + at);
                float4* o = reinterpret_cast<float4*>(static_cast<float*>(dst) + at);
                const int n4 = count >> 2;
                done = n4 << 2;
                for (int k0 = threadIdx.x; k0 < n4; k0 += 8 * NORM_THREADS) {
                    uint2 x[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (k0 + u * NORM_THREADS < n4) x[u] = q[k0 + u * NORM_THREADS];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int k = k0 + u * NORM_THREADS;
                        if (k >= n4) break;
                        o[k] = make_float4(__uint_as_float(x[u].x << 16) * coef, __uint_as_float(x[u].x & 0xFFFF0000u) * coef, __uint_as_float(x[u].y << 16) * coef,
                                           __uint_as_float(x[u].y & 0xFFFF0000u) * coef);
                    }
                }
            } else {
                const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at);
                const int n8 = count >> 3;
                done = n8 << 3;
                for (int k0 = threadIdx.x; k0 < n8; k0 += 4 * NORM_THREADS) {
                    uint4 x[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (k0 + u * NORM_THREADS < n8) x[u] = q[k0 + u * NORM_THREADS];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int k = k0 + u * NORM_THREADS;
                        if (k >= n8) break;
                        float v[8];
                        unpack_bf16x8(x[u], v);
                        uint32_t w[4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const __nv_bfloat162 a = __floats2bfloat162_rn(v[2 * t] * coef, v[2 * t + 1] * coef);
                            w[t] = *reinterpret_cast<const uint32_t*>(&a);
                        }
                        reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + at)[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
        for (int k = done + threadIdx.x; k < count; k += NORM_THREADS) {
            const float v = sf ? static_cast<const float*>(src)[at + k] : __uint_as_float((uint32_t)static_cast<const uint16_t*>(src)[at + k] << 16);
            store_scaled(dst, at + k, v * coef, df);
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int LIST_SMALL = 64, LIST_LARGE = 768;

// Tensors [i0, ...) into the list, skipping empty ones, as many as fit; returns the next index.
template <int CAP>
static int fill_list(TensorList<CAP>& l, int i0, int n, const void* const* src, void* const* dst, const int64_t* numels, const int32_t* src_dtypes,
                     const int32_t* dst_dtypes) {
    l.n = 0, l.chunks = 0;
    int i = i0;
    for (; i < n && l.n < CAP; ++i) {
        if (numels[i] == 0) continue;
        const uint64_t chunks = (uint64_t)(numels[i] + NORM_CHUNK - 1) / NORM_CHUNK;
        if (l.n && l.chunks + chunks > 0x7FFFFFFFu) break;
        const int k = l.n++;
        l.src[k] = src[i], l.dst[k] = dst ? dst[i] : nullptr, l.numel[k] = numels[i];
        l.first[k] = l.chunks;
        l.flags[k] = (uint8_t)((src_dtypes[i] == QUARTET_F32 ? 1 : 0) | (dst && dst_dtypes[i] == QUARTET_F32 ? 2 : 0) |
                               (aligned16(src[i]) && (!dst || aligned16(dst[i])) ? 4 : 0));
        l.chunks += (uint32_t)chunks;
    }
    return i;
}

static int validate_list(int n, const void* const* src, const int64_t* numels, const int32_t* dtypes, const char* what) {
    if (n < 0) return fail(QUARTET_E_ARG, "n must be >= 0");
    if (n && (!src || !numels || !dtypes)) return fail(QUARTET_E_NULL, "%s, numels and dtypes must be non-NULL", what);
    for (int i = 0; i < n; ++i) {
        if (numels[i] < 0 || numels[i] > ((int64_t)1 << 43)) return fail(QUARTET_E_SHAPE, "tensor %d: bad element count", i);
        if (dtypes[i] != QUARTET_BF16 && dtypes[i] != QUARTET_F32) return fail(QUARTET_E_ARG, "tensor %d: dtype must be 0 (bf16) or 1 (f32)", i);
        if (numels[i] && !src[i]) return fail(QUARTET_E_NULL, "tensor %d of %s is NULL", i, what);
        if (reinterpret_cast<uintptr_t>(src[i]) & (dtypes[i] == QUARTET_F32 ? 3u : 1u)) return fail(QUARTET_E_ALIGN, "tensor %d is not aligned to its type", i);
    }
    return QUARTET_OK;
}

struct Span {
    uintptr_t begin, end;
    int index;
};

// Outputs may not share memory with one another, nor with a gradient other than their own, and with that only when they are the
// same tensor: the CTAs scale in no particular order.
static int refuse_overlap(int n, const void* const* src, void* const* dst, const int64_t* numels, const int32_t* src_dtypes, const int32_t* dst_dtypes) {
    if (n == 0) return QUARTET_OK;
    Span* out = static_cast<Span*>(malloc(sizeof(Span) * (size_t)n));
    if (!out) return fail(QUARTET_E_CUDA, "out of host memory");
    int m = 0, rc = QUARTET_OK;
    for (int i = 0; i < n; ++i) {
        const uintptr_t b = reinterpret_cast<uintptr_t>(dst[i]);
        if (numels[i]) out[m++] = Span{b, b + (uintptr_t)numels[i] * (dst_dtypes[i] == QUARTET_F32 ? 4 : 2), i};
    }
    std::sort(out, out + m, [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (int k = 1; k < m && !rc; ++k)
        if (out[k].begin < out[k - 1].end) rc = fail(QUARTET_E_ARG, "outputs %d and %d share memory", out[k - 1].index, out[k].index);
    for (int i = 0; i < n && !rc; ++i) {
        if (!numels[i]) continue;
        const uintptr_t b = reinterpret_cast<uintptr_t>(src[i]), e = b + (uintptr_t)numels[i] * (src_dtypes[i] == QUARTET_F32 ? 4 : 2);
        // the outputs are disjoint and sorted: the first that ends behind b is the first that can share memory with [b, e)
        const Span* o = std::partition_point(out, out + m, [b](const Span& a) { return a.end <= b; });
        for (; o != out + m && o->begin < e && !rc; ++o)
            if (o->index != i || o->begin != b || src_dtypes[i] != dst_dtypes[i])
                rc = fail(QUARTET_E_ARG, "gradient %d shares memory with output %d", i, o->index);
    }
    free(out);
    return rc;
}

static unsigned norm_grid(uint32_t chunks) { return chunks < 1 ? 1u : chunks < NORM_MAX_GRID ? chunks : NORM_MAX_GRID; }
// CTAs that scale: sixteen an SM, of which four are resident; 71 M fp32 elements 139 us, 143 with six, 159 with two
static unsigned clip_grid(uint32_t chunks) { return chunks < 1 ? 1u : chunks < 148 * 16 ? chunks : 148 * 16; }

template <int CAP>
static int run_partials(int n, const void* const* src, const int64_t* numels, const int32_t* dtypes, int kind, double* partials, int* used, cudaStream_t s) {
    static thread_local TensorList<CAP> l;  // too large for the stack of a small thread
    int i = 0;
    *used = 0;
    do {
        i = fill_list(l, i, n, src, nullptr, numels, dtypes, nullptr);
        // the first launch sets its partials; a later one adds to those that are set, and may not use more of them
        const bool first = *used == 0;
        const unsigned grid = first ? (i < n ? (unsigned)NORM_MAX_GRID : norm_grid(l.chunks)) : (unsigned)*used;
        auto kern = kind == 0 ? norm_partials_kernel<CAP, 0> : norm_partials_kernel<CAP, 1>;
        const int rc = check_cuda(launch_pdl(kern, dim3(grid), dim3(NORM_THREADS), 0, s, l, partials, first ? 0 : 1), "norm launch");
        if (rc) return rc;
        *used = (int)grid;
    } while (i < n);
    return QUARTET_OK;
}

static int partials_of(int n, const void* const* src, const int64_t* numels, const int32_t* dtypes, int kind, double* partials, int* used, cudaStream_t s) {
    return n <= LIST_SMALL ? run_partials<LIST_SMALL>(n, src, numels, dtypes, kind, partials, used, s)
                           : run_partials<LIST_LARGE>(n, src, numels, dtypes, kind, partials, used, s);
}

template <int CAP>
static int run_clip(int n, const void* const* src, void* const* dst, const int64_t* numels, const int32_t* src_dtypes, const int32_t* dst_dtypes, int kind,
                    const double* partials, int n_partials, double max_norm, float* norm, cudaStream_t s) {
    static thread_local TensorList<CAP> l;
    int i = 0;
    do {
        i = fill_list(l, i, n, src, dst, numels, src_dtypes, dst_dtypes);
        auto kern = kind == 0 ? clip_kernel<CAP, 0> : clip_kernel<CAP, 1>;
        const int rc = check_cuda(launch_pdl(kern, dim3(clip_grid(l.chunks)), dim3(NORM_THREADS), 0, s, l, partials, n_partials, max_norm, norm), "clip launch");
        if (rc) return rc;
        norm = nullptr;
    } while (i < n);
    return QUARTET_OK;
}

}  // namespace quartet

using namespace quartet;

extern "C" __attribute__((visibility("default"))) int quartet_grad_norm(int32_t n, const void* const* grads, const int64_t* numels, const int32_t* dtypes,
                                                                        int kind, double* workspace, double* total, float* norm, quartet_stream_t stream) {
    if (kind != 0 && kind != 1) return fail(QUARTET_E_ARG, "kind must be 0 (2-norm) or 1 (largest magnitude)");
    if (!workspace || (!total && !norm)) return fail(QUARTET_E_NULL, "need workspace, and total or norm");
    int rc = validate_list(n, grads, numels, dtypes, "grads");
    if (rc) return rc;
    if ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(total)) & 7u || reinterpret_cast<uintptr_t>(norm) & 3u)
        return fail(QUARTET_E_ALIGN, "workspace and total must be 8-byte aligned, norm 4-byte");
    if ((rc = bind_context_of(workspace))) return rc;
    if ((rc = check_device())) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int used = 0;
    if ((rc = partials_of(n, grads, numels, dtypes, kind, workspace, &used, s))) return rc;
    auto kern = kind == 0 ? norm_finish_kernel<0> : norm_finish_kernel<1>;
    return check_cuda(launch_pdl(kern, dim3(1), dim3(NORM_THREADS), 0, s, (const double*)workspace, used, total, norm), "norm launch");
}

extern "C" __attribute__((visibility("default"))) int quartet_clip_grads(int32_t n, const void* const* grads, void* const* outs, const int64_t* numels,
                                                                         const int32_t* dtypes, const int32_t* out_dtypes, int kind, double max_norm,
                                                                         const double* total, double* workspace, float* norm, quartet_stream_t stream) {
    if (kind != 0 && kind != 1) return fail(QUARTET_E_ARG, "kind must be 0 (2-norm) or 1 (largest magnitude)");
    if (!(max_norm >= 0.0)) return fail(QUARTET_E_ARG, "max_norm must be >= 0");
    if (!total && !workspace) return fail(QUARTET_E_NULL, "need workspace, or the total of quartet_grad_norm");
    int rc = validate_list(n, grads, numels, dtypes, "grads");
    if (rc) return rc;
    if ((rc = validate_list(n, const_cast<const void* const*>(outs), numels, out_dtypes, "outs"))) return rc;
    if ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(total)) & 7u || reinterpret_cast<uintptr_t>(norm) & 3u)
        return fail(QUARTET_E_ALIGN, "workspace and total must be 8-byte aligned, norm 4-byte");
    if ((rc = refuse_overlap(n, grads, outs, numels, dtypes, out_dtypes))) return rc;
    if ((rc = bind_context_of(total ? static_cast<const void*>(total) : workspace))) return rc;
    if ((rc = check_device())) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int used = 1;
    if (!total && (rc = partials_of(n, grads, numels, dtypes, kind, workspace, &used, s))) return rc;
    const double* partials = total ? total : workspace;
    return n <= LIST_SMALL ? run_clip<LIST_SMALL>(n, grads, outs, numels, dtypes, out_dtypes, kind, partials, used, max_norm, norm, s)
                           : run_clip<LIST_LARGE>(n, grads, outs, numels, dtypes, out_dtypes, kind, partials, used, max_norm, norm, s);
}
