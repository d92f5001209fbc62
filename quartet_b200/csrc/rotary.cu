// Rotary positions: in every head the pairs (x1, x2) of the first `rot` values turn by the angle pos * inv_freq[i],
//
//   y1 = s (x1 cos a - x2 sin a)      y2 = s (x1 sin a + x2 cos a)        (inverse: -a)
//
// with the pairs side by side (interleaved: 2 i, 2 i + 1) or half the rotated part apart (i, i + rot / 2); values past `rot` are
// copied.  Up to three segments (q, k, v) share one launch, each with its own strides for batch, token and head, so that
// the split of a packed projection into heads -- and, backward, its join -- is the same pass over memory as the rotation.
//
// Angles: the turn pos * inv_freq / 2 pi is taken in 64 bits and reduced there, because in 32 bits a position of 2^17 leaves an angle
// 2^-7 wrong; its fraction goes to sincospif, with the part that 32 bits lose put back to first order.  From there on it is 32 bits, the scale included:
// fp32 results are 5.8e-8 from the exact ones where rounding scale * cos once from 64 bits leaves 4.0e-8.  They cost no memory traffic
// and no table in it: a thread owns the same few pairs of a token in all heads of all segments, computes their sines and cosines once, keeps
// them in registers and walks the heads in batches, the next batch's loads under way while one is turned and stored.  Where there are few
// tokens a thread takes every split-th head, and the threads of a token share its pairs through shared memory.
// Bound by memory: each value is read and written once.
#include <algorithm>

#include "common.cuh"
#include "quant_math.cuh"

namespace quartet {

constexpr int ROT_THREADS = 256, ROT_MAX_PAIRS = 256, ROT_MAX_SEGS = 3;

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
    int64_t tokens;
    int lanes, split, per_block;  // threads a token and head group, head groups, tokens of a block
};

// Values one thread moves at a time: as many bytes (16, 8, 4, or a single value) as every row and every half of a row allows.
template <bool F32, int BYTES>
struct RotVec {
    static constexpr int N = BYTES / (F32 ? 4 : 2), WORDS = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t q[WORDS];
    // (plain loads, not read-only ones: a tensor may be turned in place)
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (BYTES == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w;
        } else if constexpr (BYTES == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            q[0] = v.x, q[1] = v.y;
        } else if constexpr (BYTES == 4) {
            q[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            q[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void copy(uint8_t* p) const {
        if constexpr (BYTES == 16)
            *reinterpret_cast<uint4*>(p) = make_uint4(q[0], q[1], q[2], q[3]);
        else if constexpr (BYTES == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(q[0], q[1]);
        else if constexpr (BYTES == 4)
            *reinterpret_cast<uint32_t*>(p) = q[0];
        else
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)q[0];
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int k = 0; k < WORDS; ++k) {
            if constexpr (F32) {
                v[k] = __uint_as_float(q[k]);
            } else {
                v[N == 1 ? 0 : 2 * k] = __uint_as_float(q[k] << 16);
                if constexpr (N > 1) v[2 * k + 1] = __uint_as_float(q[k] & 0xFFFF0000u);
            }
        }
    }
    static __device__ __forceinline__ void store(uint8_t* p, const float (&v)[N]) {
        RotVec r;
#pragma unroll
        for (int k = 0; k < WORDS; ++k) {
            if constexpr (F32) {
                r.q[k] = __float_as_uint(v[k]);
            } else if constexpr (N == 1) {
                r.q[k] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
            } else {
                const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                r.q[k] = *reinterpret_cast<const uint32_t*>(&t);
            }
        }
        r.copy(p);
    }
};

__device__ __forceinline__ int64_t position(const RotParams& p, int64_t token) {
    const int64_t b = (uint32_t)token / (uint32_t)p.T, t = token - b * p.T;
    if (!p.pos) return p.offset + t;
    const int64_t at = b * p.pos_b + t * p.pos_t;
    return p.pos_i64 ? (int64_t)__ldg(static_cast<const long long*>(p.pos) + at) : (int64_t)__ldg(static_cast<const int*>(p.pos) + at);
}
// (cosine, sine) of a pair at a position, times the scale
__device__ __forceinline__ float2 rotation(const RotParams& p, int64_t pos, int pair) {
    double turn = (double)pos * (__ldg(p.inv_freq + pair) * 0.15915494309189533577);
    turn = 2.0 * (turn - rint(turn));  // half turns, in [-1, 1]
    const float hi = (float)turn, lo = (float)(turn - (double)hi) * 3.14159265f;
    float s, c;
    sincospif(hi, &s, &c);
    return make_float2((c - s * lo) * p.scale, (s + c * lo) * (p.inverse ? -p.scale : p.scale));
}

template <bool F32, int BYTES, bool INTERLEAVED, bool SPLIT>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const __grid_constant__ RotParams p) {
    using V = RotVec<F32, BYTES>;
    // A unit is what a thread moves of every head: one vector of side-by-side pairs, two vectors half a rotated part apart (two single
    // values, in either layout), or one vector that is only copied.  The units cover a head, so a segment that is not turned (v) is
    // copied by the same units.
    constexpr bool ONE = INTERLEAVED && V::N > 1;
    constexpr int RU = ONE ? V::N : 2 * V::N, PAIRS = RU / 2, ES = F32 ? 4 : 2;
    constexpr int BATCH = SPLIT ? 1 : ONE ? 4 : 2;  // heads: 64 bytes a batch
    extern __shared__ __align__(16) float2 s_cs[];  // [token of the block][pair]
    const int ru = p.rot / RU, units = ru + (p.d - p.rot) / V::N;
    const int lane = threadIdx.x % p.lanes, rest = threadIdx.x / p.lanes, group = rest % p.split, mine = rest / p.split;
    const int pairs = p.rot >> 1;
    const int64_t token = (int64_t)blockIdx.x * p.per_block + mine;
    pdl_launch_dependents();
    pdl_wait();
    if constexpr (SPLIT) {
        for (int i = threadIdx.x; i < p.per_block * pairs; i += blockDim.x) {
            const int64_t tok = (int64_t)blockIdx.x * p.per_block + i / pairs;
            if (tok >= p.tokens) break;
            s_cs[i] = rotation(p, position(p, tok), i % pairs);
        }
        __syncthreads();
    }
    if (token >= p.tokens) return;
    const int64_t b = (uint32_t)token / (uint32_t)p.T, t = token - b * p.T;
    for (int i = lane; i < units; i += p.lanes) {
        const bool turns = i < ru, two = !ONE && turns;
        const int a1 = !turns ? p.rot + (i - ru) * V::N : ONE ? i * RU : (INTERLEAVED ? 2 * i : i * V::N);
        const int64_t gap = (int64_t)(INTERLEAVED ? 1 : p.rot >> 1) * ES;   // from the unit's first vector to its second
        const int64_t step = p.split;
        auto load = [&](V (&x1)[BATCH], V (&x2)[BATCH], int g, int h) {
            const RotSeg& sg = p.seg[g];
            const uint8_t* src = static_cast<const uint8_t*>(sg.src) + (b * sg.s_b + t * sg.s_t + h * sg.s_h + a1) * ES;
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                if (h + u * step < sg.heads) {
                    x1[u].load(src);
                    if (two) x2[u].load(src + gap);
                }
                src += step * sg.s_h * ES;
            }
        };
        auto next = [&](int& g, int& h) {
            while (g < p.n_seg && h >= p.seg[g].heads) ++g, h = group;
        };
        V x1[BATCH], x2[BATCH], y1[BATCH], y2[BATCH];
        int g = 0, h = group;
        next(g, h);
        if (g < p.n_seg) load(x1, x2, g, h);
        float cs[PAIRS], sn[PAIRS];
        if (turns) {
            const int64_t pos = SPLIT ? 0 : position(p, token);
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                const float2 v = SPLIT ? s_cs[mine * pairs + i * PAIRS + k] : rotation(p, pos, i * PAIRS + k);
                cs[k] = v.x, sn[k] = v.y;
            }
        }
#pragma unroll 1
        while (g < p.n_seg) {
            int g2 = g, h2 = h + BATCH * p.split;
            next(g2, h2);
            if (g2 < p.n_seg) load(y1, y2, g2, h2);
            const RotSeg& sg = p.seg[g];
            uint8_t* dst = static_cast<uint8_t*>(sg.dst) + (b * sg.d_b + t * sg.d_t + h * sg.d_h + a1) * ES;
            const bool turn = turns && sg.rotate;
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                if (h + u * step < sg.heads) {
                    if (!turn) {
                        x1[u].copy(dst);
                        if (two) x2[u].copy(dst + gap);
                    } else if constexpr (ONE) {
                        float v[V::N], w[V::N];
                        x1[u].get(v);
#pragma unroll
                        for (int k = 0; k < PAIRS; ++k) {
                            w[2 * k] = v[2 * k] * cs[k] - v[2 * k + 1] * sn[k];
                            w[2 * k + 1] = v[2 * k] * sn[k] + v[2 * k + 1] * cs[k];
                        }
                        V::store(dst, w);
                    } else {
                        float v1[V::N], v2[V::N], w1[V::N], w2[V::N];
                        x1[u].get(v1);
                        x2[u].get(v2);
#pragma unroll
                        for (int k = 0; k < PAIRS; ++k) {
                            w1[k] = v1[k] * cs[k] - v2[k] * sn[k];
                            w2[k] = v1[k] * sn[k] + v2[k] * cs[k];
                        }
                        V::store(dst, w1);
                        V::store(dst + gap, w2);
                    }
                }
                dst += step * sg.d_h * ES;
                x1[u] = y1[u], x2[u] = y2[u];
            }
            g = g2, h = h2;
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Whether two of the strided tensors of a launch share memory.  A tensor is the set of addresses base + sum over its axes of index * stride; two of
// them meet where the difference of their bases is a sum over all axes of coefficient * stride, each coefficient between limits.  That is
// searched axis by axis, largest stride first: what the axes behind can still reach leaves one or two coefficients of each to try where the axes
// nest, as those of views of one buffer do.
// (A launch is a few microseconds of host time: ranges that lie apart and axes that nest are told without a search, half of one in all.)
struct RotSpan {
    int64_t base, n[4], st[4];  // bytes; batch, token, head, value, an axis of one entry with stride 0
    int64_t reach;              // last value's address - first's
};
struct RotAxis {
    int64_t st, lo, hi;
};
constexpr int ROT_SEARCH = 4096;  // coefficients tried before the answer is "cannot tell"

static RotSpan rot_span(const void* p, int eb, int64_t batch, int64_t tokens, int64_t heads, int64_t d, const int64_t* st3) {
    RotSpan s{(int64_t)reinterpret_cast<uintptr_t>(p), {batch, tokens, heads, d}, {st3[0] * eb, st3[1] * eb, st3[2] * eb, eb}, 0};
    for (int i = 0; i < 4; ++i) {
        if (s.n[i] == 1) s.st[i] = 0;
        if (s.st[i] < 0) s.base += (s.n[i] - 1) * s.st[i], s.st[i] = -s.st[i];
        s.reach += (s.n[i] - 1) * s.st[i];
    }
    return s;
}
static inline int64_t floor_div(int64_t a, int64_t b) {
    if (a >= 0 && a < b) return 0;
    if (a < 0 && a >= -b) return -1;
    const int64_t q = a / b;
    return q - (q * b > a);
}

// 1: some choice of coefficients from axis i on adds up to `left` (`moved`: a choice of another address than a tensor's with itself), 0: none, -1: not
// found in ROT_SEARCH steps.  lo, hi: what the axes from i on reach.
static int rot_meets(const RotAxis* ax, int n, int i, int64_t left, int64_t lo, int64_t hi, bool moved, int& steps) {
    if (i == n) return left == 0 && moved;
    lo -= ax[i].lo * ax[i].st, hi -= ax[i].hi * ax[i].st;
    const int64_t first = std::max(ax[i].lo, -floor_div(hi - left, ax[i].st)), last = std::min(ax[i].hi, floor_div(left - lo, ax[i].st));
    for (int64_t c = first; c <= last; ++c) {
        if (--steps < 0) return -1;
        const int r = rot_meets(ax, n, i + 1, left - c * ax[i].st, lo, hi, moved || c != 0, steps);
        if (r) return r;
    }
    return 0;
}
static int rot_search(RotAxis* ax, int n, int64_t left, bool moved) {
    std::sort(ax, ax + n, [](const RotAxis& x, const RotAxis& y) { return x.st > y.st; });
    int64_t lo = 0, hi = 0;
    for (int k = 0; k < n; ++k) lo += ax[k].lo * ax[k].st, hi += ax[k].hi * ax[k].st;
    int steps = ROT_SEARCH;
    return rot_meets(ax, n, 0, left, lo, hi, moved, steps);
}
// Whether two indexes of one tensor share an address.
static int rot_folds(const RotSpan& a) {
    int64_t inner = -1;  // axes that nest: every stride is more than all smaller ones reach together
    int order[4], n = 0;
    for (int i = 0; i < 4; ++i) {
        if (a.n[i] == 1) continue;
        if (a.st[i] == 0) return 1;
        int k = n++;
        for (; k > 0 && a.st[order[k - 1]] > a.st[i]; --k) order[k] = order[k - 1];
        order[k] = i;
    }
    bool nest = true;
    for (int k = 0; k < n && nest; ++k) {
        nest = a.st[order[k]] > inner;
        inner = std::max<int64_t>(inner, 0) + (a.n[order[k]] - 1) * a.st[order[k]];
    }
    if (nest) return 0;
    RotAxis ax[4];
    for (int k = 0; k < n; ++k) {
        if (k && a.st[order[k]] == a.st[order[k - 1]]) return 1;
        ax[k] = RotAxis{a.st[order[k]], 1 - a.n[order[k]], a.n[order[k]] - 1};
    }
    return rot_search(ax, n, 0, false);
}
// Whether two tensors share an address.
static int rot_overlap(const RotSpan& a, const RotSpan& b) {
    if (a.base > b.base + b.reach || b.base > a.base + a.reach) return 0;
    RotAxis ax[8];
    int n = 0;
    auto axis = [&](int64_t st, int64_t lo, int64_t hi) {
        for (int k = 0; k < n; ++k)
            if (ax[k].st == st) {
                ax[k].lo += lo, ax[k].hi += hi;
                return;
            }
        ax[n++] = RotAxis{st, lo, hi};
    };
    for (int i = 0; i < 4; ++i) {
        if (a.st[i]) axis(a.st[i], 0, a.n[i] - 1);
        if (b.st[i]) axis(b.st[i], 1 - b.n[i], 0);
    }
    return rot_search(ax, n, b.base - a.base, true);
}
// Every value is read by one thread and written by another, in no order: a dst may be its own src as a whole and nothing else's, nor hold one
// value twice.
static int refuse_rotary_overlap(int n_seg, const RotSpan* src, const RotSpan* dst) {
    auto same = [](const RotSpan& a, const RotSpan& b) { return a.base == b.base && std::equal(a.st, a.st + 4, b.st); };
    for (int g = 0; g < n_seg; ++g) {
        if (rot_folds(dst[g])) return fail(QUARTET_E_ARG, "dst %d holds several values at one address", g);
        for (int h = 0; h < n_seg; ++h) {
            if (h < g && rot_overlap(dst[g], dst[h])) return fail(QUARTET_E_ARG, "dst %d and dst %d share memory", h, g);
            if (!(g == h && same(dst[g], src[h])) && rot_overlap(dst[g], src[h])) return fail(QUARTET_E_ARG, "dst %d shares memory with src %d", g, h);
        }
    }
    return QUARTET_OK;
}

template <bool F32, int BYTES>
static int launch_rotary(RotParams p, bool interleaved, cudaStream_t s) {
    int rc, sms = 0, heads = 1;
    if ((rc = device_sm_count(&sms))) return rc;
    constexpr int n = BYTES / (F32 ? 4 : 2);
    const int ru = interleaved && n > 1 ? n : 2 * n;
    const int units = p.rot / ru + (p.d - p.rot) / n;
    p.lanes = units < ROT_THREADS ? units : ROT_THREADS;
    for (int g = 0; g < p.n_seg; ++g) heads = p.seg[g].heads > heads ? p.seg[g].heads : heads;
    // Head groups: one, so that a pair's sine and cosine are computed once by one thread, unless the threads would then be fewer than 256 an SM (a
    // new token of each sequence; 3063 tokens of 12 fp32 heads 5.9 us with two groups, 7.7 with eight, 6.3 with one).
    p.split = 1;
    while (p.split < heads && 2 * p.split * p.lanes <= ROT_THREADS && p.tokens * p.split * p.lanes < (int64_t)sms * 256) p.split *= 2;
    p.per_block = ROT_THREADS / (p.lanes * p.split);
    const int64_t blocks = (p.tokens + p.per_block - 1) / p.per_block;
    const bool split = p.split > 1;
    void (*kern)(const RotParams) = interleaved ? (split ? rotary_kernel<F32, BYTES, true, true> : rotary_kernel<F32, BYTES, true, false>)
                                                : (split ? rotary_kernel<F32, BYTES, false, true> : rotary_kernel<F32, BYTES, false, false>);
    return check_cuda(launch_pdl(kern, dim3((unsigned)blocks), dim3(p.lanes * p.split * p.per_block),
                                 split ? (size_t)p.per_block * (p.rot / 2) * sizeof(float2) : 0, s, p),
                      "rotary launch");
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
    const int eb = f32 ? 4 : 2;
    RotParams p{};
    RotSpan srcs[ROT_MAX_SEGS], dsts[ROT_MAX_SEGS];
    // every address that a thread forms is a sum of these: their common power of two is how much it may move at once
    uint64_t bits = 16 | (uint64_t)d * eb | (uint64_t)(interleaved ? rot : rot / 2) * eb;
    for (int g = 0; g < n_seg; ++g) {
        const int64_t* st = strides6 + 6 * g;
        if (!src[g] || !dst[g]) return fail(QUARTET_E_NULL, "segment %d has a NULL pointer", g);
        if (heads[g] < 1 || heads[g] > 65536) return fail(QUARTET_E_SHAPE, "segment %d: need 1 <= heads <= 65536", g);
        if ((reinterpret_cast<uintptr_t>(src[g]) | reinterpret_cast<uintptr_t>(dst[g])) & (uintptr_t)(eb - 1))
            return fail(QUARTET_E_ALIGN, "segment %d is not aligned to its type", g);
        bits |= reinterpret_cast<uintptr_t>(src[g]) | reinterpret_cast<uintptr_t>(dst[g]);
        for (int k = 0; k < 6; ++k) bits |= (uint64_t)st[k] * (uint64_t)eb;
        srcs[g] = rot_span(src[g], eb, batch, tokens, heads[g], d, st), dsts[g] = rot_span(dst[g], eb, batch, tokens, heads[g], d, st + 3);
        p.seg[g] = RotSeg{src[g], dst[g], st[0], st[1], st[2], st[3], st[4], st[5], heads[g], rotate[g] != 0};
    }
    int rc = refuse_rotary_overlap(n_seg, srcs, dsts);
    if (rc) return rc;
    if (reinterpret_cast<uintptr_t>(inv_freq) & 7u) return fail(QUARTET_E_ALIGN, "inv_freq must be 8-byte aligned");
    if (pos && (reinterpret_cast<uintptr_t>(pos) & (pos_i64 ? 7u : 3u))) return fail(QUARTET_E_ALIGN, "pos must be aligned to its type");
    if ((rc = bind_context_of(src[0]))) return rc;
    if ((rc = check_device())) return rc;
    p.n_seg = n_seg, p.d = (int)d, p.rot = (int)rot, p.T = tokens;
    p.pos = pos, p.pos_i64 = pos_i64, p.pos_b = pos_stride_b, p.pos_t = pos_stride_t, p.offset = offset;
    p.inv_freq = inv_freq, p.scale = scale, p.inverse = inverse != 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.tokens = batch * tokens;
    const int bytes = (int)(bits & (~bits + 1));
    const bool inter = interleaved != 0;
    if (f32) return bytes == 16 ? launch_rotary<true, 16>(p, inter, s) : bytes == 8 ? launch_rotary<true, 8>(p, inter, s) : launch_rotary<true, 4>(p, inter, s);
    if (bytes >= 8) return bytes == 16 ? launch_rotary<false, 16>(p, inter, s) : launch_rotary<false, 8>(p, inter, s);
    return bytes == 4 ? launch_rotary<false, 4>(p, inter, s) : launch_rotary<false, 2>(p, inter, s);
}
