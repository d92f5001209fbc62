// The 8-bit linear layer's forward / backward as ONE host call each, like the 4-bit layer's: the kernels of the single entry points in the same
// order.  A caller in Python pays some 50 us for the forward's three calls and their nine tensors, a third of that for one.
//
//   forward   Q(x) [, Qt(x)], Q(w) [, Q(w)^T], y = Q(x) Q(w)^T
//   backward  Q(e) and / or Qt(e), dx = Q(e) Q(w), dw = Qt(e)^T Qt(x); the two products in one launch where that is quicker
#include "common.cuh"
#include "gemm_fp8.cuh"

using namespace quartet;

namespace {
inline int64_t pad128(int64_t n) { return (n + 127) / 128 * 128; }
inline int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

// Byte offsets of codes and scales in the buffers: what the forward keeps (transposes of x and w), its workspace (their rows), and the
// backward's workspace (both orientations of e).
struct Fp8Layout {
    int64_t xt, xts, wt, wts, saved;
    int64_t x, xs, w, ws, fwd;
    int64_t e, es, et, ets, bwd;
};
Fp8Layout layout_fp8(int64_t M, int64_t N, int64_t K, bool dx, bool dw) {
    Fp8Layout L{};
    auto pair = [](int64_t rows, int64_t cols, int64_t& codes, int64_t& sf, int64_t& end) {
        codes = end, sf = end + pad256(rows * pad128(cols));
        end = sf + pad256(quartet_sf_bytes(rows, pad128(cols)));
    };
    if (dw) pair(K, M, L.xt, L.xts, L.saved);
    if (dx) pair(K, N, L.wt, L.wts, L.saved);
    pair(M, K, L.x, L.xs, L.fwd);
    pair(N, K, L.w, L.ws, L.fwd);
    if (dx) pair(M, N, L.e, L.es, L.bwd);
    if (dw) pair(N, M, L.et, L.ets, L.bwd);
    return L;
}
bool bad_extents(int64_t M, int64_t N, int64_t K) { return M < 1 || N < 1 || K < 1 || M > 8388480 || N > 8388480 || K > 8388480; }
bool bad_dtype(int t) { return t != QUARTET_BF16 && t != QUARTET_F32; }
bool bad_pitch(int64_t ld, int64_t n, int dtype) { return ld < n || ld % (dtype == QUARTET_F32 ? 4 : 8) != 0; }
bool bad_align(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == QUARTET_F32 ? 3u : 1u)) != 0; }
}  // namespace

extern "C" __attribute__((visibility("default"))) int quartet_linear_fp8_train_bytes(int64_t M, int64_t N, int64_t K, int need_dx, int need_dw,
                                                                                     int64_t* bytes3) {
    if (!bytes3) return fail(QUARTET_E_NULL, "bytes3 must be non-NULL");
    if (bad_extents(M, N, K)) return fail(QUARTET_E_SHAPE, "need 1 <= M, N, K <= 8388480 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    const Fp8Layout L = layout_fp8(M, N, K, need_dx != 0, need_dw != 0);
    bytes3[0] = L.saved, bytes3[1] = L.fwd, bytes3[2] = L.bwd;
    return QUARTET_OK;
}

extern "C" __attribute__((visibility("default"))) int quartet_linear_fp8_train_fwd(const void* x, int x_dtype, const void* w, int w_dtype, int64_t M, int64_t N,
                                                                                   int64_t K, int need_dx, int need_dw, uint8_t* saved, uint8_t* workspace,
                                                                                   void* y, int y_dtype, int64_t ldy, quartet_stream_t stream) {
    // everything is checked before the first step is launched
    if (!x || !w || !workspace || !y || ((need_dx || need_dw) && !saved)) return fail(QUARTET_E_NULL, "x, w, workspace, y and (for a backward) saved must be non-NULL");
    if (bad_extents(M, N, K)) return fail(QUARTET_E_SHAPE, "need 1 <= M, N, K <= 8388480 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    if (bad_dtype(x_dtype) || bad_dtype(w_dtype) || bad_dtype(y_dtype)) return fail(QUARTET_E_ARG, "dtypes must be 0 (bf16) or 1 (f32)");
    if (bad_pitch(ldy, N, y_dtype)) return fail(QUARTET_E_SHAPE, "rows of y must start on 16-byte boundaries and hold N results");
    if (bad_align(x, x_dtype) || bad_align(w, w_dtype) || !aligned16(y) || !aligned16(saved) || !aligned16(workspace))
        return fail(QUARTET_E_ALIGN, "x and w must be aligned to their types, the other buffers to 16 bytes");
    const Fp8Layout L = layout_fp8(M, N, K, need_dx != 0, need_dw != 0);
    uint8_t *xt = need_dw ? saved + L.xt : nullptr, *xts = need_dw ? saved + L.xts : nullptr;
    uint8_t *wt = need_dx ? saved + L.wt : nullptr, *wts = need_dx ? saved + L.wts : nullptr;
    int rc = quartet_quant_fp8(x, x_dtype, M, K, QUARTET_E4M3, 0, workspace + L.x, workspace + L.xs, xt, xts, stream);
    if (rc) return rc;
    if ((rc = quartet_quant_fp8(w, w_dtype, N, K, QUARTET_E4M3, 1, workspace + L.w, workspace + L.ws, wt, wts, stream))) return rc;
    return quartet_gemm_fp8_tn(workspace + L.x, workspace + L.xs, QUARTET_E4M3, workspace + L.w, workspace + L.ws, QUARTET_E4M3, M, N, pad128(K), 1.0f, y, y_dtype,
                               ldy, stream);
}

extern "C" __attribute__((visibility("default"))) int quartet_linear_fp8_train_bwd(const void* e, int e_dtype, int64_t M, int64_t N, int64_t K, int fmt,
                                                                                   const uint8_t* saved, uint8_t* workspace, void* dx, int dx_dtype, int64_t ldx,
                                                                                   void* dw, int dw_dtype, int64_t ldw, int saved_dx, int saved_dw,
                                                                                   quartet_stream_t stream) {
    if (!dx && !dw) return QUARTET_OK;
    if (!e || !saved || !workspace) return fail(QUARTET_E_NULL, "e, saved and workspace must be non-NULL");
    if ((dx && !saved_dx) || (dw && !saved_dw)) return fail(QUARTET_E_ARG, "the forward did not keep what this gradient needs");
    if (bad_extents(M, N, K)) return fail(QUARTET_E_SHAPE, "need 1 <= M, N, K <= 8388480 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    if (bad_dtype(e_dtype) || (dx && bad_dtype(dx_dtype)) || (dw && bad_dtype(dw_dtype))) return fail(QUARTET_E_ARG, "dtypes must be 0 (bf16) or 1 (f32)");
    if (fmt != QUARTET_E4M3 && fmt != QUARTET_E5M2) return fail(QUARTET_E_ARG, "fmt must be 0 (e4m3) or 1 (e5m2)");
    if ((dx && bad_pitch(ldx, K, dx_dtype)) || (dw && bad_pitch(ldw, K, dw_dtype)))
        return fail(QUARTET_E_SHAPE, "rows of dx and dw must start on 16-byte boundaries and hold K results");
    if (bad_align(e, e_dtype) || !aligned16(saved) || !aligned16(workspace) || !aligned16(dx) || !aligned16(dw))
        return fail(QUARTET_E_ALIGN, "e must be aligned to its type, the other buffers to 16 bytes");
    const Fp8Layout S = layout_fp8(M, N, K, saved_dx != 0, saved_dw != 0), L = layout_fp8(M, N, K, dx != nullptr, dw != nullptr);
    uint8_t *ec = dx ? workspace + L.e : nullptr, *es = dx ? workspace + L.es : nullptr;
    uint8_t *et = dw ? workspace + L.et : nullptr, *ets = dw ? workspace + L.ets : nullptr;
    int rc = quartet_quant_fp8(e, e_dtype, M, N, fmt, 0, ec, es, et, ets, stream);
    if (rc) return rc;
    if (dx && dw) {
        // neither depends on the other (everything that the single entry checks has been checked above)
        if ((rc = bind_context_of(saved)) || (rc = check_device())) return rc;
        Fp8Product x{ec, saved + S.wt, {}}, y{et, saved + S.xt, {}};
        x.g.a_sf = es, x.g.b_sf = saved + S.wts, x.g.M = M, x.g.N = K, x.g.ldd = ldx, x.g.k_chunks = (int)(pad128(N) / 128);
        x.g.d = dx, x.g.d_f32 = dx_dtype == QUARTET_F32;
        y.g.a_sf = ets, y.g.b_sf = saved + S.xts, y.g.M = N, y.g.N = K, y.g.ldd = ldw, y.g.k_chunks = (int)(pad128(M) / 128);
        y.g.d = dw, y.g.d_f32 = dw_dtype == QUARTET_F32;
        x.g.a_e5m2 = y.g.a_e5m2 = fmt, x.g.alpha = y.g.alpha = 1.0f;
        return product_two(x, y, static_cast<cudaStream_t>(stream));
    }
    if (dx) return quartet_gemm_fp8_tn(ec, es, fmt, saved + S.wt, saved + S.wts, QUARTET_E4M3, M, K, pad128(N), 1.0f, dx, dx_dtype, ldx, stream);
    return quartet_gemm_fp8_tn(et, ets, fmt, saved + S.xt, saved + S.xts, QUARTET_E4M3, N, K, pad128(M), 1.0f, dw, dw_dtype, ldw, stream);
}
