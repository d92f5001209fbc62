"""Tensor-level wrappers over the C ABI.  torch supplies device memory and the
current stream; all arithmetic happens in libquartet_b200.so."""
from __future__ import annotations

import ctypes as C
import functools
import os
from array import array

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib

BF16, F32 = 0, 1
ROUND_NEAREST, ROUND_SR_PHILOX, ROUND_SR_NOISE, ROUND_SR_TLRAND = 0, 1, 2, 3
QUEST_GAUSSIAN_SCALE = 2.92247856 / 6.0
HAD_SCALE_BF16 = 0.1767578125  # bf16(32 ** -0.5)
HAD_SCALE_F32 = 0.17677669529663687
_LIST_DT = {torch.bfloat16: BF16, torch.float32: F32}
SR_OPERAND_SCALE = 4.0 / 3.0  # each absmax-quantized operand carries this factor outside its scale bytes


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return BF16
    if t.dtype == torch.float32:
        return F32
    raise ValueError(f"dtype {t.dtype} not supported (bf16 or fp32)")


def _out_dt(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return BF16
    if dtype == torch.float32:
        return F32
    raise ValueError(f"output dtype {dtype} not supported (bf16 or fp32)")


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    # the current device's stream as an address: building a torch.cuda.Stream object costs 3 us a call, this 0.1
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


class _NoSwitch:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_NO_SWITCH = _NoSwitch()


def _on(device):
    """Context that makes `device` current for the call; free when it already is (the one-process-per-GPU case)."""
    idx = device.index
    if idx is None or idx == torch.cuda.current_device():
        return _NO_SWITCH
    return torch.cuda.device(device)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("tensors must live on a CUDA device")
        if t is not None and not t.is_contiguous():
            raise ValueError("tensors must be contiguous")


def forward_mode() -> bool:
    """Whether a level of forward-mode differentiation is open.  Its inputs have no requires_grad: a call that reads their memory itself has to
    ask for them here, or their tangents are lost without a word."""
    return getattr(_forward_ad, "_current_level", 0) >= 0


def recording() -> bool:
    """Whether the call is being put into a graph (compiled, exported, traced), where only registered operators are seen."""
    return (torch.compiler.is_compiling() or torch.jit.is_tracing()) and not forward_mode()


def eagerly(fn, *args):
    """fn(*args), outside the graph where one is being compiled: a compiler calls an autograd function's forward without its forward-mode derivative."""
    return torch.compiler.disable(fn)(*args) if torch.compiler.is_compiling() else fn(*args)


def has_tangent(*ts) -> bool:
    return forward_mode() and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in ts)


def sf_bytes(rows: int, cols: int) -> int:
    return ((rows + 127) // 128 * 128) * ((cols // 32 + 3) // 4 * 4)


def quant_fwd(x, had_scale=HAD_SCALE_BF16, gaussian_scale=QUEST_GAUSSIAN_SCALE, return_mask=True):
    """[rows, cols] -> (codes [rows, cols/2] u8, sf blocked u8, mask [rows, cols/8] u8 | None)."""
    _need_cuda(x)
    rows, cols = x.shape
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=x.device)
    sf = torch.empty(sf_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    mask = torch.empty(rows, cols // 8, dtype=torch.uint8, device=x.device) if return_mask else None
    with _on(x.device):
        rc = _lib.load().quartet_quant_fwd(_ptr(x), _dt(x), rows, cols, had_scale, gaussian_scale, _ptr(codes), _ptr(sf),
                                           _ptr(mask), _stream())
    _lib.check(rc, "quartet_quant_fwd")
    return codes, sf, mask


def rms_stats(x, eps):
    """rsqrt(mean(x^2, -1) + eps) per row of [rows, cols] (bf16 / fp32) -> fp32 [rows]."""
    _need_cuda(x)
    rows, cols = x.shape
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    with _on(x.device):
        rc = _lib.load().quartet_rms_stats(_ptr(x), _dt(x), rows, cols, float(eps), _ptr(rstd), _stream())
    _lib.check(rc, "quartet_rms_stats")
    return rstd


def quant_fwd_rmsnorm(x, weight, eps, had_scale=HAD_SCALE_BF16, gaussian_scale=QUEST_GAUSSIAN_SCALE, return_mask=True):
    """Forward quantizer of RMSNorm(x) = (x * rstd).type_as(x) * weight without materialising it:
    [rows, cols], fp32 weight [cols] -> (codes, sf blocked, mask | None, rstd fp32 [rows])."""
    _need_cuda(x, weight)
    rows, cols = x.shape
    if weight.dtype != torch.float32 or weight.shape != (cols,) or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous fp32 vector with one entry per column")
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=x.device)
    sf = torch.empty(sf_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    mask = torch.empty(rows, cols // 8, dtype=torch.uint8, device=x.device) if return_mask else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    with _on(x.device):
        rc = _lib.load().quartet_quant_fwd_rmsnorm(_ptr(x), _dt(x), rows, cols, _ptr(weight), float(eps), _ptr(rstd), had_scale, gaussian_scale,
                                                   _ptr(codes), _ptr(sf), _ptr(mask), _stream())
    _lib.check(rc, "quartet_quant_fwd_rmsnorm")
    return codes, sf, mask, rstd


def quant_fwd_swiglu(h, had_scale=HAD_SCALE_BF16, gaussian_scale=QUEST_GAUSSIAN_SCALE, return_mask=True):
    """Forward quantizer of silu(h[:, :H]) * h[:, H:] without materialising it: [rows, 2H] -> (codes [rows, H/2], sf, mask | None)."""
    _need_cuda(h)
    rows, two_h = h.shape
    if two_h % 2:
        raise ValueError("h must hold the up and gate halves side by side")
    hidden = two_h // 2
    codes = torch.empty(rows, hidden // 2, dtype=torch.uint8, device=h.device)
    sf = torch.empty(sf_bytes(rows, hidden), dtype=torch.uint8, device=h.device)
    mask = torch.empty(rows, hidden // 8, dtype=torch.uint8, device=h.device) if return_mask else None
    with _on(h.device):
        rc = _lib.load().quartet_quant_fwd_swiglu(_ptr(h), _dt(h), rows, hidden, had_scale, gaussian_scale, _ptr(codes), _ptr(sf), _ptr(mask),
                                                  _stream())
    _lib.check(rc, "quartet_quant_fwd_swiglu")
    return codes, sf, mask


def swiglu(h):
    """silu(h[:, :H]) * h[:, H:] written out, [rows, 2H] -> [rows, H] in h's dtype: the values quant_fwd_swiglu quantizes."""
    _need_cuda(h)
    rows, two_h = h.shape
    if two_h % 2:
        raise ValueError("h must hold the up and gate halves side by side")
    out = torch.empty(rows, two_h // 2, dtype=h.dtype, device=h.device)
    with _on(h.device):
        rc = _lib.load().quartet_swiglu(_ptr(h), _dt(h), rows, two_h // 2, _ptr(out), _stream())
    _lib.check(rc, "quartet_swiglu")
    return out


def _sr_args(signs, signs_dev, seed, offset, noise):
    return (int(signs) & 0xFFFFFFFF, _ptr(signs_dev)), (int(seed) & (2**64 - 1), int(offset) & (2**64 - 1), _ptr(noise))


def quant_bwd(x, had_scale=HAD_SCALE_BF16, signs=0, signs_dev=None, rounding=ROUND_SR_PHILOX, seed=0, offset=0, noise=None):
    """Row-wise backward quantizer: (codes [rows, cols/2], sf blocked); value = grid * 2^(sf-127) * 4/3."""
    _need_cuda(x, noise, signs_dev)
    rows, cols = x.shape
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=x.device)
    sf = torch.empty(sf_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    (s, sd), (sd_, off, nz) = _sr_args(signs, signs_dev, seed, offset, noise)
    with _on(x.device):
        rc = _lib.load().quartet_quant_bwd(_ptr(x), _dt(x), rows, cols, had_scale, s, sd, rounding, sd_, off, nz, _ptr(codes),
                                           _ptr(sf), _stream())
    _lib.check(rc, "quartet_quant_bwd")
    return codes, sf


def quant_group32(x, kind, gaussian_scale=QUEST_GAUSSIAN_SCALE, rounding=ROUND_NEAREST, seed=0, offset=0, noise=None, return_mask=True):
    """Scaling + rounding + packing of an already rotated (or un-rotated) [rows, cols] tensor, groups of 32 along cols.
    kind 0: std-scaled round-to-nearest with clip mask -> (codes, sf, mask | None); kind 1: absmax-scaled -> (codes, sf, None)."""
    _need_cuda(x, noise)
    rows, cols = x.shape
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=x.device)
    sf = torch.empty(sf_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    mask = torch.empty(rows, cols // 8, dtype=torch.uint8, device=x.device) if (kind == 0 and return_mask) else None
    m64 = 2**64 - 1
    with _on(x.device):
        rc = _lib.load().quartet_quant_group32(_ptr(x), _dt(x), rows, cols, kind, gaussian_scale, rounding, int(seed) & m64, int(offset) & m64,
                                               _ptr(noise), _ptr(codes), _ptr(sf), _ptr(mask), _stream())
    _lib.check(rc, "quartet_quant_group32")
    return codes, sf, mask


def quant_bwd_t(x, had_scale=HAD_SCALE_BF16, signs=0, signs_dev=None, rounding=ROUND_SR_PHILOX, seed=0, offset=0, noise=None):
    """Backward quantizer of x^T: (codes_t [cols, rows/2], sf_t blocked for [cols, rows/32])."""
    _need_cuda(x, noise, signs_dev)
    rows, cols = x.shape
    codes_t = torch.empty(cols, rows // 2, dtype=torch.uint8, device=x.device)
    sf_t = torch.empty(sf_bytes(cols, rows), dtype=torch.uint8, device=x.device)
    (s, sd), (sd_, off, nz) = _sr_args(signs, signs_dev, seed, offset, noise)
    with _on(x.device):
        rc = _lib.load().quartet_quant_bwd_t(_ptr(x), _dt(x), rows, cols, had_scale, s, sd, rounding, sd_, off, nz,
                                             _ptr(codes_t), _ptr(sf_t), _stream())
    _lib.check(rc, "quartet_quant_bwd_t")
    return codes_t, sf_t


def quant_bwd_dual(x, had_scale=HAD_SCALE_BF16, signs=0, signs_dev=None, rounding=ROUND_SR_PHILOX, seed_rows=0, seed_t=0, offset=0):
    """`quant_bwd(x, seed=seed_rows)` and `quant_bwd_t(x, seed=seed_t)` from one read of x:
    (codes, sf, codes_t, sf_t), bit-identical to the two separate calls."""
    _need_cuda(x, signs_dev)
    rows, cols = x.shape
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=x.device)
    sf = torch.empty(sf_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    codes_t = torch.empty(cols, rows // 2, dtype=torch.uint8, device=x.device)
    sf_t = torch.empty(sf_bytes(cols, rows), dtype=torch.uint8, device=x.device)
    m64 = 2**64 - 1
    with _on(x.device):
        rc = _lib.load().quartet_quant_bwd_dual(_ptr(x), _dt(x), rows, cols, had_scale, int(signs) & 0xFFFFFFFF, _ptr(signs_dev), rounding,
                                                int(seed_rows) & m64, int(seed_t) & m64, int(offset) & m64, _ptr(codes), _ptr(sf),
                                                _ptr(codes_t), _ptr(sf_t), _stream())
    _lib.check(rc, "quartet_quant_bwd_dual")
    return codes, sf, codes_t, sf_t


def requant_t(codes, sf, in_scale=1.0, had_scale=HAD_SCALE_BF16, signs=0, signs_dev=None, rounding=ROUND_SR_PHILOX, seed=0,
              offset=0, noise=None):
    """MXFP4 [rows, cols] -> backward-quantized transpose (codes_t [cols, rows/2], sf_t)."""
    _need_cuda(codes, sf, noise, signs_dev)
    rows, cols = codes.shape[0], codes.shape[1] * 2
    codes_t = torch.empty(cols, rows // 2, dtype=torch.uint8, device=codes.device)
    sf_t = torch.empty(sf_bytes(cols, rows), dtype=torch.uint8, device=codes.device)
    (s, sd), (sd_, off, nz) = _sr_args(signs, signs_dev, seed, offset, noise)
    with _on(codes.device):
        rc = _lib.load().quartet_requant_t(_ptr(codes), _ptr(sf), rows, cols, in_scale, had_scale, s, sd, rounding, sd_, off,
                                           nz, _ptr(codes_t), _ptr(sf_t), _stream())
    _lib.check(rc, "quartet_requant_t")
    return codes_t, sf_t


def gemm_mxfp4_tn(a, a_sf, b, b_sf, alpha=1.0, mask=None, had_scale=HAD_SCALE_BF16, out_dtype=torch.bfloat16, out=None):
    """D[M,N] = alpha * A[M,K] . B[N,K]^T on packed e2m1 operands with blocked E8M0 scales."""
    _need_cuda(a, a_sf, b, b_sf, mask, out)
    M, K = a.shape[0], a.shape[1] * 2
    N = b.shape[0]
    if b.shape[1] * 2 != K:
        raise ValueError(f"contraction extents differ: {K} vs {b.shape[1] * 2}")
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    with _on(a.device):
        rc = _lib.load().quartet_gemm_mxfp4_tn(_ptr(a), _ptr(a_sf), _ptr(b), _ptr(b_sf), M, N, K, alpha, _ptr(mask), had_scale,
                                               _ptr(out), _out_dt(out.dtype), _stream())
    _lib.check(rc, "quartet_gemm_mxfp4_tn")
    return out


# One host call per direction for the whole layer (quartet_linear_fwd / quartet_linear_bwd): the same kernels as the
# single entry points.  FUSED_LAYER_CALLS = False makes the layer code call the entry points one by one instead
# (what the benchmark's per-kernel timing pass does).
FUSED_LAYER_CALLS = True


def linear_fwd(x2, w, had_scale_x, had_scale_w, out_dtype, gaussian_scale=QUEST_GAUSSIAN_SCALE):
    """x2 [M, K] (M a multiple of 128), w [N, K] -> (y [M, N], xc, xs, xm, wc, ws, wm)."""
    _need_cuda(x2, w)
    M, K = x2.shape
    N = w.shape[0]
    dev = x2.device
    u8 = torch.uint8
    xc, xs, xm = torch.empty(M, K // 2, dtype=u8, device=dev), torch.empty(sf_bytes(M, K), dtype=u8, device=dev), torch.empty(M, K // 8, dtype=u8, device=dev)
    wc, ws, wm = torch.empty(N, K // 2, dtype=u8, device=dev), torch.empty(sf_bytes(N, K), dtype=u8, device=dev), torch.empty(N, K // 8, dtype=u8, device=dev)
    y = torch.empty(M, N, dtype=out_dtype, device=dev)
    with _on(dev):
        rc = _lib.load().quartet_linear_fwd(_ptr(x2), _dt(x2), _ptr(w), _dt(w), M, N, K, had_scale_x, had_scale_w, gaussian_scale, _ptr(xc), _ptr(xs),
                                            _ptr(xm), _ptr(wc), _ptr(ws), _ptr(wm), _ptr(y), _out_dt(out_dtype), _stream())
    _lib.check(rc, "quartet_linear_fwd")
    return y, xc, xs, xm, wc, ws, wm


def linear_bwd(e2, xc, xs, xm, wc, ws, wm, had_scale_b, rounding, seeds, alpha, had_scale_x, had_scale_w, x_dtype, w_dtype, need_dx=True,
               need_dw=True, signs=0, signs_dev=None, offset=0):
    """e2 [M, N] (M a multiple of 128) and the packed outputs of linear_fwd -> (dx [M, K] | None, dw [N, K] | None)."""
    _need_cuda(e2, xc, xs, xm, wc, ws, wm, signs_dev)
    M, N = e2.shape
    K = wc.shape[1] * 2
    dev = e2.device
    lib = _lib.load()
    work = torch.empty(lib.quartet_linear_bwd_workspace_bytes(M, N, K), dtype=torch.uint8, device=dev)
    dx = torch.empty(M, K, dtype=x_dtype, device=dev) if need_dx else None
    dw = torch.empty(N, K, dtype=w_dtype, device=dev) if need_dw else None
    m64 = 2**64 - 1
    seeds4 = (C.c_uint64 * 4)(*[int(v) & m64 for v in seeds])
    with _on(dev):
        rc = lib.quartet_linear_bwd(_ptr(e2), _dt(e2), M, N, K, _ptr(xc), _ptr(xs), _ptr(xm), _ptr(wc), _ptr(ws), _ptr(wm), had_scale_b,
                                    int(signs) & 0xFFFFFFFF, _ptr(signs_dev), rounding, seeds4, int(offset) & m64, alpha, had_scale_x, had_scale_w,
                                    _ptr(work), _ptr(dx), _out_dt(x_dtype), _ptr(dw), _out_dt(w_dtype), _stream())
    _lib.check(rc, "quartet_linear_bwd")
    return dx, dw


def gemm_mxfp4_tn_scatter(a, a_sf, b, b_sf, owner_ptrs, rows_per_owner, alpha=1.0, mask=None, had_scale=HAD_SCALE_BF16):
    """The fp32 product of `gemm_mxfp4_tn` with rows [o*rows_per_owner, (o+1)*rows_per_owner) stored to the
    device address owner_ptrs[o] (a dense [rows_per_owner, N] matrix, possibly in another GPU's memory)."""
    _need_cuda(a, a_sf, b, b_sf, mask)
    M, K = a.shape[0], a.shape[1] * 2
    N = b.shape[0]
    if b.shape[1] * 2 != K:
        raise ValueError(f"contraction extents differ: {K} vs {b.shape[1] * 2}")
    arr = (C.c_void_p * len(owner_ptrs))(*[int(x) for x in owner_ptrs])
    with _on(a.device):
        rc = _lib.load().quartet_gemm_mxfp4_tn_scatter(_ptr(a), _ptr(a_sf), _ptr(b), _ptr(b_sf), M, N, K, alpha, _ptr(mask), had_scale,
                                                       C.cast(arr, C.c_void_p), len(owner_ptrs), rows_per_owner, _stream())
    _lib.check(rc, "quartet_gemm_mxfp4_tn_scatter")


def shard_reduce(slots_ptr, n_slots, slot_elems, scale, out):
    """out[i] = scale * sum_s slots[s*slot_elems + i]; `slots_ptr` is a device address, `out` an fp32 tensor."""
    _need_cuda(out)
    if out.dtype != torch.float32 or not out.is_contiguous() or out.numel() != slot_elems:
        raise ValueError("out must be a contiguous fp32 tensor of slot_elems elements")
    with _on(out.device):
        rc = _lib.load().quartet_shard_reduce(int(slots_ptr), n_slots, slot_elems, scale, _ptr(out), _stream())
    _lib.check(rc, "quartet_shard_reduce")
    return out


def peer_alloc(nbytes, device):
    """(device address, 64-byte handle) of a buffer other processes of the node can map."""
    ptr, handle = C.c_void_p(), C.create_string_buffer(64)
    with torch.cuda.device(device):
        rc = _lib.load().quartet_peer_alloc(nbytes, C.byref(ptr), C.cast(handle, C.c_void_p))
    _lib.check(rc, "quartet_peer_alloc")
    return ptr.value, handle.raw


def peer_open(handle, device):
    ptr, buf = C.c_void_p(), C.create_string_buffer(bytes(handle), 64)
    with torch.cuda.device(device):
        rc = _lib.load().quartet_peer_open(C.cast(buf, C.c_void_p), C.byref(ptr))
    _lib.check(rc, "quartet_peer_open")
    return ptr.value


def peer_close(ptr, device):
    with torch.cuda.device(device):
        _lib.check(_lib.load().quartet_peer_close(int(ptr)), "quartet_peer_close")


def peer_copy(dst_ptr, src_ptr, nbytes, device):
    """Asynchronous copy between device addresses on the current stream (DMA engines, no SM)."""
    with torch.cuda.device(device):
        _lib.check(_lib.load().quartet_peer_copy(int(dst_ptr), int(src_ptr), nbytes, _stream()), "quartet_peer_copy")


def peer_free(ptr, device):
    with torch.cuda.device(device):
        _lib.check(_lib.load().quartet_peer_free(int(ptr)), "quartet_peer_free")


def probe_copy_ingress(region_mb=48, iters=4000, stages=6, chunk=16384, producers=2, device="cuda"):
    """Bytes per clock one SM takes in through bulk asynchronous copies (see csrc/probe_ingress.cu)."""
    src = torch.ones(region_mb << 20, dtype=torch.uint8, device=device)
    cycles = torch.zeros(1024, dtype=torch.int64, device=device)
    out = C.c_double(0.0)
    with torch.cuda.device(src.device):
        rc = _lib.load().quartet_probe_copy_ingress(_ptr(src), src.numel(), iters, stages, chunk, producers, _ptr(cycles), C.byref(out), _stream())
    _lib.check(rc, "quartet_probe_copy_ingress")
    return out.value


def probe_copy_ingress_noalloc(src, iters=4000, stages=6, chunk=16384, producers=2):
    """`probe_copy_ingress` on a caller-provided uint8 device tensor; neither this wrapper nor the library allocates."""
    _need_cuda(src)
    out = C.c_double(0.0)
    with torch.cuda.device(src.device):
        rc = _lib.load().quartet_probe_copy_ingress_noalloc(_ptr(src), src.numel() * src.element_size(), iters, stages, chunk, producers,
                                                            C.byref(out), _stream())
    _lib.check(rc, "quartet_probe_copy_ingress_noalloc")
    return out.value


def fold_signs(draw, word):
    """word (int64[1] or int32[1] device tensor, low 32 bits used) ^= bits j where draw[j] == 0; draw = the 32 zeros / ones
    of the reference's torch.randint(0, 2, (32,)) call (mxfp4.py:52-60), bf16 or fp32."""
    _need_cuda(draw, word)
    if draw.numel() != 32:
        raise ValueError("draw must hold 32 values")
    with _on(word.device):
        rc = _lib.load().quartet_fold_signs(_ptr(draw), _dt(draw), _ptr(word), _stream())
    _lib.check(rc, "quartet_fold_signs")
    return word


def unrotate_mask(g, mask=None, had_scale=HAD_SCALE_BF16, out_dtype=None):
    """((g * mask).view(-1, 32) @ H^T).view_as(g)"""
    _need_cuda(g, mask)
    out = torch.empty_like(g, dtype=out_dtype or g.dtype)
    cols = g.shape[-1]
    rows = g.numel() // cols
    with _on(g.device):
        rc = _lib.load().quartet_unrotate_mask(_ptr(g), _dt(g), _ptr(mask), rows, cols, had_scale, _ptr(out), _out_dt(out.dtype),
                                               _stream())
    _lib.check(rc, "quartet_unrotate_mask")
    return out


def dequant(codes, sf, scale=1.0, dtype=torch.float32):
    """codes [rows, cols/2] + blocked sf -> [rows, cols] values grid * 2^(sf-127) * scale."""
    _need_cuda(codes, sf)
    rows, cols = codes.shape[0], codes.shape[1] * 2
    out = torch.empty(rows, cols, dtype=dtype, device=codes.device)
    with _on(codes.device):
        rc = _lib.load().quartet_dequant(_ptr(codes), _ptr(sf), rows, cols, scale, _ptr(out), _out_dt(dtype), _stream())
    _lib.check(rc, "quartet_dequant")
    return out


# ------------------------------------------------------------------------------------------------
# 8-bit block-scaled linear layer
# ------------------------------------------------------------------------------------------------
E4M3, E5M2 = 0, 1
_F8 = {torch.float8_e4m3fn: E4M3, torch.float8_e5m2: E5M2}


def _f8(dtype) -> int:
    if dtype not in _F8:
        raise ValueError(f"8-bit dtype {dtype} not supported (float8_e4m3fn or float8_e5m2)")
    return _F8[dtype]


def _pad128(n: int) -> int:
    return (n + 127) // 128 * 128


def quant_fp8(x, dtype=torch.float8_e4m3fn, square=False, rows=True, transpose=False):
    """[R, C] (bf16 / fp32) -> (codes [R, pad128(C)], sf blocked u8, codes_t [C, pad128(R)], sf_t): 8-bit values with a power-of-two scale
    for each block of 128 along the contraction, 1 x 128 or (square) 128 x 128.  `rows` / `transpose` choose the orientations; the
    other pair is None."""
    _need_cuda(x)
    if x.dim() != 2:
        raise ValueError("x must have two dimensions")
    if not (rows or transpose):
        raise ValueError("nothing to quantize: rows and transpose are both False")
    fmt, (R, K), dev = _f8(dtype), x.shape, x.device
    codes = sf = codes_t = sf_t = None
    if rows:
        codes = torch.empty(R, _pad128(K), dtype=dtype, device=dev)
        sf = torch.empty(sf_bytes(R, _pad128(K)), dtype=torch.uint8, device=dev)
    if transpose:
        codes_t = torch.empty(K, _pad128(R), dtype=dtype, device=dev)
        sf_t = torch.empty(sf_bytes(K, _pad128(R)), dtype=torch.uint8, device=dev)
    xdt = _dt(x)
    if R and K:
        with _on(dev):
            rc = _lib.load().quartet_quant_fp8(_ptr(x), xdt, R, K, fmt, int(bool(square)), _ptr(codes), _ptr(sf), _ptr(codes_t), _ptr(sf_t), _stream())
        _lib.check(rc, "quartet_quant_fp8")
    return codes, sf, codes_t, sf_t


def _need_codes(codes, sf, what):
    _need_cuda(codes, sf)
    if codes.dim() != 2 or codes.shape[1] % 128 or sf.dtype != torch.uint8 or sf.numel() != sf_bytes(codes.shape[0], codes.shape[1]):
        raise ValueError(f"{what}: codes [rows, multiple of 128] and the blocked uint8 scales that belong to them are needed")
    if sf.device != codes.device:
        raise ValueError(f"{what}: codes and scales are on different devices")


def dequant_fp8(codes, sf, cols=None, scale=1.0, dtype=torch.float32):
    """Codes of quant_fp8 and their scales -> [rows, cols] values (cols: without the padding; default all columns)."""
    _need_codes(codes, sf, "dequant_fp8")
    rows, pitch = codes.shape
    cols = pitch if cols is None else int(cols)
    if not 0 <= pitch - cols < 128:
        raise ValueError(f"{cols} columns do not belong to codes of {pitch}")
    out = torch.empty(rows, cols, dtype=dtype, device=codes.device)
    if out.numel():
        with _on(codes.device):
            rc = _lib.load().quartet_dequant_fp8(_ptr(codes), _ptr(sf), rows, cols, _f8(codes.dtype), scale, _ptr(out), _out_dt(dtype), _stream())
        _lib.check(rc, "quartet_dequant_fp8")
    return out


def _padded_out(lead, cols, dtype, dev):
    """[*lead, cols] whose rows start on 16-byte boundaries, and their pitch in elements.  No view of another tensor, even where the rows are
    padded: what an autograd function returns could not be changed in place otherwise."""
    per = 16 // dtype.itemsize
    pitch = (cols + per - 1) // per * per
    if pitch == cols:
        return torch.empty(*lead, cols, dtype=dtype, device=dev), pitch
    strides, step = [1], pitch
    for n in reversed(lead):
        strides.append(step)
        step *= max(n, 1)
    return torch.empty_strided((*lead, cols), strides[::-1], dtype=dtype, device=dev), pitch


def gemm_fp8_tn(a, a_sf, b, b_sf, alpha=1.0, out_dtype=torch.bfloat16):
    """D[M, N] = alpha * A[M, K] . B[N, K]^T on 8-bit codes with blocked E8M0 scales, as quant_fp8 makes them.  Where a row of D is no
    multiple of 16 bytes, D's rows are padded in memory so that they start on one."""
    _need_codes(a, a_sf, "gemm_fp8_tn (a)")
    _need_codes(b, b_sf, "gemm_fp8_tn (b)")
    (M, K), N = a.shape, b.shape[0]
    if b.shape[1] != K:
        raise ValueError(f"contraction extents differ: {K} vs {b.shape[1]}")
    if a.device != b.device:
        raise ValueError("operands are on different devices")
    fa, fb, dd = _f8(a.dtype), _f8(b.dtype), _out_dt(out_dtype)
    if M == 0 or N == 0 or K == 0:
        return torch.zeros(M, N, dtype=out_dtype, device=a.device)
    out, pitch = _padded_out((M,), N, out_dtype, a.device)
    with _on(a.device):
        rc = _lib.load().quartet_gemm_fp8_tn(_ptr(a), _ptr(a_sf), fa, _ptr(b), _ptr(b_sf), fb, M, N, K, alpha, _ptr(out), dd, pitch, _stream())
    _lib.check(rc, "quartet_gemm_fp8_tn")
    return out


GEMM_FP8_FORMS = ("stream", "pairs", "rows_256", "rows_128", "rows_128_two", "rows_few")


def gemm_fp8_form(M, N, K):
    """(form, ways the contraction is split) of a product of these extents (K a multiple of 128) on the current device."""
    form, splits = C.c_int32(0), C.c_int32(0)
    _lib.check(_lib.load().quartet_gemm_fp8_form(M, N, K, C.byref(form), C.byref(splits)), "quartet_gemm_fp8_form")
    return GEMM_FP8_FORMS[form.value], splits.value


def linear_fp8(x, w, w_sf, out_dtype=None):
    """x [..., K] times a packed weight (codes [N, pad128(K)] and scales of quant_fp8(weight, square=True)) -> [..., N]: x is quantized in
    blocks of 128 (e4m3) and multiplied.  The serving form of quantization.fp8_linear; not differentiable: an x that wants a gradient, or has a
    tangent, is refused (call it under torch.no_grad() or on x.detach())."""
    if (x.requires_grad and torch.is_grad_enabled()) or has_tangent(x):
        raise RuntimeError("linear_fp8 has no derivative: call it under torch.no_grad() or on x.detach(), or use quantization.fp8_linear")
    _need_codes(w, w_sf, "linear_fp8")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have at least one column")
    if (x.shape[-1] + 127) // 128 * 128 != w.shape[1]:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {w.shape[1]}")
    if x.device != w.device:
        raise ValueError("x and the weight are on different devices")
    dtype = out_dtype or x.dtype
    if recording():
        return torch.ops.quartet_b200.linear_fp8(x, w, w_sf, dtype)
    return _linear_fp8(x, w, w_sf, dtype)


def _linear_fp8(x, w, w_sf, dtype):
    shape, dev, N = x.shape, w.device, w.shape[0]
    if not x.is_contiguous():
        x = x.contiguous()
    K = shape[-1]
    M = x.numel() // K
    xd, wd, yd = _dt(x), _f8(w.dtype), _out_dt(dtype)
    y, pitch = _padded_out(shape[:-1], N, dtype, dev)
    if M and N:
        lib = _lib.load()
        nbytes = lib.quartet_linear_fp8_workspace_bytes(M, K)
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        with _on(dev):
            rc = lib.quartet_linear_fp8(x.data_ptr(), xd, M, K, w.data_ptr(), w_sf.data_ptr(), wd, N, 1.0, None if work is None else work.data_ptr(),
                                        y.data_ptr(), yd, pitch, _stream())
        if rc:
            _lib.check(rc, "quartet_linear_fp8")
    return y


@functools.lru_cache(maxsize=4096)
def _fp8_train_bytes(M, N, K, need_dx, need_dw):
    out = (C.c_int64 * 3)()
    _lib.check(_lib.load().quartet_linear_fp8_train_bytes(M, N, K, need_dx, need_dw, C.addressof(out)), "quartet_linear_fp8_train_bytes")
    return tuple(out)


def fp8_linear_fwd(x, w, need_dx, need_dw, out_dtype):
    """x [..., K], w [N, K] -> (y [..., N], saved): the 8-bit layer's forward in one call; saved is what fp8_linear_bwd takes."""
    _need_cuda(x, w)
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1] or w.device != x.device:
        raise ValueError(f"x [..., K] and w [N, K] on one device are needed, not {tuple(x.shape)} and {tuple(w.shape)}")
    (N, K), dev = w.shape, x.device
    M = x.numel() // K if K else x.shape[:-1].numel()
    xd, wd, yd = _dt(x), _dt(w), _out_dt(out_dtype)
    y, pitch = _padded_out(x.shape[:-1], N, out_dtype, dev)
    need_dx, need_dw = 1 if need_dx else 0, 1 if need_dw else 0
    if not (M and N and K):
        return y.zero_(), torch.empty(0, dtype=torch.uint8, device=dev)
    saved_bytes, work_bytes, _ = _fp8_train_bytes(M, N, K, need_dx, need_dw)
    saved, work = torch.empty(saved_bytes, dtype=torch.uint8, device=dev), torch.empty(work_bytes, dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = _lib.load().quartet_linear_fp8_train_fwd(x.data_ptr(), xd, w.data_ptr(), wd, M, N, K, need_dx, need_dw, saved.data_ptr() if saved_bytes else None,
                                                      work.data_ptr(), y.data_ptr(), yd, pitch, _stream())
    if rc:
        _lib.check(rc, "quartet_linear_fp8_train_fwd")
    return y, saved


def fp8_linear_bwd(e2, saved, K, grad_dtype, x_dtype, w_dtype, need_dx, need_dw, saved_dx, saved_dw):
    """e2 [M, N] and the forward's saved buffer (made with need_dx = saved_dx, need_dw = saved_dw) -> (dx [M, K] | None, dw [N, K] | None)."""
    _need_cuda(e2, saved)
    if e2.dim() != 2 or saved.device != e2.device:
        raise ValueError("e [M, N] and the kept buffer on one device are needed")
    (M, N), dev = e2.shape, e2.device
    ed, fmt = _dt(e2), _f8(grad_dtype)
    # the library sees an address only: the buffer's size is what tells whether it was kept for these extents
    if M and N and K and (saved.dtype != torch.uint8 or saved.numel() != _fp8_train_bytes(M, N, K, 1 if saved_dx else 0, 1 if saved_dw else 0)[0]):
        raise ValueError(f"the kept buffer does not belong to a layer of {M} x {N}, K {K}")
    dx, ldx = _padded_out((M,), K, x_dtype, dev) if need_dx else (None, 0)
    dw, ldw = _padded_out((N,), K, w_dtype, dev) if need_dw else (None, 0)
    if not (M and N and K):
        return None if dx is None else dx.zero_(), None if dw is None else dw.zero_()
    work = torch.empty(_fp8_train_bytes(M, N, K, 1 if need_dx else 0, 1 if need_dw else 0)[2], dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = _lib.load().quartet_linear_fp8_train_bwd(e2.data_ptr(), ed, M, N, K, fmt, saved.data_ptr(), work.data_ptr(), dx.data_ptr() if need_dx else None,
                                                      _out_dt(x_dtype), ldx, dw.data_ptr() if need_dw else None, _out_dt(w_dtype), ldw, 1 if saved_dx else 0,
                                                      1 if saved_dw else 0, _stream())
    if rc:
        _lib.check(rc, "quartet_linear_fp8_train_bwd")
    return dx, dw


# ------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------
def rotary(segments, inv_freq, positions=None, offset=0, interleaved=True, scale=1.0, inverse=False):
    """Turns (or copies) up to three tensors in one launch.  segments: (src, dst, rotate), src and dst [batch, tokens, heads, d] views of any
    strides whose last axis is contiguous.  positions: int32 / int64 [tokens] or [batch, tokens], or None for offset, offset + 1, ...
    inv_freq: float64 [rot / 2].  A dst may be its own src; one that shares memory with anything else, or with itself, is refused."""
    x0 = segments[0][0]
    B, T, _, d = x0.shape
    dev, dtype = x0.device, x0.dtype
    srcs, dsts, strides, heads, turns = [], [], [], [], []
    for src, dst, rotate in segments:
        shape = src.shape
        if src.device != dev or dst.device != dev:
            raise ValueError("tensors must live on one CUDA device")
        if src.dtype != dtype or dst.dtype != dtype or shape != dst.shape or len(shape) != 4 or shape[0] != B or shape[1] != T or shape[3] != d:
            raise ValueError("segments must agree in dtype, batch, tokens and d")
        a, b = src.stride(), dst.stride()
        if d > 1 and (a[3] != 1 or b[3] != 1):
            raise ValueError("the values of a head must be adjacent")
        srcs.append(src.data_ptr()), dsts.append(dst.data_ptr()), heads.append(shape[2]), turns.append(1 if rotate else 0)
        strides += [a[0], a[1], a[2], b[0], b[1], b[2]]
    rotary_raw(srcs + dsts, rotary_plan(strides, heads, turns), dev, dtype, B, T, d, inv_freq, positions, offset, interleaved, scale, inverse)


def rotary_plan(strides, heads, turns):
    """The host arrays of a launch that do not change with the tensors' addresses: element strides (batch, token, head of src and dst) of each
    segment, its heads and whether it is turned."""
    longs, ints = array("q", strides), array("i", [*heads, *turns])
    return longs, ints, longs.buffer_info()[0], ints.buffer_info()[0]


def rotary_raw(ptrs, plan, dev, dtype, B, T, d, inv_freq, positions, offset, interleaved, scale, inverse):
    """The launch behind rotary(): ptrs (sources, then destinations) and plan (rotary_plan) of segments that the caller has checked; inv_freq and
    positions are checked here."""
    n = len(ptrs) >> 1
    if dev.type != "cuda":
        raise ValueError("tensors must live on a CUDA device")
    if inv_freq.device != dev or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 vector on the tensors' device")
    pos_ptr, i64, pb, pt = None, 0, 0, 0
    if positions is not None:
        if positions.device != dev or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64 on the tensors' device")
        if positions.shape == (T,):
            pt = positions.stride(0)
        elif positions.shape == (B, T):
            pb, pt = positions.stride()
        else:
            raise ValueError(f"positions must have shape ({T},) or ({B}, {T}), not {tuple(positions.shape)}")
        pos_ptr, i64 = positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0
    if dtype not in _LIST_DT:
        raise ValueError(f"dtype {dtype} not supported (bf16 or fp32)")
    if B * T == 0:
        return
    addresses = array("q", ptrs)
    at, (_, _, strides, ints) = addresses.buffer_info()[0], plan
    with _on(dev):
        rc = _lib.load().quartet_rotary(n, at, at + 8 * n, strides, ints, ints + 4 * n, _LIST_DT[dtype], B, T, d, 2 * inv_freq.shape[0], 1 if interleaved else 0,
                                        pos_ptr, i64, pb, pt, offset, inv_freq.data_ptr(), scale, 1 if inverse else 0, _stream())
    if rc:
        _lib.check(rc, "quartet_rotary")


# ------------------------------------------------------------------------------------------------
# norm over many tensors, and clipping by it
# ------------------------------------------------------------------------------------------------
NORM_PARTIALS = 1024


def _dense(t) -> bool:
    """Whether the elements fill one stretch of memory, in whatever order of the axes."""
    if t.is_contiguous():
        return True
    want = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _tensor_list(ts, dev, what):
    """Host arrays (addresses, element counts, dtypes) of the tensors."""
    idx = dev.index
    try:
        dts = array("i", [_LIST_DT[t.dtype] for t in ts])
    except KeyError:
        dts = None
    if dts is None or dev.type != "cuda" or any([t.get_device() != idx for t in ts]) or not all([t.is_contiguous() or _dense(t) for t in ts]):
        raise ValueError(f"{what} must be dense bf16 or fp32 tensors on one CUDA device")
    return array("q", [t.data_ptr() for t in ts]), array("q", [t.numel() for t in ts]), dts


def _at(a) -> int:
    return a.buffer_info()[0]


def _norm_kind(norm_type) -> int:
    norm_type = float(norm_type)
    if norm_type == 2:
        return 0
    if norm_type == float("inf"):
        return 1
    raise ValueError(f"norm_type must be 2 or inf, not {norm_type}")


def grad_norm(tensors, norm_type=2.0, total=False):
    """Norm over all elements of the tensors (bf16 / fp32, mixed): fp32 scalar on their device.  total=True returns instead what ranks that hold
    different tensors combine: the float64 sum of squares, shape [1] (for the maximum norm, the maximum)."""
    tensors, kind = list(tensors), _norm_kind(norm_type)
    if not tensors:
        raise ValueError("need at least one tensor")
    dev = tensors[0].device
    ptrs, numels, dts = _tensor_list(tensors, dev, "tensors")
    work = torch.empty(NORM_PARTIALS + 1, dtype=torch.float64, device=dev)
    out = work[NORM_PARTIALS:] if total else torch.empty((), dtype=torch.float32, device=dev)
    with _on(dev):
        rc = _lib.load().quartet_grad_norm(len(tensors), _at(ptrs), _at(numels), _at(dts), kind, _ptr(work), _ptr(out) if total else None, None if total else _ptr(out),
                                           _stream())
    _lib.check(rc, "quartet_grad_norm")
    return out


def clip_grads(tensors, max_norm, norm_type=2.0, out=None, total=None):
    """Scales the tensors by min(1, max_norm / (norm + 1e-6)), in place or into `out` (a tensor for each, fp32 or bf16, of its size and layout);
    returns the norm before (fp32 scalar on the device; nothing waits for it).  total: a float64 [1] as grad_norm(..., total=True) returns it, e.g.
    summed over ranks, to use in place of the tensors' own."""
    tensors, kind = list(tensors), _norm_kind(norm_type)
    if not tensors:
        raise ValueError("need at least one tensor")
    dev = tensors[0].device
    ptrs, numels, dts = _tensor_list(tensors, dev, "tensors")
    optrs, odts = ptrs, dts
    if out is not None:
        out = list(out)
        optrs, onumels, odts = _tensor_list(out, dev, "out")
        # contiguous tensors of one size lie alike in memory; others have to agree in shape and strides
        if onumels != numels or not all([(o.is_contiguous() and t.is_contiguous()) or (o.shape == t.shape and o.stride() == t.stride())
                                         for o, t in zip(out, tensors)]):
            raise ValueError("out must hold a tensor of the same size and layout for each of the tensors")
    if total is not None and not (total.is_cuda and total.device == dev and total.dtype == torch.float64 and total.numel() == 1):
        raise ValueError("total must be one float64 value on the tensors' device")
    work = torch.empty(NORM_PARTIALS, dtype=torch.float64, device=dev) if total is None else None
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with _on(dev):
        rc = _lib.load().quartet_clip_grads(len(tensors), _at(ptrs), _at(optrs), _at(numels), _at(dts), _at(odts), kind, float(max_norm), _ptr(total), _ptr(work), _ptr(norm), _stream())
    _lib.check(rc, "quartet_clip_grads")
    torch.autograd.graph.increment_version(tensors if out is None else out)  # a graph that saved one of them then refuses to use it
    return norm


def device_status() -> int:
    """Fault word of the current device (0 = no kernel ever gave up on a bounded wait); clears it."""
    st = C.c_int32(0)
    _lib.check(_lib.load().quartet_device_status(C.byref(st)), "quartet_device_status")
    return st.value


# Every wait inside the kernels is bounded: a kernel that gives up leaves its tiles unwritten and records the
# fact in the fault word instead of hanging.  Nothing reads that word on the hot path (it costs a device
# synchronisation), so a caller that wants wrong results turned into an exception either polls device_status()
# itself at a point where it synchronises anyway, or sets QUARTET_CHECK_FAULTS=1: the layer's backward and
# the gradient exchange's wait() then check the word and raise.
CHECK_FAULTS = os.environ.get("QUARTET_CHECK_FAULTS", "0") not in ("", "0")


def raise_on_fault(where: str) -> None:
    if CHECK_FAULTS:
        word = device_status()
        if word:
            raise _lib.QuartetError(f"{where}: a kernel gave up on a bounded wait (fault word {word:#x}); its results are incomplete")


def unpack_mask(mask_u8: torch.Tensor) -> torch.Tensor:
    """[rows, cols/8] bit-packed (LSB first) -> bool [rows, cols]  (benchmark_mxfp4.ipynb:975-979 `_unpack_mask`)."""
    bits = torch.arange(8, device=mask_u8.device, dtype=torch.uint8)
    return ((mask_u8.unsqueeze(-1) >> bits) & 1).bool().reshape(*mask_u8.shape[:-1], mask_u8.shape[-1] * 8)
