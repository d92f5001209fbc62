"""Refusals of the rotary, 8-bit and gradient-norm entry points before anything touches a device, their host-side helpers, and the
sharded clipping over two gloo ranks (the kernels stand in as torch operations there)."""
import ctypes as C
import math
import os

import pytest
import torch

import __graft_entry__ as entry
from quartet_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    entry.build()
    return _lib.load()


@pytest.fixture(scope="module")
def p():
    buf = (C.c_uint8 * 65536)()
    base = (C.addressof(buf) + 255) & ~255
    yield lambda off=0: C.c_void_p(base + off)
    del buf


def test_quant_fp8_refusals(lib, p):
    f = lib.quartet_quant_fp8
    assert f(None, 0, 1, 128, 0, 0, p(), p(), None, None, None) == -1
    assert f(p(), 0, 1, 128, 0, 0, None, None, None, None, None) == -1
    assert f(p(), 0, 1, 128, 0, 0, p(), None, None, None, None) == -1
    assert f(p(), 0, 1, 128, 0, 0, None, None, p(), None, None) == -1
    assert f(p(), 2, 1, 128, 0, 0, p(), p(), None, None, None) == -4
    assert f(p(), 0, 1, 128, 2, 0, p(), p(), None, None, None) == -4
    assert f(p(), 0, 1, 128, 0, 2, p(), p(), None, None, None) == -4
    for rows, cols in ((0, 128), (1, 0), (-1, 128), (8388481, 128), (1, 1 << 30)):
        assert f(p(), 0, rows, cols, 0, 0, p(), p(), None, None, None) == -2
    assert f(p(1), 0, 1, 128, 0, 0, p(), p(), None, None, None) == -3
    assert f(p(2), 1, 1, 128, 0, 0, p(), p(), None, None, None) == -3
    assert f(p(), 0, 1, 128, 0, 0, p(8), p(), None, None, None) == -3
    assert f(p(), 0, 1, 128, 0, 0, p(), p(), p(), p(4), None) == -3
    g = lib.quartet_dequant_fp8
    assert g(None, p(), 1, 1, 0, 1.0, p(), 1, None) == -1
    assert g(p(), p(), 1, 1, 3, 1.0, p(), 1, None) == -4
    assert g(p(), p(), 1, 1, 0, 1.0, p(), 2, None) == -4
    assert g(p(), p(), 0, 1, 0, 1.0, p(), 1, None) == -2
    assert g(p(4), p(), 1, 1, 0, 1.0, p(), 1, None) == -3


def test_gemm_fp8_refusals(lib, p):
    def f(a=p(), asf=p(), fa=0, b=p(), bsf=p(), fb=0, M=4, N=8, K=128, d=p(), dt=0, ldd=8):
        return lib.quartet_gemm_fp8_tn(a, asf, fa, b, bsf, fb, M, N, K, 1.0, d, dt, ldd, None)

    for name in ("a", "asf", "b", "bsf", "d"):
        assert f(**{name: None}) == -1
        assert f(**{name: p(8)}) == -3
    assert f(fa=2) == -4 and f(fb=-1) == -4 and f(dt=2) == -4
    assert f(M=0) == -2 and f(N=0) == -2 and f(K=0) == -2 and f(K=100) == -2 and f(M=8388481) == -2 and f(N=8388481, ldd=1 << 24) == -2
    assert f(ldd=7) == -2 and f(N=9, ldd=8) == -2 and f(N=9, ldd=12) == -2 and f(N=9, ldd=10, dt=1) == -2


def test_linear_fp8_refusals(lib, p):
    def f(x=p(), xd=0, M=4, K=200, w=p(), sf=p(), wd=0, N=8, work=p(), y=p(), yd=0, ldy=8):
        return lib.quartet_linear_fp8(x, xd, M, K, w, sf, wd, N, 1.0, work, y, yd, ldy, None)

    assert lib.quartet_linear_fp8_workspace_bytes(8, 200) == 0 and lib.quartet_linear_fp8_workspace_bytes(9, 200) == 9 * 256 + 128 * 8
    for M in (4, 40):
        for name in ("x", "w", "sf", "y"):
            assert f(M=M, **{name: None}) == -1
        for name in ("w", "sf", "y"):
            assert f(M=M, **{name: p(8)}) == -3
        assert f(M=M, x=p(1)) == -3 and f(M=M, x=p(2), xd=1) == -3
        assert f(M=M, xd=2) == -4 and f(M=M, wd=2) == -4 and f(M=M, yd=2) == -4
        assert f(M=M, N=0) == -2 and f(M=M, K=0) == -2 and f(M=M, N=9) == -2 and f(M=M, ldy=12) == -2
    assert f(M=0) == -2 and f(M=8388481) == -2 and f(M=9, work=None) == -1 and f(M=9, work=p(8)) == -3


def test_layer_refusals(lib, p):
    b3 = (C.c_int64 * 3)()
    assert lib.quartet_linear_fp8_train_bytes(0, 1, 1, 1, 1, b3) == -2 and lib.quartet_linear_fp8_train_bytes(1, 1, 1, 1, 1, None) == -1
    assert lib.quartet_linear_fp8_train_bytes(200, 100, 300, 1, 1, b3) == 0
    xt, wt = 300 * 256 + 384 * 8, 300 * 128 + 384 * 4          # transposes of x and w: codes and scales, in 256-byte units
    assert list(b3) == [xt + wt, 200 * 384 + 256 * 12 + 100 * 384 + 128 * 12, 200 * 128 + 256 * 4 + 100 * 256 + 128 * 8]
    assert lib.quartet_linear_fp8_train_bytes(200, 100, 300, 0, 0, b3) == 0 and b3[0] == 0 and b3[2] == 0

    def fwd(x=p(), xd=0, w=p(), wd=1, M=4, N=8, K=200, sv=p(), wk=p(), y=p(), yd=0, ldy=8):
        return lib.quartet_linear_fp8_train_fwd(x, xd, w, wd, M, N, K, 1, 1, sv, wk, y, yd, ldy, None)

    for name in ("x", "w", "sv", "wk", "y"):
        assert fwd(**{name: None}) == -1
    for name in ("sv", "wk", "y"):
        assert fwd(**{name: p(8)}) == -3
    assert fwd(x=p(1)) == -3 and fwd(w=p(2)) == -3 and fwd(xd=2) == -4 and fwd(wd=2) == -4 and fwd(yd=2) == -4
    assert fwd(M=0) == -2 and fwd(N=0) == -2 and fwd(K=0) == -2 and fwd(K=8388481) == -2 and fwd(ldy=7) == -2 and fwd(ldy=12) == -2

    def bwd(e=p(), ed=0, M=4, N=8, K=200, fmt=0, sv=p(), wk=p(), dx=p(), xd=0, ldx=200, dw=p(), wd=1, ldw=200, sx=1, sw=1):
        return lib.quartet_linear_fp8_train_bwd(e, ed, M, N, K, fmt, sv, wk, dx, xd, ldx, dw, wd, ldw, sx, sw, None)

    for name in ("e", "sv", "wk"):
        assert bwd(**{name: None}) == -1
    for name in ("sv", "wk", "dx", "dw"):
        assert bwd(**{name: p(8)}) == -3
    assert bwd(dx=None, dw=None, e=None) == 0 and bwd(e=p(1)) == -3
    assert bwd(sx=0) == -4 and bwd(sw=0) == -4 and bwd(fmt=2) == -4 and bwd(ed=2) == -4 and bwd(xd=2) == -4 and bwd(wd=2) == -4
    assert bwd(M=0) == -2 and bwd(ldx=199) == -2 and bwd(ldw=202) == -2


def test_rotary_refusals(lib, p):
    def f(n=1, src=(p(),), dst=(p(1024),), strides=(0,) * 18, heads=(1,), rotate=(1,), dt=0, batch=1, tokens=1, d=64, rot=64, pos=None, i64=1, inv=p(2048)):
        m = max(len(src), 1)
        pad = lambda v, k: list(v) + [0] * (k - len(v))  # noqa: E731
        arr = lambda v: (C.c_void_p * m)(*[x.value if x else None for x in v])  # noqa: E731
        return lib.quartet_rotary(n, arr(src) if src else None, arr(dst), (C.c_int64 * 18)(*strides), (C.c_int32 * 3)(*pad(heads, 3)), (C.c_int32 * 3)(*pad(rotate, 3)), dt,
                                  batch, tokens, d, rot, 1, pos, i64, 0, 0, 0, inv, 1.0, 0, None)

    assert f(n=0) == -4 and f(n=4) == -4 and f(dt=3) == -4
    assert f(src=(None,)) == -1 and f(dst=(None,)) == -1 and f(inv=None) == -1 and f(src=()) == -1
    assert f(batch=0) == -2 and f(tokens=0) == -2 and f(batch=1 << 16, tokens=1 << 15) == -2
    assert f(rot=63) == -2 and f(rot=66) == -2 and f(rot=0) == -2 and f(d=1024, rot=514) == -2 and f(heads=(0,)) == -2
    assert f(src=(p(1),)) == -3 and f(dst=(p(2),), dt=1) == -3 and f(inv=p(4)) == -3 and f(pos=p(4)) == -3 and f(pos=p(2), i64=0) == -3


def test_grad_list_refusals(lib, p):
    def lists(ptrs, numels, dts):
        n = len(ptrs)
        return n, (C.c_void_p * n)(*[x.value if x else None for x in ptrs]), (C.c_int64 * n)(*numels), (C.c_int32 * n)(*dts)

    def norm(ptrs, numels, dts, kind=0, work=p(4096), total=p(8192), out=None):
        n, a, b, c = lists(ptrs, numels, dts)
        return lib.quartet_grad_norm(n, a, b, c, kind, work, total, out, None)

    assert norm([p()], [4], [1], kind=2) == -4 and norm([p()], [4], [2]) == -4
    assert norm([None], [4], [1]) == -1 and norm([p()], [4], [1], work=None) == -1 and norm([p()], [4], [1], total=None) == -1
    assert norm([p()], [-1], [1]) == -2 and norm([p(2)], [4], [1]) == -3 and norm([p(1)], [4], [0]) == -3
    assert norm([p()], [4], [1], work=p(4)) == -3 and norm([p()], [4], [1], out=p(2)) == -3
    assert lib.quartet_grad_norm(1, None, None, None, 0, p(), p(), None, None) == -1 and lib.quartet_grad_norm(-1, None, None, None, 0, p(), p(), None, None) == -4

    def clip(ptrs, outs, numels, dts, odts=None, max_norm=1.0, total=None, work=p(4096)):
        n, a, b, c = lists(ptrs, numels, dts)
        _, o, _, oc = lists(outs, numels, odts or dts)
        return lib.quartet_clip_grads(n, a, o, b, c, oc, 0, max_norm, total, work, None, None)

    assert clip([p()], [p()], [4], [1], max_norm=-1.0) == -4 and clip([p()], [p()], [4], [1], max_norm=math.nan) == -4
    assert clip([p()], [p()], [4], [1], work=None) == -1 and clip([p()], [None], [4], [1]) == -1
    # outputs that share memory: with one another, with another gradient, with their own at an offset or in another type
    assert clip([p(), p(256)], [p(512), p(520)], [4, 4], [1, 1]) == -4
    assert clip([p(), p(256)], [p(512), p(8)], [4, 4], [1, 1]) == -4
    assert clip([p(), p()], [p(), p()], [4, 4], [1, 1]) == -4
    assert clip([p()], [p(4)], [4], [1]) == -4 and clip([p(16)], [p()], [8], [1]) == -4
    assert clip([p()], [p()], [4], [0], [1]) == -4
    assert clip([p(0), p(64), p(16)], [p(0), p(64), p(16)], [4, 4, 13], [1, 1, 1]) == -4
    assert b"share memory" in lib.quartet_last_error_string()


def test_wrappers_refuse_host_tensors():
    from quartet_b200 import ops
    from quartet_b200.clip import clip_grad_norm_
    from quartet_b200.quantization import Fp8Linear, fp8_linear
    from quartet_b200.rotary import apply_rotary, rotary_frequencies, rotary_qkv

    x, inv = torch.zeros(2, 128), rotary_frequencies(64)[0]
    with pytest.raises(ValueError):
        ops.quant_fp8(x)
    with pytest.raises(ValueError):
        fp8_linear(x, x)
    with pytest.raises(ValueError):
        Fp8Linear(128, 64)(x)
    with pytest.raises(ValueError):
        Fp8Linear(128, 64, grad_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        apply_rotary(torch.zeros(1, 2, 3, 64), None, inv)
    with pytest.raises(ValueError):
        rotary_qkv(torch.zeros(1, 2, 192), 1, 1, inv)
    with pytest.raises(ValueError):
        ops.grad_norm([x])
    w = torch.nn.Parameter(x)
    w.grad = x.clone()
    with pytest.raises(ValueError):
        clip_grad_norm_([w], 1.0)


def test_frequencies():
    from quartet_b200.rotary import rotary_frequencies

    inv, s = rotary_frequencies(128)
    assert s == 1.0 and inv.dtype == torch.float64 and torch.equal(inv, 10000.0 ** -(torch.arange(0, 128, 2, dtype=torch.float64) / 128))
    lin, _ = rotary_frequencies(128, scaling={"kind": "linear", "factor": 4.0})
    assert torch.equal(lin, inv / 4)
    ntk, _ = rotary_frequencies(128, scaling={"kind": "ntk", "factor": 4.0})
    assert ntk[0] == inv[0] and abs(ntk[-1] * 4 / inv[-1] - 1) < 1e-12
    bands, _ = rotary_frequencies(128, 500000.0, {"kind": "bands", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 4.0})
    base, _ = rotary_frequencies(128, 500000.0)
    turns = 8192 * base / (2 * math.pi)
    assert torch.equal(bands[turns > 4], base[turns > 4]) and torch.allclose(bands[turns < 1], base[turns < 1] / 8, rtol=1e-15)
    mid = (turns < 4) & (turns > 1)
    assert bool(((bands < base) & (bands > base / 8))[mid].all())
    yarn, s = rotary_frequencies(128, scaling={"kind": "yarn", "factor": 16.0, "original_length": 4096})
    assert abs(s - (0.1 * math.log(16) + 1)) < 1e-12 and yarn[0] == inv[0] and abs(yarn[-1] * 16 / inv[-1] - 1) < 1e-12
    assert rotary_frequencies(128, scaling={"kind": "yarn", "factor": 2.0, "original_length": 4096, "attention_factor": 1.0})[1] == 1.0
    for bad in ({"kind": "other"}, {"kind": "linear", "factor": 0.5}, {"kind": "linear", "factor": 2.0, "typo": 1}, {"kind": "bands", "factor": 2.0, "original_length": 10,
                                                                                                              "low": 4.0, "high": 1.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling=bad)
    for bad in (0, 63, -2):
        with pytest.raises(ValueError):
            rotary_frequencies(bad)


def _shard_rank(rank, port, inf, nan, out):
    import torch.distributed as dist

    from quartet_b200 import clip, ops

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)

    def total_of(ts, kind, total=False):
        flat = torch.cat([t.double().reshape(-1) for t in ts])
        return flat.abs().max().reshape(1) if kind == math.inf else flat.square().sum().reshape(1)

    def scale(ts, max_norm, kind=2.0, out=None, total=None):
        n = total[0] if kind == math.inf else total[0].sqrt()
        for t in ts:
            t.mul_(float((max_norm / (n + 1e-6)).clamp(max=1.0)))
        return n.float()

    ops.grad_norm, ops.clip_grads = total_of, scale
    g = torch.Generator().manual_seed(0)
    full, rest = torch.randn(8, 5, generator=g), torch.randn(7, generator=g)
    p, q = torch.nn.Parameter(torch.zeros(8, 5)), torch.nn.Parameter(torch.zeros(7))
    p.grad_shard, q.grad = full[4 * rank:4 * rank + 4].clone(), rest.clone()
    if nan and rank == 1:
        p.grad_shard[2, 3] = math.nan
    n = clip.clip_grad_norm_([p, q], 0.5, math.inf if inf else 2.0)
    both = torch.cat([full.reshape(-1), rest]).double()
    want = both.abs().max() if inf else both.norm()
    ok = abs(n.item() - want.item()) < 1e-6 and torch.allclose(p.grad_shard, full[4 * rank:4 * rank + 4] * (0.5 / want).float(), rtol=1e-5)
    if nan:
        ok = math.isnan(n.item()) and bool(torch.isnan(p.grad_shard).all()) and bool(torch.isnan(q.grad).all())
    out[rank] = ok if nan else ok and torch.allclose(q.grad, rest * (0.5 / want).float(), rtol=1e-5)
    dist.destroy_process_group()


@pytest.mark.parametrize("inf,nan", [(False, False), (True, False), (False, True), (True, True)])
def test_sharded_clip_over_two_ranks(inf, nan):
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    with ctx.Manager() as m:
        out = m.dict()
        mp.spawn(_shard_rank, args=(port, inf, nan, out), nprocs=2)
        assert dict(out) == {0: True, 1: True}


def test_sharded_gradients_need_a_group():
    from quartet_b200.clip import clip_grad_norm_

    w = torch.nn.Parameter(torch.zeros(4))
    w.grad_shard = torch.zeros(2)
    with pytest.raises(RuntimeError):
        clip_grad_norm_([w], 1.0)
