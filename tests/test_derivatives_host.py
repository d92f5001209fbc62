"""Derivatives of the rotary and 8-bit entry points that do not go through requires_grad: forward mode and recorded traces.  The kernels stand in
as torch operations on the host."""
import pytest
import torch
from torch.autograd import forward_ad as fwad

from quartet_b200 import ops, torch_ops
from quartet_b200.quantization import fp8_linear
from quartet_b200.rotary import apply_rotary, rotary_frequencies, rotary_qkv


def _turned(x, inv, positions, offset, interleaved, scale, inverse):
    b, t = x.shape[:2]
    pos = (offset + torch.arange(t)).expand(b, t) if positions is None else positions.expand(b, t)
    a = (-1.0 if inverse else 1.0) * pos.double()[..., None, None] * inv
    c, s, r = a.cos() * scale, a.sin() * scale, 2 * inv.numel()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y = x.double().clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y.to(x.dtype)


@pytest.fixture(autouse=True)
def host_kernels(monkeypatch):
    def rotary(segments, inv, positions=None, offset=0, interleaved=True, scale=1.0, inverse=False):
        for src, dst, rotate in segments:  # through numpy: nothing that a derivative or a recorder could see
            y = _turned(torch.from_numpy(src.detach().numpy().copy()), inv, positions, offset, interleaved, scale, inverse) if rotate else src
            dst.detach().numpy()[...] = y.numpy()

    def split(qkv, n_head, n_kv_head, inv, positions, offset, interleaved, scale, head_major):
        b, t, w = qkv.shape
        d = w // (n_head + 2 * n_kv_head)
        raw = torch.from_numpy(qkv.detach().numpy().copy())
        out = []
        for i, (z, h) in enumerate(zip(raw.split([n_head * d, n_kv_head * d, n_kv_head * d], -1), (n_head, n_kv_head, n_kv_head))):
            z = z.unflatten(-1, (h, d))
            z = _turned(z, inv, positions, offset, interleaved, scale, False) if i < 2 else z
            y = qkv.new_empty((b, h, t, d) if head_major else (b, t, h, d))
            y.detach().numpy()[...] = (z.transpose(1, 2) if head_major else z).numpy()
            out.append(y)
        return tuple(out)

    def join(dq, dk, dv, inv, positions, offset, interleaved, scale, head_major):
        view = (lambda z: z.transpose(1, 2)) if head_major else (lambda z: z)
        q, k, v = (view(torch.from_numpy(z.detach().numpy().copy())) for z in (dq, dk, dv))
        parts = [_turned(q, inv, positions, offset, interleaved, scale, True), _turned(k, inv, positions, offset, interleaved, scale, True), v]
        y = torch.cat([z.flatten(2) for z in parts], -1)
        out = dq.new_empty(y.shape)
        out.detach().numpy()[...] = y.numpy()
        return out

    monkeypatch.setattr(ops, "rotary", rotary)
    monkeypatch.setattr(torch_ops, "split_heads", split)
    monkeypatch.setattr(torch_ops, "join_heads", join)


INV = rotary_frequencies(16)[0]
POS = torch.tensor([[3, 1, 7, 1000], [0, 5, 5, 9]])


@pytest.mark.parametrize("interleaved", [True, False])
def test_apply_rotary_forward_mode(interleaved):
    q, k, dq, dk = torch.randn(2, 4, 3, 16), torch.randn(2, 4, 1, 16), torch.randn(2, 4, 3, 16), torch.randn(2, 4, 1, 16)
    f = lambda a, b: apply_rotary(a, b, INV, POS, interleaved=interleaved, scale=1.5)  # noqa: E731
    with fwad.dual_level():
        yq, yk = f(fwad.make_dual(q, dq), fwad.make_dual(k, dk))
        (pq, tq), (pk, tk) = fwad.unpack_dual(yq), fwad.unpack_dual(yk)
        only, none = apply_rotary(fwad.make_dual(q, dq), None, INV, POS, interleaved=interleaved, scale=1.5)
        t_only = fwad.unpack_dual(only).tangent
        mixed_q, mixed_k = f(fwad.make_dual(q, dq), k)          # one of the two alone
        t_mixed, t_none = fwad.unpack_dual(mixed_q).tangent, fwad.unpack_dual(mixed_k).tangent
        plain = fwad.unpack_dual(f(q, k)[0])
    want_q, want_k = f(dq, dk)                                  # the rotation is linear
    assert torch.equal(tq, want_q) and torch.equal(tk, want_k) and torch.equal(t_only, want_q) and torch.equal(t_mixed, want_q)
    assert none is None and (t_none is None or not t_none.any()) and plain.tangent is None
    assert torch.equal(pq, f(q, k)[0]) and torch.equal(pk, f(q, k)[1])


def test_apply_rotary_forward_over_reverse():
    q, e, de = torch.randn(1, 4, 2, 16, requires_grad=True), torch.randn(1, 4, 2, 16), torch.randn(1, 4, 2, 16)
    with fwad.dual_level():
        y = apply_rotary(q, None, INV, scale=1.5)[0]
        (g,) = torch.autograd.grad(y, (q,), fwad.make_dual(e, de))
        tangent = fwad.unpack_dual(g).tangent
    (want,) = torch.autograd.grad(apply_rotary(q, None, INV, scale=1.5)[0], (q,), de)
    assert tangent is not None and torch.equal(tangent, want)


@pytest.mark.parametrize("head_major", [True, False])
def test_rotary_qkv_forward_mode(head_major):
    x, dx = torch.randn(2, 4, 5 * 16), torch.randn(2, 4, 5 * 16)
    f = lambda z: rotary_qkv(z, 3, 1, INV, POS, scale=1.5, head_major=head_major)  # noqa: E731
    with fwad.dual_level():
        outs = f(fwad.make_dual(x, dx))
        tangents = [fwad.unpack_dual(z).tangent for z in outs]
    assert all(t is not None and torch.equal(t, w) for t, w in zip(tangents, f(dx)))
    # its gradient's tangent is refused like its gradient's gradient
    z = x.clone().requires_grad_()
    with fwad.dual_level(), pytest.raises(RuntimeError, match="not differentiable twice"):
        outs = f(z)
        torch.autograd.grad(outs, (z,), [fwad.make_dual(torch.ones_like(o), torch.ones_like(o)) for o in outs])


def _opaque(x, w, dt):
    y = torch.empty(*x.shape[:-1], w.shape[0], dtype=dt)
    y.detach().numpy()[...] = x.detach().numpy() @ w.detach().numpy().T
    return y


def _fp8_on_host(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(ops, "fp8_linear_fwd", lambda x, w, need_dx, need_dw, dt: (_opaque(x, w, dt), torch.zeros(8)))
    monkeypatch.setattr(ops, "fp8_linear_bwd", lambda e, saved, K, gd, xd, wd, need_dx, need_dw, sx, sw: (torch.ones(e.shape[0], K), torch.ones(e.shape[1], K)))


def test_fp8_linear_refuses_forward_mode(monkeypatch):
    _fp8_on_host(monkeypatch)
    x, w = torch.randn(3, 8), torch.randn(5, 8)
    with fwad.dual_level():
        assert fwad.unpack_dual(fp8_linear(x, w)).tangent is None
        for a, b in ((fwad.make_dual(x, x), w), (x, fwad.make_dual(w, w))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                fp8_linear(a, b)
        xg = x.clone().requires_grad_()
        y = fp8_linear(xg, w)
        with pytest.raises(RuntimeError, match="not differentiable twice"):
            torch.autograd.grad(y, (xg,), fwad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_compiled_calls_keep_tangents():
    q, dq, x = torch.randn(2, 4, 3, 16), torch.randn(2, 4, 3, 16), torch.randn(2, 4, 5 * 16)
    f = torch.compile(lambda a: apply_rotary(a, None, INV, scale=1.5)[0] * 1.0, backend="aot_eager")
    g = torch.compile(lambda a: rotary_qkv(a, 3, 1, INV, scale=1.5)[2] * 1.0, backend="aot_eager")
    f(q), g(x)                                                  # compiled without
    with fwad.dual_level():
        t, u = (fwad.unpack_dual(z).tangent for z in (f(fwad.make_dual(q, dq)), g(fwad.make_dual(x, x))))
    assert t is not None and torch.equal(t, apply_rotary(dq, None, INV, scale=1.5)[0])
    assert u is not None and torch.equal(u, rotary_qkv(x, 3, 1, INV)[2])


@pytest.mark.parametrize("grad", [False, True])
def test_traces_record_the_rotation(grad):
    q, k, x = torch.randn(2, 4, 3, 16), torch.randn(2, 4, 1, 16), torch.randn(2, 4, 5 * 16)
    for t in (q, k, x):
        t.requires_grad_(grad)
    f = torch.jit.trace(lambda a, b: apply_rotary(a, b, INV, scale=1.5), (q, k))
    g = torch.jit.trace(lambda z: rotary_qkv(z, 3, 1, INV, scale=1.5), (x,))
    q2, k2, x2 = (torch.randn_like(t) for t in (q, k, x))
    assert all(torch.equal(a, b) for a, b in zip(f(q2, k2), apply_rotary(q2, k2, INV, scale=1.5)))
    assert all(torch.equal(a, b) for a, b in zip(g(x2), rotary_qkv(x2, 3, 1, INV, scale=1.5)))


def test_trace_records_the_8_bit_layer(monkeypatch):
    _fp8_on_host(monkeypatch)
    w = torch.randn(5, 8)
    f = torch.jit.trace(lambda a: fp8_linear(a, w), (torch.randn(2, 3, 8),))
    x = torch.randn(2, 3, 8)
    assert torch.equal(f(x), fp8_linear(x, w))


def test_the_packed_form_refuses_what_it_cannot_differentiate():
    x, w, sf = torch.randn(3, 256), torch.zeros(8, 256, dtype=torch.float8_e4m3fn), torch.zeros(ops.sf_bytes(8, 256), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="no derivative"):
        ops.linear_fp8(x.clone().requires_grad_(), w, sf)
    with fwad.dual_level(), pytest.raises(RuntimeError, match="no derivative"):
        ops.linear_fp8(fwad.make_dual(x, x), w, sf)
    with torch.no_grad(), pytest.raises(ValueError):            # a leaf of a model that is served: only the device is wrong here
        ops.linear_fp8(x.clone().requires_grad_(), w, sf)


def test_the_packed_form_is_compiled_and_traced_as_one_operator(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_linear_fp8", lambda a, b, c, dt: _opaque(torch.nn.functional.pad(a.detach(), (0, 56)), b.float(), dt))
    w, sf = torch.randn(8, 256).to(torch.float8_e4m3fn), torch.zeros(ops.sf_bytes(8, 256), dtype=torch.uint8)
    x, z = torch.randn(2, 3, 200), torch.randn(2, 3, 200)
    f = lambda a: ops.linear_fp8(a, w, sf) * 2  # noqa: E731
    want = f(x)
    assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(x), want) and want.shape == (2, 3, 8)
    assert torch.equal(torch.jit.trace(f, (x,))(z), f(z))
    with pytest.raises(Exception, match="no derivative"):
        torch.compile(f, fullgraph=True, backend="aot_eager")(x.clone().requires_grad_())


def test_forward_mode_does_not_load_the_compiler():
    """Loading it takes seconds; only a call inside compiled code needs it."""
    import os
    import subprocess
    import sys

    code = """if True:
        import sys, torch
        from torch.autograd import forward_ad as fwad
        from quartet_b200 import ops, rotary
        ops.rotary = lambda segments, *a: [dst.detach().copy_(src.detach()) for src, dst, _ in segments]
        x = torch.randn(1, 2, 1, 8)
        with fwad.dual_level():
            y = rotary.apply_rotary(fwad.make_dual(x, x + 1), None, torch.ones(4, dtype=torch.float64))[0]
            assert torch.equal(fwad.unpack_dual(y).tangent, x + 1)
        sys.exit('torch._dynamo' in sys.modules)"""
    assert subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__)))).returncode == 0
