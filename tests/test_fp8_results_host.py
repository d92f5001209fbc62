"""What fp8_linear hands back, with the library's launches replaced: results that belong to nobody else, in every shape."""
import contextlib

import pytest
import torch

import __graft_entry__ as entry
from quartet_b200 import _lib, ops
from quartet_b200.quantization import fp8_linear


class _Lib:
    """The library's host functions, and launches that do nothing."""

    def __init__(self, real):
        self.real = real

    def __getattr__(self, name):
        if name in ("quartet_linear_fp8_train_fwd", "quartet_linear_fp8_train_bwd"):
            return lambda *a: 0
        return getattr(self.real, name)


@pytest.fixture(autouse=True)
def no_launches(monkeypatch):
    entry.build()
    lib = _Lib(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(ops, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)


@pytest.mark.parametrize("shape", [(5, 256), (2, 3, 256), (256,), (1, 1, 2, 256), (0, 256), (3, 0, 256)])
@pytest.mark.parametrize("n", [64, 77, 1])
def test_results_can_be_changed_in_place(shape, n):
    x, w = torch.randn(shape, requires_grad=True), torch.randn(n, 256, requires_grad=True)
    y = fp8_linear(x, w)
    assert y.shape == (*shape[:-1], n) and not y._is_view()
    y.add_(torch.ones(n))
    torch.relu_(y)
    y.sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape
    with torch.no_grad():
        assert fp8_linear(x, w).shape == (*shape[:-1], n)
    # rows start on 16-byte boundaries
    assert y.numel() == 0 or all(s % 4 == 0 for s, extent in zip(y.stride()[:-1], y.shape) if extent > 1)


def test_operands_that_do_not_belong_together_are_refused(monkeypatch):
    """What the library cannot see from addresses: extents that differ, and a kept buffer that is not this backward's."""
    x, w, e = torch.zeros(40, 256), torch.zeros(64, 256), torch.zeros(40, 64)
    for a, b in ((x, torch.zeros(64, 128)), (torch.zeros(40, 300), w), (x, w[0]), (torch.zeros(()), w)):
        with pytest.raises(ValueError):
            ops.fp8_linear_fwd(a, b, True, True, torch.float32)
    with pytest.raises(ValueError):
        ops.fp8_linear_fwd(x, w, True, True, torch.float16)
    y, saved = ops.fp8_linear_fwd(x, w, True, True, torch.float32)
    back = lambda e=e, s=saved, K=256, dx=True, dw=True, sx=True, sw=True: ops.fp8_linear_bwd(e, s, K, torch.float8_e4m3fn, torch.float32, torch.float32, dx, dw, sx, sw)  # noqa: E731
    assert [t.shape for t in back()] == [(40, 256), (64, 256)]
    only = ops.fp8_linear_fwd(x, w, False, True, torch.float32)[1]
    assert back(s=only, dx=False, sx=False)[0] is None
    for bad in (dict(s=saved[:-1]), dict(s=only), dict(s=saved.float()), dict(e=torch.zeros(300, 64)), dict(e=torch.zeros(40, 200)), dict(K=1024), dict(e=e[0]),
                dict(s=torch.empty(0, dtype=torch.uint8)), dict(sx=False, dx=False)):
        with pytest.raises(ValueError):
            back(**bad)
    assert back(e=torch.zeros(0, 64), s=torch.empty(0, dtype=torch.uint8))[1].shape == (64, 256)


@pytest.mark.parametrize("shape", [(0, 256), (3, 0, 256), (1, 256), (3, 5, 256), (300, 256)])
@pytest.mark.parametrize("need", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("n", [64, 77])
def test_operators_keep_the_shapes_they_state(shape, need, n):
    """What the compiler is told of the layer's operators is what they return, without tokens too."""
    from torch._subclasses import FakeTensorMode

    x, w = torch.randn(shape), torch.randn(n, 256)
    fwd, bwd = torch.ops.quartet_b200.fp8_linear_fwd, torch.ops.quartet_b200.fp8_linear_bwd
    f8, f32 = torch.float8_e4m3fn, torch.float32
    real = fwd(x, w, f8, f32, *need)
    e = torch.zeros(*shape[:-1], n)
    back = bwd(e, real[1], 256, f8, f32, f32, *need)
    with FakeTensorMode() as mode:
        fx, fw, fe = (mode.from_tensor(t) for t in (x, w, e))
        told = fwd(fx, fw, f8, f32, *need)
        told_back = bwd(fe, told[1], 256, f8, f32, f32, *need)
    for a, b in zip((*real, *back), (*told, *told_back)):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
