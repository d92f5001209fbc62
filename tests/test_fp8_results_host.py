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
