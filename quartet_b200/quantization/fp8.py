"""A linear layer on 8-bit operands with a power-of-two scale for each block of 128, for the layers that four bits cost too much -- the
reference leaves its head un-quantized (src/models/llama.py:197).

    y  = Q(x) Q(w)^T            x in blocks of 1 x 128, w in blocks of 128 x 128, both e4m3
    dx = Q(e) Q(w)              e in blocks of 1 x 128 along the outputs (grad_dtype)
    dw = Qt(e)^T Qt(x)          both in blocks of 128 tokens

A square block of w is a block of its transpose too, so the backward multiplies by exactly the weight the forward used.
Saved for backward: one byte per value of x and w.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import ops, torch_ops  # noqa: F401  (torch_ops registers the operators that a compiled model calls)
from .producers import _out_dtype


def _forward(x, w, need_dx, need_dw, out_dtype):
    return ops.fp8_linear_fwd(x if x.is_contiguous() else x.contiguous(), w if w.is_contiguous() else w.contiguous(), need_dx, need_dw, out_dtype)


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, grad_dtype, out_dtype):
        need_dx, need_dw = ctx.needs_input_grad[:2]
        y, saved = _forward(x, w, need_dx, need_dw, out_dtype)
        ctx.save_for_backward(saved)
        ctx.x_shape, ctx.args, ctx.kept = x.shape, (w.shape[1], grad_dtype, x.dtype, w.dtype), (need_dx, need_dw)
        return y

    @staticmethod
    def backward(ctx, e):
        if torch.is_grad_enabled() or ops.has_tangent(e):
            raise RuntimeError("fp8_linear is not differentiable twice")
        need_dx, need_dw = ctx.needs_input_grad[:2]
        if not (need_dx or need_dw):
            return None, None, None, None
        e2 = e if e.dim() == 2 else e.reshape(-1, e.shape[-1])
        if e2.dtype not in (torch.bfloat16, torch.float32):
            e2 = e2.float()
        dx, dw = ops.fp8_linear_bwd(e2 if e2.is_contiguous() else e2.contiguous(), ctx.saved_tensors[0], *ctx.args, need_dx, need_dw, *ctx.kept)
        if ops.CHECK_FAULTS:
            ops.raise_on_fault("8-bit linear backward")
        if dx is not None and len(ctx.x_shape) != 2:
            dx = dx.view(ctx.x_shape)
        return dx, (dw if dw is None or dw.is_contiguous() else dw.contiguous()), None, None


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, *, grad_dtype: torch.dtype = torch.float8_e4m3fn, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] (bf16 / fp32) times weight [N, K]^T on 8-bit operands, differentiable in both.  out_dtype: bf16 or fp32; by default autocast's, else
    x's.  For a weight that does not change, pack it once (ops.quant_fp8(weight, square=True)) and call ops.linear_fp8."""
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"x [..., K] and weight [N, K] are needed, not {tuple(x.shape)} and {tuple(weight.shape)}")
    if not (x.is_cuda and weight.device == x.device):
        raise ValueError("x and weight must live on one CUDA device")
    ops._f8(grad_dtype)
    out_dtype = out_dtype or _out_dtype(x, x.dtype)
    if ops.recording():
        # a compiled graph is guarded on what needs a gradient; a trace is not, and may be called with other inputs, so it keeps both transposes
        need_dx, need_dw = (True, True) if torch.jit.is_tracing() else [torch.is_grad_enabled() and t.requires_grad for t in (x, weight)]
        return torch.ops.quartet_b200.fp8_linear_fwd(x, weight, grad_dtype, out_dtype, need_dx, need_dw)[0]
    if ops.forward_mode():  # the function has no such derivative, and says so where an input has a tangent
        return ops.eagerly(_Fp8LinearFn.apply, x, weight, grad_dtype, out_dtype)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _Fp8LinearFn.apply(x, weight, grad_dtype, out_dtype)
    return _forward(x, weight, False, False, out_dtype)[0]  # nothing is kept, so neither transpose is made


class Fp8Linear(nn.Linear):
    """nn.Linear whose products run on 8-bit operands (fp8_linear); parameters and state_dict are nn.Linear's."""

    def __init__(self, in_features, out_features, bias=False, grad_dtype=torch.float8_e4m3fn, **kwargs):
        super().__init__(in_features, out_features, bias=bias, **kwargs)
        ops._f8(grad_dtype)
        self.grad_dtype = grad_dtype

    def forward(self, x):
        y = fp8_linear(x, self.weight, grad_dtype=self.grad_dtype)
        return y if self.bias is None else y + self.bias.to(y.dtype)

    def export_fp8(self):
        """The weight as 8-bit codes [N, pad128(K)] and blocked E8M0 scales: what ops.linear_fp8 takes."""
        with torch.no_grad():
            return ops.quant_fp8(self.weight.detach().contiguous(), square=True)[:2]
