"""Rotary positions for the q and k that a quantized projection produces (LlamaAttention, src/models/llama.py:117-158 of the reference,
whose pairs are interleaved).

    inv_freq, scale = rotary_frequencies(head_dim, base=10000.0, scaling=None, device=...)
    q, k = apply_rotary(q, k, inv_freq, positions)                      # [batch, tokens, heads, d], any strides
    q, k, v = rotary_qkv(qkv, n_head, n_kv_head, inv_freq)              # packed projection -> heads, one pass over memory

Both are differentiable, in reverse and in forward mode; the backward of rotary_qkv writes the packed gradient that the projection's backward reads.
"""
from __future__ import annotations

import math

import torch

from . import ops, torch_ops


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: dict | None = None, device=None):
    """(inv_freq float64 [rot_dim / 2], scale): angles per position and the factor of the rotated values.

    scaling, for contexts longer than the trained one:
      {"kind": "linear", "factor": f}     positions divided by f
      {"kind": "ntk", "factor": f}        base raised so that the slowest pair is divided by f and the fastest kept
      {"kind": "bands", "factor": f, "original_length": L, "low": 1.0, "high": 4.0}
                                          pairs that turn fewer than `low` times in L tokens divided by f, those that turn more than `high`
                                          times kept, a linear mixture between
      {"kind": "yarn", "factor": f, "original_length": L, "beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": None}
                                          the mixture as a ramp over the pair index, and scale = 0.1 ln f + 1
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and at least 2")
    if not base > 0:
        raise ValueError("base must be positive")
    exponent = torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim
    inv, scale = base ** -exponent, 1.0
    if scaling is not None:
        opts = dict(scaling)
        kind, f = opts.pop("kind", None), float(opts.pop("factor", 1.0))
        if not 1.0 <= f < math.inf:
            raise ValueError("factor must be finite and at least 1")
        if kind in ("bands", "yarn"):
            length = float(opts.pop("original_length", 0.0))
            if not length > 0:
                raise ValueError(f"{kind} scaling needs an original_length above 0")
        if kind == "linear":
            inv = inv / f
        elif kind == "ntk":
            if rot_dim < 4:
                raise ValueError("ntk scaling needs at least two pairs")
            inv = (base * f ** (rot_dim / (rot_dim - 2))) ** -exponent
        elif kind == "bands":
            low, high = float(opts.pop("low", 1.0)), float(opts.pop("high", 4.0))
            if not 0 < low < high:
                raise ValueError("need 0 < low < high")
            keep = ((length * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
            inv = (1.0 - keep) * inv / f + keep * inv
        elif kind == "yarn":
            fast, slow = float(opts.pop("beta_fast", 32.0)), float(opts.pop("beta_slow", 1.0))
            if not 0 < slow <= fast:
                raise ValueError("need 0 < beta_slow <= beta_fast")
            if base == 1.0:
                raise ValueError("yarn scaling needs a base other than 1")

            def pair(turns):
                return rot_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot_dim - 1)
            ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            inv = inv / f * ramp + inv * (1.0 - ramp)
            factor = opts.pop("attention_factor", None)
            scale = 0.1 * math.log(f) + 1.0 if factor is None else float(factor)
        else:
            raise ValueError(f"unknown scaling kind {kind!r}")
        if opts:
            raise ValueError(f"unknown scaling options {sorted(opts)}")
    return inv.to(device), scale


def _adjacent(x):
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _turn(xs, inv_freq, positions, offset, interleaved, scale, inverse):
    xs = [_adjacent(x) for x in xs]
    outs = [torch.empty_like(x) for x in xs]
    ops.rotary([(x, y, True) for x, y in zip(xs, outs)], inv_freq, positions, offset, interleaved, scale, inverse)
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, offset, interleaved, scale, inverse):
        ctx.save_for_backward(inv_freq, positions)
        ctx.save_for_forward(inv_freq, positions)
        ctx.args = (offset, interleaved, scale, inverse)
        ctx.set_materialize_grads(False)
        if k is None:
            return _turn((q,), inv_freq, positions, *ctx.args)[0], None
        return tuple(_turn((q, k), inv_freq, positions, *ctx.args))

    @staticmethod
    def backward(ctx, dq, dk):
        inv_freq, positions = ctx.saved_tensors
        offset, interleaved, scale, inverse = ctx.args
        need_q, need_k = dq is not None and ctx.needs_input_grad[0], dk is not None and ctx.needs_input_grad[1]
        gs = ([dq] if need_q else []) + ([dk] if need_k else [])
        if not gs:
            return (None,) * 8
        if torch.is_grad_enabled() or ops.forward_mode():  # create_graph, or tangents: the gradient is a rotation too
            outs = _turn_by_mode(gs[0], gs[1] if len(gs) == 2 else None, inv_freq, positions, offset, interleaved, scale, not inverse)
        else:
            outs = _turn(gs, inv_freq, positions, offset, interleaved, scale, not inverse)
        return outs[0] if need_q else None, outs[-1 if len(gs) == 2 else 0] if need_k else None, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *unused):
        inv_freq, positions = ctx.saved_tensors
        return _Rotary.apply(tq, None, inv_freq, positions, *ctx.args)  # linear: the tangent turns alike (k: _turn_by_mode sends it alone)


def _turn_by_mode(q, k, *args):
    """_Rotary.apply; with a level of forward mode open each tensor by itself, as either may be without a tangent."""
    if k is None or not ops.forward_mode():
        return _Rotary.apply(q, k, *args)
    return _Rotary.apply(q, None, *args)[0], _Rotary.apply(k, None, *args)[0]


def _check_heads(x, what):
    if x.dim() != 4:
        raise ValueError(f"{what} must be [batch, tokens, heads, d]")


def apply_rotary(q, k, inv_freq, positions=None, *, offset=0, interleaved=True, scale=1.0):
    """Turns q and k (k may be None), [batch, tokens, heads, d] views of any strides; heads may differ.  The first 2 * len(inv_freq) values of
    each head are rotated (times `scale`), the rest is copied.  positions: int32 / int64 [tokens] or [batch, tokens]; None: offset + token."""
    _check_heads(q, "q")
    if k is not None:
        _check_heads(k, "k")
    if ops.recording():
        turn = torch.ops.quartet_b200.rotary
        return (turn(q, inv_freq, positions, offset, interleaved, scale, False),
                None if k is None else turn(k, inv_freq, positions, offset, interleaved, scale, False))
    if ops.forward_mode():
        return ops.eagerly(_turn_by_mode, q, k, inv_freq, positions, offset, interleaved, scale, False)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, inv_freq, positions, offset, interleaved, scale, False)
    if k is None:
        return _turn((q,), inv_freq, positions, offset, interleaved, scale, False)[0], None
    return tuple(_turn((q, k), inv_freq, positions, offset, interleaved, scale, False))


class _RotaryQKV(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, n_head, n_kv_head, inv_freq, positions, offset, interleaved, scale, head_major):
        ctx.save_for_backward(inv_freq, positions)
        ctx.save_for_forward(inv_freq, positions)
        ctx.heads, ctx.args = (n_head, n_kv_head), (offset, interleaved, scale, head_major)
        return torch_ops.split_heads(qkv, n_head, n_kv_head, inv_freq, positions, offset, interleaved, scale, head_major)

    @staticmethod
    def backward(ctx, dq, dk, dv):
        inv_freq, positions = ctx.saved_tensors
        if torch.is_grad_enabled() or ops.has_tangent(dq, dk, dv):
            raise RuntimeError("rotary_qkv is not differentiable twice: use apply_rotary under create_graph")
        return torch_ops.join_heads(dq, dk, dv, inv_freq, positions, *ctx.args), None, None, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, t, *unused):
        return _RotaryQKV.apply(t, *ctx.heads, *ctx.saved_tensors, *ctx.args)


def rotary_qkv(qkv, n_head, n_kv_head, inv_freq, positions=None, *, offset=0, interleaved=True, scale=1.0, head_major=True):
    """The packed projection [batch, tokens, (n_head + 2 n_kv_head) d] split into q, k, v with q and k turned: [batch, heads, tokens, d]
    (head_major, what scaled_dot_product_attention takes) or [batch, tokens, heads, d], each contiguous."""
    if qkv.dim() != 3 or n_head < 1 or n_kv_head < 1 or qkv.shape[2] % (n_head + 2 * n_kv_head) or qkv.shape[2] == 0:
        raise ValueError("qkv must be [batch, tokens, (n_head + 2 n_kv_head) * d]")
    if ops.recording():
        return torch.ops.quartet_b200.rotary_qkv(qkv, n_head, n_kv_head, inv_freq, positions, offset, interleaved, scale, head_major)
    if ops.forward_mode():
        return ops.eagerly(_RotaryQKV.apply, qkv, n_head, n_kv_head, inv_freq, positions, offset, interleaved, scale, head_major)
    if torch.is_grad_enabled() and qkv.requires_grad:
        return _RotaryQKV.apply(qkv, n_head, n_kv_head, inv_freq, positions, offset, interleaved, scale, head_major)
    return torch_ops.split_heads(qkv, n_head, n_kv_head, inv_freq, positions, offset, interleaved, scale, head_major)
