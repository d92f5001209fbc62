"""clip_grad_norm_ for the training loop around the quantized layers (src/optim/base.py:203-204 of the reference calls torch's).

One pass over the gradients for the norm and one to scale them, in two launches; nothing waits for the device.  Weights whose gradient lives
as a shard on each rank (shard.PeerWgradScatter leaves it in `weight.grad_shard`) are clipped by the norm over all ranks' shards.
"""
from __future__ import annotations

import torch
import torch.distributed as dist

from . import ops


def _shard_of(p):
    """The weight's shard of this step, or None; refused while its exchange is in flight, as the shard found there would be an older one."""
    record = getattr(p, "grad_shard_record", None)
    if record is not None:
        if record.in_flight:
            raise RuntimeError("a weight's gradient is still being exchanged: call wait() of its PeerWgradScatter before clipping")
        if record.stale:
            return None
    return getattr(p, "grad_shard", None)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, group=None) -> torch.Tensor:
    """Scales the gradients in place so that their norm (2 or inf) is at most max_norm; returns the norm before, fp32, on the device.

    Gradients are dense bf16 or fp32 tensors on one device.  A parameter with a `grad_shard` and no `grad` counts as sharded: the norm is
    taken over the shards of all ranks of `group` (every rank then has to make this call); gradients in `.grad` are taken to be the
    same on every rank.  A PeerWgradScatter's wait() has to come first: this call raises while one of the parameters' exchanges is in flight.  A shard
    that was clipped before is left out once the sink has been given further exchanges (a layer that took no part in the step).
    error_if_nonfinite reads the norm back, and raises before anything is scaled."""
    norm_type = float(norm_type)
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    whole = [p.grad for p in parameters if p.grad is not None]
    sharded = [(p, s) for p in parameters if p.grad is None and (s := _shard_of(p)) is not None]
    shards = [s for _, s in sharded]
    grads = whole + shards
    if not grads:
        return torch.zeros(())
    total = None
    if shards:
        if not dist.is_initialized():
            raise RuntimeError("sharded gradients need an initialised process group")
        total = ops.grad_norm(shards, norm_type, total=True)
        if norm_type == float("inf"):
            # gathered, not reduced: a library's maximum may drop a NaN, torch's does not
            every = [torch.empty_like(total) for _ in range(dist.get_world_size(group))]
            dist.all_gather(every, total, group=group)
            total = torch.cat(every).max().reshape(1)
        else:
            dist.all_reduce(total, op=dist.ReduceOp.SUM, group=group)
        if whole:
            rest = ops.grad_norm(whole, norm_type, total=True)
            total = torch.maximum(total, rest) if norm_type == float("inf") else total + rest
    elif error_if_nonfinite:
        total = ops.grad_norm(whole, norm_type, total=True)
    if error_if_nonfinite and not bool(torch.isfinite(total)):
        raise RuntimeError(f"the total norm of order {norm_type} of the gradients is not finite")
    norm = ops.clip_grads(grads, max_norm, norm_type, total=total)
    for p, _ in sharded:
        record = getattr(p, "grad_shard_record", None)
        if record is not None:
            record.clipped_at = record.count.submitted
    return norm
