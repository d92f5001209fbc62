"""Clipping of the shards that a PeerWgradScatter really leaves behind, step after step: its bookkeeping runs, with streams, peer memory and
kernels replaced by host stand-ins."""
import contextlib
import pickle

import pytest
import torch
import torch.distributed as dist


class _Stream:
    def __init__(self, *a, **k):
        pass

    def wait_event(self, e):
        pass

    wait_stream = wait_event


class _Event:
    landed = False

    def record(self, stream=None):
        pass

    def query(self):
        return _Event.landed


class _Ops:
    """One rank: the scattered product leaves its values in slot memory, the sum of the slots reads them back."""

    def __init__(self):
        self.slots, self.next = {}, 1 << 20

    def peer_alloc(self, nbytes, device):
        self.next += 1 << 24
        return self.next, b""

    def gemm_mxfp4_tn_scatter(self, a, a_sf, b, b_sf, dst, rpo, alpha, mask=None, had_scale=None):
        self.slots[dst[0]] = a.clone()

    def shard_reduce(self, ptr, world, elems, scale, out):
        out.copy_(self.slots[ptr])

    def raise_on_fault(self, what):
        pass


@pytest.fixture
def sink(monkeypatch):
    from quartet_b200 import clip, ops
    from quartet_b200.shard import PeerWgradScatter

    def gather(out, obj, group=None):
        out[0] = obj

    for name, value in (("Stream", _Stream), ("Event", _Event), ("current_stream", lambda d=None: _Stream()), ("stream", lambda s: contextlib.nullcontext())):
        monkeypatch.setattr(torch.cuda, name, value)
    for name, value in (("get_world_size", lambda g=None: 1), ("get_rank", lambda g=None: 0), ("get_backend", lambda g=None: "nccl"), ("is_initialized", lambda: True),
                        ("all_reduce", lambda t, op=None, group=None: None), ("all_gather_object", gather)):
        monkeypatch.setattr(dist, name, value)
    monkeypatch.setattr(_Event, "landed", False)
    monkeypatch.setattr(ops, "grad_norm", lambda ts, kind=2.0, total=False: torch.cat([t.double().reshape(-1) for t in ts]).square().sum().reshape(1))

    def scale(ts, max_norm, kind=2.0, out=None, total=None):
        n = total[0].sqrt()
        for t in ts:
            t.mul_(float((max_norm / (n + 1e-6)).clamp(max=1.0)))
        return n.float()

    monkeypatch.setattr(ops, "clip_grads", scale)
    s = PeerWgradScatter(device="cpu")
    s.ops = _Ops()
    s.clip = clip.clip_grad_norm_
    return s


def _weight():
    return torch.nn.Parameter(torch.zeros(256, 256))


def _backward(sink, weight, value):
    sink.wgrad(weight, torch.full((256, 256), value), None, None, None, 1.0, None, 1.0)


def test_a_shard_still_in_flight_is_refused(sink):
    w, v = _weight(), _weight()
    _backward(sink, w, 1.0)
    with pytest.raises(RuntimeError, match=r"wait\(\)"):
        sink.clip([w], 1.0)
    sink.wait()
    assert abs(sink.clip([w], 1.0).item() - 256.0) < 1e-3
    assert abs(w.grad_shard[0, 0].item() - 1 / 256) < 1e-7
    # the next step: the shard found there is the last step's, whose clipping would leave the new one as it is
    _backward(sink, w, 2.0)
    old = w.grad_shard.clone()
    with pytest.raises(RuntimeError, match=r"wait\(\)"):
        sink.clip([w], 1.0)
    assert torch.equal(w.grad_shard, old)
    # whether an exchange happens to have landed differs from rank to rank: the answer may not
    _Event.landed = True
    _backward(sink, v, 2.0)
    with pytest.raises(RuntimeError, match=r"wait\(\)"):
        sink.clip([w], 1.0)
    sink.wait()
    assert abs(sink.clip([w, v], 1.0).item() - 512.0 * 2 ** 0.5) < 1e-2


def test_a_shard_of_an_earlier_step_does_not_count(sink):
    w, v = _weight(), _weight()
    _backward(sink, w, 3.0)
    _backward(sink, v, 4.0)
    sink.wait()
    assert abs(sink.clip([w, v], 1.0).item() - 256.0 * 5) < 1e-2
    _backward(sink, w, 3.0)                                   # v takes no part in this step
    sink.wait()
    kept = v.grad_shard.clone()
    assert abs(sink.clip([w, v], 1.0).item() - 256.0 * 3) < 1e-2
    assert torch.equal(v.grad_shard, kept)
    assert abs(sink.clip([w, v], 1e6).item() - 1.0) < 1e-3    # a second look in the same step counts what the first did
    _backward(sink, v, 4.0)
    sink.wait()
    assert abs(sink.clip([w, v], 1.0).item() - 256.0 * 4) < 1e-2


def test_groups_of_one_step_are_clipped_one_after_the_other(sink):
    w, v = _weight(), _weight()
    for value in (3.0, 5.0):
        _backward(sink, w, value)
        _backward(sink, v, 2 * value)
        sink.wait()
        assert abs(sink.clip([w], 1.0).item() - 256.0 * value) < 1e-2
        assert abs(sink.clip([v], 1.0).item() - 512.0 * value) < 1e-2
    # one that was not clipped yet counts, whatever else was exchanged since
    _backward(sink, w, 1.0)
    _backward(sink, v, 1.0)
    sink.wait()
    sink.clip([w], 1.0)
    _backward(sink, w, 1.0)
    sink.wait()
    assert abs(sink.clip([v], 1.0).item() - 256.0) < 1e-2


def test_a_weight_with_a_shard_can_be_pickled(sink):
    w = _weight()
    _backward(sink, w, 1.0)
    sink.wait()
    assert torch.equal(pickle.loads(pickle.dumps(w)).grad_shard, w.grad_shard)
