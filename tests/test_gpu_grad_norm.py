"""The norm over many tensors and clipping by it, against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import ops

    return ops


def norm64(ts, inf=False):
    if inf:
        return max((t.detach().double().abs().max().item() for t in ts if t.numel()), default=0.0)
    return math.sqrt(math.fsum(t.detach().double().square().sum().item() for t in ts))


def check(ops, ts, max_norm, outs=None, inf=False):
    before = [t.clone() for t in ts]
    want = norm64(ts, inf)
    n = ops.grad_norm(ts, math.inf if inf else 2.0)
    # One rounding to fp32 (2^-24).  Sums are in 64 bits (their error is far below it), but four squares of bf16 values are added in 32
    # before: the square is exact, a fused add and an add round the sum of squares by 2^-24 each, which is 2^-24 of its root.
    bf16 = any(t.dtype == torch.bfloat16 for t in ts)
    assert abs(n.item() - want) <= 2.0 ** -24 * (2 if bf16 and not inf else 1) * want * (1 + 1e-6)
    m = ops.clip_grads(ts, max_norm, math.inf if inf else 2.0, out=outs)
    assert m.dtype == torch.float32 and torch.equal(m, n)
    c = min(1.0, max_norm / (want + 1e-6))
    for b, o in zip(before, outs if outs is not None else ts):
        w = b.double() * c
        # the factor and the product are rounded to fp32, the result to its type
        lim = w.abs() * (2.0 ** -23 + 2.0 ** -47) + 2.0 ** -149
        lim = lim + (torch.finfo(o.dtype).eps / 2) * (w.abs() + lim) if o.dtype == torch.bfloat16 else lim
        assert bool(((o.double() - w).abs() <= lim).all())
    if outs is not None:
        assert all(torch.equal(a, b) for a, b in zip(ts, before))


SETS = {"one": [(1,)], "odd": [(1,), (3,), (5, 7), (8191,), (8192,), (8193,), (100, 129)], "mixed": [(640,), (1920, 640), (0,), (33, 3, 5), (16,), (2, 0)],
        "many": [(i % 37 + 1,) for i in range(70)], "more": [(i % 11 + 1, 3) for i in range(1700)]}


@pytest.mark.parametrize("name", SETS)
@pytest.mark.parametrize("kind", ["f32", "bf16", "both"])
@pytest.mark.parametrize("inf", [False, True])
def test_norm_and_clip(ops, name, kind, inf):
    g = torch.Generator(device="cuda").manual_seed(len(name))
    pick = lambda i: torch.bfloat16 if kind == "bf16" or (kind == "both" and i % 2) else torch.float32  # noqa: E731
    make = lambda: [(torch.randn(s, generator=g, device="cuda") * 10.0 ** (i % 5 - 3)).to(pick(i)) for i, s in enumerate(SETS[name])]  # noqa: E731
    for max_norm in (0.01, 1e9, 0.0):
        check(ops, make(), max_norm, inf=inf)
    ts = make()
    check(ops, ts, 0.25, [torch.empty_like(t, dtype=torch.float32) for t in ts], inf)
    check(ops, ts, 0.25, [torch.empty_like(t, dtype=torch.bfloat16) for t in ts], inf)
    check(ops, ts, 1e9, [torch.empty_like(t, dtype=torch.float32) for t in ts], inf)
    a, b = ops.grad_norm(ts), ops.grad_norm(ts)
    assert torch.equal(a, b)


def test_large_and_unaligned_and_reordered(ops):
    g = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn(5_000_001, generator=g, device="cuda")
    ts = [flat[1:3_000_000], flat[3_000_001:5_000_001].view(1000, 2000).t(),
          torch.randn(4, 6, 8, generator=g, device="cuda").permute(2, 0, 1), torch.randn(999, generator=g, device="cuda").bfloat16()[1:]]
    check(ops, ts, 1.0, [torch.empty_like(t) for t in ts])
    check(ops, ts, 1.0)
    assert flat[0].abs() > 0 and not torch.equal(flat[1:3], flat[3:5])


def test_squares_that_leave_fp32(ops):
    for dt, room in ((torch.float32, 1), (torch.bfloat16, 2)):
        for s in (1e30, 1e-30, 1e-40, 1e-9, 3e18, 1e19):
            ts = [torch.full((1000,), s, device="cuda", dtype=dt), torch.full((3,), s, device="cuda", dtype=dt), torch.zeros(64, device="cuda", dtype=dt)]
            ts[2][5] = s
            n = ops.grad_norm(ts).item()
            want = norm64(ts)
            assert abs(n - want) <= max(room * 2.0 ** -24 * want * 1.0001, 2.0 ** -150)
    assert abs(ops.clip_grads([torch.full((4,), 3e38, device="cuda")], 1.0).item()) == math.inf  # the norm itself is past fp32 ...
    t = torch.full((4,), 3e38, device="cuda")
    ops.clip_grads([t], 1.0)
    assert torch.allclose(t, torch.full_like(t, 0.5))                                             # ... the clipping is not


@pytest.mark.parametrize("inf", [False, True])
def test_values_that_are_not_finite(ops, inf):
    kind = math.inf if inf else 2.0
    for bad in (math.inf, -math.inf, math.nan):
        for dt in (torch.float32, torch.bfloat16):
            ts = [torch.ones(5000, device="cuda", dtype=dt), torch.ones(7, device="cuda", dtype=dt)]
            ts[0][4321] = bad
            ref = [t.float().cpu().clone() for t in ts]
            n = ops.clip_grads(ts, 1.0, kind)
            if math.isnan(bad):
                assert math.isnan(n.item()) and all(bool(torch.isnan(t).all()) for t in ts)
            else:
                assert n.item() == math.inf
                assert all(torch.equal(t.float().cpu().nan_to_num(nan=9.0), (r * 0.0).nan_to_num(nan=9.0)) for t, r in zip(ts, ref))


def test_agrees_with_torch_on_parameters_and_shards(ops, monkeypatch):
    from quartet_b200 import clip

    torch.manual_seed(0)
    a, b = (torch.nn.Sequential(torch.nn.Linear(64, 300), torch.nn.Linear(300, 7)).cuda() for _ in range(2))
    for p, q in zip(a.parameters(), b.parameters()):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    list(a.parameters())[1].grad = list(b.parameters())[1].grad = None
    n, m = clip.clip_grad_norm_(a.parameters(), 0.7), torch.nn.utils.clip_grad_norm_([q for q in b.parameters() if q.grad is not None], 0.7)
    assert abs(n.item() - m.item()) < 1e-6 * m.item()
    assert all(torch.allclose(p.grad, q.grad, rtol=1e-6, atol=0) for p, q in zip(a.parameters(), b.parameters()) if p.grad is not None)
    # shards: the sum over ranks is what clips (two ranks that hold equal shards, by a stand-in for the collective)
    p, q = torch.nn.Parameter(torch.zeros(300, 5, device="cuda")), torch.nn.Parameter(torch.zeros(9, device="cuda"))
    p.grad_shard, q.grad = torch.randn(150, 5, device="cuda"), torch.randn(9, device="cuda")
    want = math.sqrt(2 * norm64([p.grad_shard]) ** 2 + norm64([q.grad]) ** 2)
    before = p.grad_shard.clone()
    monkeypatch.setattr(clip.dist, "is_initialized", lambda: True)
    monkeypatch.setattr(clip.dist, "all_reduce", lambda t, op=None, group=None: t.mul_(2))
    n = clip.clip_grad_norm_([p, q], 0.5)
    assert abs(n.item() - want) <= 2.0 ** -24 * want * 1.0001
    assert torch.allclose(p.grad_shard, before * (0.5 / (want + 1e-6)), rtol=2.0 ** -22, atol=0)
    q.grad[0] = math.nan
    kept = p.grad_shard.clone()
    with pytest.raises(RuntimeError):
        clip.clip_grad_norm_([p, q], 0.5, error_if_nonfinite=True)
    assert torch.equal(p.grad_shard, kept)
    assert clip.clip_grad_norm_([torch.nn.Parameter(torch.zeros(1))], 1.0).item() == 0


def test_captured_on_another_stream(ops):
    ts = [torch.randn(1000, 33, device="cuda"), torch.randn(5, device="cuda").bfloat16()]
    outs = [torch.empty_like(t) for t in ts]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.clip_grads(ts, 1.0, out=outs)
    torch.cuda.current_stream().wait_stream(s)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        n = ops.clip_grads(ts, 1.0, out=outs)
    with torch.cuda.graph(second):
        k = ops.grad_norm(ts[:1])
    ts[0].mul_(3.0)
    first.replay(), second.replay()
    assert torch.equal(n, ops.grad_norm(ts)) and torch.equal(k, ops.grad_norm(ts[:1]))
    assert torch.allclose(outs[0], ts[0] / n, rtol=1e-5)


def test_refusals(ops):
    x = torch.randn(64, 64, device="cuda")
    bad = [lambda: ops.grad_norm([]), lambda: ops.grad_norm([x.cpu()]), lambda: ops.grad_norm([x.half()]), lambda: ops.grad_norm([x[:, ::2]]),
           lambda: ops.grad_norm([x], 3.0), lambda: ops.clip_grads([x], -1.0), lambda: ops.clip_grads([x], math.nan), lambda: ops.clip_grads([x, x], 1.0),
           lambda: ops.clip_grads([x[:10], x[5:20]], 1.0), lambda: ops.clip_grads([x], 1.0, out=[]), lambda: ops.clip_grads([x], 1.0, out=[x[:1]]),
           lambda: ops.clip_grads([x.view(-1)[:100]], 1.0, out=[x.view(-1)[4:104]]), lambda: ops.clip_grads([x], 1.0, out=[x.t()]),
           lambda: ops.clip_grads([x], 1.0, total=torch.ones(1, device="cuda"))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert ops.grad_norm([x, x]).item() > 0   # the same tensor twice counts twice in a norm; clipped twice it is refused


def test_clipping_is_seen_by_a_graph_that_saved_a_gradient(ops):
    """As after any change in place: the backward of a graph that saved the gradient raises, and does not use the scaled values."""
    w = torch.full((300,), 3.0, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((w * w).sum(), w, create_graph=True)
    kept = g.detach()
    loss = (kept * w).sum()
    ops.clip_grads([kept], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    out, kept = torch.empty(300, device="cuda"), torch.ones(300, device="cuda")
    version, before = out._version, kept._version
    ops.clip_grads([kept], 1.0, out=[out])
    assert out._version > version and kept._version == before
