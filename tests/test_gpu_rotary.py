"""Rotary positions against the rotation in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import rotary

    return rotary


def turn(x, pos, inv_freq, scale, interleaved, sign=1.0):
    """(rotation in 64 bits, magnitudes that its error bound is relative to) of x [b, t, h, d]"""
    x = x.double().cpu()
    a = sign * pos.double().cpu()[..., None, None] * inv_freq.cpu()
    c, s = a.cos() * scale, a.sin() * scale
    r = 2 * inv_freq.numel()
    i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y, m = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    m[..., i] = m[..., j] = (x[..., i].abs() + x[..., j].abs()) * abs(scale)
    return y, m


def check(got, want, m):
    """cos and sin are off by at most 2^-22 (sincospi one ulp, the correction, the scale: four roundings at 1), the two products and the
    sum add 2^-23 of the magnitudes; then half a step of the type."""
    err = (got.cpu().double() - want).abs()
    lim = (2.0 ** -22 + 2.0 ** -23) * m
    lim = lim + (torch.finfo(got.dtype).eps / 2) * (want.abs() + lim) + 1e-40
    lim = torch.where(m == 0, torch.zeros_like(lim), lim)  # values that are only copied
    assert bool((err <= lim).all()), (err / lim.clamp_min(1e-45)).max().item()


@pytest.mark.parametrize("b,t,hq,hk,d,rot", [(1, 1, 1, 1, 2, 2), (2, 1, 32, 8, 128, 128), (1, 5, 3, 1, 96, 64), (3, 17, 5, 5, 128, 128), (2, 33, 4, 2, 80, 20),
                                             (1, 130, 2, 1, 100, 50), (2, 7, 3, 3, 7, 6), (1, 3, 2, 2, 512, 512), (1, 4, 9, 3, 256, 64), (2, 40, 3, 2, 72, 72), (1, 50, 2, 2, 68, 36), (3, 9, 4, 1, 66, 66)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_apply_and_gradient(R, b, t, hq, hk, d, rot, dtype, interleaved):
    g = torch.Generator().manual_seed(b + t + d)
    q, k = (torch.randn(b, t, h, d, generator=g).to(dtype).cuda().requires_grad_() for h in (hq, hk))
    inv, _ = R.rotary_frequencies(rot, device="cuda")
    pos = torch.randint(-5, 1 << 20, (b, t), generator=g)
    for p in (pos, pos[0].to(torch.int32)):
        yq, yk = R.apply_rotary(q, k, inv, p.cuda(), interleaved=interleaved, scale=1.25)
        gq, gk = (torch.randn(z.shape, generator=g).to(dtype).cuda() for z in (yq, yk))
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
        for x, y, e, dx in ((q, yq, gq, dq), (k, yk, gk, dk)):
            check(y.detach(), *turn(x.detach(), p, inv, 1.25, interleaved))
            check(dx, *turn(e, p, inv, 1.25, interleaved, -1.0))


@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hk,d,rot,t", [(5, 5, 128, 128, 9), (8, 2, 64, 32, 33), (3, 1, 36, 12, 5), (2, 2, 20, 20, 1)])
def test_packed_projection_and_gradient(R, head_major, dtype, hq, hk, d, rot, t):
    b = 2
    g = torch.Generator().manual_seed(d + t)
    qkv = torch.randn(b, t, (hq + 2 * hk) * d, generator=g).to(dtype).cuda().requires_grad_()
    inv, _ = R.rotary_frequencies(rot, device="cuda")
    outs = R.rotary_qkv(qkv, hq, hk, inv, offset=1000, interleaved=False, head_major=head_major)
    pos = 1000 + torch.arange(t)
    parts = [z.detach().unflatten(-1, (-1, d)) for z in qkv.split([hq * d, hk * d, hk * d], -1)]
    view = (lambda z: z.transpose(1, 2)) if head_major else (lambda z: z)
    for i, (z, src) in enumerate(zip(outs, parts)):
        assert z.is_contiguous()
        if i < 2:
            check(view(z.detach()), *turn(src, pos, inv, 1.0, False))
        else:
            assert torch.equal(view(z.detach()), src)
    gs = [torch.randn(z.shape, generator=g).to(dtype).cuda() for z in outs]
    (dqkv,) = torch.autograd.grad(outs, (qkv,), gs, retain_graph=True)
    for i, (dz, e) in enumerate(zip(dqkv.split([hq * d, hk * d, hk * d], -1), gs)):
        if i < 2:
            check(dz.unflatten(-1, (-1, d)), *turn(view(e), pos, inv, 1.0, False, -1.0))
        else:
            assert torch.equal(dz.unflatten(-1, (-1, d)), view(e))
    # gradients that are expanded, transposed, or absent
    (a,) = torch.autograd.grad(outs[0].sum(), (qkv,), retain_graph=True)
    ones = torch.ones(b, t, hq, d)
    check(a[..., :hq * d].unflatten(-1, (-1, d)), *turn(ones, pos, inv, 1.0, False, -1.0))
    assert bool((a[..., hq * d:] == 0).all())


def test_gradient_against_differences(R):
    """The rotation is linear: the difference of two forwards along a direction is the gradient's product with it."""
    g = torch.Generator().manual_seed(3)
    q, dv, e = (torch.randn(2, 9, 3, 64, generator=g).cuda() for _ in range(3))
    inv, _ = R.rotary_frequencies(64, device="cuda")
    q.requires_grad_()
    y = R.apply_rotary(q, None, inv, offset=70000)[0]
    (dx,) = torch.autograd.grad(y, (q,), e)
    with torch.no_grad():
        diff = (R.apply_rotary(q + dv, None, inv, offset=70000)[0].double() - y.double()) * e.double()
    along = (dx.double() * dv.double()).sum()
    # each of the 3456 values of a forward is off by at most 2^-21 of magnitudes up to 8, and q + dv by 2^-24 of itself
    assert abs((diff.sum() - along).item()) < q.numel() * 3 * 8 * 4 * 2.0 ** -21


def test_views_streams_positions_and_empty(R):
    inv, _ = R.rotary_frequencies(64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(2, 11, 3 * 4 * 64, generator=g, device="cuda", dtype=torch.bfloat16)
    q, k, _ = (z.unflatten(-1, (4, 64)) for z in base.split(4 * 64, -1))            # slices of a packed projection
    want = [R.apply_rotary(z.contiguous(), None, inv)[0] for z in (q, k)]
    got = R.apply_rotary(q, k, inv)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hm = q.transpose(1, 2).contiguous().transpose(1, 2)                               # head-major memory
    y, none = R.apply_rotary(hm, None, inv)
    assert none is None and torch.equal(y, want[0]) and y.stride() == hm.stride()
    odd = torch.empty(2 * 11 * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 11, 4, 64).copy_(q)   # not 16-byte aligned
    assert torch.equal(R.apply_rotary(odd, None, inv)[0], want[0])
    assert torch.equal(R.apply_rotary(q[:, :, :1].expand(2, 11, 4, 64), None, inv)[0][:, :, 2], want[0][:, :, 0])
    inner = torch.empty(2, 11, 64, 4, device="cuda", dtype=torch.bfloat16).transpose(2, 3).copy_(q)               # heads innermost
    assert torch.equal(R.apply_rotary(inner, None, inv)[0], want[0])
    pos = torch.arange(11, device="cuda")
    for p in (pos, pos.int(), pos.expand(2, 11), torch.stack([pos, pos], -1)[:, 0], pos.repeat(2, 1).T.contiguous().T):
        assert torch.equal(R.apply_rotary(q, None, inv, p)[0], want[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = R.apply_rotary(q, None, inv)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(z, want[0])
    for shape in ((0, 11, 4, 64), (2, 0, 4, 64)):
        assert R.apply_rotary(torch.empty(shape, device="cuda"), None, inv)[0].shape == shape
    assert [z.shape for z in R.rotary_qkv(torch.empty(2, 0, 12 * 64, device="cuda"), 4, 4, inv)] == [(2, 4, 0, 64)] * 3
    # in place, through the low-level call
    from quartet_b200 import ops

    x = q.contiguous()
    ops.rotary([(x, x, True)], inv)
    assert torch.equal(x, want[0])


def test_captured_and_compiled(R):
    inv, _ = R.rotary_frequencies(64, device="cuda")
    qkv = torch.randn(2, 16, 8 * 64, device="cuda", requires_grad=True)
    gs = [torch.randn(2, h, 16, 64, device="cuda") for h in (4, 2, 2)]

    def step(z):
        outs = R.rotary_qkv(z, 4, 2, inv)
        return (*outs, *torch.autograd.grad(outs, (z,), gs))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(qkv)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(qkv)
    with torch.no_grad():
        qkv.copy_(torch.randn_like(qkv))
    graph.replay()
    want = step(qkv)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    comp = torch.compile(lambda z: R.rotary_qkv(z, 4, 2, inv), fullgraph=True)
    got = comp(qkv)
    assert all(torch.equal(a, b) for a, b in zip((*got, *torch.autograd.grad(got, (qkv,), gs)), want))
    q = torch.randn(1, 5, 3, 64, device="cuda", requires_grad=True)
    y = R.apply_rotary(q, None, inv)[0]
    z = torch.compile(lambda v: R.apply_rotary(v, None, inv)[0], fullgraph=True)(q)
    e = torch.randn_like(y)
    assert torch.equal(y, z) and torch.equal(*(torch.autograd.grad(v, (q,), e)[0] for v in (y, z)))


def test_refusals(R):
    inv, _ = R.rotary_frequencies(64, device="cuda")
    q = torch.randn(2, 3, 4, 64, device="cuda")
    bad = [lambda: R.apply_rotary(q.half(), None, inv), lambda: R.apply_rotary(q, q.bfloat16(), inv), lambda: R.apply_rotary(q.cpu(), None, inv),
           lambda: R.apply_rotary(q, None, inv.float()), lambda: R.apply_rotary(q, None, inv.cpu()), lambda: R.apply_rotary(q[..., :32], None, inv),
           lambda: R.apply_rotary(q, None, inv, torch.arange(4, device="cuda")), lambda: R.apply_rotary(q, None, inv, torch.arange(3.0, device="cuda")),
           lambda: R.apply_rotary(q[0], None, inv), lambda: R.rotary_qkv(q, 2, 1, inv), lambda: R.rotary_qkv(q.flatten(2), 3, 1, inv),
           lambda: R.apply_rotary(q, None, inv, torch.arange(3)), lambda: R.apply_rotary(q, q[:, :2], inv)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_gradient_of_the_gradient(R):
    """apply_rotary's gradient is itself a rotation, so a second derivative goes through; the packed form refuses one."""
    inv, _ = R.rotary_frequencies(16, device="cuda")
    q = torch.randn(1, 4, 2, 16, device="cuda", requires_grad=True)
    e = torch.randn(1, 4, 2, 16, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(R.apply_rotary(q, None, inv, scale=1.5)[0], (q,), e, create_graph=True)
    (de,) = torch.autograd.grad(dx, (e,), torch.ones_like(dx))
    check(de, *turn(torch.ones_like(dx), torch.arange(4), inv, 1.5, True))
    qkv = torch.randn(1, 4, 3 * 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(R.rotary_qkv(qkv, 1, 1, inv)[0].sum(), (qkv,), create_graph=True)


def test_destinations_that_share_memory_are_refused(R):
    from quartet_b200 import ops

    inv, _ = R.rotary_frequencies(64, device="cuda")
    buf = torch.randn(2, 5, 12, 64, device="cuda")
    q, k = buf[:, :, :4], buf[:, :, 4:8]
    fresh = torch.empty(2, 5, 4, 64, device="cuda")
    want = R.apply_rotary(q, None, inv)[0]
    bad = [[(q, buf[:, :, 1:5], True)], [(q, fresh[:, :, :1].expand(2, 5, 4, 64), True)], [(q, fresh, True), (k, fresh, True)], [(q, k, True), (k, fresh, True)],
           [(q, buf.view(-1)[1:2 * 5 * 4 * 64 + 1].view(2, 5, 4, 64), True)]]
    kept = buf.clone()
    for segments in bad:
        with pytest.raises(ValueError, match="share|one address"):
            ops.rotary(segments, inv)
    assert torch.equal(buf, kept)
    ops.rotary([(q, buf[:, :, 8:], True), (k, k, True)], inv)                # disjoint parts of one buffer, one of them in place
    assert torch.equal(buf[:, :, 8:], want) and torch.equal(k, R.apply_rotary(kept[:, :, 4:8], None, inv)[0])
