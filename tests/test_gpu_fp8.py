"""The 8-bit block-scaled linear layer: quantizers bit for bit, the product and the layer within the bounds of their arithmetic."""
import pytest
import torch

from tests import fp8_oracle as fo

pytestmark = pytest.mark.gpu
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import ops

    return ops


def _x(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    x.view(-1)[:: 53] *= 30.0
    if rows > 2:
        x[rows // 2] = 0.0                                     # a row of empty blocks
        x[0, : min(cols, 128)] = 0.0
        x[0, 0] = 1.75 * 2.0 ** 5                              # MAX times a power of two: the scale is exact
        x[1, :1] = 1e-38
    return x.to(dtype)


def _codes(c):
    return c.cpu().float().double()


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (2, 127), (3, 640), (127, 129), (128, 128), (129, 257), (200, 1000), (384, 136), (33, 4100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_quantizer_equals_the_definition(ops, rows, cols, dtype, square, fmt):
    x = _x(rows, cols, dtype, rows * 7 + cols)
    got = ops.quant_fp8(x.cuda(), fmt, square=square, transpose=True)
    for (codes, sf), src in (((got[0], got[1]), x), ((got[2], got[3]), x.T)):
        want, e = fo.quantize(src, fmt, square)
        assert codes.dtype == fmt and codes.shape == want.shape
        assert torch.equal(_codes(codes), want)
        assert torch.equal(sf.cpu(), fo.blocked(e, src.shape[0]))
        v = ops.dequant_fp8(codes, sf, src.shape[1])
        assert torch.equal(v.cpu().double(), fo.values(src, fmt, square).float().double())
    only = ops.quant_fp8(x.cuda(), fmt, square=square)
    assert torch.equal(only[0].view(torch.uint8), got[0].view(torch.uint8)) and torch.equal(only[1], got[1]) and only[2] is None
    only = ops.quant_fp8(x.cuda(), fmt, square=square, rows=False, transpose=True)
    assert torch.equal(only[2].view(torch.uint8), got[2].view(torch.uint8)) and torch.equal(only[3], got[3]) and only[0] is None


@pytest.mark.parametrize("rows,cols", [(2600, 2903), (2600, 2902), (2611, 2900), (300, 121), (1, 9)])
@pytest.mark.parametrize("offset", [0, 1, 2, 8])
@pytest.mark.parametrize("square", [False, True])
def test_quantizer_reads_rows_wherever_they_start(ops, rows, cols, offset, square):
    """Rows that start on any even byte, between values that are not numbers, in more tiles than CTAs: as from a padded copy with aligned rows."""
    flat = torch.full((rows * cols + 64,), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = flat[offset:offset + rows * cols].view(rows, cols)
    x.copy_(_x(rows, cols, torch.bfloat16, rows + cols))
    padded = torch.zeros(rows, -(-cols // 128) * 128, dtype=torch.bfloat16, device="cuda")
    padded[:, :cols] = x
    want, got = (ops.quant_fp8(t, E4M3, square=square, transpose=True) for t in (padded, x))
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    assert torch.equal(got[2].view(torch.uint8), want[2][:cols].view(torch.uint8))
    # [column blocks, row blocks, 32, 4, 4]: the bytes of columns past the last one are zeros, where the padded copy has those of columns of zeros
    blocks = want[3].view(-1, -(-rows // 128), 32, 4, 4).clone()
    if cols % 128:
        blocks[-1] *= (torch.arange(128).view(4, 32).T < cols % 128).cuda()[None, :, :, None]
    assert torch.equal(got[3].view_as(blocks), blocks)
    only = ops.quant_fp8(x, E4M3, square=square)
    assert torch.equal(only[0].view(torch.uint8), got[0].view(torch.uint8)) and torch.equal(only[1], got[1])
    only = ops.quant_fp8(x, E4M3, square=square, rows=False, transpose=True)
    assert torch.equal(only[2].view(torch.uint8), got[2].view(torch.uint8)) and torch.equal(only[3], got[3])


def test_quantizer_rounds_every_code_boundary_to_even(ops):
    """Every value of the formats and every midpoint between two, in a block whose scale is 1."""
    for fmt, top in ((E4M3, 448.0), (E5M2, 57344.0)):
        all8 = torch.arange(0, 256, dtype=torch.uint8).view(fmt).float()
        v = all8[torch.isfinite(all8)].unique()
        mid = torch.cat([v, (v[1:] + v[:-1]) / 2, -v])
        n = -(-mid.numel() // 127)
        x = torch.full((n, 128), top)
        x[:, 1:] = torch.nn.functional.pad(mid, (0, n * 127 - mid.numel())).view(n, 127)
        codes, sf, _, _ = ops.quant_fp8(x.cuda(), fmt)
        want, e = fo.quantize(x, fmt)
        assert bool((e == 0).all()) and torch.equal(sf.cpu(), fo.blocked(e, n))
        assert torch.equal(_codes(codes), want)


def test_extremes_and_blocks_that_are_not_finite(ops):
    x = torch.zeros(6, 256)
    x[0, 3], x[1, 3], x[2, 5], x[3, 200] = float("inf"), float("nan"), 3.4e38, float("-inf")
    x[4, :4] = torch.tensor([1e-45, 1e-40, -2e-39, 0.0])
    x[5, 0], x[5, 1] = 1e30, 1e-30
    for fmt in (E4M3, E5M2):
        codes, sf, codes_t, sf_t = ops.quant_fp8(x.cuda(), fmt, transpose=True)
        v = ops.dequant_fp8(codes, sf, 256).cpu()
        bad = torch.zeros(6, 2, dtype=torch.bool)
        bad[0, 0] = bad[1, 0] = bad[3, 1] = True
        assert torch.equal(torch.isnan(v).view(6, 2, 128).all(2), bad) and torch.equal(torch.isnan(v).view(6, 2, 128).any(2), bad)
        ok = x.clone()
        ok[0, :128] = ok[1, :128] = 0
        ok[3, 128:] = 0
        want = fo.values(ok, fmt)
        good = ~bad.repeat_interleave(128, 1)
        assert torch.equal(v.double()[good], want.float().double()[good])
        vt = ops.dequant_fp8(codes_t, sf_t, 6).cpu()
        assert torch.equal(torch.isnan(vt).any(1), ~torch.isfinite(x).all(0)) and torch.equal(torch.isnan(vt).all(1), ~torch.isfinite(x).all(0))
        # a NaN block reaches exactly the results it belongs to
        w = torch.ones(128, 256, device="cuda")
        y = ops.linear_fp8(x.cuda(), *ops.quant_fp8(w, square=True)[:2]).cpu()
        if fmt == E4M3:
            assert torch.equal(torch.isnan(y).all(1), bad.any(1)) and torch.equal(torch.isnan(y).any(1), bad.any(1))


def _bound(absum, K, y, out_dtype):
    """fp32 sums of K exact products, at most 2^-23 of the magnitudes lost at each addition in any order, then the output's rounding."""
    b = K * 2.0 ** -23 * absum
    return b + (torch.finfo(out_dtype).eps / 2) * (y.abs() + b) + 1e-40


def _product(ops, M, N, K, fa=E4M3, fb=E4M3, out_dtype=torch.float32, seed=0, alpha=1.0):
    g = torch.Generator().manual_seed(seed + M + N + K)
    a, b = torch.randn(M, K, generator=g) * 3, torch.randn(N, K, generator=g) * 0.02
    av, bv = fo.values(a, fa), fo.values(b, fb, True)
    (ac, asf, _, _), (bc, bsf, _, _) = ops.quant_fp8(a.cuda(), fa), ops.quant_fp8(b.cuda(), fb, square=True)
    y = ops.gemm_fp8_tn(ac, asf, bc, bsf, alpha, out_dtype)
    want = alpha * (av @ bv.T)
    err = (y.cpu().double() - want).abs()
    lim = _bound(abs(alpha) * (av.abs() @ bv.abs().T), fo.pad128(K), want, out_dtype)
    print(M, N, K, "worst of bound", (err / lim).max().item(), "relative", (err.norm() / want.norm()).item())
    assert y.dtype == out_dtype and y.shape == (M, N)
    assert bool((err <= lim).all())
    assert ops.device_status() == 0


SIZES = [(1, 1, 1), (1, 128, 128), (1, 257, 640), (5, 130, 127), (16, 512, 1024), (17, 96, 384), (33, 640, 129), (64, 1000, 512), (65, 264, 2048), (100, 100, 100),
         (128, 128, 4096), (129, 255, 640), (250, 1024, 300), (256, 256, 256), (257, 513, 1152), (384, 128, 1408), (511, 264, 520), (1021, 640, 640),
         (1024, 2051, 256), (2048, 520, 384),
         (65, 4099, 128), (96, 4096, 640), (200, 2300, 256), (255, 3000, 384), (300, 257, 8192), (2000, 256, 128)]


@pytest.mark.parametrize("mnk", SIZES)
def test_product_within_its_bound(ops, mnk):
    _product(ops, *mnk)
    _product(ops, *mnk, out_dtype=torch.bfloat16, alpha=0.375)


@pytest.mark.parametrize("mnk", [(130, 4010, 8192), (257, 1999, 8192),                      # 256 rows of A in a CTA, one and two blocks of them
                                 (300, 11003, 640), (66, 19000, 256),                       # more tiles than SMs, two to an SM
                                 (100, 640, 4096), (140, 1200, 2000), (129, 4096, 1000),    # clusters of eight, four and two
                                 (2300, 4101, 256), (2300, 4100, 140), (60000, 100, 128), (40001, 203, 100), (38000, 64, 128)])  # pairs
def test_product_in_every_form(ops, mnk):
    _product(ops, *mnk)
    _product(ops, *mnk, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("fa,fb", [(E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
def test_product_of_mixed_formats(ops, fa, fb):
    _product(ops, 200, 320, 900, fa, fb)
    _product(ops, 3, 320, 900, fa, fb)
    _product(ops, 512, 768, 900, fa, fb)


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 40, 300])
@pytest.mark.parametrize("K,N", [(1, 1), (127, 130), (640, 515), (1000, 64), (4096, 300), (2300, 1025)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_packed_weight_equals_quantizer_then_product(ops, M, K, N, dtype):
    """The one-call form and, for few rows, the one-launch form: the same codes, so the same sums up to their order."""
    x = _x(M, K, dtype, M + K)
    if K > 300:
        x[0, 299] = float("nan")
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(N)) * 0.02
    wc, ws = ops.quant_fp8(w.cuda(), square=True)[:2]
    y = ops.linear_fp8(x.cuda(), wc, ws)
    y32 = ops.linear_fp8(x.cuda(), wc, ws, torch.float32)
    assert y.dtype == dtype and y.shape == (M, N)
    keep = x.clone()
    if K > 300:
        assert bool(torch.isnan(y[0]).all())
        keep[0] = 0
    xv, wv = fo.values(keep, E4M3), fo.values(w, E4M3, True)
    want, s = xv @ wv.T, xv.abs() @ wv.abs().T
    rows = slice(1, None) if K > 300 else slice(None)
    for got, dt in ((y, dtype), (y32, torch.float32)):
        assert bool(((got.cpu().double() - want).abs() <= _bound(s, fo.pad128(K), want, dt))[rows].all())
    assert ops.device_status() == 0


def test_product_takes_a_scale_for_every_32(ops):
    """The product itself reads one scale byte per 32 values: scales that differ inside a block of 128 count."""
    from oracle import ref_math as rm

    for M, N, K in ((70, 150, 256), (512, 512, 512)):
        g = torch.Generator().manual_seed(M)
        a, b = (torch.randn(n, K, generator=g).to(E4M3) for n in (M, N))
        ae, be = (torch.randint(120, 134, (n, K // 32), generator=g, dtype=torch.uint8) for n in (M, N))
        av, bv = (c.double() * fo.two(e.int() - 127).repeat_interleave(32, 1) for c, e in ((a, ae), (b, be)))
        y = ops.gemm_fp8_tn(a.cuda(), rm.to_blocked(ae).cuda(), b.cuda(), rm.to_blocked(be).cuda(), out_dtype=torch.float32)
        want = av @ bv.T
        assert bool(((y.cpu().double() - want).abs() <= _bound(av.abs() @ bv.abs().T, K, want, torch.float32)).all())


def test_product_leaves_memory_beside_its_result_alone(ops):
    """Rows of D behind the last and columns up to the row pitch keep what they held."""
    from quartet_b200 import _lib

    for M, N, K in ((5, 131, 256), (300, 515, 256), (511, 1003, 128)):
        for dt, code in ((torch.bfloat16, 0), (torch.float32, 1)):
            a, b = torch.randn(M, K, device="cuda"), torch.randn(N, K, device="cuda")
            (ac, asf, _, _), (bc, bsf, _, _) = ops.quant_fp8(a), ops.quant_fp8(b, square=True)
            want = ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=dt)
            buf = torch.full((M + 130, (N + 15) // 8 * 8), 7.0, dtype=dt, device="cuda")
            rc = _lib.load().quartet_gemm_fp8_tn(ops._ptr(ac), ops._ptr(asf), 0, ops._ptr(bc), ops._ptr(bsf), 0, M, N, K, 1.0, ops._ptr(buf), code, buf.shape[1],
                                                 ops._stream())
            assert rc == 0
            assert torch.equal(buf[:M, :N], want) and bool((buf[M:] == 7).all()) and bool((buf[:, N:] == 7).all())


def test_large_products_leave_memory_beside_their_result_alone(ops):
    """As above, where pairs of CTAs store whole 16-byte units and the rest value by value, and where rows are split between CTAs."""
    from quartet_b200 import _lib

    for M, N, K in ((2300, 4101, 128), (2300, 4100, 128), (40001, 199, 128), (40001, 65, 128), (300, 11003, 256), (130, 4010, 8192)):
        for dt, code in ((torch.bfloat16, 0), (torch.float32, 1)):
            a, b = torch.randn(M, K, device="cuda"), torch.randn(N, K, device="cuda")
            (ac, asf, _, _), (bc, bsf, _, _) = ops.quant_fp8(a), ops.quant_fp8(b, square=True)
            want = ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=dt)
            buf = torch.full((M + 130, (N + 15) // 8 * 8), 7.0, dtype=dt, device="cuda")
            rc = _lib.load().quartet_gemm_fp8_tn(ops._ptr(ac), ops._ptr(asf), 0, ops._ptr(bc), ops._ptr(bsf), 0, M, N, K, 1.0, ops._ptr(buf), code, buf.shape[1],
                                                 ops._stream())
            assert rc == 0
            assert torch.equal(buf[:M, :N], want) and bool((buf[M:] == 7).all()) and bool((buf[:, N:] == 7).all())
    assert ops.device_status() == 0


def test_products_repeat_bit_for_bit(ops):
    for M, N, K in ((1, 4096, 4096), (7, 512, 11008), (300, 640, 4096), (1024, 1024, 1024)):
        a, b = torch.randn(M, K, device="cuda"), torch.randn(N, K, device="cuda") * 0.02
        (ac, asf, _, _), (bc, bsf, _, _) = ops.quant_fp8(a), ops.quant_fp8(b, square=True)
        first = ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=torch.float32)
        assert all(torch.equal(first, ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=torch.float32)) for _ in range(5))


@pytest.mark.parametrize("M,K,N", [(65, 64, 300), (128, 256, 5000), (300, 4000, 100), (1000, 700, 900), (2050, 515, 1030), (4096, 640, 1920), (300, 2600, 2600),
                                   (513, 8000, 257), (4100, 100, 4100)])
@pytest.mark.parametrize("gd", [E4M3, E5M2])
def test_both_gradients_equal_each_alone(ops, M, K, N, gd):
    """The two products of a backward pass, which may share a launch, against each by itself (another form may add in another order)."""
    x, w, e = torch.randn(M, K, device="cuda"), torch.randn(N, K, device="cuda") * 0.05, torch.randn(M, N, device="cuda").bfloat16()
    _, saved = ops.fp8_linear_fwd(x, w, True, True, torch.bfloat16)
    both = ops.fp8_linear_bwd(e, saved, K, gd, torch.float32, torch.bfloat16, True, True, True, True)
    dx, _ = ops.fp8_linear_bwd(e, saved, K, gd, torch.float32, torch.bfloat16, True, False, True, True)
    _, dw = ops.fp8_linear_bwd(e, saved, K, gd, torch.float32, torch.bfloat16, False, True, True, True)
    ev, et = (ops.dequant_fp8(c, s, n).double().abs() for c, s, n in ((*ops.quant_fp8(e, gd)[:2], N), (*ops.quant_fp8(e.T.contiguous(), gd)[:2], M)))
    wv, xt = ops.dequant_fp8(*ops.quant_fp8(w, square=True)[:2], K).double().abs(), ops.dequant_fp8(*ops.quant_fp8(x.T.contiguous())[:2], M).double().abs()
    for got, want, absum, k in ((both[0], dx, ev @ wv, N), (both[1], dw, et @ xt.T, M)):
        lim = 2 * fo.pad128(k) * 2.0 ** -23 * absum
        lim = lim + torch.finfo(got.dtype).eps * (want.double().abs() + lim) + 1e-40
        assert bool(((got.double() - want.double()).abs() <= lim).all())
    again = ops.fp8_linear_bwd(e, saved, K, gd, torch.float32, torch.bfloat16, True, True, True, True)
    assert torch.equal(again[0], both[0]) and torch.equal(again[1], both[1]) and ops.device_status() == 0


@pytest.mark.parametrize("M,K,N", [(1, 128, 128), (7, 100, 65), (130, 640, 1000), (256, 384, 512), (513, 257, 640)])
@pytest.mark.parametrize("xd,wd,gd", [(torch.bfloat16, torch.float32, E4M3), (torch.float32, torch.float32, E5M2), (torch.bfloat16, torch.bfloat16, E5M2)])
def test_layer_and_its_gradients(ops, M, K, N, xd, wd, gd):
    from quartet_b200.quantization import fp8_linear

    x, w, e = _x(M, K, xd, 1), (torch.randn(N, K, generator=torch.Generator().manual_seed(2)) * 0.02).to(wd), _x(M, N, xd, 3)
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = fp8_linear(xg, wg, grad_dtype=gd)
    y.backward(e.cuda())
    wants = fo.layer(x, w, e, gd)
    f8 = E4M3
    absx, absw = fo.values(x, f8).abs(), fo.values(w, f8, True).abs()
    abse, abset = fo.values(e, gd).abs(), fo.values(e.T, gd).abs()
    sums = (absx @ absw.T, abse @ absw, abset @ fo.values(x.T, f8).T.abs())
    for name, got, want, s, k, dt in zip(("y", "dx", "dw"), (y.detach(), xg.grad, wg.grad), wants, sums, (K, N, M), (xd, xd, wd)):
        assert got.dtype == dt and got.shape == want.shape, name
        assert bool(((got.cpu().double() - want).abs() <= _bound(s, fo.pad128(k), want, dt)).all()), name


def test_layer_gradient_against_differences(ops):
    """The products are linear in each operand once the operands are on the 8-bit grid: with such inputs (scale 1) a difference of two
    forwards is the gradient's product exactly up to the sums' rounding."""
    from quartet_b200.quantization import fp8_linear

    g = torch.Generator().manual_seed(5)
    M, K, N = 128, 256, 128
    grid = lambda r, c: torch.randint(-8, 9, (r, c), generator=g).float()  # noqa: E731

    def pin(t):  # every block of either orientation holds 448, so that every scale is 1 and small integers are codes
        t[torch.arange(t.shape[0]), torch.arange(t.shape[0]) % 128] = 448.0
        t[:, 128:] = torch.where(torch.arange(t.shape[0])[:, None] % 128 == torch.arange(t.shape[1] - 128)[None] % 128, torch.tensor(448.0), t[:, 128:])
        return t

    x, w, e = pin(grid(M, K)), pin(grid(N, K)), pin(grid(M, N))
    dxv, dwv = grid(M, K), grid(N, K)
    dxv[x == 448], dwv[w == 448] = 0, 0
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    fp8_linear(xg, wg).backward(e.cuda())
    f = lambda a, b: (fp8_linear(a.cuda(), b.cuda()).double() * e.cuda().double()).sum().item()  # noqa: E731
    # x + d and x - d stay on the grid: integers up to 16
    for t, d, grad, call in ((x, dxv, xg.grad, lambda v: f(v, w)), (w, dwv, wg.grad, lambda v: f(x, v))):
        diff = (call(t + d) - call(t - d)) / 2
        along = (grad.double().cpu() * d.double()).sum().item()
        size = (grad.double().cpu().abs() * d.double().abs()).sum().item() + 448.0 * 448 * K
        assert abs(diff - along) <= 2.0 ** -20 * size * 4


def test_layer_shapes_strides_streams_and_empty_batches(ops):
    from quartet_b200.quantization import Fp8Linear, fp8_linear

    torch.manual_seed(0)
    lin = Fp8Linear(200, 77, bias=True).cuda()
    x = torch.randn(4, 3, 200, device="cuda", dtype=torch.bfloat16)
    y = lin(x)
    assert y.shape == (4, 3, 77)
    big = torch.randn(4, 3, 400, device="cuda", dtype=torch.bfloat16)
    big[..., ::2] = x
    assert torch.equal(lin(big[..., ::2]), y)                               # strided input
    assert torch.equal(lin(x.transpose(0, 1)).transpose(0, 1), y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = lin(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, y)
    e = torch.empty(0, 200, device="cuda").requires_grad_()
    out = fp8_linear(e, lin.weight)
    assert out.shape == (0, 77)
    lin.weight.grad = None
    out.sum().backward()
    assert e.grad.shape == (0, 200) and bool((lin.weight.grad == 0).all())
    # a gradient that is expanded, and one of the inputs only
    lin.weight.grad = None
    xr = x.clone().requires_grad_()
    lin(xr).sum().backward()
    assert xr.grad.shape == x.shape and lin.weight.grad.is_contiguous()
    frozen = lin.weight.detach()
    xr.grad = None
    fp8_linear(xr, frozen).sum().backward()
    assert xr.grad is not None
    codes, sf = lin.export_fp8()
    assert torch.allclose(ops.linear_fp8(x, codes, sf).float(), fp8_linear(x, frozen).float(), rtol=2.0 ** -7, atol=1e-5)
    assert ops.linear_fp8(x[:0], codes, sf).shape == (0, 3, 77)
    assert list(lin.state_dict()) == ["weight", "bias"]


def test_layer_without_gradients_keeps_nothing(ops, monkeypatch):
    from quartet_b200.quantization import Fp8Linear

    seen, real = [], ops.fp8_linear_fwd
    monkeypatch.setattr(ops, "fp8_linear_fwd", lambda x, w, need_dx, need_dw, dt: seen.append((need_dx, need_dw)) or real(x, w, need_dx, need_dw, dt))
    lin, x = Fp8Linear(200, 96, device="cuda"), torch.randn(3, 5, 200, device="cuda")
    want = lin(x)
    assert want.requires_grad and seen == [(False, True)]
    with torch.no_grad():
        got = lin(x)
    with torch.inference_mode():
        inf = lin(x)
    lin.requires_grad_(False)
    assert torch.equal(got, want) and torch.equal(inf, want) and torch.equal(lin(x), want) and not got.requires_grad
    assert seen[1:] == [(False, False)] * 3


def test_layer_captured_and_replayed(ops):
    """Forward and backward in one graph, replayed on new inputs; a second graph beside it does not disturb it."""
    from quartet_b200.quantization import fp8_linear

    w = (torch.randn(640, 384, device="cuda") * 0.02).requires_grad_()
    xs = [torch.randn(200, 384, device="cuda").requires_grad_() for _ in range(2)]
    e = torch.randn(200, 640, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            torch.autograd.grad(fp8_linear(x, w), (x, w), e)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fp8_linear(x, w)
            outs.append([y, *torch.autograd.grad(y, (x, w), e)])
        graphs.append(g)
    with torch.no_grad():
        for x in xs:
            x.copy_(torch.randn_like(x))
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for x, got in zip(xs, outs):
        y = fp8_linear(x, w)
        want = [y, *torch.autograd.grad(y, (x, w), e)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layer_compiled_equals_eager(ops):
    from quartet_b200.quantization import Fp8Linear

    torch.manual_seed(1)
    lin = Fp8Linear(256, 136).cuda()
    x = torch.randn(3, 50, 256, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = lin(x)
        comp = torch.compile(lin, fullgraph=True)
        z = comp(x)
    assert y.dtype == torch.bfloat16 and torch.equal(y, z)
    g = torch.randn_like(y)
    want = torch.autograd.grad(y, (x, lin.weight), g)
    got = torch.autograd.grad(z, (x, lin.weight), g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(ops):
    from quartet_b200.quantization import fp8_linear

    x = torch.randn(4, 256, device="cuda")
    c, sf, _, _ = ops.quant_fp8(x)
    for call in (lambda: ops.quant_fp8(x.half()), lambda: ops.quant_fp8(x[:, ::2]), lambda: ops.quant_fp8(x, torch.int8), lambda: ops.quant_fp8(x, rows=False),
                 lambda: ops.quant_fp8(x.cpu()), lambda: ops.quant_fp8(x[0]), lambda: ops.gemm_fp8_tn(c, sf, c[:, :128].contiguous(), sf),
                 lambda: ops.gemm_fp8_tn(c, sf[:-1], c, sf), lambda: ops.gemm_fp8_tn(c.view(torch.uint8), sf, c, sf),
                 lambda: ops.gemm_fp8_tn(c, sf, c, sf, out_dtype=torch.float16), lambda: ops.linear_fp8(x[:, :100], c, sf), lambda: ops.dequant_fp8(c, sf, 100),
                 lambda: fp8_linear(x, x[:, :128]), lambda: fp8_linear(x[:, :0], x[:, :0]), lambda: ops.linear_fp8(x[:, :0], c, sf), lambda: fp8_linear(x.cpu(), x), lambda: fp8_linear(x, x, grad_dtype=torch.int8)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
