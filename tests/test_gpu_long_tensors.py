"""Tensors of more than 2^31 elements: what lies past that offset equals the same call on a slice of its own, or has a known value."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    if torch.cuda.get_device_properties(0).total_memory < 64 << 30:
        pytest.skip("needs 64 GB")
    from quartet_b200 import ops

    return ops


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _bytes(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("cols", [31008, 31003])
@pytest.mark.parametrize("square", [False, True])
def test_quantizer(ops, cols, square):
    rows, tail = 70001, 70001 - 546 * 128
    x = torch.randn(rows, cols, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    codes, sf, codes_t, sf_t = ops.quant_fp8(x, square=square, transpose=True)
    want, wsf, want_t, wsf_t = ops.quant_fp8(x[-tail:].clone(), square=square, transpose=True)
    assert torch.equal(_bytes(codes[-tail:]), _bytes(want)) and torch.equal(sf[-wsf.numel():], wsf)
    blocks = (rows + 127) // 128   # scales of the transpose: [column blocks, row blocks, 512]
    assert torch.equal(_bytes(codes_t)[:, 546 * 128:], _bytes(want_t)) and torch.equal(sf_t.view(-1, blocks, 512)[:, -1], wsf_t.view(-1, 512))
    last = ops.dequant_fp8(codes, sf, cols, dtype=torch.bfloat16)[-tail:]
    assert torch.equal(last, ops.dequant_fp8(want, wsf, cols, dtype=torch.bfloat16))
    only = ops.quant_fp8(x, square=square)
    assert torch.equal(_bytes(only[0][-tail:]), _bytes(want))


def _close(got, want, absum, k):
    """both sums of k exact products in fp32, in whatever order; then the output's rounding, of both"""
    lim = 2 * (k * 2.0 ** -23 * absum)
    lim = lim + torch.finfo(got.dtype).eps * (want.double().abs() + lim)
    assert bool(((got.double() - want.double()).abs() <= lim).all())


@pytest.mark.parametrize("n", [31008, 31003])
def test_product_with_a_long_result(ops, n):
    m, k = 70001, 128
    a, b = torch.randn(m, k, device="cuda"), torch.randn(n, k, device="cuda")
    (ac, asf, _, _), (bc, bsf, _, _) = ops.quant_fp8(a), ops.quant_fp8(b, square=True)
    y = ops.gemm_fp8_tn(ac, asf, bc, bsf)
    tail = m - 546 * 128
    tc, tsf, _, _ = ops.quant_fp8(a[-tail:].clone())
    absum = ops.dequant_fp8(tc, tsf).double().abs() @ ops.dequant_fp8(bc, bsf).double().abs().T
    _close(y[-tail:], ops.gemm_fp8_tn(tc, tsf, bc, bsf), absum, k)


@pytest.mark.parametrize("m", [1, 16, 100, 300])
def test_product_with_a_long_weight(ops, m):
    n, k = 70001, 31104
    w = torch.empty(n, k, device="cuda", dtype=torch.bfloat16).normal_()
    wc, wsf = ops.quant_fp8(w, square=True)[:2]
    x = torch.randn(m, k, device="cuda").bfloat16()
    tail = n - 546 * 128
    tc, tsf = ops.quant_fp8(w[-tail:].clone(), square=True)[:2]
    xc, xsf = ops.quant_fp8(x)[:2]
    absum = ops.dequant_fp8(xc, xsf).double().abs() @ ops.dequant_fp8(tc, tsf).double().abs().T
    _close(ops.linear_fp8(x, wc, wsf, out_dtype=torch.float32)[:, -tail:], ops.linear_fp8(x, tc, tsf, out_dtype=torch.float32), absum, k)
    assert ops.device_status() == 0


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(ops, interleaved):
    from quartet_b200 import rotary

    t, h, d = 131075, 16, 1030
    inv, _ = rotary.rotary_frequencies(128, device="cuda")
    q = torch.empty(1, t, h, d, device="cuda", dtype=torch.bfloat16).normal_()
    assert q.numel() > 2 ** 31
    y, _ = rotary.apply_rotary(q, None, inv, interleaved=interleaved)
    want, _ = rotary.apply_rotary(q[:, -3:].clone(), None, inv, offset=t - 3, interleaved=interleaved)
    assert torch.equal(y[:, -3:], want)
    del q
    heads = 2 * h + 2 * h
    packed = torch.empty(1, t // 2, heads * d, device="cuda", dtype=torch.bfloat16).normal_()
    got = rotary.rotary_qkv(packed, 2 * h, h, inv, interleaved=interleaved)
    want = rotary.rotary_qkv(packed[:, -3:].clone(), 2 * h, h, inv, offset=t // 2 - 3, interleaved=interleaved)
    assert packed.numel() > 2 ** 31 and all(torch.equal(a[:, :, -3:], b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_and_clip(ops, dtype):
    g = torch.zeros(2 ** 31 + 12345, device="cuda", dtype=dtype)
    g[0], g[2 ** 31 + 7], g[-1] = 3.0, 4.0, 12.0
    assert ops.grad_norm([g]).item() == 13.0 and ops.grad_norm([g], float("inf")).item() == 12.0
    assert ops.clip_grads([g], 6.5).item() == 13.0
    coef = torch.tensor(6.5 / (13.0 + 1e-6), dtype=torch.float64).float()
    assert torch.equal(g[[0, 2 ** 31 + 7, -1]].cpu(), (torch.tensor([3.0, 4.0, 12.0]) * coef).to(dtype)) and int(torch.count_nonzero(g)) == 3
