"""Scales of every size in the 8-bit product: what a pair of them makes of a sum, whatever either would make of it alone."""
import pytest
import torch

from tests import fp8_oracle as fo

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import ops

    return ops


def _blocked32(e):
    """Scale bytes [rows, K / 32] as the kernels lay them out."""
    rows, n = e.shape
    out = torch.zeros(fo.pad128(rows) // 128, n // 4, 32, 4, 4, dtype=torch.uint8)
    r = torch.arange(rows)
    out[r // 128, :, r % 32, r % 128 // 32, :] = e.view(rows, n // 4, 4)
    return out.reshape(-1)


def _check(ops, a, ae, b, be, K):
    av, bv = (c.double() * fo.two(e.int() - 127).repeat_interleave(32, 1) for c, e in ((a, ae), (b, be)))
    y = ops.gemm_fp8_tn(a.cuda(), _blocked32(ae).cuda(), b.cuda(), _blocked32(be).cuda(), out_dtype=torch.float32).cpu().double()
    want = av @ bv.T
    # sums of K exact products, at most 2^-23 of the magnitudes lost at each addition; results below the normal range are rounded to 2^-149
    # at each addition
    lim = K * 2.0 ** -23 * (av.abs() @ bv.abs().T) + want.abs() * 2.0 ** -24 + K * 2.0 ** -149
    assert bool(((y - want).abs() <= lim).all()), ((y - want).abs() / lim).max().item()


# (byte of B's scales, byte of A's): far apart, the least and the largest, both small
PAIRS = [(237, 67), (67, 237), (0, 187), (187, 0), (1, 254), (254, 1), (254, 0), (0, 254), (127, 127), (200, 150), (64, 64), (60, 66), (10, 10), (0, 0)]


@pytest.mark.parametrize("M", [1, 8, 9, 70])
@pytest.mark.parametrize("wb,xb", PAIRS)
def test_products_of_any_two_scales(ops, M, wb, xb):
    if M > 8 and 2 < wb + xb < 129:
        pytest.skip("sums below the normal range: how the tensor core rounds them is its own")
    g = torch.Generator().manual_seed(M + wb)
    N, K = 150, 256
    a, b = (torch.randn(n, K, generator=g).to(E4M3) for n in (M, N))
    ae, be = (torch.full((n, K // 32), v, dtype=torch.uint8) for n, v in ((M, xb), (N, wb)))
    _check(ops, a, ae, b, be, K)


@pytest.mark.parametrize("M", [1, 8, 9, 70])
def test_scales_far_apart_within_a_block_of_128(ops, M):
    """Every group of 32 with a pair of scales of its own, their products between 2^-30 and 2^30."""
    g = torch.Generator().manual_seed(M)
    N, K = 150, 512
    a, b = (torch.randn(n, K, generator=g).to(E4M3) for n in (M, N))
    up = torch.randint(-110, 111, (1, K // 32), generator=g)
    ae = (127 + up + torch.randint(-15, 16, (M, K // 32), generator=g)).to(torch.uint8)
    be = (127 - up + torch.randint(-15, 16, (N, K // 32), generator=g)).to(torch.uint8)
    _check(ops, a, ae, b, be, K)


@pytest.mark.parametrize("M", [1, 3, 8])
def test_rows_of_zeros_beside_others(ops, M):
    """Rows of zeros have the least scale; with them in the same instruction the others keep their results to the last bit."""
    x, w = torch.randn(M, 1000, device="cuda"), torch.randn(300, 1000, device="cuda") * 0.02
    w[128:256] = 0.0
    want = ops.linear_fp8(x, *ops.quant_fp8(w, square=True)[:2])
    wide = torch.cat([x, torch.zeros(8 - M, 1000, device="cuda")]) if M < 8 else x
    got = ops.linear_fp8(wide, *ops.quant_fp8(w, square=True)[:2])
    assert torch.equal(got[:M], want) and bool((got[M:] == 0).all()) and bool((want[:, 128:256] == 0).all())
    exact = fo.values(x.cpu(), E4M3) @ fo.values(w.cpu(), E4M3, True).T
    s = fo.values(x.cpu(), E4M3).abs() @ fo.values(w.cpu(), E4M3, True).abs().T
    assert bool(((want.cpu().double() - exact).abs() <= 1024 * 2.0 ** -23 * s + exact.abs() * 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reading_back_with_a_factor_rounds_once(ops, dtype):
    """code 2^(b - 127) scale, where the scale and the block's power of two alone leave fp32 or its normal range."""
    codes = torch.tensor([2.0 ** -9, -3 * 2.0 ** -9, 2.0 ** -6, 1.125, 448.0, 0.0]).repeat(64)[:256].view(2, 128).to(E4M3)
    for byte, scale in ((250, 1024.0), (254, 0.3), (0, 0.3), (1, 1e-3), (100, 3e38), (127, 1.1), (40, 7e-13)):
        sf = _blocked32(torch.full((2, 4), byte, dtype=torch.uint8)).cuda()
        got = ops.dequant_fp8(codes.cuda(), sf, scale=scale, dtype=dtype).cpu()
        want = codes.double() * 2.0 ** (byte - 127) * torch.tensor(scale).double()      # the factor itself is fp32
        f32 = want.float()                                                              # rounds, overflows and underflows as one product does
        assert torch.equal(got, f32.to(dtype)), (byte, scale)


@pytest.mark.parametrize("n", [64, 77])
def test_results_changed_in_place_before_the_backward(ops, n):
    from quartet_b200.quantization import fp8_linear

    x, w = torch.randn(2, 9, 200, device="cuda"), torch.randn(n, 200, device="cuda") * 0.05
    grads = []
    for inplace in (False, True):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = fp8_linear(a, b)
        y = y.mul_(0.5).add_(1.0) if inplace else y * 0.5 + 1.0
        y.square().sum().backward()
        grads.append((y.detach(), a.grad, b.grad))
    assert all(torch.equal(u, v) for u, v in zip(*grads))


@pytest.mark.parametrize("n", [64, 77])
def test_compiled_layer_with_few_tokens_or_none(ops, n):
    from quartet_b200.quantization import Fp8Linear

    torch.manual_seed(0)
    lin = Fp8Linear(200, n).cuda()
    comp = torch.compile(lin, fullgraph=True, dynamic=False)
    for tokens in (0, 1, 5):
        grads = []
        for f in (lin, comp):
            x = torch.randn(2, tokens, 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).requires_grad_()
            lin.weight.grad = None
            y = f(x)
            y.square().sum().backward()
            grads.append((y.detach(), x.grad, lin.weight.grad.clone()))
        assert grads[0][0].shape == (2, tokens, n)
        assert all(torch.equal(a, b) for a, b in zip(*grads))
