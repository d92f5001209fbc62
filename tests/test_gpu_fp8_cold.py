"""The product from cold memory, where copies of operands and scales arrive late and in any order: the same bits as from a warm cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import ops

    return ops


# (form, M, N, K): contractions longer than any ring of buffers, several rounds of tiles for the CTA pairs
CASES = [("pairs", 4310, 3886, 1474), ("pairs", 4190, 5517, 1253), ("pairs", 3741, 2647, 919), ("pairs", 8192, 2048, 4096), ("rows_256", 130, 4010, 8192),
         ("rows_128", 512, 768, 900), ("rows_128_two", 300, 11003, 640), ("rows_few", 33, 4096, 4096), ("stream", 3, 4010, 4096)]


@pytest.mark.parametrize("form,M,N,K", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_cold_and_warm_agree(ops, form, M, N, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(K)
    make = lambda rows: torch.randn(rows, K, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))  # noqa: E731
    a, b = (ops.quant_fp8(make(rows))[:2] for rows in (M, N))
    assert ops.gemm_fp8_form(M, N, a[0].shape[1])[0] == form
    flush = torch.empty(64 << 20, device="cuda")                # twice the L2
    want = ops.gemm_fp8_tn(*a, *b, out_dtype=dtype)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(400):
        flush.fill_(i)
        wrong += (ops.gemm_fp8_tn(*a, *b, out_dtype=dtype) != want).any()
    assert wrong.item() == 0 and ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_first_and_second_run_of_changing_sizes_agree(ops, dtype):
    """New operands each time, other work between their quantizers and the product: the first run finds everything cold, the second nothing."""
    import random

    r, g = random.Random(7), torch.Generator(device="cuda").manual_seed(7)
    f8 = (torch.float8_e4m3fn, torch.float8_e5m2)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(600):
        M, N, K = r.randint(2200, 5000), r.randint(2200, 5600), r.randint(600, 1500)
        ops_ab = []
        for rows in (M, N):
            x = torch.randn(rows, K, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))
            ops_ab.append(ops.quant_fp8(x, r.choice(f8), square=r.random() < 0.5)[:2])
        for codes, sf in ops_ab:
            ops.dequant_fp8(codes, sf).double()
        first, second = (ops.gemm_fp8_tn(*ops_ab[0], *ops_ab[1], out_dtype=dtype) for _ in range(2))
        wrong += (first != second).any()
    assert wrong.item() == 0 and ops.device_status() == 0


@pytest.mark.parametrize("M,K,N", [(1000, 2000, 3000), (2048, 1030, 4096), (4096, 640, 8000)])
def test_both_gradients_from_cold_memory(ops, M, K, N):
    """The backward's two products, in one launch of CTA pairs where that is quicker: every first run against the next."""
    g = torch.Generator(device="cuda").manual_seed(M)
    evict = torch.empty(64 << 20, device="cuda")
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(150):
        x, w, e = (torch.randn(s, generator=g, device="cuda", dtype=torch.bfloat16) for s in ((M, K), (N, K), (M, N)))
        x, e = (t * torch.exp(2 * torch.randn(M, 1, generator=g, device="cuda")).bfloat16() for t in (x, e))
        _, saved = ops.fp8_linear_fwd(x, w, True, True, torch.bfloat16)
        evict.fill_(i)
        first, second = (ops.fp8_linear_bwd(e, saved, K, torch.float8_e5m2, torch.bfloat16, torch.float32, True, True, True, True) for _ in range(2))
        for a, b in zip(first, second):
            wrong += (a != b).any()
    assert wrong.item() == 0 and ops.device_status() == 0
