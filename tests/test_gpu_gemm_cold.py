"""The 4-bit product from cold memory: the first run of new operands against the second, bit for bit."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import ops

    return ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_first_and_second_run_agree(ops, dtype):
    """New operands each time, other work between their quantizers and the product: the first run finds everything cold, the second nothing."""
    r, g = random.Random(3), torch.Generator(device="cuda").manual_seed(3)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    evict = torch.empty(64 << 20, device="cuda")                # twice the L2
    for i in range(600):
        M, N, K = 256 * r.randint(8, 20), 256 * r.randint(8, 22), 128 * r.randint(8, 30)
        a, b = (ops.quant_fwd(torch.randn(rows, K, generator=g, device="cuda").mul_(torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))).bfloat16())[:2]
                for rows in (M, N))
        evict.fill_(i)
        first, second = (ops.gemm_mxfp4_tn(*a, *b, out_dtype=dtype) for _ in range(2))
        wrong += (first != second).any()
    assert wrong.item() == 0 and ops.device_status() == 0
