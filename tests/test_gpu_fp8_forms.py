"""Every form of the 8-bit product by itself: formats that differ, a scale for every 32 values, and the same bits every time.  Each size is checked to
take the form that it stands for, so that a change of the rule that picks cannot take a form out of these tests unseen."""
import pytest
import torch

from tests import fp8_oracle as fo
from tests.test_gpu_fp8 import _bound, _product
from tests.test_gpu_fp8_scales import _blocked32

pytestmark = pytest.mark.gpu
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2

FORMS = {"stream": (3, 4010, 1024), "rows_few": (33, 1200, 900), "rows_128": (512, 768, 900), "rows_128_two": (300, 11003, 640), "rows_256": (130, 4010, 8192),
         "pairs": (2300, 4101, 256)}


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__ as entry

    entry.build()
    from quartet_b200 import ops

    return ops


@pytest.mark.parametrize("form", FORMS)
def test_sizes_take_the_form_they_stand_for(ops, form):
    M, N, K = FORMS[form]
    assert ops.gemm_fp8_form(M, N, fo.pad128(K))[0] == form and set(FORMS) == set(ops.GEMM_FP8_FORMS)
    with pytest.raises(ValueError):
        ops.gemm_fp8_form(M, N, 100)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fa,fb", [(E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
def test_mixed_formats(ops, form, fa, fb):
    _product(ops, *FORMS[form], fa, fb)


@pytest.mark.parametrize("form", FORMS)
def test_a_scale_for_every_32(ops, form):
    M, N, K = FORMS[form]
    K = fo.pad128(K)
    g = torch.Generator().manual_seed(M)
    a, b = (torch.randn(n, K, generator=g).to(E4M3) for n in (M, N))
    ae, be = (torch.randint(120, 134, (n, K // 32), generator=g, dtype=torch.uint8) for n in (M, N))
    av, bv = (c.double() * fo.two(e.int() - 127).repeat_interleave(32, 1) for c, e in ((a, ae), (b, be)))
    y = ops.gemm_fp8_tn(a.cuda(), _blocked32(ae).cuda(), b.cuda(), _blocked32(be).cuda(), out_dtype=torch.float32)
    want = av @ bv.T
    assert bool(((y.cpu().double() - want).abs() <= _bound(av.abs() @ bv.abs().T, K, want, torch.float32)).all())
    assert ops.device_status() == 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_every_time(ops, form, dtype):
    M, N, K = FORMS[form]
    a, b = torch.randn(M, K, device="cuda"), torch.randn(N, K, device="cuda") * 0.02
    (ac, asf, _, _), (bc, bsf, _, _) = ops.quant_fp8(a), ops.quant_fp8(b, square=True)
    first = ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=dtype)
    assert all(torch.equal(first, ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=dtype)) for _ in range(20))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                              # beside another product
        other = [ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=dtype) for _ in range(5)]
    mine = [ops.gemm_fp8_tn(ac, asf, bc, bsf, out_dtype=dtype) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, t) for t in other + mine)
