"""Forward-mode derivatives and recorded traces of the rotary and 8-bit calls, with the kernels themselves."""
import pytest
import torch
from torch.autograd import forward_ad as fwad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    import __graft_entry__ as entry

    entry.build()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tangents_turn_like_values(dtype):
    from quartet_b200.rotary import apply_rotary, rotary_frequencies, rotary_qkv

    inv, _ = rotary_frequencies(64, device="cuda")
    q, k, x, dq, dk, dx = (torch.randn(s, device="cuda").to(dtype) for s in ((2, 7, 4, 80), (2, 7, 2, 80), (2, 7, 8 * 80)) * 2)
    with fwad.dual_level():
        out = apply_rotary(fwad.make_dual(q, dq), fwad.make_dual(k, dk), inv, scale=1.25)
        outs = rotary_qkv(fwad.make_dual(x, dx), 4, 2, inv)
        got = [fwad.unpack_dual(z) for z in (*out, *outs)]
    values, tangents = (*apply_rotary(q, k, inv, scale=1.25), *rotary_qkv(x, 4, 2, inv)), (*apply_rotary(dq, dk, inv, scale=1.25), *rotary_qkv(dx, 4, 2, inv))
    for (p, t), v, w in zip(got, values, tangents):
        assert t is not None and torch.equal(p, v) and torch.equal(t, w)


def test_the_8_bit_layer_refuses_tangents():
    from quartet_b200.quantization import fp8_linear

    x, w = torch.randn(5, 256, device="cuda"), torch.randn(64, 256, device="cuda")
    with fwad.dual_level():
        assert torch.equal(fp8_linear(x, w), fp8_linear(x, w))
        with pytest.raises((RuntimeError, NotImplementedError)):
            fp8_linear(fwad.make_dual(x, x), w)


def test_traced_calls_compute():
    from quartet_b200.quantization import fp8_linear
    from quartet_b200.rotary import apply_rotary, rotary_frequencies, rotary_qkv

    inv, _ = rotary_frequencies(64, device="cuda")
    w = torch.randn(72, 256, device="cuda")
    for f, shape in ((lambda a: apply_rotary(a, None, inv)[0], (2, 7, 4, 64)), (lambda a: rotary_qkv(a, 2, 1, inv), (2, 7, 4 * 64)), (lambda a: fp8_linear(a, w), (3, 5, 256))):
        for grad in (False, True):
            x, z = (torch.randn(shape, device="cuda", requires_grad=grad) for _ in range(2))
            got, want = torch.jit.trace(f, (x,))(z), f(z)
            for a, b in zip(*((v if isinstance(v, tuple) else (v,)) for v in (got, want))):
                assert torch.equal(a, b) and a.requires_grad == grad
                if grad:
                    assert torch.equal(*(torch.autograd.grad(v.float().sum(), (z,), retain_graph=True)[0] for v in (a, b)))


@pytest.mark.parametrize("m", [1, 40])
@pytest.mark.parametrize("n", [64, 77])
def test_the_packed_form_compiled_and_traced(m, n):
    from quartet_b200 import ops

    w, sf = ops.quant_fp8(torch.randn(n, 200, device="cuda"), square=True)[:2]
    f = lambda a: ops.linear_fp8(a, w, sf, torch.bfloat16) * 2  # noqa: E731
    x, z = torch.randn(m, 1, 200, device="cuda"), torch.randn(m, 1, 200, device="cuda")
    assert torch.equal(torch.compile(f, fullgraph=True)(x), f(x))
    assert torch.equal(torch.jit.trace(f, (x,))(z), f(z))
    # calls that are no operators break a compiled graph, and compute what they do outside one
    g = lambda a: ops.dequant_fp8(*ops.quant_fp8(a.view(m, 200))[:2], 200) * 2  # noqa: E731
    assert torch.equal(torch.compile(g)(x), g(x))
