"""Steps of a layer whose weight gradient leaves through a PeerWgradScatter, clipped by clip_grad_norm_: one rank, so that its own memory is the peer's."""
import random

import pytest
import torch
import torch.distributed as dist

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def group():
    import __graft_entry__ as entry

    entry.build()
    torch.cuda.set_device(0)
    dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1)
    yield
    dist.destroy_process_group()


def _layer(k, n):
    from quartet_b200.quantization import BACKWARD_SCHEMES, QUANTIZER_CLASSES, QuantizedLinear

    return QuantizedLinear(k, n, bias=False, weight_quantizer=QUANTIZER_CLASSES["QuestMXFP4Quantizer"](), activation_quantizer=QUANTIZER_CLASSES["QuestMXFP4Quantizer"](),
                           gradient_quantizer=QUANTIZER_CLASSES["AlbertTsengQuantizer"](stochastic=True, rerotate="signs"),
                           backward_scheme=BACKWARD_SCHEMES["Q(E)Q(Wt)t_Q(Et)Q(Xt)t"]()).cuda()


def test_steps_with_clipping(group):
    from quartet_b200.clip import clip_grad_norm_
    from quartet_b200.shard import PeerWgradScatter

    torch.manual_seed(0)
    a, b = _layer(512, 256), _layer(256, 512)
    sink = PeerWgradScatter()
    a.wgrad_sink = b.wgrad_sink = sink
    weights = [a.weight, b.weight]
    x = torch.randn(256, 512, device="cuda", dtype=torch.bfloat16)

    def backward(layer, inp):
        random.seed(1), torch.manual_seed(1)
        y = layer(inp.detach().requires_grad_())
        y.backward(torch.ones_like(y))

    for step in range(3):
        backward(a, x * (step + 1))
        if step != 1:
            backward(b, x[:, :256])
        with pytest.raises(RuntimeError, match=r"wait\(\)"):
            clip_grad_norm_(weights, 1.0)
        got = [t.clone() for t in sink.wait()]
        kept = None if step == 0 else b.weight.grad_shard.clone()
        want = torch.cat([t.double().flatten() for t in got]).norm().item()
        n = clip_grad_norm_(weights, 1.0).item()
        assert want > 1.0 and abs(n - want) <= 2.0 ** -23 * want
        for w, t in zip(weights, got):
            assert torch.allclose(w.grad_shard, t * (1.0 / (want + 1e-6)), rtol=2.0 ** -22, atol=0)
        if step == 1:                                        # b took no part: neither counted nor scaled again
            assert torch.equal(b.weight.grad_shard, kept)
    sink.close()
