"""The operators around the 4-bit layers together, as a training step uses them: rotary positions on the packed projection of a
QuantizedLinear, an 8-bit head, and clipping before the optimizer -- against the same model with each of them written in torch."""
import copy
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tests import fp8_oracle as fo
from tests.llama_harness import Block, TinyLlama, rotary

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Q():
    import __graft_entry__ as entry

    entry.build()
    import quartet_b200.quantization as q

    return q


class FusedBlock(Block):
    """The harness block with the packed projection split and turned in one pass."""

    def forward(self, x):
        from quartet_b200.rotary import rotary_qkv

        b, t, d = x.shape
        qkv = self.rmsnorm_linear(x, self.ln1.weight, self.ln1.eps, self.c_attn)
        q, k, v = rotary_qkv(qkv, self.n_head, self.n_kv_head, self.inv_freq)
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=self.n_kv_head != self.n_head)
        x = x + self.attn_proj(y.transpose(1, 2).reshape(b, t, d))
        return x + self.swiglu_linear(self.rmsnorm_linear(x, self.ln2.weight, self.ln2.eps, self.w12), self.c_proj)


class _PlainHead(torch.autograd.Function):
    """The 8-bit layer's definition in 64 bits, and its gradient's."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return fo.layer(x.cpu(), w.cpu(), torch.zeros(x.shape[0], w.shape[0]), torch.float8_e4m3fn)[0].float().to(x.device)

    @staticmethod
    def backward(ctx, e):
        x, w = ctx.saved_tensors
        _, dx, dw = fo.layer(x.cpu(), w.cpu(), e.cpu(), torch.float8_e4m3fn)
        return dx.float().to(x.device), dw.float().to(x.device)


class PlainHead(nn.Linear):
    def forward(self, x):
        return _PlainHead.apply(x.reshape(-1, x.shape[-1]), self.weight).view(*x.shape[:-1], -1)


def build(Q, n_kv_head):
    torch.manual_seed(0)
    plain = TinyLlama(Q, vocab=500, d=512, n_layer=2, n_head=4, n_kv_head=n_kv_head, gkw={"stochastic": False}, fuse_producers=True).cuda()
    fused = copy.deepcopy(plain)
    from quartet_b200.rotary import rotary_frequencies

    inv, _ = rotary_frequencies(128, device="cuda")
    for blk in fused.blocks:
        blk.__class__, blk.inv_freq = FusedBlock, inv
    for model, cls in ((plain, PlainHead), (fused, Q.Fp8Linear)):
        head = cls(512, 500, bias=False).cuda()
        head.weight = model.lm_head.weight
        model.lm_head = head
    return plain, fused


@pytest.mark.parametrize("n_kv_head", [None, 2])
def test_step_against_the_model_in_torch(Q, n_kv_head):
    from quartet_b200 import ops
    from quartet_b200.clip import clip_grad_norm_

    assert rotary is not None
    plain, fused = build(Q, n_kv_head)
    idx, tgt = (torch.randint(0, 500, (2, 96), generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2))
    losses = []
    for model in (plain, fused):
        loss = model(idx, tgt)
        loss.backward()
        losses.append(loss.item())
    # The forward differs by the last places of the rotation and of the head's sums, which move a 4-bit code now and then
    assert abs(losses[0] - losses[1]) < 1e-3 * losses[0]
    for (n, a), (_, b) in zip(plain.named_parameters(), fused.named_parameters()):
        cos = F.cosine_similarity(a.grad.flatten().double(), b.grad.flatten().double(), dim=0).item()
        assert cos > 0.99 and abs(a.grad.norm() / b.grad.norm() - 1).item() < 0.02, (n, cos)
    grads = [p.grad.clone() for p in fused.parameters()]
    want = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    norm = clip_grad_norm_(fused.parameters(), 0.5 * want)
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    for g, p in zip(grads, fused.parameters()):
        assert torch.allclose(p.grad, g * 0.5, rtol=1e-5, atol=0)
    assert ops.device_status() == 0


def test_steps_run_under_autocast_and_compiled(Q):
    from quartet_b200 import ops
    from quartet_b200.clip import clip_grad_norm_

    _, model = build(Q, 2)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    idx = torch.randint(0, 500, (2, 128), device="cuda")
    tgt = torch.roll(idx, -1, 1)
    eager = []
    for step in (model, torch.compile(model)):
        for _ in range(2):
            opt.zero_grad(set_to_none=True)
            with torch.autocast("cuda", dtype=torch.bfloat16):
                loss = step(idx, tgt)
            loss.backward()
            n = clip_grad_norm_(model.parameters(), 1.0)
            eager.append((loss.item(), n.item()))
            assert all(torch.isfinite(p.grad).all() for p in model.parameters())
            after = math.sqrt(sum(p.grad.double().square().sum().item() for p in model.parameters()))
            assert after <= 1.0 + 1e-6 or n.item() < 1.0
            opt.step()
    assert all(math.isfinite(v) for pair in eager for v in pair)
    assert ops.device_status() == 0
