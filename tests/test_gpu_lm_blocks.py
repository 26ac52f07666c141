"""The hybrid LM on the block kernels: residual norms, gated feed-forward
blocks, the AdamW step and the 8-bit head together.

Loss and gradients against the same model in float64 on the CPU with a plain
gated block and unfused norms.  The gated block rounds its operands and hidden
values to bf16 (2^-8 each at most); three blocks deep the gradients stay within
2e-2 of their largest entry, the bound that the package's bf16 paths are held
to.
"""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

gpu = pytest.mark.gpu


class PlainGated(torch.nn.Module):
    def __init__(self, like):
        super().__init__()
        for name in ("gate", "up", "down"):
            linear = getattr(like, name)
            new = torch.nn.Linear(linear.in_features, linear.out_features, bias=False)
            new.weight.data.copy_(linear.weight.data)
            setattr(self, name, new)
        self.activation = like.activation

    def forward(self, x):
        g = self.gate(x)
        act = {"silu": F.silu, "gelu": F.gelu, "relu2": lambda t: F.relu(t).square()}[self.activation](g)
        return self.down(act * self.up(x))


def _pair(gated, **kw):
    from thetascan_b200.lm import HybridLM
    torch.manual_seed(3)
    ours = HybridLM(vocab=256, d_model=128, n_layers=3, n_heads=2, mixer_layers=(), gated=gated, fused_norms=True, **kw)
    ref = HybridLM(vocab=256, d_model=128, n_layers=3, n_heads=2, mixer_layers=(), gated=gated)
    ref.load_state_dict(ours.state_dict())
    for block in ref.blocks:
        block.mlp = PlainGated(block.mlp)
    return ours.cuda(), ref.double()


@gpu
@pytest.mark.parametrize("gated", ["silu", "gelu", "relu2"])
@pytest.mark.parametrize("length", [2, 130])
def test_loss_and_gradients(gated, length):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    ours, ref = _pair(gated)
    tokens = torch.randint(0, 256, (3, length), generator=torch.Generator().manual_seed(7))
    loss, want = ours.loss(tokens.cuda()), ref.loss(tokens)
    loss.backward()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-3 * float(want.detach())
    got = dict(ours.named_parameters())
    for name, p in ref.named_parameters():
        a, b = got[name].grad.double().cpu(), p.grad
        assert float((a - b).abs().max()) <= 2e-2 * float(b.abs().max()), name


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trains_with_a_mixer_and_quantizes_its_head(bits):
    # eight sequences by heart: the loss of a fixed batch falls below half of the uniform log 256 = 5.5
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import AdamW
    from thetascan_b200.lm import HybridLM, gn_mixer_config
    torch.manual_seed(4)
    model = HybridLM(vocab=256, d_model=128, n_layers=3, n_heads=2, mixer_layers=(1,), mixer_config=gn_mixer_config(128, 2),
                     gated="silu", fused_norms=True).cuda()
    opt = AdamW(model.parameters(), lr=3e-3, betas=(0.9, 0.95), weight_decay=0.0, state_bits=bits)
    tokens = torch.randint(0, 256, (8, 33), generator=torch.Generator().manual_seed(7)).cuda()
    losses = []
    for _ in range(60):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model.loss(tokens)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[0] > 5 and losses[-1] < 2.75, losses[::10]
    with torch.no_grad():
        want = model(tokens[:, :-1])
        model.quantize_head()
        got = model(tokens[:, :-1]).float()
    # codes of both factors within 2^-4 of their values, independently over 128 terms: a few percent of the logits' norm
    assert 0 < float((got - want).norm()) <= 0.06 * float(want.norm())
    assert model(tokens[:, :-1]).requires_grad   # with gradients: the exact head


@gpu
def test_quantized_model_compiles_into_one_graph():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    torch._dynamo.reset()
    model, _ = _pair("silu")
    model.quantize_head()
    tokens = torch.randint(0, 256, (3, 20), generator=torch.Generator().manual_seed(7)).cuda()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = model(tokens)
        got = torch.compile(model, fullgraph=True, backend="aot_eager")(tokens)
    # the same kernels; a stream that rounds elsewhere may move a code by a step, 2^-4 of one of 128 terms
    assert got.dtype == want.dtype and got.shape == want.shape
    assert float((got.float() - want.float()).norm()) <= 0.02 * float(want.float().norm())


def test_default_model_is_unchanged_on_the_cpu():
    # the options off: the modules, their order and their initial values are what they were
    from thetascan_b200.lm import HybridLM
    torch.manual_seed(0)
    m = HybridLM(vocab=64, d_model=32, n_layers=2, n_heads=2, mixer_layers=())
    assert [n for n, _ in m.named_parameters() if n.startswith("blocks.0.")] == [
        "blocks.0.norm1.weight", "blocks.0.norm2.weight", "blocks.0.mix.qkv.weight", "blocks.0.mix.out.weight",
        "blocks.0.mlp.up.weight", "blocks.0.mlp.down.weight"]
    assert torch.isfinite(m.loss(torch.randint(0, 64, (2, 9))))
