"""A small hybrid language model around the b200 mixer (baseline config 5).

The reference trains its mixers inside an external GPT host that it does not
ship (benchmarks/parameter-golf/prepare_harness.py:649-740 patches
``build_mixer`` and ``Block`` into a cloned training script).  This module is
a self-contained host of the same shape -- for exercising the mixer under
autograd, bf16 autocast, data-parallel training and AdamW, and for timing a
whole training step:

* token embedding of a 1024-entry vocabulary, tied to the output head;
* nine pre-norm residual blocks ``x + mix(norm(x))``, ``x + mlp(norm(x))``
  with RMS norms, d_model 512, 8 heads, MLP hidden width 2 x d_model
  (squared-ReLU);
* the two middle blocks mix with a ThetaScan-GN mixer of this package
  (``thetascan_b200.ThetaScan``; the expanded GN layout of the reference's
  ``gn_expanded_reference_v0_1`` preset, config.py:832-862: shared k/q
  projection, learned relu2 threshold, 2x random feature expansion,
  two-stage feature-mass read, one fast recency branch -- at memory
  multiplier 2, m = 256, the widest the scan kernels take), the others with
  causal softmax attention (``scaled_dot_product_attention``, RoPE on q/k).

The mixer's output projection starts at zero, as the reference's adapter
initialises it (thetascan_benchmark_adapter.py:83).

Options of the same model on this package's block kernels: ``gated`` (the
feed-forward block is a :class:`GatedFFN` of that activation), ``fused_norms``
(each norm takes the previous branch's addition to the residual stream with
it), training by :class:`AdamW` with states in 32 or 8 bits, and
:meth:`HybridLM.quantize_head` (inference logits from an 8-bit norm and an
8-bit vocabulary projection).  ``python -m thetascan_b200.lm`` trains such a
model on uniform-random tokens for a few steps and reports loss, time and the
8-bit head's agreement.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .config import GNConfig, RoPEConfig, TemporalConfig, ThetaScanConfig
from .ffn import GatedFFN
from .mixer import ThetaScan
from .norm import add_rms_norm, rms_norm, rms_norm_8bit


def gn_mixer_config(d_model: int = 512, n_heads: int = 8, memory_multiplier: int = 2) -> ThetaScanConfig:
    """The expanded GN mixer layout of config 5 at memory multiplier 2."""
    return ThetaScanConfig(
        d_model=d_model, n_heads=n_heads, memory_multiplier=memory_multiplier, feature_expansion=2,
        share_key_query=True, output_gate=False, family="gn",
        gn=GNConfig(nonlinearity="relu2_threshold", jacobian_steps=1, read_normalization="both_feature_mass"),
        rope=RoPEConfig(mode="partial", fraction=0.5, base=10_000.0),
        temporal=TemporalConfig(mode="bank", bank_mode="fast", recency_branches=1, retention_inits=(0.9,),
                                blend_mode="free"))


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x):
        return F.rms_norm(x, (x.shape[-1],), self.weight, self.eps)


def _rope(x, base: float = 10_000.0):
    """Adjacent-pair rotation of all channels of ``x [B,H,T,d]`` (f32 phases)."""
    B, H, T, d = x.shape
    inv = 1.0 / (base ** (torch.arange(0, d, 2, dtype=torch.float32, device=x.device) / d))
    ang = torch.outer(torch.arange(T, dtype=torch.float32, device=x.device), inv)
    cos, sin = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), dim=-1).flatten(-2)


class CausalAttention(nn.Module):
    def __init__(self, d_model: int, n_heads: int):
        super().__init__()
        self.n_heads = n_heads
        self.qkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.out = nn.Linear(d_model, d_model, bias=False)

    def forward(self, x):
        B, T, D = x.shape
        q, k, v = self.qkv(x).view(B, T, 3, self.n_heads, D // self.n_heads).permute(2, 0, 3, 1, 4)
        y = F.scaled_dot_product_attention(_rope(q), _rope(k), v, is_causal=True)
        return self.out(y.transpose(1, 2).reshape(B, T, D))


class MLP(nn.Module):
    def __init__(self, d_model: int, ratio: int):
        super().__init__()
        self.up = nn.Linear(d_model, ratio * d_model, bias=False)
        self.down = nn.Linear(ratio * d_model, d_model, bias=False)

    def forward(self, x):
        return self.down(F.relu(self.up(x)).square())


class Block(nn.Module):
    def __init__(self, d_model: int, n_heads: int, mlp_ratio: int, mixer: nn.Module, gated: str | None = None):
        super().__init__()
        self.norm1, self.norm2 = RMSNorm(d_model), RMSNorm(d_model)
        self.mix = mixer
        self.mlp = MLP(d_model, mlp_ratio) if gated is None else GatedFFN(d_model, mlp_ratio * d_model, gated)

    def forward(self, x):
        x = x + self.mix(self.norm1(x))
        return x + self.mlp(self.norm2(x))

    def forward_fused(self, branch, stream):
        """The block on a residual ``stream`` that the previous ``branch``
        (None: nothing) still has to be added to; returns its own last branch
        and the stream before that."""
        y, stream = _add_norm(self.norm1, branch, stream)
        y, stream = _add_norm(self.norm2, self.mix(y), stream)
        return self.mlp(y), stream


def _add_norm(norm, branch, stream):
    if branch is None:
        return rms_norm(stream, norm.weight, norm.eps), stream
    return add_rms_norm(branch.to(stream.dtype), stream, norm.weight, norm.eps)


def _rows_8bit(w):
    """e4m3 codes and f32 scales of the rows of ``w`` (largest magnitude to 448)."""
    w = w.detach().float()
    scale = w.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100) / 448
    return (w / scale).to(torch.float8_e4m3fn), scale


class HybridLM(nn.Module):
    """Nine-block hybrid LM; blocks in ``mixer_layers`` use the GN mixer."""

    def __init__(self, vocab: int = 1024, d_model: int = 512, n_layers: int = 9, n_heads: int = 8,
                 mlp_ratio: int = 2, mixer_layers=(3, 4), mixer_config: ThetaScanConfig | None = None,
                 mixer_factory=None, gated: str | None = None, fused_norms: bool = False):
        """``mixer_factory(config)`` builds a mixer module (default: this
        package's ThetaScan; a test passes the reference's own to compare).
        ``gated``: the activation of gated feed-forward blocks (default: the
        plain squared-ReLU MLP).  ``fused_norms``: residual additions within
        the norms' kernels (CUDA only)."""
        super().__init__()
        self.fused_norms = fused_norms
        self.head_8bit = None
        self.embed = nn.Embedding(vocab, d_model)
        nn.init.normal_(self.embed.weight, std=0.02)
        cfg = mixer_config if mixer_config is not None else gn_mixer_config(d_model, n_heads)
        factory = mixer_factory if mixer_factory is not None else ThetaScan
        blocks = []
        for i in range(n_layers):
            if i in mixer_layers:
                mixer = factory(cfg)
                mixer.zero_output_projection_()
            else:
                mixer = CausalAttention(d_model, n_heads)
            blocks.append(Block(d_model, n_heads, mlp_ratio, mixer, gated))
        self.blocks = nn.ModuleList(blocks)
        self.norm = RMSNorm(d_model)
        # residual-branch outputs of the attention and MLP blocks (the mixers
        # keep their zero output projection)
        for name, p in self.named_parameters():
            if name.endswith("mlp.down.weight") or name.endswith("mix.out.weight"):
                nn.init.normal_(p, std=0.02 / math.sqrt(2 * n_layers))

    def quantize_head(self) -> None:
        """Keep the vocabulary projection in 8 bits for inference: from now on
        calls without gradients take the final norm as e4m3 codes with a scale
        per row and multiply codes by codes (CUDA; the embedding keeps its
        type).  Call again after the weights change."""
        self.head_8bit = _rows_8bit(self.embed.weight)

    def _head(self, branch, stream):
        norm = self.norm
        if self.head_8bit is not None and not torch.is_grad_enabled():
            residual = None if branch is None else branch.to(stream.dtype)
            codes, scales, *_ = rms_norm_8bit(stream, norm.weight, norm.eps, residual=residual)
            weight, weight_scale = self.head_8bit
            logits = torch._scaled_mm(codes.reshape(-1, codes.shape[-1]), weight.t(), scales.reshape(-1, 1),
                                      weight_scale.t(), out_dtype=torch.bfloat16)
            return logits.view(*codes.shape[:-1], -1)
        y = norm(stream) if branch is None and not self.fused_norms else _add_norm(norm, branch, stream)[0]
        return F.linear(y, self.embed.weight)

    def forward(self, tokens):
        x = self.embed(tokens)
        if not self.fused_norms:
            for block in self.blocks:
                x = block(x)
            return self._head(None, x)
        branch = None
        for block in self.blocks:
            branch, x = block.forward_fused(branch, x)
        return self._head(branch, x)

    def loss(self, tokens):
        """Next-token cross entropy of ``tokens [B,T]`` (predicting 1..T-1)."""
        logits = self(tokens[:, :-1])
        return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), tokens[:, 1:].reshape(-1))


def main() -> None:
    """Train a gated hybrid model on random tokens with this package's norms, feed-forward blocks and optimizer."""
    import argparse
    import time

    from .optim import AdamW

    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--gated", default="silu", choices=("silu", "gelu", "relu2"))
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    torch.manual_seed(0)
    model = HybridLM(gated=a.gated, fused_norms=True).cuda()
    optimizer = AdamW(model.parameters(), lr=3e-4, betas=(0.9, 0.95), weight_decay=0.1, state_bits=a.state_bits)
    data = torch.randint(0, model.embed.num_embeddings, (a.batch, a.tokens + 1), device="cuda")
    for step in range(a.steps):
        torch.cuda.synchronize()
        start = time.perf_counter()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model.loss(data)
        loss.backward()
        optimizer.step()
        optimizer.zero_grad()
        torch.cuda.synchronize()
        print(f"step {step + 1}: loss {loss.detach().item():.4f}, {(time.perf_counter() - start) * 1e3:.1f} ms")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = model(data[:, :-1]).float()
        model.quantize_head()
        got = model(data[:, :-1]).float()
    print(f"8-bit head: logits within {float((got - want).norm() / want.norm()):.3f} of the bf16 head's, "
          f"{float((got.argmax(-1) == want.argmax(-1)).float().mean()) * 100:.1f} % of the tokens the same")


if __name__ == "__main__":
    main()
