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
8-bit vocabulary projection).  With ``window`` the attention layers see a
sliding window (:func:`thetascan_b200.window_attention`), and
:meth:`HybridLM.generate` goes on from a prompt token by token, with ring caches
and scan states whose size does not depend on the length.  ``python -m thetascan_b200.lm`` trains such a
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
from .sample import sample_tokens
from .seqpar import ScanStream
from .window import WindowCache, window_attention


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


def _rope(x, base: float = 10_000.0, start: int = 0):
    """Adjacent-pair rotation of all channels of ``x [B,H,T,d]`` (f32 phases),
    whose first token is at position ``start``."""
    B, H, T, d = x.shape
    inv = 1.0 / (base ** (torch.arange(0, d, 2, dtype=torch.float32, device=x.device) / d))
    ang = torch.outer(torch.arange(start, start + T, dtype=torch.float32, device=x.device), inv)
    cos, sin = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), dim=-1).flatten(-2)


class AttentionStream(WindowCache):
    """The ring cache of one layer and the tokens that the sequences, all of one
    length, have had; ``lengths`` (int32, on the device) is the same number for
    each, and the layers of a model share it."""

    def __init__(self, lengths, n_heads: int, head_dim: int, window: int, sinks: int):
        super().__init__(lengths.shape[0], n_heads, head_dim, window, sinks, device=lengths.device)
        self.lengths, self.position = lengths, 0

    def attend(self, q, k, v):
        """The attention of the next tokens, ``[B,H,T,d]`` bf16, which enter the cache."""
        T, start = q.shape[2], self.position
        self.position += T
        if T == 1:
            return self.step(q, k, v, self.lengths)
        slots = self.keys.shape[2]
        window = slots - self.sinks
        past_k, past_v = k, v
        if start:
            # what the piece still sees, in order: the first tokens, then the last ones (differences of
            # positions within the window are right even where tokens between the two are left out)
            order = torch.arange(start, device=q.device)
            if start > slots:
                order = torch.cat((order[:self.sinks], order[start - window:]))
            order = torch.where(order < self.sinks, order, self.sinks + (order - self.sinks) % window)
            past_k, past_v = (torch.cat((t[:, :, order], new), 2) for t, new in ((self.keys, k), (self.values, v)))
        y = window_attention(q, past_k, past_v, window, self.sinks)
        self.extend(k, v, self.lengths)
        return y


class CausalAttention(nn.Module):
    """Causal softmax attention; with a ``window`` each token sees that many last
    tokens and the ``sinks`` first ones, in bf16 (CUDA only)."""

    def __init__(self, d_model: int, n_heads: int, window: int | None = None, sinks: int = 0):
        super().__init__()
        if window is None and sinks:
            raise ValueError("first tokens that stay visible (sinks) need a window")
        self.n_heads, self.window, self.sinks = n_heads, window, sinks
        self.qkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.out = nn.Linear(d_model, d_model, bias=False)

    def forward(self, x, stream: AttentionStream | None = None):
        B, T, D = x.shape
        q, k, v = self.qkv(x).view(B, T, 3, self.n_heads, D // self.n_heads).permute(2, 0, 3, 1, 4)
        start = 0 if stream is None else stream.position
        q, k = _rope(q, start=start), _rope(k, start=start)
        if self.window is None:
            y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        else:
            half = [t.to(torch.bfloat16) for t in (q, k, v)]
            y = window_attention(*half, self.window, self.sinks) if stream is None else stream.attend(*half)
            y = y.to(q.dtype)
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

    def forward(self, x, *state):
        x = x + self.mix(self.norm1(x), *state)
        return x + self.mlp(self.norm2(x))

    def forward_fused(self, branch, stream, *state):
        """The block on a residual ``stream`` that the previous ``branch``
        (None: nothing) still has to be added to; returns its own last branch
        and the stream before that."""
        y, stream = _add_norm(self.norm1, branch, stream)
        y, stream = _add_norm(self.norm2, self.mix(y, *state), stream)
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
                 mixer_factory=None, gated: str | None = None, fused_norms: bool = False, window: int | None = None,
                 sinks: int = 0):
        """``mixer_factory(config)`` builds a mixer module (default: this
        package's ThetaScan; a test passes the reference's own to compare).
        ``gated``: the activation of gated feed-forward blocks (default: the
        plain squared-ReLU MLP).  ``fused_norms``: residual additions within
        the norms' kernels (CUDA only).  ``window``, ``sinks``: attention over
        the last ``window`` tokens and the first ``sinks`` (CUDA only), with
        which the model can :meth:`generate`."""
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
                mixer = CausalAttention(d_model, n_heads, window, sinks)
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

    def stream(self, batch: int) -> "ModelStream":
        """The start of ``batch`` sequences that come in pieces (see :meth:`extend`)."""
        return ModelStream(self, batch)

    @torch.no_grad()
    def extend(self, tokens, stream: "ModelStream"):
        """Logits ``[B,vocab]`` behind the last of the ``tokens [B,T]`` that the
        sequences of the ``stream`` go on by.  The whole work on a token does not
        depend on how many came before it."""
        if tokens.ndim != 2 or tokens.shape[0] != stream.lengths.shape[0] or tokens.shape[1] < 1:
            raise ValueError(f"extend: tokens must be [{stream.lengths.shape[0]}, at least 1], got {tuple(tokens.shape)}")
        if stream.model is not self:
            raise ValueError("extend: another model's stream")
        if stream.broken:
            raise RuntimeError("extend: an earlier call ended with an error, and the stream's layers are not alike")
        stream.broken = True
        x, branch = self.embed(tokens), None
        for block, state in zip(self.blocks, stream.layers):
            if self.fused_norms:
                branch, x = block.forward_fused(branch, x, state)
            else:
                x = block(x, state)
        stream.lengths += tokens.shape[1]
        stream.broken = False
        return self._head(None if branch is None else branch[:, -1:], x[:, -1:])[:, 0]

    @torch.no_grad()
    def generate(self, tokens, count: int, *, temperature=1.0, top_k=None, top_p=None, min_p=None,
                 generator: torch.Generator | None = None, stream: "ModelStream | None" = None):
        """``count`` further tokens ``[B,count]`` of the sequences that ``tokens
        [B,T]`` begin (or, with a ``stream``, go on), drawn by
        :func:`thetascan_b200.sample_tokens` with its settings.  A row of logits
        that are all NaN or minus infinity gives -1, and that sequence goes on as
        if it had been token 0, as it does for a -1 among the ``tokens``."""
        if count < 1:
            raise ValueError(f"generate: count must be >= 1, got {count}")
        stream = self.stream(tokens.shape[0]) if stream is None else stream
        uniform = torch.rand(count, tokens.shape[0], dtype=torch.float32, device=tokens.device, generator=generator)
        got = []
        for row in uniform:
            logits = self.extend(tokens.clamp_min(0), stream)
            tokens = sample_tokens(logits, row, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)[:, None]
            got.append(tokens)
        return torch.cat(got, 1)

    def loss(self, tokens):
        """Next-token cross entropy of ``tokens [B,T]`` (predicting 1..T-1)."""
        logits = self(tokens[:, :-1])
        return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), tokens[:, 1:].reshape(-1))


class ModelStream:
    """What a :class:`HybridLM` keeps of its sequences: a ring cache of each
    attention layer, the scan states of each mixer."""

    @torch.inference_mode(False)   # what it keeps is changed in place, in that mode or not
    def __init__(self, model: HybridLM, batch: int):
        if batch < 1:
            raise ValueError(f"a stream needs at least one sequence, got {batch}")
        self.model, self.broken = model, False
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=model.embed.weight.device)
        self.layers = []
        for block in model.blocks:
            mix = block.mix
            if isinstance(mix, ThetaScan):
                self.layers.append(ScanStream())
            elif isinstance(mix, CausalAttention) and mix.window is not None:
                width = mix.qkv.in_features // mix.n_heads
                self.layers.append(AttentionStream(self.lengths, mix.n_heads, width, mix.window, mix.sinks))
            else:
                raise TypeError("a stream needs attention with a window and this package's mixers")


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
    ap.add_argument("--window", type=int, help="attention over so many last tokens")
    ap.add_argument("--sinks", type=int, default=0, help="and over so many first ones")
    ap.add_argument("--generate", type=int, default=0, metavar="N", help="let the model go on by N tokens (needs --window)")
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    if a.generate and a.window is None:
        ap.error("--generate needs --window")
    if a.sinks and a.window is None:
        ap.error("--sinks needs --window")
    torch.manual_seed(0)
    model = HybridLM(gated=a.gated, fused_norms=True, window=a.window, sinks=a.sinks).cuda()
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
    if a.generate:
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            stream = model.stream(a.batch)
            first = model.generate(data, 1, top_k=50, stream=stream)
            torch.cuda.synchronize()
            start = time.perf_counter()
            got = model.generate(first, a.generate, top_k=50, stream=stream)
            torch.cuda.synchronize()
        print(f"{got.numel()} tokens behind {tuple(data.shape)}: {(time.perf_counter() - start) * 1e3 / a.generate:.2f} ms a step")


if __name__ == "__main__":
    main()
