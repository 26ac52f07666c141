"""The gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T``.

* :func:`gated_ffn` -- the function, with its gradients;
* :class:`GatedFFN` -- the module, with ``torch.nn.Linear`` weight layouts.

The kernels (``csrc/ffn.cu``) form both projections, the activation and the
product in one launch and the down projection in a second.  For a backward
pass the block keeps its input and 8 bytes per hidden value (10 with up to 32
rows): ``h`` in bf16 and both projections in 24 bits.  bf16 operands, f32 accumulators.  Any number of
rows; widths that are multiples of 8.

What is rounded on the way: ``h`` to bf16 between the two launches, and ``dg``
and ``du`` in the backward, as operands of the next product.  A result's error
is then 2.35e-3 of its norm, where its own rounding to bf16 alone is 1.66e-3.
With up to 32 rows, where a few large hidden values may carry a result, each of
the three passes in two bf16 parts, which leaves the result's own rounding
alone; so the same row comes out the same within that rounding, not to the bit,
from a call with more rows.  The output does not depend on whether gradients are
wanted, and a compiled call computes what the eager one does.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib

LIB = "thetascan_b200"
ACTIVATIONS = ("gelu", "relu2", "silu")
KEPT_BLOCK = 6144   # bytes kept for each 32 rows x 32 hidden columns
TWO_PART_ROWS = 32  # rows up to which h is kept in two parts


def _kept_bytes(rows, hidden):
    return -(-rows // 32) * -(-hidden // 32) * KEPT_BLOCK


def _or_empty(t, like, dtype=None):
    return like.new_empty(0, dtype=dtype) if t is None else t


@torch.library.custom_op(f"{LIB}::gated_ffn_fwd", mutates_args=())
def gated_ffn_fwd(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: str,
                  keep: bool) -> tuple[Tensor, Tensor, Tensor]:
    """The block's output, and what its backward reads: h and the projections (empty unless ``keep``)."""
    y, h, kept = _lib.host().ffn_fwd(x, w_gate, w_up, w_down, activation, keep)
    return y, _or_empty(h, x), _or_empty(kept, x, torch.uint8)


@gated_ffn_fwd.register_fake
def _(x, w_gate, w_up, w_down, activation, keep):
    rows, hidden = x.numel() // x.shape[-1], w_gate.shape[0]
    parts = 2 if rows <= TWO_PART_ROWS else 1
    return (x.new_empty(*x.shape[:-1], w_down.shape[0]), x.new_empty((parts * rows, hidden) if keep else (0,)),
            x.new_empty(_kept_bytes(rows, hidden) if keep else 0, dtype=torch.uint8))


@torch.library.custom_op(f"{LIB}::gated_ffn_bwd", mutates_args=())
def gated_ffn_bwd(dy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, h: Tensor, kept: Tensor,
                  activation: str, wanted: list[bool]) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients of x, w_gate, w_up, w_down (empty where not wanted)."""
    grads = _lib.host().ffn_bwd(dy, x, w_gate, w_up, w_down, h, kept, activation, wanted)
    return tuple(_or_empty(g, x) for g in grads)


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, h, kept, activation, wanted):
    return tuple(t.new_empty(t.shape if need else (0,)) for t, need in zip((x, w_gate, w_up, w_down), wanted))


class _TracedFFN(torch.autograd.Function):
    """The autograd node as a tracing compiler sees it; eager calls have theirs in ``csrc/host.cpp``."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        y, h, kept = gated_ffn_fwd(x, w_gate, w_up, w_down, activation, True)
        ctx.activation = activation
        ctx.save_for_backward(x, w_gate, w_up, w_down, h, kept)
        return y

    @staticmethod
    def backward(ctx, dy):
        wanted = list(ctx.needs_input_grad[:4])
        grads = gated_ffn_bwd(dy, *ctx.saved_tensors, ctx.activation, wanted)
        return (*(t if need else None for t, need in zip(grads, wanted)), None)


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: str = "silu") -> Tensor:
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T`` over the last dimension of
    ``x [..., width]``; ``w_gate`` and ``w_up`` are ``[hidden, width]``,
    ``w_down`` is ``[width_out, hidden]``, all bf16.  ``activation`` is
    ``"silu"``, ``"gelu"`` (exact) or ``"relu2"`` (``max(g, 0)^2``)."""
    if torch.compiler.is_compiling():
        if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
            return _TracedFFN.apply(x, w_gate, w_up, w_down, activation)
        return gated_ffn_fwd(x, w_gate, w_up, w_down, activation, False)[0]
    return _lib.host().gated_ffn(x, w_gate, w_up, w_down, activation)


class GatedFFN(nn.Module):
    """Gated feed-forward block with weights ``gate`` and ``up`` ``[hidden,
    d_model]`` and ``down`` ``[d_model, hidden]`` (no biases).  Operands are
    rounded to bf16 where they are kept wider; the output has the type of the
    input."""

    def __init__(self, d_model: int, hidden: int, activation: str = "silu", *, device=None,
                 dtype: Optional[torch.dtype] = None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {ACTIVATIONS}, got {activation!r}")
        if d_model < 8 or hidden < 8 or d_model % 8 or hidden % 8:
            raise NotImplementedError("gated_ffn: widths must be nonzero multiples of 8")
        kw = dict(bias=False, device=device, dtype=dtype)
        self.gate, self.up = nn.Linear(d_model, hidden, **kw), nn.Linear(d_model, hidden, **kw)
        self.down = nn.Linear(hidden, d_model, **kw)
        self.activation = activation

    def forward(self, x):
        bf = torch.bfloat16
        y = gated_ffn(x.to(bf), self.gate.weight.to(bf), self.up.weight.to(bf), self.down.weight.to(bf),
                      self.activation)
        return y.to(x.dtype)
