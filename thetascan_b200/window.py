"""Causal attention over a sliding window, with first tokens that stay visible.

The query at position ``i`` sees the keys at ``j <= i`` with ``i - j < window``
or ``j < sinks``:

* :func:`window_attention` -- many queries at a time (training, prompts, the
  next piece of a long prompt), with gradients;
* :func:`window_attention_step` -- one new token of each sequence over a ring
  cache of ``sinks + window`` slots, which it enters;
* :func:`window_cache_extend` -- copies a prompt's keys and values into such a
  cache;
* :class:`WindowCache` -- the cache's tensors with these two as methods.

bf16 tensors ``[batch, heads, tokens, head width]`` of any strides (channels
contiguous and 16-byte steps are read in place, others are copied first), head
widths that are multiples of 8 up to 128, key heads that several query heads
share.  Scores, softmax statistics and sums are f32; the weights are rounded to
bf16 as operands of the product with the values, and so are the scores'
gradients.  The results do not depend on timing.

``lengths`` (int32, one per sequence) ends the sequences of a padded batch:
positions at or behind a sequence's length are seen by none and see none; their
rows of the output and of the gradients are zero, and what lies in them does not
matter.  (An infinity or NaN within a sequence may reach the rows of other
positions within its 128: a hidden pair's weight of zero is multiplied by it.)
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import _lib

LIB = "thetascan_b200"


def _token_major(t: Tensor) -> Tensor:
    """An empty ``[B, H, T, D]`` whose heads lie together for each token."""
    b, h, n, d = t.shape
    return t.new_empty(b, n, h, d).transpose(1, 2)


@torch.library.custom_op(f"{LIB}::window_fwd", mutates_args=())
def window_fwd(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, scale: float, lengths: Optional[Tensor],
               keep: bool) -> tuple[Tensor, Tensor]:
    """The attention, and the log-sum-exp of its rows for the backward (empty unless ``keep``)."""
    y, lse = _lib.host().window_fwd(q, k, v, window, sinks, scale, lengths, keep)
    return y, q.new_empty(0, dtype=torch.float32) if lse is None else lse


@window_fwd.register_fake
def _(q, k, v, window, sinks, scale, lengths, keep):
    b, h, n, _ = q.shape
    return _token_major(q), q.new_empty((b, h, -(-n // 128) * 128) if keep else (0,), dtype=torch.float32)


@torch.library.custom_op(f"{LIB}::window_bwd", mutates_args=())
def window_bwd(dy: Tensor, q: Tensor, k: Tensor, v: Tensor, y: Tensor, lse: Tensor, window: int, sinks: int, scale: float,
               lengths: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients of q, k and v."""
    return _lib.host().window_bwd(dy, q, k, v, y, lse, window, sinks, scale, lengths)


@window_bwd.register_fake
def _(dy, q, k, v, y, lse, window, sinks, scale, lengths):
    return _token_major(q), _token_major(k), _token_major(v)


@torch.library.custom_op(f"{LIB}::window_step", mutates_args=("keys", "values"))
def window_step(q: Tensor, k: Tensor, v: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, sinks: int,
                scale: float) -> Tensor:
    """One token's attention; its key and value enter the cache."""
    return _lib.host().window_step(q, k, v, keys, values, lengths, sinks, scale)


@window_step.register_fake
def _(q, k, v, keys, values, lengths, sinks, scale):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{LIB}::window_extend", mutates_args=("keys", "values"))
def window_extend(k: Tensor, v: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, sinks: int,
                  new: Optional[Tensor]) -> None:
    """Keys and values of new tokens into the cache."""
    _lib.host().window_extend(k, v, keys, values, lengths, sinks, new)


@window_extend.register_fake
def _(k, v, keys, values, lengths, sinks, new):
    return None


class _TracedWindow(torch.autograd.Function):
    """The autograd node as a tracing compiler sees it; eager calls have theirs in ``csrc/host.cpp``."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, lengths):
        y, lse = window_fwd(q, k, v, window, sinks, scale, lengths, True)
        ctx.sizes = window, sinks, scale
        ctx.save_for_backward(q, k, v, y, lse, lengths)
        return y

    @staticmethod
    def backward(ctx, dy):
        *kept, lengths = ctx.saved_tensors
        return (*window_bwd(dy, *kept, *ctx.sizes, lengths), None, None, None, None)


def _scale(scale, q):
    return 1 / math.sqrt(q.shape[-1]) if scale is None else float(scale)


def window_attention(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int = 0, *, scale: Optional[float] = None,
                     lengths: Optional[Tensor] = None) -> Tensor:
    """``softmax(scale q k^T) v`` over the visible keys, ``[B, H, T, D]`` bf16.

    ``q`` is ``[B, H, T, D]``, ``k`` and ``v`` are ``[B, G, S, D]`` with ``G``
    dividing ``H`` (query head ``h`` reads key head ``h // (H // G)``) and
    ``S >= T``: the queries are the last ``T`` of ``S`` positions.  ``scale`` is
    ``D ** -0.5`` unless given.  ``lengths`` ``[B]`` counts each sequence's
    positions.  The output's heads lie together for each token."""
    if torch.compiler.is_compiling():
        scale = _scale(scale, q)
        if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
            return _TracedWindow.apply(q, k, v, window, sinks, scale, lengths)
        return window_fwd(q, k, v, window, sinks, scale, lengths, False)[0]
    return _lib.host().window_attention(q, k, v, window, sinks, scale, lengths)


def window_attention_step(q: Tensor, k: Tensor, v: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, sinks: int = 0, *,
                          scale: Optional[float] = None) -> Tensor:
    """The attention of one new token of each sequence, ``q [B, H, 1, D]``.

    ``keys`` and ``values`` ``[B, G, sinks + window, D]`` are the ring cache:
    position ``j`` lies in slot ``j`` below ``sinks``, in slot ``sinks + (j -
    sinks) % window`` above.  The token's ``k`` and ``v`` ``[B, G, 1, D]`` enter
    it at position ``lengths[b]``, the number of tokens before it.  ``lengths``
    (int32) is not changed, so that the layers of a model can share it; a
    negative one marks a row without a sequence, for which nothing is written and
    the output is zero.  For inference: no gradient."""
    if torch.compiler.is_compiling():
        _lib.refuse_gradient("window_attention_step", q, k, v, keys, values)
        return window_step(q, k, v, keys, values, lengths, sinks, _scale(scale, q))
    return _lib.host().window_step(q, k, v, keys, values, lengths, sinks, scale)


def window_cache_extend(k: Tensor, v: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, sinks: int = 0, *,
                        new: Optional[Tensor] = None) -> None:
    """Copy new tokens' ``k`` and ``v`` ``[B, G, T, D]`` into a ring cache (see
    :func:`window_attention_step`) behind ``lengths`` tokens: those that the cache
    has slots for.  ``new`` (int32) counts each sequence's tokens among the ``T``.
    ``lengths`` is not changed; slots that no new token falls into are left as
    they were, and so is the whole row of a negative length."""
    if torch.compiler.is_compiling():
        _lib.refuse_gradient("window_cache_extend", k, v, keys, values)
        return window_extend(k, v, keys, values, lengths, sinks, new)
    return _lib.host().window_extend(k, v, keys, values, lengths, sinks, new)


class WindowCache:
    """A ring cache of ``sinks + window`` keys and values for each of ``batch``
    sequences: ``keys`` and ``values``, without the lengths, which the layers of a
    model share."""

    @torch.inference_mode(False)   # what it keeps is changed in place, in that mode or not
    def __init__(self, batch: int, heads: int, head_dim: int, window: int, sinks: int = 0, *, device=None):
        if window < 1 or sinks < 0:
            raise ValueError(f"window must be >= 1 and sinks >= 0, got {window} and {sinks}")
        shape = (batch, heads, sinks + window, head_dim)
        self.sinks = sinks
        self.keys, self.values = (torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(2))

    def extend(self, k: Tensor, v: Tensor, lengths: Tensor, *, new: Optional[Tensor] = None) -> None:
        window_cache_extend(k, v, self.keys, self.values, lengths, self.sinks, new=new)

    def step(self, q: Tensor, k: Tensor, v: Tensor, lengths: Tensor, *, scale: Optional[float] = None) -> Tensor:
        return window_attention_step(q, k, v, self.keys, self.values, lengths, self.sinks, scale=scale)
