"""The choice of a token from logits, by given uniform numbers.

:func:`sample_tokens` filters by temperature, top-k, top-p and min-p and draws a
token for each row in one kernel (``csrc/sample.cu``) that reads the logits once.
The result is a function of its arguments: probabilities are summed as integers
of 2^-40 of the largest one, in no particular order.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor

from . import _lib

LIB = "thetascan_b200"


@torch.library.custom_op(f"{LIB}::sample", mutates_args=())
def _sample(logits: Tensor, uniform: Tensor, temperature: float, temperatures: Optional[Tensor], top_k: Optional[int],
            top_ks: Optional[Tensor], top_p: float, top_ps: Optional[Tensor], min_p: float, min_ps: Optional[Tensor],
            logprobs: bool) -> tuple[Tensor, Tensor]:
    """Tokens and their log-probabilities (empty unless wanted); each setting as a number or a tensor."""
    settings = (temperatures if temperatures is not None else temperature, top_ks if top_ks is not None else top_k,
                top_ps if top_ps is not None else top_p, min_ps if min_ps is not None else min_p)
    got = _lib.host().sample(logits, uniform, *settings, logprobs)
    return got if logprobs else (got, logits.new_empty(0, dtype=torch.float32))


@_sample.register_fake
def _(logits, uniform, temperature, temperatures, top_k, top_ks, top_p, top_ps, min_p, min_ps, logprobs):
    return (logits.new_empty(uniform.shape, dtype=torch.int64),
            logits.new_empty(uniform.shape if logprobs else (0,), dtype=torch.float32))


def sample_tokens(logits: Tensor, uniform: Tensor, *, temperature: Union[float, Tensor] = 1.0,
                  top_k: Union[int, Tensor, None] = None, top_p: Union[float, Tensor, None] = None,
                  min_p: Union[float, Tensor, None] = None, return_logprobs: bool = False):
    """A token for each row of ``logits [..., vocabulary]`` (f32 or bf16), int64.

    Tokens rank by falling logit, the lower index first among equals.  Of them
    ``top_k`` keeps the first so many, ``top_p`` the shortest prefix of those that
    holds this share of their probability, ``min_p`` those of that with at least
    this share of the largest probability.  The token is the first, by index, at
    which the running sum of the kept probabilities exceeds ``uniform`` (f32, in
    ``[0, 1)``, one for each row) times their total.

    Each setting is one number or a tensor with a value for each row (f32;
    ``top_k`` of an integer type).  ``temperature`` 0 takes the largest logit.
    Numbers out of range raise ``ValueError``; in a tensor they have a meaning
    (which is cheaper than looking): a temperature that is not above 0 is 0,
    ``top_k`` below 1, ``top_p`` from 1 on and ``min_p`` up to 0 do not filter,
    ``top_p`` up to 0 keeps one token, ``min_p`` above 1 is 1, and an infinite
    temperature is the largest number.

    A NaN or minus infinity is a masked token; a row of nothing else gives -1.
    Infinities share a row's probability.  A token under 2^-41 of the largest
    probability is never drawn.  With ``return_logprobs`` the result is ``(tokens,
    logprobs)``: ``log_softmax(logits / temperature)`` at the token, before the
    filters (with temperature 1 in a greedy row; minus infinity for token -1)."""
    if not torch.compiler.is_compiling():
        return _lib.host().sample(logits, uniform, temperature, top_k, top_p, min_p, return_logprobs)
    if return_logprobs and torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("sample_tokens: the log-probabilities have no gradient: call it under torch.no_grad()")

    def split(value, off):
        return (off, value) if isinstance(value, Tensor) else (off if value is None else value, None)

    tokens, logprobs = _sample(logits.detach(), uniform, *split(temperature, 1.0), *split(top_k, None), *split(top_p, 1.0),
                               *split(min_p, 0.0), return_logprobs)
    return (tokens, logprobs) if return_logprobs else tokens
