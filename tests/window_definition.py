"""Attention over a sliding window with first tokens, from its definition in 64 bits, with bounds of what the kernels'
roundings can do to it.

The kernels round the weights p to bf16 before the product with the values, and p and ds before the products of the
gradients; every result is rounded once.  A rounding to bf16 is off by at most 2^-8 of the value.  f32 enters by the
scores (a sum of up to 128 products), exp2 and the sums: ``F32`` of the magnitudes covers it.  delta = dy.y takes the
rounded y."""
from __future__ import annotations

import torch

HALF = 2.0 ** -8
F32 = 2e-4


def visible(q_tokens, tokens, window, sinks, lengths, device):
    i = torch.arange(tokens - q_tokens, tokens, device=device)[:, None]
    j = torch.arange(tokens, device=device)
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    if lengths is None:
        return seen[None, None]
    n = lengths.to(device).view(-1, 1, 1, 1)
    return seen & (i < n) & (j < n)


def attention(q, k, v, window, sinks, scale, lengths=None, dy=None):
    """``(y, (dq, dk, dv), bounds)`` of 64-bit inputs; bounds of y and, with ``dy``, of the gradients."""
    share = q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    seen = visible(q.shape[2], k.shape[2], window, sinks, lengths, q.device)
    s = (q @ kk.transpose(-1, -2) * scale).masked_fill(~seen, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -torch.inf, 0))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    y = p @ vv
    size = p @ vv.abs()
    y_off = (HALF + F32) * size + HALF * y.abs()
    if dy is None:
        return y, None, (y_off,)

    def shared(t):
        return t.unflatten(1, (k.shape[1], share)).sum(2)

    dp = dy @ vv.transpose(-1, -2)
    ds = p * (dp - (dy * y).sum(-1, keepdim=True))
    pt, dst = p.transpose(-1, -2), ds.transpose(-1, -2)
    dq, dk, dv = ds @ kk * scale, shared(dst @ q) * scale, shared(pt @ dy)
    # ds: its own rounding, f32 in p and in dp, and y's error in delta
    ds_off = HALF * ds.abs() + p * (F32 * (dy.abs() @ vv.abs().transpose(-1, -2) + (dy * y).abs().sum(-1, keepdim=True)) +
                                    (dy.abs() * y_off).sum(-1, keepdim=True)) * (1 + HALF)
    off = (ds_off @ kk.abs() * scale + HALF * dq.abs(), shared(ds_off.transpose(-1, -2) @ q.abs()) * scale + HALF * dk.abs(),
           shared(pt @ dy.abs()) * (HALF + F32) + HALF * dv.abs())
    return y, (dq, dk, dv), (y_off, *off)
