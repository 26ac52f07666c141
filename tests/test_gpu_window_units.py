"""Windowed attention with more units (query or key tiles, or pairs of them) than the 148 CTAs that take them, so that a CTA
has several: the orders in which they come with and without lengths, at both widths of the kernels, and first tokens whose
queries are split among CTAs in several sequences.  Against the definition in 64 bits (window_definition.py, which derives
the bounds)."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_window import _make, _within, win  # noqa: F401  (win: a fixture)
from window_definition import attention

gpu = pytest.mark.gpu


def _check(win, q, k, v, dy, window, sinks, lengths):  # noqa: F811
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = win.window_attention(*leaves, window, sinks, lengths=lengths)
    grads = torch.autograd.grad(y, leaves, dy)
    for b in range(q.shape[0]):   # one sequence at a time: the definition has every pair in 64 bits
        s = slice(b, b + 1)
        want, want_grads, bounds = attention(*(t[s].double() for t in (q, k, v)), window, sinks, 1 / math.sqrt(q.shape[-1]),
                                             None if lengths is None else lengths[s], dy[s].double())
        for got, w, bound in zip((y.detach(), *grads), (want, *want_grads), bounds):
            _within(got[s], w, bound)
    with torch.no_grad():
        assert torch.equal(win.window_attention(q, k, v, window, sinks, lengths=lengths), y)
    again = torch.autograd.grad(win.window_attention(*leaves, window, sinks, lengths=lengths), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


# batch, heads, kv_heads, tokens, past, dim, window, sinks; pairs of query tiles, query tiles and key tiles are each above 148
CASES = [
    (5, 8, 8, 900, 0, 64, 256, 4), (5, 8, 8, 1000, 0, 64, 70, 0), (2, 12, 6, 1700, 0, 128, 200, 130), (2, 12, 6, 1700, 0, 128, 600, 0),
    (3, 20, 5, 1300, 200, 80, 300, 5), (3, 18, 6, 1290, 0, 48, 129, 300), (20, 6, 2, 500, 70, 96, 100, 1), (160, 1, 1, 300, 0, 128, 40, 2)]


def _units(batch, heads, kv_heads, tokens, past):
    share, tiles = heads // kv_heads, -(-tokens // 128)
    return batch * kv_heads * min(-(-share * tiles // 2), -(-(tokens + past) // 128))


@gpu
@pytest.mark.parametrize("case", CASES)
def test_more_units_than_ctas(win, case):  # noqa: F811
    batch, heads, kv_heads, tokens, past, dim, window, sinks = case
    assert _units(*case[:5]) > 148
    q, k, v, dy, _ = _make(batch, heads, kv_heads, tokens, past, dim, False, seed=tokens)
    _check(win, q, k, v, dy, window, sinks, None)


@gpu
@pytest.mark.parametrize("case", CASES)
def test_more_units_than_ctas_of_any_length(win, case):  # noqa: F811
    batch, heads, kv_heads, tokens, past, dim, window, sinks = case
    q, k, v, dy, lengths = _make(batch, heads, kv_heads, tokens, past, dim, True, seed=tokens + 1)
    lengths[-1] = tokens + past
    lengths[batch // 2] = past + 1
    _check(win, q, k, v, dy, window, sinks, lengths)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ragged", [False, True])
def test_split_first_tokens_of_several_sequences(win, dim, ragged):  # noqa: F811
    # few units, so that the split ones come in every order; three chunks of eight query tiles, two tiles of first tokens
    q, k, v, dy, lengths = _make(3, 4, 2, 2300, 100, dim, ragged, seed=7)
    _check(win, q, k, v, dy, 150, 200, lengths)


@gpu
def test_a_sequence_alone_and_in_a_batch(win):  # noqa: F811
    # the order of units changes no result
    q, k, v, dy, _ = _make(5, 8, 8, 900, 0, 64, False, seed=3)

    def step(s):
        leaves = [t[s].detach().requires_grad_(True) for t in (q, k, v)]
        y = win.window_attention(*leaves, 256, 4)
        return y.detach(), *torch.autograd.grad(y, leaves, dy[s])

    together = step(slice(None))
    for b in range(5):
        s = slice(b, b + 1)
        assert all(torch.equal(a[s], one) for a, one in zip(together, step(s)))


@gpu
@pytest.mark.parametrize("batch,kv_heads,tokens,dim", [(20, 8, 1300, 64), (8, 8, 5000, 64), (8, 8, 5000, 128)])
@pytest.mark.parametrize("ragged", [False, True])
def test_first_tokens_in_fewer_chunks(win, batch, kv_heads, tokens, dim, ragged):  # noqa: F811
    # 1280 and 512 key tiles of first tokens: their queries in one and in four chunks, in place of two and five
    q, k, v, dy, lengths = _make(batch, kv_heads, kv_heads, tokens, 0, dim, ragged, seed=2)
    _check(win, q, k, v, dy, 100, 1000, lengths)
