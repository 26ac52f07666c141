"""Windowed attention and its ring cache on the GPU against the definition in 64 bits (window_definition.py, which
derives the bounds)."""
from __future__ import annotations

import math

import pytest
import torch

from window_definition import F32, HALF, attention

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def win():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import window
    return window


def _make(batch, heads, kv_heads, tokens, past, dim, ragged, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(n, h, scale=1.0):
        return (torch.randn(batch, n, h, dim, generator=g, device="cuda") * scale).to(BF16).transpose(1, 2)

    lengths = None
    if ragged:
        lengths = torch.randint(0, tokens + past + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = 0 if seed % 2 else tokens + past
    return normal(tokens, heads, 1.5), normal(tokens + past, kv_heads), normal(tokens + past, kv_heads), normal(tokens, heads), lengths


def _within(got, want, bound):
    assert got.shape == want.shape and got.dtype == BF16
    over = (got.double() - want).abs() - bound - 1e-6
    assert not torch.isnan(got).any() and float(over.max()) <= 0, float(over.max())


# batch, heads, kv_heads, tokens, past, dim, window, sinks, ragged
CASES = [
    (1, 1, 1, 1, 0, 64, 16, 0, False), (1, 1, 1, 128, 0, 64, 128, 0, False), (2, 2, 2, 300, 0, 64, 100, 0, False),
    (1, 2, 1, 512, 0, 128, 128, 4, False), (2, 6, 2, 517, 0, 80, 150, 3, True), (3, 3, 3, 700, 0, 64, 64, 130, True),
    (2, 4, 4, 260, 777, 128, 200, 20, False), (1, 5, 1, 390, 100, 96, 9, 1, False), (2, 3, 1, 300, 0, 64, 100, 300, False),
    (1, 2, 2, 1, 500, 64, 100, 7, False), (2, 2, 1, 1000, 0, 128, 4000, 0, True), (2, 9, 3, 333, 55, 8, 40, 200, True),
    (1, 1, 1, 2000, 0, 16, 1, 0, False), (4, 1, 1, 129, 3, 64, 2, 129, True), (1, 8, 1, 255, 0, 120, 127, 1, False),
    (1, 4, 2, 2500, 0, 128, 260, 16, False), (5, 1, 1, 64, 64, 40, 10_000_000, 5, True), (1, 1, 1, 1300, 0, 64, 1, 257, False)]


@gpu
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(win, case):
    batch, heads, kv_heads, tokens, past, dim, window, sinks, ragged = case
    q, k, v, dy, lengths = _make(batch, heads, kv_heads, tokens, past, dim, ragged, seed=tokens)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = win.window_attention(*leaves, window, sinks, lengths=lengths)
    grads = torch.autograd.grad(y, leaves, dy)
    want, want_grads, bounds = attention(*(t.double() for t in (q, k, v)), window, sinks, 1 / math.sqrt(dim), lengths, dy.double())
    for got, w, bound in zip((y.detach(), *grads), (want, *want_grads), bounds):
        _within(got, w, bound)
    with torch.no_grad():
        assert torch.equal(win.window_attention(q, k, v, window, sinks, lengths=lengths), y)
    again = torch.autograd.grad(win.window_attention(*leaves, window, sinks, lengths=lengths), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # no order of sums depends on timing


@gpu
@pytest.mark.parametrize("batch,heads,kv_heads,tokens,past,dim,sinks", [(64, 2, 1, 300, 0, 64, 3), (65, 2, 2, 200, 30, 64, 0), (33, 3, 1, 140, 7, 72, 140)])
def test_many_sequences_of_any_length(win, batch, heads, kv_heads, tokens, past, dim, sinks):
    q, k, v, dy, lengths = _make(batch, heads, kv_heads, tokens, past, dim, True, seed=batch)
    lengths[5:9], lengths[20:24] = tokens + past, 0   # equal ones among them
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = win.window_attention(*leaves, 90, sinks, lengths=lengths)
    grads = torch.autograd.grad(y, leaves, dy)
    want, want_grads, bounds = attention(*(t.double() for t in (q, k, v)), 90, sinks, 1 / math.sqrt(dim), lengths, dy.double())
    for got, w, bound in zip((y.detach(), *grads), (want, *want_grads), bounds):
        _within(got, w, bound)


@gpu
def test_rows_that_see_nothing_are_zero(win):
    q, k, v, dy, _ = _make(3, 4, 2, 200, 100, 64, False)
    lengths = torch.tensor([0, 150, 100], dtype=torch.int32, device="cuda")   # none, 50 queries, keys but no query
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = win.window_attention(*leaves, 30, 2, lengths=lengths)
    dq, dk, dv = torch.autograd.grad(y, leaves, dy)
    assert not y[0].any() and not y[2].any() and not y[1, :, 50:].any() and y[1, :, 49].any()
    for g in (dk, dv):
        assert not g[0].any() and not g[2].any() and not g[1, :, 150:].any() and g[1, :, 149].any()
    assert not dq[0].any() and not dq[2].any() and not dq[1, :, 50:].any()


@gpu
@pytest.mark.parametrize("dim,past,window,sinks", [(64, 0, 100, 4), (128, 0, 300, 0), (80, 77, 150, 130), (128, 40, 64, 200)])
@pytest.mark.parametrize("filling", [math.nan, math.inf])
def test_what_lies_behind_a_sequence_does_not_matter(win, dim, past, window, sinks, filling):
    q, k, v, dy, _ = _make(4, 4, 2, 330, past, dim, False, seed=dim)
    lengths = torch.tensor([330 + past, 257 + past, 1 + past, 0], dtype=torch.int32, device="cuda")
    behind = torch.arange(330 + past, device="cuda")[None] >= lengths[:, None]
    got = []
    for fill in (0.0, filling):
        parts = [t.masked_fill(behind[:, None, -t.shape[2]:, None], fill) for t in (q, k, v, dy)]
        leaves = [t.requires_grad_(True) for t in parts[:3]]
        y = win.window_attention(*leaves, window, sinks, lengths=lengths)
        got.append((y.detach(), *torch.autograd.grad(y, leaves, parts[3])))
    for a, b in zip(*got):
        assert torch.isfinite(b).all() and torch.equal(a, b)


@gpu
def test_layouts(win):
    g = torch.Generator("cuda").manual_seed(3)
    qkv = torch.randn(2, 150, 3, 4, 64, generator=g, device="cuda").to(BF16)
    q, k, v = qkv.permute(2, 0, 3, 1, 4)
    want = win.window_attention(*(t.contiguous() for t in (q, k, v)), 40, 3)
    assert torch.equal(win.window_attention(q, k, v, 40, 3), want)
    # a base that is no multiple of 16 bytes, channels that are not contiguous, keys that all heads share by expansion
    flat = torch.empty(2 * 4 * 150 * 64 + 1, dtype=BF16, device="cuda")
    odd = flat[1:].view(2, 4, 150, 64).copy_(q)
    assert torch.equal(win.window_attention(odd, k, v, 40, 3), want)
    turned = k.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(win.window_attention(q, turned, v, 40, 3), want)
    one_k, one_v = k[:, :1], v[:, :1]
    shared = win.window_attention(q, one_k, one_v, 40, 3)
    leaf_k, leaf_v = (t.detach().requires_grad_(True) for t in (one_k, one_v))
    y = win.window_attention(q, leaf_k.expand(2, 4, 150, 64), leaf_v.expand(2, 4, 150, 64), 40, 3)
    assert torch.equal(y, shared)
    by_expansion = torch.autograd.grad(y, (leaf_k, leaf_v), q)
    by_sharing = torch.autograd.grad(win.window_attention(q, leaf_k, leaf_v, 40, 3), (leaf_k, leaf_v), q)
    for a, b in zip(by_expansion, by_sharing):   # four roundings and three sums in bf16, against one rounding
        assert float((a.double() - b.double()).abs().max()) <= 8 * HALF * float(b.abs().max())
    # a gradient that comes expanded
    q1 = q.detach().requires_grad_(True)
    a, = torch.autograd.grad(win.window_attention(q1, k, v, 40, 3).sum(), q1)
    b, = torch.autograd.grad(win.window_attention(q1, k, v, 40, 3), q1, torch.ones_like(q))
    assert torch.equal(a, b)


@gpu
def test_scale_and_large_scores(win):
    q, k, v, _, _ = _make(1, 2, 2, 300, 0, 64, False)
    # scores up to a few hundred: the softmax is nearly one-hot, and its reference moves by large steps
    scale = 4.0
    got = win.window_attention(q, k, v, 90, 2, scale=scale)
    want, _, (bound,) = attention(q.double(), k.double(), v.double(), 90, 2, scale)
    # f32 scores of magnitude 500 are off by up to 500 * 2^-23 * a few: 2e-4 of a weight
    _within(got, want, bound + 1e-3)


@gpu
def test_empty_sizes(win):
    for shape in [(0, 2, 5, 64), (2, 2, 0, 64)]:
        q = torch.zeros(shape, dtype=BF16, device="cuda", requires_grad=True)
        k = torch.zeros(shape[0], 2, shape[2] + 3, 64, dtype=BF16, device="cuda", requires_grad=True)
        y = win.window_attention(q, k, k, 4)
        assert y.shape == shape
        y.sum().backward()
        assert k.grad.shape == k.shape and not k.grad.any()


@gpu
def test_streams_graphs_and_devices(win):
    q, k, v, dy, _ = _make(2, 4, 2, 300, 0, 64, False)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def step():
        y = win.window_attention(*leaves, 70, 3)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs of the same call, replayed in turn with other inputs
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        leaves[0].copy_(leaves[0].flip(2))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
def test_refusals(win):
    q, k, v, dy, _ = _make(2, 4, 2, 20, 0, 64, False)
    attend = win.window_attention
    for bad in (lambda: attend(q.float(), k, v, 4), lambda: attend(q[0], k, v, 4), lambda: attend(q, k, v[:, :1], 4),
                lambda: attend(q, k[:, :, :10], v[:, :, :10], 4), lambda: attend(q[:, :3], k, v, 4),
                lambda: attend(q, k, v, 0), lambda: attend(q, k, v, 4, -1), lambda: attend(q, k, v, 4, scale=0.0),
                lambda: attend(q, k, v, 4, scale=math.nan), lambda: attend(q, k, v, 4, lengths=torch.zeros(2, device="cuda")),
                lambda: attend(q, k, v, 4, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        attend(q[..., :12], k[..., :12], v[..., :12], 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        attend(q, k.cpu(), v, 4)
    leaf = q.detach().requires_grad_(True)
    y = attend(leaf, k, v, 4)
    dq, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
    assert dq.shape == q.shape
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(y, leaf, dy.detach().requires_grad_(True), create_graph=True)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            attend(fwd.make_dual(q, q), k, v, 4)


@gpu
def test_compiles_into_one_graph(win):
    torch._dynamo.reset()
    q, k, v, dy, lengths = _make(2, 4, 2, 150, 0, 64, True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def f(q, k, v):
        return win.window_attention(q, k, v, 40, 3, lengths=lengths) * 2

    want = torch.autograd.grad(f(*leaves), leaves, dy)
    got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ ring cache

def _slot(position, window, sinks):
    return position if position < sinks else sinks + (position - sinks) % window


# batch, heads, kv_heads, dim, window, sinks, tokens of each sequence before the new one
STEPS = [
    (1, 1, 1, 64, 16, 0, [0]), (1, 8, 8, 64, 256, 4, [255]), (3, 4, 2, 128, 40, 4, [0, 3, 4]), (4, 8, 1, 96, 100, 7, [6, 7, 106, 107]),
    (2, 20, 1, 64, 33, 1, [1000, 33]), (3, 40, 2, 128, 17, 0, [16, 17, 5]), (2, 16, 1, 8, 1, 3, [2, 9]), (2, 6, 2, 40, 500, 200, [199, 5000]),
    (1, 16, 2, 128, 3000, 64, [100_000]), (2, 2, 2, 64, 1, 0, [0, 7]), (3, 9, 3, 120, 130, 30, [-1, 0, 1_000_000_007])]


@gpu
@pytest.mark.parametrize("case", STEPS)
def test_token_over_the_ring_cache(win, case):
    batch, heads, kv_heads, dim, window, sinks, before = case
    g = torch.Generator("cuda").manual_seed(window)
    qkv = torch.randn(batch, 1, heads + 2 * kv_heads, dim, generator=g, device="cuda").to(BF16)
    q, k, v = qkv.transpose(1, 2).split((heads, kv_heads, kv_heads), 1)
    q = q * 1.5
    keys, values = (torch.randn(batch, kv_heads, sinks + window, dim, generator=g, device="cuda").to(BF16) for _ in range(2))
    lengths = torch.tensor(before, dtype=torch.int32, device="cuda")
    for b, n in enumerate(before):   # slots that were never filled may hold anything
        keys[b, :, max(n, 0):] = math.nan if n < sinks + window else 0
        values[b, :, max(n, 0):] = math.inf if n < sinks + window else 0
    old = keys.clone(), values.clone()
    with torch.no_grad():
        y = win.window_attention_step(q, k, v, keys, values, lengths, sinks)
    assert lengths.tolist() == before and y.shape == q.shape
    for b, n in enumerate(before):
        if n < 0:
            assert not y[b].any() and torch.equal(keys[b].nan_to_num(), old[0][b].nan_to_num())
            continue
        slot, filled = _slot(n, window, sinks), min(n + 1, sinks + window)
        for buffer, was, new in ((keys, old[0], k), (values, old[1], v)):
            was[b, :, slot] = new[b, :, 0]
            assert torch.equal(buffer[b].view(torch.int16), was[b].view(torch.int16))
        kk, vv = (t[b:b + 1, :, :filled].double() for t in (keys, values))
        # the one query at the end of the filled slots sees them all
        want, _, (bound,) = attention(q[b:b + 1].double(), kk, vv, filled, 0, 1 / math.sqrt(dim))
        _within(y[b:b + 1], want, bound)


@gpu
def test_generation_is_the_attention_over_everything(win):
    # a prompt of uneven lengths, then tokens one at a time past the window: the rows of one call over all of it
    batch, heads, kv_heads, dim, window, sinks, total = 3, 6, 2, 64, 40, 3, 130
    q, k, v, _, _ = _make(batch, heads, kv_heads, total, 0, dim, False)
    prompt = torch.tensor([1, 37, 90], dtype=torch.int32, device="cuda")
    want, _, (bound,) = attention(q.double(), k.double(), v.double(), window, sinks, dim ** -0.5)
    cache = win.WindowCache(batch, kv_heads, dim, window, sinks, device="cuda")
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        y = win.window_attention(q[:, :, :90], k[:, :, :90], v[:, :, :90], window, sinks, lengths=prompt)
        cache.extend(k[:, :, :90], v[:, :, :90], lengths, new=prompt)
        lengths += prompt
        for b, n in enumerate(prompt.tolist()):
            _within(y[b:b + 1, :, :n], want[b:b + 1, :, :n], bound[b:b + 1, :, :n])
        for _ in range(40):
            at = lengths.long().view(-1, 1, 1, 1)
            now = [t.gather(2, at.expand(-1, t.shape[1], 1, dim)) for t in (q, k, v)]
            y = cache.step(*now, lengths)
            for b, n in enumerate(lengths.tolist()):
                _within(y[b], want[b, :, n:n + 1], bound[b, :, n:n + 1])
            lengths += 1


@gpu
@pytest.mark.parametrize("window,sinks,tokens", [(16, 0, 5), (16, 3, 40), (1, 2, 7), (100, 30, 20), (7, 0, 1)])
def test_extension_of_the_cache(win, window, sinks, tokens):
    before, new = [0, sinks, 3 * window + 1, 2, 5, -1], [tokens, tokens - 1, tokens, 0, tokens + 9, tokens]
    batch, heads, dim = len(before), 2, 24
    g = torch.Generator("cuda").manual_seed(tokens)
    k, v = (torch.randn(batch, tokens, heads, dim, generator=g, device="cuda").to(BF16).transpose(1, 2) for _ in range(2))
    keys, values = (torch.randn(batch, heads, sinks + window, dim, generator=g, device="cuda").to(BF16) for _ in range(2))
    want = keys.clone(), values.clone()
    for b in range(batch):
        for t in range(min(new[b], tokens) if before[b] >= 0 else 0):
            slot = _slot(before[b] + t, window, sinks)
            want[0][b, :, slot], want[1][b, :, slot] = k[b, :, t], v[b, :, t]
    with torch.no_grad():
        win.window_cache_extend(k, v, keys, values, torch.tensor(before, dtype=torch.int32, device="cuda"), sinks,
                                new=torch.tensor(new, dtype=torch.int32, device="cuda"))
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])


@gpu
def test_cache_behind_two_to_the_31_elements(win):
    window, dim = (1 << 25) + 5, 64
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    keys, values = (torch.zeros(1, 1, window, dim, dtype=BF16, device="cuda") for _ in range(2))
    lengths = torch.tensor([window - 3], dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(0)
    k, v = (torch.randn(1, 1, 2, dim, generator=g, device="cuda").to(BF16) * 30 for _ in range(2))
    with torch.no_grad():
        win.window_cache_extend(k, v, keys, values, lengths, new=None)
        lengths += 2
        q = k[:, :, 1:] * 0.1
        y = win.window_attention_step(q, k[:, :, 1:], v[:, :, :1], keys, values, lengths)
    assert torch.equal(keys[0, 0, -3:-1], k[0, 0]) and torch.equal(keys[0, 0, -1], k[0, 0, 1])
    # the last key, twice in the cache, outweighs all others; their values are v[1] and v[0]
    s = q[0, 0, 0].double() @ k[0, 0, 1].double() / 8
    assert float(s) - math.log(window) > 20
    assert float((y[0, 0, 0].double() - (v[0, 0, 0].double() + v[0, 0, 1].double()) / 2).abs().max()) <= 2 * (2 * HALF + F32) * 100


@gpu
def test_step_in_a_graph_and_compiled(win):
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v = (torch.randn(2, 4, 1, 64, generator=g, device="cuda").to(BF16) for _ in range(3))

    def fresh():
        return win.WindowCache(2, 4, 64, 8, 2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")

    def tokens(cache, lengths, count, step):
        out = []
        for _ in range(count):
            out.append(step(cache, lengths).clone())
            lengths += 1
        return torch.stack(out)

    def call(cache, lengths):
        return win.window_attention_step(q, k * (1 + lengths.view(-1, 1, 1, 1)).to(BF16), v, cache.keys, cache.values, lengths, 2)

    with torch.no_grad():
        want = tokens(*fresh(), 14, call)
        cache, lengths = fresh()
        call(cache, lengths)
        cache.keys.zero_(), cache.values.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(cache, lengths)
        cache.keys.zero_(), cache.values.zero_()
        assert torch.equal(tokens(cache, lengths, 14, lambda *_: (graph.replay(), y)[1]), want)
        torch._dynamo.reset()
        assert torch.equal(tokens(*fresh(), 14, torch.compile(call, fullgraph=True, backend="aot_eager")), want)


@gpu
def test_cache_refusals(win):
    cache = win.WindowCache(2, 2, 64, 8, 2, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 1, 64, dtype=BF16, device="cuda")
    k = q[:, :2]
    for bad in (lambda: cache.step(q, k, k, lengths.long()), lambda: cache.step(q[:, :3], k, k, lengths),
                lambda: win.window_attention_step(q, k, k, cache.keys, cache.values, lengths, 10),
                lambda: win.window_attention_step(q, k, k, cache.keys, cache.values, lengths, -1),
                lambda: cache.step(q.repeat(1, 1, 2, 1), k, k, lengths), lambda: cache.step(q, k, k, lengths, scale=-1.0),
                lambda: cache.extend(k[:1], k[:1], lengths), lambda: cache.extend(k, k, lengths, new=lengths[:1]),
                lambda: win.window_attention_step(q, k, k, cache.keys[:, :, :1].expand(-1, -1, 10, -1), cache.values, lengths, 2),
                lambda: win.window_attention_step(q, k, k, cache.keys.transpose(2, 3).contiguous().transpose(2, 3), cache.values,
                                                  lengths, 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no gradient"):
        cache.step(q.detach().requires_grad_(True), k, k, lengths)
    version = cache.keys._version
    cache.step(q, k, k, lengths)
    assert cache.keys._version > version


@gpu
def test_backward_in_a_thread_that_has_made_no_call():
    # the tensor maps are made in the thread of the backward pass, which may not have met the device before
    import subprocess
    import sys
    code = ("import torch\nfrom thetascan_b200 import window_attention\n"
            "q, k, v = (torch.ones(1, 2, 5, 64, dtype=torch.bfloat16, device='cuda', requires_grad=True) for _ in range(3))\n"
            "window_attention(q, k, v, 4).backward(torch.ones_like(q))\nassert v.grad.any()\n")
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)
