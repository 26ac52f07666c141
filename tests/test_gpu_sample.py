"""The choice of tokens against its definition in 64 bits.

Sums of probabilities are exact to 2^-29 of each term, so the kept set is the definition's (a cut that falls on a
border within that has odds of about 1e-6 a row) and the token is one whose stretch of the running mass holds uniform *
total within 1e-8 of the total."""
from __future__ import annotations

import math

import pytest
import torch

gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def sample():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import sample_tokens
    return sample_tokens


def _kept(x, temperature, top_k, top_p, min_p):
    """Odds of one row's tokens that are left, by index (zero: not), and of all of them."""
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.max()
    if top == -math.inf:
        return None, None
    t = temperature if temperature > 0 else 1.0
    z = torch.where(x == top, 0.0, (x - top) / t)
    odds = torch.exp(z)
    order = torch.argsort(x, descending=True, stable=True)
    if temperature <= 0:
        order = order[:1]
    else:
        if top_k:
            order = order[:top_k]
        if top_p is not None and top_p < 1:
            mass = odds[order]
            order = order[mass.cumsum(0) - mass < max(top_p * float(mass.sum()), 1e-300)]
        if min_p:
            order = order[z[order] >= math.log(min(min_p, 1.0))]
    left = torch.zeros_like(odds)
    left[order] = odds[order]
    return left, odds


def _check(tokens, logits, uniform, temperature=1.0, top_k=None, top_p=None, min_p=None, logprobs=None):
    def of(value, i):
        return value[i].item() if torch.is_tensor(value) else value

    for i, token in enumerate(tokens.tolist()):
        t = of(temperature, i)
        left, odds = _kept(logits[i], t, of(top_k, i), of(top_p, i), of(min_p, i))
        if left is None:
            assert token == -1 and (logprobs is None or logprobs[i] == -math.inf)
            continue
        assert left[token] > 0, (i, token)
        sums = left.cumsum(0)
        total = float(sums[-1])
        at = min(max(float(uniform[i]), 0.0), 1.0) * total
        assert float(sums[token] - left[token]) <= at + 1e-8 * total and at <= float(sums[token]) + 1e-8 * total, (i, token)
        if logprobs is not None:
            want = math.log(float(odds[token])) - math.log(float(odds.sum()))
            assert abs(float(logprobs[i]) - want) <= 2.0 ** -23 * abs(want) + 1e-8


def _logits(rows, vocab, dtype, seed=0, spread=2.5):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype), torch.rand(rows, generator=g, device="cuda")


SETTINGS = [
    dict(), dict(temperature=0.0), dict(temperature=0.6, top_k=1), dict(top_k=7), dict(top_p=0.9), dict(min_p=0.1),
    dict(temperature=1.3, top_k=400, top_p=0.95, min_p=0.01), dict(top_k=10 ** 6, top_p=1.0, min_p=0.0), dict(top_p=1e-9),
    dict(temperature=30.0, top_p=0.5), dict(temperature=1e-3, top_p=0.5), dict(temperature=100.0, top_k=900)]


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (9, 1024), (4, 2049), (6, 16391), (2, 50_257), (1, 300_001)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_settings(sample, rows, vocab, dtype):
    logits, uniform = _logits(rows, vocab, dtype, seed=vocab)
    for settings in SETTINGS:
        tokens, logprobs = sample(logits, uniform, return_logprobs=True, **settings)
        assert tokens.dtype == torch.int64 and tokens.shape == (rows,) and logprobs.dtype == F32
        _check(tokens, logits, uniform, logprobs=logprobs, **settings)
        assert torch.equal(sample(logits, uniform, **settings), tokens)


@gpu
def test_each_row_its_own_settings(sample):
    rows = 40
    logits, uniform = _logits(rows, 5000, F32, seed=1)
    g = torch.Generator("cuda").manual_seed(2)
    settings = dict(temperature=torch.rand(rows, generator=g, device="cuda") * 1.5, top_k=torch.randint(-1, 300, (rows,), generator=g, device="cuda"),
                    top_p=torch.rand(rows, generator=g, device="cuda") * 1.2, min_p=torch.rand(rows, generator=g, device="cuda") * 0.2)
    settings["temperature"][::5] = 0
    meant = dict(settings, top_k=settings["top_k"].clamp_min(0))
    tokens, logprobs = sample(logits, uniform, return_logprobs=True, **settings)
    _check(tokens, logits, uniform, logprobs=logprobs, **meant)
    assert torch.equal(sample(logits, uniform, **dict(settings, top_k=settings["top_k"].to(torch.int32))), tokens)
    # values out of range have the documented meaning
    wild = dict(temperature=torch.tensor([-1.0, math.nan, 1.0, 1.0]), top_k=torch.tensor([2 ** 40, 0, -5, 3]),
                top_p=torch.tensor([2.0, 0.5, -1.0, math.nan]), min_p=torch.tensor([-1.0, 0.0, 0.0, 5.0]))
    got = sample(logits[:4], uniform[:4], **{n: t.cuda() for n, t in wild.items()})
    best = logits[:4].argmax(-1)
    assert got.tolist() == best.tolist()   # greedy, greedy, one token of top_p, min_p 1


@gpu
@pytest.mark.parametrize("vocab", [700, 5000, 40_000, 140_000])
def test_equal_logits(sample, vocab):
    # ties go to the lowest index, at every cut: all equal, two values, few values
    for kind in range(3):
        g = torch.Generator("cuda").manual_seed(kind)
        logits = torch.zeros(3, vocab, device="cuda")
        if kind:
            logits = torch.randint(0, 2 if kind == 1 else 9, (3, vocab), generator=g, device="cuda") * (0.125 if kind == 1 else 2.0 ** -9)
        uniform = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24], device="cuda")
        for settings in (dict(), dict(top_k=513), dict(top_k=vocab - 1), dict(top_p=0.37), dict(top_k=600, top_p=0.9), dict(temperature=0.0),
                         dict(min_p=1.0), dict(top_k=550, top_p=0.99, min_p=0.95)):
            _check(sample(logits, uniform, **settings), logits, uniform, **settings)
    # of equals, all with the same mass: exactly the first ones
    logits = torch.zeros(1, vocab, device="cuda")
    last = sample(logits, torch.tensor([1 - 2.0 ** -24], device="cuda"), top_k=600)
    assert last.item() == 599


@gpu
def test_many_values_in_one_bin(sample):
    # a bin of the histogram holds 64ths of a nat at temperature 1: thousands of different logits in it
    g = torch.Generator("cuda").manual_seed(0)
    logits = 3 + torch.rand(4, 30_000, generator=g, device="cuda") * 1e-3
    logits[:, 17] = 4.0
    uniform = torch.rand(4, generator=g, device="cuda")
    for settings in (dict(top_k=12_345), dict(top_p=0.4), dict(top_k=20_000, top_p=0.7), dict(temperature=50.0, top_p=0.6)):
        _check(sample(logits, uniform, **settings), logits, uniform, **settings)


@gpu
def test_masked_tokens(sample):
    logits, uniform = _logits(8, 2000, F32, seed=3)
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 1:] = -math.inf
    logits[3, ::2] = math.nan
    logits[4, 5] = logits[4, 900] = math.inf
    logits[5] = -math.inf
    logits[5, 1999] = -3e38
    logits[6, :1000] = 3e38
    logits[7, :] = -0.0
    logits[7, 9] = 0.0
    for settings in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5), dict(top_k=30, top_p=0.8, min_p=0.1)):
        tokens, logprobs = sample(logits, uniform, return_logprobs=True, **settings)
        assert tokens[0] == -1 and tokens[1] == -1 and tokens[2] == 0 and tokens[3] % 2 == 1 and tokens[4] in (5, 900) and tokens[5] == 1999
        clean = logits.clone()
        clean[4] = torch.where(logits[4] == math.inf, 0.0, -math.inf)
        _check(tokens, clean, uniform, logprobs=logprobs, **settings)
    assert sample(logits, uniform, temperature=0.0)[7] == 0   # minus zero is zero: the first


@gpu
def test_logits_and_temperatures_at_the_ends_of_f32(sample):
    least = torch.finfo(F32).min
    logits = torch.full((8, 3000), -math.inf, device="cuda")
    logits[:, 7] = math.nan
    logits[0, 1000:1010] = least                                   # a mask of the type's lowest value, and nothing else
    logits[1, ::3] = least
    logits[1, 1] = torch.nextafter(torch.tensor(least), torch.tensor(0.0))
    logits[2, 100:1100] = torch.randn(1000, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    logits[3, ::2] = torch.linspace(-1, 1, 1500, device="cuda") * 3.4e38
    logits[4, 5:9] = torch.tensor([-3e38, 3e38, 0.0, 1.0], device="cuda")
    logits[5, 2000:] = least
    logits[5, 2001] = 1.0
    logits[6, 50:60] = math.inf
    logits[7, ::5] = least / 2
    temperature = torch.tensor([1.0, 0.5, 3e38, 1e38, 2e38, 1.0, 3e38, 0.0], device="cuda")
    clean = logits.clone()
    clean[6] = torch.where(logits[6] == math.inf, 0.0, -math.inf)   # infinities share a row's probability
    for seed in range(4):
        uniform = torch.rand(8, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")
        for settings in (dict(), dict(top_k=4), dict(top_p=0.6), dict(top_k=600, top_p=0.9, min_p=0.01), dict(min_p=0.3)):
            tokens, logprobs = sample(logits, uniform, temperature=temperature, return_logprobs=True, **settings)
            _check(tokens, clean, uniform, temperature=temperature, logprobs=logprobs, **settings)
    temperature[:] = math.inf
    tokens = sample(logits, uniform, temperature=temperature)
    assert (clean[torch.arange(8), tokens] > -math.inf).all()


@gpu
def test_uniform_at_its_ends(sample):
    logits, _ = _logits(4, 300, F32, seed=4)
    ends = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, math.nan], device="cuda")
    tokens = sample(logits, ends, top_k=20)
    kept = [sorted(row.topk(20).indices.tolist()) for row in logits]
    assert tokens.tolist() == [kept[0][0], kept[1][-1], kept[2][-1], kept[3][0]]


@gpu
def test_frequencies(sample):
    # evenly spaced uniforms: each kept token is drawn as often as its share says, to one draw
    logits, _ = _logits(1, 50, F32, seed=5, spread=1.0)
    n = 4096
    tokens = sample(logits.expand(n, -1), (torch.arange(n, device="cuda") + 0.5) / n, top_p=0.8)
    left, _ = _kept(logits[0], 1.0, None, 0.8, None)
    counts = torch.bincount(tokens, minlength=50).double()
    assert float((counts - left / left.sum() * n).abs().max()) <= 1


@gpu
def test_layouts_streams_and_graphs(sample):
    wide, uniform = _logits(12, 3001, BF16, seed=6)
    logits = wide[::2, 1:2500]
    want = sample(logits.contiguous(), uniform[:6], top_k=40, top_p=0.9)
    assert torch.equal(sample(logits, uniform[:6], top_k=40, top_p=0.9), want)
    assert torch.equal(sample(logits.reshape(2, 3, -1), uniform[:6].view(2, 3), top_k=40, top_p=0.9), want.view(2, 3))
    assert torch.equal(sample(logits.t().contiguous().t(), uniform[:6], top_k=40, top_p=0.9), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        u = uniform[:6].clone()
        sample(logits, u, top_k=40, top_p=0.9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = sample(logits, u, top_k=40, top_p=0.9)
        u.copy_(uniform[6:])
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, sample(logits, uniform[6:], top_k=40, top_p=0.9))
    torch._dynamo.reset()
    compiled = torch.compile(lambda x, u, t: sample(x, u, temperature=t, top_k=40, return_logprobs=True), fullgraph=True, backend="aot_eager")
    t = torch.full((6,), 0.7, device="cuda")
    for a, b in zip(compiled(logits, uniform[:6], t), sample(logits, uniform[:6], temperature=t, top_k=40, return_logprobs=True)):
        assert torch.equal(a, b)


@gpu
def test_refusals_and_empty(sample):
    logits, uniform = _logits(3, 10, F32)
    for bad in (lambda: sample(logits, uniform[:2]), lambda: sample(logits, uniform.double()), lambda: sample(logits.half(), uniform),
                lambda: sample(logits, uniform, temperature=-0.5), lambda: sample(logits, uniform, temperature=math.inf),
                lambda: sample(logits, uniform, temperature=math.nan), lambda: sample(logits, uniform, top_k=0),
                lambda: sample(logits, uniform, top_p=0.0), lambda: sample(logits, uniform, top_p=1.5),
                lambda: sample(logits, uniform, min_p=-0.1), lambda: sample(logits, uniform, min_p=1.1),
                lambda: sample(logits, uniform, temperature=uniform[:2]), lambda: sample(logits, uniform, top_k=uniform),
                lambda: sample(logits, uniform, top_p=uniform.double()), lambda: sample(logits[:, :0], uniform)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no gradient"):
        sample(logits.requires_grad_(True), uniform, return_logprobs=True)
    assert sample(logits, uniform).shape == (3,)
    assert sample(logits[:0].detach(), uniform[:0]).shape == (0,)
