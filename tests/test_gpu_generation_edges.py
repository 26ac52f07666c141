"""Calls of the generation operators that their documentation allows and few programs make: offsets past 32 bits, one row
without a batch, inference mode, compiled models, streams side by side."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_generate import NEAR, _model, _off
from test_gpu_sample import _check, sample  # noqa: F401  (sample: a fixture)
from test_gpu_window import _within, win  # noqa: F401  (win: a fixture)
from window_definition import attention

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


@gpu
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_over_more_than_two_to_the_31_elements(win, token_major):  # noqa: F811
    heads, tokens, dim, last = 120, 150_001, 128, 300
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator("cuda").manual_seed(0)

    def normal(h):
        shape = (1, tokens, h, dim) if token_major else (1, h, tokens, dim)
        t = torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=g)
        return t.transpose(1, 2) if token_major else t

    q, k, v, dy = normal(heads), normal(2), normal(2), normal(heads)
    assert q.numel() > 1 << 31
    dy[:, :, :-last] = 0     # what is before it has no gradient, but that of the keys it sees
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = win.window_attention(*leaves, 64, 2)
    dq, dk, dv = torch.autograd.grad(y, leaves, dy)
    q, k, v, y = (t.detach() for t in (q, k, v, y))
    assert not dq[:, ::17, :-last].any() and not dk[:, :, 2:-last - 64].any()
    # the last rows of the heads of the second key head; the gradient of a key is the sum of all of them
    s = slice(heads // 2, heads)
    near = torch.cat((torch.arange(2), torch.arange(tokens - last - 64, tokens))).cuda()   # the keys that these see, in order
    want, want_grads, bounds = attention(q[:, s, -last:].double(), k[:, 1:, near].double(), v[:, 1:, near].double(), 64, 2,
                                         1 / math.sqrt(dim), None, dy[:, s, -last:].double())
    for got, w, bound in zip((y[:, s, -last:], dq[:, s, -last:], dk[:, 1:, near], dv[:, 1:, near]), (want, *want_grads), bounds):
        _within(got, w, bound)


@gpu
def test_choice_over_more_than_two_to_the_31_logits(sample):  # noqa: F811
    rows, vocab = 17_000, 128_257
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    g = torch.Generator("cuda").manual_seed(0)
    logits = torch.empty(rows, vocab, dtype=BF16, device="cuda").normal_(generator=g)
    uniform = torch.rand(rows, generator=g, device="cuda")
    tokens, logprobs = sample(logits, uniform, top_k=70, return_logprobs=True)
    at = torch.tensor([0, 8000, rows - 2, rows - 1], device="cuda")
    _check(tokens[at], logits[at], uniform[at], top_k=70, logprobs=logprobs[at])


@gpu
def test_one_row_without_a_batch(sample):  # noqa: F811
    g = torch.Generator("cuda").manual_seed(0)
    logits, uniform = torch.randn(1, 700, generator=g, device="cuda"), torch.rand(1, generator=g, device="cuda")
    token, logprob = sample(logits[0], uniform[0], top_k=torch.tensor(9, device="cuda"), top_p=0.9, return_logprobs=True)
    assert token.shape == logprob.shape == ()
    _check(token[None], logits, uniform, top_k=9, top_p=0.9, logprobs=logprob[None])


@gpu
def test_generation_in_inference_mode_and_training_after_it():
    model = _model(24, 2, gated="silu", fused_norms=True).cuda()
    tokens = torch.randint(0, 256, (2, 37), generator=torch.Generator().manual_seed(0)).cuda()
    want = model.generate(tokens, 6, top_k=9, generator=torch.Generator("cuda").manual_seed(1))
    with torch.inference_mode():
        got = model.generate(tokens, 6, top_k=9, generator=torch.Generator("cuda").manual_seed(1))
    assert torch.equal(got, want)
    loss = model.loss(torch.cat((tokens, want), 1)[:, :38])
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


@gpu
def test_compiled_model_with_windowed_attention():
    torch._dynamo.reset()
    tokens = torch.randint(0, 256, (2, 65), generator=torch.Generator().manual_seed(0)).cuda()
    grads = []
    for compiled in (False, True):
        model = _model(24, 2, mixer_layers=(), gated="silu", fused_norms=True).cuda()
        call = torch.compile(model, fullgraph=True, backend="aot_eager") if compiled else model
        logits = call(tokens[:, :-1])
        loss = torch.nn.functional.cross_entropy(logits.float().flatten(0, 1), tokens[:, 1:].flatten())
        loss.backward()
        grads.append([logits.detach(), *(p.grad for p in model.parameters())])
    for a, b in zip(*grads):
        assert _off(a, b) < NEAR


@gpu
def test_streams_side_by_side(win, sample):  # noqa: F811
    # the same calls on two CUDA streams at once, on tensors of their own: what each gives alone
    def work(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        q, k, v, dy = (torch.randn(3, 6, 700, 128, generator=g, device="cuda").to(BF16) for _ in range(4))
        logits, uniform = torch.randn(40, 60_000, generator=g, device="cuda"), torch.rand(40, generator=g, device="cuda")

        def run():
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            y = win.window_attention(*leaves, 150, 140)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy), sample(logits, uniform, top_k=600, top_p=0.9))
        return run

    runs = [work(0), work(1)]
    want = [r() for r in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = [[] for _ in runs]
    for _ in range(10):
        for i, (r, stream) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(stream):
                got[i].append(r())
    torch.cuda.synchronize()
    for many, one in zip(got, want):
        assert all(torch.equal(a, b) for each in many for a, b in zip(each, one))


@gpu
def test_a_stream_through_inference_mode_and_out_of_it():
    model = _model(24, 2, gated="silu", fused_norms=True).cuda()
    tokens = torch.randint(0, 256, (2, 80), generator=torch.Generator().manual_seed(0)).cuda()
    stream = model.stream(2)
    want = [model.extend(tokens[:, s], stream) for s in (slice(0, 40), slice(40, 41), slice(41, 80))]
    for inside in ((True, False, True), (False, True, False), (True, True, False)):
        with torch.inference_mode(inside[0]):
            stream = model.stream(2)
        for one, s, w in zip(inside, (slice(0, 40), slice(40, 41), slice(41, 80)), want):
            with torch.inference_mode(one):
                got = model.extend(tokens[:, s], stream)
            assert torch.equal(got, w)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_minus_infinity_alone_give_no_number(win, dim):  # noqa: F811
    # a row whose visible scores are all minus infinity: 0 / 0, not the zero of a row that sees nothing; in every form
    g = torch.Generator("cuda").manual_seed(0)
    q, k, v = (torch.randn(2, 2, 150, dim, generator=g, device="cuda").to(BF16) for _ in range(3))
    q[1, :, 149] = 0
    q[1, :, 149, 0] = math.inf
    k[..., 0] = -1
    lengths = torch.tensor([100, 150], dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y = win.window_attention(*leaves, 40, 2, lengths=lengths)
    with torch.no_grad():
        cache = win.WindowCache(2, 2, dim, 40, 2, device="cuda")
        cache.extend(k[:, :, :149], v[:, :, :149], torch.zeros_like(lengths), new=lengths - 1)
        step = cache.step(q[:, :, 149:], k[:, :, 149:], v[:, :, 149:], lengths - 1)
    assert torch.isnan(y[1, :, 149]).all() and torch.isnan(step[1]).all()
    assert torch.isfinite(y[:, :, :149]).all() and not y[0, :, 100:].any()
    dq, = torch.autograd.grad(y, leaves[0], torch.ones_like(y))
    assert torch.isnan(dq[1, :, 149]).all() and torch.isfinite(dq[0]).all() and not dq[0, :, 100:].any()
