"""Settings of the choice of tokens: every integer type of ``top_k``, refusals of compiled calls, masses at the precision
that the choice states."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_sample import sample  # noqa: F401  (a fixture)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64,
                                   torch.uint64])
def test_top_k_of_any_integer_type(sample, dtype):  # noqa: F811
    g = torch.Generator("cuda").manual_seed(0)
    logits, uniform = torch.randn(5, 400, generator=g, device="cuda"), torch.rand(5, generator=g, device="cuda")
    wanted = [1, 2, 50, 127, 0]
    want = torch.cat([sample(logits[i:i + 1], uniform[i:i + 1], top_k=k or None) for i, k in enumerate(wanted)])
    assert torch.equal(sample(logits, uniform, top_k=torch.tensor(wanted).to(dtype).cuda()), want)
    # more than there are tokens, or less than one: no filter
    open_ = sample(logits, uniform)
    for limit in (torch.iinfo(dtype).max, torch.iinfo(dtype).min):
        if 1 <= limit < 400:
            continue
        assert torch.equal(sample(logits, uniform, top_k=torch.tensor([limit] * 5, dtype=dtype).cuda()), open_)


@gpu
def test_compiled_calls_refuse_what_eager_ones_refuse(sample):  # noqa: F811
    torch._dynamo.reset()
    logits, uniform = torch.randn(3, 10, device="cuda"), torch.rand(3, device="cuda")
    for settings in (dict(temperature=-0.5), dict(top_k=0), dict(top_k=-3), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=1.1)):
        compiled = torch.compile(lambda x, u, s=settings: sample(x, u, **s), fullgraph=True, backend="aot_eager")
        for call in (lambda x, u: sample(x, u, **settings), compiled):
            with pytest.raises(ValueError):
                call(logits, uniform)
    for settings in (dict(), dict(top_k=4), dict(top_k=10 ** 9), dict(top_k=torch.full((3,), 4, device="cuda"))):
        compiled = torch.compile(lambda x, u, s=settings: sample(x, u, **s), fullgraph=True, backend="aot_eager")
        assert torch.equal(compiled(logits, uniform), sample(logits, uniform, **settings))


@gpu
def test_masses_at_their_stated_precision(sample):
    """Two tokens, the second of mass m beside the first's 1: top_p keeps it as long as 1 < top_p (1 + m).  With top_p on
    either side of that by ``off`` of m, which of the two is drawn shows whether m is right to that.

    A mass is rounded to units of 2^-40, by half of one at most; the series of the exponential, a distance in 64 bits and
    top_p itself are off by less than 1e-12 of it together."""
    g = torch.Generator().manual_seed(1)
    draws = torch.rand(400, 3, generator=g, dtype=torch.float64).tolist()
    uniform = torch.tensor([1 - 2.0 ** -24], device="cuda")
    logits, settings, wanted = [], [], []
    for a, b, c in draws:
        top, temperature = float(torch.tensor(2 + 10 * a, dtype=torch.float32)), 0.4 + b
        other = float(torch.tensor(top - temperature * 1.2 * c - 1e-3, dtype=torch.float32))
        m = math.exp((other - top) / temperature)
        off = 2.0 ** -41 / m + 1e-12
        for sign in (1, -1):
            logits.append([top, other])
            settings.append(dict(temperature=temperature, top_p=1 / (1 + m * (1 + sign * off))))
            wanted.append(0 if sign > 0 else 1)
    logits = torch.tensor(logits, dtype=torch.float32, device="cuda")
    got = torch.cat([sample(logits[i:i + 1], uniform, **s) for i, s in enumerate(settings)])
    wrong = (got != torch.tensor(wanted, device="cuda")).nonzero()[:, 0].tolist()
    assert not wrong, (len(wrong), [settings[i] for i in wrong[:3]])
