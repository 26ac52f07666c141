"""The scan's token step against its definition in 64 bits and against the scan of whole segments.

Bounds: the state's update is one multiplication and one fused one in f32 (after a product k v of its own rounding):
4 * 2^-24 of |a S| + |k v|.  A read sums up to 256 products in f32, each of a state that far off: 260 * 2^-24 of the sum
of magnitudes, and its own rounding to bf16 (2^-8) where the streams are bf16."""
from __future__ import annotations

import pytest
import torch

gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def scan():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import scan
    return scan


def _make(batch, heads, dk, dv, unit, kinds, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q, k = (normal(batch, 1, heads, dk).to(dtype).transpose(1, 2) for _ in range(2))
    v = normal(batch, 1, heads, dv).to(dtype).transpose(1, 2)
    rets = [None if kind == "sum" else torch.log(torch.rand(*((heads,) if kind == "head" else (batch, heads, 1, 1)),
                                                            generator=g, device="cuda") * 0.5 + 0.5) for kind in kinds]
    return q, k, v, rets, normal(batch, heads, len(kinds), dk, dv + unit)


def _check(got, state, before, q, k, v, rets, unit):
    q, k, v = q.double(), k.double(), v.double()
    if unit:
        v = torch.cat([v, torch.ones_like(v[..., :1])], -1)
    for i, r in enumerate(rets):
        keep = torch.ones(1, 1, 1, 1, device=q.device) if r is None else r.reshape(-1, q.shape[1], 1, 1)
        old, new = before[:, :, i].double() * torch.exp(keep.double() if r is not None else keep * 0.0), k.transpose(-1, -2) * v
        want = old + new
        off = 4 * 2.0 ** -24 * (old.abs() + new.abs())
        # exp of the retention in f32: two units in the last place
        off = off + 4 * 2.0 ** -24 * old.abs()
        assert (state[:, :, i].double() - want).abs().sub(off).max() <= 0
        read = q @ want
        bound = 270 * 2.0 ** -24 * (q.abs() @ (old.abs() + new.abs())) + (2.0 ** -8 if got[i].dtype == BF16 else 0) * read.abs()
        assert got[i].shape == read.shape
        assert (got[i].double() - read).abs().sub(bound).max() <= 0


CASES = [
    (1, 1, 1, 1, 0, ("sum",)), (1, 8, 256, 64, 1, ("sum", "head")), (3, 2, 17, 5, 1, ("head", "sum", "gate")),
    (40, 5, 33, 200, 0, ("gate",)), (2, 3, 256, 256, 0, ("sum", "head", "head", "sum")), (1, 1, 255, 255, 1, ("head",)),
    (70, 16, 128, 64, 1, ("sum", "head")), (2, 1, 7, 129, 0, ("head", "gate"))]


@gpu
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_against_the_definition(scan, case, dtype):
    batch, heads, dk, dv, unit, kinds = case
    q, k, v, rets, state = _make(batch, heads, dk, dv, unit, kinds, dtype, seed=dk)
    before = state.clone()
    got = scan.linattn_views_step(q, k, v, rets, state, append_unit=bool(unit))
    assert len(got) == len(kinds) and all(o.dtype == dtype for o in got)
    _check(got, state, before, q, k, v, rets, unit)
    again = before.clone()
    twice = scan.linattn_views_step(q, k, v, rets, again, append_unit=bool(unit))
    assert torch.equal(again, state) and all(torch.equal(a, b) for a, b in zip(got, twice))


@gpu
def test_continues_a_scanned_prompt(scan):
    # the state that a prompt's scan leaves, then tokens one by one: the scan of it all
    g = torch.Generator("cuda").manual_seed(5)
    q, k, v = (torch.randn(2, 4, 70, d, generator=g, device="cuda").to(BF16) for d in (64, 64, 48))
    rets = [None, torch.log(torch.tensor([0.5, 0.9, 0.99, 0.999], device="cuda"))]
    want, end = scan.linattn_views_stream(q, k, v, rets, append_unit=True)
    with torch.no_grad():
        _, state = scan.linattn_views_stream(q[:, :, :60], k[:, :, :60], v[:, :, :60], rets, append_unit=True)
        for t in range(60, 70):
            got = scan.linattn_views_step(*(x[:, :, t:t + 1] for x in (q, k, v)), rets, state, append_unit=True)
            for a, b in zip(got, want):
                # the whole scan's products are bf16 (2^-8 of the terms)
                assert float((a.float() - b[:, :, t:t + 1].float()).norm()) <= 2e-2 * float(b[:, :, t:t + 1].float().norm())
    assert float((state - end).norm()) <= 1e-2 * float(end.norm())


@gpu
def test_streams_graphs_and_compilation(scan):
    q, k, v, rets, state = _make(2, 3, 40, 24, 1, ("sum", "head"), F32)
    first = state.clone()

    def tokens(step, state):
        return torch.stack([torch.stack(step(state)).clone() for _ in range(5)])

    def call(state):
        return scan.linattn_views_step(q, k, v, rets, state, append_unit=True)

    want = tokens(call, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(tokens(call, first.clone()), want)
        held = first.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call(held)
        held.copy_(first)
        assert torch.equal(tokens(lambda s: (graph.replay(), out)[1], held), want)
    torch.cuda.current_stream().wait_stream(side)
    torch._dynamo.reset()
    assert torch.equal(tokens(torch.compile(call, fullgraph=True, backend="aot_eager"), first.clone()), want)


@gpu
def test_refusals_and_empty(scan):
    q, k, v, rets, state = _make(2, 3, 16, 8, 0, ("sum", "head"), F32)
    step = scan.linattn_views_step
    assert step(q, k, v, [], state) == ()
    for bad in (lambda: step(q, k, v, rets, state[:, :, :1]), lambda: step(q, k, v, rets, state.transpose(3, 4)),
                lambda: step(q, k, v, rets, state.double()), lambda: step(q, k, v, [None, rets[1][:2]], state),
                lambda: step(q.repeat(1, 1, 2, 1), k, v, rets, state), lambda: step(q, k[..., :8], v, rets, state),
                lambda: step(q, k, v, rets, state[:1].expand(2, -1, -1, -1, -1))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: step(q.to(BF16), k, v, rets, state), lambda: step(q.half(), k.half(), v.half(), rets, state),
                lambda: step(q, k, v, [None] * 5, torch.zeros(2, 3, 5, 16, 8, device="cuda"))):
        with pytest.raises(NotImplementedError):
            bad()
    with pytest.raises(RuntimeError, match="no gradient"):
        step(q.detach().requires_grad_(True), k, v, rets, state)
    with pytest.raises(RuntimeError, match="in place"):
        step(q, k, v, rets, state.clone().requires_grad_(True))
    none = torch.zeros(0, 3, 1, 16, device="cuda")
    assert step(none, none, none, [None], torch.zeros(0, 3, 1, 16, 16, device="cuda"))[0].shape == (0, 3, 1, 16)
    version = state._version
    step(q, k, v, rets, state)
    assert state._version > version
