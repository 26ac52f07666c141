"""Windowed attention, the token steps and the choice of tokens under the other ways of taking derivatives: each is either
right or refused with an error."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import thetascan_b200
    return thetascan_b200


def _inputs(dim=64):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, h, 200, dim, generator=g).to(BF16).cuda() for h in (4, 2, 2))
    return q, k, v, torch.tensor([200, 131], dtype=torch.int32, device="cuda")


def _attention(ts, lengths):
    return lambda q, k, v: ts.window_attention(q, k, v, 50, 3, lengths=lengths)


def _steps(ts):
    """Calls without a gradient, of one tensor."""
    from thetascan_b200.scan import linattn_views_step
    one = torch.ones(2, 2, 1, 64, dtype=BF16, device="cuda")
    cache = ts.WindowCache(2, 2, 64, 8, 2, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    state, uniform = torch.zeros(2, 2, 1, 64, 64, device="cuda"), torch.zeros(2, device="cuda")
    return [(lambda t: ts.window_attention_step(t, one, one, cache.keys, cache.values, lengths, 2), one),
            (lambda t: ts.window_cache_extend(t, one, cache.keys, cache.values, lengths, 2), one),
            (lambda t: linattn_views_step(t, one, one, [None], state), one),
            (lambda t: ts.sample_tokens(t, uniform), torch.zeros(2, 9, device="cuda"))]


@gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(ts, requires_grad):
    *inputs, lengths = _inputs()
    f = _attention(ts, lengths)
    for i in range(3):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(inputs[i].clone().requires_grad_(requires_grad), torch.ones_like(inputs[i]))
            args = [dual if j == i else u for j, u in enumerate(inputs)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(*args)
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    y = f(*leaves)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaves, dy)
    for f, t in _steps(ts):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(t.clone(), torch.ones_like(t)))


@gpu
def test_transforms_are_refused(ts):
    # functorch's wrapped tensors have no memory of their own
    *inputs, lengths = _inputs()
    f = _attention(ts, lengths)
    for call, t in [(lambda t: f(t, *inputs[1:]), inputs[0]), *_steps(ts)]:
        many = t[None].expand(3, *t.shape)
        with pytest.raises(Exception):
            torch.vmap(call)(many)
        with pytest.raises(Exception):
            torch.func.grad(lambda t: call(t).float().sum())(t)
        with pytest.raises(Exception):
            torch.func.jvp(lambda t: call(t).float().sum(), (t,), (t,))


@gpu
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("dim", [64, 80])
def test_checkpointing_gives_the_same_gradients(ts, reentrant, dim):
    from torch.utils.checkpoint import checkpoint
    *inputs, lengths = _inputs(dim)
    f, grads = _attention(ts, lengths), []
    for call in (f, lambda *t: checkpoint(f, *t, use_reentrant=reentrant)):
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        y = call(*leaves)
        y.backward(torch.ones_like(y))
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@gpu
def test_saved_tensors_pass_through_their_hooks(ts):
    *inputs, lengths = _inputs()
    f = _attention(ts, lengths)
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    want = torch.autograd.grad(f(*leaves).float().sum(), leaves)
    count = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: count.append(t.shape) or t.cpu(), lambda t: t.cuda()):
        y = f(*leaves)
    assert len(count) >= 5   # q, k, v, the result and the rows' sums; the lengths too
    got = torch.autograd.grad(y.float().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_gradients_of_some_inputs_alone(ts):
    *inputs, lengths = _inputs()
    f = _attention(ts, lengths)
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    want = torch.autograd.grad(f(*leaves).float().sum(), leaves)
    for i in range(3):
        args = [t.clone().requires_grad_(i == n) for n, t in enumerate(inputs)]
        got, = torch.autograd.grad(f(*args).float().sum(), args[i])
        assert torch.equal(got, want[i])


@gpu
def test_what_the_backward_needs_may_not_change(ts):
    # a length, an input or the result written over before the backward pass is found, as PyTorch finds it
    *inputs, lengths = _inputs()
    for which in range(5):
        own = lengths.clone()
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        y = _attention(ts, own)(*leaves)
        with torch.no_grad():
            (own, *leaves, y)[which].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, torch.ones_like(y))


@gpu
def test_one_tensor_as_keys_and_values(ts):
    *inputs, lengths = _inputs()
    f = _attention(ts, lengths)
    q, kv = inputs[0].clone().requires_grad_(True), inputs[1].clone().requires_grad_(True)
    both, = torch.autograd.grad(f(q, kv, kv).float().sum(), kv)
    k, v = (kv.detach().clone().requires_grad_(True) for _ in range(2))
    dk, dv = torch.autograd.grad(f(q, k, v).float().sum(), (k, v))
    assert torch.equal(both, dk + dv)


@gpu
def test_the_result_is_no_view(ts):
    *inputs, lengths = _inputs()
    y = _attention(ts, lengths)(*(t.clone().requires_grad_(True) for t in inputs))
    assert not y._is_view()
    y.clone().mul_(2), y.mul_(2)   # in place, as on any result
    torch._dynamo.reset()
    compiled = torch.compile(_attention(ts, lengths), fullgraph=True, backend="aot_eager")
    with torch.no_grad():
        assert compiled(*inputs).stride() == _attention(ts, lengths)(*inputs).stride()
    for shape in [(0, 2, 5, 64), (2, 2, 0, 64)]:
        q = torch.zeros(shape, dtype=BF16, device="cuda")
        assert ts.window_attention(q, q, q, 4).shape == shape
