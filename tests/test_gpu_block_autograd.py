"""The norm, the gated block and the AdamW step under the other ways of taking
derivatives: each is either right or refused with an error.
"""
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


def _inputs(rows=40):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: (torch.randn(*s, generator=g) / 8).to(BF16).cuda()  # noqa: E731
    return r(rows, 64), r(128, 64), r(128, 64), r(64, 128), r(64)


def _calls(ts):
    """Name of the operator, the function, its inputs."""
    x, wg, wu, wd, w = _inputs()
    return [("rms_norm", ts.rms_norm, (x, w)), ("add_rms_norm", lambda *t: ts.add_rms_norm(*t)[0], (x, x.flip(0), w)),
            ("rms_norm_8bit", lambda *t: ts.rms_norm_8bit(*t)[1], (x, w)), ("gated_ffn", ts.gated_ffn, (x, wg, wu, wd))]


@gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(ts, requires_grad):
    for name, f, inputs in _calls(ts):
        for i, t in enumerate(inputs):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t.clone().requires_grad_(requires_grad and name != "rms_norm_8bit"), torch.ones_like(t))
                args = [dual if j == i else u for j, u in enumerate(inputs)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*args)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*args)
                with forward_ad._set_fwd_grad_enabled(False), torch.no_grad():
                    f(*args)   # asked for without
        f(*inputs)


@gpu
def test_forward_mode_over_a_backward_pass_is_refused(ts):
    for name, f, inputs in _calls(ts):
        if name == "rms_norm_8bit":
            continue
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        y = f(*leaves)
        with forward_ad.dual_level():
            dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaves, dy)


@gpu
def test_forward_mode_through_a_step_is_refused(ts):
    p, g, m, v = (torch.ones(64, device="cuda") for _ in range(4))
    with forward_ad.dual_level():
        for which in range(2):
            args = [forward_ad.make_dual(t, t.clone()) if i == which else t for i, t in enumerate((p, g))]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ts.adamw_step([args[0]], [args[1]], [m], [v], step=1, lr=0.1)
    assert (p == 1).all() and (m == 1).all()


@gpu
def test_transforms_are_refused(ts):
    # functorch's wrapped tensors have no memory of their own
    for _, f, inputs in _calls(ts):
        many = inputs[0][None].expand(3, *inputs[0].shape)
        with pytest.raises(Exception):
            torch.vmap(lambda t: f(t, *inputs[1:]))(many)
        with pytest.raises(Exception):
            torch.func.grad(lambda t: f(t, *inputs[1:]).float().sum())(inputs[0])
        with pytest.raises(Exception):
            torch.func.jvp(lambda t: f(t, *inputs[1:]).float().sum(), (inputs[0],), (inputs[0],))


@gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointing_gives_the_same_gradients(ts, reentrant):
    from torch.utils.checkpoint import checkpoint
    for name, f, inputs in _calls(ts):
        if name == "rms_norm_8bit":
            continue
        grads = []
        for call in (f, lambda *t: checkpoint(f, *t, use_reentrant=reentrant)):
            leaves = [t.clone().requires_grad_(True) for t in inputs]
            y = call(*leaves)
            y.backward(torch.ones_like(y))
            grads.append([t.grad for t in leaves])
        assert all(torch.equal(a, b) for a, b in zip(*grads)), name


@gpu
def test_saved_tensors_pass_through_their_hooks(ts):
    for name, f, inputs in _calls(ts):
        if name == "rms_norm_8bit":
            continue
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        want = torch.autograd.grad(f(*leaves).float().sum(), leaves)
        count = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: count.append(t.shape) or t.cpu(), lambda t: t.cuda()):
            y = f(*leaves)
        assert len(count) >= 3, name
        got = torch.autograd.grad(y.float().sum(), leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


@gpu
def test_one_tensor_as_both_terms_of_the_sum(ts):
    # its gradient is the sum of both terms'
    x, *_, w = _inputs()
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    y, s = ts.add_rms_norm(a, a, w)
    (y.float().sum() + 3 * s.float().sum()).backward()
    c = x.clone().requires_grad_(True)
    y2, s2 = ts.add_rms_norm(b, c, w)
    (y2.float().sum() + 3 * s2.float().sum()).backward()
    assert torch.equal(y, y2) and torch.equal(a.grad, b.grad + c.grad) and torch.equal(b.grad, c.grad)


@gpu
@pytest.mark.parametrize("rows", [8, 300])
def test_forward_and_backward_in_a_graph(ts, rows):
    x, wg, wu, wd, w = _inputs(rows)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd, w)]

    def step():
        y, s = ts.add_rms_norm(x, x.detach(), w)
        z = ts.gated_ffn(y, wg, wu, wd)
        return [z.detach(), *torch.autograd.grad((z, s), leaves, (torch.ones_like(z), torch.ones_like(s)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        for t in leaves:
            t.mul_(1.25)
    want = step()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
