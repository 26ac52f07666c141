"""Token steps and the cache's extension have no gradient: inputs that want one are refused, in eager and compiled calls."""
from __future__ import annotations

import pytest
import torch

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import thetascan_b200
    return thetascan_b200


def _calls(ts):
    """Name, the call, its tensors that could want a gradient, and the ones it writes."""
    from thetascan_b200.scan import linattn_views_step
    one = [torch.ones(2, 2, 1, 64, dtype=BF16, device="cuda") for _ in range(3)]
    a, b = (ts.WindowCache(2, 2, 64, 8, 2, device="cuda") for _ in range(2))
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    state, decay = torch.zeros(2, 2, 2, 64, 64, device="cuda"), torch.zeros(2, device="cuda")
    return [("step", lambda q, k, v, a, b: ts.window_attention_step(q, k, v, a, b, lengths, 2), one, [a.keys, a.values]),
            ("extend", lambda k, v, a, b: ts.window_cache_extend(k, v, a, b, lengths, 2), one[1:], [b.keys, b.values]),
            ("scan", lambda q, k, v, r, s: linattn_views_step(q, k, v, [None, r], s), [*one, decay], [state])]


@gpu
@pytest.mark.parametrize("compiled", [False, True])
def test_gradients_are_refused(ts, compiled):
    for name, f, inputs, written in _calls(ts):
        was = [t.clone() for t in written]
        for i in range(len(inputs)):
            if compiled:
                torch._dynamo.reset()
            call = torch.compile(f, backend="aot_eager") if compiled else f
            args = [t.clone().requires_grad_(True) if i == n else t for n, t in enumerate(inputs)]
            with pytest.raises(RuntimeError, match="no gradient|no autograd formula"):
                call(*args, *written)
            assert all(torch.equal(a, b) for a, b in zip(was, written)), name   # and nothing is written
        with torch.no_grad():
            args = [t.clone().requires_grad_(True) for t in inputs]
            call(*args, *written)
        assert not all(torch.equal(a, b) for a, b in zip(was, written)), name
