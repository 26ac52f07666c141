"""Windowed attention, the scan's token step and the choice of tokens on the host (no GPU): the C entries refuse what
they cannot do before anything is launched, CPU tensors raise, and the formulas that the GPU tests compare with agree
with differences."""
from __future__ import annotations

import ctypes

import pytest
import torch

from thetascan_b200 import _lib, sample_tokens, window_attention, window_attention_step, window_cache_extend
from thetascan_b200.scan import linattn_views_step
from thetascan_b200.window import WindowCache

BAD, NOT_BUILT = _lib.TS_ERR_VALUE, _lib.TS_ERR_NOT_IMPLEMENTED
THERE = 1 << 20   # a pointer that is never followed: aligned, not null


def _window(**over):
    a = _lib.WindowArgs(batch=1, heads=2, kv_heads=1, dim=64, q_tokens=4, kv_tokens=8, window=4, sinks=1, scale=0.125)
    a.q = a.k = a.v = a.y = THERE
    for n in ("q_strides", "k_strides", "v_strides", "y_strides"):
        setattr(a, n, _lib.c_longlong_3(1024, 64, 128))
    for n, x in over.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(batch=0), BAD), (dict(q_tokens=0), BAD), (dict(kv_tokens=3), BAD), (dict(heads=3, kv_heads=2), BAD),
    (dict(window=0), BAD), (dict(sinks=-1), BAD), (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD),
    (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(q=None), BAD), (dict(y=None), BAD),
    (dict(dim=12), NOT_BUILT), (dict(dim=136), NOT_BUILT), (dict(dim=0), NOT_BUILT), (dict(q=THERE + 8), BAD),
    (dict(k_strides=_lib.c_longlong_3(1024, 64, 100)), BAD), (dict(kv_tokens=(1 << 30) + 8), NOT_BUILT)])
def test_window_refuses(over, code):
    lib = _lib.load()
    assert lib.ts_b200_window_fwd(ctypes.byref(_window(**over)), None) == code
    assert _lib.last_error()[1]


def test_window_backward_refuses():
    lib = _lib.load()
    a, g = _window(lse=THERE), _lib.WindowGradArgs()
    assert lib.ts_b200_window_bwd(ctypes.byref(a), ctypes.byref(g), None) == BAD
    g.dy = g.dq = g.dk = g.dv = g.workspace = THERE
    g.workspace_bytes = lib.ts_b200_window_bwd_workspace_bytes(ctypes.byref(a)) - 1
    assert lib.ts_b200_window_bwd(ctypes.byref(a), ctypes.byref(g), None) == BAD
    assert "workspace" in _lib.last_error()[1]
    g.workspace_bytes += 1
    g.dq_strides = _lib.c_longlong_3(4, 8, 8)
    assert lib.ts_b200_window_bwd(ctypes.byref(a), ctypes.byref(g), None) == BAD
    assert lib.ts_b200_window_bwd_workspace_bytes(ctypes.byref(_window(window=0))) == 0


def _cache(**over):
    c = _lib.WindowCacheArgs(batch=1, kv_heads=1, dim=64, window=4, sinks=0, keys=THERE, values=THERE, lengths=THERE)
    c.keys_strides = c.values_strides = _lib.c_longlong_3(256, 256, 64)
    for n, x in over.items():
        setattr(c, n, x)
    return c


@pytest.mark.parametrize("over,code", [
    (dict(batch=0), BAD), (dict(window=0), BAD), (dict(sinks=-1), BAD), (dict(keys=None), BAD), (dict(lengths=None), BAD),
    (dict(values=THERE + 2), BAD), (dict(keys_strides=_lib.c_longlong_3(256, 256, 60)), BAD), (dict(dim=20), NOT_BUILT),
    (dict(batch=1 << 17), NOT_BUILT)])
def test_cache_entries_refuse(over, code):
    lib = _lib.load()
    step = _lib.WindowStepArgs(cache=_cache(**over), heads=2, scale=0.1, q=THERE, k=THERE, v=THERE, y=THERE)
    assert lib.ts_b200_window_step(ctypes.byref(step), None) == code
    extend = _lib.WindowExtendArgs(cache=_cache(**over), tokens=3, k=THERE, v=THERE)
    assert lib.ts_b200_window_extend(ctypes.byref(extend), None) == code


def test_step_and_extend_refuse():
    lib = _lib.load()
    for over in (dict(heads=0), dict(scale=0.0), dict(q=None), dict(y=None), dict(k=THERE + 4),
                 dict(q_strides=_lib.c_longlong_2(64, 4))):
        a = _lib.WindowStepArgs(cache=_cache(), heads=2, scale=0.1, q=THERE, k=THERE, v=THERE, y=THERE)
        for n, x in over.items():
            setattr(a, n, x)
        assert lib.ts_b200_window_step(ctypes.byref(a), None) == BAD, over
    for over in (dict(tokens=0), dict(k=None), dict(v=THERE + 4)):
        a = _lib.WindowExtendArgs(cache=_cache(), tokens=1, k=THERE, v=THERE)
        for n, x in over.items():
            setattr(a, n, x)
        assert lib.ts_b200_window_extend(ctypes.byref(a), None) == BAD, over


@pytest.mark.parametrize("over,code", [
    (dict(batch=0), BAD), (dict(dk=0), NOT_BUILT), (dict(dk=257), NOT_BUILT), (dict(dv=257), NOT_BUILT), (dict(dv=1), NOT_BUILT),
    (dict(v_append_unit=2), BAD), (dict(n_retentions=0), BAD), (dict(n_retentions=5), BAD), (dict(state=None), BAD),
    (dict(dtype=7), BAD)])
def test_scan_step_refuses(over, code):
    a = _lib.ScanStepArgs(batch=1, heads=1, dk=16, dv=9, v_append_unit=1, dtype=0, q=THERE, k=THERE, v=THERE, n_retentions=1,
                          state=THERE, out=THERE)
    for n, x in over.items():
        setattr(a, n, x)
    assert _lib.load().ts_b200_scan_step(ctypes.byref(a), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(rows=0), BAD), (dict(vocab=0), BAD), (dict(vocab=(1 << 21) + 1), NOT_BUILT), (dict(logits=None), BAD),
    (dict(uniform=None), BAD), (dict(tokens=None), BAD), (dict(dtype=9), BAD)])
def test_sample_refuses(over, code):
    a = _lib.SampleArgs(rows=1, vocab=8, dtype=0, logits=THERE, row_stride=8, uniform=THERE, temperature_value=1.0,
                        top_p_value=1.0, tokens=THERE)
    for n, x in over.items():
        setattr(a, n, x)
    assert _lib.load().ts_b200_sample(ctypes.byref(a), None) == code


def test_null_arguments_are_refused():
    lib = _lib.load()
    for name in ("window_step", "window_extend", "scan_step", "sample", "window_fwd"):
        assert getattr(lib, f"ts_b200_{name}")(None, None) == BAD
    assert lib.ts_b200_window_bwd_workspace_bytes(None) == 0


def test_cpu_tensors_raise():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    one, state = q[:, :, :1], torch.zeros(1, 2, 1, 64, 64)
    cache = WindowCache(1, 2, 64, window=4, sinks=1)
    lengths = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        window_attention(q, q, q, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        window_attention_step(one, one, one, cache.keys, cache.values, lengths, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        window_cache_extend(q, q, cache.keys, cache.values, lengths, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        linattn_views_step(one, one, one, [None], state)
    with pytest.raises(RuntimeError, match="CUDA"):
        sample_tokens(torch.zeros(2, 8), torch.zeros(2))


def test_cache_sizes():
    cache = WindowCache(3, 2, 64, window=5, sinks=2)
    assert cache.keys.shape == (3, 2, 7, 64) and cache.values.dtype == torch.bfloat16 and not cache.keys.any()
    with pytest.raises(ValueError):
        WindowCache(1, 1, 64, window=0)


def test_definition_agrees_with_differences():
    from window_definition import attention
    g = torch.Generator().manual_seed(0)
    q = torch.randn(1, 4, 5, 8, generator=g, dtype=torch.float64)
    k, v = (torch.randn(1, 2, 7, 8, generator=g, dtype=torch.float64) for _ in range(2))
    dy = torch.randn(1, 4, 5, 8, generator=g, dtype=torch.float64)
    lengths = torch.tensor([6])
    _, grads, _ = attention(q, k, v, 2, 1, 0.3, lengths, dy)
    for i, grad in enumerate(grads):
        step = torch.randn(grad.shape, generator=g, dtype=torch.float64) * 1e-5
        at = [[t + (s * step if n == i else 0) for n, t in enumerate((q, k, v))] for s in (1, -1)]
        up, down = (float((attention(*a, 2, 1, 0.3, lengths, dy)[0] * dy).sum()) for a in at)
        assert abs((up - down) / 2 - float((grad * step).sum())) <= 1e-8 * float(step.norm() * grad.norm())


def _generating(monkeypatch, chosen):
    """A model whose work and choice are replaced; what reaches each of the two."""
    from thetascan_b200 import lm
    model = lm.HybridLM(vocab=16, d_model=64, n_layers=1, n_heads=1, mixer_layers=(), window=4)
    fed, drawn = [], []
    monkeypatch.setattr(model, "extend", lambda tokens, stream: (fed.append(tokens.clone()), torch.zeros(2, 16))[1])

    def choose(logits, uniform, **settings):
        drawn.append(uniform)
        return chosen.clone()

    monkeypatch.setattr(lm, "sample_tokens", choose)
    return model, fed, drawn


def test_a_row_without_a_token_goes_on(monkeypatch):
    """A row of masked logits has no token: -1, which is no place in the embedding."""
    model, fed, _ = _generating(monkeypatch, torch.tensor([-1, 5]))
    got = model.generate(torch.tensor([[1, 2], [3, 4]]), 3)
    assert got.tolist() == [[-1] * 3, [5] * 3]
    model.generate(got[:, -1:], 1, stream=model.stream(2))   # as a caller goes on from there
    assert [t.tolist() for t in fed] == [[[1, 2], [3, 4]], [[0], [5]], [[0], [5]], [[0], [5]]]


def test_uniform_numbers_are_f32_whatever_the_default(monkeypatch):
    model, _, drawn = _generating(monkeypatch, torch.tensor([1, 5]))
    was = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.float64)
        model.generate(torch.tensor([[1, 2], [3, 4]]), 2)
    finally:
        torch.set_default_dtype(was)
    assert [u.dtype for u in drawn] == [torch.float32] * 2   # what the choice takes


@pytest.mark.parametrize("over,said", [(dict(lse=THERE + 4), "lse"), (dict(workspace=THERE + 8), "workspace")])
def test_window_backward_refuses_what_its_copies_cannot_read(over, said):
    """Both are read by copies of 16-byte pieces, which end the context at another address."""
    lib = _lib.load()
    a, g = _window(lse=THERE), _lib.WindowGradArgs()
    g.dy = g.dq = g.dk = g.dv = g.workspace = THERE
    for n in ("dy", "dq", "dk", "dv"):
        setattr(g, f"{n}_strides", _lib.c_longlong_3(1024, 64, 128))
    g.workspace_bytes = lib.ts_b200_window_bwd_workspace_bytes(ctypes.byref(a))
    for n, x in over.items():
        setattr(a if hasattr(a, n) else g, n, x)
    assert lib.ts_b200_window_bwd(ctypes.byref(a), ctypes.byref(g), None) == BAD
    assert said in _lib.last_error()[1] and "16-byte" in _lib.last_error()[1]


@pytest.mark.parametrize("dim", [64, 128])
def test_workspace_of_many_first_tokens_is_bounded(dim):
    """Sums of first tokens' key tiles, [channels x 128] f32 of dk and dv for each chunk of queries: no more of them than
    keep the SMs at work, whatever the sizes."""
    lib = _lib.load()
    for batch, kv_heads, tokens, sinks in [(1, 1, 1 << 20, 128), (1, 8, 16384, 4096), (64, 8, 16384, 4096), (4, 8, 1 << 20, 1 << 19), (512, 16, 4096, 1)]:
        a = _window(batch=batch, heads=kv_heads, kv_heads=kv_heads, dim=dim, q_tokens=tokens, kv_tokens=tokens, window=100, sinks=sinks)
        stats = batch * kv_heads * tokens * 4
        got = lib.ts_b200_window_bwd_workspace_bytes(ctypes.byref(a))
        assert stats <= got <= stats + 16 * 148 * 2 * dim * 128 * 4, (batch, kv_heads, tokens, sinks, got - stats)


def test_a_stream_begun_in_inference_mode_goes_on_outside():
    """What a stream keeps is changed in place by later calls, which PyTorch refuses for tensors made in inference mode."""
    from thetascan_b200 import lm, seqpar
    model = lm.HybridLM(vocab=16, d_model=64, n_layers=2, n_heads=1, mixer_layers=(1,), window=4,
                        mixer_config=lm.gn_mixer_config(64, 1))
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 1, 9, n, generator=g) for n in (6, 6, 4))

    def scan(q, k, v, retentions, *, append_unit=False):
        return [(q @ k.transpose(-1, -2)).tril() @ torch.cat((v, torch.ones_like(v[..., :1])), -1) for _ in retentions]

    def piece(scans, s):
        with scans.piece(q[:, 0, s]):
            return seqpar.sharded_reads(scans, scan, q[:, :, s], k[:, :, s], v[:, :, s], (None,), append_unit=True)[0]

    with torch.inference_mode():
        stream, scans = model.stream(2), seqpar.ScanStream()
        first = piece(scans, slice(0, 5)).clone()
    with torch.no_grad():
        stream.lengths += 3
        stream.layers[0].keys.zero_()
        got = torch.cat((first, piece(scans, slice(5, 9))), 2)
    want, = scan(q, k, v, (None,))
    assert float((got - want).abs().max()) <= 9 * 6 * 2.0 ** -23 * float(want.abs().max())   # sums of 54 products
