"""The residual norm's kernels against its definition in float64.

The definition: s = round(x + r) in the stream's type, y = s rstd w.  Bounds,
derived before any run: a result is rounded once to its type, half a unit in
the last place, so at most 2^-8 of its value in bf16; what precedes it is f32
arithmetic whose relative error is below 2e-6 for these widths (a sum of n
squares has a relative error under n 2^-24 in the worst order, and is summed in
pairs here).  Gradients that add terms of both signs are measured against the
largest entry.
"""
from __future__ import annotations

import pytest
import torch

gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


@pytest.fixture(scope="module")
def norm():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import norm
    return norm


def _make(shape, dtype, wdtype, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(dtype).cuda()
    r = (3 * torch.randn(shape, generator=g)).to(dtype).cuda() if residual else None
    w = (1 + 0.2 * torch.randn(shape[-1], generator=g)).to(wdtype).cuda()
    return x, r, w


def _definition(x, r, w, eps=EPS):
    s = x if r is None else (x.double() + r.double()).to(x.dtype)
    s = s.double()
    return s * (s.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double(), s


def _close(got, want, dtype):
    """Half a unit in the last place of the type, and 2e-6 of the value or of the largest entry before it."""
    assert got.dtype == dtype and got.shape == want.shape
    step = 2.0 ** -8 if dtype == BF16 else 0.0
    bound = want.abs() * (step + 2e-6) + 2e-6 * want.abs().max()
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())


CASES = [(1, 1), (1, 7), (3, 64), (2, 128), (5, 333), (257, 512), (33, 520), (9, 1024), (4, 1537), (3, 2048), (7, 4104),
         (2, 8192), (3, 8200), (2, 16384), (3, 16383)]


@gpu
@pytest.mark.parametrize("rows,width", CASES)
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(norm, rows, width, dtype, wdtype, residual):
    x, r, w = _make((rows, width), dtype, wdtype, seed=rows * 17 + width, residual=residual)
    want, s = _definition(x, r, w)
    got = norm.add_rms_norm(x, r, w, EPS) if residual else norm.rms_norm(x, w, EPS)
    if residual:
        got, total = got
        assert torch.equal(total.double(), s)
    _close(got, want, dtype)


@gpu
@pytest.mark.parametrize("rows,width", CASES)
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("residual", [True, False])
def test_backward_is_the_formulas(norm, rows, width, dtype, wdtype, residual):
    x, r, w = _make((rows, width), dtype, wdtype, seed=rows + width, residual=residual)
    g = torch.Generator().manual_seed(9)
    dy = torch.randn((rows, width), generator=g).to(dtype).cuda()
    ds = torch.randn((rows, width), generator=g).to(dtype).cuda()
    leaves = [t.clone().requires_grad_(True) for t in ((x, r, w) if residual else (x, w))]
    if residual:
        got = torch.autograd.grad(norm.add_rms_norm(*leaves, EPS), leaves, (dy, ds))
        assert torch.equal(got[0], got[1])
    else:
        got = torch.autograd.grad(norm.rms_norm(*leaves, EPS), leaves, dy)
    _, s = _definition(x, r, w)
    s = s.requires_grad_(True)
    w64 = w.double().requires_grad_(True)
    y = s * (s.square().mean(-1, keepdim=True) + EPS).rsqrt() * w64
    want = torch.autograd.grad((y * dy.double()).sum() + ((s * ds.double()).sum() if residual else 0), (s, w64))
    _close(got[0], want[0], dtype)
    _close(got[-1], want[1], wdtype)


@gpu
def test_backward_is_the_difference_of_its_forward(norm):
    # f32, along a random direction: central differences of step h have an error of h^2 times a third derivative of
    # order one and 2^-23 of the loss's terms / h from rounding; h = 1e-2 leaves both under 1e-3 of the slope's scale
    x, r, w = _make((6, 96), F32, F32, seed=3)
    g = torch.Generator().manual_seed(4)
    dy, ds, along = (torch.randn(6, 96, generator=g).cuda() for _ in range(3))
    xl = x.clone().requires_grad_(True)
    y, s = norm.add_rms_norm(xl, r, w, EPS)
    slope = (torch.autograd.grad((y, s), xl, (dy, ds))[0].double() * along.double()).sum()

    def loss(t):
        y, s = norm.add_rms_norm(t, r, w, EPS)
        return (y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()

    h = 1e-2
    diff = (loss(x + h * along) - loss(x - h * along)) / (2 * h)
    assert abs(float(diff - slope)) <= 1e-3 * float((dy.norm() + ds.norm()) * along.norm())


@gpu
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("rows,width", CASES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("residual", [True, False])
def test_8bit(norm, group, rows, width, dtype, residual):
    x, r, w = _make((rows, width), dtype, dtype, seed=rows * 3 + width, residual=residual)
    want, s = _definition(x, r, w)
    with torch.no_grad():
        got = norm.rms_norm_8bit(x, w, EPS, residual=r, group=group)
    assert len(got) == (3 if residual else 2)
    if residual:
        assert torch.equal(got[2].double(), s)
    codes, scales = got[:2]
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    parts = want.split(group or width, -1)
    top = torch.stack([p.abs().amax(-1) for p in parts], -1).clamp_min(2.0 ** -100)
    assert scales.shape == top.shape
    assert ((scales.double() * 448 / top - 1).abs() <= 4e-6).all()
    # a code is at most half its step from the value: 2^-4 of it, or 2^-10 of the scale among the smallest
    each = scales.double().repeat_interleave(group or width, -1)[:, :width]
    bound = (want.abs() * 2.0 ** -4).maximum(each * 2.0 ** -10) * (1 + 1e-4)
    assert ((codes.double() * each - want).abs() <= bound).all()
    assert int((codes.view(torch.uint8) & 0x7F).max()) == 0x7E  # the largest magnitude gets the largest code


@gpu
def test_rows_of_zeros_and_non_finite_rows(norm):
    x = torch.zeros(4, 200, device="cuda", dtype=BF16)
    x[1] = 1.0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    w = torch.ones(200, device="cuda", dtype=BF16)
    y = norm.rms_norm(x, w, EPS)
    assert (y[0] == 0).all() and (y[1] == 1).all() and y[2].isnan().all()
    assert y[3, 7].isnan() and (y[3, :7] == 0).all()
    codes, scales = norm.rms_norm_8bit(x[:2], w, EPS, group=128)
    assert (codes[0].float() == 0).all() and (scales > 0).all() and scales.isfinite().all()
    xl = x[:1].clone().requires_grad_(True)
    dx, = torch.autograd.grad(norm.rms_norm(xl, w, EPS), xl, torch.ones_like(xl))
    assert (dx == 1000.0).all()  # rstd = 1e3 at eps = 1e-6


@gpu
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("width", [200, 203, 1000, 8200])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_8bit_of_non_finite_rows(norm, dtype, width, group):
    # a scale is the largest magnitude's: NaN where one of its values is (an infinity's row is 0 * inf there), and so are
    # its codes; the other groups and rows are what they are without it
    x, _, w = _make((6, width), dtype, F32, seed=width)
    clean = norm.rms_norm_8bit(x, w, EPS, group=group)
    bad = x.clone()
    bad[1, 5], bad[2, width - 1], bad[3, 130] = float("nan"), float("inf"), float("-inf")
    codes, scales = norm.rms_norm_8bit(bad, w, EPS, group=group)
    y = norm.rms_norm(bad.float(), w, EPS)
    nan = torch.stack([p.isnan().any(-1) for p in y.split(group or width, -1)], -1)
    assert nan[1].all() and nan[2, -1] and nan[3].any() and not nan[[0, 4, 5]].any()
    assert torch.equal(scales.isnan(), nan)
    assert torch.equal(codes.float().isnan(), nan.repeat_interleave(group or width, -1)[:, :width])
    for row in (0, 4, 5):
        assert torch.equal(scales[row], clean[1][row]) and torch.equal(codes[row].float(), clean[0][row].float())
    spoilt = w.clone()
    spoilt[150] = float("nan")
    codes, scales = norm.rms_norm_8bit(x, spoilt, EPS, group=group)
    hit = torch.arange(scales.shape[1], device="cuda") == (150 // group if group else 0)
    assert torch.equal(scales.isnan(), hit.expand(6, -1))
    assert torch.equal(scales[:, ~hit], clean[1][:, ~hit])


@gpu
def test_leading_dimensions_strides_and_alignment(norm):
    g = torch.Generator().manual_seed(1)
    big = torch.randn(3, 5, 2, 72, generator=g).to(BF16).cuda()
    w = torch.ones(64, device="cuda")
    for x in (big[..., :64], big[..., 1:65], big[:, ::2, 1, :64], big.transpose(0, 1)[..., 8:72], big[:1, :, :, :64].expand(3, 5, 2, 64)):
        want, s = _definition(x, x.flip(0), w)
        y, total = norm.add_rms_norm(x, x.flip(0), w, EPS)
        _close(y, want, BF16)
        assert torch.equal(total.double(), s)
    x = big[..., 1:65].requires_grad_(True)
    got, = torch.autograd.grad(norm.rms_norm(x, w, EPS).float().sum(), x)   # an expanded gradient
    s = big[..., 1:65].double().requires_grad_(True)
    want, = torch.autograd.grad((s * (s.square().mean(-1, keepdim=True) + EPS).rsqrt()).sum(), s)
    _close(got, want, BF16)


@gpu
def test_empty_and_unused_outputs(norm):
    w = torch.ones(32, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, 32, device="cuda", requires_grad=True)
    y, s = norm.add_rms_norm(x, x, w)
    dx, dw = torch.autograd.grad(y.sum() + s.sum(), (x, w))
    assert dx.shape == x.shape and (dw == 0).all()
    x = torch.randn(2, 32, device="cuda", requires_grad=True)
    _, s = norm.add_rms_norm(x, x.detach(), w)
    dx, dw = torch.autograd.grad(s.sum(), (x, w), allow_unused=True)
    assert (dx == 1).all() and dw is None
    assert norm.rms_norm_8bit(torch.zeros(0, 32, device="cuda"), w.detach(), group=128)[1].shape == (0, 1)


@gpu
def test_gradients_do_not_depend_on_timing(norm):
    x, r, w = _make((5000, 512), BF16, F32)
    dy = torch.randn_like(x)

    def once():
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
        return torch.autograd.grad(norm.add_rms_norm(*leaves), leaves, (dy, dy))

    a = once()
    for _ in range(3):
        for p, q in zip(a, once()):
            assert torch.equal(p, q)


@gpu
def test_on_another_stream(norm):
    x, r, w = _make((2000, 512), BF16, F32)
    want = norm.add_rms_norm(x, r, w)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm.add_rms_norm(x, r, w)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@gpu
def test_compiles_into_one_graph(norm):
    x, r, w = _make((64, 256), BF16, F32)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]

    def f(x, r, w):
        y, s = norm.add_rms_norm(x, r, w)
        return (y.float() + s.float()).square().sum()

    want = torch.autograd.grad(f(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves), leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("residual", [False, True])
def test_compiled_inference_runs_what_eager_inference_runs(norm, residual, monkeypatch):
    # bit for bit, and with nothing kept for a backward pass unless one is wanted
    torch._dynamo.reset()
    x, r, w = _make((40, 256), BF16, F32, residual=residual)
    f = norm.add_rms_norm if residual else norm.rms_norm
    args = (x, r, w) if residual else (x, w)
    outputs = lambda y: y if residual else (y,)  # noqa: E731
    kept, host = [], norm._lib.host()

    class Host:
        def __getattr__(self, name):
            if name != "norm_fwd":
                return getattr(host, name)
            return lambda *a: kept.append(a[-1]) or host.norm_fwd(*a)

    want = outputs(f(*args))
    compiled = torch.compile(lambda *t: f(*t), fullgraph=True, backend="aot_eager")
    monkeypatch.setattr(norm._lib, "host", lambda: Host())
    assert all(torch.equal(a, b) for a, b in zip(outputs(compiled(*args)), want))
    with torch.no_grad():
        got = outputs(compiled(*args[:-1], w.clone().requires_grad_(True)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert kept == [False, False]
    got = outputs(compiled(*args[:-1], w.clone().requires_grad_(True)))
    assert got[0].requires_grad and torch.equal(got[0].detach(), want[0]) and kept[2:] == [True]


@gpu
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("residual", [False, True])
def test_8bit_compiles_into_one_graph(norm, residual, group):
    torch._dynamo.reset()
    x, r, w = _make((3, 20, 200), BF16, F32, residual=residual)
    f = lambda x, w: norm.rms_norm_8bit(x, w, residual=r, group=group)  # noqa: E731
    want = f(x, w)
    compiled = torch.compile(f, fullgraph=True, backend="aot_eager")
    got = compiled(x, w)
    assert len(got) == len(want) == (3 if residual else 2)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.float(), b.float())
    w.requires_grad_(True)
    with torch.no_grad():
        assert torch.equal(compiled(x, w)[1], want[1])
    with pytest.raises(Exception, match="no gradient"):
        compiled(x, w)


@gpu
def test_refusals(norm):
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    for bad in (dict(x=x.half()), dict(w=w.half()), dict(w=w[:32]), dict(eps=-1.0), dict(w=w[None])):
        with pytest.raises(ValueError):
            norm.rms_norm(bad.get("x", x), bad.get("w", w), bad.get("eps", EPS))
    with pytest.raises(ValueError):
        norm.add_rms_norm(x, x[:1], w)
    with pytest.raises(ValueError):
        norm.add_rms_norm(x, x.bfloat16(), w)
    with pytest.raises(ValueError):
        norm.rms_norm_8bit(x, w, group=64)
    with pytest.raises(RuntimeError):
        norm.rms_norm_8bit(x.requires_grad_(True), w)
    with pytest.raises(NotImplementedError):
        norm.rms_norm(torch.zeros(1, 16385, device="cuda"), torch.ones(16385, device="cuda"))
    with pytest.raises(RuntimeError):
        norm.rms_norm(x.detach(), w.cpu())


@gpu
def test_custom_op_refuses_what_does_not_fit(norm):
    x, w, rstd = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda"), torch.ones(4, device="cuda")
    for bad in ((x[:2], None, x, w, rstd), (x, x[:2], x, w, rstd), (x, None, x, w[:32], rstd), (x, None, x, w, rstd[:3]),
                (x.bfloat16(), None, x, w, rstd)):
        with pytest.raises(ValueError):
            norm.norm_bwd(*bad, EPS)


@gpu
def test_second_gradient_is_refused(norm):
    x, w = torch.ones(2, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(norm.rms_norm(x, w).sum(), x, create_graph=True)


def test_refuses_cpu_tensors():
    from thetascan_b200 import rms_norm
    with pytest.raises(RuntimeError):
        rms_norm(torch.zeros(2, 8), torch.ones(8))


def test_c_entry_refuses_bad_arguments():
    import ctypes
    from thetascan_b200 import _lib
    lib = _lib.load()
    assert lib.ts_b200_norm_fwd(None, None) == _lib.TS_ERR_VALUE
    a = _lib.NormArgs()
    a.rows, a.width, a.x, a.weight, a.y = 1, 20000, 256, 256, 256
    assert lib.ts_b200_norm_fwd(ctypes.byref(a), None) == _lib.TS_ERR_NOT_IMPLEMENTED
    a.width, a.residual = 64, 256
    assert lib.ts_b200_norm_fwd(ctypes.byref(a), None) == _lib.TS_ERR_VALUE   # no output for the sum
    a.residual, a.group = None, 96
    assert lib.ts_b200_norm_fwd(ctypes.byref(a), None) == _lib.TS_ERR_NOT_IMPLEMENTED
    a.group = 0
    g = _lib.NormGradArgs()
    assert lib.ts_b200_norm_bwd(ctypes.byref(a), ctypes.byref(g), None) == _lib.TS_ERR_VALUE
