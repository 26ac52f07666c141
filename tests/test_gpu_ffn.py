"""The gated feed-forward block's kernels against its formula in float64.

Bounds, derived before any run.  bf16 rounds a value by at most 2^-8 of it (U).
The kernels round the hidden values (h, dg, du) and each result once and
accumulate in f32, so a result sum_j a_j b_j with rounded a_j is off by at most
U sum_j |a_j b_j| + U |result|; f32 sums, the activation's fast exponential
and the projections that are kept in 24 bits (2^-16 of each of two) add less
than 4e-5 sum_j |a_j b_j| (with what cancels inside a_j counted by its terms).  Over many entries the roundings are independent, each
of root mean square at most U / sqrt(3), so the norm of the error is within
U sqrt(2/3) = 3.2e-3 of the result's (checked at 3.3e-3).
"""
from __future__ import annotations

import math

import pytest
import torch

gpu = pytest.mark.gpu
BF16 = torch.bfloat16
U = 2.0 ** -8


@pytest.fixture(scope="module")
def ffn():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import _lib, ffn
    yield ffn
    assert _lib.device_status(torch.cuda.current_stream().cuda_stream) == 0


def _make(rows, width, hidden, out, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(BF16).cuda()  # noqa: E731
    return (r(rows, width), r(hidden, width, scale=1.5 / math.sqrt(width)), r(hidden, width, scale=1 / math.sqrt(width)),
            r(out, hidden, scale=1 / math.sqrt(hidden)), r(rows, out))


def _act(g, kind):
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if kind == "gelu":
        s = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * s, s + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g.clamp_min(0).square(), 2 * g.clamp_min(0)


def _formula(x, wg, wu, wd, dy, kind):
    """Outputs, and for each the sum of magnitudes that its bound is made of."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg.T, x @ wu.T
    a, slope = _act(g, kind)
    h = a * u
    dh = dy @ wd
    du, dg = dh * a, dh * u * slope
    # f32 error inside the hidden values is relative to the terms of their sums
    terms_dh = dy.abs() @ wd.abs()
    t = dict(h=a.abs() * (x.abs() @ wu.abs().T) + slope.abs() * u.abs() * (x.abs() @ wg.abs().T),
             du=terms_dh * a.abs() + dh.abs() * slope.abs() * (x.abs() @ wg.abs().T),
             dg=terms_dh * (u * slope).abs() + dh.abs() * (x.abs() @ wu.abs().T) * slope.abs()
             + (dh * u).abs() * 2 * (x.abs() @ wg.abs().T))
    want = (h @ wd.T, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h)
    rounded = (h.abs() @ wd.abs().T, dg.abs() @ wg.abs() + du.abs() @ wu.abs(), dg.abs().T @ x.abs(), du.abs().T @ x.abs(),
               dy.abs().T @ h.abs())
    summed = (t["h"] @ wd.abs().T, t["dg"] @ wg.abs() + t["du"] @ wu.abs(), t["dg"].T @ x.abs(), t["du"].T @ x.abs(),
              dy.abs().T @ t["h"])
    return want, [U * r + 4e-5 * (r + s) for r, s in zip(rounded, summed)]


def _close(got, want, bound, what):
    assert got.dtype == BF16 and got.shape == want.shape
    off = (got.double() - want).abs()
    assert (off <= bound + U * want.abs() + 1e-30).all(), (what, float((off - bound - U * want.abs()).max()))
    if want.numel() >= 4096:
        assert float(off.norm()) <= 3.3e-3 * float(want.norm()), (what, float(off.norm() / want.norm()))


NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")
SHAPES = [
    # rows, width, hidden, width_out: one token, few rows, tile edges, ragged everything
    (1, 8, 8, 8), (1, 512, 1024, 512), (2, 64, 128, 64), (5, 264, 136, 72), (8, 1024, 2056, 1024), (9, 128, 512, 128),
    (16, 520, 1032, 520), (17, 72, 264, 8), (31, 256, 256, 256), (33, 256, 256, 256), (64, 512, 512, 512), (65, 192, 320, 448),
    (127, 64, 128, 256), (128, 64, 256, 264), (129, 136, 120, 64), (255, 256, 384, 256), (256, 512, 1024, 512), (257, 256, 256, 512),
    # few rows past wide weights, with a ragged end of each
    (12, 136, 2376, 600), (30, 264, 2440, 1192),
    # a long inner length and few tiles: split products, forward and backward
    (100, 64, 4096, 64), (5000, 64, 72, 64), (3001, 128, 384, 320),
    # several tiles for each pair of SMs
    (20011, 64, 264, 136), (9000, 328, 1304, 328),
]


@gpu
@pytest.mark.parametrize("rows,width,hidden,out", SHAPES)
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu2"])
def test_block_is_the_formulas(ffn, rows, width, hidden, out, kind):
    *inputs, dy = _make(rows, width, hidden, out, seed=rows + width)
    want, bound = _formula(*inputs, dy, kind)
    with torch.no_grad():
        _close(ffn.gated_ffn(*inputs, kind), want[0], bound[0], "inference")
    leaves = [t.requires_grad_(True) for t in inputs]
    y = ffn.gated_ffn(*leaves, kind)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    for name, g, w, b in zip(NAMES, got, want, bound):
        _close(g.detach(), w, b, name)


# The down product split among clusters of three pairs (one tile, ragged ones, twenty), and the few rows' wide kernels at
# both ends of their rows and where their width begins.
MORE_SHAPES = [
    (40, 128, 1536, 256), (33, 72, 1480, 8), (300, 136, 1672, 264), (1000, 64, 2560, 1280),
    (9, 64, 2568, 640), (12, 136, 2376, 616), (16, 1024, 4096, 1024), (32, 256, 256, 256), (32, 512, 2376, 1192),
]


@gpu
@pytest.mark.parametrize("rows,width,hidden,out", MORE_SHAPES)
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu2"])
def test_block_is_the_formulas_where_the_split_changes(ffn, rows, width, hidden, out, kind):
    test_block_is_the_formulas(ffn, rows, width, hidden, out, kind)


@gpu
@pytest.mark.parametrize("rows,width,hidden,out", [(1, 1024, 4096, 4096), (7, 520, 1032, 1024), (12, 136, 2376, 616),
                                                   (16, 520, 1032, 520), (31, 256, 256, 256), (32, 512, 2376, 1192)])
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu2"])
def test_few_rows_carry_their_results_rounding_alone(ffn, rows, width, hidden, out, kind):
    # h goes to the product in two bf16 parts, within 2^-16 of it, which the 4e-5 covers: what is left is the result's
    # rounding, U at most and uniform, so U / sqrt 12 = 1.13e-3 of a value at an even mantissa and up to sqrt 3 of that
    # near a power of two; 1.9e-3 of the norm is over both, and under the 2.35e-3 of h in one part
    *inputs, dy = _make(rows, width, hidden, out, seed=rows + 1)
    want, bound = _formula(*inputs, dy, kind)
    x, wg, wu, wd = (t.double() for t in inputs)
    h = _act(x @ wg.T, kind)[0] * (x @ wu.T)
    alone = bound[0] - U * (h.abs() @ wd.abs().T)
    with torch.no_grad():
        y = ffn.gated_ffn(*inputs, kind)
    off = (y.double() - want[0]).abs()
    assert (off <= alone + U * want[0].abs()).all()
    assert float(off.norm()) <= 1.9e-3 * float(want[0].norm())


@gpu
@pytest.mark.parametrize("rows,width,hidden,out", [(1, 1024, 512, 4096), (2, 680, 512, 680), (3, 1296, 488, 1296), (8, 520, 1032, 600),
                                                   (16, 72, 136, 264), (17, 264, 392, 264), (32, 512, 1336, 512)])
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu2"])
def test_few_rows_carry_their_gradients_rounding_alone(ffn, rows, width, hidden, out, kind):
    # as above for the results of a call with gradients: h, dg and du in two parts each, g and u within 2^-15 (which is
    # 6.1e-5 of the sums of magnitudes for the two of them: 1e-4 is allowed)
    *inputs, dy = _make(rows, width, hidden, out, seed=rows + 2)
    want, _ = _formula(*inputs, dy, kind)
    x, wg, wu, wd = (t.double() for t in inputs)
    g, u, dh = x @ wg.T, x @ wu.T, dy.double() @ wd
    a, slope = _act(g, kind)
    at_x, at_g, at_u = x.abs(), x.abs() @ wg.abs().T, x.abs() @ wu.abs().T
    terms = dy.double().abs() @ wd.abs()
    du = terms * a.abs() + dh.abs() * slope.abs() * at_g
    dg = terms * (u * slope).abs() + dh.abs() * slope.abs() * at_u + 2 * (dh * u).abs() * at_g
    h = a.abs() * at_u + slope.abs() * u.abs() * at_g
    sums = (h @ wd.abs().T, dg @ wg.abs() + du @ wu.abs(), dg.T @ at_x, du.T @ at_x, dy.double().abs().T @ h)
    with torch.no_grad():
        alone = ffn.gated_ffn(*inputs, kind)
    leaves = [t.requires_grad_(True) for t in inputs]
    y = ffn.gated_ffn(*leaves, kind)
    assert torch.equal(y.detach(), alone)   # the forward with gradients is the one without
    for name, got, ref, magnitude in zip(NAMES, (y.detach(), *torch.autograd.grad(y, leaves, dy)), want, sums):
        off = (got.double() - ref).abs()
        assert (off <= 1e-4 * magnitude + U * ref.abs()).all(), name
        assert float(off.norm()) <= 1.9e-3 * float(ref.norm()), name


@gpu
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu2"])
def test_activation_over_its_range(ffn, kind):
    # one row, w_up = 1, and for each gate value a second hidden value that takes act(g) rounded to bf16 away again
    # (act(64) is 64 to the last bit, or 4096 for relu2): what comes out is act(g) less that, so an error of act(g) shows
    # at 2^-17 of it.  Allowed: 3.5e-5, of which 2^-16 are for the two parts of h and the result's own rounding, and 2e-5
    # for the activation (far out in gelu's and silu's tails; exponentials of large arguments).
    g = torch.linspace(-12, 12, 512).to(BF16)
    exact = g.double() * torch.erfc(-g.double() / math.sqrt(2)) / 2 if kind == "gelu" else _act(g.double(), kind)[0]
    near = exact.to(BF16)
    back = 4096.0 if kind == "relu2" else 64.0
    wg, wu = torch.zeros(1024, 8, dtype=BF16), torch.zeros(1024, 8, dtype=BF16)
    wg[:512, 0], wg[512:, 0] = g, 64.0
    wu[:512, 0], wu[512:, 0] = 1.0, near / back
    eye = torch.eye(512, dtype=BF16)
    x = torch.zeros(1, 8, dtype=BF16)
    x[0, 0] = 1
    with torch.no_grad():
        y = ffn.gated_ffn(x.cuda(), wg.cuda(), wu.cuda(), torch.cat([eye, -eye], 1).cuda(), kind)[0].double().cpu()
    off = (y - (exact - near.double())).abs()
    assert (off <= (2 * 2.0 ** -17 + 2e-5) * exact.abs()).all(), float((off / exact.abs().clamp_min(1e-300)).max())


@gpu
def test_gradient_is_the_difference_of_the_forward(ffn):
    # along the gradient, a step of 5 % of x: the difference of two forwards of N rounded outputs is off by at most
    # 5 deviations of their noise (3.2e-3 |y| |dy| / sqrt(N) each), and by 2 % for its own curvature
    x, wg, wu, wd, dy = _make(300, 128, 256, 128, seed=5)
    leaf = x.clone().requires_grad_(True)
    y = ffn.gated_ffn(leaf, wg, wu, wd)
    grad = torch.autograd.grad(y, leaf, dy)[0].double()
    step = grad / grad.norm() * x.double().norm() * 0.05
    up, down = (x.double() + step).to(BF16), (x.double() - step).to(BF16)
    loss = lambda t: (ffn.gated_ffn(t, wg, wu, wd).double() * dy.double()).sum()  # noqa: E731
    change, slope = float(loss(up) - loss(down)), float((grad * (up.double() - down.double())).sum())
    noise = 5 * 2 * 3.2e-3 * float(y.double().norm() * dy.double().norm()) / math.sqrt(y.numel())
    assert noise < 0.1 * abs(slope)
    assert abs(change - slope) <= noise + 0.02 * abs(slope)


@gpu
def test_only_wanted_gradients(ffn):
    x, wg, wu, wd, dy = _make(300, 64, 128, 64)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    every = torch.autograd.grad(ffn.gated_ffn(*leaves), leaves, dy)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, wg, wu, wd))]
        only, = torch.autograd.grad(ffn.gated_ffn(*some), some[i], dy)
        assert torch.equal(only, every[i])


@gpu
def test_results_do_not_depend_on_timing(ffn):
    x, wg, wu, wd, dy = _make(5000, 64, 264, 64)

    def once():
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = ffn.gated_ffn(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    a = once()
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(a, once()))


@gpu
def test_rows_are_independent(ffn):
    # a NaN or infinite row stays its own: the others are what they are without it
    x, wg, wu, wd, _ = _make(300, 128, 256, 128)
    want = ffn.gated_ffn(x, wg, wu, wd)
    bad = x.clone()
    bad[7, 3], bad[260, 0] = float("nan"), float("inf")
    got = ffn.gated_ffn(bad, wg, wu, wd)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[7] = keep[260] = False
    assert torch.equal(got[keep], want[keep]) and got[7].isnan().all()
    y = ffn.gated_ffn(bad[:8], wg, wu, wd)
    assert torch.isfinite(y[:7]).all() and y[7].isnan().all()


@gpu
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu2"])
@pytest.mark.parametrize("rows", [4, 70])
def test_non_finite_weights_show(ffn, rows, kind):
    # one hidden value is NaN, plus or minus infinity by its gate alone: outputs and gradients are finite, infinite or
    # NaN where the formula's are
    x, wg, wu, wd, dy = _make(rows, 64, 128, 64, seed=1)
    x = x.abs() + 0.5
    x[rows // 2] = 0.25
    for value in (float("nan"), float("inf"), -float("inf")):
        gate = wg.clone()
        gate[77] = value
        leaves = [t.clone().requires_grad_(True) for t in (x, gate, wu, wd)]
        wide = [t.detach().double().requires_grad_(True) for t in leaves]
        g = wide[0] @ wide[1].T
        want = (_act(g, kind)[0] * (wide[0] @ wide[2].T)) @ wide[3].T
        y = ffn.gated_ffn(*leaves, kind)
        with torch.no_grad():
            results = [(y, want), (ffn.gated_ffn(*leaves, kind), want)]
        # the gradients' formula, as NaN-free subexpressions differ between ways to write a derivative
        dh = dy.double() @ wide[3]
        slope = _act(g, kind)[1]
        dg, du = dh * (wide[0] @ wide[2].T) * slope, dh * _act(g, kind)[0]
        grads = torch.autograd.grad(y, leaves, dy)
        results += [(grads[1], dg.T @ wide[0]), (grads[2], du.T @ wide[0]), (grads[0], dg @ wide[1] + du @ wide[2])]
        for got, ref in results:
            assert torch.equal(got.isnan(), ref.isnan()), (value, kind)
            assert torch.equal(got.isinf(), ref.isinf()), (value, kind)


@gpu
@pytest.mark.parametrize("rows", [1, 4, 32, 70])
def test_infinite_down_weights_show(ffn, rows):
    # h times an infinity is infinite with h's sign, whatever is left of h's rounding: also for an h of few bits (the last
    # rows' x is 0.5 in one place, and its weights are powers of two), and NaN for an h of zero
    x, wg, wu, wd, _ = _make(rows, 64, 128, 64, seed=2)
    wg[5], wu[5] = 2.0, 4.0
    x[rows - 1] = 0
    if rows > 1:
        x[rows - 2] = 0
        x[rows - 2, 7] = 0.5
    wd = wd.clone()
    wd[9, 5], wd[11, 5] = float("inf"), -float("inf")
    with torch.no_grad():
        y = ffn.gated_ffn(x, wg, wu, wd, "relu2")
    want = (_act(x.double() @ wg.double().T, "relu2")[0] * (x.double() @ wu.double().T)) @ wd.double().T
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    assert torch.equal(y[y.isinf()].double(), want[want.isinf()])


@gpu
@pytest.mark.parametrize("rows", [3, 70])
def test_strides_leading_dimensions_and_alignment(ffn, rows):
    g = torch.Generator().manual_seed(3)
    big = torch.randn(2, rows, 3, 160, generator=g).to(BF16).cuda()
    _, wg, wu, wd, _ = _make(1, 128, 256, 128)
    wide = torch.zeros(256, 200, dtype=BF16, device="cuda")
    wide[:, 8:136] = wg
    turned = wd.T.contiguous().T
    for x in (big[..., :128], big[..., 8:136], big[..., 1:129], big[:, :, 1, 32:], big.transpose(0, 2)[..., :128],
              big[:, :1, :, :128].expand(2, rows, 3, 128), big[0, 0, 0, :128]):
        want, bound = _formula(x.reshape(-1, 128), wg, wu, wd, torch.zeros(x.reshape(-1, 128).shape, device="cuda"), "silu")
        for weights in ((wg, wu, wd), (wide[:, 8:136], wu, turned)):
            got = ffn.gated_ffn(x, *weights)
            assert got.shape == x.shape
            _close(got.reshape(-1, 128), want[0], bound[0], "y")
    x = big[..., 1:129].requires_grad_(True)
    dx, = torch.autograd.grad(ffn.gated_ffn(x, wg, wu, wd).float().sum(), x)   # an expanded gradient
    want, bound = _formula(x.detach().reshape(-1, 128), wg, wu, wd, torch.ones(x.numel() // 128, 128, device="cuda"), "silu")
    _close(dx.reshape(-1, 128), want[1], bound[1], "dx")


@gpu
def test_empty(ffn):
    _, wg, wu, wd, _ = _make(1, 64, 128, 64)
    leaves = [torch.zeros(2, 0, 64, dtype=BF16, device="cuda", requires_grad=True), wg.requires_grad_(True)]
    y = ffn.gated_ffn(leaves[0], leaves[1], wu, wd)
    dx, dw = torch.autograd.grad(y.sum(), leaves)
    assert y.shape == (2, 0, 64) and dx.shape == (2, 0, 64) and (dw == 0).all()


@gpu
def test_on_another_stream_and_in_a_graph(ffn):
    for rows in (4, 700):
        x, wg, wu, wd, _ = _make(rows, 128, 256, 128)
        want = ffn.gated_ffn(x, wg, wu, wd)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ffn.gated_ffn(x, wg, wu, wd)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ffn.gated_ffn(x, wg, wu, wd)
        x.copy_(x.flip(0))
        for _ in range(2):
            graph.replay()
        assert torch.equal(got, want.flip(0))


@gpu
def test_module_rounds_wider_weights(ffn):
    torch.manual_seed(0)
    m = ffn.GatedFFN(64, 128, "gelu").cuda()
    x = torch.randn(50, 64, device="cuda", requires_grad=True)
    y = m(x)
    assert y.dtype == torch.float32
    y.sum().backward()
    want = ffn.gated_ffn(x.detach().to(BF16), *(l.weight.detach().to(BF16) for l in (m.gate, m.up, m.down)), "gelu")
    assert torch.equal(y.detach(), want.float())
    assert all(p.grad.dtype == torch.float32 and p.grad.abs().sum() > 0 for p in m.parameters()) and x.grad.dtype == torch.float32


@gpu
def test_compiles_into_one_graph(ffn):
    x, wg, wu, wd, _ = _make(64, 64, 128, 64)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    f = lambda *t: ffn.gated_ffn(*t).float().square().sum()  # noqa: E731
    want = torch.autograd.grad(f(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves), leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("rows", [1, 32, 300])
def test_compiled_inference_runs_what_eager_inference_runs(ffn, rows):
    # bit for bit, also where only the mode or only the inputs say that no gradient is wanted; the op keeps nothing
    torch._dynamo.reset()   # the modes and sizes below are each a compilation of the same function
    x, wg, wu, wd, _ = _make(rows, 128, 512, 128)
    f = lambda *t: ffn.gated_ffn(*t, "gelu")  # noqa: E731
    want = f(x, wg, wu, wd)
    compiled = torch.compile(f, fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(x, wg, wu, wd), want)
    with torch.no_grad():
        assert torch.equal(compiled(x, wg.clone().requires_grad_(True), wu, wd), want)
    with torch.inference_mode():
        assert torch.equal(compiled(x, wg, wu, wd), want)
    y = compiled(x, wg.clone().requires_grad_(True), wu, wd)
    assert y.requires_grad and torch.equal(y.detach(), f(x, wg.clone().requires_grad_(True), wu, wd).detach())
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with torch.no_grad():
        y = compiled(x, wg, wu, wd)
    assert torch.cuda.max_memory_allocated() - base < rows * (512 * 4 + 128 * 2) + 8192   # h and y, not g and u
    assert torch.equal(y, want)


@gpu
def test_refusals(ffn):
    x, wg, wu, wd, _ = _make(4, 64, 128, 64)
    for bad in ((x.float(), wg, wu, wd), (x, wg.half(), wu, wd), (x, wg[:64], wu, wd), (x, wg, wu, wd[:, :64]), (x[:, :32], wg, wu, wd),
                (x, wg[0], wu[0], wd)):
        with pytest.raises(ValueError):
            ffn.gated_ffn(*bad)
    with pytest.raises(ValueError):
        ffn.gated_ffn(x, wg, wu, wd, "tanh")
    with pytest.raises(NotImplementedError):
        ffn.gated_ffn(x, wg[:100], wu[:100], wd[:, :100])
    with pytest.raises(RuntimeError):
        ffn.gated_ffn(x, wg.cpu(), wu, wd)


@gpu
def test_custom_op_refuses_what_does_not_fit(ffn):
    x, wg, wu, wd, dy = _make(40, 64, 128, 64)
    _, h, kept = ffn.gated_ffn_fwd(x, wg, wu, wd, "silu", True)
    all_ = [True] * 4
    assert len(ffn.gated_ffn_bwd(dy, x, wg, wu, wd, h, kept, "silu", all_)) == 4
    for bad in ((dy[:3], x, wg, wu, wd, h, kept), (dy, x[:8], wg, wu, wd, h, kept), (dy, x, wg, wu, wd, h[:8], kept),
                (dy, x, wg, wu, wd, h, kept[:-1]), (dy.float(), x, wg, wu, wd, h, kept)):
        with pytest.raises(ValueError):
            ffn.gated_ffn_bwd(*bad, "silu", all_)
    moved = torch.empty(kept.numel() + 4, dtype=torch.uint8, device="cuda")[4:]
    with pytest.raises(ValueError, match="aligned"):
        ffn.gated_ffn_bwd(dy, x, wg, wu, wd, h, moved, "silu", all_)


def test_refuses_cpu_tensors_and_widths():
    from thetascan_b200 import GatedFFN, gated_ffn
    with pytest.raises(RuntimeError):
        gated_ffn(*(torch.zeros(8, 8, dtype=BF16) for _ in range(4)))
    with pytest.raises(NotImplementedError):
        GatedFFN(60, 128)
    with pytest.raises(ValueError):
        GatedFFN(64, 128, "tanh")


def test_c_entry_refuses_bad_arguments():
    import ctypes
    from thetascan_b200 import _lib
    lib = _lib.load()
    assert lib.ts_b200_ffn_fwd(None, None) == _lib.TS_ERR_VALUE
    a = _lib.FfnArgs()
    a.rows, a.width, a.hidden, a.width_out = 4, 64, 100, 64
    assert lib.ts_b200_ffn_fwd(ctypes.byref(a), None) == _lib.TS_ERR_NOT_IMPLEMENTED
    assert lib.ts_b200_ffn_fwd_workspace_bytes(ctypes.byref(a)) == 0
    a.hidden = 128
    assert lib.ts_b200_ffn_fwd(ctypes.byref(a), None) == _lib.TS_ERR_VALUE      # null pointers
    # room for h (in two parts for few rows) and for dg and du
    assert lib.ts_b200_ffn_fwd_workspace_bytes(ctypes.byref(a)) >= 2 * 4 * 128 * 2
    assert lib.ts_b200_ffn_bwd_workspace_bytes(ctypes.byref(a)) >= 2 * 4 * 128 * 2
    a.x = a.w_gate = a.w_up = a.w_down = a.y = 256
    assert lib.ts_b200_ffn_fwd(ctypes.byref(a), None) == _lib.TS_ERR_VALUE      # no workspace
    a.h = 256
    assert lib.ts_b200_ffn_fwd(ctypes.byref(a), None) == _lib.TS_ERR_VALUE      # h without the projections
    a.rows, a.hidden = 33, 136
    assert lib.ts_b200_ffn_kept_bytes(ctypes.byref(a)) == 2 * 5 * 6144
    from thetascan_b200 import ffn
    assert ffn._kept_bytes(33, 136) == 2 * 5 * 6144
    a.activation = 9
    assert lib.ts_b200_ffn_fwd(ctypes.byref(a), None) == _lib.TS_ERR_VALUE
