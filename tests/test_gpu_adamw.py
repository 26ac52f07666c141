"""The AdamW step's kernel against its formula in float64.

Bounds, derived before any run: the step is a few f32 operations (the quotient
by an approximate division, 2 units in the last place), so the parameter's
change is within 1e-6 of itself and the result within a unit in the last
place of its type; the moments are two products and a sum, within 2^-22.  An
8-bit code lies within one of its steps (1/8 of the value, or 2^-9 of the
scale) of the f32 value.
"""
from __future__ import annotations

import math

import pytest
import torch

gpu = pytest.mark.gpu
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = (1, 7, 8, 255, 256, 257, 1000, 4096, 4099, 70001)


@pytest.fixture(scope="module")
def optim():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from thetascan_b200 import optim
    return optim


def _formula(p, g, m, v, step, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p - lr * weight_decay * p - lr / (1 - b1 ** step) * m / ((v / (1 - b2 ** step)).sqrt() + eps), m, v


def _case(sizes, pdtype, gdtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda n, s=1.0: (torch.randn(n, generator=gen) * s).cuda()  # noqa: E731
    ps = [r(n) for n in sizes]
    gs = [r(n, 0.01).to(gdtype) for n in sizes]
    ms = [r(n, 0.01) for n in sizes]
    vs = [r(n, 0.01).square() for n in sizes]
    return [p.to(pdtype) for p in ps], gs, ms, vs, ps


def _within_ulp(got, want, dtype, slack):
    ulp = want.abs() * (2.0 ** -8 if dtype == BF16 else 2.0 ** -23)
    assert ((got.double() - want).abs() <= ulp + slack).all()


@gpu
@pytest.mark.parametrize("pdtype,gdtype", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("master", [False, True])
def test_step_is_the_formulas(optim, pdtype, gdtype, master):
    if master and pdtype == F32:
        pytest.skip("masters belong to bf16 parameters")
    ps, gs, ms, vs, p32 = _case(SIZES, pdtype, gdtype)
    start = [(p32[i] if master else ps[i]).double() for i in range(len(SIZES))]
    want = [_formula(p, g.double(), m.double(), v.double(), 5, **HYPER) for p, g, m, v in zip(start, gs, ms, vs)]
    optim.adamw_step(ps, gs, ms, vs, step=5, **HYPER, masters=p32 if master else None)
    for i, (p, m, v) in enumerate(want):
        change = (p - start[i]).abs()
        _within_ulp(ps[i], p, pdtype, 1e-6 * change)
        if master:
            _within_ulp(p32[i], p, F32, 1e-6 * change)
        assert ((ms[i].double() - m).abs() <= 2.0 ** -22 * (m.abs() + 0.02)).all()
        assert ((vs[i].double() - v).abs() <= 2.0 ** -22 * v + 1e-40).all()


def _decode(codes, scales):
    return codes.double() * scales.double().repeat_interleave(256)[:codes.numel()]


@gpu
@pytest.mark.parametrize("pdtype,gdtype,master", [(F32, F32, False), (BF16, BF16, False), (BF16, F32, True)])
def test_8bit_step(optim, pdtype, gdtype, master):
    ps, gs, _, _, p32 = _case(SIZES, pdtype, gdtype, seed=2)
    zeros = lambda k: [torch.zeros(n, device="cuda", dtype=k) for n in SIZES]  # noqa: E731
    scales = lambda: [torch.zeros(optim.state_scales(n), device="cuda") for n in SIZES]  # noqa: E731
    m, r, ms, rs = zeros(E4M3), zeros(E4M3), scales(), scales()
    for step in (1, 2, 3):
        start = [(p32[i] if master else ps[i]).double() for i in range(len(SIZES))]
        want = [_formula(p, g.double(), _decode(a, sa), _decode(b, sb).square(), step, **HYPER)
                for p, g, a, sa, b, sb in zip(start, gs, m, ms, r, rs)]
        optim.adamw_step(ps, gs, m, r, step=step, **HYPER, masters=p32 if master else None, exp_avg_scales=ms,
                         exp_avg_sq_scales=rs, seed=11)
        for i, (p, first, second) in enumerate(want):
            _within_ulp(ps[i], p, pdtype, 2e-6 * (p - start[i]).abs())
            for value, codes, scale in ((first, m[i], ms[i]), (second.sqrt(), r[i], rs[i])):
                top = torch.stack([b.abs().max() for b in value.split(256)])
                assert ((scale.double() * 448 - top).abs() <= 1e-6 * top).all()
                each = scale.double().repeat_interleave(256)[:value.numel()]
                off = (_decode(codes, scale) - value).abs()
                assert (off <= (value.abs() / 8).maximum(each * 2.0 ** -9) * (1 + 1e-5)).all()
            assert ((r[i].float() > 0) | (second == 0)).all()


@gpu
def test_8bit_rounding_is_right_on_average(optim):
    # one value 0.3 of the block's largest in every element but one: its code is one of two neighbours; over n
    # elements the mean is within 5 standard deviations, 5 * step / 2 / sqrt(n), of the value
    n = 256 * 400
    g = torch.full((n,), 0.3, device="cuda")
    g[::256] = 1.0
    args = [[torch.zeros(n, device="cuda", dtype=E4M3)] for _ in range(2)]
    scales = [[torch.zeros(n // 256, device="cuda")] for _ in range(2)]
    p = [torch.zeros(n, device="cuda")]
    optim.adamw_step(p, [g], *args, step=1, **HYPER, exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1], seed=5)
    for codes, scale, value in ((args[0][0], scales[0][0], 0.1 * 0.3), (args[1][0], scales[1][0], math.sqrt(0.05) * 0.3)):
        x = _decode(codes, scale).view(-1, 256)[:, 1:]
        step = float(x.max() - x.min())
        assert 0 < step <= value / 8 * 1.001
        assert abs(float(x.mean()) - value) <= 5 * step / 2 / math.sqrt(x.numel())


@gpu
def test_8bit_rounding_follows_its_key(optim):
    def once(seed, ordinals):
        ps, gs, _, _, _ = _case((5000, 5000), F32, F32)
        gs[1] = gs[0]
        m, r = ([torch.zeros(5000, device="cuda", dtype=E4M3) for _ in range(2)] for _ in range(2))
        ms, rs = ([torch.zeros(20, device="cuda") for _ in range(2)] for _ in range(2))
        optim.adamw_step(ps, gs, m, r, step=1, **HYPER, exp_avg_scales=ms, exp_avg_sq_scales=rs, seed=seed,
                         ordinals=ordinals)
        return [t.view(torch.uint8) for t in m + r]

    a = once(1, [0, 1])
    assert all(torch.equal(x, y) for x, y in zip(a, once(1, [0, 1])))
    assert not torch.equal(a[0], a[1]) and not torch.equal(a[0], once(2, [0, 1])[0])
    assert torch.equal(a[1], once(1, [1, 0])[0])


@gpu
def test_many_tensors_mixed_kinds_and_alignment(optim):
    # more tensors than one launch takes, sizes of zero among them, views that start at odd elements
    gen = torch.Generator().manual_seed(8)
    sizes = [int(torch.randint(0, 700, (1,), generator=gen)) for _ in range(900)]
    flat = [torch.randn(sum(sizes) + 900, generator=gen).cuda() for _ in range(3)]
    flat.append(torch.rand(sum(sizes) + 900, generator=gen).cuda())
    lists, at = [[] for _ in flat], 0
    for i, n in enumerate(sizes):
        for x, f in zip(lists, flat):
            x.append(f[at + i:at + i + n])
        at += n
    ps = [p.to(BF16) if i % 3 == 0 else p.clone() for i, p in enumerate(lists[0])]
    want = [_formula(p.double(), g.double(), m.double(), v.double(), 2, **HYPER) for p, g, m, v in zip(ps, *lists[1:])]
    start = [p.double() for p in ps]
    optim.adamw_step(ps, lists[1], lists[2], lists[3], step=2, **HYPER)
    for p, m, v, (wp, wm, wv), s in zip(ps, lists[2], lists[3], want, start):
        _within_ulp(p, wp, p.dtype, 1e-6 * (wp - s).abs())
        assert ((m.double() - wm).abs() <= 2.0 ** -22 * (wm.abs() + 2)).all()
        assert ((v.double() - wv).abs() <= 2.0 ** -21 * wv).all()


def _mix32(x):
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


@gpu
def test_8bit_states_are_the_formulas_to_the_bit(optim):
    # each sum, product, root and quotient rounded to f32 by itself (the CPU's are), the code's random rounding in float64
    # (exact).  The kernel's root is the next value in one case of a million: of 4000 blocks' scales at most one may be
    # off, and in the other blocks a code where its value is within 2^-20 of a step's end, at most ten in a million.
    n, seed = 4000 * 256, 17
    b1, b2 = HYPER["betas"]
    f = lambda v: torch.tensor(v, dtype=F32)  # noqa: E731
    gen = torch.Generator().manual_seed(12)
    m, r = (torch.zeros(n, device="cuda", dtype=E4M3) for _ in range(2))
    ms, rs = (torch.zeros(n // 256, device="cuda") for _ in range(2))
    p = torch.zeros(n, device="cuda")
    for step in (1, 2, 3):
        g = torch.randn(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen) - 7)
        state = [(c.cpu().float().view(-1, 256) * s.cpu()[:, None]).view(-1) for c, s in ((m, ms), (r, rs))]
        optim.adamw_step([p], [g.cuda()], [m], [r], step=step, **HYPER, exp_avg_scales=[ms], exp_avg_sq_scales=[rs], seed=seed)
        first = f(b1) * state[0] + f(1 - b1) * g
        root = (f(b2) * (state[1] * state[1]) + f(1 - b2) * (g * g)).double().sqrt().float()   # the CPU's f32 root is not rounded correctly
        word = _mix32(torch.arange(n) ^ _mix32(torch.tensor(_mix32((seed + 0x9E3779B9 * step) & 0xFFFFFFFF))))
        for x, codes, scales, u in ((first, m, ms, word & 0xFFFF), (root, r, rs, word >> 16)):
            blocks = x.view(-1, 256)
            want = blocks.abs().amax(1) * f(1 / 448)
            same = scales.cpu() == want
            assert int((~same).sum()) <= 1
            a = (blocks.abs() / want[:, None]).double()
            size = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
            code = (torch.floor(a / size + u.view(-1, 256) / 65536) * size).clamp_max(448.0)
            if codes is r:
                code = torch.where(blocks > 0, code.clamp_min(2.0 ** -9), code)
            got = codes.cpu().double().view(-1, 256)
            assert int(((got != code * blocks.sign().double()) & same[:, None]).sum()) <= 10


@gpu
def test_step_inside_a_compiled_function(optim):
    # the step is not traced: the graph breaks around it and goes on with what it wrote
    def f(p, g, m, v):
        optim.adamw_step([p], [g * 2], [m], [v], step=1, **HYPER)
        return p * 2 + m

    torch._dynamo.reset()
    make = lambda: [torch.rand(300, generator=torch.Generator().manual_seed(i)).cuda() for i in range(4)]  # noqa: E731
    a, b = make(), make()
    want, got = f(*a), torch.compile(f, backend="aot_eager")(*b)
    assert torch.equal(want, got) and all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_8bit_special_values(optim):
    n = 1024
    g = torch.zeros(n, device="cuda")
    g[300] = float("nan")
    g[600] = 1e-30
    m, r = (torch.zeros(n, device="cuda", dtype=E4M3) for _ in range(2))
    ms, rs = (torch.zeros(4, device="cuda") for _ in range(2))
    p = torch.ones(n, device="cuda")
    optim.adamw_step([p], [g], [m], [r], step=1, **HYPER, exp_avg_scales=[ms], exp_avg_sq_scales=[rs])
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[300] = True
    assert torch.equal(p.isnan(), bad) and torch.equal(m.float().isnan(), bad) and torch.equal(r.float().isnan(), bad)
    assert ms.isfinite().all() and rs.isfinite().all()
    assert (m.float()[:256] == 0).all() and (r.float()[:256] == 0).all()


@gpu
@pytest.mark.parametrize("size", [1e-21, 1e-12, 1e6, 1e12])
def test_8bit_step_at_extreme_magnitudes(optim, size):
    # the first step moves by lr (with eps = 0) whatever the gradient's size; v itself is 1e-42 to 1e24
    gen = torch.Generator().manual_seed(3)
    g = (size * (1 + torch.rand(700, generator=gen))).cuda()
    m, r = (torch.zeros(700, device="cuda", dtype=E4M3) for _ in range(2))
    ms, rs = (torch.zeros(3, device="cuda") for _ in range(2))
    p = torch.zeros(700, device="cuda")
    optim.adamw_step([p], [g], [m], [r], step=1, lr=1.0, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0, exp_avg_scales=[ms],
                     exp_avg_sq_scales=[rs])
    assert ((p + 1).abs() <= 1e-5).all()
    for codes, scale, c in ((m, ms, 0.1), (r, rs, math.sqrt(0.05))):
        off = (_decode(codes, scale) - c * g.double()).abs()
        assert (off <= c * g.double() / 8 * 1.0001).all()


@gpu
@pytest.mark.parametrize("pdtype,gdtype,master", [(F32, F32, False), (BF16, BF16, False), (BF16, F32, True)])
@pytest.mark.parametrize("size", [2e14, 3e14, 1e16, 1e19, 1e25, 1e37])
def test_8bit_step_of_large_finite_gradients(optim, size, pdtype, gdtype, master):
    # the first step moves by lr (with eps = 0) whatever the gradient's size, in the blocks with one large gradient, the
    # whole one and the ragged last one, as in those without.  f32: a few roundings and an approximate quotient, 1e-5;
    # the gradient's own rounding cancels.  A block's small values keep their step, and the least code.
    gen = torch.Generator().manual_seed(6)
    g = torch.rand(700, generator=gen) + 1
    g[:256] *= size
    g[256:] *= 1e-3
    g[600] = size
    g = g.to(gdtype).cuda()
    m, r = (torch.zeros(700, device="cuda", dtype=E4M3) for _ in range(2))
    ms, rs = (torch.zeros(3, device="cuda") for _ in range(2))
    p, p32 = torch.zeros(700, device="cuda", dtype=pdtype), torch.zeros(700, device="cuda")
    optim.adamw_step([p], [g], [m], [r], step=1, lr=1.0, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0, exp_avg_scales=[ms],
                     exp_avg_sq_scales=[rs], masters=[p32] if master else None)
    for value in (p, p32) if master else (p,):
        _within_ulp(value, torch.full((700,), -1.0, device="cuda", dtype=torch.float64), value.dtype, 1e-5)
    for codes, scale, c in ((m, ms, 0.1), (r, rs, math.sqrt(0.05))):
        want = c * g.double()
        top = torch.stack([b.max() for b in want.split(256)])
        assert ((scale.double() * 448 - top).abs() <= 1e-6 * top).all()
        each = scale.double().repeat_interleave(256)[:700]
        assert ((_decode(codes, scale) - want).abs() <= (want / 8).maximum(each * 2.0 ** -9) * 1.0001).all()
    assert (r.float() > 0).all()


@gpu
@pytest.mark.parametrize("pdtype,gdtype,master", [(F32, F32, False), (BF16, BF16, False), (BF16, F32, True)])
@pytest.mark.parametrize("size", [1e-18, 1e-20, 1e-21, 1e-22, 1e-24, 1e-27])
def test_8bit_step_of_tiny_gradients(optim, size, pdtype, gdtype, master):
    # as above: steps of lr whatever the gradient's size, next to zeros (whose step is 0 / 0 with eps = 0: left out) and
    # next to ordinary values
    gen = torch.Generator().manual_seed(7)
    g = (torch.rand(700, generator=gen) + 1) * size
    g[256:400] = 1e-3
    g[3] = g[650] = 0
    g = g.to(gdtype).cuda()
    m, r = (torch.zeros(700, device="cuda", dtype=E4M3) for _ in range(2))
    ms, rs = (torch.zeros(3, device="cuda") for _ in range(2))
    p, p32 = torch.zeros(700, device="cuda", dtype=pdtype), torch.zeros(700, device="cuda")
    optim.adamw_step([p], [g], [m], [r], step=1, lr=1.0, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0, exp_avg_scales=[ms],
                     exp_avg_sq_scales=[rs], masters=[p32] if master else None)
    there = g != 0
    for value in (p, p32) if master else (p,):
        _within_ulp(value[there], torch.full((698,), -1.0, device="cuda", dtype=torch.float64), value.dtype, 1e-5)
    for codes, scale, c in ((m, ms, 0.1), (r, rs, math.sqrt(0.05))):
        want = c * g.double()
        top = torch.stack([b.max() for b in want.split(256)])
        assert ((scale.double() * 448 - top).abs() <= 1e-6 * top).all()
        each = scale.double().repeat_interleave(256)[:700]
        assert ((_decode(codes, scale) - want).abs() <= (want / 8).maximum(each * 2.0 ** -9) * 1.0001).all()
    assert torch.equal(r.float() > 0, there)


@gpu
def test_8bit_roots_without_gradients_fade_evenly(optim):
    # no gradient and no first moment: the root shrinks by sqrt(b2) a step at every size down to the least scale
    sizes = torch.tensor([1e-15, 1e-18, 1e-21, 1e-24, 1e-27], dtype=torch.float64)
    n = 256 * len(sizes)
    m, r = torch.zeros(n, device="cuda", dtype=E4M3), torch.full((n,), 448.0, device="cuda").to(E4M3)
    ms, rs = torch.zeros(len(sizes), device="cuda"), (sizes / 448).float().cuda()
    start, g = rs.double(), torch.zeros(n, device="cuda")
    p = torch.ones(n, device="cuda")
    optim.adamw_step([p], [g], [m], [r], step=9, **HYPER, exp_avg_scales=[ms], exp_avg_sq_scales=[rs])
    assert ((rs.double() / start - math.sqrt(0.95)).abs() <= 1e-6).all()
    assert ((p.double() - (1 - HYPER["lr"] * HYPER["weight_decay"])).abs() <= 1e-6).all()


@gpu
@pytest.mark.parametrize("size", [1e-24, 1e-3, 1e16, 1e30])
def test_8bit_steps_go_on_at_any_magnitude_and_alignment(optim, size):
    # five steps on views that start at odd elements: the decoded states follow the average of what went in, whose codes
    # are within 1/16 of a step (2^-3 of the value at most) each time, and the parameter moves by lr within the sum of
    # both moments' errors (5 * 2^-3 in the worst order)
    n = 1000
    gen = torch.Generator().manual_seed(9)
    hold = lambda dtype: torch.zeros(n + 3, device="cuda", dtype=dtype)[3:]  # noqa: E731
    m, r, p, g = hold(E4M3), hold(E4M3), hold(F32), hold(F32)
    ms, rs = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    g.copy_((1 + 0.1 * torch.rand(n, generator=gen)) * size)
    for step in range(1, 6):
        before = p.clone()
        optim.adamw_step([p], [g], [m], [r], step=step, lr=1.0, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0,
                         exp_avg_scales=[ms], exp_avg_sq_scales=[rs], seed=3)
        assert ((p - before + 1).abs() <= 5 * 2.0 ** -3).all()
        assert ((p - before).mean() + 1).abs() <= 0.02
        for codes, scale, c in ((m, ms, 1 - 0.9 ** step), (r, rs, math.sqrt(1 - 0.95 ** step))):
            assert ((_decode(codes, scale) / (c * g.double()) - 1).abs() <= 5 * 2.0 ** -3).all()


@gpu
def test_8bit_infinite_value_makes_its_block_non_finite(optim):
    g = torch.ones(600, device="cuda")
    g[10] = float("inf")
    m, r = (torch.zeros(600, device="cuda", dtype=E4M3) for _ in range(2))
    ms, rs = (torch.zeros(3, device="cuda") for _ in range(2))
    p = torch.ones(600, device="cuda")
    optim.adamw_step([p], [g], [m], [r], step=1, **HYPER, exp_avg_scales=[ms], exp_avg_sq_scales=[rs])
    assert not p[10].isfinite() and p[:10].isfinite().all() and p[11:].isfinite().all()
    for codes, scale in ((m, ms), (r, rs)):
        x = _decode(codes, scale)
        assert not x[:256].isfinite().any() and x[256:].isfinite().all() and (x[256:] > 0).all()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, True)])
def test_optimizer_learns_and_resumes(optim, bits, dtype, master):
    # a quadratic bowl from the origin: Adam moves about lr a step, so 300 steps of 1e-2 reach targets within 1
    torch.manual_seed(0)
    target = torch.rand(33, 65, device="cuda") * 2 - 1
    make = lambda ps: optim.AdamW(ps, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.0, state_bits=bits, master_weights=master)  # noqa: E731

    def steps(p, frozen, opt, count):
        for _ in range(count):
            opt.zero_grad()
            ((p.float() - target).square().sum() * 0.5).backward()
            opt.step()

    p = torch.zeros(33, 65, device="cuda", dtype=dtype, requires_grad=True)
    frozen = torch.zeros(4, device="cuda", requires_grad=True)
    opt = make([p, frozen])
    steps(p, frozen, opt, 300)
    assert float((p.float() - target).abs().mean()) < 0.02 and (frozen == 0).all()
    q = p.detach().clone().requires_grad_(True)
    again = make([q, frozen])
    again.load_state_dict(opt.state_dict())
    for k, v in opt.state[p].items():
        w = again.state[q][k]
        assert w == v if k == "step" else (w.dtype == v.dtype and w is not v and torch.equal(w.view(torch.uint8), v.view(torch.uint8)))
    steps(p, frozen, opt, 3)
    steps(q, frozen, again, 3)
    assert torch.equal(p, q)


@gpu
def test_optimizer_groups_follow_torch(optim):
    # the same steps as torch.optim.AdamW on its single-tensor path; both are f32, so a few units in the last place apart
    torch.manual_seed(1)
    a = [torch.randn(n, device="cuda", requires_grad=True) for n in (5, 300, 4097)]
    b = [t.detach().clone().requires_grad_(True) for t in a]
    groups = lambda x: [dict(params=x[:2], lr=1e-3), dict(params=x[2:], weight_decay=0.0)]  # noqa: E731
    ours, theirs = optim.AdamW(groups(a), lr=2e-3), torch.optim.AdamW(groups(b), lr=2e-3, foreach=False)
    for i in range(5):
        for x, y in zip(a, b):
            x.grad = torch.randn_like(x)
            y.grad = x.grad.clone()
        if i == 2:
            a[1].grad = b[1].grad = None   # its count of steps falls behind the others'
        ours.step()
        theirs.step()
    for x, y in zip(a, b):
        assert ((x - y).abs() <= 1e-6 * (1 + y.abs())).all()


@gpu
def test_step_is_refused_in_a_graph_and_seen_by_autograd(optim):
    p = torch.ones(64, device="cuda", requires_grad=True)
    args = [[torch.zeros(64, device="cuda")] for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            torch.zeros(1, device="cuda")
            optim.adamw_step([p], *args, step=1, **HYPER)
    loss = (p * p).sum()
    optim.adamw_step([p], *args, step=1, **HYPER)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@gpu
def test_refusals(optim):
    p, g, m, v = ([torch.ones(300, device="cuda")] for _ in range(4))
    ok = dict(step=1, **HYPER)
    optim.adamw_step([], [], [], [], **ok)
    for bad in (dict(step=0), dict(step=1.5), dict(betas=(1.0, 0.9)), dict(lr=-1.0), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            optim.adamw_step(p, g, m, v, **{**ok, **bad})
    for lists in ((p, [], m, v), (p, g, [], v), (p, [g[0][:299]], m, v), (p, g, [m[0].bfloat16()], v), ([p[0].half()], g, m, v),
                  (p, [g[0].half()], m, v), ([torch.ones(10, 30, device="cuda").T], g, m, v), (p, [g[0].cpu()], m, v)):
        with pytest.raises(ValueError):
            optim.adamw_step(*lists, **ok)
    with pytest.raises(ValueError):
        optim.adamw_step(p, g, m, v, **ok, masters=[p[0].clone()])
    with pytest.raises(ValueError):
        optim.adamw_step(p, g, m, v, **ok, exp_avg_scales=[m[0][:2]], exp_avg_sq_scales=[m[0][:2]])
    code = [torch.zeros(300, device="cuda", dtype=E4M3)]
    with pytest.raises(ValueError):
        optim.adamw_step(p, g, code, code, **ok)
    with pytest.raises(ValueError):
        optim.adamw_step(p, g, code, code, **ok, exp_avg_scales=[m[0][:1]], exp_avg_sq_scales=[m[0][:2]])
    assert (p[0] == 1).all()
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0))):
        with pytest.raises(ValueError):
            optim.AdamW([torch.ones(3, device="cuda", requires_grad=True)], **bad)
    with pytest.raises(ValueError):
        optim.AdamW([torch.ones(3, 4, device="cuda").T.requires_grad_(True)])
    with pytest.raises(RuntimeError):
        optim.adamw_step([torch.ones(3)], [torch.ones(3)], [torch.ones(3)], [torch.ones(3)], **ok)


def test_a_refused_step_does_not_count():
    # on the CPU every step is refused; the bias corrections of the next one must not move
    from thetascan_b200 import AdamW
    p = torch.ones(8, requires_grad=True)
    opt = AdamW([p])
    p.grad = torch.ones(8)
    for _ in range(2):
        with pytest.raises(RuntimeError):
            opt.step()
    assert opt.state[p]["step"] == 0
    p.grad = torch.sparse_coo_tensor([[1]], [1.0], (8,))
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    assert opt.state[p]["step"] == 0 and (p == 1).all()


@gpu
def test_steps_after_a_refused_one(optim):
    a, b = (torch.ones(300, device="cuda", requires_grad=True) for _ in range(2))
    x, y = optim.AdamW([a]), optim.AdamW([b])
    for i in range(3):
        a.grad = torch.full((300,), 0.5 + i, device="cuda")
        b.grad = a.grad.clone()
        if i == 1:
            x.param_groups[0]["betas"] = (2.0, 0.9)
            with pytest.raises(ValueError):
                x.step()
            x.param_groups[0]["betas"] = (0.9, 0.999)
        x.step()
        y.step()
    assert torch.equal(a, b) and x.state[a]["step"] == 3


def test_options_of_a_group_are_checked_as_the_defaults_are():
    from thetascan_b200 import AdamW
    p, q = torch.ones(8, requires_grad=True), torch.ones(8, requires_grad=True)
    opt = AdamW([p])
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([dict(params=[q], **bad)])
        with pytest.raises(ValueError):
            AdamW([q], **bad)
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[q], **bad))
        assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[q], state_bits=8, lr=0.5))
    assert opt.param_groups[1]["state_bits"] == 8


@gpu
def test_lists_are_of_the_parameters_shapes_or_flat(optim):
    make = lambda *shape: torch.rand(shape, generator=torch.Generator().manual_seed(1)).cuda()  # noqa: E731
    args = [make(4, 6) for _ in range(5)]
    args[0] = args[0].bfloat16()
    for i in range(1, 5):
        for shape in ((6, 4), (4, 3, 2)):
            bad = [t.reshape(shape) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(ValueError):
                optim.adamw_step(*([t] for t in bad[:4]), step=1, **HYPER, masters=[bad[4]])
    flat = [t.clone().reshape(-1) if i else t.clone() for i, t in enumerate(args)]
    for lists in (args, flat):
        optim.adamw_step(*([t] for t in lists[:4]), step=1, **HYPER, masters=[lists[4]])
    assert all(torch.equal(a, b.view(4, 6)) for a, b in zip(args, flat))


def test_c_entry_refuses_bad_arguments():
    import ctypes
    from thetascan_b200 import _lib
    lib = _lib.load()
    assert lib.ts_b200_adamw(None, None) == _lib.TS_ERR_VALUE
    t = _lib.AdamWTensor()
    t.n = 4
    a = _lib.AdamWArgs()
    a.count, a.tensors, a.step, a.state_bits = 1, ctypes.addressof(t), 1, 32
    assert lib.ts_b200_adamw(ctypes.byref(a), None) == _lib.TS_ERR_VALUE      # null pointers
    a.state_bits = 16
    assert lib.ts_b200_adamw(ctypes.byref(a), None) == _lib.TS_ERR_NOT_IMPLEMENTED
    a.state_bits, a.step = 32, 0
    assert lib.ts_b200_adamw(ctypes.byref(a), None) == _lib.TS_ERR_VALUE
    a.step, a.master = 1, 1
    assert lib.ts_b200_adamw(ctypes.byref(a), None) == _lib.TS_ERR_VALUE      # a master behind an f32 parameter
