"""Operators around the mixer, as they are timed and checked: the root-mean-square norm that adds the residual (with its
backward pass, and with an output in 8 bits), the gated feed-forward block (with its backward pass), and the AdamW step
over many tensors (32-bit and 8-bit states).

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges, ``prepare`` makes what a program holds
before the call, ``run`` is one call: with ``own`` the framework's operator, without it the same operator in elementary
torch operations in 32 bits.  ``exact`` evaluates the definition in 64 bits.
"""
import math
import random

import torch

own = False

EPS = 1e-6              # of the norm
E4M3_MAX = 448.0        # largest value of the 8-bit type
TINY = 2.0 ** -100      # smallest largest magnitude that a scale is made for
STATE_BLOCK = 256       # elements of an 8-bit optimizer state that share a scale
LR, BETAS, ADAM_EPS, DECAY = 1e-3, (0.9, 0.95), 1e-8, 0.1
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step of four sequences: latency
        dict(name="norm_step", op="norm", mode="forward", rows=4, width=1024, dtype="bf16", weight="bf16", residual=True, group=0),
        # the hybrid language model's training batch (64 x 1024 tokens of width 512) with the framework's f32 weights
        dict(name="norm_train", op="norm", mode="train", rows=65536, width=512, dtype="bf16", weight="f32", residual=True, group=0),
        # the first norm of a float32 model (nothing to add yet) whose width no vector load divides
        dict(name="norm_train_odd_f32", op="norm", mode="train", rows=4099, width=1537, dtype="f32", weight="f32", residual=False, group=0),
        # a prompt's activations on their way into an 8-bit projection, a scale for each 128 columns
        dict(name="norm_8bit", op="norm", mode="8bit", rows=16384, width=2048, dtype="bf16", weight="bf16", residual=True, group=128),
        # one token: the weights are read once
        dict(name="ffn_token", op="ffn", mode="forward", rows=1, width=1024, hidden=4096, activation="silu"),
        # a prompt of no round length
        dict(name="ffn_prompt", op="ffn", mode="forward", rows=1531, width=1024, hidden=2816, activation="gelu"),
        # the hybrid language model's training batch and widths
        dict(name="ffn_train", op="ffn", mode="train", rows=65536, width=512, hidden=1024, activation="relu2"),
        # a wider model's training batch
        dict(name="ffn_train_wide", op="ffn", mode="train", rows=8192, width=2048, hidden=5632, activation="silu"),
        # a few small tensors (an adapter's): latency
        dict(name="adamw_small", op="adamw", layout="ragged", tensors=6, total=20000, param="f32", grad="f32", bits=32),
        # the hybrid language model in f32
        dict(name="adamw_lm", op="adamw", layout="lm", layers=9, width=512, hidden=1024, param="f32", grad="f32", bits=32),
        # bf16 parameters with f32 masters, tensors of uneven sizes
        dict(name="adamw_master", op="adamw", layout="ragged", tensors=40, total=120_000_001, param="bf16+master", grad="bf16", bits=32),
        # a larger model in bf16 with states in 8 bits
        dict(name="adamw_8bit", op="adamw", layout="lm", layers=12, width=1024, hidden=4096, param="bf16", grad="bf16", bits=8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _not(n, other):
    return n + 8 if n == other else n


def draw(rng):
    op = rng.choice(["norm", "ffn", "adamw"])
    if op == "norm":
        width = _not(_log(rng, 64, 16384), 3072)
        if rng.random() < 0.6:
            width = _not(max(64, width // 64 * 64), 3072)
        rows = _log(rng, 1, max(1, min(65536, (1 << 25) // width)))
        mode = rng.choice(["forward", "train", "8bit"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        return dict(op=op, mode=mode, rows=_not(rows, 3072), width=width, dtype=dtype, weight=rng.choice(["f32", dtype]),
                    residual=rng.random() < 0.7, group=rng.choice([0, 128]) if mode == "8bit" else 0)
    if op == "ffn":
        mode = rng.choice(["forward", "forward", "train"])
        width = _not(_log(rng, 256, 2048) // 8 * 8, 3072)
        hidden = _not(_log(rng, 256, 5632) // 8 * 8, 3072)
        most = int(1.6e12 / ((18 if mode == "train" else 6) * width * hidden))
        rows = _not(_log(rng, 1, max(1, min(65536, most))), 3072)
        return dict(op=op, mode=mode, rows=rows, width=width, hidden=hidden, activation=rng.choice(["silu", "gelu", "relu2"]))
    bits = rng.choice([32, 8])
    param = rng.choice(["f32", "bf16", "bf16+master"])
    grad = rng.choice(["f32", "bf16"]) if param == "bf16+master" else param
    if rng.random() < 0.3:
        return dict(op=op, layout="lm", layers=rng.randint(1, 12), width=rng.choice([256, 512, 1024]), hidden=_not(rng.randint(32, 512) * 8, 3072),
                    param=param, grad=grad, bits=bits)
    total = _log(rng, 1000, 120_000_000)
    return dict(op=op, layout="ragged", tensors=min(_log(rng, 1, 200), total // 20), total=total, param=param, grad=grad, bits=bits)


def _sizes(case):
    """Element counts of the optimizer case's tensors."""
    if case["layout"] == "lm":
        d, h = case["width"], case["hidden"]
        block = [d, d * d, d * d, d * d, d * d, d, d * h, d * h, d * h]
        return [1024 * d] + block * case["layers"] + [d]
    rng = random.Random(case["total"] * 1009 + case["tensors"])
    share = [math.exp(rng.uniform(0, 5)) for _ in range(case["tensors"])]
    got = [max(1, int(case["total"] * s / sum(share))) for s in share]
    got[-1] += max(0, case["total"] - sum(got))
    return got


# --------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    if case["op"] == "norm":
        rows, width, t = case["rows"], case["width"], DTYPES[case["dtype"]]
        spread = torch.exp(0.5 * normal(width))  # channels of a residual stream differ in size
        state = dict(case=case, x=normal(rows, width, dtype=t), weight=(1 + 0.2 * normal(width)).to(DTYPES[case["weight"]]))
        if case["residual"]:
            state["residual"] = (normal(rows, width) * 3 * spread).to(t)
        if case["mode"] == "train":
            state["dy"] = normal(rows, width, dtype=t)
            if case["residual"]:
                state["dsum"] = normal(rows, width, dtype=t)
        return state
    if case["op"] == "ffn":
        rows, d, h, t = case["rows"], case["width"], case["hidden"], torch.bfloat16
        state = dict(case=case, x=normal(rows, d, dtype=t), w_gate=normal(h, d, scale=1.5 / math.sqrt(d), dtype=t),
                     w_up=normal(h, d, scale=1.0 / math.sqrt(d), dtype=t), w_down=normal(d, h, scale=1.0 / math.sqrt(h), dtype=t))
        if case["mode"] == "train":
            state["dy"] = normal(rows, d, dtype=t)
        return state

    # The tensors are views of flat buffers, each at a multiple of 64 elements (its scales back to back).
    sizes = _sizes(case)
    starts, blocks, at, at_block = [], [], 0, 0
    for n in sizes:
        starts.append(at)
        blocks.append(at_block)
        at += -(-n // 64) * 64
        at_block += -(-n // STATE_BLOCK)

    def views(flat):
        return [flat[a:a + n] for a, n in zip(starts, sizes)]

    master = normal(at, scale=0.05)
    sigma = torch.exp(1.5 * normal(at) - 7)
    m = normal(at).mul_(0.3).mul_(sigma)
    r = sigma.mul_(0.5 + torch.rand(at, generator=gen, device="cuda"))
    grad = normal(at).mul_(r).to(DTYPES[case["grad"]])
    state = dict(case=case, step=50 + seed % 50, seed=seed % 1_000_003)
    flat = dict(param=master if case["param"] == "f32" else master.to(torch.bfloat16))
    if case["param"] == "bf16+master":
        flat["master"] = master
    if case["bits"] == 32:
        flat |= dict(exp_avg=m, exp_avg_sq=r.square_())
    else:
        for name, x in (("exp_avg", m), ("exp_avg_sq", r)):
            code = torch.zeros(at, dtype=torch.float8_e4m3fn, device="cuda")
            scale = torch.zeros(at_block, device="cuda")
            for a, b, n in zip(starts, blocks, sizes):
                k = -(-n // STATE_BLOCK)
                y = torch.zeros(k * STATE_BLOCK, device="cuda")
                y[:n] = x[a:a + n]
                y = y.view(k, STATE_BLOCK)
                scale[b:b + k] = y.abs().amax(1) / E4M3_MAX
                y = y / scale[b:b + k, None].clamp_min(TINY)
                if name == "exp_avg_sq":
                    y = y.clamp_min(2.0 ** -9)
                code[a:a + n] = y.view(-1)[:n].to(torch.float8_e4m3fn)
            flat[name] = code
            flat[name + "_scale"] = scale
        for name in ("exp_avg_scale", "exp_avg_sq_scale"):
            state[name + "s"] = [flat[name][b:b - (-n // STATE_BLOCK)] for b, n in zip(blocks, sizes)]
    for name in ("param", "master", "exp_avg", "exp_avg_sq"):
        if name in flat:
            state[name + "s"] = views(flat[name])
    state.update(flat=flat, grads=views(grad))
    return state


# --------------------------------------------------------------------------- one pass

def run(state):
    return {"norm": _run_norm, "ffn": _run_ffn, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_norm(s):
    return _own_norm(s) if own else _plain_norm(s)


def _run_ffn(s):
    return _own_ffn(s) if own else _plain_ffn(s)


def _run_adamw(s):
    """The states and parameters change in place; the next pass is the next step."""
    s["step"] += 1
    (_own_adamw if own else _plain_adamw)(s)
    return s["flat"]


def _own_norm(s):
    from thetascan_b200 import add_rms_norm, rms_norm, rms_norm_8bit
    case, residual = s["case"], s.get("residual")
    if case["mode"] == "8bit":
        return rms_norm_8bit(s["x"], s["weight"], EPS, residual=residual, group=case["group"] or None)
    if case["mode"] == "forward":
        with torch.no_grad():
            return rms_norm(s["x"], s["weight"], EPS) if residual is None else add_rms_norm(s["x"], residual, s["weight"], EPS)
    x, weight = s["x"].detach().requires_grad_(True), s["weight"].detach().requires_grad_(True)
    if residual is None:
        y = rms_norm(x, weight, EPS)
        return (y.detach(), *torch.autograd.grad(y, (x, weight), s["dy"]))
    y, total = add_rms_norm(x, residual, weight, EPS)
    return (y.detach(), total.detach(), *torch.autograd.grad((y, total), (x, weight), (s["dy"], s["dsum"])))


def _plain_norm(s):
    case, x, w = s["case"], s["x"], s["weight"].float()
    total = x if s.get("residual") is None else (x.float() + s["residual"].float()).to(x.dtype)  # the residual stream, as it is stored
    a = total.float()
    inv = (a.square().mean(-1, keepdim=True) + EPS).rsqrt()
    unit = a * inv
    y = unit * w
    streams = () if s.get("residual") is None else (total,)
    if case["mode"] == "8bit":
        group = case["group"] or case["width"]
        n = -(-case["width"] // group)
        padded = torch.zeros(case["rows"], n * group, device=y.device)
        padded[:, :case["width"]] = y
        scale = padded.view(-1, n, group).abs().amax(-1).clamp_min(TINY) / E4M3_MAX
        code = (padded.view(-1, n, group) / scale[..., None]).view(-1, n * group)[:, :case["width"]]
        return (code.to(torch.float8_e4m3fn), scale, *streams)
    if case["mode"] == "forward":
        return y.to(x.dtype) if not streams else (y.to(x.dtype), total)
    dy = s["dy"].float()
    du = dy * w
    dx = (du - unit * (du * unit).mean(-1, keepdim=True)) * inv
    if streams:
        dx = dx + s["dsum"].float()
    return (y.to(x.dtype), *streams, dx.to(x.dtype), (dy * unit).sum(0).to(s["weight"].dtype))


def _own_ffn(s):
    from thetascan_b200 import gated_ffn
    weights = [s["w_gate"], s["w_up"], s["w_down"]]
    if s["case"]["mode"] == "forward":
        with torch.no_grad():
            return gated_ffn(s["x"], *weights, activation=s["case"]["activation"])
    leaves = [t.detach().requires_grad_(True) for t in (s["x"], *weights)]
    y = gated_ffn(*leaves, activation=s["case"]["activation"])
    return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))


def _plain_ffn(s):
    kind = s["case"]["activation"]
    x, wg, wu, wd = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    t = s["x"].dtype
    g, u = x @ wg.T, x @ wu.T
    if kind == "silu":
        gate = torch.sigmoid(g)
        act = g * gate
    elif kind == "gelu":
        gate = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        act = g * gate
    else:
        gate = g.clamp_min(0)
        act = gate.square()
    h = act * u
    y = (h @ wd.T).to(t)
    if s["case"]["mode"] == "forward":
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    if kind == "silu":
        slope = gate * (1 + g * (1 - gate))
    elif kind == "gelu":
        slope = gate + g * torch.exp(-0.5 * g.square()) / math.sqrt(2 * math.pi)
    else:
        slope = 2 * gate
    du, dg = dh * act, dh * u * slope
    return y, (dg @ wg + du @ wu).to(t), (dg.T @ x).to(t), (du.T @ x).to(t), (dy.T @ h).to(t)


def _own_adamw(s):
    from thetascan_b200 import adamw_step
    adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=s["step"], lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY,
               masters=s.get("masters"), exp_avg_scales=s.get("exp_avg_scales"), exp_avg_sq_scales=s.get("exp_avg_sq_scales"), seed=s["seed"])


def _plain_adamw(s):
    b1, b2 = BETAS
    c1, c2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]
    if s["case"]["bits"] == 8:
        masters = s.get("masters") or [None] * len(s["params"])
        [_plain_adamw_8bit(i, s["seed"], s["step"], c1, c2, *t) for i, t in enumerate(zip(
            s["params"], masters, s["grads"], s["exp_avgs"], s["exp_avg_scales"], s["exp_avg_sqs"], s["exp_avg_sq_scales"]))]
        return
    m, v = s["exp_avgs"], s["exp_avg_sqs"]
    p = s.get("masters") or ([t.float() for t in s["params"]] if s["case"]["param"] == "bf16" else s["params"])
    g = s["grads"] if s["case"]["grad"] == "f32" else [t.float() for t in s["grads"]]
    torch._foreach_mul_(m, b1)
    torch._foreach_add_(m, g, alpha=1 - b1)
    torch._foreach_mul_(v, b2)
    torch._foreach_addcmul_(v, g, g, value=1 - b2)
    below = torch._foreach_div(v, c2)
    torch._foreach_sqrt_(below)
    torch._foreach_add_(below, ADAM_EPS)
    torch._foreach_mul_(p, 1 - LR * DECAY)
    torch._foreach_addcdiv_(p, m, below, value=-LR / c1)
    if p is not s["params"]:
        torch._foreach_copy_(s["params"], p)


def _mix(x):
    """A low-bias mixing of 32-bit words (held in int64): two rounds of shift, exclusive or and multiplication."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _mix_int(x):
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _tensor_key(seed, step, i):
    """The word that a tensor's rounding in this step is keyed with."""
    return _mix_int(_mix_int((seed + 0x9E3779B9 * step) & 0xFFFFFFFF) ^ i)


def _stochastic(a, u):
    """Magnitudes a <= 448 on the 8-bit type's grid: down, or up where the fraction of a step and u in [0, 1) reach one."""
    _, e = torch.frexp(a)
    exponent = (e - 1).clamp_min(-6) - 3
    return (torch.floor(torch.ldexp(a, -exponent) + u).ldexp(exponent)).clamp_max(E4M3_MAX)


def _in_blocks(x, k):
    padded = torch.zeros(k * STATE_BLOCK, dtype=x.dtype, device=x.device)
    padded[:x.numel()] = x
    return padded.view(k, STATE_BLOCK)


def _plain_adamw_8bit(i, seed, step, c1, c2, param, master, grad, m_code, m_scale, r_code, r_scale):
    (b1, b2), n, k = BETAS, param.numel(), m_scale.numel()
    g = grad.float()
    m = (_in_blocks(m_code.float(), k) * m_scale[:, None]).view(-1)[:n]
    r = (_in_blocks(r_code.float(), k) * r_scale[:, None]).view(-1)[:n]
    m = b1 * m + (1 - b1) * g
    v = b2 * r.square() + (1 - b2) * g.square()
    p = param.float() if master is None else master
    p = p * (1 - LR * DECAY) - (LR / c1) * m / ((v / c2).sqrt() + ADAM_EPS)
    param.copy_(p)
    if master is not None:
        master.copy_(p)
    word = _mix(torch.arange(n, device=g.device) ^ _tensor_key(seed, step, i))
    for x, code, scale, u in ((m, m_code, m_scale, word & 0xFFFF), (v.sqrt(), r_code, r_scale, word >> 16)):
        y = _in_blocks(x, k)
        top = y.abs().amax(1)
        scale.copy_(torch.where(top < TINY, 0, top / E4M3_MAX))
        q = _stochastic(y.abs() / scale[:, None].clamp_min(TINY / E4M3_MAX), _in_blocks(u.float() / 65536, k))
        if code is r_code:
            q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q)
        code.copy_((q * y.sign()).view(-1)[:n])


# --------------------------------------------------------------------------- work

def work(case):
    """The bytes and operations that one pass cannot do without: inputs once, outputs once."""
    if case["op"] == "norm":
        n, size = case["rows"] * case["width"], BYTES[case["dtype"]]
        streams = 2 if case["residual"] else 1
        moved = n * size * (streams + streams)          # x, residual -> y, sum
        if case["mode"] == "8bit":
            moved += n * (1 - size) + 4 * case["rows"] * (-(-case["width"] // case["group"]) if case["group"] else 1)
        if case["mode"] == "train":
            moved += n * size * (streams + 1)           # dy, dsum -> dx
        return dict(bytes=moved + case["width"] * BYTES[case["weight"]] * (2 if case["mode"] == "train" else 1), flops=n * (14 if case["mode"] == "train" else 5))
    if case["op"] == "ffn":
        rows, d, h = case["rows"], case["width"], case["hidden"]
        train = case["mode"] == "train"
        return dict(bytes=2 * ((4 if train else 2) * rows * d + (6 if train else 3) * d * h), flops=(18 if train else 6) * rows * d * h)
    n = sum(_sizes(case))
    moved = n * BYTES[case["grad"]] + {"f32": 8, "bf16": 4, "bf16+master": 10}[case["param"]] * n
    moved += 16 * n if case["bits"] == 32 else 4 * n + 16 * sum(-(-k // STATE_BLOCK) for k in _sizes(case))
    return dict(bytes=moved, flops=15 * n)


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "ffn": _exact_ffn, "adamw": _exact_adamw}[case["op"]](s)


def _exact_norm(s):
    case, x, w = s["case"], s["x"].double(), s["weight"].double()
    streams = []
    if case["residual"]:
        streams = [(x + s["residual"].double()).to(s["x"].dtype)]  # part of the definition: the sum is stored, and the norm is the stored one's
        x = streams[0].double()
    size = torch.sqrt(torch.linalg.vector_norm(x, dim=1) ** 2 / case["width"] + EPS)
    y = x / size[:, None] * w
    if case["mode"] == "8bit":
        codes, scales = [], []
        for part in y.split(case["group"] or case["width"], 1):
            scales.append(torch.clamp(part.abs().max(1).values, min=TINY) / E4M3_MAX)
            codes.append((part / scales[-1][:, None]).float().to(torch.float8_e4m3fn).double())
        return (torch.cat(codes, 1), torch.stack(scales, 1), *streams)
    if case["mode"] == "forward":
        return (y, *streams) if streams else y
    dy = s["dy"].double()
    along = torch.einsum("rc,rc,c->r", dy, x, w) / (case["width"] * size ** 3)
    dx = dy * w / size[:, None] - x * along[:, None]
    if streams:
        dx += s["dsum"].double()
    return (y, *streams, dx, torch.einsum("rc,rc,r->c", dy, x, 1 / size))


def _exact_ffn(s):
    case = s["case"]
    rows = case["rows"]
    wg, wu, wd = (s[n].double() for n in ("w_gate", "w_up", "w_down"))
    ys, dxs, dwg, dwu, dwd = [], [], 0, 0, 0
    for at in range(0, rows, 16384):
        x = s["x"][at:at + 16384].double()
        g = torch.einsum("rd,hd->rh", x, wg)
        u = torch.einsum("rd,hd->rh", x, wu)
        with torch.enable_grad():
            leaf = g.clone().requires_grad_(True)
            if case["activation"] == "silu":
                act = leaf / (1 + torch.exp(-leaf))
            elif case["activation"] == "gelu":
                act = leaf * torch.special.ndtr(leaf)
            else:
                act = torch.relu(leaf) ** 2
            slope, = torch.autograd.grad(act.sum(), leaf)
        act = act.detach()
        ys.append(torch.einsum("rh,dh->rd", act * u, wd))
        if case["mode"] == "forward":
            continue
        dy = s["dy"][at:at + 16384].double()
        dh = torch.einsum("rd,dh->rh", dy, wd)
        dwd = dwd + torch.einsum("rd,rh->dh", dy, act * u)
        dg, du = dh * u * slope, dh * act
        dxs.append(torch.einsum("rh,hd->rd", dg, wg) + torch.einsum("rh,hd->rd", du, wu))
        dwg = dwg + torch.einsum("rh,rd->hd", dg, x)
        dwu = dwu + torch.einsum("rh,rd->hd", du, x)
    y = torch.cat(ys)
    return y if case["mode"] == "forward" else (y, torch.cat(dxs), dwg, dwu, dwd)


def _exact_adamw(s):
    case, (b1, b2), step = s["case"], BETAS, s["step"] + 1
    flat = s["flat"]
    out = {name: t.double() for name, t in flat.items()}

    def place(name, i, values):
        """Where tensor i of `name` lies in its flat buffer."""
        view = s[name + "s"][i]
        a = view.storage_offset() - flat[name].storage_offset()
        out[name][a:a + view.numel()] = values

    for i, grad in enumerate(s["grads"]):
        g = grad.double()
        n = g.numel()
        if case["bits"] == 32:
            m, v = s["exp_avgs"][i].double(), s["exp_avg_sqs"][i].double()
        else:
            m, v = (s[name + "s"][i].double() * s[name + "_scales"][i].double().repeat_interleave(STATE_BLOCK)[:n] for name in ("exp_avg", "exp_avg_sq"))
            v = v ** 2
        m = m + (1 - b1) * (g - m)
        v = v + (1 - b2) * (g * g - v)
        p = (s["masters"] if "masters" in s else s["params"])[i].double()
        p = p - LR * (DECAY * p + m / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + ADAM_EPS))
        place("param", i, p)
        if "masters" in s:
            place("master", i, p)
        if case["bits"] == 32:
            place("exp_avg", i, m)
            place("exp_avg_sq", i, v)
            continue
        word = _mix(torch.arange(n, device=g.device) ^ _tensor_key(s["seed"], step, i))
        for name, x, u in (("exp_avg", m, word % 65536), ("exp_avg_sq", v.sqrt(), word // 65536)):
            top = torch.stack([b.abs().max() for b in x.split(STATE_BLOCK)]) if n < 100_000 else _in_blocks(x, -(-n // STATE_BLOCK)).abs().amax(1)
            scale = torch.where(top < TINY, torch.zeros_like(top), top / E4M3_MAX)
            a = x.abs() / scale.clamp_min(TINY / E4M3_MAX).repeat_interleave(STATE_BLOCK)[:n]
            step_size = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
            q = torch.clamp(torch.floor(a / step_size + u.double() / 65536) * step_size, max=E4M3_MAX)
            if name == "exp_avg_sq":
                q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
            place(name, i, q * x.sign())
            place(name + "_scale", i, scale)
    return out
