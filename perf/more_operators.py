"""Operators of training and generation around the mixer, as they are timed and checked: causal attention over a sliding
window with first tokens that stay visible (training, prompts, single tokens over a ring cache), the token step of the
decayed multi-view scan, and the choice of a token from logits (temperature, top-k, top-p, min-p).

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges, ``prepare`` makes what a program holds
before the call, ``run`` is one call: with ``own`` the framework's operator, without it the same operator in elementary
torch operations in 32 bits (64 for a choice's cumulative sums).  ``exact`` evaluates the definition in 64 bits.

Attention: the query at position i sees the keys at j <= i with i - j < window or j < sinks, j and i below the
sequence's length; a row that sees nothing is zero.  The ring cache holds position j in slot j below ``sinks`` and in
slot sinks + (j - sinks) mod window above.

Scan step: S <- exp(log_alpha) S + k^T [v | 1], read q S, for each view.

Choice: tokens in the order of falling logits (lower index first among equals); the first top_k of them; of these the
shortest prefix that holds top_p of their mass; of these the ones with at least min_p times the largest probability;
the first token, by index, at which the cumulative mass of what is left exceeds ``uniform`` times its total.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
QUERY_BLOCK = 128       # queries that share a span of keys in the plain form


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # the hybrid language model's training batch (64 x 1024 tokens, 8 heads of 64) with windowed attention blocks
        dict(name="attn_train_lm", op="attention", mode="train", batch=64, tokens=1024, past=0, heads=8, kv_heads=8, dim=64, window=256, sinks=4, ragged=False),
        # one long document, shared key heads
        dict(name="attn_train_long", op="attention", mode="train", batch=1, tokens=16384, past=0, heads=16, kv_heads=4, dim=128, window=2048, sinks=16, ragged=False),
        # fine-tuning on a padded batch of texts of uneven length, a head width that is no power of two, no sinks
        dict(name="attn_train_ragged", op="attention", mode="train", batch=6, tokens=1999, past=0, heads=10, kv_heads=5, dim=80, window=500, sinks=0, ragged=True),
        # prompts of uneven length, their last window kept in the cache
        dict(name="attn_prompt", op="attention", mode="prompt", batch=5, tokens=4001, past=0, heads=16, kv_heads=8, dim=128, window=1024, sinks=4, ragged=True),
        # the next piece of a long prompt over the keys before it
        dict(name="attn_piece", op="attention", mode="piece", batch=2, tokens=1000, past=7001, heads=8, kv_heads=8, dim=64, window=1500, sinks=128, ragged=False),
        # one token of one sequence in the hybrid language model: latency
        dict(name="attn_token", op="attention", mode="token", batch=1, heads=8, kv_heads=8, dim=64, window=256, sinks=4),
        # one token of each of many sequences, wide cache
        dict(name="attn_tokens", op="attention", mode="token", batch=64, heads=32, kv_heads=8, dim=128, window=4096, sinks=64),
        # one token through a mixer of the hybrid language model (8 heads, 256 features, the sum and one recency view)
        dict(name="scan_token", op="scan", batch=1, heads=8, dk=256, dv=64, views=2, unit=True, gated=False, dtype="bf16"),
        # one token of each of many sequences, float32 streams
        dict(name="scan_tokens", op="scan", batch=192, heads=16, dk=256, dv=64, views=2, unit=True, gated=False, dtype="f32"),
        # the hybrid language model's vocabulary, a few sequences: latency
        dict(name="sample_lm", op="sample", rows=4, vocab=1024, dtype="f32", spread=2.0, temperature=0.8, top_k=50, top_p=None, min_p=None, per_row=False, logprobs=False),
        # a serving batch on a large vocabulary, every filter, settings of each request's own (some greedy)
        dict(name="sample_serving", op="sample", rows=64, vocab=128_257, dtype="bf16", spread=2.5, temperature=0.9, top_k=1000, top_p=0.95, min_p=0.02, per_row=True, logprobs=False),
        # rollouts of a training run: top-p alone, with the log-probabilities
        dict(name="sample_rollout", op="sample", rows=512, vocab=50_257, dtype="f32", spread=2.5, temperature=1.0, top_k=None, top_p=0.9, min_p=None, per_row=False, logprobs=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1e15)


def draw(rng):
    while True:
        case = _draw(rng)
        if _cost(case) <= 9e-4:
            return case


def _draw(rng):
    op = rng.choice(["attention", "attention", "scan", "sample"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 5, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        dim = rng.choice([64, 128, 64, 128, 8 * rng.randint(2, 16)])
        sinks = rng.choice([0, 1, 4, rng.randint(2, 200)])
        mode = rng.choice(["train", "train", "prompt", "piece", "token", "token"])
        if mode == "token":
            return dict(op=op, mode=mode, batch=_log(rng, 1, 128), heads=heads, kv_heads=kv_heads, dim=dim, window=_log(rng, 16, 8192), sinks=sinks)
        tokens = _log(rng, 1 if mode == "piece" else 100, 16384)
        return dict(op=op, mode=mode, batch=_log(rng, 1, max(1, min(64, 65536 // tokens))), tokens=tokens, past=_log(rng, 1, 16000) if mode == "piece" else 0,
                    heads=heads, kv_heads=kv_heads, dim=dim, window=_log(rng, 16, 4096), sinks=sinks, ragged=rng.random() < 0.4)
    if op == "scan":
        return dict(op=op, batch=_log(rng, 1, 256), heads=rng.choice([1, 3, 4, 8, 16]), dk=rng.choice([64, 128, 256, rng.randint(8, 256)]), dv=rng.choice([64, 128, rng.randint(8, 200)]),
                    views=rng.randint(1, 4), unit=rng.random() < 0.6, gated=rng.random() < 0.3, dtype=rng.choice(["bf16", "f32"]))
    return dict(op=op, rows=_log(rng, 1, 512), vocab=_log(rng, 100, 200_000), dtype=rng.choice(["bf16", "f32"]), spread=rng.uniform(1.5, 3.5), temperature=round(rng.uniform(0.4, 1.4), 3),
                top_k=rng.choice([None, _log(rng, 1, 2000)]), top_p=rng.choice([None, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([None, round(rng.uniform(0.005, 0.2), 4)]),
                per_row=rng.random() < 0.4, logprobs=rng.random() < 0.5)


def _lengths(case):
    """Tokens of each sequence of a padded batch (the longest fills it)."""
    total = case["tokens"] + case["past"]
    if not case["ragged"]:
        return [total] * case["batch"]
    rng = random.Random(total * 131 + case["batch"])
    return [total] + [rng.randint(1, total) for _ in range(case["batch"] - 1)]


def _filled(case):
    """Tokens that each sequence of a decoding batch has had: one just begun, most beyond their window."""
    rng = random.Random(case["window"] * 131 + case["batch"])
    most = 2 * (case["window"] + case["sinks"])
    got = [rng.randint(case["window"] // 2, most) for _ in range(case["batch"])]
    if case["batch"] > 1:
        got[1] = 0
    return got


# --------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "attention":
        b, h, g, d, t = case["batch"], case["heads"], case["kv_heads"], case["dim"], torch.bfloat16
        if case["mode"] == "token":
            # the new token's q, k, v are parts of one projection
            q, k, v = normal(b, 1, h + 2 * g, d, dtype=t).transpose(1, 2).split((h, g, g), 1)
            slots = case["sinks"] + case["window"]
            lengths = torch.tensor(_filled(case), dtype=torch.int32, device="cuda")
            empty = torch.arange(slots, device="cuda") >= lengths[:, None]
            keys, values = (normal(b, g, slots, d, dtype=t).masked_fill_(empty[:, None, :, None], 0) for _ in range(2))
            return dict(case=case, q=q * 1.5, k=k, v=v, keys=keys, values=values, lengths=lengths)
        n, past = case["tokens"], case["past"]
        q = (normal(b, n, h, d, dtype=t) * 1.5).transpose(1, 2)
        k, v = (normal(b, n + past, g, d, dtype=t).transpose(1, 2) for _ in range(2))
        state = dict(case=case, q=q, k=k, v=v, lengths=torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None)
        if case["mode"] == "train":
            state["dy"] = normal(b, n, h, d, dtype=t).transpose(1, 2)
        if case["mode"] == "prompt":
            slots = case["sinks"] + case["window"]
            state["keys"], state["values"] = (torch.zeros(b, g, slots, d, dtype=t, device="cuda") for _ in range(2))
            state["filled"] = torch.zeros(b, dtype=torch.int32, device="cuda")
        return state
    if case["op"] == "scan":
        b, h, t = case["batch"], case["heads"], DTYPES[case["dtype"]]
        width = case["dv"] + int(case["unit"])
        # positive features that sum to one, as the mixers' maps give them
        q, k = (torch.softmax(2 * normal(b, h, 1, case["dk"]), -1).to(t) for _ in range(2))
        retentions = [None]
        for _ in range(case["views"] - 1):
            retentions.append(torch.log(0.5 + 0.499 * uniform(*((b, h, 1, 1) if case["gated"] else (h,)))))
        state = normal(b, h, case["views"], case["dk"], width, scale=0.1)
        if case["unit"]:
            state[..., -1] = 0.2 + uniform(b, h, case["views"], case["dk"])
        return dict(case=case, q=q, k=k, v=normal(b, h, 1, case["dv"], dtype=t), retentions=retentions, state=state)
    rows, vocab = case["rows"], case["vocab"]
    logits = normal(rows, vocab, scale=case["spread"]).to(DTYPES[case["dtype"]])
    banned = torch.randint(0, vocab, (vocab // 100,), generator=gen, device="cuda")
    logits[:, banned] = -math.inf
    settings = {name: case[name] for name in ("temperature", "top_k", "top_p", "min_p")}
    if case["per_row"]:
        greedy = uniform(rows) < 0.1
        settings["temperature"] = (case["temperature"] * (0.7 + 0.6 * uniform(rows))).masked_fill_(greedy, 0)
        if case["top_k"] is not None:
            settings["top_k"] = (case["top_k"] * uniform(rows)).to(torch.int32) + 1
        if case["top_p"] is not None:
            settings["top_p"] = case["top_p"] * (0.8 + 0.2 * uniform(rows))
        if case["min_p"] is not None:
            settings["min_p"] = case["min_p"] * uniform(rows)
    return dict(case=case, logits=logits, uniform=uniform(rows), settings=settings)


# --------------------------------------------------------------------------- one pass

def run(state):
    return {"attention": _run_attention, "scan": _run_scan, "sample": _run_sample}[state["case"]["op"]](state)


def _run_attention(s):
    return _own_attention(s) if own else _plain_attention(s)


def _run_scan(s):
    """The state changes in place; the next pass is the next token."""
    return (*(_own_scan if own else _plain_scan)(s), s["state"])


def _run_sample(s):
    return _own_sample(s) if own else _plain_sample(s)


def _own_attention(s):
    from thetascan_b200 import window_attention, window_attention_step, window_cache_extend
    case, window, sinks = s["case"], s["case"]["window"], s["case"]["sinks"]
    if case["mode"] == "train":
        leaves = [s[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
        y = window_attention(*leaves, window, sinks, lengths=s["lengths"])
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    with torch.no_grad():
        if case["mode"] == "token":
            y = window_attention_step(s["q"], s["k"], s["v"], s["keys"], s["values"], s["lengths"], sinks)
            return y, s["keys"], s["values"]
        y = window_attention(s["q"], s["k"], s["v"], window, sinks, lengths=s["lengths"])
        if case["mode"] == "piece":
            return y
        window_cache_extend(s["k"], s["v"], s["keys"], s["values"], s["filled"], sinks, new=s["lengths"])
        return y, s["keys"], s["values"]


def _plain_window(q, k, v, window, sinks, lengths):
    """The attention in blocks of queries, each against the span of keys that its window reaches and the first keys."""
    b, h, n, d = q.shape
    g, total = k.shape[1], k.shape[2]
    past, window, sinks, blocks = total - n, min(window, total), min(sinks, total), -(-n // QUERY_BLOCK)
    behind = blocks * QUERY_BLOCK - n
    pad = torch.nn.functional.pad
    qb = pad(q.float(), (0, 0, 0, behind)).view(b, g, h // g, blocks, QUERY_BLOCK, d)
    kf, vf = k.float(), v.float()
    span = window - 1 + QUERY_BLOCK
    kb, vb = (pad(t, (0, 0, window - 1, behind))[:, :, past:].unfold(2, span, QUERY_BLOCK).transpose(-1, -2) for t in (kf, vf))
    at = past + torch.arange(blocks * QUERY_BLOCK, device=q.device).view(blocks, QUERY_BLOCK, 1)
    near = at[:, :1] - window + 1 + torch.arange(span, device=q.device)
    first = torch.arange(sinks, device=q.device)
    length = torch.full((b,), total, device=q.device) if lengths is None else lengths
    length = length.view(b, 1, 1, 1, 1, 1)
    seen = torch.cat([((near <= at) & (at - near < window) & (near >= sinks)).expand(b, 1, 1, -1, -1, -1) & (near < length),
                      (first <= at).expand(b, 1, 1, -1, -1, -1) & (first < length)], -1) & (at < length)
    scores = torch.cat([qb @ kb[:, :, None].transpose(-1, -2), qb @ kf[:, :, None, None, :sinks].transpose(-1, -2)], -1) * (1 / math.sqrt(d))
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.detach().amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - top)
    total_p = p.sum(-1, keepdim=True)
    y = (p[..., :span] @ vb[:, :, None] + p[..., span:] @ vf[:, :, None, None, :sinks]) / total_p.masked_fill(total_p == 0, 1)
    return y.reshape(b, h, blocks * QUERY_BLOCK, d)[:, :, :n].to(q.dtype)


def _plain_extend(k, v, keys, values, filled, sinks, new):
    b, slots, n = keys.shape[0], keys.shape[2], k.shape[2]
    window = slots - sinks
    count = torch.full_like(filled, n) if new is None else new
    after = filled + count
    # each slot's newest position, where it is one of the new tokens
    slot = torch.arange(slots, device=k.device)
    last = after[:, None] - 1
    newest = torch.where(slot < sinks, slot, slot + torch.div(last - slot, window, rounding_mode="floor") * window)
    source = newest - filled[:, None]
    fresh = ((newest <= last) & (source >= 0) & (newest >= slot))[:, None, :, None]
    index = source.clamp(0, n - 1)[:, None, :, None].expand(b, k.shape[1], slots, k.shape[3])
    keys.copy_(torch.where(fresh, k.gather(2, index), keys))
    values.copy_(torch.where(fresh, v.gather(2, index), values))


def _plain_attention(s):
    case, window, sinks = s["case"], s["case"]["window"], s["case"]["sinks"]
    if case["mode"] == "train":
        leaves = [s[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
        y = _plain_window(*leaves, window, sinks, s["lengths"])
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if case["mode"] == "token":
        q, keys, values, lengths = s["q"], s["keys"], s["values"], s["lengths"]
        b, h, _, d = q.shape
        row = torch.arange(b, device=q.device)
        slot = torch.where(lengths < sinks, lengths, sinks + (lengths - sinks) % window).long()
        keys[row, :, slot], values[row, :, slot] = s["k"][:, :, 0], s["v"][:, :, 0]
        seen = (torch.arange(keys.shape[2], device=q.device) <= lengths[:, None])[:, None, None]
        scores = q.float().reshape(b, keys.shape[1], -1, d) @ keys.float().transpose(-1, -2) * (1 / math.sqrt(d))
        scores = scores.masked_fill(~seen, -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        y = p @ values.float() / p.sum(-1, keepdim=True)
        return y.reshape(b, h, 1, d).to(q.dtype), keys, values
    with torch.no_grad():
        y = _plain_window(s["q"], s["k"], s["v"], window, sinks, s["lengths"])
    if case["mode"] == "piece":
        return y
    _plain_extend(s["k"], s["v"], s["keys"], s["values"], s["filled"], sinks, s["lengths"])
    return y, s["keys"], s["values"]


def _own_scan(s):
    from thetascan_b200.scan import linattn_views_step
    return linattn_views_step(s["q"], s["k"], s["v"], s["retentions"], s["state"], append_unit=s["case"]["unit"])


def _plain_scan(s):
    q, k, v, state = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    if s["case"]["unit"]:
        v = torch.cat([v, torch.ones_like(v[..., :1])], -1)
    one = torch.zeros(1, 1, 1, 1, device=q.device)
    keep = torch.cat([(one if r is None else r.reshape(-1, q.shape[1], 1, 1)).expand(*q.shape[:2], 1, 1) for r in s["retentions"]], 2).exp()
    state.mul_(keep[..., None])
    state.add_((k.transpose(-1, -2) * v)[:, :, None])
    reads = (q.transpose(-1, -2)[:, :, None] * state).sum(-2)
    return tuple(reads[:, :, i:i + 1].to(s["q"].dtype) for i in range(reads.shape[2]))


def _own_sample(s):
    from thetascan_b200 import sample_tokens
    return sample_tokens(s["logits"], s["uniform"], return_logprobs=s["case"]["logprobs"], **s["settings"])


def _column(value, like):
    """A setting as a column in 64 bits, a row of it for each row of logits."""
    return (value.double() if torch.is_tensor(value) else torch.full((like.shape[0],), value, dtype=torch.float64, device=like.device))[:, None]


def _plain_sample(s):
    logits, settings = s["logits"], s["settings"]
    rows, vocab = logits.shape
    temperature = _column(settings["temperature"], logits)
    greedy = temperature <= 0
    values, order = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    scaled = (values.double() - values[:, :1]) / torch.where(greedy, 1, temperature)
    weight = torch.exp(scaled)
    kept = torch.isfinite(values)
    rank = torch.arange(vocab, device=logits.device)
    if settings["top_k"] is not None:
        kept = kept & (rank < _column(settings["top_k"], logits))
    mass = weight * kept
    if settings["top_p"] is not None:
        sums = mass.cumsum(-1)
        kept = kept & (sums - mass < _column(settings["top_p"], logits) * sums[:, -1:])
    if settings["min_p"] is not None:
        kept = kept & (scaled >= _column(settings["min_p"], logits).log())
    kept = kept & (~greedy | (rank < 1))
    by_index = torch.zeros_like(weight).scatter_(1, order, weight * kept)
    sums = by_index.cumsum(-1)
    token = (sums > s["uniform"].double()[:, None] * sums[:, -1:]).to(torch.uint8).argmax(-1)
    if not s["case"]["logprobs"]:
        return token
    place = (order == token[:, None]).to(torch.uint8).argmax(-1, keepdim=True)
    return token, (scaled.gather(1, place) - weight.sum(-1, keepdim=True).log())[:, 0].float()


# --------------------------------------------------------------------------- work

def _pairs(case):
    """Query-key pairs of one head that are visible, over the batch."""
    window, sinks = case["window"], case["sinks"]
    count = 0
    for length in _lengths(case):
        at = torch.arange(case["past"], max(case["past"], length), dtype=torch.int64)
        # positions up to i, less those that are neither near nor first
        count += int((at + 1 - (at + 1 - window - sinks).clamp_min(0)).sum())
    return count


def work(case):
    """The bytes and operations that one pass cannot do without: inputs once, outputs once."""
    if case["op"] == "attention":
        b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        if case["mode"] == "token":
            seen = sum(min(n + 1, case["window"] + case["sinks"]) for n in _filled(case))
            return dict(bytes=2 * d * (2 * seen * g + 2 * b * h + 2 * b * g), flops=4 * d * h * seen)
        q, kv, train = b * case["tokens"] * h * d, b * (case["tokens"] + case["past"]) * g * d, case["mode"] == "train"
        if case["mode"] == "piece":     # keys that some query sees
            n, total = case["tokens"], case["tokens"] + case["past"]
            kv = b * g * d * (total - max(0, case["past"] - case["window"] + 1 - case["sinks"]))
        moved = 2 * ((4 if train else 2) * q + (4 if train else 2) * kv)
        if case["mode"] == "prompt":
            moved += 4 * d * g * sum(min(n, case["window"] + case["sinks"]) for n in _lengths(case))
        return dict(bytes=moved, flops=(14 if train else 4) * d * h * _pairs(case))
    if case["op"] == "scan":
        size, width = BYTES[case["dtype"]], case["dv"] + int(case["unit"])
        heads = case["batch"] * case["heads"]
        state = heads * case["views"] * case["dk"] * width
        return dict(bytes=8 * state + size * heads * (2 * case["dk"] + case["dv"] + case["views"] * width), flops=5 * state)
    n = case["rows"] * case["vocab"]
    return dict(bytes=n * BYTES[case["dtype"]] + case["rows"] * (16 if case["logprobs"] else 12), flops=8 * n)


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "scan": _exact_scan, "sample": _exact_sample}[case["op"]](s)


def _exact_attention(s):
    case = s["case"]
    if case["mode"] == "token":
        return _exact_token(s)
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    (b, h, n, d), (g, total) = q.shape, k.shape[1:3]
    past, share, window, sinks = total - n, h // g, case["window"], case["sinks"]
    lengths = [total] * b if s["lengths"] is None else s["lengths"].tolist()
    y = torch.zeros_like(q)
    if case["mode"] == "train":
        dy, dq, dk, dv = s["dy"].double(), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i, length in enumerate(lengths):
        for low in range(past, length, 1024):
            high = min(low + 1024, length)
            at = torch.arange(low, high, device=q.device)[:, None]
            keys = torch.arange(high, device=q.device)
            keys = keys[(keys < sinks) | (keys > low - window)]
            hidden = (keys > at) | ((at - keys >= window) & (keys >= sinks))
            rows = slice(low - past, high - past)
            for head in range(g):
                heads = slice(head * share, (head + 1) * share)
                kk, vv, qq = k[i, head, keys], v[i, head, keys], q[i, heads, rows]
                logits = torch.einsum("hqd,kd->hqk", qq, kk) / d ** 0.5
                logits.masked_fill_(hidden, -math.inf)
                p = torch.softmax(logits, -1)
                out = torch.einsum("hqk,kd->hqd", p, vv)
                y[i, heads, rows] = out
                if case["mode"] == "train":
                    go = dy[i, heads, rows]
                    dv[i, head].index_add_(0, keys, torch.einsum("hqk,hqd->kd", p, go))
                    ds = p * (torch.einsum("hqd,kd->hqk", go, vv) - (go * out).sum(-1, keepdim=True)) / d ** 0.5
                    dq[i, heads, rows] = torch.einsum("hqk,kd->hqd", ds, kk)
                    dk[i, head].index_add_(0, keys, torch.einsum("hqk,hqd->kd", ds, qq))
    if case["mode"] == "train":
        return y, dq, dk, dv
    if case["mode"] == "piece":
        return y
    keys, values = s["keys"].double(), s["values"].double()
    for i, length in enumerate(lengths):
        for buffer, new in ((keys, s["k"]), (values, s["v"])):
            buffer[i, :, :min(sinks, length)] = new[i, :, :min(sinks, length)].double()
            kept = torch.arange(max(sinks, length - window), max(sinks, length), device=q.device)
            buffer[i, :, sinks + (kept - sinks) % window] = new[i, :, kept].double()
    return y, keys, values


def _exact_token(s):
    case, window, sinks = s["case"], s["case"]["window"], s["case"]["sinks"]
    share = case["heads"] // case["kv_heads"]
    y, keys, values, lengths = s["q"].double(), s["keys"].clone(), s["values"].clone(), s["lengths"].tolist()
    for i, n in enumerate(lengths):
        slot = n if n < sinks else sinks + (n - sinks) % window
        keys[i, :, slot], values[i, :, slot] = s["k"][i, :, 0], s["v"][i, :, 0]
        seen = min(n + 1, sinks + window)
        for head in range(case["kv_heads"]):
            heads = slice(head * share, (head + 1) * share)
            logits = torch.einsum("hd,kd->hk", s["q"][i, heads, 0].double(), keys[i, head, :seen].double()) / case["dim"] ** 0.5
            y[i, heads, 0] = torch.einsum("hk,kd->hd", torch.softmax(logits, -1), values[i, head, :seen].double())
    return y, keys.double(), values.double()


def _exact_scan(s):
    q, k, v, state = (s[n].double() for n in ("q", "k", "v", "state"))
    if s["case"]["unit"]:
        v = torch.nn.functional.pad(v, (0, 1), value=1.0)
    reads = []
    for i, r in enumerate(s["retentions"]):
        if r is not None:
            state[:, :, i] *= torch.exp(r.double().reshape(-1, q.shape[1], 1, 1))
        state[:, :, i] += torch.einsum("bhti,bhtj->bhij", k, v)
        reads.append(torch.einsum("bhti,bhij->bhtj", q, state[:, :, i]))
    return (*reads, state)


def _exact_sample(s):
    tokens, logprobs = [], []
    settings = {name: value.double().tolist() if torch.is_tensor(value) else [value] * s["case"]["rows"] for name, value in s["settings"].items()}
    for i, u in enumerate(s["uniform"].double().tolist()):
        t, top_k, top_p, min_p = (settings[name][i] for name in ("temperature", "top_k", "top_p", "min_p"))
        x = s["logits"][i].double()
        z = x / (t if t > 0 else 1)
        odds = torch.exp(z - z.max())
        order = torch.argsort(x, descending=True, stable=True)
        count = 1 if t <= 0 else len(order) if top_k is None else int(top_k)
        order = order[:count]
        if top_p is not None:
            before = torch.cumsum(odds[order], 0) - odds[order]
            order = order[before < top_p * odds[order].sum()]
        if min_p is not None:
            order = order[z[order] - z.max() >= math.log(min_p)]
        order = order[odds[order] > 0].sort().values
        sums = torch.cumsum(odds[order], 0)
        token = order[torch.searchsorted(sums, u * sums[-1], right=True).clamp_max(len(order) - 1)]
        tokens.append(token)
        logprobs.append(torch.log_softmax(z, 0)[token])
    tokens = torch.stack(tokens)
    return (tokens, torch.stack(logprobs)) if s["case"]["logprobs"] else tokens
