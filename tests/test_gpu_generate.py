"""The hybrid model token by token: windowed attention over ring caches, mixers over their scan states and the choice of
tokens, run together as a server runs them, against the model's forward over whole sequences."""
from __future__ import annotations

import copy

import pytest
import torch

from thetascan_b200 import sample_tokens
from thetascan_b200.config import KernelConfig, RoPEConfig, TemporalConfig, ThetaScanConfig
from thetascan_b200.lm import CausalAttention, HybridLM, gn_mixer_config, main
from thetascan_b200.mixer import ThetaScan
from thetascan_b200.seqpar import ScanStream

gpu = pytest.mark.gpu


def _model(window=None, sinks=0, mixer_layers=(1,), **kw):
    torch.manual_seed(2)
    model = HybridLM(vocab=256, d_model=128, n_layers=3, n_heads=2, mixer_layers=mixer_layers,
                     mixer_config=gn_mixer_config(128, 2), window=window, sinks=sinks, **kw)
    with torch.no_grad():   # every branch as large as the stream that it is added to
        model.embed.weight.normal_(std=0.5)
        for block in model.blocks:
            out = block.mix.out if isinstance(block.mix, CausalAttention) else block.mix._core.proj_out
            out.weight.normal_(std=0.3)
            block.mlp.down.weight.normal_(std=0.1)
    return model


def _off(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm().clamp_min(1e-30))   # nothing against nothing is 0


# An attention layer rounds q, k, v, its weights and its output to bf16, and a mixer of the whole sequence its streams: a
# rounding is 2^-8 / sqrt(12) of a value's step in the mean, under 2^-9 of its norm.  Whole and in pieces they are
# rounded at other places: twice that, of about 8 roundings, in three branches of the size of the stream, in quadrature:
# 2 sqrt(24) 2^-9 = 0.02.
NEAR = 0.02


@gpu
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("window,sinks,pieces", [
    (16, 3, [70]), (16, 3, [1] * 40), (16, 0, [33, 1, 1, 20, 15]), (1, 2, [3, 1, 9]), (64, 1, [20, 1, 70, 1, 2]), (300, 4, [150, 1])])
def test_pieces_equal_the_whole(window, sinks, pieces, fused):
    model = _model(window, sinks, gated="silu" if fused else None, fused_norms=fused).cuda()
    tokens = torch.randint(0, 256, (3, sum(pieces)), generator=torch.Generator().manual_seed(4)).cuda()
    with torch.no_grad():
        want = model(tokens)
        alone = model(tokens[:, -1:])[:, -1]
    stream, at = model.stream(3), 0
    for n in pieces:
        got = model.extend(tokens[:, at:at + n], stream)
        at += n
        assert _off(got, want[:, at - 1]) < NEAR, at
    assert stream.lengths.tolist() == [at] * 3
    assert _off(alone, want[:, -1]) > 10 * NEAR   # what came before matters


@gpu
def test_wide_window_is_causal_attention():
    ours, plain = _model(500, 2).cuda(), _model().cuda()
    tokens = torch.randint(0, 256, (2, 200), generator=torch.Generator().manual_seed(5)).cuda()
    a, b = ours.loss(tokens), plain.loss(tokens)
    with torch.no_grad():
        assert _off(ours(tokens), plain(tokens)) < NEAR
    a.backward(), b.backward()
    for (name, p), q in zip(ours.named_parameters(), plain.parameters()):
        # the gradients' own roundings (P, dS, dq, dk, dv and y again) beside the forward's
        assert _off(p.grad, q.grad) < 3 * NEAR, name


@gpu
def test_generation_is_the_stepwise_choice():
    model = _model(24, 2, gated="silu", fused_norms=True).cuda()
    tokens = torch.randint(0, 256, (4, 50), generator=torch.Generator().manual_seed(6)).cuda()
    settings = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    got = model.generate(tokens, 30, generator=torch.Generator("cuda").manual_seed(7), **settings)
    again = model.generate(tokens, 30, generator=torch.Generator("cuda").manual_seed(7), **settings)
    assert got.shape == (4, 30) and got.dtype == torch.int64 and torch.equal(got, again)
    uniform = torch.rand(30, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    stream, new = model.stream(4), tokens
    for i in range(30):
        new = sample_tokens(model.extend(new, stream), uniform[i], **settings)[:, None]
        assert torch.equal(new[:, 0], got[:, i])
    # a stream goes on where it was; temperature 0 takes the largest logit
    stream = model.stream(4)
    first = model.generate(tokens, 5, temperature=0, stream=stream)
    rest = model.generate(first[:, -1:], 6, temperature=0, stream=stream)
    assert torch.equal(torch.cat((first, rest), 1), model.generate(tokens, 11, temperature=0))
    assert torch.equal(first[:, 0], model.extend(tokens, model.stream(4)).float().argmax(-1))


@gpu
def test_generation_under_autocast_and_8bit_head():
    model = _model(24, 2, gated="silu", fused_norms=True).cuda()
    tokens = torch.randint(0, 256, (2, 40), generator=torch.Generator().manual_seed(8)).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with torch.no_grad():
            want = model(tokens)[:, -1]
        assert _off(model.extend(tokens, model.stream(2)), want) < 2 * NEAR   # the projections in bf16 too
        model.quantize_head()
        assert model.generate(tokens, 4).shape == (2, 4)


def _config(kind):
    common = dict(d_model=128, n_heads=2, rope=RoPEConfig(mode="partial", fraction=0.5))
    if kind == "gn":
        return gn_mixer_config(128, 2)
    if kind == "sum":
        return ThetaScanConfig(memory_multiplier=4, family="kernel", kernel=KernelConfig(feature_map="relu2_ridge"),
                               temporal=TemporalConfig(mode="sum"), **common)
    bank = TemporalConfig(mode="bank", bank_mode=kind, recency_branches=2, retention_inits=(0.9, 0.99))
    return ThetaScanConfig(memory_multiplier=2, family="kernel",
                           kernel=KernelConfig(feature_map="projected_bspline", bspline_basis_count=16), temporal=bank, **common)


@gpu
@pytest.mark.parametrize("kind", ["gn", "sum", "fast", "stale"])
def test_mixer_in_pieces(kind):
    torch.manual_seed(3)
    mixer = ThetaScan(_config(kind)).cuda()
    with torch.no_grad():
        mixer._core.proj_out.weight.normal_(std=0.1)
        mixer._core.W2[0].normal_(0.0, 0.2)
        if mixer._core.fade_eta is not None:
            mixer._core.fade_eta.normal_(0.0, 0.5)
    x = torch.randn(2, 150, 128, generator=torch.Generator().manual_seed(9)).cuda()
    with torch.no_grad():
        want = mixer(x)
        stream, got, at = ScanStream(), [], 0
        for n in (70, 1, 1, 48, 30):
            got.append(mixer(x[:, at:at + n], stream))
            at += n
        assert stream.position == at == 150
    # float32 against float32 (a division by a mass may magnify the sums' 2^-24); the whole GN mixer has bf16 streams
    assert _off(torch.cat(got, 1), want) < (NEAR if kind == "gn" else 2e-4)


@gpu
def test_stream_refusals():
    model = _model(8, 1).cuda()
    stream = model.stream(2)
    tokens = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        model.extend(tokens[:1], stream)
    with pytest.raises(ValueError):
        model.extend(tokens[:, :0], stream)
    with pytest.raises(ValueError):
        copy.deepcopy(model).extend(tokens, stream)
    with pytest.raises(ValueError):
        model.generate(tokens, 0)
    model.extend(tokens, stream)
    mixer, scan = model.blocks[1].mix, stream.layers[1]
    x = torch.zeros(2, 1, 128, device="cuda")
    with pytest.raises(RuntimeError):   # with gradients
        mixer(x, scan)
    with torch.no_grad(), pytest.raises(ValueError):
        mixer(x[:1], scan)
    with torch.no_grad(), pytest.raises(ValueError):
        mixer(x[:, :0], scan)
    model.extend(tokens, stream)        # a refusal leaves the stream as it was
    assert stream.lengths.tolist() == [6, 6] and scan.position == 6
    other = ThetaScan(_config("stale")).cuda()
    with torch.no_grad(), pytest.raises(Exception):
        other(x, scan)
    with torch.no_grad(), pytest.raises(RuntimeError):   # its states are not whole any more
        mixer(x, scan)


@gpu
def test_command_generates(monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["lm", "--steps", "1", "--batch", "2", "--tokens", "64", "--window", "16", "--sinks", "2", "--generate", "3"])
    main()
    assert "6 tokens behind (2, 65)" in capsys.readouterr().out


def test_refusals_on_the_host(monkeypatch):
    with pytest.raises(ValueError):
        CausalAttention(64, 2, None, 3)
    with pytest.raises(TypeError):
        _model().stream(1)
    with pytest.raises(ValueError):
        _model(4).stream(0)
    monkeypatch.setattr("sys.argv", ["lm", "--generate", "3"])
    with pytest.raises(SystemExit):
        main()


def test_scan_stream_in_pieces_on_the_host():
    """The algebra of longer pieces, with the definition of the scan in 64 bits."""
    from thetascan_b200 import seqpar
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 3, 40, n, generator=g, dtype=torch.float64) for n in (6, 6, 4))
    la = -torch.rand(3, generator=g, dtype=torch.float64) * 0.3
    ahead = torch.arange(40, dtype=torch.float64)
    gap = (ahead[:, None] - ahead[None]).clamp_min(0)

    def scan(q, k, v, retentions, *, append_unit=False, stale=None):
        vv = torch.cat((v, v.new_ones(*v.shape[:3], 1)), -1) if append_unit else v
        n = q.shape[2]
        outs = []
        for i, r in enumerate(retentions):
            w = torch.ones(1, n, n, dtype=torch.float64) if r is None else torch.exp(r[:, None, None] * gap[:n, :n])
            w = 1 - w if stale and stale[i] else w
            outs.append((q @ k.transpose(-1, -2) * w.tril()) @ vv)
        return outs

    retentions, stale = (None, la, la), (False, False, True)
    want = scan(q, k, v, retentions, append_unit=True, stale=stale)
    stream, got, at = ScanStream(), [[], [], []], 0
    for n in (13, 2, 25):
        s = slice(at, at + n)
        with stream.piece(q[:, 0, s]):
            for out, r in zip(got, seqpar.sharded_reads(stream, scan, q[:, :, s], k[:, :, s], v[:, :, s], retentions, append_unit=True, stale=stale)):
                out.append(r)
        at += n
    for a, b in zip(got, want):
        # the states and the results are kept in 32 bits: sums of up to 40 x 6 products
        assert float((torch.cat(a, 2) - b).abs().max()) < 240 * 2.0 ** -23 * float(b.abs().max())
