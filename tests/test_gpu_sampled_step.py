"""Sampling many continuations of one prompt, its operators together: prefill and steps whose products run in 8-bit integers,
attention over shared pages, tokens drawn from the cut distribution; eager, captured and through the model.

Where the 8-bit codes of a second product's rows are rounded from fp32 results of a first, a result near the middle between two
codes may round either way: those elements are counted, and what a code less or more of each would change is allowed."""
import math

import pytest
import torch

import oracle
from gpu_util import announce, device
from oracle import int8, sampling
from q35hip import layers, ops
from q35hip import model as gm
from q35hip import workloads
from q35hip.workloads import Q35Config, quantize_rows_int8

pytestmark = pytest.mark.gpu
H24 = 2.0 ** -24


def mlp_params(H, I, seed=0):
    g = torch.Generator().manual_seed(seed)
    p = {}
    for name, (o, i) in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
        p[name + ".q"], p[name + ".s"] = quantize_rows_int8(torch.randn(o, i, generator=g) * i ** -0.5)
        p[name] = p[name + ".q"].float() * p[name + ".s"][:, None]
    return {k: v.to(device()) for k, v in p.items()}


@pytest.mark.parametrize("M,H,I", [(9, 64, 64), (40, 256, 384), (130, 128, 1000 // 64 * 64)])
@pytest.mark.parametrize("normed", [False, True])
def test_mlp(M, H, I, normed):
    """x + MLP against 64 bits. An activation is within 16 * 2^-24 of itself, relative (two products of three roundings and the
    sigmoid's), and 32 (1 + |gate|) covers the gate's error in it; a code flips where the quotient is that near to a half."""
    announce(f"mlp act_int8 M{M} H{H} I{I} normed {normed}")
    p = mlp_params(H, I)
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, H, generator=g) * 2
    w = torch.randn(H, generator=g) * 0.2
    xd = x.to(device())
    res = xd.clone()
    cap = torch.zeros(M, 1, I, device=device())
    if normed:
        out = gm.mlp(p, res, res, prenorm=(None, w.to(device()), 1e-6), act_int8=True, capture=cap)
        h = int8.norm_rows(x, w)
    else:
        out = gm.mlp(p, ops.quantize_rows(xd), res, capture=cap)
        h = x
    assert out is res
    c = {k: v.cpu() for k, v in p.items()}
    q, s = int8.quantize_rows(h)
    gate, up = int8.product(q, s, c["gate_proj.q"], c["gate_proj.s"]), int8.product(q, s, c["up_proj.q"], c["up_proj.s"])
    act = gate * torch.sigmoid(gate) * up
    near = 32 * H24 * (1 + gate.abs()) * act.abs()
    assert bool(((cap[:, 0].double().cpu() - act).abs() <= near).all())
    q2, s2 = int8.quantize_rows(act)
    t = act / s2.double()[:, None]
    flips = ((t - t.floor() - 0.5).abs() <= near / s2.double()[:, None] + 127 * 33 * H24).double()
    want = x.double() + int8.product(q2, s2, c["down_proj.q"], c["down_proj.s"])
    wd = c["down_proj.q"].double().abs() * c["down_proj.s"].double()[:, None]
    # the row's scale follows its largest activation: its relative error is that of one
    scale = (near / act.abs().clamp_min(1e-300)).amax(-1, keepdim=True) + H24
    allowed = (flips * s2.double()[:, None]) @ wd.T + (q2.double().abs() * s2.double()[:, None]) @ wd.T * (scale + 4 * H24) \
        + 2 * H24 * (want.abs() + x.double().abs())
    assert bool(((res.double().cpu() - want).abs() <= allowed).all())


def test_mlp_refuses_rows_in_8_bits_without_their_weights():
    p = mlp_params(64, 64)
    for k in ("gate_proj", "up_proj", "down_proj"):
        p[k + ".s"] = p[k + ".s"][:, None].contiguous()
    x = torch.randn(9, 64, device=device())
    with pytest.raises(ValueError, match="one scale per row"):
        gm.mlp(p, ops.quantize_rows(x), x)
    w = torch.zeros(64, 64, device=device())
    with pytest.raises(ValueError, match="one scale per row"):
        layers.linear(ops.quantize_rows(x), w)
    wq, ws = quantize_rows_int8(torch.randn(64, 64))
    with pytest.raises(ValueError, match="no prenorm"):
        layers.linear(ops.quantize_rows(x), w, wq.to(device()), ws.to(device()), prenorm=(None, w[0], 1e-6, None))


def step_inputs(B, fmt, blocks=6, page=16, own=3, V=1000):
    """An attention layer's weights, pages that B sequences share the first `blocks` of, and an LM head."""
    dev, g = device(), torch.Generator().manual_seed(B)
    H, Hq, Hkv, D = 128, 4, 2, 256
    p = {}
    for name, (o, i) in (("q_proj", (Hq * 2 * D, H)), ("k_proj", (Hkv * D, H)), ("v_proj", (Hkv * D, H)), ("o_proj", (H, Hq * D))):
        q, s = quantize_rows_int8(torch.randn(o, i, generator=g) * i ** -0.5)
        p[name + ".q"], p[name + ".s"], p[name] = q.to(dev), s.to(dev), (q.float() * s[:, None]).to(dev)
    for name in ("q_norm", "k_norm"):
        p[name] = torch.randn(D, generator=g).to(dev) * 0.1
    table = torch.empty(B, blocks + own, dtype=torch.int32)
    table[:, :blocks] = torch.arange(blocks, dtype=torch.int32)
    table[:, blocks:] = blocks + torch.arange(B * own, dtype=torch.int32).view(B, own)
    pages = ops.kv_pages(blocks + B * own, Hkv, page, dev, fmt)
    prompt = torch.randn(1, blocks * page, H, generator=g).to(dev)
    first = table[:1].to(dev)
    layers.gated_attention_layer_paged(prompt, p, pages, first, torch.zeros(1, dtype=torch.int32, device=dev), act_int8=True)
    head, hs = quantize_rows_int8(torch.randn(V, H, generator=g))
    return dict(p=p, pages=pages, table=table.to(dev), blocks=blocks, pos=torch.full((B,), blocks * page, dtype=torch.int32, device=dev),
                head=head.to(dev), hs=hs.to(dev), emb=torch.randn(V, H, generator=g).to(dev), norm=torch.randn(H, generator=g).to(dev) * 0.1,
                temperature=torch.rand(B, generator=g).to(dev) + 0.2, top_k=torch.randint(0, 60, (B,), generator=g, dtype=torch.int32).to(dev))


def step(s, ids, u):
    """One token for every sequence: embedding, the layer on its normed rows, the head's product, the draw."""
    x = s["emb"].index_select(0, ids).unsqueeze(1)
    layers.gated_attention_layer_paged(x, s["p"], s["pages"], s["table"], s["pos"], prenorm=(None, s["norm"], 1e-6, None), residual=x,
                                       shared_blocks=s["blocks"], act_int8=True)
    logits = ops.gemm_i8(ops.add_rmsnorm_i8_(x[:, 0], None, s["norm"], 1e-6), s["head"], s["hs"])
    nxt = ops.sample_tokens(logits, u, temperature=s["temperature"], top_k=s["top_k"], top_p=0.9, min_p=0.01)
    return x, logits, nxt


@pytest.mark.parametrize("B,fmt", [(9, "bf16"), (12, "int4"), (33, "int4")])
def test_steps_eager_and_captured(B, fmt):
    """Several steps, each captured one's replay against the eager one of the same state (equal bits: no atomics in them), with
    eager work between; the draw against the 64-bit oracle on the step's own logits; the layer against the plain attention
    over the same pages."""
    announce(f"steps {fmt} B{B}")
    s = step_inputs(B, fmt)
    dev = device()
    ids = torch.arange(B, dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(1)
    us = torch.rand(20, B, generator=g).to(dev)
    g_ids, g_u = ids.clone(), us[0].clone()
    start = [t.clone() for t in s["pages"] if t is not None]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s, g_ids, g_u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, glogits, gnxt = step(s, g_ids, g_u)

    def restore(state):
        for t, v in zip([t for t in s["pages"] if t is not None], state):
            t.copy_(v)
    restore(start)
    for i in range(20):
        state = [t.clone() for t in s["pages"] if t is not None]
        x, logits, nxt = step(s, ids, us[i])
        plain = s["emb"].index_select(0, ids).unsqueeze(1)
        layers.gated_attention_layer_paged(plain, s["p"], s["pages"], s["table"], s["pos"], prenorm=(None, s["norm"], 1e-6, None),
                                           residual=plain)
        assert oracle.rel_err(x.cpu(), plain.cpu()) <= 3e-2, i  # (activations of 8 bits: 2 products of 0.3 to 0.9 %)
        torch.cuda.synchronize()
        restore(state)
        g_ids.copy_(ids)
        g_u.copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gx, x) and torch.equal(glogits, logits) and torch.equal(gnxt, nxt), i
        want, _ = sampling.sample_tokens(logits.cpu(), us[i].cpu(), s["temperature"].cpu(), s["top_k"].cpu(), 0.9, 0.01)
        assert torch.equal(nxt.cpu(), want), i
        ids = nxt
        s["pos"].add_(1)


def config():
    return Q35Config(vocab=300, hidden=128, inter=256, layers=4, n_heads=2, n_kv=1, head_dim=256, lin_k_heads=2, lin_v_heads=2,
                     lin_dk=128, lin_dv=128)


def in_doubles(monkeypatch):
    """The 8-bit operators as plain 64-bit torch code."""
    def quantize(x):
        q, s = int8.quantize_rows(x)
        return ops.RowsI8(q, s)

    def norm(x, y, w, eps=1e-6):
        if y is not None:
            x += y
        return quantize(int8.norm_rows(x, w, eps))

    def gemm(x, W, ws, out=None, epilogue="store", pushes=None, T=1, capture=None):
        y = int8.product(x.q, x.s, W, ws)
        if epilogue == "swiglu":
            y = int8.swiglu(y)
        if epilogue == "add":
            out += y
            return out
        return y.float()
    monkeypatch.setattr(ops, "quantize_rows", quantize)
    monkeypatch.setattr(ops, "add_rmsnorm_i8_", norm)
    monkeypatch.setattr(ops, "gemm_i8", gemm)


@pytest.mark.parametrize("rows,T", [(2, 70), (12, 17)])
@pytest.mark.parametrize("mlp_only", [False, True])
def test_model(rows, T, mlp_only, monkeypatch):
    """Prefill and steps with act_int8 against the same model with the 8-bit operators in doubles. They differ by fp32
    roundings, and where one of these turns a code by one: 0.25 % of a row's product at these widths (4 / 127 / sqrt(128)), in
    at most each of the 16 products of a token: 2e-2 with their sum in squares and a factor of two."""
    announce(f"model act_int8 rows {rows} T{T} mlp only {mlp_only}")
    cfg = config()
    W = workloads.init_weights(cfg, seed=3, group=128 if mlp_only else 0, mlp_group=0)
    ids = torch.randint(0, cfg.vocab, (rows, T + 3), generator=torch.Generator().manual_seed(5))
    m = gm.HybridModel(cfg, W, device(), max_len=128, rows=rows, deterministic=True, act_int8=True)
    plain = gm.HybridModel(cfg, W, device(), max_len=128, rows=rows, deterministic=True)
    got, full = [], []
    for mm, out in ((m, got), (plain, full)):
        out.append(mm.forward(ids[:, :T])[0].cpu())
        for i in range(3):
            out.append(mm.decode_step(ids[:, T + i].to(device())).cpu())
    in_doubles(monkeypatch)
    m.reset()
    want = [m.forward(ids[:, :T])[0].cpu()]
    for i in range(3):
        want.append(m.decode_step(ids[:, T + i].to(device())).cpu())
    for a, b, f in zip(got, want, full):
        assert oracle.rel_err(a, b) <= 2e-2
        assert not torch.equal(a, f)  # the 8-bit operators ran


@pytest.mark.parametrize("rows,T", [(2, 4), (1, 8), (8, 1)])
def test_few_rows_are_as_without(rows, T):
    """Up to 8 rows in all: the same bits as a model without act_int8, in prefill and steps."""
    announce(f"model act_int8, few rows {rows} T{T}")
    cfg = config()
    W = workloads.init_weights(cfg, seed=3, group=0)
    ids = torch.randint(0, cfg.vocab, (rows, T), generator=torch.Generator().manual_seed(5))
    a, b = (gm.HybridModel(cfg, W, device(), max_len=64, rows=rows, deterministic=True, act_int8=i) for i in (True, False))
    assert torch.equal(a.forward(ids)[0], b.forward(ids)[0])
    assert torch.equal(a.decode_step(ids[:, 0].to(device())), b.decode_step(ids[:, 0].to(device())))


def test_model_refuses():
    W = workloads.init_weights(config(), seed=3)
    with pytest.raises(ValueError, match="act_int8"):
        gm.HybridModel(config(), W, device(), max_len=64, rows=1, act_int8=True)
    m = gm.HybridModel(config(), W, device(), max_len=64, rows=2)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="u must be"):
        gm.sampled(m, ids, 4, u=torch.zeros(2, 3, device=device()))


@pytest.mark.parametrize("graph", [False, True])
def test_sampled(graph):
    """Tokens of sampled() against the oracle's draws from the model's logits, which a deterministic model repeats."""
    announce(f"sampled graph {graph}")
    cfg, steps, rows = config(), 6, 3
    W = workloads.init_weights(cfg, seed=4, group=0)
    m = gm.HybridModel(cfg, W, device(), max_len=64, rows=rows, deterministic=True)
    ids = torch.randint(0, cfg.vocab, (rows, 9), generator=torch.Generator().manual_seed(6))
    if graph:
        m.enable_decode_graph()
    u = torch.rand(rows, steps, generator=torch.Generator().manual_seed(7))
    temperature = torch.tensor([0.0, 0.7, 30.0])
    toks = gm.sampled(m, ids, steps, u=u.to(device()), temperature=temperature.to(device()), top_k=50, top_p=0.95)
    m.reset()
    logits = m.forward(ids)[0]
    for i in range(steps):
        want, _ = sampling.sample_tokens(logits.cpu(), u[:, i], temperature, 50, 0.95)
        assert torch.equal(toks[:, i], want.long()), i
        logits = m.decode_step(want.to(device()))
    m.reset()
    greedy, _ = gm.greedy(m, ids, steps)
    m.reset()
    again = gm.sampled(m, ids, steps, temperature=0.0)
    assert torch.equal(again, greedy)
    m.reset()
    assert gm.sampled(m, ids, 0).shape == (rows, 0)
    m.reset()
    gen = torch.Generator(device=device()).manual_seed(8)
    a = gm.sampled(m, ids, steps, generator=gen, temperature=5.0)
    m.reset()
    assert torch.equal(a, gm.sampled(m, ids, steps, generator=gen.manual_seed(8), temperature=5.0))


def test_many_rows_in_a_decode_graph():
    """12 rows with act_int8: the captured step's replays, with eager work between, against the eager steps of another model, and
    sampled() through the graph against sampled() without."""
    announce("model act_int8, decode graph of 12 rows")
    cfg, rows = config(), 12
    W = workloads.init_weights(cfg, seed=9, group=0)
    eager, graph = (gm.HybridModel(cfg, W, device(), max_len=64, rows=rows, deterministic=True, act_int8=True) for _ in range(2))
    graph.enable_decode_graph()
    ids = torch.randint(0, cfg.vocab, (rows, 7), generator=torch.Generator().manual_seed(2))
    a, b = eager.forward(ids)[0], graph.forward(ids)[0]
    assert torch.equal(a, b)
    for step in range(6):
        nxt = ops.sample_tokens(a, torch.full((rows,), 0.1 * step + 0.05, device=device()), top_k=40)
        a, b = eager.decode_step(nxt).clone(), graph.decode_step(nxt).clone()
        torch.cuda.synchronize()
        assert torch.equal(a, b), step
    u = torch.rand(rows, 5, generator=torch.Generator().manual_seed(3)).to(device())
    eager.reset()
    graph.reset()
    assert torch.equal(gm.sampled(eager, ids, 5, u=u, top_p=0.9), gm.sampled(graph, ids, 5, u=u, top_p=0.9))
