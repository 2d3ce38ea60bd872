"""The operators for sampling on tensors that stand for others (vmap, functionalization, negated views), in traces and compiled
functions, from two threads, at the largest sizes, and on random numbers that are none: what plain calls give."""
import math
import threading

import pytest
import torch

from gpu_util import announce, device
from oracle import sampling
from q35hip import ops
from test_gpu_paged import columns, make, to

pytestmark = pytest.mark.gpu


def inputs(B=4, V=3001, K=128, N=200, seed=0):
    dev, g = device(), torch.Generator().manual_seed(seed)
    return ((torch.randn(B, V, generator=g) * 2).to(dev), torch.rand(3, B, generator=g).to(dev), torch.randn(B, K, generator=g).to(dev),
            torch.randint(-127, 128, (N, K), generator=g).to(torch.int8).to(dev), torch.rand(N, generator=g).to(dev),
            torch.randn(K, generator=g).to(dev))


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def attention(g, q, gate):
    return ops.gated_attention_paged_shared(q, gate, g["pages"], g["table"], g["pos"], g["cos"], g["sin"], 2, lens=g["lens"])


def pages(fmt, seed=0):
    g = make(fmt, 3, 2, 4, 2, 16, [70, 40, 33], lens=[2, 1, 2], seed=seed)
    g["table"][:, :2] = g["table"][0, :2].clone()
    return to(g, device())


def test_vmap():
    x, us, r, W, ws, w = inputs()
    announce("sampling ops under vmap")
    tok, pr = torch.vmap(lambda u: ops.sample_tokens(x, u, top_k=9, want_probs=True))(us)
    for i, u in enumerate(us):
        assert same((tok[i], pr[i]), ops.sample_tokens(x, u, top_k=9, want_probs=True))
    xs = torch.stack([x, -x])
    out = torch.vmap(lambda x: ops.filter_logits(x, top_p=0.4))(xs)
    assert same(out, [ops.filter_logits(a, top_p=0.4) for a in xs])
    q, s = torch.vmap(lambda r: tuple(ops.quantize_rows(r)))(torch.stack([r, 3 * r]))
    assert same((q[1], s[1]), ops.quantize_rows(3 * r))
    g = pages("int4")
    q, gate, _, _ = columns(g["y"], 4, 2)
    out = torch.vmap(lambda q: attention(g, q, gate))(torch.stack([q, -q]))
    assert same(out, [attention(g, q, gate), attention(g, -q, gate)])


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_negated_views_and_functional_tensors(fmt):
    x, us, r, W, ws, w = inputs()
    g = pages(fmt)
    q, gate, _, _ = columns(g["y"], 4, 2)
    announce(f"sampling ops {fmt}, negated views and functional tensors")
    assert torch.equal(attention(g, torch._neg_view(q), -gate), attention(g, -q, -gate))
    assert torch.equal(torch.func.functionalize(lambda q: attention(g, q, gate))(-q), attention(g, -q, gate))
    assert torch.equal(ops.sample_tokens(torch._neg_view(x), us[0]), ops.sample_tokens(-x, us[0]))
    assert torch.equal(torch.func.functionalize(lambda x: ops.filter_logits(x, top_k=5))(x), ops.filter_logits(x, top_k=5))
    assert same(ops.quantize_rows(torch._neg_view(r)), ops.quantize_rows(-r))
    assert torch.equal(ops.gemm_i8(ops.quantize_rows(r), W, torch._neg_view(ws)), ops.gemm_i8(ops.quantize_rows(r), W, -ws))


@pytest.mark.parametrize("how", ["compiled", "traced"])
def test_recorded(how):
    """A whole step recorded on one set of inputs and run on another."""
    x, us, r, W, ws, w = inputs()
    g = pages("bf16")
    q, gate, _, _ = columns(g["y"], 4, 2)

    def step(q, x, r, y, u):
        o = attention(g, q, gate)
        n = ops.add_rmsnorm_i8_(r, y, w)
        a = ops.gemm_i8(n, W, ws, epilogue="swiglu")
        b = ops.gemm_i8(ops.quantize_rows(r), W, ws)
        return o, a, b, n[0], n[1], ops.sample_tokens(ops.filter_logits(x, top_k=50), u, top_p=0.9), r
    announce(f"sampling ops {how}")
    y = torch.ones_like(r)
    if how == "compiled":
        f = torch.compile(step, fullgraph=True, backend="eager")
    else:
        f = torch.jit.trace(step, (q, x, r.clone(), y, us[0]), check_trace=False)
    got = f(2 * q, -x, 2 * r, y, us[1])
    assert same(got, step(2 * q, -x, 2 * r, y, us[1]))


def test_calls_from_two_threads():
    dev = device()
    data = [inputs(seed=i) for i in range(2)]
    gs = [pages(f, i) for i, f in enumerate(("bf16", "int4"))]

    def run(i):
        x, us, r, W, ws, w = data[i]
        q, gate, _, _ = columns(gs[i]["y"], 4, 2)
        return (attention(gs[i], q, gate), *ops.sample_tokens(x, us[0], top_p=0.8, want_probs=True),
                ops.gemm_i8(ops.add_rmsnorm_i8_(r, None, w), W, ws))
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    bad = []

    def many(i):
        try:
            with torch.cuda.device(dev), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    out = run(i)
                    torch.cuda.current_stream().synchronize()
                    if not same(out, want[i]):
                        bad.append(i)
        except Exception as e:  # (to the thread that asserts)
            bad.append(e)
    announce("sampling calls from two threads")
    threads = [threading.Thread(target=many, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not bad and not any(t.is_alive() for t in threads), bad


def test_random_numbers_that_are_none():
    """Outside 0 .. 1 and NaN: a kept token all the same."""
    V = 5000
    x = torch.randn(6, V, generator=torch.Generator().manual_seed(2)).to(device())
    u = torch.tensor([math.nan, -1.0, 2.0, math.inf, -math.inf, 0.5], device=device())
    announce("sample: random numbers that are none")
    for cuts in (dict(top_k=5), dict(top_p=0.3), dict()):
        tok, pr = ops.sample_tokens(x, u, want_probs=True, **cuts)
        assert bool(((tok >= 0) & (tok < V)).all())
        assert bool((pr.gather(1, tok.long()[:, None]) > 0).all())


@pytest.mark.parametrize("cuts", [dict(top_k=2000), dict(top_p=0.6), dict(top_k=3000000, top_p=0.999, min_p=1e-6)], ids=str)
def test_the_largest_vocabulary(cuts):
    V = 1 << 22
    x = torch.randn(2, V, generator=torch.Generator().manual_seed(3)) * 1.5
    u = torch.tensor([0.25, 0.9])
    announce(f"sample V{V} {cuts}")
    tok, pr = ops.sample_tokens(x.to(device()), u.to(device()), want_probs=True, **cuts)
    want, wp = sampling.sample_tokens(x, u, **cuts)
    assert torch.equal(tok.cpu(), want)
    assert torch.equal(pr.cpu() > 0, wp > 0)
    assert bool(((pr.double().cpu() - wp).abs() <= 2.0 ** -23 * wp + 2.0 ** -149).all())


def test_rows_past_32_bits():
    """More than 2^31 logits: the last rows' offsets need more than 32 bits, of logits and outputs."""
    B, V = 520, 1 << 22
    announce(f"sample B{B} V{V}")
    dev = device()
    x = torch.full((B, V), -20.0, device=dev)
    at = (torch.arange(B, device=dev) * 8009) % V
    x[torch.arange(B, device=dev), at] = 5.0
    x[torch.arange(B, device=dev), V - 1] = 4.0
    u = torch.full((B,), 0.999, device=dev)
    tok, pr = ops.sample_tokens(x, u, top_k=2, want_probs=True)
    assert bool((tok == V - 1).all())
    rows = torch.tensor([0, 511, 512, 519], device=dev)
    for r in rows.tolist():
        kept = pr[r].nonzero()[:, 0]
        assert sorted(kept.tolist()) == sorted({int(at[r]), V - 1})
    del pr
    out = ops.filter_logits(x, top_k=2)
    for r in rows.tolist():
        assert int((out[r] > -math.inf).sum()) == 2 and float(out[r, V - 1]) == 4.0


def test_products_past_32_bits():
    """Rows of q, and results, at offsets past 2^31."""
    dev = device()
    announce("gemm_i8 past 32 bits")
    M, K, N = 70001, 64, 33000
    W = torch.ones(N, K, dtype=torch.int8, device=dev)
    W[1::2] = -1
    s, ws = torch.rand(M, device=dev), torch.rand(N, device=dev)
    wide = torch.zeros(M, 40000, dtype=torch.int8, device=dev)  # 2.8e9 bytes
    wide[:, :K] = torch.arange(M, device=dev).remainder(100)[:, None].to(torch.int8)
    y = ops.gemm_i8((wide[:, :K], s), W, ws)
    for m in (0, 1, 53687, 65535, 65536, M - 1):
        want = torch.full((N,), float(K * (m % 100)), device=dev)
        want[1::2] *= -1
        want = want * s[m] * ws
        assert bool(((y[m] - want).abs() <= 3.2 * 2.0 ** -24 * want.abs()).all()), m
    x = torch.zeros(M, 40000, dtype=torch.bfloat16, device=dev)
    x[:, 100:164] = torch.arange(M, device=dev).remainder(200)[:, None].to(torch.bfloat16)
    q, s = ops.quantize_rows(x[:, 100:164])
    assert bool((q.float() == torch.where(s[:, None] > 0, 127.0, 0.0)).all())
    assert torch.equal(s, (x[:, 100].double() / 127).float())


@pytest.mark.parametrize("V", [4092, 4093, 16379, 16380, 16381, 16385])
def test_where_short_rows_end(V):
    """Around the longest row that one block takes, at each distance from 16 bytes; first and last tokens kept and drawn."""
    announce(f"sample short rows V{V}")
    g = torch.Generator().manual_seed(V)
    for off in range(4):
        wide = torch.full((3, V + 8), 90.0)
        x = torch.randn(3, V, generator=g) * 3
        x[0, 0], x[1, V - 1], x[2, [0, V - 1]] = 12.0, 12.0, 11.0
        wide[:, off:off + V] = x
        view = wide.to(device())[:, off:off + V]
        u = torch.tensor([0.1, 0.5, 0.9])
        for cuts in (dict(), dict(top_k=30), dict(top_k=2000, top_p=0.99), dict(top_p=0.97, min_p=1e-3)):
            tok, pr = ops.sample_tokens(view, u.to(device()), want_probs=True, **cuts)
            want, wp = sampling.sample_tokens(x, u, **cuts)
            assert torch.equal(tok.cpu(), want)
            assert torch.equal(pr.cpu() > 0, wp > 0)
            kept = ops.filter_logits(view, **cuts).cpu()
            assert torch.equal(kept, sampling.filter_logits(x, **cuts))
