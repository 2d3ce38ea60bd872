"""The paged-cache ops on tensors that stand for others (vmap, functionalization, negated views), under autograd, in traces and
compiled functions: what the plain calls give."""
import pytest
import torch

from gpu_util import announce, device
from q35hip import ops
from test_gpu_paged import append, attend, columns, make, to

pytestmark = pytest.mark.gpu


def drafts(B, K, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    dev = device()
    return (torch.randn(B, K + 1, V, generator=g).to(dev), torch.randint(0, V, (B, K), generator=g).int().to(dev),
            torch.rand(5, B, K + 1, generator=g).to(dev))


def test_vmap():
    """Mapped over any argument, the first or another."""
    x, ids, us = drafts(3, 2, 1000)
    announce("paged ops under vmap")
    want = [ops.verify_drafts(x, ids, u) for u in us]
    n, tok = torch.vmap(lambda u: ops.verify_drafts(x, ids, u))(us)
    assert all(torch.equal(n[i], w[0]) and torch.equal(tok[i], w[1]) for i, w in enumerate(want))
    g = to(make("int4", 2, 3, 4, 2, 16, [70, 33], lens=[3, 2]), device())
    q, gate, _, _ = columns(g["y"], 4, 2)
    qs = torch.stack([q, 2 * q, -q])
    rest = (g["pages"], g["table"], g["pos"], g["cos"], g["sin"])
    out = torch.vmap(lambda q: ops.gated_attention_paged(q, gate, *rest))(qs)
    assert all(torch.equal(out[i], ops.gated_attention_paged(qs[i], gate, *rest)) for i in range(3))
    pos = torch.tensor([[0, 3], [5, 1]], dtype=torch.int32, device=q.device)
    k, v = torch.vmap(lambda p: ops.paged_kv_rows(g["pages"], g["table"], p, 9))(pos)
    for i in range(2):
        wk, wv = ops.paged_kv_rows(g["pages"], g["table"], pos[i], 9)
        assert torch.equal(k[i], wk) and torch.equal(v[i], wv)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_negated_views_and_functional_tensors(fmt):
    g = to(make(fmt, 2, 3, 4, 2, 16, [70, 33], lens=[3, 2]), device())
    q, gate, _, _ = columns(g["y"], 4, 2)
    rest = (g["pages"], g["table"], g["pos"], g["cos"], g["sin"])
    announce(f"paged attention {fmt}, negated views and functional tensors")
    want = ops.gated_attention_paged(-q, -gate, *rest)
    for a, b in ((-q, torch._neg_view(gate)), (torch._neg_view(q), -gate)):
        assert torch.equal(ops.gated_attention_paged(a, b, *rest), want)
    assert torch.equal(torch.func.functionalize(lambda q: ops.gated_attention_paged(q, -gate, *rest))(-q), want)


def test_parameters_and_inputs_that_ask_for_a_gradient():
    """Parameters are tensors like others; autograd is told that there is no gradient, as by every op of the package."""
    g = to(make("bf16", 2, 3, 4, 2, 16, [70, 33], lens=[3, 2]), device())
    q, gate, _, _ = columns(g["y"], 4, 2)
    rest = (g["pages"], g["table"], g["pos"], g["cos"], g["sin"])
    announce("paged attention, parameters")
    want = ops.gated_attention_paged(q, gate, *rest, q_norm_w=g["qw"])
    w = torch.nn.Parameter(g["qw"])
    with torch.no_grad():
        assert torch.equal(ops.gated_attention_paged(q, gate, *rest, q_norm_w=w), want)
    out = ops.gated_attention_paged(q, gate, *rest, q_norm_w=w)
    assert torch.equal(out, want) and out.requires_grad


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_compiled_whole(fmt):
    g = to(make(fmt, 2, 3, 4, 2, 16, [70, 33], lens=[3, 2]), device())
    x, ids, us = drafts(2, 2, 500)
    other = dict(g, pages=tuple(None if p is None else p.clone() for p in g["pages"]))

    def step(y, pages, u):
        q, gate, k, v = columns(y, 4, 2)
        rope = (g["cos"], g["sin"])
        ops.paged_kv_append_(k, v, pages, g["table"], g["pos"], *rope, lens=g["lens"], k_norm_w=g["kw"])
        o = ops.gated_attention_paged(q, gate, pages, g["table"], g["pos"], *rope, lens=g["lens"])
        return o, *ops.paged_kv_rows(pages, g["table"], g["pos"], 3), *ops.verify_drafts(x, ids, u)
    announce(f"paged ops compiled {fmt}")
    got = torch.compile(step, fullgraph=True, backend="eager")(g["y"], other["pages"], us[0])
    want = step(g["y"], g["pages"], us[0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(g["pages"], other["pages"]):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_a_trace_run_on_other_inputs(fmt):
    """torch.jit.trace records the ops: what it gives for other queries, keys and random numbers is what the calls give."""
    g = to(make(fmt, 2, 3, 4, 2, 16, [70, 33], lens=[3, 2]), device())
    x, ids, us = drafts(2, 2, 500)
    other = tuple(None if p is None else p.clone() for p in g["pages"])

    def step(y, u, *pages):
        q, gate, k, v = columns(y, 4, 2)
        rope = (g["cos"], g["sin"])
        ops.paged_kv_append_(k, v, pages, g["table"], g["pos"], *rope, lens=g["lens"], k_norm_w=g["kw"])
        o = ops.gated_attention_paged(q, gate, pages, g["table"], g["pos"], *rope, lens=g["lens"])
        return o, *ops.paged_kv_rows(pages, g["table"], g["pos"], 3), *ops.verify_drafts(x, ids, u)
    announce(f"paged ops traced {fmt}")
    traced = torch.jit.trace(step, (g["y"], us[0], *(p.clone() for p in g["pages"] if p is not None)), check_trace=False)
    y = 0.5 * g["y"].flip(0)
    got = traced(y, us[1], *(p for p in other if p is not None))
    want = step(y, us[1], *g["pages"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(g["pages"], other):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_token_drawn_from_the_stack_s_logits():
    """K = 0 on what the hybrid stack gives: the oracle's tokens for the same logits, and what the next step takes."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))
    from oracle import paged
    from q35hip import model
    from tiny_weights import tiny_config, tiny_inputs, tiny_weights
    dev, cfg = device(), tiny_config()
    ids, _ = tiny_inputs(cfg)
    m = model.HybridModel(cfg, tiny_weights(cfg), dev, max_len=256, rows=2)
    announce("tokens drawn from the stack's logits")
    logits, _ = m.forward(ids)
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        u = torch.rand(2, 1, generator=g)
        n, tok = ops.verify_drafts(logits[:, None], logits.new_empty(2, 0, dtype=torch.int32), u.to(dev), temperature=0.7)
        want = paged.verify_drafts(logits[:, None].cpu(), torch.empty(2, 0, dtype=torch.int32), u, temperature=0.7)
        assert torch.equal(n.cpu(), want[0]) and torch.equal(tok.cpu(), want[1])
        logits, _ = m.forward(tok)


@pytest.mark.parametrize("T", [1, 3])
def test_layer_with_parameters_outside_no_grad(T):
    """Weights as nn.Parameter with grad mode on: the layer's values, with and without a residual, as under no_grad."""
    from q35hip import layers
    dev = device()
    g = torch.Generator().manual_seed(3)
    p = {n: torch.nn.Parameter((torch.randn(*s, generator=g) * 0.05).to(dev))
         for n, s in (("q_proj", (1024, 256)), ("k_proj", (256, 256)), ("v_proj", (256, 256)), ("o_proj", (256, 512)),
                      ("q_norm", (256,)), ("k_norm", (256,)))}
    x, res = (torch.randn(2, T, 256, generator=g).to(dev) for _ in range(2))
    table = torch.tensor([[0, 3], [2, 1]], dtype=torch.int32, device=dev)
    pos = torch.tensor([0, 20], dtype=torch.int32, device=dev)
    announce(f"paged layer with parameters, T {T}")
    out = []
    for grad in (False, True):
        pages = ops.kv_pages(4, 1, 16, dev, "int4")
        with torch.set_grad_enabled(grad):
            a = layers.gated_attention_layer_paged(x, dict(p), pages, table, pos)
            b = layers.gated_attention_layer_paged(x, dict(p), pages, table, pos, residual=res.clone(), fixed_order=True)
        out.append((a.detach(), b.detach(), *pages))
    for a, b in zip(*out):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_calls_from_two_threads():
    """Each thread on a stream of its own (the extension gives the interpreter lock up in a call): the results of one."""
    import threading
    dev = device()
    gs = [to(make(fmt, 2, 3, 8, 2, 64, [900, 130], lens=[3, 2], seed=i), dev) for i, fmt in enumerate(("bf16", "int4"))]
    want = [attend(g) for g in gs]
    x, ids, us = drafts(3, 2, 20000)
    drawn = ops.verify_drafts(x, ids, us[0])
    torch.cuda.synchronize()
    bad = []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    out, n = attend(gs[i]), ops.verify_drafts(x, ids, us[0])
                    torch.cuda.current_stream().synchronize()
                    if not (torch.equal(out, want[i]) and all(torch.equal(a, b) for a, b in zip(n, drawn))):
                        bad.append(i)
        except Exception as e:  # (to the thread that asserts)
            bad.append(e)
    announce("paged calls from two threads")
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not bad and not any(t.is_alive() for t in threads), bad
