"""Attention over a paged cache whose sequences share their first pages, against oracle/paged.py in 64 bits with the bounds of
test_gpu_paged.py, and against gated_attention_paged, which reads the shared pages once per sequence."""
import math

import pytest
import torch

from gpu_util import announce, device
from oracle import paged
from q35hip import Q35Error, layers, ops
from test_gpu_paged import check_attention, columns, make, to

pytestmark = pytest.mark.gpu


def shared(fmt, B, T, Hq, Hkv, ps, blocks, ctx, **kw):
    """make() with the first `blocks` entries of every table row those of row 0."""
    d = make(fmt, B, T, Hq, Hkv, ps, ctx, **kw)
    d["table"][:, :blocks] = d["table"][0, :blocks].clone()
    return dict(d, blocks=blocks)


def attend(d, **kw):
    q, gate, _, _ = columns(d["y"], d["Hq"], d["Hkv"])
    return ops.gated_attention_paged_shared(q, kw.pop("gate", gate), d["pages"], d["table"], d["pos"], d["cos"], d["sin"],
                                            kw.pop("blocks", d["blocks"]), lens=d["lens"], q_norm_w=d["qw"], **kw)


CASES = [  # B, T, Hq, Hkv, page, shared blocks, contexts, lens
    (1, 1, 8, 2, 16, 1, [17], None), (3, 1, 8, 2, 64, 4, [300, 257, 400], None), (4, 1, 4, 4, 16, 20, [321, 330, 400, 336], None),
    (5, 1, 8, 1, 32, 3, [100, 97, 130, 98, 99], None), (9, 1, 16, 2, 128, 8, [1025 + 50 * i for i in range(9)], None),
    (2, 5, 8, 2, 16, 10, [170, 200], [5, 2]), (6, 4, 6, 2, 64, 5, [330, 324, 400, 350, 321, 333], [0, 4, 1, 3, 2, 4]),
    (3, 20, 8, 2, 32, 6, [212, 230, 260], [20, 7, 13]), (2, 70, 8, 2, 256, 2, [600, 700], None), (33, 1, 8, 2, 16, 70, [1150] * 33, None)]


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("B,T,Hq,Hkv,ps,blocks,ctx,lens", CASES)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_shared(fmt, B, T, Hq, Hkv, ps, blocks, ctx, lens, out_dtype):
    d = shared(fmt, B, T, Hq, Hkv, ps, blocks, ctx, seed=B + T, lens=lens)
    announce(f"paged shared {fmt} B{B} T{T} heads {Hq}/{Hkv} page {ps} shared {blocks} ctx {ctx[:3]} {out_dtype}")
    out = attend(to(d, device()), out_dtype=out_dtype)
    check_attention(d, out)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_bf16_queries_no_gate_no_norm(fmt):
    d = shared(fmt, 4, 2, 8, 2, 16, 12, [200, 210, 230, 260], dtype=torch.bfloat16, norm=False, rot=0)
    announce(f"paged shared {fmt} bare")
    out = attend(to(d, device()), gate=None, out_dtype=torch.float32)
    check_attention(d, out, gated=False)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_sequences_inside_and_outside_the_shared_part(fmt):
    """Sequences that end inside the shared part or just behind it, that have no token here, that start below 0 or past the
    table, and a table that is shared whole."""
    d = shared(fmt, 8, 3, 8, 2, 16, 9, [3, 16, 144, 145, 147, 200, 100, 150], lens=[3, 3, 3, 3, 3, 0, 2, 3], nb=14)
    d["pos"][6], d["pos"][7] = -1, 14 * 16 - 2
    g = to(d, device())
    announce(f"paged shared {fmt} inside")
    for blocks in (9, 1, 14):
        d["table"][:, :blocks] = d["table"][0, :blocks].clone()
        check_attention(d, attend(to(d, device()), blocks=blocks))
    whole = to(dict(d, table=d["table"][:1].expand(8, 14)), device())
    whole["table"] = d["table"][:1].to(device()).expand(8, 14)
    check_attention(d, attend(whole, blocks=14))
    assert g["table"].shape == (8, 14)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_pages_that_the_table_does_not_name(fmt):
    d = shared(fmt, 3, 2, 8, 2, 16, 6, [120, 130, 140])
    d["table"][:, 2] = -1
    d["table"][:, 5] = 1 << 20
    d["table"][1, 7] = -7
    announce(f"paged shared {fmt} missing pages")
    check_attention(d, attend(to(d, device())))
    d["table"][:, :6] = -1
    check_attention(d, attend(to(d, device())))
    d["table"][:] = -1
    assert bool((attend(to(d, device())) == 0).all())


def test_garbage_behind_a_short_sequence():
    """Infinities and NaN in the shared rows that a short sequence does not see, in rows behind the last token, in pages that no
    table names."""
    d = shared("bf16", 3, 1, 8, 2, 16, 8, [40, 129, 131], nb=10)
    kp, vp = (p.clone() for p in d["pages"][:2])
    t = d["table"]
    for p in (kp, vp):
        p[t[0, 3:8].long()] = math.nan          # behind row 0's 40 tokens, seen by no one else below
        p[t[1, 8].long(), :, 1:] = math.inf     # behind row 1's last token
        p[t[2, 9].long()] = math.nan
    only = dict(d, pages=(kp, vp, None, None))
    want = paged.gated_attention_paged(*columns(d["y"], 8, 2)[:2], only["pages"], t, d["pos"], d["cos"], d["sin"], None, d["qw"])
    announce("paged shared garbage")
    out = attend(to(only, device()), out_dtype=torch.float32).cpu().double()
    assert not bool(out[0].isnan().any()) and float((out[0] - want[0]).abs().max()) < 0.05
    assert bool(out[1:].isnan().all())  # they see the rows of NaN
    for p, q in zip((kp, vp), d["pages"]):
        p[t[0, 3:8].long()] = q[t[0, 3:8].long()]
    check_attention(d, attend(to(only, device()), out_dtype=torch.float32))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_against_the_unshared_form(fmt):
    """Long shared parts and large batches: within the bounds of two such results."""
    for B, T, ps, blocks, own in ((32, 1, 64, 128, 200), (3, 1, 64, 32, 64), (64, 4, 128, 40, 300), (2, 60, 32, 100, 100)):
        g = torch.Generator().manual_seed(B)
        n = blocks * ps
        ctx = [n + T + int(torch.randint(0, own, (1,), generator=g)) for _ in range(B)]
        d = to(shared(fmt, B, T, 8, 2, ps, blocks, ctx, seed=B), device())
        announce(f"paged shared {fmt} against unshared B{B} T{T} shared {n}")
        a = attend(d, out_dtype=torch.float32)
        q, gate, _, _ = columns(d["y"], 8, 2)
        b = ops.gated_attention_paged(q, gate, d["pages"], d["table"], d["pos"], d["cos"], d["sin"], q_norm_w=d["qw"],
                                      out_dtype=torch.float32)
        assert float((a - b).norm() / b.norm()) < 2.5e-3 and not bool(a.isnan().any())
        z = attend(d, blocks=0, out_dtype=torch.float32)
        assert torch.equal(z, b)


def test_captured_layer_and_two_streams():
    """The layer with shared blocks in a graph that follows tables, positions and lengths; and on two streams at once."""
    dev = device()
    B, ps, blocks, nb = 4, 16, 6, 9
    g = torch.Generator().manual_seed(0)
    Hq, Hkv, D, hidden = 8, 2, 256, 512
    p = {n: (0.05 * torch.randn(r, hidden, generator=g)).to(dev) for n, r in
         (("q_proj", 2 * Hq * D), ("k_proj", Hkv * D), ("v_proj", Hkv * D))}
    p["o_proj"] = (0.05 * torch.randn(hidden, Hq * D, generator=g)).to(dev)
    p["q_norm"], p["k_norm"] = torch.zeros(D, device=dev), torch.zeros(D, device=dev)
    for fmt in ("bf16", "int4"):
        pages = ops.kv_pages(blocks + B * (nb - blocks), Hkv, ps, dev, fmt)
        table = torch.cat([torch.arange(blocks).expand(B, blocks),
                           blocks + torch.arange(B * (nb - blocks)).view(B, -1)], 1).int().contiguous().to(dev)
        prompt = torch.randn(1, blocks * ps, hidden, generator=g).to(dev)
        layers.gated_attention_layer_paged(prompt, p, pages, table[:1], torch.zeros(1, dtype=torch.int32, device=dev))
        pos = torch.full((B,), blocks * ps, dtype=torch.int32, device=dev)
        x = torch.randn(B, 1, hidden, generator=g).to(dev)
        announce(f"paged shared layer {fmt}")
        a = layers.gated_attention_layer_paged(x, p, pages, table, pos, shared_blocks=blocks)
        b = layers.gated_attention_layer_paged(x, p, pages, table, pos)
        assert float((a - b).norm() / b.norm()) < 3e-3
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layers.gated_attention_layer_paged(x, p, pages, table, pos, shared_blocks=blocks)
        for i in range(4):
            x.copy_(torch.randn(B, 1, hidden, generator=g).to(dev))
            pos.add_(1)
            graph.replay()
            want = layers.gated_attention_layer_paged(x, p, pages, table, pos, shared_blocks=blocks)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    d = to(shared("int4", 5, 1, 8, 2, 16, 30, [500, 490, 600, 481, 550]), dev)
    want = attend(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [attend(d) for _ in range(5)]
    b = [attend(d) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in a + b)


def test_empty_and_refusals():
    d = to(shared("bf16", 3, 2, 8, 2, 16, 6, [120, 130, 140]), device())
    q, gate, _, _ = columns(d["y"], 8, 2)
    announce("paged shared refusals")
    nb = d["table"].shape[1]
    empty = dict(d, y=d["y"][:0], table=d["table"][:0], pos=d["pos"][:0])
    assert attend(empty).shape == (0, 2, 2048)
    for bad in (lambda: attend(d, blocks=-1), lambda: attend(d, blocks=nb + 1), lambda: attend(d, gate=gate[:, :1]),
                lambda: attend(dict(d, table=d["table"].long())), lambda: attend(dict(d, cos=d["cos"][:8], sin=d["sin"][:8])),
                lambda: attend(dict(d, pos=d["pos"].cpu())), lambda: attend(d, out_dtype=torch.float16)):
        with pytest.raises(Q35Error):
            bad()
