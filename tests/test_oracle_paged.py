"""Pins of oracle/paged.py and the host-side refusals of the paged-cache and draft-verification entry points (CPU)."""
import ctypes
import math

import pytest
import torch

import oracle
import q35hip
from oracle import paged
from q35hip import ops


def test_nibble_orders_are_the_documented_formulas():
    for g in range(4):
        for a in range(4):
            for u in range(2):
                for j in range(8):
                    assert paged.nibble_of("k")[64 * g + 16 * a + 8 * u + j] == 64 * a + 16 * g + 8 * u + j
        for c in range(16):
            for e in range(4):
                assert paged.nibble_of("v")[64 * g + 4 * c + e] == 16 * c + 4 * g + e


def test_pack_round_trip_and_values():
    gen = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 16, (5, 256), generator=gen, dtype=torch.uint8)
    for w in "kv":
        packed = paged.pack_rows(codes, w)
        assert packed.shape == (5, 128) and torch.equal(paged.unpack_rows(packed, w), codes)
    s = torch.rand(5, 4, generator=gen).bfloat16()
    v = paged.row_values(paged.pack_rows(codes, "v"), s, "v")
    assert v[3, 130] == (int(codes[3, 130]) - 8) * float(s[3, 2])


def test_quantizer_error_bound_zeros_and_values_that_are_not_finite():
    """|x - value| <= s / 2 away from the largest values; there the scale's own rounding (2^-8) adds 7 s 2^-8."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(64, 256, generator=gen)
    x[3, 64:128] = 0
    codes, s = paged.quantize_rows(x)
    v = paged.row_values(paged.pack_rows(codes, "k"), s, "k")
    sd = s.double().repeat_interleave(64, -1)
    assert bool(((v - x.double()).abs() <= sd * (0.5 + 7 * 2 ** -8)).all())
    assert float(s[3, 1]) == 0 and bool((v[3, 64:128] == 0).all())
    x[5, 70] = math.inf
    x[6, 200] = math.nan
    codes, s = paged.quantize_rows(x)
    assert torch.isnan(s).nonzero().tolist() == [[5, 1], [6, 3]]
    assert bool((codes[5, 64:128] == 8).all())


@pytest.mark.parametrize("T", [1, 3])
def test_attention_and_append_against_the_dense_oracle(T):
    gen = torch.Generator().manual_seed(T)
    B, Hq, Hkv, ps, nb = 2, 4, 2, 16, 3
    pos = torch.tensor([20, 7], dtype=torch.int32)
    n = nb * ps
    cos, sin = oracle.rope_tables(n, oracle.rope_inv_freq())
    dense_k = torch.randn(B, Hkv, n, 256, generator=gen).bfloat16()
    dense_v = torch.randn(B, Hkv, n, 256, generator=gen).bfloat16()
    table = torch.randperm(B * nb, generator=gen).view(B, nb).int()
    pages = [torch.zeros(B * nb, Hkv, ps, 256, dtype=torch.bfloat16) for _ in range(2)] + [None, None]
    for b in range(B):
        for j in range(nb):
            pages[0][int(table[b, j])] = dense_k[b, :, j * ps:(j + 1) * ps]
            pages[1][int(table[b, j])] = dense_v[b, :, j * ps:(j + 1) * ps]
    q = torch.randn(B, T, Hq, 256, generator=gen).bfloat16()
    gate = torch.randn(B, T, Hq, 256, generator=gen).bfloat16()
    ref = oracle.gated_attention_cached(q, dense_k, dense_v, gate.flatten(2), pos, cos, sin, dtype=torch.float64)
    got = paged.gated_attention_paged(q, gate, pages, table, pos, cos, sin)
    assert oracle.rel_err(got, ref) < 1e-12
    # the rows written through the table are the rows read back
    k = torch.randn(B, T, Hkv, 256, generator=gen)
    v = torch.randn(B, T, Hkv, 256, generator=gen)
    paged.paged_append(k, v, pages, table, pos, cos, sin)
    kr, vr = paged.paged_rows(pages, table, pos, T)
    for b in range(B):
        at = slice(int(pos[b]), int(pos[b]) + T)
        want = oracle.apply_partial_rope(k[b:b + 1].double(), cos[at].double(), sin[at].double())[0]
        assert torch.equal(kr[b], want.transpose(0, 1).bfloat16().double())
    assert torch.equal(vr, v.transpose(1, 2).bfloat16().double())


def test_verification_draws_from_the_target():
    """Drafts drawn from q, kept or replaced by the rule: integrated over a grid of both random numbers, the first token's
    distribution is p (the property that defines the rule)."""
    V, N = 5, 60
    gen = torch.Generator().manual_seed(3)
    logits = torch.randn(1, 2, V, generator=gen)
    q = torch.softmax(torch.randn(V, generator=gen).double(), 0).float()
    p = torch.softmax(logits[0, 0].double(), 0)
    grid = (torch.arange(N) + 0.5) / N
    u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).view(-1, 2).float()
    n = u.shape[0]
    out = torch.zeros(V, dtype=torch.float64)
    for x in range(V):
        _, tok = paged.verify_drafts(logits.expand(n, 2, V), torch.full((n, 1), x, dtype=torch.int32), u,
                                     draft_probs=q.expand(n, 1, V))
        out += float(q[x]) * torch.bincount(tok[:, 0].long(), minlength=V).double() / n
    # each of the V drafts' regions is counted on a grid of step 1 / N: at most V + 1 borders, 1 / N each
    assert float((out - p).abs().max()) <= (V + 1) / N * float(q.max()) + 1e-6


def test_verification_greedy_and_empty_rows():
    logits = torch.tensor([[[0., 3., 3.], [1., 0., 2.]], [[-math.inf] * 3, [0., 0., 0.]]])
    ids = torch.tensor([[1], [0]], dtype=torch.int32)
    n, tok = paged.verify_drafts(logits, ids, torch.full((2, 2), 0.9), temperature=0.0)
    assert n.tolist() == [1, 0] and tok.tolist() == [[1, 2], [0, -1]]


# ---------------------------------------------------------------- refusals (nothing is launched)
FAKE = 0x1000


def _append(k=FAKE, ksb=512, kst=512, ksh=256, dt=0, w=FAKE, rot=64, cos=FAKE, table=FAKE, ld=4, nb=4, pos=FAKE, kp=FAKE,
            ks=FAKE, fmt=4, n=8, ps=64, B=2, T=1, H=2, D=256):
    return q35hip.lib().q35_paged_kv_append(k, ksb, kst, ksh, FAKE, 512, 512, 256, dt, w, 1e-6, cos, FAKE, rot, table, ld,
                                            nb, pos, None, kp, FAKE, ks, FAKE, fmt, n, ps, B, T, H, D, None)


def test_append_refusals():
    for kw in (dict(k=None), dict(pos=None), dict(table=None), dict(kp=None), dict(B=0), dict(T=0), dict(H=0), dict(n=0),
               dict(nb=0), dict(ps=0), dict(ld=3), dict(ks=None), dict(cos=None), dict(rot=-8), dict(rot=63),
               dict(ksb=-4)):
        assert _append(**kw) == 1, kw
    for kw in (dict(D=128), dict(ps=8), dict(ps=48), dict(ps=2048), dict(fmt=2), dict(dt=2), dict(rot=62), dict(k=FAKE + 4),
               dict(kst=514), dict(w=FAKE + 4), dict(kp=FAKE + 8), dict(B=70000), dict(n=1 << 40), dict(nb=1 << 27, ld=1 << 27)):
        assert _append(**kw) == 2, kw


def _rows(kp=FAKE, out=FAKE, ks=FAKE, fmt=4, T=3, D=256, ps=16):
    return q35hip.lib().q35_paged_kv_rows(kp, FAKE, ks, FAKE, fmt, 8, ps, FAKE, 4, 4, FAKE, None, out, FAKE, 2, T, 2, D,
                                          None)


def test_rows_refusals():
    for kw in (dict(kp=None), dict(out=None), dict(ks=None), dict(T=0)):
        assert _rows(**kw) == 1, kw
    for kw in (dict(out=FAKE + 8), dict(fmt=3), dict(D=64), dict(ps=24)):
        assert _rows(**kw) == 2, kw


def _attn(q=FAKE, qst=2048, gate=FAKE, gst=2048, dt=0, w=None, rot=64, out=FAKE, odt=1, B=2, T=1, Hq=8, Hkv=2, D=256, fmt=1,
          ps=64, nb=4, splits=0, ws=FAKE, wsb=1 << 30):
    return q35hip.lib().q35_gated_attn_paged(q, 2048, qst, 256, gate, 2048, gst, 256, dt, w, 1e-6, FAKE, FAKE, rot, FAKE,
                                             FAKE, None, None, fmt, 8, ps, FAKE, nb, nb, FAKE, None, out, odt, B, T, Hq,
                                             Hkv, D, 0.0625, splits, ws, wsb, None)


def test_attention_refusals():
    for kw in (dict(q=None), dict(out=None), dict(Hq=7), dict(Hq=0), dict(fmt=4), dict(rot=33), dict(T=0)):
        assert _attn(**kw) == 1, kw
    for kw in (dict(odt=2), dict(dt=4), dict(out=FAKE + 8), dict(q=FAKE + 8), dict(gate=FAKE + 8), dict(gst=2046),
               dict(w=FAKE + 4), dict(rot=68), dict(D=128), dict(Hq=8192), dict(T=1 << 25)):
        assert _attn(**kw) == 2, kw
    need = q35hip.lib().q35_gated_attn_paged_workspace_bytes(2, 1, 8, 2, 256, 16, 64, 0)
    assert need == 2 * 8 * 8 * 258 * 4  # eight runs, of 128 keys each
    assert _attn(nb=16, wsb=need - 1) == 3 and _attn(nb=16, ws=None) == 3 and _attn(nb=16, ws=FAKE + 8) == 3
    assert _attn(splits=2, wsb=2 * 8 * 2 * 258 * 4 - 1) == 3  # 256 keys asked for in two runs
    assert q35hip.lib().q35_gated_attn_paged_workspace_bytes(2, 1, 8, 3, 256, 4, 64, 0) == 0


def _verify(x=FAKE, lsp=100, ids=FAKE, probs=None, psp=100, u=FAKE, T=1.0, n=FAKE, B=2, K=3, V=100, ws=FAKE, wsb=1 << 30):
    return q35hip.lib().q35_verify_drafts(x, 400, lsp, ids, 3, probs, 300, psp, u, 4, None, None, ctypes.c_float(T), n,
                                          FAKE, B, K, V, ws, wsb, None)


def test_verify_refusals():
    for kw in (dict(x=None), dict(u=None), dict(n=None), dict(ids=None), dict(B=0), dict(K=-1), dict(V=0), dict(lsp=99),
               dict(probs=FAKE, psp=99), dict(T=-1.0), dict(T=math.nan)):
        assert _verify(**kw) == 1, kw
    assert _verify(K=256) == 2 and _verify(B=65535, K=1) == 2
    need = q35hip.lib().q35_verify_drafts_workspace_bytes(2, 3, 100)
    assert need > 0 and _verify(wsb=need - 1) == 3 and _verify(ws=None) == 3 and _verify(ws=FAKE + 8) == 3


def test_ops_refuse_cpu_tensors_and_bad_formats():
    pages = ops.kv_pages(4, 2, 16, "cpu", "int4")
    assert pages.k.shape == (4, 2, 16, 128) and pages.v_scale.shape == (4, 2, 16, 4)
    table, pos = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x, tab = torch.zeros(1, 1, 2, 256), torch.zeros(32, 32)
    for call in (lambda: ops.paged_kv_append_(x, x, pages, table, pos, tab, tab),
                 lambda: ops.paged_kv_rows(pages, table, pos, 4),
                 lambda: ops.gated_attention_paged(x, None, pages, table, pos, tab, tab),
                 lambda: ops.verify_drafts(torch.zeros(1, 2, 9), pos[:, None], torch.zeros(1, 2))):
        with pytest.raises(q35hip.Q35Error, match="no CPU|HIP device"):
            call()
    with pytest.raises(ValueError, match="fmt"):
        ops.kv_pages(4, 2, 16, "cpu", "fp8")
    with pytest.raises(ValueError, match="page_size"):
        ops.kv_pages(4, 2, 24, "cpu")
    with pytest.raises(q35hip.Q35Error, match="out_dtype"):
        ops.gated_attention_paged(x, None, pages, table, pos, tab, tab, out_dtype=torch.float16)
