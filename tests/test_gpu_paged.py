"""Paged KV cache on the GPU: append, rows read back and the attention over the pages against oracle/paged.py in 64 bits.

Bounds. Append: bf16 rows within one rounding (2^-8 relative) of the 64-bit values plus the fp32 arithmetic in front of it
(2^-18 of the row's largest value); 4-bit codes and scales equal. Attention, per output value, with w the softmax weights:
  2^-8 sum w |v|            each weight rounded to bf16 once
  2 d sum w |v|             scores off by d sum |q k| scale, a weight's numerator and the sum of all both moving: fp32 norm,
                            rotation and sums (2^-16) and q's own rounding, bf16 hi + lo (2^-17) against bf16 keys, so
                            d = 2^-15; against 4-bit codes fp16 (half a step is 2^-12 of q), so d = 2^-12 + 2^-15
  2^-16 sum w |v|           exponentials, sums and divisions in fp32
  (n / 32 + 16) 2^-19 sum w s   fp32 sums over n keys of offset codes (at most 31 s each, in n / 32 products per wave)
  2^-8 |out| (2^-23 for fp32)   the output's own rounding, with 2^-20 |out| of the gate
"""
import math

import pytest
import torch

from gpu_util import announce, device
from oracle import paged
from q35hip import layers, ops, workloads

pytestmark = pytest.mark.gpu


def make(fmt, B, T, Hq, Hkv, ps, ctx, seed=0, dtype=torch.float32, lens=None, nb=None, norm=True, rot=64):
    """CPU inputs: y's columns as strided views, a pool of pages with every row written, a shuffled table."""
    g = torch.Generator().manual_seed(seed)
    nb = -(-max(ctx) // ps) + 1 if nb is None else nb
    n = B * nb + 2
    y = torch.randn(B, T, 2 * (Hq + Hkv) * 256, generator=g).to(dtype)
    pk, pv = (torch.randn(n, Hkv, ps, 256, generator=g) for _ in range(2))
    if fmt == "bf16":
        pages = (pk.bfloat16(), pv.bfloat16(), None, None)
    else:
        (kc, ks), (vc, vs) = paged.quantize_rows(pk), paged.quantize_rows(pv)
        pages = (paged.pack_rows(kc, "k"), paged.pack_rows(vc, "v"), ks, vs)
    cos, sin = workloads.rope_tables(nb * ps, partial_rotary_factor=rot / 256)
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    pos = torch.tensor([c - (T if lens is None else lens[b]) for b, c in enumerate(ctx)], dtype=torch.int32)
    return dict(y=y, pages=pages, table=torch.randperm(n, generator=g)[:B * nb].view(B, nb).int(), pos=pos, lens=lens_t,
                cos=cos, sin=sin, qw=0.1 * torch.randn(256, generator=g) if norm else None,
                kw=0.1 * torch.randn(256, generator=g) if norm else None, Hq=Hq, Hkv=Hkv, fmt=fmt)


def columns(y, Hq, Hkv):
    q, k, v = y.split([2 * Hq * 256, Hkv * 256, Hkv * 256], -1)
    q = q.unflatten(-1, (Hq, 512))
    return q[..., :256], q[..., 256:], k.unflatten(-1, (Hkv, 256)), v.unflatten(-1, (Hkv, 256))


def to(d, dev):
    out = dict(d)
    for k, v in d.items():
        if torch.is_tensor(v):
            out[k] = v.to(dev)
    out["pages"] = tuple(None if p is None else p.to(dev) for p in d["pages"])
    return out


def attend(d, **kw):
    q, gate, _, _ = columns(d["y"], d["Hq"], d["Hkv"])
    return ops.gated_attention_paged(q, kw.pop("gate", gate), d["pages"], d["table"], d["pos"], d["cos"], d["sin"],
                                     lens=d["lens"], q_norm_w=d["qw"], **kw)


def check_attention(d, out, gated=True, **kw):
    q, gate, _, _ = columns(d["y"], d["Hq"], d["Hkv"])
    ref, amp, prod, step = paged.gated_attention_paged(q, gate if gated else None, d["pages"], d["table"], d["pos"],
                                                       d["cos"], d["sin"], d["lens"], d["qw"], spread=True, **kw)
    n = d["table"].shape[1] * d["pages"][0].shape[2]
    last = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -23
    q_off = 2.0 ** -15 + (2.0 ** -12 if d["fmt"] == "int4" else 0)
    bound = (2.0 ** -8 + 2 * q_off * prod + 2.0 ** -16) * amp + (n / 32 + 16) * 2.0 ** -19 * step \
        + (last + 2.0 ** -20) * ref.abs() * (1 + 2.0 ** -7) + 1e-30
    err = (out.double().cpu() - ref).abs()
    worst = float((err / bound).max())
    assert not bool(out.isnan().any()) and worst <= 1, worst
    assert bool((out.cpu()[ref == 0] == 0).all())
    return worst


def append(d):
    _, _, k, v = columns(d["y"], d["Hq"], d["Hkv"])
    ops.paged_kv_append_(k, v, d["pages"], d["table"], d["pos"], d["cos"], d["sin"], lens=d["lens"], k_norm_w=d["kw"])


def oracle_append(d):
    _, _, k, v = columns(d["y"], d["Hq"], d["Hkv"])
    pages = tuple(None if p is None else p.clone() for p in d["pages"])
    paged.paged_append(k, v, pages, d["table"], d["pos"], d["cos"], d["sin"], d["lens"], d["kw"])
    return pages


def same_pages(fmt, got, want):
    if fmt == "int4":
        for a, b in zip(got, want):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
        return
    for a, b in zip(got[:2], want[:2]):
        a, b = a.double().cpu(), b.double()
        bound = b.abs() * 2.0 ** -8 * 2 + b.abs().amax(-1, keepdim=True) * 2.0 ** -18
        assert bool(((a - b).abs() <= bound).all())


APPEND = [  # B, T, Hq, Hkv, page, contexts, lens
    (1, 1, 8, 2, 16, [1], None), (3, 1, 8, 2, 64, [700, 64, 65], None), (2, 5, 8, 2, 16, [20, 33], [5, 2]),
    (3, 4, 4, 4, 32, [40, 4, 31], [0, 4, 1]), (1, 77, 8, 1, 128, [200], None), (2, 130, 6, 2, 256, [130, 300], [130, 77]),
    (1, 3, 1, 1, 1024, [1500], None)]


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hq,Hkv,ps,ctx,lens", APPEND)
def test_append(fmt, dtype, B, T, Hq, Hkv, ps, ctx, lens):
    d = make(fmt, B, T, Hq, Hkv, ps, ctx, seed=T, dtype=dtype, lens=lens)
    want, g = oracle_append(d), to(d, device())
    announce(f"paged append {fmt} {dtype} B{B} T{T} Hkv{Hkv} page {ps} ctx {ctx} lens {lens}")
    append(g)
    same_pages(fmt, g["pages"], want)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("norm,rot", [(False, 64), (True, 0), (False, 0), (True, 256), (True, 8)])
def test_append_without_norm_and_other_rotations(fmt, norm, rot):
    d = make(fmt, 2, 3, 2, 2, 16, [10, 35], norm=norm, rot=rot)
    want, g = oracle_append(d), to(d, device())
    announce(f"paged append {fmt} norm {norm} rot {rot}")
    append(g)
    same_pages(fmt, g["pages"], want)


def test_bf16_append_is_bitwise_the_front_end():
    """The rows that attn_prep writes into a dense cache, through the table."""
    dev = device()
    B, T, ps, nb = 3, 37, 16, 5
    d = to(make("bf16", B, T, 8, 2, ps, [37, 50, 80], nb=nb), dev)
    kc, vc = (torch.zeros(B, 2, nb * ps, 256, dtype=torch.bfloat16, device=dev) for _ in range(2))
    announce("paged append bf16 against attn_prep")
    ops.attn_prep(d["y"], d["qw"], d["kw"], d["cos"], d["sin"], d["pos"], kc, vc, num_heads=8, num_kv_heads=2)
    append(d)
    k, v = ops.paged_kv_rows(d["pages"], d["table"], d["pos"], T)
    for b in range(B):
        at = int(d["pos"][b])
        assert torch.equal(k[b], kc[b, :, at:at + T]) and torch.equal(v[b], vc[b, :, at:at + T])


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_append_ties_zeros_and_values_that_are_not_finite(fmt):
    """Values on the border between two codes go to the even one, a zero group stays zero, and a group that holds an
    infinity or NaN reads back as NaN in 4 bits without touching its neighbours."""
    d = make(fmt, 1, 4, 1, 1, 16, [9], norm=False, rot=0)
    v = d["y"][..., -256:].view(1, 4, 4, 64)
    v[0, 0, 0] = torch.arange(64) % 14 * 1.5 - 10.5  # s = 1.5: ties and codes
    v[0, 0, 1] = torch.arange(64) % 29 * 0.375 - 5.25  # s = 0.75: multiples of s / 2
    v[0, 1, 2] = 0
    v[0, 2, 3, 5], v[0, 3, 0, 63] = math.inf, math.nan
    want, g = oracle_append(d), to(d, device())
    announce(f"paged append {fmt} ties")
    append(g)
    if fmt == "int4":
        same_pages(fmt, g["pages"], want)
    else:
        # equal values; which of the NaNs a NaN is rounded to is not stated
        assert torch.allclose(g["pages"][1].cpu().float(), want[1].float(), rtol=0, atol=0, equal_nan=True)
    _, rows = ops.paged_kv_rows(g["pages"], g["table"], g["pos"], 4)
    nan = rows[0, 0].isnan()
    if fmt == "int4":
        assert bool(nan[2, 192:].all()) and bool(nan[3, :64].all()) and int(nan.sum()) == 128
        assert torch.equal(rows[0, 0, 0, :64].cpu().float(), torch.round(d["y"][0, 0, -256:-192] / 1.5) * 1.5)


def test_append_scales_near_a_tie():
    """Among 65,536 groups of normed and rotated keys some scales lie so near the middle of two bf16 numbers that fp32 puts
    them onto it: rounded to fp32 and then to bf16, as stated, and not straight to bf16."""
    d = make("int4", 1, 4096, 4, 4, 256, [4096], seed=2)
    want, g = oracle_append(d), to(d, device())
    _, _, k, _ = columns(d["y"], 4, 4)
    at = torch.arange(4096)
    x = paged._norm(k, d["kw"], 1e-6)[0]
    x = paged.apply_partial_rope(x, d["cos"][at].double(), d["sin"][at].double())
    m = x.unflatten(-1, (4, 64)).abs().amax(-1) / 7
    near = m.float()
    assert int(((near.view(torch.int32) & 0xFFFF) == 0x8000).logical_and(near.double() != m).sum()) >= 1
    announce("paged append int4, scales near a tie")
    append(g)
    same_pages("int4", g["pages"], want)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_append_leaves_everything_else_alone(fmt):
    """Tokens past lens, at positions below 0 or past the table, and on entries that name no page are not written."""
    d = make(fmt, 4, 6, 2, 2, 16, [6, 30, 47, 20], lens=[0, 3, 6, 6], nb=3)
    d["pos"] = torch.tensor([0, -2, 45, 14], dtype=torch.int32)  # 45 .. 50 runs past 48; 14 .. 19 over two pages
    d["table"][3, 0], d["table"][1, 1] = -1, d["pages"][0].shape[0]
    want, g = oracle_append(d), to(d, device())
    announce(f"paged append {fmt} outside")
    append(g)
    same_pages(fmt, g["pages"], want)


ROWS = [(1, 1, 1, 16, [0], None), (2, 40, 2, 16, [0, 7], [40, 13]), (3, 130, 4, 64, [0, 100, 1], [130, 0, 64]),
        (1, 1000, 2, 256, [24], None)]


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("B,T,Hkv,ps,pos,lens", ROWS)
def test_rows(fmt, B, T, Hkv, ps, pos, lens):
    d = make(fmt, B, 1, Hkv, Hkv, ps, [p + T for p in pos])
    d["pos"], d["lens"] = torch.tensor(pos, dtype=torch.int32), None if lens is None else torch.tensor(lens, dtype=torch.int32)
    d["table"][0, 0] = -1 if B > 1 else d["table"][0, 0]
    want = paged.paged_rows(d["pages"], d["table"], d["pos"], T, d["lens"])
    g = to(d, device())
    announce(f"paged rows {fmt} B{B} T{T} Hkv{Hkv} page {ps} pos {pos}")
    got = ops.paged_kv_rows(g["pages"], g["table"], g["pos"], T, lens=g["lens"])
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b.bfloat16())


ATTN = [  # B, T, Hq, Hkv, page, contexts, lens
    (1, 1, 8, 2, 16, [1], None), (1, 1, 8, 2, 64, [31], None), (2, 1, 8, 2, 16, [33, 129], None),
    (3, 1, 4, 4, 32, [700, 1, 300], None), (2, 1, 8, 1, 128, [1000, 513], None), (1, 1, 16, 1, 64, [257], None),
    (2, 1, 6, 2, 256, [400, 90], None), (3, 4, 8, 2, 16, [200, 4, 37], [4, 4, 1]), (2, 5, 8, 2, 32, [600, 150], [5, 0]),
    (1, 7, 3, 1, 16, [100], None), (2, 33, 8, 2, 64, [33, 290], None), (1, 130, 4, 2, 128, [300], None),
    (2, 9, 24, 1, 64, [70, 9], [9, 3])]


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hq,Hkv,ps,ctx,lens", ATTN)
def test_attention(fmt, dtype, B, T, Hq, Hkv, ps, ctx, lens):
    d = make(fmt, B, T, Hq, Hkv, ps, ctx, seed=7 * T + B, dtype=dtype, lens=lens)
    g = to(d, device())
    announce(f"paged attention {fmt} {dtype} B{B} T{T} Hq{Hq} Hkv{Hkv} page {ps} ctx {ctx} lens {lens}")
    out = attend(g)
    print(f"worst error {check_attention(d, out):.3f} of its bound")
    assert torch.equal(out, attend(g))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("splits", [1, 2, 3, 8, 100])
@pytest.mark.parametrize("T", [1, 6])
def test_attention_splits(fmt, splits, T):
    """One run (no merge), few and as many as the capacity holds; rows shorter than a run, and runs past a row's end."""
    d = make(fmt, 3, T, 8, 2, 64, [1100, 130, T], seed=splits)
    g = to(d, device())
    announce(f"paged attention {fmt} T{T} splits {splits}")
    check_attention(d, attend(g, splits=splits))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("kw", [dict(norm=False), dict(rot=0), dict(rot=256, norm=False)])
def test_attention_plain_queries_no_gate_fp32_output(fmt, kw):
    d = make(fmt, 2, 2, 8, 2, 32, [90, 400], **kw)
    g = to(d, device())
    announce(f"paged attention {fmt} {kw}")
    check_attention(d, attend(g, gate=None, out_dtype=torch.float32, scale=0.05), gated=False, scale=0.05)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_attention_peaked_and_rising_scores(fmt):
    """Scores that rise along the keys by tens of nats and near one-hot rows: the running maximum moves in every run."""
    d = make(fmt, 1, 2, 8, 2, 64, [900], norm=False, rot=0)
    q, _, _, _ = columns(d["y"], 8, 2)
    q *= 12.0
    g = to(d, device())
    announce(f"paged attention {fmt} peaked")
    check_attention(d, attend(g))
    check_attention(d, attend(g, splits=1))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T", [1, 5])
def test_attention_masked_places_hold_anything(fmt, T):
    """Rows of the pages past a sequence's end, on entries that name no page, and (for earlier tokens of a call) of later
    tokens hold NaN and infinities: no output that does not attend to them changes."""
    d = make(fmt, 2, T, 8, 2, 16, [70, 41], seed=3)
    g = to(d, device())
    clean = attend(g)
    pages = tuple(None if p is None else p.clone() for p in d["pages"])
    for b in range(2):
        end = int(d["pos"][b]) + T
        for at in range(end, d["table"].shape[1] * 16):
            page, row = int(d["table"][b, at // 16]), at % 16
            for i in (0, 1) if fmt == "bf16" else (2, 3):
                pages[i][page, :, row] = math.nan if at % 2 else math.inf
        if T > 1:  # the last token's own value row: only it may see it
            at = end - 1
            page, row = int(d["table"][b, at // 16]), at % 16
            pages[1 if fmt == "bf16" else 3][page, :, row] = -math.inf
    spare = [p for p in range(d["pages"][0].shape[0]) if p not in d["table"].flatten().tolist()]
    for i in (0, 1) if fmt == "bf16" else (2, 3):
        pages[i][spare] = math.nan
    announce(f"paged attention {fmt} T{T} garbage in masked places")
    out = attend(dict(g, pages=tuple(None if p is None else p.to(g["y"].device) for p in pages)))
    keep = slice(0, T - 1) if T > 1 else slice(0, 1)
    assert torch.equal(out[:, keep], clean[:, keep])
    if T > 1:
        assert not bool(torch.isfinite(out[:, -1]).any())


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_attention_infinite_values_that_are_attended_to(fmt):
    """Plus and minus infinity and NaN in values (bf16): as sums of them; a key with NaN makes its readers NaN."""
    d = make(fmt, 1, 3, 2, 1, 16, [50], norm=False)
    if fmt == "bf16":
        v = d["pages"][1]
        page = int(d["table"][0, 2])  # keys 32 .. 47
        v[page, 0, 3, 10], v[page, 0, 4, 11], v[page, 0, 5, 12] = math.inf, -math.inf, math.nan
        v[page, 0, 3, 13], v[page, 0, 4, 13] = math.inf, -math.inf
        v[int(d["table"][0, 3]), 0, 0, 20] = math.inf  # key 48, the second token's own
    else:
        d["pages"][3][int(d["table"][0, 2]), 0, 3, 0] = math.nan
    announce(f"paged attention {fmt} infinities")
    out = attend(to(d, device())).float().cpu().view(3, 2, 256)
    if fmt == "bf16":
        assert bool((out[:, :, 10] == math.inf).all()) and bool((out[:, :, 11] == -math.inf).all())
        assert bool(out[:, :, [12, 13]].isnan().all())
        assert bool(torch.isfinite(out[0, :, 20]).all()) and bool((out[1:, :, 20] == math.inf).all())
        rest = [i for i in range(256) if i not in (10, 11, 12, 13, 20)]
        assert bool(torch.isfinite(out[..., rest]).all())
    else:
        assert bool(out[..., :64].isnan().all()) and bool(torch.isfinite(out[..., 64:]).all())


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T,splits", [(1, 1), (1, 3), (5, 1), (5, 3)])
def test_attention_scores_that_are_nan(fmt, T, splits):
    """A query that is NaN, and a key that is NaN and alone in its wave's last round: NaN for the heads they reach, and for
    no other."""
    n = 257 if T == 1 else 261  # key 256 is the only one of its 32 that the first token sees
    d = make(fmt, 3, T, 4, 2, 16, [n, n, n])
    d["y"][0, 0, 512 * 1 + 7] = math.nan  # row 0, token 0, head 1
    page, row = int(d["table"][1, 256 // 16]), 256 % 16  # row 1, key 256 of key head 1
    if fmt == "bf16":
        d["pages"][0][page, 1, row, 3] = math.nan
    else:
        d["pages"][2][page, 1, row, 0] = math.nan
    announce(f"paged attention {fmt} NaN scores T {T} splits {splits}")
    nan = attend(to(d, device()), splits=splits).view(3, T, 4, 256).isnan().cpu()
    assert bool((nan.any(-1) == nan.all(-1)).all())
    want = torch.zeros(3, T, 4, dtype=torch.bool)
    want[0, 0, 1] = True
    want[1, :, 2:] = True
    assert torch.equal(nan.any(-1), want)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T", [1, 4])
def test_attention_rows_that_see_nothing(fmt, T):
    """Positions below 0 and past the table, no tokens, and rows all of whose pages are missing give zeros."""
    d = make(fmt, 5, T, 8, 2, 16, [40, T, T, 30, 33], lens=[T] * 5, nb=3)
    d["pos"] = torch.tensor([40, -T, -1, 10, 48 - T + 1 if T > 1 else 48], dtype=torch.int32)
    d["lens"][0] = 0
    d["table"][3, 0] = 99999  # the row's only page
    d["table"][4, 1] = -5
    g = to(d, device())
    announce(f"paged attention {fmt} T{T} rows that see nothing")
    out = attend(g)
    check_attention(d, out)
    assert not bool(out[0].any()) and not bool(out[1].any())
    if T == 1:
        assert not bool(out[2:].any())


def test_sliced_table_and_a_page_shared_by_two_rows():
    """A table that is a slice of a wider one; a prefix page that two rows read."""
    d = make("int4", 2, 1, 8, 2, 16, [40, 45], nb=3)
    d["table"][1, 0] = d["table"][0, 0]
    g = to(d, device())
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=device())
    wide[:, 4:7] = g["table"]
    announce("paged attention, sliced table")
    out = attend(dict(g, table=wide[:, 4:7]))
    check_attention(d, out)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_a_serving_run(fmt):
    """As they are used together: a prompt in two chunks of different lengths per row, then steps of three drafts each
    checked by the attention of four tokens, refused drafts overwritten by the next step; against the oracle's pages."""
    dev = device()
    B, Hq, Hkv, ps, nb = 3, 8, 2, 16, 8
    d = make(fmt, B, 1, Hq, Hkv, ps, [1, 1, 1], nb=nb)
    ref_pages = tuple(None if p is None else p.clone() for p in d["pages"])
    g = to(d, dev)
    gen = torch.Generator().manual_seed(11)
    pos = torch.zeros(B, dtype=torch.int32)
    announce(f"paged serving run {fmt}")
    for step, (T, lens) in enumerate([(23, [23, 9, 16]), (40, [40, 1, 33]), (4, [4, 4, 4]), (4, [4, 1, 3]), (4, [2, 4, 4])]):
        y = torch.randn(B, T, 2 * (Hq + Hkv) * 256, generator=gen)
        lens = torch.tensor(lens, dtype=torch.int32)
        cur = dict(d, y=y, pos=pos, lens=lens, pages=ref_pages)
        ref_pages = oracle_append(cur)
        cur["pages"] = ref_pages
        gcur = dict(g, y=y.to(dev), pos=pos.to(dev), lens=lens.to(dev))
        append(gcur)
        same_pages(fmt, g["pages"], ref_pages)
        cur["pages"] = tuple(None if p is None else p.cpu() for p in g["pages"])
        check_attention(cur, attend(gcur))
        if step < 2:
            pos = pos + lens
        else:  # the target keeps some of the drafts
            V = 97
            logits, u = torch.randn(B, T, V, generator=gen), torch.rand(B, T, generator=gen)
            ids = logits[:, :-1].argmax(-1).int()
            n, tok = ops.verify_drafts(logits.to(dev), ids.to(dev), u.to(dev), lens=(lens - 1).to(dev))
            rn, rtok = paged.verify_drafts(logits, ids, u, lens=lens - 1)
            assert torch.equal(n.cpu(), rn) and torch.equal(tok.cpu(), rtok)
            pos = pos + rn + 1


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_captured_step_follows_the_positions(fmt):
    """Append and attention in a HIP graph, replayed with eager work between: each replay equals the eager calls."""
    dev = device()
    d = make(fmt, 3, 2, 8, 2, 16, [300, 20, 100], lens=[2, 1, 2], nb=24)
    g = to(d, dev)
    eager = dict(g, pages=tuple(None if p is None else p.clone() for p in g["pages"]), pos=g["pos"].clone(),
                 lens=g["lens"].clone(), y=g["y"].clone())
    announce(f"paged capture {fmt}")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append(g)
        out = attend(g)
    for step in range(4):
        y = torch.randn(g["y"].shape, generator=torch.Generator().manual_seed(step)).to(dev)
        for x in (g, eager):
            x["y"].copy_(y)
        graph.replay()
        append(eager)
        want = attend(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(g["pages"], eager["pages"]):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for x in (g, eager):
            x["pos"] += x["lens"]


def test_another_stream_and_calls_side_by_side():
    """Two streams at once, each with its own cache: the results of calls one after the other."""
    dev = device()
    ds = [to(make("int4", 2, 1, 8, 2, 64, [900, 800], seed=s), dev) for s in range(2)]
    want = [attend(d) for d in ds]
    torch.cuda.synchronize()
    announce("paged attention on two streams")
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attend(ds[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_pages_past_32_bits(fmt):
    """Pages more than 2^32 bytes into the pool (and, in bf16, 2^31 elements)."""
    dev = device()
    d = make(fmt, 2, 3, 4, 2, 64, [150, 70], lens=[3, 2])
    nb = d["table"].shape[1]
    row = 512 if fmt == "bf16" else 128
    n = (1 << 32) // (2 * 64 * row) + 2 * nb + 2
    announce(f"paged {fmt} pages past 32 bits")
    want_pages = oracle_append(d)
    g = to(d, dev)
    small = g["pages"]
    m = small[0].shape[0]
    big = tuple(None if p is None else torch.empty(n, *p.shape[1:], dtype=p.dtype, device=dev) for p in small)
    for p, q in zip(big, small):
        if p is not None:
            p[n - m:] = q
    far = dict(g, pages=big, table=g["table"] + (n - m))
    append(far)
    same_pages(fmt, [None if p is None else p[n - m:] for p in big], want_pages)
    after = dict(d, pages=tuple(None if p is None else p[n - m:].cpu() for p in big))
    check_attention(after, attend(far))
    k, v = ops.paged_kv_rows(big, far["table"], torch.zeros_like(far["pos"]), 70)
    wk, wv = paged.paged_rows(after["pages"], d["table"], torch.zeros_like(d["pos"]), 70)
    assert torch.equal(k.cpu().double(), wk.bfloat16().double()) and torch.equal(v.cpu().double(), wv.bfloat16().double())


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_attention_over_a_prompt(fmt):
    """A prompt's own tokens from position 0 on, ragged, six heads over two."""
    d = make(fmt, 2, 700, 6, 2, 64, [700, 333], lens=[700, 333])
    announce(f"paged attention {fmt} prompt of 700")
    check_attention(d, attend(to(d, device())))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T,Hq,lens", [(9, 4, [9, 4]), (12, 4, [12, 1]), (17, 3, [0, 17]), (13, 5, [13, 13])])
def test_attention_rows_over_three_to_five_tiles(fmt, T, Hq, lens):
    """36, 48, 51 and 65 query rows of one key head, over keys in one run and in several."""
    d = make(fmt, 2, T, Hq, 1, 16, [600, 40], lens=lens)
    announce(f"paged attention {fmt} T {T} heads {Hq} lens {lens}")
    g = to(d, device())
    for splits in (0, 1, 4):
        check_attention(d, attend(g, splits=splits))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("B,T,nb", [(2, 1, 2), (2, 1, 3), (2, 1, 4), (2, 6, 2), (2, 6, 3), (40, 1, 3), (40, 6, 4), (70, 1, 2),
                                    (130, 2, 3)])
def test_attention_over_tables_of_two_to_four_rounds(fmt, B, T, nb):
    """Tables of 256 to 512 keys for few rows and many: one block of eight waves, of four, or several and their merge."""
    ctx = [128 * nb - (37 * b) % (128 * nb - T) for b in range(B)]
    d = make(fmt, B, T, 4, 2, 128, ctx, nb=nb)
    announce(f"paged attention {fmt} B {B} T {T} table of {128 * nb}")
    g = to(d, device())
    out = attend(g)
    check_attention(d, out)
    if B == 2:
        check_attention(d, attend(g, splits=1))


@pytest.mark.parametrize("T", [1, 6])
def test_attention_more_splits_than_rounds(T):
    d = make("int4", 2, T, 8, 2, 32, [3000, 130])
    announce(f"paged attention T {T}, 5000 splits")
    check_attention(d, attend(to(d, device()), splits=5000))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T", [1, 6])
def test_attention_over_four_million_keys(fmt, T):
    """A table that names one page 4096 times: the page's keys, each as often as a token sees it. The splits make a block's
    run 8192 keys (the n of the bound's sums)."""
    ps, blocks = 1024, 4096
    d = make(fmt, 1, T, 4, 2, ps, [T], norm=False, rot=0, nb=1)
    cap = ps * blocks
    d["pos"] = torch.tensor([cap - T], dtype=torch.int32)
    q, gate, _, _ = columns(d["y"], 4, 2)
    page = int(d["table"][0, 0])
    g = to(d, device())
    g["table"] = g["table"].expand(1, blocks).contiguous()
    announce(f"paged attention {fmt} T {T} over 4194304 keys")
    out = attend(g, splits=512).cpu().double().view(T, 4, 256)
    k, v = (paged.row_values(d["pages"][i][page], None if d["pages"][2 + i] is None else d["pages"][2 + i][page], w)
            for i, w in ((0, "k"), (1, "v")))  # [Hkv, page, 256]
    sv = torch.zeros_like(v) if d["pages"][3] is None else d["pages"][3][page].double().repeat_interleave(64, -1)
    for t in range(T):
        often = blocks - (torch.arange(ps) > ps - T + t).double()
        for h in range(4):
            w = often * torch.exp(k[h // 2] @ q[0, t, h].double() / 16)
            w = w / w.sum()
            sg = torch.sigmoid(gate[0, t, h].double())
            ref, amp, step = (w @ v[h // 2]) * sg, (w @ v[h // 2].abs()) * sg, (w @ sv[h // 2]) * sg
            prod = float((k[h // 2].abs() @ q[0, t, h].double().abs()).max()) / 16
            q_off = 2.0 ** -15 + (2.0 ** -12 if fmt == "int4" else 0)
            bound = (2.0 ** -8 + 2 * q_off * prod + 2.0 ** -16) * amp + (8192 / 32 + 16) * 2.0 ** -19 * step \
                + (2.0 ** -8 + 2.0 ** -20) * ref.abs() * (1 + 2.0 ** -7)
            assert float(((out[t, h] - ref).abs() / bound).max()) <= 1


def test_append_of_tiny_values_without_eps():
    """Squares below the smallest normal number, and an eps of 0: the codes of 64 bits all the same."""
    d = make("int4", 1, 40, 2, 2, 16, [40])
    scale = 10.0 ** -torch.arange(40).float()[:, None]
    d["y"] = d["y"] * scale
    _, _, k, v = columns(d["y"], 2, 2)
    pages = tuple(p.clone() for p in d["pages"])
    paged.paged_append(k, v, pages, d["table"], d["pos"], d["cos"], d["sin"], d["lens"], d["kw"], eps=0.0)
    g = to(d, device())
    _, _, k, v = columns(g["y"], 2, 2)
    announce("paged append of tiny values")
    ops.paged_kv_append_(k, v, g["pages"], g["table"], g["pos"], g["cos"], g["sin"], k_norm_w=g["kw"], eps=0.0)
    same_pages("int4", g["pages"], pages)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_calls_through_the_dispatcher(fmt):
    """torch.ops, a dispatch mode and inference mode give what the plain calls give; meta tensors the shapes."""
    from torch.utils._python_dispatch import TorchDispatchMode
    dev = device()
    g = to(make(fmt, 2, 3, 8, 2, 16, [70, 33], lens=[3, 2]), dev)
    announce(f"paged calls through the dispatcher {fmt}")
    other = dict(g, pages=tuple(None if p is None else p.clone() for p in g["pages"]))
    append(g)
    want = attend(g)
    rows = ops.paged_kv_rows(g["pages"], g["table"], g["pos"], 3, lens=g["lens"])
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Record():
        append(other)
        got = attend(other)
        got_rows = ops.paged_kv_rows(other["pages"], g["table"], g["pos"], 3, lens=g["lens"])
    assert {"q35.paged_kv_append_.default", "q35.gated_attn_paged.default", "q35.paged_kv_rows.default"} <= set(seen)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(got_rows, rows))
    for a, b in zip(g["pages"], other["pages"]):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with torch.inference_mode():
        assert torch.equal(attend(g), want)
    meta = {k: v.to("meta") if torch.is_tensor(v) else v for k, v in g.items()}
    meta["pages"] = tuple(None if p is None else p.to("meta") for p in g["pages"])
    out = attend(meta)
    assert out.shape == want.shape and out.dtype == want.dtype and out.device.type == "meta"


def test_graphs_on_two_streams_share_nothing():
    """Two captured steps replayed at once on two streams, several times."""
    dev = device()
    gs, outs, want = [], [], []
    announce("paged graphs on two streams")
    for s in range(2):
        g = to(make("int4", 2, 2, 8, 2, 64, [3000, 2500], seed=s), dev)
        want.append(attend(g))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attend(g)
        gs.append((graph, g))
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for (graph, _), s in zip(gs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T,lens", [(1, None), (3, [3, 0]), (40, [40, 17])])
def test_layer(fmt, T, lens):
    """The attention layer over pages, with an o_proj of 1 so that its output is the attention's: its projection's columns
    through the oracle. Then with a residual, added in place."""
    dev = device()
    d = make(fmt, 2, T, 2, 1, 32, [T + 30, (lens or [T] * 2)[1] + 5], lens=lens)
    g = torch.Generator().manual_seed(T)
    p = {n: (torch.randn(w, 512, generator=g) * 0.05).to(dev) for n, w in (("q_proj", 1024), ("k_proj", 256), ("v_proj", 256))}
    p["o_proj"] = torch.eye(512, device=dev)
    p["q_norm"], p["k_norm"] = d["qw"].to(dev), d["kw"].to(dev)
    x = torch.randn(2, T, 512, generator=g).to(dev)
    gpu = to(d, dev)
    announce(f"paged attention layer {fmt} T {T} lens {lens}")
    out = layers.gated_attention_layer_paged(x, p, gpu["pages"], gpu["table"], gpu["pos"], lens=gpu["lens"])
    d["y"] = layers.linear(x, layers.attn_in_weight(p)).cpu()
    d["cos"], d["sin"] = (t.cpu() for t in layers.rope_tables(d["table"].shape[1] * 32, 64, 1e7, dev))
    want = oracle_append(d)
    same_pages(fmt, gpu["pages"], want)
    d["pages"] = tuple(None if t is None else t.cpu() for t in gpu["pages"])
    check_attention(d, out)
    res = torch.randn(2, T, 512, generator=g).to(dev)
    got = layers.gated_attention_layer_paged(x, p, gpu["pages"], gpu["table"], gpu["pos"], lens=gpu["lens"],
                                             residual=res.clone(), fixed_order=True)
    assert torch.equal(got, res + out)


def test_layer_in_int8_against_the_dense_layer():
    """int8 weights, a prompt and then steps of one token: the dense layer's outputs but for the two attentions' roundings
    (2^-8 a weight and 2^-8 an output of each, over sum w |v|, carried through |o_proj|)."""
    dev = device()
    g = torch.Generator().manual_seed(5)
    H, Hq, Hkv = 512, 4, 2
    p = {}
    for n, (r, c) in dict(q_proj=(Hq * 512, H), k_proj=(Hkv * 256, H), v_proj=(Hkv * 256, H), o_proj=(H, Hq * 256)).items():
        q = torch.randint(-127, 128, (r, c), generator=g, dtype=torch.int8)
        s = torch.full((r, c // 128), 0.001)
        p[n + ".q"], p[n + ".s"] = q.to(dev), s.to(dev)
        p[n] = (q.float() * 0.001).to(dev)
    p["q_norm"], p["k_norm"] = (0.1 * torch.randn(256, generator=g).to(dev) for _ in range(2))
    announce("paged attention layer in int8 against the dense one")
    B, n, blocks = 2, 64, 2
    kc, vc = (torch.zeros(B, Hkv, 128, 256, dtype=torch.bfloat16, device=dev) for _ in range(2))
    pages = ops.kv_pages(B * blocks, Hkv, 64, dev)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=dev)
    at = 0
    for T in (n, 1, 1, 5):
        x = torch.randn(B, T, H, generator=g).to(dev)
        pos = torch.full((B,), at, dtype=torch.int32, device=dev)
        got = layers.gated_attention_layer_paged(x, p, pages, table, pos)
        want = layers.gated_attention_layer(x, p, kc, vc, at if T == n else pos)
        k, v = ops.paged_kv_rows(pages, table, torch.zeros_like(pos), 128)
        # (bitwise where both read the projection in fp32, and one rounding apart otherwise)
        assert bool(((k.float() - kc.float()).abs() <= kc.float().abs() * 2.0 ** -7 + 1e-6).all())
        vmax = vc[:, :, :at + T].abs().amax((2, 3)).float().amax(1)  # >= sum w |v|
        bound = (2 * (2.0 ** -8 + 2.0 ** -8) + 2.0 ** -12) * vmax[:, None, None] * p["o_proj"].abs().sum(-1)
        assert bool(((got - want).abs() <= bound).all())
        at += T


def test_refusals_on_the_device():
    dev = device()
    d = to(make("int4", 1, 1, 8, 2, 16, [5]), dev)
    q, gate, k, v = columns(d["y"], 8, 2)
    kp, vp, ks, vs = d["pages"]
    a = (d["table"], d["pos"], d["cos"], d["sin"])
    announce("paged refusals")
    from q35hip import Q35Error
    for call in (lambda: ops.gated_attention_paged(q, gate, (kp, vp), *a),                      # no scales
                 lambda: ops.gated_attention_paged(q, gate[:, :, :4], d["pages"], *a),          # gate unlike q
                 lambda: ops.gated_attention_paged(q.half(), None, d["pages"], *a),             # dtype
                 lambda: ops.gated_attention_paged(q[..., :128], None, d["pages"], *a),         # head dim
                 lambda: ops.gated_attention_paged(q, None, d["pages"], d["table"].long(), *a[1:]),
                 lambda: ops.gated_attention_paged(q, None, d["pages"], d["table"].cpu(), *a[1:]),
                 lambda: ops.gated_attention_paged(q, None, d["pages"], d["table"], d["pos"], d["cos"][:8], d["sin"][:8]),
                 lambda: ops.gated_attention_paged(q[:, :, :7], None, d["pages"], *a),          # 7 heads over 2
                 lambda: ops.paged_kv_append_(k, v[..., :0], d["pages"], *a),
                 lambda: ops.paged_kv_append_(k, v.bfloat16(), d["pages"], *a),
                 lambda: ops.paged_kv_append_(k[:, :, :1], v[:, :, :1], d["pages"], *a),
                 lambda: ops.paged_kv_append_(k, v, (kp.float(), vp.float(), ks, vs), *a),
                 lambda: ops.paged_kv_append_(k, v, (kp, vp, ks.float(), vs.float()), *a),
                 lambda: ops.paged_kv_rows(d["pages"], d["table"], d["pos"].long(), 3)):
        with pytest.raises(Q35Error):
            call()
    assert ops.gated_attention_paged(q[:, :0], None, d["pages"], *a).shape == (1, 0, 2048)
