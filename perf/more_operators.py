"""The operators of a step that samples many continuations of one prompt, as cases that can be timed and compared.

A case is a dict of plain values with a "kind":

  attn     gated causal grouped attention over a paged KV cache whose sequences share their first pages (one prompt, many
           continuations), the shared keys read once for all of them
  sample   one token per row drawn from softmax(logits / temperature) cut by top-k, top-p and min-p, from given random
           numbers; with the probabilities it was drawn from where a draft model hands them on
  filter   the logits of several positions per row with what the same cuts drop at -inf (what a check of drafts takes)
  proj     a projection in 8-bit integers: residual rows normed with (1 + w), quantised with one scale a row, times int8
           weights with one scale an output channel
  gate     the same with the gate and up projections interleaved and silu(gate) * up as the result
  down     activations quantised with one scale a row, times int8 weights

Order of the cuts: temperature, then the top_k most likely tokens (0: all), then of these the most likely whose sum ahead
of them is below top_p of these tokens' sum, then those of at least min_p of the most likely one's probability; the most
likely token always stays, ties go to the lowest index, temperature 0 is the argmax. The token is the lowest index whose
running sum over the kept ones exceeds u of the whole.

Rows in 8 bits: s = fp32(max|x| / 127), codes rint(x / s) (half to even), both of the exact x.

Pages as in perf/operators.py: k, v [pages, Hkv, page size, 256] bf16, or 4 bits with one bf16 scale per group of 64 dims:
codes [pages, Hkv, page size, 128] bytes, scales [pages, Hkv, page size, 4]. A code n stands for (n - 8) s. Bytes of a row,
in nibbles (low first): keys hold dims 64 g + 16 a + 8 u + j at nibble 64 a + 16 g + 8 u + j (g, a < 4, u < 2, j < 8);
values dims 64 g + 4 c + e at nibble 16 c + 4 g + e (g, e < 4, c < 16).

Sizes are those of the Qwen3.5-0.8B shape (8 query and 2 key heads of 256, rotation of 64 dims, hidden 1024, 3584
neurons, vocabulary 151,936) and of serving batches around it. Three rows are a steering experiment (boosted, as it is,
suppressed).
"""
import math
import os
import sys

import torch

own = False
if os.path.join(os.getcwd(), "duo-mech-interp_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "duo-mech-interp_amd"))

DEV = "cuda"
D, ROT, THETA, EPS, VOCAB = 256, 64, 1e7, 1e-6, 151936
HALF, GROUP, NG = ROT // 2, 64, D // 64
INF = math.inf


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one token of three steered rows behind one prompt held in 4 bits (layers below the steered one)
        dict(name="attn_step_r3", kind="attn", fmt="int4", B=3, T=1, shared=2048, own=64, page=64, hq=8, hkv=2, q="f32"),
        # one token of 32 samples of a long prompt, bf16 pages
        dict(name="attn_step_b32", kind="attn", fmt="bf16", B=32, T=1, shared=8192, own=500, page=64, hq=8, hkv=2, q="f32"),
        # four drafted tokens each of 64 answers about one long document held in 4 bits
        dict(name="attn_drafts_b64", kind="attn", fmt="int4", B=64, T=4, shared=32768, own=1000, page=128, hq=8, hkv=2,
             q="f32"),
        # the next token of three steered rows
        dict(name="sample_r3", kind="sample", B=3, V=VOCAB, temp=0.7, top_k=20, top_p=0.95, min_p=0.0, probs=False),
        # a draft model's tokens for a serving batch, every request with its own settings, and their probabilities
        dict(name="sample_mixed_b32", kind="sample", B=32, V=VOCAB, temp=-1.0, top_k=0, top_p=1.0, min_p=0.0, probs=True),
        # a large batch, nucleus sampling alone
        dict(name="sample_b256", kind="sample", B=256, V=VOCAB, temp=1.0, top_k=0, top_p=0.9, min_p=0.0, probs=False),
        # the target's logits behind up to four drafts of one row
        dict(name="filter_r1", kind="filter", B=1, P=5, V=VOCAB, temp=0.7, top_k=50, top_p=0.95, min_p=0.0),
        # the same for a serving batch
        dict(name="filter_b32", kind="filter", B=32, P=5, V=VOCAB, temp=0.8, top_k=0, top_p=0.95, min_p=0.02),
        # the attention's input projections of a decode step of 32 samples
        dict(name="proj_b32", kind="proj", M=32, N=5120, K=1024),
        # one row's down projection of a short prompt: an odd number of tokens
        dict(name="down_333", kind="down", M=333, N=1024, K=3584),
        # the neurons of a prompt on three rows
        dict(name="gate_3x2048", kind="gate", M=6144, N=7168, K=1024),
        # down projections of a large prefill batch
        dict(name="down_16k", kind="down", M=16384, N=1024, K=3584),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cuts(rng):
    return dict(temp=rng.choice([0.3, 0.7, 1.0, 1.3]), top_k=rng.choice([0, 0, _log(rng, 1, 500)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
                min_p=rng.choice([0.0, 0.0, round(math.exp(rng.uniform(math.log(0.001), math.log(0.3))), 4)]))


def draw(rng):
    kind = rng.choice(["attn", "attn", "sample", "filter", "proj", "gate", "down"])
    if kind == "attn":
        hq, hkv = rng.choice([(8, 2), (8, 2), (8, 2), (4, 4), (8, 1), (16, 2), (6, 2)])
        T = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 64)])
        B = _log(rng, 1, max(1, min(128, 1280 // (T * hq))))
        page = rng.choice([16, 32, 64, 128, 256])
        shared = _log(rng, 16, 32768) // page * page
        return dict(kind=kind, fmt=rng.choice(["bf16", "int4"]), B=B, T=T, shared=shared, own=T + _log(rng, 1, 1500),
                    page=page, hq=hq, hkv=hkv, q=rng.choice(["f32", "f32", "bf16"]))
    if kind == "sample":
        V = _log(rng, 100, VOCAB)
        return dict(dict(kind=kind, B=_log(rng, 1, 256), V=V, probs=rng.random() < 0.4), **_cuts(rng))
    if kind == "filter":
        B, P = _log(rng, 1, 32), rng.randint(1, 5)
        return dict(dict(kind=kind, B=B, P=P, V=_log(rng, 100, VOCAB)), **_cuts(rng))
    K = 64 * rng.choice([4, 8, 9, 16, 16, 25, 32, 56])
    N = {"gate": 2 * _log(rng, 64, 3584), "proj": _log(rng, 64, 8224), "down": _log(rng, 64, 2048)}[kind]
    return dict(kind=kind, M=_log(rng, 1, min(16384, 45_000_000_000 // (N * K))), N=N, K=K)


# ---------------------------------------------------------------- inputs
def _pool(g, c, n_pages):
    shape = (n_pages, c["hkv"], c["page"], D)
    k, v = (torch.randn(shape, generator=g, device=DEV) for _ in range(2))
    if c["fmt"] == "bf16":
        return k.bfloat16(), v.bfloat16(), None, None
    out = []
    for x in (k, v):
        x = x.unflatten(-1, (NG, GROUP))
        s = (x.abs().amax(-1) / 7).bfloat16()
        n = (x / s.float().unsqueeze(-1)).round().clamp(-7, 7).to(torch.uint8) + 8
        out.append((n.flatten(-2), s))
    (kc, ks), (vc, vs) = out
    kc = kc.unflatten(-1, (4, 4, 2, 8)).transpose(-4, -3).flatten(-4)
    vc = vc.unflatten(-1, (4, 16, 4)).transpose(-3, -2).flatten(-3)
    return kc[..., 0::2] | (kc[..., 1::2] << 4), vc[..., 0::2] | (vc[..., 1::2] << 4), ks, vs


def _tables(n):
    inv = 1.0 / (THETA ** (torch.arange(0, ROT, 2, dtype=torch.int64).float() / ROT))
    a = torch.arange(n, dtype=torch.float32)[:, None] * inv[None, :]
    return a.cos().to(DEV), a.sin().to(DEV)


def _logits(g, rows, V):
    """Rows from sure to undecided: likelihoods that fall with a power of the token's rank, and noise on them."""
    a = 1.1 + 1.9 * torch.rand(rows, 1, generator=g, device=DEV)
    rank = torch.rand(rows, V, generator=g, device=DEV).argsort(-1).float()
    return -a * torch.log(2 + rank) + 0.6 * torch.randn(rows, V, generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c, s = case, dict(case=case)
    kind = c["kind"]
    if kind in ("sample", "filter"):
        B, V = c["B"], c["V"]
        rows = B * c.get("P", 1)
        x = _logits(g, rows, V)
        s["x"] = x if kind == "sample" else x.view(B, c["P"], V)
        s["u"] = torch.rand(B, generator=g, device=DEV)
        s["cuts"] = {k: c[k] for k in ("top_k", "top_p", "min_p")}
        s["cuts"]["temperature"] = c["temp"]
        if c["temp"] < 0:  # each request's own settings; some rows greedy, some without a cut
            def pick(values, dtype=torch.float32):
                at = torch.randint(0, len(values), (B,), generator=g, device=DEV)
                return torch.tensor(values, device=DEV, dtype=dtype)[at]
            s["cuts"] = dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.2]), top_k=pick([0, 0, 20, 50], torch.int32),
                             top_p=pick([1.0, 0.8, 0.9, 0.95]), min_p=pick([0.0, 0.0, 0.05]))
        return s
    if kind == "attn":
        B, T, ps = c["B"], c["T"], c["page"]
        n_sh, n_own = c["shared"] // ps, -(-c["own"] // ps)
        nb = n_sh + n_own
        total = n_sh + B * n_own + 3
        s["pages"] = _pool(g, c, total)
        at = torch.randperm(total, generator=g, device=DEV).int()
        s["table"] = torch.cat([at[:n_sh].expand(B, n_sh), at[n_sh:n_sh + B * n_own].view(B, n_own)], 1).contiguous()
        s["blocks"] = n_sh
        # continuations of unequal length; the new tokens are their last ones
        own_n = c["own"] - torch.randint(0, c["own"] // 2 + 1, (B,), generator=g, device=DEV)
        own_n[0] = c["own"]
        lens = torch.full((B,), T, device=DEV)
        if 1 < T < 16:
            lens = torch.randint(1, T + 1, (B,), generator=g, device=DEV)
        lens = torch.minimum(lens, own_n)
        s["lens"], s["pos"] = lens.int(), (c["shared"] + own_n - lens).int()
        s["cos"], s["sin"] = _tables(nb * ps)
        y = torch.randn(B, T, 2 * (c["hq"] + c["hkv"]) * D, generator=g, device=DEV) * 0.7
        y = y if c["q"] == "f32" else y.bfloat16()
        # columns of the fused projection output: [q | gate] per query head, then k, then v
        qg = y[..., :2 * c["hq"] * D].unflatten(-1, (c["hq"], 2 * D))
        s["q"], s["gate"] = qg[..., :D], qg[..., D:]
        s["q_norm"] = 0.1 * torch.randn(D, generator=g, device=DEV)
        return s
    M, N, K = c["M"], c["N"], c["K"]
    x = torch.randn(M, K, generator=g, device=DEV)
    if kind == "down":  # activations of gated neurons: a few large ones in a row
        x = torch.nn.functional.silu(1.5 * x) * torch.randn(M, K, generator=g, device=DEV)
    else:  # a residual stream: a few channels much larger than the others
        x = x * torch.where(torch.rand(K, generator=g, device=DEV) < 0.01, 12.0, 1.0)
        s["norm"] = 0.1 * torch.randn(K, generator=g, device=DEV)
    s["x"] = x
    w = 0.02 * torch.randn(N, K, generator=g, device=DEV)
    s["ws"] = w.abs().amax(1) / 127
    s["w"] = (w / s["ws"][:, None]).round().clamp(-127, 127).to(torch.int8)
    return s


# ---------------------------------------------------------------- plain forms
def _values(b, sc, which):
    """fp32 values of packed codes [..., 128] with scales [..., 4]."""
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    if which == "k":
        n = n.unflatten(-1, (4, 4, 2, 8)).transpose(-4, -3).flatten(-4)
    else:
        n = n.unflatten(-1, (16, 4, 4)).transpose(-3, -2).flatten(-3)
    return ((n.float() - 8).unflatten(-1, (NG, GROUP)) * sc.float().unsqueeze(-1)).flatten(-2)


def _attn(s):
    c = s["case"]
    B, T, hq, hkv, ps = c["B"], c["T"], c["hq"], c["hkv"], c["page"]
    G, P = hq // hkv, s["blocks"] * ps
    t = torch.arange(T, device=DEV)
    at, ok = s["pos"].long()[:, None] + t, t < s["lens"][:, None]
    at = at.where(ok, torch.zeros_like(at))
    q = s["q"].float()
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * (1 + s["q_norm"])
    co, si = s["cos"][at].unsqueeze(2), s["sin"][at].unsqueeze(2)
    a, b, rest = q.split([HALF, HALF, D - ROT], -1)
    q = torch.cat([a * co - b * si, b * co + a * si, rest], -1) * D ** -0.5
    q = q.unflatten(2, (hkv, G)).permute(0, 2, 1, 3, 4).reshape(B, hkv, T * G, D)

    def kv(table):  # [..., blocks] -> k, v [..., Hkv, keys, 256]
        x = [None if p is None else p[table.long()].transpose(-4, -3).flatten(-3, -2) for p in s["pages"]]
        if c["fmt"] == "int4":
            return _values(x[0], x[2], "k"), _values(x[1], x[3], "v")
        return x[0].float(), x[1].float()
    # the shared keys once, for the rows of all sequences together
    k0, v0 = kv(s["table"][0, :s["blocks"]])
    k1, v1 = kv(s["table"][:, s["blocks"]:])
    qa = q.transpose(0, 1).reshape(hkv, B * T * G, D)
    x0 = torch.matmul(qa, k0.transpose(-1, -2))
    x0 = x0.view(hkv, B, T * G, P).transpose(0, 1)
    x1 = torch.matmul(q, k1.transpose(-1, -2))
    x = torch.cat([x0, x1], -1).view(B, hkv, T, G, -1)
    see = (torch.arange(x.shape[-1], device=DEV) <= at[:, :, None]) & ok[:, :, None]
    x = x.masked_fill(~see[:, None, :, None], -INF)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-3e38))
    z = p.sum(-1)
    p = p.flatten(2, 3)
    o = torch.matmul(p[..., :P].transpose(0, 1).reshape(hkv, B * T * G, P), v0).view(hkv, B, T * G, D).transpose(0, 1)
    o = o + torch.matmul(p[..., P:], v1)
    o = o.view(B, hkv, T, G, D) / torch.where(z > 0, z, torch.ones_like(z))[..., None]
    o = o.permute(0, 2, 1, 3, 4).reshape(B, T, hq, D) / (1 + torch.exp(-s["gate"].float()))
    return o.flatten(2).to(torch.bfloat16)


def _kept(x, cuts):
    """x [rows, V] -> the tokens from the most likely one down, their weights in 64 bits (the first one's is 1), and which of
    them are kept (the first ones)."""
    def col(v):
        return v[:, None] if torch.is_tensor(v) else torch.full((x.shape[0], 1), v, device=DEV)
    t, k, p, m = (col(cuts[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    d = xs.double()
    w = torch.exp((d - d[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)).double())
    rank = torch.arange(x.shape[1], device=DEV)
    keep = (k <= 0) | (rank < k)
    w0 = w * keep
    ahead = w0.cumsum(-1) - w0
    keep = keep & ((p >= 1) | (ahead < p.double() * w0.sum(-1, keepdim=True))) & (w >= m.double())
    return order, w, torch.where(t > 0, keep | (rank == 0), rank == 0)


def _sample(s):
    c = s["case"]
    order, w, keep = _kept(s["x"], s["cuts"])
    w = w * keep
    run = w.cumsum(-1)
    over = run > s["u"].double()[:, None] * run[:, -1:]
    at = torch.where(over.any(-1), over.int().argmax(-1), keep.sum(-1) - 1)
    token = order.gather(1, at[:, None])[:, 0].int()
    return (token, torch.zeros_like(w).scatter(1, order, w / run[:, -1:]).float()) if c["probs"] else token


def _filter(s):
    x = s["x"]
    order, _, keep = _kept(x.flatten(0, 1), s["cuts"])
    return torch.where(torch.zeros_like(keep).scatter(1, order, keep).view_as(x), x, torch.full_like(x, -INF))


def _codes(x):
    """x [M, K] in 64 bits (a code is a rounding decision: there it hangs on no order of a sum) -> codes and scales."""
    sc = (x.abs().amax(-1, keepdim=True) / 127).float()
    d = sc.double()
    return torch.where(d > 0, x / d, torch.zeros_like(x)).round().clamp(-127, 127).float(), sc


def _product(s):
    c = s["case"]
    x = s["x"].double()
    if c["kind"] != "down":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + s["norm"].double())
    q, sc = _codes(x)
    y = torch.matmul(q, s["w"].float().T) * sc * s["ws"]
    if c["kind"] == "gate":
        a, b = y[:, 0::2], y[:, 1::2]
        y = a / (1 + torch.exp(-a)) * b
    return y


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"attn": _attn, "sample": _sample, "filter": _filter}.get(kind, _product)(s)
    from q35hip import ops
    if kind == "attn":
        return ops.gated_attention_paged_shared(s["q"], s["gate"], s["pages"], s["table"], s["pos"], s["cos"], s["sin"],
                                                s["blocks"], lens=s["lens"], q_norm_w=s["q_norm"], eps=EPS)
    if kind == "sample":
        return ops.sample_tokens(s["x"], s["u"], want_probs=c["probs"], **s["cuts"])
    if kind == "filter":
        return ops.filter_logits(s["x"], **s["cuts"])
    rows = ops.quantize_rows(s["x"]) if kind == "down" else ops.add_rmsnorm_i8_(s["x"], None, s["norm"], EPS)
    return ops.gemm_i8(rows, s["w"], s["ws"], epilogue="swiglu" if kind == "gate" else "store")


# ---------------------------------------------------------------- work
def work(case):
    c = case
    kind = c["kind"]
    if kind in ("sample", "filter"):
        n = c["B"] * c.get("P", 1) * c["V"]
        return dict(bytes=4 * n * (2 if kind == "filter" or c["probs"] else 1), flops=3 * n)
    if kind == "attn":
        row = 2 * c["hkv"] * (2 * D if c["fmt"] == "bf16" else D // 2 + 2 * NG)  # a token's keys and values
        B, T, own_n = c["B"], c["T"], 0.75 * c["own"]  # continuations are up to half shorter than the longest
        new = B * (T if T == 1 or T >= 16 else (T + 1) / 2)
        el = 4 if c["q"] == "f32" else 2
        return dict(bytes=(c["shared"] + B * own_n) * row + new * c["hq"] * D * (2 * el + 2),
                    flops=4 * new * (c["shared"] + own_n) * c["hq"] * D)
    M, N, K = c["M"], c["N"], c["K"]
    return dict(bytes=4 * M * K + N * (K + 4) + 4 * M * (N // 2 if kind == "gate" else N), flops=2 * M * N * K)


# ---------------------------------------------------------------- 64-bit results, from the definitions
def _dims_of(which):
    """The dim at each nibble of a row."""
    order = [0] * D
    for g in range(4):
        for i in range(64):
            if which == "k":
                order[64 * (i // 16) + 16 * g + i % 16] = 64 * g + i
            else:
                order[16 * (i // 4) + 4 * g + i % 4] = 64 * g + i
    return torch.tensor(order, device=DEV)


def _row64(pages, which, page, row):
    """Row `row` of page `page` (both [n]) of all heads in 64 bits: [n, Hkv, 256]."""
    codes, scale = (pages[0], pages[2]) if which == "k" else (pages[1], pages[3])
    if scale is None:
        return codes[page, :, row].double()
    b = codes[page, :, row].long()
    out = torch.empty(*b.shape[:-1], D, dtype=torch.float64, device=DEV)
    at = _dims_of(which)
    out[..., at[0::2]] = (b % 16 - 8).double()
    out[..., at[1::2]] = (b // 16 - 8).double()
    return out * scale[page, :, row].double().repeat_interleave(GROUP, -1)


def _exact_attn(s):
    c = s["case"]
    hq, hkv, ps = c["hq"], c["hkv"], c["page"]
    out = torch.zeros(c["B"], c["T"], hq * D, dtype=torch.float64, device=DEV)
    pos, lens, table = s["pos"].tolist(), s["lens"].tolist(), s["table"].long()
    for b in range(c["B"]):
        n = lens[b]
        at = torch.arange(pos[b] + n, device=DEV)
        kk, vv = (_row64(s["pages"], w, table[b, at // ps], at % ps) for w in "kv")  # [keys, Hkv, D]
        new = at[pos[b]:]
        x = s["q"][b, :n].double()
        x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * (s["q_norm"].double() + 1)
        turn = torch.complex(s["cos"][new].double(), s["sin"][new].double())[:, None]
        z = torch.complex(x[..., :HALF].contiguous(), x[..., HALF:ROT].contiguous()) * turn
        x = torch.cat([z.real, z.imag, x[..., ROT:]], -1)
        for h in range(hq):
            y = x[:, h] @ kk[:, h * hkv // hq].T / 16
            y = torch.where(at[None] > new[:, None], -INF, y)
            out[b, :n, h * D:(h + 1) * D] = y.softmax(-1) @ vv[:, h * hkv // hq] * s["gate"][b, :n, h].double().sigmoid()
    return out


def _exact_cut(x, t, k, p, m):
    """One row of doubles -> the kept tokens' probabilities, token by token down the sorted row."""
    V = x.shape[0]
    down = torch.argsort(-x, stable=True)
    if t <= 0:
        n = 1
    else:
        e = ((x[down] - x[down[0]]) / t).exp()
        n = min(k, V) if k > 0 else V
        if p < 1:
            run = e[:n].cumsum(0)
            n = 1 + int((run[:n - 1] < p * run[-1]).sum())
        n = max(1, min(n, int((e >= m).sum())))
    out = torch.zeros_like(x)
    out[down[:n]] = ((x[down[:n]] - x[down[0]]) / t).softmax(0) if t > 0 else 1.0
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "sample" and not c["probs"]:
        return None  # whole numbers, held to be equal
    s = prepare(case, seed)
    if c["kind"] == "attn":
        return _exact_attn(s)
    if c["kind"] in ("sample", "filter"):
        x = s["x"].flatten(0, -2)
        rows = []
        for i in range(x.shape[0]):
            t, k, p, m = ((v[i].item() if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float32).item())
                          for v in (s["cuts"][n] for n in ("temperature", "top_k", "top_p", "min_p")))
            rows.append(_exact_cut(x[i].double(), t, int(k), p, m))
        probs = torch.stack(rows)
        if c["kind"] == "sample":
            return None, probs
        return torch.where(probs > 0, x.double(), -INF).view_as(s["x"])
    x = s["x"].double()
    if c["kind"] != "down":
        x = x / (x.square().sum(1, keepdim=True) / c["K"] + EPS).sqrt() * (s["norm"].double() + 1)
    scale = (x.abs().max(1).values / 127).float().double()
    n = torch.round(x / scale[:, None].clamp_min(1e-300)).clamp(-127, 127)
    y = torch.empty(c["M"], c["N"], dtype=torch.float64, device=DEV)
    for i in range(0, c["M"], 4096):  # whole numbers below 2^53: exact
        y[i:i + 4096] = n[i:i + 4096] @ s["w"].double().T
    y *= scale[:, None] * s["ws"].double()
    return torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2] if c["kind"] == "gate" else y
