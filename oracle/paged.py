"""Paged KV cache, attention over it and the check of drafted tokens, on the CPU in 64 bits (test infrastructure only).

  quantize_rows / row_values   the 4-bit row format: one bf16 scale s = bf16(fp32(max |x| / 7)) per group of 64 dims, codes
                               8 + clamp(rint(x / s), -7, 7), standing for (code - 8) s
  pack_rows / unpack_rows      the order of the codes in a row's 128 bytes (include/q35hip.h)
  paged_append                 k norm with (1 + w), rotation, and the writes through the block table
  paged_rows                   rows read back in the dense caches' layout
  gated_attention_paged        HF:656-698 over the keys that the table names, token by token
  verify_drafts                acceptance by u q < p, then the inverse CDF of max(p - q, 0) or p

Pinned (tests/test_oracle_paged.py): packing against the dim-by-dim formula and round trips, the format's error bound and
exact values, the attention against oracle.gated_attention_cached on dense caches, the verification's distribution against
the target's by integration over a grid of random numbers.
"""
import math

import torch

from .attention import apply_partial_rope

GROUP, D = 64, 256


def nibble_of(which):
    """The nibble at which each dim of a row lies."""
    d = torch.arange(D)
    g, i = d // 64, d % 64
    if which == "k":
        return 64 * (i // 16) + 16 * g + i % 16
    return 16 * (i // 4) + 4 * g + i % 4


def quantize_rows(x):
    """x [..., 256] -> codes [..., 256] (uint8, dims in order), scales [..., 4] bf16."""
    g = x.double().unflatten(-1, (D // GROUP, GROUP))
    finite = torch.isfinite(g).all(-1)
    s = (torch.where(finite[..., None], g, 0.0).abs().amax(-1) / 7).float().to(torch.bfloat16)
    sd = s.double()[..., None]
    n = torch.where((sd > 0) & finite[..., None], g / sd, 0.0).round().clamp(-7, 7)
    s = torch.where(finite, s, torch.tensor(math.nan, dtype=torch.bfloat16))
    return (torch.nan_to_num(n) + 8).to(torch.uint8).flatten(-2), s


def pack_rows(codes, which):
    at = nibble_of(which)
    nib = torch.empty_like(codes)
    nib[..., at] = codes
    return nib[..., 0::2] | nib[..., 1::2] << 4


def unpack_rows(packed, which):
    nib = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    return nib[..., nibble_of(which)]


def row_values(packed, scale, which):
    """The doubles that a 4-bit row stands for (bf16 rows: themselves)."""
    if scale is None:
        return packed.double()
    n = unpack_rows(packed, which).double() - 8
    return (n.unflatten(-1, (D // GROUP, GROUP)) * scale.double()[..., None]).flatten(-2)


def _norm(x, w, eps):
    x = x.double()
    if w is None:
        return x
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (1 + w.double())


def _places(pages, table, pos, lens, T):
    """(b, t, position, page, row in it) of every token that is there; page None where the table names none."""
    n_pages, ps = pages[0].shape[0], pages[0].shape[2]
    cap = table.shape[1] * ps
    for b in range(table.shape[0]):
        n = T if lens is None else min(max(int(lens[b]), 0), T)
        for t in range(n):
            at = int(pos[b]) + t
            if 0 <= at < cap:
                page = int(table[b, at // ps])
                yield b, t, at, page if 0 <= page < n_pages else None, at % ps


def paged_append(k, v, pages, table, pos, cos, sin, lens=None, k_norm_w=None, eps=1e-6):
    """Writes into `pages` (a tuple of CPU tensors) in place; bf16 pages get the 64-bit values rounded once."""
    kp, vp, ks, vs = pages
    kn = _norm(k, k_norm_w, eps)
    for b, t, at, page, row in _places(pages, table, pos, lens, k.shape[1]):
        if page is None:
            continue
        kr = apply_partial_rope(kn[b:b + 1, t:t + 1], cos[at:at + 1].double(), sin[at:at + 1].double())[0, 0]
        for x, dst, sc, which in ((kr, kp, ks, "k"), (v[b, t].double(), vp, vs, "v")):
            if sc is None:
                dst[page, :, row] = x.to(dst.dtype)
            else:
                codes, s = quantize_rows(x)
                dst[page, :, row], sc[page, :, row] = pack_rows(codes, which), s


def paged_rows(pages, table, pos, T, lens=None):
    """(k, v) [B, Hkv, T, 256] doubles, zeros where there is no token."""
    out = [torch.zeros(table.shape[0], pages[0].shape[1], T, D, dtype=torch.float64) for _ in range(2)]
    for b, t, at, page, row in _places(pages, table, pos, lens, T):
        if page is not None:
            for o, i, which in ((out[0], 0, "k"), (out[1], 1, "v")):
                sc = pages[2 + i]
                o[b, :, t] = row_values(pages[i][page, :, row], None if sc is None else sc[page, :, row], which)
    return tuple(out)


def gated_attention_paged(q, gate, pages, table, pos, cos, sin, lens=None, q_norm_w=None, eps=1e-6, scale=None,
                          spread=False):
    """[B, T, Hq * 256] doubles. spread: also sum_j w_j |v_j| sigmoid(gate), the sum of q and k's absolute products and
    sum_j w_j s_j (the 4-bit value scale of each dim's group, zeros for bf16), for error bounds."""
    B, T, Hq, _ = q.shape
    Hkv, ps, n_pages = pages[0].shape[1], pages[0].shape[2], pages[0].shape[0]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, T, Hq * D, dtype=torch.float64)
    amp, prod, step = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    qn = _norm(q, q_norm_w, eps)
    cap = table.shape[1] * ps
    for b in range(B):
        n = T if lens is None else min(max(int(lens[b]), 0), T)
        last = min(int(pos[b]) + n, cap)
        if n == 0 or last <= 0:
            continue
        at = torch.arange(last)
        page, row = table[b, at // ps].long(), at % ps
        named = (page >= 0) & (page < n_pages)
        page = page.where(named, torch.zeros_like(page))
        k, v = (row_values(pages[i][page, :, row], None if pages[2 + i] is None else pages[2 + i][page, :, row], w)
                for i, w in ((0, "k"), (1, "v")))
        sv = torch.zeros_like(v) if pages[3] is None else pages[3][page, :, row].double().repeat_interleave(GROUP, -1)
        for t in range(n):
            p = int(pos[b]) + t
            if not 0 <= p < cap:
                continue
            keys = torch.nonzero(named[:p + 1])[:, 0]
            if keys.numel() == 0:
                continue
            qt = apply_partial_rope(qn[b:b + 1, t:t + 1], cos[p:p + 1].double(), sin[p:p + 1].double())[0, 0]
            for h in range(Hq):
                kk, vv = k[keys, h // G], v[keys, h // G]
                w = torch.softmax(kk @ qt[h] * scale, 0)
                g = 1.0 if gate is None else torch.sigmoid(gate[b, t, h].double())
                sl = slice(h * D, (h + 1) * D)
                out[b, t, sl] = (w @ vv) * g
                if spread:
                    amp[b, t, sl] = (w @ vv.abs()) * g
                    prod[b, t, sl] = (kk.abs() @ qt[h].abs()).max() * abs(scale)
                    step[b, t, sl] = (w @ sv[keys, h // G]) * g
    return (out, amp, prod, step) if spread else out


def verify_drafts(logits, draft_ids, u, draft_probs=None, lens=None, temperature=1.0):
    """(n_accept [B], tokens [B, K + 1]) int32, position by position."""
    B, K, V = logits.shape[0], logits.shape[1] - 1, logits.shape[2]
    n_out = torch.zeros(B, dtype=torch.int32)
    tokens = torch.full((B, K + 1), -1, dtype=torch.int32)

    def target(x, T):
        x = torch.nan_to_num(x.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        m = x.max()
        if m == -math.inf:
            return None
        if T <= 0:
            w = torch.zeros(V, dtype=torch.float64)
            w[int((x == m).nonzero()[0])] = 1
            return w
        w = torch.where(x == m, 1.0, torch.where(x == -math.inf, 0.0, torch.exp((x - m) / T)))
        return w / w.sum()
    for b in range(B):
        T = float(temperature[b]) if torch.is_tensor(temperature) else float(temperature)
        n = K if lens is None else min(max(int(lens[b]), 0), K)
        i, token = 0, None
        while i < n:
            p, x = target(logits[b, i], T), int(draft_ids[b, i])
            q = 1.0 if draft_probs is None else (float(draft_probs[b, i, x]) if 0 <= x < V else 0.0)
            if p is None or not 0 <= x < V or not float(u[b, i]) * q < float(p[x]):
                break
            tokens[b, i] = x
            i += 1
        p = target(logits[b, i], T)
        if p is None:
            token = 0
        else:
            r = p
            if i < n:
                less = torch.zeros(V, dtype=torch.float64)
                if draft_probs is not None:
                    less = draft_probs[b, i].double()
                elif 0 <= int(draft_ids[b, i]) < V:
                    less[int(draft_ids[b, i])] = 1
                left = torch.nan_to_num(p - less, nan=0.0).clamp_min(0)
                r = left if left.sum() > 0 else p
            run = r.cumsum(0)
            over = (run > float(u[b, K]) * run[-1]).nonzero()
            token = int(over[0]) if over.numel() else int((r > 0).nonzero()[-1])
        tokens[b, i] = token
        n_out[b] = i
    return n_out, tokens
