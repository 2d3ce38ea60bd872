"""Truncated sampling on the CPU in 64 bits (test infrastructure only).

  kept_tokens     the tokens that top-k, top-p and min-p keep of one row, from the most likely down, and their weights
  sample_tokens   the token that a random number falls on, and the probabilities it is drawn from
  filter_logits   the logits with what is cut at -inf

Pinned (tests/test_oracle_sampling.py): the cuts against sorted probabilities token by token, the draw's distribution by
integration over a grid of random numbers, and against verify_drafts where nothing is cut.
"""
import math

import torch


def kept_tokens(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x [V] -> (indices in order, weights relative to the first): the kept ones; none where no logit is above -inf."""
    x = torch.nan_to_num(x.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    V = x.numel()
    order = torch.argsort(x, descending=True, stable=True)
    m = x[order[0]]
    if m == -math.inf:
        return order[:0], x[:0]
    if not temperature > 0:
        return order[:1], torch.ones(1, dtype=torch.float64)
    xs = x[order]
    w = torch.where(xs == m, 1.0, torch.where(xs == -math.inf, 0.0, torch.exp((xs - m) / temperature)))
    n = top_k if 0 < top_k < V else V
    if top_p < 1:
        total, ahead, keep = float(w[:n].sum()), 0.0, 0
        run = torch.cat([torch.zeros(1, dtype=torch.float64), w[:n].cumsum(0)[:-1]])
        keep = int((run < max(top_p, 0.0) * total).sum())
        n = max(keep, 1)
    if min_p > 0:
        n = max(min(n, int((w >= min_p).sum())), 1)
    return order[:n], w[:n]


def _setting(v, b):
    return v[b].item() if torch.is_tensor(v) else torch.tensor(v, dtype=torch.float32).item()


def _settings(b, temperature, top_k, top_p, min_p):
    return _setting(temperature, b), int(top_k[b]) if torch.is_tensor(top_k) else int(top_k), _setting(top_p, b), \
        _setting(min_p, b)


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens [B] int32, probabilities [B, V] doubles)."""
    B, V = logits.shape
    tokens, probs = torch.zeros(B, dtype=torch.int32), torch.zeros(B, V, dtype=torch.float64)
    for b in range(B):
        at, w = kept_tokens(logits[b], *_settings(b, temperature, top_k, top_p, min_p))
        if at.numel() == 0:
            continue
        run = w.cumsum(0)
        over = (run > float(u[b]) * run[-1]).nonzero()
        tokens[b] = at[int(over[0])] if over.numel() else at[int((w > 0).nonzero()[-1])]
        probs[b, at] = w / run[-1]
    return tokens, probs


def filter_logits(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """[B, V] or [B, P, V]: what is cut, and NaN, at -inf."""
    x = logits if logits.dim() == 3 else logits[:, None]
    out = torch.full_like(x, -math.inf)
    for b in range(x.shape[0]):
        for p in range(x.shape[1]):
            at, _ = kept_tokens(x[b, p], *_settings(b, temperature, top_k, top_p, min_p))
            out[b, p, at] = torch.nan_to_num(x[b, p, at], nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    return out.view_as(logits)
