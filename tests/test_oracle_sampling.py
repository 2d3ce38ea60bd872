"""oracle/sampling.py against the definition token by token."""
import math

import pytest
import torch

from oracle import paged, sampling


def slow_kept(x, T, k, p, m):
    """One cut after the other on a list of (weight, index)."""
    top = max(x)
    ws = sorted(((math.exp((v - top) / T), i) for i, v in enumerate(x)), key=lambda t: (-t[0], t[1]))
    if k > 0:
        ws = ws[:k]
    if p < 1:
        total, ahead, kept = math.fsum(w for w, _ in ws), 0.0, []
        for w, i in ws:
            if kept and not ahead < p * total:
                break
            kept.append((w, i))
            ahead += w
        ws = kept
    return [i for n, (w, i) in enumerate(ws) if n == 0 or w >= m]


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.0, 0, 0.8, 0.0), (1.3, 0, 1.0, 0.1),
                                     (0.9, 12, 0.9, 0.05), (1.0, 3, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 1, 0.5, 2.0)])
def test_cuts_token_by_token(seed, T, k, p, m):
    x = 2 * torch.randn(40, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
    x[7] = x[3]  # a tie
    at, w = sampling.kept_tokens(x, T, k, p, m)
    assert at.tolist() == slow_kept(x.tolist(), T, k, p, m)
    assert torch.allclose(w, torch.exp((x[at] - x.max()) / T))


def test_the_draw_s_distribution():
    x = torch.randn(1, 9, generator=torch.Generator().manual_seed(1)) * 1.5
    _, probs = sampling.sample_tokens(x, torch.zeros(1), 0.8, 6, 0.9, 0.02)
    n = 20000
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(torch.cat([sampling.sample_tokens(x, u[i:i + 1], 0.8, 6, 0.9, 0.02)[0] for i in range(0, n, 10)]).long(),
                         minlength=9) / (n / 10)
    assert float((got - probs[0]).abs().max()) < 2 * 10 / n * 9 and float(probs.sum()) == pytest.approx(1)
    assert bool(((probs > 0) == (got > 0)).all())


def test_nothing_cut_is_the_softmax():
    x = torch.randn(3, 50, generator=torch.Generator().manual_seed(2))
    _, probs = sampling.sample_tokens(x, torch.zeros(3), 0.7)
    assert torch.allclose(probs, torch.softmax(x.double() / torch.tensor(0.7).double(), -1))
    assert torch.equal(sampling.filter_logits(x), x)
    tok, _ = sampling.sample_tokens(x, torch.full((3,), 0.9), 0.0)
    assert tok.tolist() == x.argmax(-1).tolist()
    want = paged.verify_drafts(x[:, None], torch.zeros(3, 0, dtype=torch.int32), torch.zeros(3, 1), temperature=0.0)[1][:, 0]
    assert torch.equal(tok, want)


def test_missing_logits():
    x = torch.tensor([[-math.inf] * 4, [math.nan, 1.0, -math.inf, 0.0], [math.inf, 0.0, math.inf, 1.0]])
    tok, p = sampling.sample_tokens(x, torch.tensor([0.5, 0.99, 0.6]))
    assert tok.tolist() == [0, 3, 2] and p[0].sum() == 0 and p[2].tolist() == [0.5, 0, 0.5, 0]
    f = sampling.filter_logits(x, top_k=1)
    assert f[0].tolist() == [-math.inf] * 4 and f[1].tolist() == [-math.inf, 1.0, -math.inf, -math.inf]
