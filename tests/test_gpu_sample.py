"""Truncated sampling on the GPU against oracle/sampling.py in 64 bits: tokens and what is cut are equal.

Probabilities: w / sum with w in 64 bits, sums of whole numbers of 2^-S of the largest weight (S = 62 - log2 V: at most V 2^-S / 2
= 2^-26 of the sum for 2^18 tokens), rounded once to fp32: 2^-24 + 2^-26 relative, and 2^-149 where that is more.
"""
import math

import pytest
import torch

from gpu_util import announce, device
from oracle import paged, sampling
from q35hip import Q35Error, ops

pytestmark = pytest.mark.gpu


def logits(B, V, seed=0, a=1.5, noise=0.6):
    g = torch.Generator().manual_seed(seed)
    rank = torch.stack([torch.randperm(V, generator=g) for _ in range(B)]).float()
    return -a * torch.log(2 + rank) + noise * torch.randn(B, V, generator=g)


def both(x, u, **cuts):
    dev = device()
    up = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in cuts.items()}
    xd = x.to(dev)
    tok, probs = ops.sample_tokens(xd, u.to(dev), want_probs=True, **up)
    assert torch.equal(ops.sample_tokens(xd, u.to(dev), **up), tok)
    cut = ops.filter_logits(xd, **up)
    want, p = sampling.sample_tokens(x, u, **cuts)
    assert tok.dtype == torch.int32 and torch.equal(tok.cpu(), want), (tok.cpu(), want)
    assert torch.equal(cut.cpu(), sampling.filter_logits(x, **cuts))
    err = (probs.double().cpu() - p).abs()
    assert bool((err <= (2.0 ** -24 + 2.0 ** -26) * p + 2.0 ** -149).all()), float((err / p.clamp_min(1e-40)).max())
    return want


CUTS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.99),
        dict(min_p=0.1), dict(top_p=0.95, min_p=0.02, temperature=0.6), dict(top_k=300, top_p=0.999, min_p=1e-4, temperature=1.7),
        dict(top_k=7, min_p=0.5), dict(top_p=0.0), dict(min_p=1.0), dict(min_p=3.0), dict(temperature=0.05), dict(temperature=30.0, top_p=0.7)]


@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 3), (2, 61), (3, 1000), (2, 4096), (2, 4099), (1, 20001), (2, 65539)])
@pytest.mark.parametrize("cuts", CUTS, ids=str)
def test_cuts(B, V, cuts):
    u = torch.rand(B, generator=torch.Generator().manual_seed(V))
    announce(f"sample B{B} V{V} {cuts}")
    both(logits(B, V, seed=V), u, **cuts)


@pytest.mark.parametrize("a,noise", [(1.1, 0.6), (3.0, 0.3), (0.0, 2.5), (0.0, 0.05), (0.0, 0.0)])
def test_full_vocabulary(a, noise):
    """Sure rows, undecided ones (a nucleus of tens of thousands), flat ones and one where all logits are equal."""
    V = 151936
    x = logits(2, V, seed=int(10 * a + 100 * noise), a=a, noise=noise)
    u = torch.tensor([0.37, 0.993])
    for cuts in (dict(), dict(top_p=0.9), dict(top_k=40, top_p=0.95, temperature=0.7), dict(top_k=100000), dict(min_p=0.05),
                 dict(top_k=60000, top_p=0.97, min_p=1e-3, temperature=1.2)):
        announce(f"sample V{V} a {a} noise {noise} {cuts}")
        both(x, u, **cuts)


def test_settings_per_row():
    B, V = 7, 5003
    x, u = logits(B, V, seed=3), torch.rand(B, generator=torch.Generator().manual_seed(4))
    announce("sample per row")
    both(x, u, temperature=torch.tensor([0.0, -1.0, 0.5, 1.0, 2.0, 0.8, 1.0]),
         top_k=torch.tensor([0, 3, -5, 10, 99999, 1, 200], dtype=torch.int32),
         top_p=torch.tensor([0.5, 1.0, 0.9, 2.0, 0.7, 0.1, -1.0]), min_p=torch.tensor([0.1, 0.0, -1.0, 0.01, 0.0, 0.9, 0.3]))


def test_ties_are_cut_by_index():
    """Equal logits across every border: the lowest indices stay."""
    V = 9001
    x = torch.zeros(3, V)
    x[1, 4000:4100] = 1.0
    x[2, ::3] = 2.0
    x[2, 1::3] = -0.0
    u = torch.tensor([0.999, 0.5, 0.25])
    announce("sample ties")
    for cuts in (dict(top_k=10), dict(top_k=150), dict(top_p=0.25), dict(top_p=0.5), dict(top_k=3500, top_p=0.875), dict(min_p=0.9),
                 dict(top_k=77, min_p=1.0)):
        both(x, u, **cuts)


def test_many_ties_in_the_border():
    """More tokens of one value than a block holds in LDS, across each border."""
    V = 40000
    x = torch.full((2, V), -3.0)
    x[:, 7::2] = 1.25
    x[1, 20000] = 2.0
    u = torch.tensor([0.731, 0.4])
    announce("sample many ties")
    for cuts in (dict(top_k=9000), dict(top_p=0.75), dict(top_k=15000, top_p=0.5), dict(min_p=0.4), dict(top_k=30000)):
        both(x, u, **cuts)


def test_masked_infinite_and_missing_logits():
    V = 5000
    x = logits(8, V, seed=9)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, ::2] = math.nan
    x[4, [3, 4999]] = math.inf
    x[5, 10:] = torch.finfo(torch.float32).min
    x[6] = math.inf
    x[7] = 1e-42 * torch.arange(V)
    u = torch.full((8,), 0.6)
    announce("sample masks")
    for cuts in (dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.2), dict(temperature=0.0), dict(top_k=20, top_p=0.5, min_p=0.01)):
        want = both(x, u, **cuts)
        assert int(want[0]) == 0 and int(want[1]) == 0 and int(want[2]) == 0


def test_borders_of_the_random_numbers():
    x = torch.full((5, 9000), -math.inf)
    x[:, [8000, 4096, 17]] = 0.0
    announce("sample borders")
    tok = both(x, torch.tensor([0.0, 1 / 3, 2 / 3, 1 - 2.0 ** -24, 1.0]))
    assert tok.tolist()[0] == 17 and tok.tolist()[3:] == [8000, 8000]


def test_strides_positions_and_odd_rows():
    """Rows that start off 16 bytes, several positions, wider tensors around them, strided random numbers."""
    dev = device()
    B, P, V = 3, 4, 4101
    wide = torch.full((B, P + 1, V + 6), 50.0)
    for off in range(4):
        x = torch.stack([logits(P, V, seed=10 * b + off) for b in range(B)])
        wide[:, :P, off:off + V] = x
        t, k = torch.tensor([0.7, 1.0, 0.0]), torch.tensor([0, 30, 4], dtype=torch.int32)
        announce(f"filter strides {off}")
        got = ops.filter_logits(wide.to(dev)[:, :P, off:off + V], temperature=t.to(dev), top_k=k.to(dev), top_p=0.9)
        assert torch.equal(got.cpu(), sampling.filter_logits(x, t, k, 0.9))
        u = torch.rand(B, 5)
        tok = ops.sample_tokens(wide.to(dev)[:, 1, off:off + V], u.to(dev)[:, 3], top_p=0.9)
        assert torch.equal(tok.cpu(), sampling.sample_tokens(x[:, 1], u[:, 3], top_p=0.9)[0])


def test_the_cut_distribution_through_verification():
    """A draft model's tokens with their probabilities, checked against the target's logits under the same cuts: what the
    oracles give, and over many random numbers the kept and drawn tokens follow the target's cut distribution."""
    dev = device()
    B, V = 4000, 24
    g = torch.Generator().manual_seed(2)
    cuts = dict(temperature=0.8, top_k=12, top_p=0.9)
    xd, xt = (2 * torch.randn(1, V, generator=g) for _ in range(2))
    u = torch.rand(B, 3, generator=g)
    announce("sample, filter, verify")
    draft, q = ops.sample_tokens(xd.expand(B, V).to(dev), u[:, 2].contiguous().to(dev), want_probs=True, **cuts)
    target = ops.filter_logits(xt.expand(B, 2, V).contiguous().to(dev), **cuts)
    n, tok = ops.verify_drafts(target, draft[:, None], u[:, :2].contiguous().to(dev), draft_probs=q[:, None], temperature=0.8)
    _, p = sampling.sample_tokens(xt, torch.zeros(1), **cuts)
    got = torch.bincount(tok[:, 0].long().cpu(), minlength=V) / B
    assert float((got - p[0]).abs().max()) < 5 * 0.5 / math.sqrt(B) and bool((got[p[0] == 0] == 0).all())
    wn, wt = paged.verify_drafts(target.cpu(), draft[:, None].cpu(), u[:, :2], q[:, None].cpu(), None, 0.8)
    assert torch.equal(n.cpu(), wn) and torch.equal(tok.cpu(), wt)


def test_captured_and_side_by_side():
    dev = device()
    x = logits(4, 30011, seed=6).to(dev)
    u = torch.rand(4, generator=torch.Generator().manual_seed(1)).to(dev)
    cuts = dict(temperature=0.9, top_p=0.9, top_k=torch.tensor([0, 10, 0, 5000], dtype=torch.int32, device=dev))

    def step():
        return (*ops.sample_tokens(x, u, want_probs=True, **cuts), ops.filter_logits(x, **cuts))
    announce("sample capture")
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        u.copy_(torch.rand(4, generator=torch.Generator().manual_seed(i)).to(dev))
        x.copy_(logits(4, 30011, seed=20 + i).to(dev))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [step() for _ in range(3)]
    b = [step() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for s, t in zip(a, b) for p, q in zip(s, t))


def test_empty_and_refusals():
    dev = device()
    x, u = torch.zeros(3, 10, device=dev), torch.zeros(3, device=dev)
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,) and ops.filter_logits(x[:0]).shape == (0, 10)
    announce("sample refusals")
    for bad in (lambda: ops.sample_tokens(x.double(), u), lambda: ops.sample_tokens(x[None], u), lambda: ops.sample_tokens(x, u[:2]),
                lambda: ops.sample_tokens(x, u.double()), lambda: ops.sample_tokens(x.T, u), lambda: ops.sample_tokens(x[:, :0], u),
                lambda: ops.sample_tokens(x.cpu(), u), lambda: ops.sample_tokens(x, u.cpu()),
                lambda: ops.sample_tokens(x, u, temperature=-1.0), lambda: ops.sample_tokens(x, u, temperature=math.nan),
                lambda: ops.sample_tokens(x, u, top_p=math.nan), lambda: ops.sample_tokens(x, u, min_p=math.nan),
                lambda: ops.sample_tokens(x, u, top_k=u), lambda: ops.sample_tokens(x, u, top_p=u[:2]),
                lambda: ops.sample_tokens(x, u, temperature=u.cpu()), lambda: ops.filter_logits(x[0]),
                lambda: ops.filter_logits(torch.zeros(1, (1 << 22) + 1, device=dev))):
        with pytest.raises(Q35Error):
            bad()
