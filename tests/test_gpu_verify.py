"""Verification of drafted tokens on the GPU: whole numbers, equal to oracle/paged.py's in 64 bits."""
import math

import pytest
import torch

from gpu_util import announce, device
from oracle import paged
from q35hip import Q35Error, ops

pytestmark = pytest.mark.gpu


def make(B, K, V, seed=0, probs=False, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g) * spread
    near = logits[:, :K] + torch.randn(B, K, V, generator=g)
    q = near.softmax(-1) if probs else None
    ids = (torch.multinomial(q.view(B * K, V), 1, generator=g).view(B, K) if probs and K else near.argmax(-1)).int()
    return logits, ids, torch.rand(B, K + 1, generator=g), q, torch.randint(0, K + 1, (B,), generator=g).int()


def both(logits, ids, u, q=None, lens=None, temperature=1.0):
    dev = device()
    up = [None if x is None else x.to(dev) for x in (logits, ids, u, q, lens)]
    t = temperature.to(dev) if torch.is_tensor(temperature) else temperature
    got = ops.verify_drafts(up[0], up[1], up[2], draft_probs=up[3], lens=up[4], temperature=t)
    want = paged.verify_drafts(logits, ids, u, q, lens, temperature)
    for a, b in zip(got, want):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), (a.cpu(), b)
    return want


@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (1, 1, 2), (3, 0, 1000), (4, 3, 97), (2, 4, 4096), (2, 4, 4097), (3, 2, 20001),
                                   (2, 7, 12288), (5, 15, 130)])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_verify(B, K, V, probs, temperature):
    x, ids, u, q, lens = make(B, K, V, seed=V + K, probs=probs)
    announce(f"verify B{B} K{K} V{V} probs {probs} T {temperature}")
    both(x, ids, u, q, None, temperature)
    both(x, ids, u, q, lens, temperature)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_full_vocabulary(probs):
    """A flat distribution over 151,936 tokens (a running sum in 32 bits would miss tokens), and a peaked one."""
    for spread in (0.05, 3.0):
        x, ids, u, q, lens = make(3, 2, 151936, seed=int(spread * 10), probs=probs, spread=spread)
        announce(f"verify V151936 spread {spread} probs {probs}")
        both(x, ids, u, q, lens)
        both(x, ids, u, q, torch.zeros(3, dtype=torch.int32), 1.0)


def test_verify_temperature_per_row_and_strided_inputs():
    B, K, V = 4, 3, 5003
    x, ids, u, q, lens = make(B, K, V, probs=True)
    t = torch.tensor([0.0, 0.5, 1.0, 2.0])
    announce("verify strides")
    want = both(x, ids, u, q, lens, t)
    dev = device()
    wide = torch.full((B, K + 3, V + 5), 99.0, device=dev)
    wide[:, 1:K + 2, 3:V + 3] = x.to(dev)
    wq = torch.full((B, K, V + 1), 0.5, device=dev)
    wq[..., 1:] = q.to(dev)
    wide_ids, wu = torch.full((B, 9), 7, dtype=torch.int32, device=dev), torch.zeros(B, 11, device=dev)
    wide_ids[:, 2:2 + K], wu[:, 5:6 + K] = ids.to(dev), u.to(dev)
    got = ops.verify_drafts(wide[:, 1:K + 2, 3:V + 3], wide_ids[:, 2:2 + K], wu[:, 5:6 + K], draft_probs=wq[..., 1:],
                            lens=lens.to(dev), temperature=t.to(dev))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_verify_borders_of_the_random_numbers():
    """u = 0 takes the first token with weight; the largest fp32 below 1 the last reachable; 1 itself the last with weight;
    u q = p refuses."""
    x = torch.full((4, 1, 9000), -math.inf)
    x[:, 0, [5, 4096, 8999]] = torch.tensor([0.0, 0.0, 0.0])
    u = torch.tensor([[0.0], [1 / 3], [1 - 2 ** -24], [1.0]])
    ids = torch.zeros(4, 0, dtype=torch.int32)
    announce("verify borders")
    _, tok = both(x, ids, u)
    assert tok[:, 0].tolist()[0] == 5 and tok[:, 0].tolist()[2:] == [8999, 8999]
    x = torch.tensor([[[0.0, 0.0], [0.0, 0.0]]])  # p = 1/2, drafted for certain
    for v, n in ((0.5, 0), (0.5 - 2 ** -25, 1)):
        got = both(x, torch.tensor([[1]], dtype=torch.int32), torch.tensor([[v, 0.9]]))
        assert got[0].tolist() == [n]


def test_verify_masked_infinite_and_missing_logits():
    V = 6000
    x, ids, u, _, _ = make(6, 2, V, seed=9)
    x[0] = -math.inf                       # no winner: nothing kept, token 0
    x[1, 0] = math.nan
    x[1, 0, 77] = 1.0                      # NaN counts as nothing
    ids[1, 0] = 77
    x[2, 0, [3, 5999]] = math.inf          # infinities share the mass
    ids[2, 0] = 5999
    x[3, :, 1:] = torch.finfo(torch.float32).min  # the type's lowest value as a mask
    ids[3] = 0
    ids[4, 0], ids[5, 1] = -1, V           # drafts that are no token
    announce("verify masks")
    for t in (0.0, 1.0):
        n, tok = both(x, ids, u, None, None, t)
        assert int(n[0]) == 0 and int(tok[0, 0]) == 0 and int(n[1]) >= 1 and int(n[3]) == 2 and int(n[4]) == 0


def test_verify_nothing_left_behind_a_refusal():
    """q = p to the last bit and more (an fp32 q that sums to over 1): the drawn token falls back on p."""
    x = torch.zeros(1, 2, 8)
    q = torch.full((1, 1, 8), 0.2)
    announce("verify fallback")
    n, tok = both(x, torch.tensor([[2]], dtype=torch.int32), torch.tensor([[0.9, 0.6]]), q)
    assert n.tolist() == [0] and tok[0].tolist() == [4, -1]


def test_verify_captured_and_side_by_side():
    """In a graph, replayed on new numbers with eager calls between; and on two streams at once."""
    dev = device()
    x, ids, u, q, lens = (t.to(dev) for t in make(3, 4, 30000, seed=4, probs=True))
    announce("verify capture")
    ops.verify_drafts(x, ids, u, draft_probs=q, lens=lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_drafts(x, ids, u, draft_probs=q, lens=lens)
    for step in range(4):
        u.copy_(torch.rand(3, 5, generator=torch.Generator().manual_seed(step)).to(dev))
        graph.replay()
        want = ops.verify_drafts(x, ids, u, draft_probs=q, lens=lens)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.verify_drafts(x, ids, u, draft_probs=q, lens=lens))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_verify_refusals_on_the_device():
    dev = device()
    x, ids, u, q, lens = (t.to(dev) for t in make(2, 3, 50, probs=True))
    announce("verify refusals")
    for call in (lambda: ops.verify_drafts(x.half(), ids, u), lambda: ops.verify_drafts(x, ids.long(), u),
                 lambda: ops.verify_drafts(x, ids[:, :2], u), lambda: ops.verify_drafts(x, ids, u[:, :3]),
                 lambda: ops.verify_drafts(x, ids, u, draft_probs=q[..., :49]),
                 lambda: ops.verify_drafts(x, ids, u, lens=lens.long()), lambda: ops.verify_drafts(x, ids.cpu(), u),
                 lambda: ops.verify_drafts(x, ids, u, temperature=-1.0),
                 lambda: ops.verify_drafts(x, ids, u, temperature=float("nan")),
                 lambda: ops.verify_drafts(x, ids, u, temperature=torch.ones(3, device=dev))):
        with pytest.raises(Q35Error):
            call()


def test_verify_infinite_temperature_and_nan_draft_probabilities():
    """The tokens above -inf alike; a NaN among the draft's probabilities refuses its draft and leaves its token undrawn."""
    x, ids, u, q, lens = make(4, 2, 5000, seed=3, probs=True)
    x[:, :, 1000:3000] = -math.inf
    announce("verify infinite temperature, NaN probabilities")
    both(x, ids, u, q, lens, math.inf)
    both(x, ids, u, q, lens, torch.tensor([math.inf, 1.0, 0.0, -2.0]))
    q[:, :, 77] = math.nan
    ids[0, 0] = ids[1, 1] = 77
    n, _ = both(x, ids, u, q)
    assert int(n[0]) == 0 and int(n[1]) <= 1


def test_verify_most_drafts_and_largest_vocabulary():
    x, ids, u, q, _ = make(2, 255, 300, seed=8, probs=True, spread=0.1)
    q = x[:, :-1].softmax(-1)  # nearly every draft is kept
    announce("verify K 255, V 4194304")
    n, _ = both(x, ids, u, q)
    x, ids, u, q, _ = make(1, 1, 4194304, seed=8, spread=0.5)
    both(x, ids, u, q)
    dev = device()
    with pytest.raises(Q35Error):
        ops.verify_drafts(torch.zeros(1, 1, 4194305, device=dev), torch.zeros(1, 0, dtype=torch.int32, device=dev),
                          torch.zeros(1, 1, device=dev))
    with pytest.raises(Q35Error):
        ops.verify_drafts(torch.zeros(1, 257, 8, device=dev), torch.zeros(1, 256, dtype=torch.int32, device=dev),
                          torch.zeros(1, 257, device=dev))


def test_verify_rows_past_32_bits():
    """Rows of logits more than 2^32 bytes apart."""
    dev = device()
    x, ids, u, q, lens = make(2, 1, 3001, seed=12)
    announce("verify rows past 32 bits")
    far = (1 << 31) + 64  # elements
    pool = torch.empty(far + 2 * 3001, device=dev)
    wide = pool.as_strided((2, 2, 3001), (far, 3001, 1))
    wide.copy_(x.to(dev))
    got = ops.verify_drafts(wide, ids.to(dev), u.to(dev))
    want = paged.verify_drafts(x, ids, u)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_verify_broadcast_logits():
    """One row's logits for every sequence, as an expanded view, each with its own random numbers."""
    dev = device()
    x, ids, u, q, _ = make(5, 3, 4099, seed=21, probs=True)
    announce("verify broadcast logits")
    one, qone = x[:1].to(dev), q[:1].to(dev)
    ids = ids[:1].expand(5, 3)
    got = ops.verify_drafts(one.expand(5, 4, 4099), ids.to(dev).contiguous(), u.to(dev),
                            draft_probs=qone.expand(5, 3, 4099))
    want = paged.verify_drafts(x[:1].expand(5, 4, 4099), ids, u, q[:1].expand(5, 3, 4099))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
