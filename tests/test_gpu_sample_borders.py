"""Truncated sampling where a border can go wrong, against oracle/sampling.py in 64 bits: what is kept and drawn is equal."""
import math

import pytest
import torch

import q35hip
from gpu_util import announce, device
from oracle import sampling
from q35hip import ops
from test_gpu_sample import logits

pytestmark = pytest.mark.gpu


def same(x, u, **cuts):
    """Tokens and cut logits of x [B, V], device against oracle."""
    dev = device()
    up = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in cuts.items()}
    tok, cut = ops.sample_tokens(x.to(dev), u.to(dev), **up).cpu(), ops.filter_logits(x.to(dev), **up).cpu()
    want = sampling.filter_logits(x, **cuts)
    kept, asked = (cut > -float("inf")).sum(-1), (want > -float("inf")).sum(-1)
    assert torch.equal(cut, want), (kept.tolist(), asked.tolist())
    assert torch.equal(tok, sampling.sample_tokens(x, u, **cuts)[0])


@pytest.mark.parametrize("V", [16391, 40000])
def test_long_rows_behind_kernels_that_use_all_of_lds(V):
    """The smallest value of min-p is found with the table that the block has filled, not with what was in LDS before."""
    dev = device()
    B = 48
    g = torch.Generator().manual_seed(V)
    x, u = logits(B, V, seed=V), torch.rand(B, generator=g)
    cuts = dict(min_p=torch.exp(-8 * torch.rand(B, generator=g)), top_p=torch.where(torch.rand(B, generator=g) < 0.5, 0.97, 1.0))
    rows = ops.quantize_rows(torch.randn(4096, 1024, generator=g).to(dev))
    W = torch.randint(-127, 128, (7168, 1024), generator=g).to(torch.int8).to(dev)
    xd, ud, up = x.to(dev), u.to(dev), {k: v.to(dev) for k, v in cuts.items()}
    announce(f"min-p of rows of {V} behind large tiles")
    want = sampling.sample_tokens(x, u, **cuts)[0]
    for _ in range(4):
        ops.gemm_i8(rows, W, torch.ones(7168, device=dev), epilogue="swiglu")
        tok = ops.sample_tokens(xd, ud, **up)
        assert torch.equal(tok.cpu(), want)
    same(x, u, **cuts)


def border_rows(V, temps, ps, seed):
    """Rows whose largest logit M lies 0 to 2 steps of fp32 beside -T ln m, so that the border of min-p lies next to 0, where fp32
    is finest; the others on both sides of 0 from 1e-9 on, and anywhere. Returns logits, temperatures, min-ps."""
    g = torch.Generator().manual_seed(seed)
    t, m = (a.flatten() for a in torch.meshgrid(torch.tensor(temps), torch.tensor(ps), indexing="ij"))
    t, m = t.repeat(5), m.repeat(5)
    top = -t.double() * m.double().log()
    top = top.float()
    for i, steps in enumerate((-2, -1, 0, 1, 2)):
        at = slice(i * len(temps) * len(ps), (i + 1) * len(temps) * len(ps))
        for _ in range(abs(steps)):
            top[at] = torch.nextafter(top[at], torch.tensor(float("inf") if steps > 0 else -float("inf")))
    x = torch.rand(t.numel(), V, generator=g) * 1.5 * t[:, None] - t[:, None]
    x[1::2] -= 0.6 * t[1::2, None]  # (every other row: the border's own tokens alone)
    near = torch.cat([torch.zeros(1), 10.0 ** -torch.arange(3, 10)])
    x[:, 1:1 + near.numel()] = near
    x[:, 10:10 + near.numel()] = -near
    x = torch.minimum(x, top[:, None])
    x[:, 20] = top
    # nothing lies so near a border that 64 bits could not tell
    w = torch.exp((x.double() - top[:, None].double()) / t[:, None].double()) / m[:, None].double()
    assert float((w - 1).abs().min()) > 1e-13
    return x, t, m


TEMPS = [0.05, 0.3, 0.5, 0.6, 0.7, 0.8, 0.9, 1.0, 1.2, 1.5, 2.0, 5.0]
MINS = [1e-4, 1e-3, 0.005, 0.01, 0.02, 0.03, 0.05, 0.1, 0.2, 0.3, 0.5, 0.9]


@pytest.mark.parametrize("V", [33, 5000])
@pytest.mark.parametrize("cuts", [dict(), dict(top_k=30), dict(top_k=1500), dict(top_p=0.98), dict(top_k=40, top_p=0.9)], ids=str)
def test_min_p_whose_border_is_next_to_zero(V, cuts):
    x, t, m = border_rows(V, TEMPS, MINS, V)
    announce(f"min-p next to 0, V{V} {cuts}")
    same(x, torch.linspace(0, 0.999, x.shape[0]), temperature=t, min_p=m, **cuts)


@pytest.mark.parametrize("cuts", [dict(), dict(top_k=30), dict(top_p=0.98)], ids=str)
def test_min_p_of_long_rows_next_to_zero(cuts):
    x, t, m = border_rows(20011, [0.5, 0.7, 1.0, 1.2], [0.01, 0.02, 0.1, 0.3], 1)
    announce(f"min-p next to 0, long rows {cuts}")
    same(x, torch.linspace(0, 0.999, x.shape[0]), temperature=t, min_p=m, **cuts)


def test_min_p_of_one_number():
    """The plain settings, as numbers: 0.01 of the largest keeps what is above 0 here."""
    announce("min-p numbers")
    for m, t, top in ((0.01, 1.0, 4.60517025), (0.01, 0.5, 2.30258512), (0.02, 0.7, 2.73841596)):
        x = torch.full((1, 100), -0.5)
        x[0, 7], x[0, 50:60], x[0, 60:70] = top, 0.25, -0.25
        same(x, torch.tensor([0.98]), temperature=t, min_p=m)
        assert sampling.filter_logits(x, temperature=t, min_p=m).isfinite().sum() == 11


@pytest.mark.parametrize("V", [50, 20000])
def test_min_p_at_infinite_temperature(V):
    """Every finite logit weighs 1, which is at least any min-p up to 1."""
    x = logits(3, V, seed=V)
    x[1, ::3], x[2, 1::2] = -float("inf"), float("nan")
    announce(f"min-p at an infinite temperature V{V}")
    for m in (0.5, 1.0):
        same(x, torch.tensor([0.1, 0.6, 0.9]), temperature=float("inf"), min_p=m)


@pytest.mark.parametrize("V", [40, 5000, 20000])
def test_min_p_above_one_keeps_the_first_token(V):
    """No weight is more than the first one's: it alone stays, also where others equal it."""
    x = torch.zeros(4, V)
    x[1, V // 2:V // 2 + 9] = 1.0
    x[2] = float("inf")
    x[3, ::2] = -0.0
    u = torch.tensor([0.9, 0.95, 0.99, 0.5])
    announce(f"min-p above 1 V{V}")
    for cuts in (dict(min_p=1.5), dict(min_p=float("inf")), dict(min_p=3.0, top_k=5), dict(min_p=3.0, top_k=3000), dict(min_p=2.0, top_p=0.9),
                 dict(min_p=1.0, top_k=12), dict(min_p=torch.tensor([1.1, 0.5, 4.0, 0.0])),
                 dict(min_p=2.0, temperature=torch.tensor([0.0, 5.0, 0.1, float("inf")]))):
        same(x, u, **cuts)


def test_numbers_beside_tensors_are_not_read():
    """From C: where a row has its own settings the one number says nothing, also not which kernels run."""
    dev = device()
    B, V = 3, 20000
    x, u = logits(B, V, seed=5), torch.tensor([0.2, 0.7, 0.95])
    own = dict(temperature=torch.tensor([1.0, 0.8, 1.2]), top_k=torch.tensor([0, 5, 2000], dtype=torch.int32),
               top_p=torch.tensor([0.9, 1.0, 0.95]), min_p=torch.tensor([0.0, 0.1, 0.01]))
    one = dict(temperature=0.0, top_k=1, top_p=0.0, min_p=9.0)
    L = q35hip.lib()
    size = L.q35_sample_tokens_workspace_bytes(B, 1, V)
    ws, tok = torch.empty(size, dtype=torch.uint8, device=dev), torch.full((B,), -1, dtype=torch.int32, device=dev)
    xd, ud, up = x.to(dev), u.to(dev), {n: t.to(dev) for n, t in own.items()}
    for names in (("temperature", "top_k", "top_p", "min_p"), ("min_p",), ("top_k", "min_p"), ("temperature",), ("top_k", "top_p")):
        args = []
        for n in ("temperature", "top_k", "top_p", "min_p"):
            # (a number of no effect where the rows have none of their own)
            plain = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)[n]
            args += [up[n].data_ptr() if n in names else None, one[n] if n in names else plain]
        announce(f"sample from C, {names}")
        assert L.q35_sample_tokens(xd.data_ptr(), V, V, ud.data_ptr(), 1, *args, tok.data_ptr(), 0, None, B, 1, V, ws.data_ptr(),
                                   size, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(tok.cpu(), sampling.sample_tokens(x, u, **{n: own[n] for n in names})[0])


@pytest.mark.parametrize("bits", [9, 16, 18, 22])
def test_borders_behind_a_flat_tail(bits):
    """One token and a flat tail of 2^bits - 1 whose weights are about half of 2^-S, the unit of the sums (S = min(62 - bits, 50)).
    Each weight is off by half a unit and 2e-12 of itself, so a sum by e = 2^bits 2^-(S + 1) + 2e-12 of it, and the border of
    top-p and the draw lie where sums within 2 e (the whole's and the running one's) put them: a place in the tail is not
    known better than that, and what is kept is a first part of the order in any case."""
    V, S = 1 << bits, min(62 - bits, 50)
    u = torch.tensor([0.5, 1 - 2.0 ** -24])
    for halves in (0.5, 0.98, 1.02, 1.5, 3.0, 1000.0):  # of a weight in units of 2^-(S + 1)
        x = torch.full((2, V), math.log(halves) - (S + 1) * math.log(2.0))
        x[:, V // 3] = 0.0
        w = math.exp(float(x[0, 0]))  # (of the logit in fp32)
        Z = 1 + (V - 1) * w
        e = 2 * (V * 2.0 ** -(S + 1) + 2e-12 * Z) + 2.0 ** -S
        for p in (0.999, 1 - 2.0 ** -20, 1 - 2.0 ** -22, 1 - 2.0 ** -24):
            announce(f"flat tail V{V}, {halves} halves of a unit, top-p {p}")
            cut = ops.filter_logits(x.to(device()), top_p=p).cpu()
            kept = (cut > -math.inf).nonzero()[:, 1].view(2, -1)[0]
            n = kept.numel() - 1  # of the tail
            order = torch.cat([torch.tensor([V // 3]), torch.arange(V - 1) + (torch.arange(V - 1) >= V // 3)])
            assert torch.equal(kept, order[:n + 1].sort().values)
            assert 1 + n * w >= p * Z - e and (n == 0 or 1 + (n - 1) * w <= p * Z + e)
        tok = ops.sample_tokens(x.to(device()), u.to(device())).cpu()
        assert int(tok[0]) == V // 3
        at = int((order == tok[1]).nonzero())
        assert 1 + at * w >= float(u[1]) * Z - e and (at == 0 or 1 + (at - 1) * w <= float(u[1]) * Z + e)
