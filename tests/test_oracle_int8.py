"""oracle/int8.py against exact fractions and Python integers."""
from fractions import Fraction

import torch

from oracle import int8


def test_codes_are_exact_quotients():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20, 64, generator=g) * 3
    x[0] = torch.arange(64) * 0.5          # ties: a scale of 2^-2 (31.75 / 127) makes quotients of n + 1/2
    x[0, 1::2] += 0.125
    x[0, 63] = 31.75
    x[1] = 0
    q, s = int8.quantize_rows(x)
    for r in range(20):
        d = Fraction(float(s[r]))
        for k in range(64):
            v = Fraction(float(x[r, k]))
            want = round(v / d) if d else 0  # (Python rounds half to even)
            assert int(q[r, k]) == max(-127, min(127, want))
    assert float(s[0]) == 0.25 and int(q.abs().max()) == 127


def test_rows_that_are_not_finite():
    x = torch.ones(3, 8)
    x[1, 3], x[2, 0] = float("nan"), float("inf")
    q, s = int8.quantize_rows(x)
    assert s.isnan().tolist() == [False, True, True] and int(q[1:].abs().max()) == 0


def test_product_in_whole_numbers():
    g = torch.Generator().manual_seed(1)
    q = torch.randint(-127, 128, (3, 40), generator=g).to(torch.int8)
    W = torch.randint(-127, 128, (5, 40), generator=g).to(torch.int8)
    y = int8.product(q, torch.ones(3), W, torch.ones(5))
    for m in range(3):
        for n in range(5):
            assert int(y[m, n]) == sum(int(a) * int(b) for a, b in zip(q[m].tolist(), W[n].tolist()))
    y = torch.randn(2, 6, generator=g).double()
    assert torch.allclose(int8.swiglu(y), torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2])
