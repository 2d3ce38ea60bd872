"""Products in 8-bit integers with scales per token and channel, on the CPU in 64 bits (test infrastructure only).

  quantize_rows    s = fp32(max |x| / 127), codes rint(x / s) half to even; a row with a value that is not finite: codes 0, NaN
  norm_rows        x * rsqrt(mean x^2 + eps) * (1 + w) in 64 bits (HF:720-734)
  product          (sum_k q W) s w_scale, the sum in whole numbers
  swiglu           silu(gate) * up of interleaved (gate, up) columns (HF:704-717)

Pinned (tests/test_oracle_int8.py): codes against exact fractions, products against Python integers.
"""
import torch


def quantize_rows(x):
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    safe = torch.where(finite[..., None], x, 0.0)
    s = (safe.abs().amax(-1) / 127).float()
    d = s.double()[..., None]
    q = torch.where(d > 0, safe / torch.where(d > 0, d, 1.0), 0.0).round().clamp(-127, 127).to(torch.int8)
    return q, torch.where(finite, s, torch.nan)


def norm_rows(x, w, eps=1e-6):
    x = x.double()
    return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (1 + w.double())


def product(q, s, W, w_scale):
    """Doubles: |sum| stays below 2^53."""
    return (q.double() @ W.double().T) * s.double()[..., None] * w_scale.double()


def swiglu(y):
    g, u = y[..., 0::2], y[..., 1::2]
    return g * torch.sigmoid(g) * u
