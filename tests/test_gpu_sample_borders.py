"""Truncated sampling where a border can go wrong, against oracle/sampling.py in 64 bits: what is kept and drawn is equal."""
import pytest
import torch

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
