"""Rows in 8 bits on the GPU where the scale is subnormal, against oracle/int8.py: codes and scales are equal."""
import pytest
import torch

from gpu_util import announce, device
from oracle import int8
from q35hip import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [8, 512, 1024, 3584])
def test_codes_where_the_scale_is_subnormal(K):
    """Scales of one to a few units of 2^-149: rounded by up to a third, the quotients pass 127 and the codes stay there."""
    tops = torch.tensor([1, 63, 64, 126, 127, 128, 190, 191, 254, 300, 317, 318, 444, 1000, 20000], dtype=torch.float64)
    x = torch.arange(K, dtype=torch.float64) / (K - 1) * 2 - 1
    x = ((x * tops[:, None]).round() * 2.0 ** -149).float()
    x[:, 0], x[:, -1] = -x[:, -1], x[:, -1].clone()
    wq, ws = int8.quantize_rows(x)
    assert int((x.double().abs().amax(-1) / ws.double().clamp_min(1e-300))[6]) == 190
    announce(f"quantize_rows subnormal K{K}")
    q, s = ops.quantize_rows(x.to(device()))
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws) and int(q.abs().max()) == 127
