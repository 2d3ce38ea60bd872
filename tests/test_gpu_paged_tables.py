"""The paged cache with rotation tables, block tables and batches out of the ordinary."""
import pytest
import torch

from gpu_util import announce, device
from oracle import paged
from q35hip import Q35Error, ops
from test_gpu_paged import append, make, oracle_append, same_pages, to

pytestmark = pytest.mark.gpu


def test_append_with_large_rotation_tables():
    """Tables that hold a scale beside the angles (cos and sin up to 4096): among 16 million rotated values some lie so near a
    tie that fp32 would give them the neighbouring code; codes and scales are those of 64 bits all the same."""
    d = make("int4", 2, 4096, 8, 8, 256, [4096, 4096], seed=6, rot=256)
    d["cos"], d["sin"] = d["cos"] * 4096, d["sin"] * 4096
    want, g = oracle_append(d), to(d, device())
    announce("paged append int4, large rotation tables")
    append(g)
    same_pages("int4", g["pages"], want)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_rows_of_65535_sequences(fmt):
    """As many sequences as the append and the attention take, two heads each; 65536 are refused."""
    dev = device()
    d = make(fmt, 1, 1, 2, 2, 16, [16 * 40], nb=40)
    B, T = 65535, 3
    table = torch.randint(0, 42, (B, 2), generator=torch.Generator().manual_seed(1)).int()
    pos = (torch.arange(B) % 31).int()  # (32 rows a table: some end past it)
    g = to(d, dev)
    announce(f"paged rows {fmt} of 65535 sequences")
    got = ops.paged_kv_rows(g["pages"], table.to(dev), pos.to(dev), T)
    at = pos.long()[:, None] + torch.arange(T)
    page, row = table.long().gather(1, (at // 16).clamp_max(1)), at % 16
    for x, i, which in zip(got, (0, 1), "kv"):
        sc = d["pages"][2 + i]
        values = paged.row_values(d["pages"][i], sc, which).bfloat16()  # [pages, 2, 16, 256]
        want = values[page, :, row] * (at < 32)[:, :, None, None]
        assert torch.equal(x.cpu(), want.transpose(1, 2))
    with pytest.raises(Q35Error):
        ops.paged_kv_rows(g["pages"], table[:1].expand(B + 1, 2).contiguous().to(dev), torch.zeros(B + 1, dtype=torch.int32, device=dev), 1)
