"""The paged cache with rotation tables, block tables and batches out of the ordinary."""
import pytest
import torch

from gpu_util import announce, device
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
