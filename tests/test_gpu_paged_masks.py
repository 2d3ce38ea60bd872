"""Garbage in masked places of a paged cache, over keys of several rounds, blocks of four and eight waves, and joined runs."""
import math

import pytest
import torch

from gpu_util import announce, device
from test_gpu_paged import attend, check_attention, make, to

pytestmark = pytest.mark.gpu

# keys of the table, contexts: ends in the second, third and fifth round of 128 keys, one key into one, and at its border; for
# 70 rows the blocks that a CU holds differ
CASES = [(256, [200, 129]), (384, [300, 261]), (384, [257, 383]), (512, [500, 256]), (640, [600, 300]),
         (384, [384 - 7 * (b % 50) for b in range(70)])]


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("keys,ctx", CASES)
def test_masked_places_hold_anything(fmt, T, splits, keys, ctx):
    """Rows past a sequence's end, pages that no entry names (a whole round's entries of one row among them), the first page of
    the pool, and for earlier tokens the last token's own value: NaN and infinities change no output that does not attend to
    them, bit for bit, and the outputs are those of the formula."""
    B = len(ctx)
    d = make(fmt, B, T, 4, 1, 16, ctx, seed=keys + B, nb=keys // 16)
    used = d["table"] == 0
    d["table"][used] = min(set(range(d["pages"][0].shape[0])) - set(d["table"].flatten().tolist()))
    if keys > 256:
        d["table"][1, 8:16] = torch.tensor([-1, 99999] * 4, dtype=torch.int32)
    d["table"][0, 3] = -7
    announce(f"paged attention {fmt} T{T} splits {splits} garbage over {keys} keys, {B} rows")
    g = to(d, device())
    clean = attend(g, splits=splits)
    check_attention(d, clean)
    pages = tuple(None if p is None else p.clone() for p in d["pages"])
    spare = sorted(set(range(pages[0].shape[0])) - set(d["table"].flatten().tolist()))
    assert 0 in spare
    for i in (0, 1) if fmt == "bf16" else (2, 3):
        pages[i][spare] = math.nan
        pages[i][spare[0], :, ::2] = math.inf
        for b in range(B):
            for at in range(ctx[b], keys):
                page = int(d["table"][b, at // 16])
                if 0 <= page < pages[0].shape[0]:
                    pages[i][page, :, at % 16] = (math.nan, math.inf, -math.inf)[at % 3]
    last = [b for b in range(B) if T > 1 and 0 <= int(d["table"][b, (ctx[b] - 1) // 16]) < pages[0].shape[0]]
    for b in last:
        pages[1 if fmt == "bf16" else 3][int(d["table"][b, (ctx[b] - 1) // 16]), :, (ctx[b] - 1) % 16] = -math.inf
    out = attend(dict(g, pages=tuple(None if p is None else p.to(device()) for p in pages)), splits=splits)
    keep = slice(0, T - 1) if T > 1 else slice(0, 1)
    assert torch.equal(out[:, keep], clean[:, keep])
    if T > 1:
        assert not bool(torch.isfinite(out[last, -1]).any())
