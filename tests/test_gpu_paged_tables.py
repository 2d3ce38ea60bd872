"""The paged cache with rotation tables, block tables and batches out of the ordinary."""
import pytest
import torch

from gpu_util import announce, device
from oracle import paged
from q35hip import Q35Error, layers, ops
from test_gpu_paged import append, attend, check_attention, make, oracle_append, same_pages, to

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


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_a_captured_layer(fmt):
    """The attention layer in a HIP graph: refused while its rotation tables are not there, and once they are each replay at
    new positions gives what the eager call gives."""
    dev = device()
    g = torch.Generator().manual_seed(7)
    B, nb = 3, 6
    p = {n: (torch.randn(*s, generator=g) * 0.05).to(dev)
         for n, s in (("q_proj", (1024, 256)), ("k_proj", (256, 256)), ("v_proj", (256, 256)), ("o_proj", (256, 512)))}
    p["q_norm"], p["k_norm"] = (0.1 * torch.randn(256, generator=g).to(dev) for _ in range(2))
    table = torch.randperm(B * nb, generator=g).view(B, nb).int().to(dev)
    mine, eager = (ops.kv_pages(B * nb, 1, 32, dev, fmt) for _ in range(2))
    x, pos = torch.randn(B, 1, 256, generator=g).to(dev), torch.zeros(B, dtype=torch.int32, device=dev)
    theta = 1e7 + (fmt == "int4")  # (tables of this test's own)
    announce(f"paged layer captured {fmt}")
    with pytest.raises(Q35Error, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            layers.gated_attention_layer_paged(x, p, mine, table, pos, rope_theta=theta + 2)
    layers.gated_attention_layer_paged(x, p, mine, table, pos, rope_theta=theta)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layers.gated_attention_layer_paged(x, p, mine, table, pos, rope_theta=theta)
    for step in range(5):
        x.copy_(torch.randn(B, 1, 256, generator=g).to(dev))
        graph.replay()
        want = layers.gated_attention_layer_paged(x, p, eager, table, pos, rope_theta=theta)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(mine, eager):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        pos += torch.tensor([1, 0, 1], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
@pytest.mark.parametrize("T", [1, 5])
def test_one_table_for_all_rows(fmt, T):
    """Several rows of queries over one sequence's pages, its table expanded: as with the table repeated."""
    d = make(fmt, 3, T, 8, 2, 16, [300, 290, 17], seed=9)
    d["table"] = d["table"][:1].repeat(3, 1)
    g = to(d, device())
    announce(f"paged {fmt} T{T}, an expanded table")
    one = dict(g, table=g["table"][:1].expand(3, -1))
    out = attend(one)
    check_attention(d, out)
    assert torch.equal(out, attend(g))
    for a, b in zip(*(ops.paged_kv_rows(x["pages"], x["table"], x["pos"], T) for x in (one, g))):
        assert torch.equal(a, b)
