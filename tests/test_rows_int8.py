"""What the layers refuse of rows in 8 bits, without a GPU: arguments that such rows cannot follow are not dropped in silence."""
import pytest
import torch

from q35hip import layers, model, ops


def rows(*shape):
    return ops.RowsI8(torch.zeros(*shape, dtype=torch.int8), torch.ones(shape[:-1]))


def mlp_params(H=64, I=128):
    p = {}
    for n, shape in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
        p[n], p[n + ".q"], p[n + ".s"] = torch.zeros(shape), torch.zeros(shape, dtype=torch.int8), torch.ones(shape[0])
    return p


def test_mlp_of_rows_in_8_bits_takes_no_prenorm():
    """The add and the norm that prenorm asks for cannot follow the rounding."""
    p, x = mlp_params(), torch.zeros(2, 6, 64)
    for y in (None, torch.ones(2, 6, 64)):
        with pytest.raises(ValueError, match="prenorm"):
            model.mlp(p, rows(2, 6, 64), x, prenorm=(y, torch.zeros(64), 1e-6))
    assert bool((x == 0).all())


def test_linear_of_rows_in_8_bits_takes_no_prenorm_and_no_conv():
    w, q, s = torch.zeros(256, 64), torch.zeros(256, 64, dtype=torch.int8), torch.ones(256)
    for M in (1, 3, 20):
        with pytest.raises(ValueError, match="prenorm"):
            layers.linear(rows(M, 1, 64), w, q, s, prenorm=(None, torch.zeros(64), 1e-6, None))
        with pytest.raises(ValueError, match="conv"):
            layers.linear(rows(M, 1, 64), w, q, s, conv=(torch.zeros(128, 4), None, torch.zeros(M, 128, 3)))
        with pytest.raises(ValueError, match="one scale per row"):
            layers.linear(rows(M, 1, 64), w, q, torch.ones(256, 2))
