"""Sizes of layers in training that the C interface has no bits for are refused before any device work (no GPU)."""
import pytest
import torch

from neutronbench_amd import layers
from neutronbench_amd.layout import SampledLayer

MOST = 1 << 32


def of(*shape):
    return torch.empty(*shape, dtype=torch.bfloat16, device="meta")


@pytest.mark.parametrize("rows,columns", [(MOST, 1), (MOST + 8, 4), (1, MOST + 8)])
def test_rows_and_columns_of_more_than_32_bits(rows, columns):
    with pytest.raises(ValueError, match="2\\^32"):
        layers.DropoutOp(layers.Dropout(0.5, 1)).forward(of(rows, columns))
    with pytest.raises(ValueError, match="2\\^32"):
        layers.DenseOp().forward(of(rows, columns), of(4, columns))
    with pytest.raises(ValueError, match="2\\^32"):
        layers.DenseOp().forward(of(4, columns), of(rows, columns))
    sg = SampledLayer()
    sg.v_size, sg.src_size, sg.e_size = rows, 5, 0
    with pytest.raises(ValueError, match="2\\^32"):
        layers.DotAttentionOp(sg, 1).forward(of(rows, columns), of(5, columns), of(5, columns))
