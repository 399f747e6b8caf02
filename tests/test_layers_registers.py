"""Registers of the kernels of layers in training, as their launches count on (no GPU)."""
import pytest
from test_kernel_registers import kernels  # noqa: F401  (a fixture)

# (name, kernels, most vector registers of a lane, most bytes of scratch memory of a lane)
EXPECTED = [
    ("dense_rows_kernelIf", 4, 256, 0), ("dense_rows_kernelINS_4Bf16E", 4, 168, 0), ("dense_rows_kernelINS_3F16E", 4, 168, 0),
    ("dense_wide_kernel", 6, 256, 0), ("dense_weight_kernelIf", 2, 256, 0), ("dense_weight_kernelINS_4Bf16ELb1E", 3, 168, 0),
    ("dense_few_kernel", 6, 128, 0), ("dense_columns_kernel", 3, 64, 0), ("dense_sum_kernel", 3, 64, 0),
    # attention: lanes of a head 1, 2, 4, 8 and 16; the block's 1,024 threads leave 128 registers, one of which may go to memory
    ("dot_block_kernel", 30, 128, 8), ("join_dot_spans_kernel", 9, 128, 0),
    ("dot_rows_kernelINS_4Bf16", 30, 256, 0), ("dot_rows_kernelINS_3F16", 30, 256, 0), ("dot_rows_kernelIf", 30, 256, 16),
    ("16dot_spans_kernelINS_4Bf16", 75, 256, 0), ("16dot_spans_kernelINS_3F16", 75, 256, 0), ("16dot_spans_kernelIf", 75, 256, 12),
]


@pytest.mark.parametrize("kernel,number,most,scratch", EXPECTED)
def test_registers(kernels, kernel, number, most, scratch):  # noqa: F811
    found = [k for name, k in kernels.items() if kernel in name]
    assert len(found) == number
    for k in found:
        assert k[".vgpr_count"] <= most and k[".private_segment_fixed_size"] <= scratch
