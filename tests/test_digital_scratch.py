"""Scratch memory of the digital operators: what the kernels use, and no more, without a GPU."""
import ctypes as C

import pytest

from aihwkit_amd import _cabi

CUS = 256                                        # compute units of an MI355X


@pytest.mark.parametrize("rows, cols, workgroups", [
    (1, 768, 1), (16, 768, 1), (17, 768, 2), (1 << 20, 768, CUS), (50000, 64, 2 * CUS), (8192, 512, 2 * CUS), (8192, 1537, 3 * CUS),
    (8192, 4096, 3 * CUS), (100, 4096, 50), (8192, 4097, CUS), (8192, 16384, CUS), (1 << 20, 100000, CUS), (3, 1 << 24, 2),
])
def test_layer_norm_scratch_is_a_row_of_sums_for_every_workgroup(rows, cols, workgroups):
    """Weight's and bias' sums of each workgroup, floats; no workgroup has less than two rows (of eight waves up to 1024 columns)."""
    assert _cabi.lib().rpu_layer_norm_backward_scratch(rows, cols) == workgroups * 2 * cols * 4
