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


def adapters(n, rank, size):
    return _cabi.Adapters(a_dev=1 << 40, b_dev=1 << 41, scale_dev=1 << 42, n=n, in_size=size, out_size=size, rank=rank, w_dtype=2, reserved=0)


@pytest.mark.parametrize("rows, n, turned", [(0, 5, 0), (1, 65535, 1), (65, 1000, 65), (8, 8, 8), (8, 9, 8), (1000, 1000, 1000), (4096, 4, 4)])
def test_adapter_scratch_has_matrices_for_no_more_adapters_than_rows(rows, n, turned):
    """A float of b^T d for every row and rank, the matrices turned (bf16), and sums of up to a chunk's rows where adapters can have
    more rows than that."""
    w = adapters(n, 16, 512)
    size = _cabi.lib().rpu_adapter_backward_scratch(C.byref(w), rows) - 4 * rows * 16 - 2 * turned * 16 * 2 * 512
    assert size % (4 * 16 * 1024) == 0 and 0 <= size // (4 * 16 * 1024) <= 2 * rows // 128
