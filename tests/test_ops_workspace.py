"""The backward pass of wide rows: its workspace holds sums of rows, and no more of them than there are wavefronts with rows."""

import ctypes

import pytest

from odc_amd import _native


def workspace(rows, width, dtype):
    _native.load_ops()
    f = ctypes.CFUNCTYPE(ctypes.c_uint64, ctypes.c_uint64, ctypes.c_uint64, ctypes.c_int32)(("odc_layer_norm_backward_workspace", _native._ops_lib))
    return f(rows, width, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("width", [3, 20000, 33001, 1 << 20, 1 << 26])
def test_a_group_has_a_row_for_each_of_its_wavefronts(dtype, width):
    for rows in (1, 2, 3, 4, 5, 63, 64, 255, 256, 257, 1000, 1024, 4096, 100_000):
        groups = workspace(rows, width, dtype) / (8 * width)
        assert groups == int(groups) and 1 <= groups <= min(256, -(-rows // 4))


@pytest.mark.parametrize("dtype,size", [(0, 2), (2, 4)])
def test_a_few_long_rows_need_little(dtype, size):
    """It was 2 GiB for an input of 512 MiB."""
    assert workspace(256, 1 << 20, dtype) <= 256 * (1 << 20) * size // 16
