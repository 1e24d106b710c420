"""Edges of the dense operators that need no GPU: the layout of split sums."""
import ctypes

import pytest

from maba_v2_architecture_b200 import _native as N


@pytest.mark.parametrize("splits,pairs", [(2, 1), (16, 1), (10, 2)])
@pytest.mark.parametrize("rows", [1, 2, 33])
def test_split_sums_stay_in_their_buffer(rows, splits, pairs):
    """A split's sums start where the one before ends, rows of ``cols`` up to a multiple of four: the
    last element stored ends a row's padding before the end of what was reserved, whatever the size."""
    reserved, reached = ctypes.c_int64(), ctypes.c_int64()
    for cols in [*range(1, 41), 100, 650, 1003, 1251, 2048]:
        rc = N.lib().maba_selftest_split_layout(rows, cols, splits, pairs, ctypes.byref(reserved), ctypes.byref(reached))
        assert rc == N.OK
        padded = (cols + 3) // 4 * 4
        assert reserved.value == 4 * splits * pairs * rows * padded
        assert reached.value == reserved.value - 4 * (padded - cols), cols


def test_split_layout_refusals():
    v = ctypes.c_int64()
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        assert N.lib().maba_selftest_split_layout(*bad, ctypes.byref(v), ctypes.byref(v)) == N.ERR_INVALID
    assert N.lib().maba_selftest_split_layout(1, 1, 1, 1, None, ctypes.byref(v)) == N.ERR_INVALID
