"""Dropout of tensors that no launch holds."""
import pytest

from helpers import capi

gpu = pytest.mark.gpu


@gpu
def test_more_elements_than_a_launch_holds_are_refused(rocm):
    """a thread takes 32 elements, a grid's dimension fewer than 2^32 threads: refused by the host, nothing is launched"""
    lib, h, x = rocm.device.lib, rocm.device.handle, rocm.zeros((4, 8))
    for rows, cols in ((2 ** 31 - 1, 128), (2 ** 30, 128), (2 ** 31 - 1, 2 ** 31 - 1)):
        for dtype in (0, 1):
            assert lib.rlt_rocm_dropout(h, dtype, x.ptr, cols, None, 0, x.ptr, cols, rows, cols, 0.5, 1, 2) == capi.RLT_E_UNSUPPORTED
    rocm.sync()
    assert not x.numpy().any()
