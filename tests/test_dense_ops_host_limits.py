"""Refusals of the dense operators' C ABI at the edges of a launch, without a
GPU: they come before any device call."""

import ctypes

from test_dense_ops_host import F16, FAKE, LIB, GroupedDesc


def test_more_work_items_than_a_grid_holds():
    """2^24 groups are accepted, but not where their tiles need a grid of 2^32
    work-items or more: an error of its own, not a failed launch."""
    lib = ctypes.CDLL(LIB)
    lib.spmm_last_error.restype = ctypes.c_char_p
    d = GroupedDesc(8, 1 << 24, 16, 16, 16, 16, 256, 0, 0, F16)
    assert lib.spmm_grouped_run(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, None, ctypes.c_size_t(0), None) == 3
    assert b"too many tiles" in lib.spmm_last_error()
