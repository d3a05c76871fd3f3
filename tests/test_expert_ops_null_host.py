"""Null pointers that the operators around experts must refuse on the host
although a tensor of no columns needs no values."""

import ctypes

from test_expert_ops_host import FAKE, ex, lib  # noqa: F401  (lib is a fixture)


def test_restore_gradient_needs_weights_of_any_width(lib):  # noqa: F811
    def back(width, weights, y=FAKE, grad=FAKE, dy=FAKE, dw=FAKE):
        return lib.spmm_expert_restore_grad_run(ctypes.byref(ex(width=width)), y, weights, FAKE, FAKE, grad, dy, dw, None)

    for width in (0, 1, 16):
        for dy, dw in ((FAKE, FAKE), (None, FAKE), (FAKE, None)):
            assert back(width, None, dy=dy, dw=dw) == 1 and b"null device pointer" in lib.spmm_last_error()
    assert back(0, None, dy=None, dw=None) == 0  # nothing is asked for
