"""The dense operators' host side, without a GPU: their entry points exist and
their C ABI refuses, before any device call, what it cannot run, and sizes its
workspaces also for empty extents."""

import ctypes
import os

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "ascend-spmm_amd", "libspmm_mi355x.so")

F16, F32, F64, BF16 = 0, 1, 2, 3
I64 = ctypes.c_int64


class NormDesc(ctypes.Structure):
    _fields_ = [("rows", I64), ("width", I64), ("x_stride", I64), ("grad_stride", I64), ("eps", ctypes.c_double),
                ("value_type", ctypes.c_int32), ("param_type", ctypes.c_int32)]


class GroupedDesc(ctypes.Structure):
    _fields_ = [("rows", I64), ("groups", I64), ("inner", I64), ("width", I64), ("x_stride", I64),
                ("grad_stride", I64), ("weight_stride", I64), ("weight_transposed", ctypes.c_int32),
                ("index_type", ctypes.c_int32), ("value_type", ctypes.c_int32)]


class OrthogonalizeDesc(ctypes.Structure):
    _fields_ = [("batch", I64), ("rows", I64), ("width", I64), ("steps", I64),
                ("coefficients", ctypes.POINTER(ctypes.c_double)), ("eps", ctypes.c_double),
                ("value_type", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.fail(f"{LIB} is not built (python ascend-spmm_amd/build.py)")
    lib = ctypes.CDLL(LIB)
    lib.spmm_last_error.restype = ctypes.c_char_p
    return lib


FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every check precedes the launch


def norm(rows=8, width=16, x_stride=None, grad_stride=None, eps=1e-5, value=F16, param=F16):
    return NormDesc(rows, width, width if x_stride is None else x_stride,
                    width if grad_stride is None else grad_stride, eps, value, param)


def test_layer_norm_refusals(lib):
    run = lambda d, x=FAKE, y=FAKE: lib.spmm_layer_norm_run(ctypes.byref(d), x, FAKE, FAKE, y, None, None, None)  # noqa: E731
    for d, code, text in ((norm(value=F64), 4, b"FP16, BF16 and FP32"), (norm(value=F16, param=BF16), 4, b"type of x or FP32"),
                          (norm(rows=-1), 4, b"negative extent"), (norm(width=0), 4, b"1 <= width"),
                          (norm(width=1 << 31), 4, b"width < 2^31"), (norm(x_stride=15), 4, b"rows of x overlap"),
                          (norm(eps=-1.0), 1, b"eps must be finite"), (norm(eps=float("nan")), 1, b"eps must be finite")):
        assert run(d) == code and text in lib.spmm_last_error()
    assert run(norm(), x=None) == 1 and b"null device pointer" in lib.spmm_last_error()
    assert run(norm(rows=0), x=None, y=None) == 0
    assert lib.spmm_layer_norm_run(None, FAKE, FAKE, FAKE, FAKE, None, None, None) == 1


def test_layer_norm_gradient_refusals(lib):
    def run(d, ws=FAKE, size=1 << 30, dw=FAKE, mean=FAKE):
        return lib.spmm_layer_norm_grad_run(ctypes.byref(d), FAKE, FAKE, mean, FAKE, FAKE, FAKE, dw, None, ws,
                                            ctypes.c_size_t(size), None)
    assert run(norm(grad_stride=8)) == 4 and b"rows of grad overlap" in lib.spmm_last_error()
    assert run(norm(), size=0) == 4 and b"workspace too small" in lib.spmm_last_error()
    assert run(norm(), ws=None) == 4
    assert run(norm(), mean=None) == 1
    size = ctypes.c_size_t(0)
    for width in (1, 100, 5000, 1 << 20):
        assert lib.spmm_layer_norm_grad_workspace(ctypes.byref(norm(rows=100000, width=width)), ctypes.byref(size)) == 0
        # one row of partial sums for each work-group or chunk of rows
        assert 0 < size.value <= 8192 * 8 * width and size.value % (8 * width) == 0
    assert lib.spmm_layer_norm_grad_workspace(ctypes.byref(norm(rows=0)), ctypes.byref(size)) == 0


def grouped(rows=8, groups=2, inner=16, width=24, x_stride=None, grad_stride=None, weight_stride=None, index=0, value=F16):
    return GroupedDesc(rows, groups, inner, width, inner if x_stride is None else x_stride,
                       width if grad_stride is None else grad_stride,
                       inner * width if weight_stride is None else weight_stride, 0, index, value)


def test_grouped_refusals(lib):
    def run(d, x=FAKE, off=FAKE):
        return lib.spmm_grouped_run(ctypes.byref(d), x, FAKE, off, FAKE, None, ctypes.c_size_t(0), None)
    for d, text in ((grouped(index=5), b"int32 or int64"), (grouped(value=F64), b"FP16, BF16 and FP32"),
                    (grouped(rows=-1), b"negative extent"), (grouped(inner=1 << 22), b"below 2^22"),
                    (grouped(x_stride=1 << 22), b"below 2^22"), (grouped(x_stride=15), b"rows of x overlap"),
                    (grouped(weight_stride=16), b"matrices of weight overlap"), (grouped(rows=1 << 31), b"below 2^31")):
        assert run(d) == 4 and text in lib.spmm_last_error()
    assert run(grouped(), x=None) == 1 and run(grouped(), off=None) == 1
    assert run(grouped(rows=0), x=None, off=None) == 0
    assert run(grouped(rows=1 << 30, width=1 << 21), x=FAKE) == 3 and b"too many tiles" in lib.spmm_last_error()

    def back(d, ws=FAKE, size=1 << 40, grad=FAKE):
        return lib.spmm_grouped_grad_run(ctypes.byref(d), FAKE, FAKE, FAKE, grad, None, FAKE, ws, ctypes.c_size_t(size), None)
    assert back(grouped(grad_stride=8)) == 4 and b"rows of grad overlap" in lib.spmm_last_error()
    assert back(grouped(), grad=None) == 1
    # many rows for one matrix: its sum is cut, and the pieces need room
    assert back(grouped(rows=100000, groups=1), size=0) == 4 and b"workspace too small" in lib.spmm_last_error()


@pytest.mark.parametrize("value", [F16, F32, BF16])
def test_workspaces_of_empty_and_odd_extents(lib, value):
    size = ctypes.c_size_t(0)
    for sizes in ((0, 3, 16, 16), (5, 2, 0, 8), (5, 2, 8, 0), (6, 0, 8, 8), (0, 0, 0, 0), (100000, 12, 128, 128),
                  (65536, 8, 1024, 2048), (1, 1, 1, 1), (33, 1000, 5, 7)):
        d = grouped(*sizes, value=value)
        assert lib.spmm_grouped_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
        assert lib.spmm_grouped_grad_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
        assert size.value < 1 << 30
    c = (ctypes.c_double * 15)(*([3.4445, -4.775, 2.0315] * 5))
    for shape in ((0, 4, 4), (1, 0, 4), (1, 4, 0), (3, 1, 1), (1, 4096, 4096), (12, 512, 1024), (1, 7, 100000)):
        d = OrthogonalizeDesc(*shape, 5, c, 1e-7, value)
        assert lib.spmm_orthogonalize_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
        assert size.value <= 64 * shape[0] * max(shape[1], 64) * max(shape[2], 64) + (1 << 28)


def test_orthogonalize_refusals(lib):
    c = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)
    nan = (ctypes.c_double * 3)(3.4445, float("nan"), 2.0315)
    make = lambda batch=1, rows=300, width=300, steps=1, coefficients=c, eps=1e-7, value=F32: OrthogonalizeDesc(  # noqa: E731
        batch, rows, width, steps, coefficients, eps, value)
    run = lambda d, u=FAKE, size=1 << 40, ws=FAKE: lib.spmm_orthogonalize_run(  # noqa: E731
        ctypes.byref(d), u, FAKE, ws, ctypes.c_size_t(size), None)
    for d, code, text in ((make(value=F64), 4, b"FP16, BF16 and FP32"), (make(batch=-1), 4, b"negative extent"),
                          (make(batch=1 << 17), 4, b"at most 65535"), (make(rows=1 << 22), 4, b"below 2^22"),
                          (make(steps=-1), 1, b"steps"), (make(coefficients=None), 1, b"null coefficients"),
                          (make(coefficients=nan), 1, b"finite"), (make(eps=-1.0), 1, b"eps")):
        assert run(d) == code and text in lib.spmm_last_error()
    assert run(make(), u=None) == 1
    assert run(make(), size=1000) == 4 and b"workspace too small" in lib.spmm_last_error()
    assert run(make(), ws=None) == 4
    assert run(make(rows=0), u=None) == 0


def test_surface():
    import spmm_npu

    for name in ("layer_norm", "grouped_matmul", "orthogonalize"):
        assert callable(getattr(spmm_npu, name)) and name in spmm_npu.__all__
    for op in ("layer_norm", "grouped_matmul"):
        assert hasattr(torch.ops.myops, op)
    x = torch.zeros(3, 4)
    for call in (lambda: spmm_npu.layer_norm(x), lambda: spmm_npu.orthogonalize(x),
                 lambda: spmm_npu.grouped_matmul(x, torch.zeros(1, 4, 4), torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="must be a GPU tensor"):
            call()
