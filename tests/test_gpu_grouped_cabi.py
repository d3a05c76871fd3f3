"""The grouped products' C entry points with what the torch operators never
pass: strides of a single row, which the descriptor leaves open, and results at
any element.

Tolerances as in test_gpu_grouped.py: one rounding of the output to its type,
and (terms + 2) 2^-24 of the terms' magnitudes."""

import ctypes
import os

import pytest
import torch

from test_dense_ops_host import BF16, F16, F32, LIB, GroupedDesc

pytestmark = pytest.mark.gpu

TYPES = [(torch.float16, F16), (torch.bfloat16, BF16), (torch.float32, F32)]
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def lib(spmm_npu):
    lib = ctypes.CDLL(LIB)
    lib.spmm_last_error.restype = ctypes.c_char_p
    return lib


def at(t):
    return ctypes.c_void_p(t.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def close(got, want, mag, terms, dtype):
    want, mag = want.cpu(), mag.cpu()
    limit = U[dtype] * want.abs() + (terms + 2) * 2.0 ** -24 * mag * (1 + U[dtype]) + 2.0 ** -24 * (dtype == torch.float16)
    return bool(((got.double().cpu() - want).abs() <= limit).all())


@pytest.mark.parametrize("stride", [0, 8, -3, 1, 1 << 40])
@pytest.mark.parametrize("dtype,value", TYPES)
@pytest.mark.parametrize("inner,width,turned", [(64, 96, 0), (64, 96, 1), (256, 384, 0), (33, 17, 0)])
def test_one_row_of_any_stride(lib, inner, width, turned, dtype, value, stride):
    g = torch.Generator(device="cuda").manual_seed(inner + width)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    x, grad, w = rand(1, inner), rand(1, width), rand(2, *((width, inner) if turned else (inner, width)))
    offsets = torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    d = GroupedDesc(1, 2, inner, width, stride, stride, inner * width, turned, 0, value)
    size = ctypes.c_size_t(0)
    assert lib.spmm_grouped_grad_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
    ws = torch.empty(max(size.value, 1), dtype=torch.uint8, device="cuda")
    y, dx, dw = torch.empty_like(grad), torch.empty_like(x), torch.full_like(w, float("nan"))
    assert lib.spmm_grouped_run(ctypes.byref(d), at(x), at(w), at(offsets), at(y), None, ctypes.c_size_t(0), stream()) == 0
    assert lib.spmm_grouped_grad_run(ctypes.byref(d), at(x), at(w), at(offsets), at(grad), at(dx), at(dw), at(ws),
                                     size, stream()) == 0, lib.spmm_last_error()
    xd, gd, wd = x.double(), grad.double(), (w[1].t() if turned else w[1]).contiguous().double()
    outer = (xd.t() * gd).t().contiguous() if turned else xd.t() * gd
    assert close(dw[1], outer, outer.abs(), 1, dtype) and not dw[0].any()
    assert close(y, xd @ wd, xd.abs() @ wd.abs(), inner, dtype)
    wt = wd.t().contiguous()
    assert close(dx, gd @ wt, gd.abs() @ wt.abs(), width, dtype)


@pytest.mark.parametrize("turned", [0, 1])
@pytest.mark.parametrize("dtype,value", TYPES)
@pytest.mark.parametrize("sizes,inner,width", [([25000, 24999], 256, 264), ([5, 0, 9], 256, 264), ([300, 700], 128, 136),
                                               ([9000], 136, 128)])
def test_results_at_any_element(lib, sizes, inner, width, dtype, value, turned):
    """out, dx and dweight one element off a 16-byte boundary: the same bits as on
    one, and nothing beside them is written."""
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    rows, groups = sum(sizes), len(sizes)
    x, grad, w = rand(rows, inner), rand(rows, width), rand(groups, *((width, inner) if turned else (inner, width)))
    offsets = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    d = GroupedDesc(rows, groups, inner, width, inner, width, inner * width, turned, 0, value)
    size = ctypes.c_size_t(0)
    assert lib.spmm_grouped_grad_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
    ws = torch.empty(max(size.value, 1), dtype=torch.uint8, device="cuda")

    def run(shift):
        flat = [torch.full((n + 2 * 64,), 7.0, device="cuda", dtype=dtype) for n in (rows * width, rows * inner, w.numel())]
        to = [ctypes.c_void_p(t.data_ptr() + (64 + shift) * t.element_size()) for t in flat]
        assert lib.spmm_grouped_run(ctypes.byref(d), at(x), at(w), at(offsets), to[0], None, ctypes.c_size_t(0), stream()) == 0
        assert lib.spmm_grouped_grad_run(ctypes.byref(d), at(x), at(w), at(offsets), at(grad), to[1], to[2], at(ws), size,
                                         stream()) == 0
        for t in flat:
            assert bool((t[:64 + shift] == 7).all()) and bool((t[t.numel() - 64 + shift:] == 7).all())
        return [t[64 + shift:t.numel() - 64 + shift] for t in flat]

    for a, b in zip(run(0), run(1)):
        assert torch.equal(a, b)
