"""orthogonalize with the result in the update's place, which the C ABI allows:
the same bits as into another tensor, for the kernel that holds a matrix in
LDS, for those of many launches, and without steps."""

import ctypes

import pytest
import torch

from test_dense_ops_host import BF16, F16, F32, LIB, OrthogonalizeDesc

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("dtype,value", [(torch.float16, F16), (torch.bfloat16, BF16), (torch.float32, F32)])
@pytest.mark.parametrize("shape", [(1, 40, 56), (5, 128, 96), (3, 33, 1100), (2, 300, 200), (1, 500, 700)])
@pytest.mark.parametrize("steps", [0, 1, 5])
def test_in_place(spmm_npu, shape, steps, dtype, value):
    u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(steps)).to(dtype)
    want = spmm_npu.orthogonalize(u, steps)
    lib = ctypes.CDLL(LIB)
    c = (ctypes.c_double * max(1, 3 * steps))(*(ABC * steps))
    d = OrthogonalizeDesc(*shape, steps, c, 1e-7, value)
    size = ctypes.c_size_t(0)
    assert lib.spmm_orthogonalize_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
    ws = torch.empty(max(1, size.value), dtype=torch.uint8, device="cuda")
    at = ctypes.c_void_p(u.data_ptr())
    assert lib.spmm_orthogonalize_run(ctypes.byref(d), at, at, ctypes.c_void_p(ws.data_ptr()), size,
                                      ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(u, want)
