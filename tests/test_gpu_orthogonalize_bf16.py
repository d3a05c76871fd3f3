"""The precision of bf16 updates: by default, with factors of 11 bits, near the
rounding of the result to 8 bits; with precise=True that rounding alone.

Tolerances, in the 2-norm: rounding to 8 bits is 1.66e-3 of a result with
evenly spread digits (2^-8 / sqrt(12) of the spacing's mean); 15 factors of 11
bits add 15 roundings of 2^-12 / sqrt(3) each, 5.5e-4 together, twice that
where weak directions grow: below 3e-3 in all, and 6e-3 where noise of 5e-3 or
less grows beside strong directions.  precise: the rounding of the exact
result, measured, and 2e-6 for fp32's own errors."""

import ctypes

import pytest
import torch

from test_dense_ops_host import BF16, LIB, OrthogonalizeDesc

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)


def exact(u):
    x = u.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    tall = x.size(-2) > x.size(-1)
    if tall:
        x = x.transpose(-2, -1).contiguous()
    a, b, c = ABC
    for _ in range(5):
        g = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.transpose(-2, -1).contiguous() if tall else x


def off_by(got, want):
    return float((got.double() - want).norm() / want.norm())


def noisy(m, n, rank, noise, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return (rand(m, rank) @ rand(rank, n) + noise * rand(m, n)).bfloat16()


CASES = [(130, 257, 20, 1.0, 3e-3), (512, 256, 40, 1.0, 3e-3), (640, 640, 80, 1.0, 3e-3), (512, 1024, 64, 1.0, 3e-3),
         (200, 260, 4, 5e-3, 6e-3), (300, 200, 4, 5e-3, 6e-3), (200, 260, 1, 1e-3, 6e-3), (700, 700, 1, 1e-3, 6e-3)]


@pytest.mark.parametrize("m,n,rank,noise,most", CASES)
def test_default(spmm_npu, m, n, rank, noise, most):
    u = noisy(m, n, rank, noise)
    assert off_by(spmm_npu.orthogonalize(u), exact(u)) <= most


@pytest.mark.parametrize("m,n,rank,noise", [c[:4] for c in CASES] + [(2000, 2100, 250, 1.0), (64, 48, 8, 1.0)])
def test_precise(spmm_npu, m, n, rank, noise):
    u = noisy(m, n, rank, noise)
    want = exact(u)
    growth = 1.0 if noise == 1.0 else 3.4445 ** 4
    assert off_by(spmm_npu.orthogonalize(u, precise=True), want) <= off_by(want.bfloat16(), want) + 2e-6 * growth


def test_precise_changes_nothing_for_others(spmm_npu):
    for dtype in (torch.float16, torch.float32):
        u = noisy(200, 300, 10, 1.0).to(dtype)
        assert torch.equal(spmm_npu.orthogonalize(u, precise=True), spmm_npu.orthogonalize(u))


def test_precise_through_the_c_abi(spmm_npu):
    """The descriptor's last field, in what was padding: 0 where it is not set."""
    class Desc(ctypes.Structure):
        _fields_ = OrthogonalizeDesc._fields_ + [("precise", ctypes.c_int32)]

    assert ctypes.sizeof(Desc) == ctypes.sizeof(OrthogonalizeDesc)
    lib = ctypes.CDLL(LIB)
    u = noisy(200, 300, 10, 1.0)
    c = (ctypes.c_double * 15)(*(ABC * 5))
    for precise in (0, 1):
        d = Desc(1, 200, 300, 5, c, 1e-7, BF16, precise)
        size = ctypes.c_size_t(0)
        assert lib.spmm_orthogonalize_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
        ws, out = torch.empty(size.value, dtype=torch.uint8, device="cuda"), torch.empty_like(u)
        p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
        assert lib.spmm_orthogonalize_run(ctypes.byref(d), p(u), p(out), p(ws), size,
                                          ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        assert torch.equal(out, spmm_npu.orthogonalize(u, precise=bool(precise)))
