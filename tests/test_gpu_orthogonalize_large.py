"""orthogonalize where the 256 x 256 tiles run it with three products of
planes, to depths of thousands.

Tolerance: the kernels state that the planes' products give what fp32 products
give, so their error against 64 bits is at most that of the same steps by fp32
library products on the same input (measured in the test), plus one unit of
fp32's rounding, 2^-24."""

import pytest
import torch

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)


def plain(u, steps, coefficients, dtype):
    x = u.to(dtype)
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    a, b, c = coefficients
    for _ in range(steps):
        g = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def off_by(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("positive", [True, False])
@pytest.mark.parametrize("steps,coefficients", [(1, (1.0, 0.0, 1.0)), (1, (0.0, 1.0, 0.0)), (5, ABC)])
@pytest.mark.parametrize("shape", [(3600, 4000), (20, 800, 8000), (6, 2000, 2100)])
def test_fp32(spmm_npu, shape, steps, coefficients, positive):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    u = torch.randn(*shape, device="cuda", generator=g)
    u = u.abs() if positive else u
    want = plain(u, steps, coefficients, torch.float64)
    library = off_by(plain(u, steps, coefficients, torch.float32), want)
    own = off_by(spmm_npu.orthogonalize(u, steps, coefficients), want)
    assert own <= library + 2.0 ** -24, (own, library)


@pytest.mark.parametrize("shape", [(3600, 4000), (12, 1024, 2048)])
def test_fp16(spmm_npu, shape):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    u = torch.randn(*shape, device="cuda", generator=g).half()
    want = plain(u, 5, ABC, torch.float64)
    rounded = off_by(want.half(), want)
    assert off_by(spmm_npu.orthogonalize(u), want) <= rounded + 2e-6
