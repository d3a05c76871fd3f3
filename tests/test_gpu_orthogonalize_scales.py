"""orthogonalize of updates whose rows, columns or whole are far smaller than
the range that a scale for the whole matrix covers: rarely active features,
and updates whose norm is far below eps.

Tolerances: fp32 results are held to what fp32 products give on the same
input (the library's error against 64 bits, measured in the test), each weak
part against its own 2-norm: at most twice that, and 2^-22 for the planes' 22
bits.  bf16 and fp16 results are rounded to 8 and 11 bits, and bf16 factors to
11: 1.25 times the rounding of the exact result."""

import pytest
import torch

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)


def plain(u, dtype, steps=5, eps=1e-7):
    x = u.to(dtype)
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.size(-2) > x.size(-1)
    if tall:
        x = x.transpose(-2, -1).contiguous()
    a, b, c = ABC
    for _ in range(steps):
        g = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.transpose(-2, -1).contiguous() if tall else x


def off_by(got, want):
    return float((got.double() - want).norm() / want.norm())


def held(u, got, part, what):
    """`part` takes the weak rows or columns of a matrix."""
    want = plain(u, torch.float64)
    assert off_by(got, want) <= limit(u, want, lambda t: t), what
    assert off_by(part(got), part(want)) <= limit(u, want, part), what


def limit(u, want, part):
    if u.dtype == torch.float32:
        return 2 * off_by(part(plain(u, torch.float32)), part(want)) + 2.0 ** -22
    return 1.25 * off_by(part(want.to(u.dtype)), part(want))


SHAPES = [(100, 140), (140, 100), (30, 400), (256, 512), (512, 256), (2, 300, 700), (1200, 200)]


@pytest.mark.parametrize("scale", [1e-3, 1e-5, 1e-7, 1e-8, 1e-14])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_weak_rows_and_columns(spmm_npu, shape, dtype, scale):
    for rows in (True, False):
        part = (lambda t: t[..., 3:11, :]) if rows else (lambda t: t[..., 3:11])  # noqa: E731
        u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(shape[-1]))
        part(u).mul_(scale)
        u = u.to(dtype)
        held(u, spmm_npu.orthogonalize(u), part, (rows, scale))


@pytest.mark.parametrize("shape", SHAPES)
def test_graded_rows_and_columns(spmm_npu, shape):
    """Scales falling from 1 to 1e-9 along the rows and along the columns: every
    row and every column on its own."""
    u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(shape[-2]))
    m, n = shape[-2:]
    for down, across in ((9, 0), (0, 9), (5, 6)):
        g = u * torch.logspace(0, -down, m, device="cuda")[:, None] * torch.logspace(0, -across, n, device="cuda")
        got, want, library = spmm_npu.orthogonalize(g).double(), plain(g, torch.float64), plain(g, torch.float32)
        for dim in (-1, -2):
            size = want.norm(dim=dim)
            own, other = ((t.double() - want).norm(dim=dim) / size for t in (got, library))
            assert float(own.max()) <= 2 * float(other.max()) + 2.0 ** -22, (down, across, dim)


@pytest.mark.parametrize("norm", [1e-6, 1e-8, 1e-10, 1e-12, 1e-13, 1e-15, 1e-16, 1e-25, 1e-30])
@pytest.mark.parametrize("shape", [(96, 128), (128, 96), (16, 16), (300, 500), (500, 300), (3, 260, 300)])
def test_updates_far_below_eps(spmm_npu, shape, norm):
    u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(shape[-1]))
    u = (u.double() * (norm / u.double().square().sum((-2, -1), keepdim=True).sqrt())).float()
    held(u, spmm_npu.orthogonalize(u), lambda t: t, norm)


@pytest.mark.parametrize("shape", [(96, 128), (300, 500), (500, 300)])
def test_bf16_far_below_eps(spmm_npu, shape):
    for norm in (1e-8, 1e-13, 1e-20, 1e-30):
        u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(shape[-1]))
        u = (u * (norm / float(u.double().norm()))).bfloat16()
        held(u, spmm_npu.orthogonalize(u), lambda t: t, norm)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(60, 90), (300, 400), (400, 300)])
def test_zero_rows_and_columns(spmm_npu, shape, dtype):
    u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    u[5] = 0
    u[:, 7] = 0
    got = spmm_npu.orthogonalize(u)
    assert not got[5].any() and not got[:, 7].any()
    held(u, got, lambda t: t, "zeros")


@pytest.mark.parametrize("shape", [(40, 30), (300, 400)])
def test_no_steps_is_the_scaled_update(spmm_npu, shape):
    """X0 alone: rounded once, from the quotient in 64 bits."""
    u = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    u[2] *= 1e-20
    want = plain(u, torch.float64, steps=0)
    assert bool(((spmm_npu.orthogonalize(u, 0).double() - want).abs() <= (2.0 ** -24 + 2.0 ** -50) * want.abs()).all())
