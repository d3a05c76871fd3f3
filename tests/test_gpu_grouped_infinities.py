"""Infinities and NaN in fp32 grouped products: wherever a product of the
factors is infinite or not a number, the result says what IEEE arithmetic
says, also against factors too small to be split into parts; results that meet
none are the same to the last bit as without them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def run(f, x, w, off, dy):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = f(x, w, off)
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy))


def wanted(x, w, off, dy):
    """In 64 bits, where none of these products or sums overflows."""
    x, w, dy, e = x.double().cpu(), w.double().cpu(), dy.double().cpu(), off.tolist()
    y, dx, dw = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w)
    for g, (a, b) in enumerate(zip(e, e[1:])):
        # one rank-one term after another: a library product may skip or reorder them
        for k in range(x.size(1)):
            y[a:b] += x[a:b, k:k + 1] * w[g, k]
        for k in range(w.size(2)):
            dx[a:b] += dy[a:b, k:k + 1] * w[g, :, k]
        for r in range(a, b):
            dw[g] += x[r, :, None] * dy[r]
    return y, dx, dw


# 2^-61 and below had zero parts, 2^-130 is below fp32's least normal value.
@pytest.mark.parametrize("small", [1.0, 2.0 ** -61, 2.0 ** -100, 2.0 ** -126, 2.0 ** -130])
@pytest.mark.parametrize("rows,inner,width", [(40, 64, 96), (70, 33, 49), (9, 128, 64), (300, 40, 130)])
def test_infinite_times_small(spmm_npu, rows, inner, width, small):
    g = torch.Generator().manual_seed(rows)
    signs = lambda *s: torch.randint(-1, 2, s, generator=g).float() * small  # noqa: E731
    x, w, dy = signs(rows, inner), signs(2, inner, width), signs(rows, width)
    off = torch.tensor([0, rows // 3, rows], dtype=torch.int32)
    clean = run(spmm_npu.grouped_matmul, x.cuda(), w.cuda(), off.cuda(), dy.cuda())
    x[1, 3], x[rows - 1, 0], x[rows - 2, 5], x[rows - 2, 6] = INF, -INF, INF, INF
    w[0, 7, 2] = -INF
    dy[2, 1], dy[rows - 3, 4] = INF, NAN
    got = run(spmm_npu.grouped_matmul, x.cuda(), w.cuda(), off.cuda(), dy.cuda())
    for a, b, c in zip(got, wanted(x, w, off, dy), clean):
        a, c = a.double().cpu(), c.double().cpu()
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a[b.isinf()], b[b.isinf()]) and b.isinf().any()
        assert torch.equal(a[b.isfinite()], c[b.isfinite()]) and b.isfinite().any()
