"""Long fp32 sums of grouped products.

Tolerance: the products of fp32 factors are split into parts whose sum is off
by at most 4 * 2^-24 of a product, and every 32 of them, together, and every
addition of such a group to the sum are rounded.  A sum of n groups added one
after another that rounds each time without preference is off by about
sqrt(n) 2^-25 of the partial sums, one that cuts to the same side by n 2^-25.
In the 2-norm over a whole result, n additions are allowed 2 sqrt(n) 2^-25 of
the partial sums' size (at most the terms' magnitudes), and the parts 2^-22."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def limit(terms):
    return 2.0 ** -22 + 2 * (terms / 32) ** 0.5 * 2.0 ** -25


def off_by(got, want, magnitude):
    """The 2-norm of the error against that of the terms' magnitudes."""
    return float((got.double() - want).norm() / magnitude.norm())


@pytest.mark.parametrize("positive", [True, False])
@pytest.mark.parametrize("rows,inner,width", [(64, 65536, 64), (512, 2048, 256), (65536, 512, 768), (131072, 130, 70),
                                              (50, 33001, 47)])
def test_long_sums(spmm_npu, rows, inner, width, positive):
    g = torch.Generator(device="cuda").manual_seed(rows + inner)
    draw = torch.rand if positive else torch.randn
    x, w, dy = (draw(*s, device="cuda", generator=g) for s in ((rows, inner), (1, inner, width), (rows, width)))
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    x.requires_grad_(True), w.requires_grad_(True)
    y = spmm_npu.grouped_matmul(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    a, b, d = x.detach().double(), w.detach()[0].double(), dy.double()
    at, bt = a.t().contiguous(), b.t().contiguous()
    for got, p, q, terms, what in ((y.detach(), a, b, inner, "y"), (dx, d, bt, width, "dx"), (dw[0], at, d, rows, "dw")):
        off = off_by(got, p @ q, p.abs() @ q.abs())
        assert off <= limit(terms), (what, off, limit(terms))
