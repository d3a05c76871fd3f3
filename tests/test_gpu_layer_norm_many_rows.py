"""layer_norm with more rows than its launches have work-groups, so that these
walk on to further rows: just past each limit, rows of a part of a wave, of
several waves, and wider than the registers hold.

Tolerances as in test_gpu_layer_norm.py."""

import pytest
import torch

from test_gpu_layer_norm import E32, TINY, U, check, make, plain

pytestmark = pytest.mark.gpu


# 4096 work-groups forward and 512 backward, of 32, 16, 4 and one row.
@pytest.mark.parametrize("rows,n,dtype", [(140001, 9, torch.float16), (70001, 128, torch.float16), (33001, 520, torch.bfloat16),
                                          (17001, 250, torch.float32), (4099, 2056, torch.float16), (4101, 1500, torch.float32)])
def test_forward_and_gradients(spmm_npu, rows, n, dtype):
    x, w, b, dy = make(rows, n, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = spmm_npu.layer_norm(x, w, b, 1e-5)
    grads = torch.autograd.grad(y, leaves, dy)
    want, bounds = plain(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    for got, ref, bound, what in zip((y.detach(), *grads), want, bounds, ("y", "dx", "dw", "db")):
        check(got, ref, bound, dtype, what)


@pytest.mark.parametrize("rows,n", [(65543, 16392)])
def test_wide_rows(spmm_npu, rows, n):
    """65536 work-groups, one row each: the rows beyond them, and some columns'
    sums over all rows."""
    dtype = torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, n, dtype=dtype, device="cuda").normal_(generator=g)
    dy = torch.empty(rows, n, dtype=dtype, device="cuda").normal_(generator=g)
    w, b = (torch.randn(n, device="cuda", generator=g).to(dtype).requires_grad_(True) for _ in range(2))
    x.requires_grad_(True)
    y = spmm_npu.layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x, y, wd, bd = x.detach(), y.detach(), w.detach(), b.detach()
    for part in (slice(0, 3), slice(65533, 65543)):
        want, bounds = plain(x[part], wd, bd, dy[part], 1e-5)
        check(y[part], want[0], bounds[0], dtype, "y")
        check(dx[part], want[1], bounds[1], dtype, "dx")
    mean = torch.empty(rows, 1, dtype=torch.float64, device="cuda")
    rstd = torch.empty_like(mean)
    for lo in range(0, rows, 4096):
        part = x[lo:lo + 4096].double()
        mean[lo:lo + 4096] = part.mean(1, keepdim=True)
        rstd[lo:lo + 4096] = 1 / torch.sqrt(part.var(1, unbiased=False, keepdim=True) + 1e-5)
    at = torch.tensor([0, 1, 255, 256, 8191, n - 2, n - 1], device="cuda")
    z, d = (x[:, at].double() - mean) * rstd, dy[:, at].double()
    terms = rows / 32 + 64
    zerr = (n / 32 + 64) * E32 * (1 + mean.abs() * rstd) * (1 + z.abs())
    for got, value, bound in ((dw[at], (d * z).sum(0), terms * E32 * (d * z).abs().sum(0) + (d.abs() * zerr).sum(0)),
                              (db[at], d.sum(0), terms * E32 * d.abs().sum(0))):
        limit = U[dtype] * value.abs() + bound * (1 + U[dtype]) + TINY[dtype]
        assert bool(((got.double() - value).abs() <= limit).all())
