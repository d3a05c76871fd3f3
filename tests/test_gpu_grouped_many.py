"""Grouped products of very many groups: right, and in time that grows with
their number, not with its square."""

import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(groups, most, inner, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + groups)
    sizes = torch.randint(0, most, (groups,), generator=g)
    off = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)])
    rows = int(off[-1]) + 5
    small = lambda *s: torch.randint(-2, 3, s, generator=g).to(dtype)  # noqa: E731  (exact sums)
    return small(rows, inner), small(groups, inner, width), small(rows, width), sizes, off


def run(f, x, w, off, dy):
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    y = f(x, w, off)
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("groups,most,inner,width", [(63, 90, 8, 16), (4095, 9, 16, 8), (4097, 300, 8, 8), (70001, 4, 8, 24),
                                                     (270001, 2, 8, 8)])
def test_products(spmm_npu, groups, most, inner, width, dtype):
    x, w, dy, sizes, off = make(groups, most, inner, width, dtype)
    y, dx, dw = run(spmm_npu.grouped_matmul, x.cuda(), w.cuda(), off.cuda(), dy.cuda())
    rows = int(off[-1])
    group = torch.repeat_interleave(torch.arange(groups), sizes)
    a, b, d = x.detach().float(), w.detach().float(), dy.float()
    want_y, want_dx = torch.zeros(dy.shape), torch.zeros(x.shape)
    for lo in range(0, rows, 1 << 16):
        part = slice(lo, min(rows, lo + (1 << 16)))
        want_y[part] = torch.bmm(a[part, None], b[group[part]])[:, 0]
        want_dx[part] = torch.bmm(d[part, None], b[group[part]].transpose(1, 2).contiguous())[:, 0]
    want_dw = torch.zeros(w.shape).index_add_(0, group, a[:rows, :, None] * d[:rows, None])
    for got, want in ((y, want_y), (dx, want_dx), (dw, want_dw)):
        assert torch.equal(got.float().cpu(), want)


@pytest.mark.parametrize("groups,rows_each", [(600, 256), (16382, 128), (16383, 128), (20000, 130)])
def test_large_tiles_of_many_groups(spmm_npu, groups, rows_each):
    """Around the number of groups that the 256 x 256 tiles take."""
    inner, width = 128, 136
    g = torch.Generator(device="cuda").manual_seed(groups)
    rows = groups * rows_each
    x = torch.randint(-2, 3, (rows, inner), generator=g, device="cuda").half()
    w = torch.randint(-2, 3, (groups, inner, width), generator=g, device="cuda").half()
    off = torch.arange(groups + 1, device="cuda") * rows_each
    off[groups // 2] += 100
    y = spmm_npu.grouped_matmul(x, w, off)
    for at in sorted({0, 1, 62, 63, 64, groups // 2 - 1, groups // 2, 4096 % groups, groups - 2, groups - 1}):
        part = slice(int(off[at]), int(off[at + 1]))
        assert torch.equal(y[part].float(), x[part].float() @ w[at].float()), at
    # every row once and by its own group
    group = torch.repeat_interleave(torch.arange(groups, device="cuda"), off.diff())
    column = torch.randint(0, width, (1,)).item()
    for lo in range(0, rows, 1 << 17):
        part = slice(lo, min(rows, lo + (1 << 17)))
        assert torch.equal(y[part, column].float(), (x[part].float() * w[group[part], :, column].float()).sum(1))


def test_time_grows_with_the_groups(spmm_npu):
    """Eight times the groups in less than 24 times the time (64 times where
    each tile scans all groups: 1.9 ms of 16384 groups against 35 us)."""
    def least(groups):
        x, w, dy, _, off = make(groups, 4, 16, 16, torch.float16)
        x, w, dy, off = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True), dy.cuda(), off.cuda()
        best = []
        for _ in range(5):
            torch.cuda.synchronize()
            start = time.perf_counter()
            y = spmm_npu.grouped_matmul(x, w, off)
            torch.cuda.synchronize()
            middle = time.perf_counter()
            torch.autograd.grad(y, (x, w), dy)
            torch.cuda.synchronize()
            best.append((middle - start, time.perf_counter() - middle))
        return [min(t) for t in zip(*best)]

    few, many = least(16384), least(131072)
    for a, b, what in zip(few, many, ("forward", "backward")):
        assert b < 24 * max(a, 50e-6), (what, a, b)
