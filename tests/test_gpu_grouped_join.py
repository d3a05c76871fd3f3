"""The weight gradient where its cut sums are joined by work-groups of 4096
sums (8388608 sums and more), by cuts and by groups, and of 1024 beside them.

Tolerances as in test_gpu_grouped.py, against 64-bit products on the GPU."""

import pytest
import torch

from test_gpu_grouped import E32, TINY, U

pytestmark = pytest.mark.gpu


# With the ranges that the rows are cut into: 7 cuts of 8 groups, 4 cuts of 3
# groups, 11 cuts of 40 groups, and 6 cuts of 12 fp32 groups (7077888 sums).
@pytest.mark.parametrize("dtype,rows,groups,inner,width", [
    (torch.bfloat16, 20011, 8, 1024, 2048), (torch.float16, 30000, 3, 1032, 2056), (torch.bfloat16, 30000, 40, 1024, 1040),
    (torch.float32, 9001, 12, 1000, 1100)])
@pytest.mark.parametrize("turned", [False, True])
def test_large_joins(spmm_npu, dtype, rows, groups, inner, width, turned):
    g = torch.Generator(device="cuda").manual_seed(rows)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    x, w, dy = rand(rows, inner), rand(groups, inner, width), rand(rows, width)
    if turned:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    edges = torch.randint(0, rows + 1, (groups - 1,), device="cuda", generator=g).sort().values
    edges = torch.cat([edges.new_zeros(1), edges, edges.new_full((1,), rows)])
    w.requires_grad_(True)
    dw, = torch.autograd.grad(spmm_npu.grouped_matmul(x, w, edges), w, dy)
    again, = torch.autograd.grad(spmm_npu.grouped_matmul(x, w, edges), w, dy)
    assert torch.equal(dw, again)
    for k, (lo, hi) in enumerate(zip(edges.tolist(), edges.tolist()[1:])):
        a, d = x[lo:hi].double().t().contiguous(), dy[lo:hi].double()
        want, mag = a @ d, a.abs() @ d.abs()
        limit = U[dtype] * want.abs() + (hi - lo + 2) * E32 * mag * (1 + U[dtype]) + TINY[dtype]
        assert bool(((dw[k].double() - want).abs() <= limit).all()), k
