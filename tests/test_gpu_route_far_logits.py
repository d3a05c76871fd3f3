"""route by softmax and a bias, and in groups, of rows whose logits are far from
zero: the choice is that of 64 bits."""

import pytest
import torch

from expert_ops_plain import INF, choose, normal
from test_gpu_route import run

pytestmark = pytest.mark.gpu

SIZES = [1e4, 1e6, 2.0 ** 20 + 1, 1e7, 1e9, 2e9, 1e10, 1e15, 1e20, 1e30, 2e38, 3e38]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts", [5, 16, 64, 65, 256, 1024])
def test_rows_far_from_zero(spmm_npu, experts, dtype):
    sizes = torch.tensor([s * sign for s in SIZES for sign in (1, -1)], dtype=torch.float64)[:, None]
    rows = len(sizes)
    bias = normal((experts,), torch.float32, experts, 0.3).cuda()
    near = sizes + normal((rows, experts), torch.float32, experts).double()
    steps = sizes * (1 - 2.0 ** -23 * (torch.arange(experts) % 5))
    below = torch.where(torch.arange(experts) % 3 == 0, sizes, sizes - sizes.abs() / 2)
    masked = torch.where(torch.arange(experts) % 2 == 0, -INF, near)
    for x in (sizes.expand(rows, experts), near, steps, below, masked):
        x = x.to(dtype).cuda()
        k = min(8, experts)
        want = choose(x, k, "softmax", bias, 1, 1)
        got = spmm_npu.route(x, k, score="softmax", bias=bias)[1].cpu()
        assert torch.equal(got, want), (got != want).any(1).nonzero().flatten().tolist()
        run(spmm_npu, x, k, "softmax", bias=bias, renormalize=False)
        if experts % 4 == 0:
            run(spmm_npu, x, 4, "softmax", bias=bias, groups=4, top_groups=2)
            run(spmm_npu, x, 4, "softmax", groups=4, top_groups=2)
            run(spmm_npu, x, 4, "softmax", groups=4, top_groups=4)
