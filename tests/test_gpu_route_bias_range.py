"""route where selection values overflow fp32, alone, two together or in their
range: the choice is that of 64 bits."""

import pytest
import torch

from expert_ops_plain import INF, choose, normal
from test_gpu_route import run

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


def same(f, x, k, score, bias, groups=1, top_groups=None):
    """Every choice as in 64 bits; weights and gradients too."""
    top_groups = groups if top_groups is None else top_groups
    want = choose(x, k, score, bias, groups, top_groups)
    _, got = f.route(x, k, score=score, bias=bias, groups=groups, top_groups=top_groups)
    assert torch.equal(got.cpu(), want), (got.cpu(), want)
    run(f, x, k, score, bias=bias, groups=groups, top_groups=top_groups)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("high,low", [(INF, 0.0), (3e38, -3e38), (INF, -3e38), (INF, -INF), (3e38, 0.0), (0.0, LOWEST)])
def test_biases_that_overflow(spmm_npu, score, high, low):
    for experts in (1, 2, 3, 8, 13, 64, 300):
        x = normal((20, experts), torch.float32, experts).cuda()
        x[1] = 0.5
        x[2, 1::2] = -INF
        x[3] = -INF
        x[4, min(2, experts):] = -INF         # two left
        x[5, 1:] = -INF                       # one left
        for at in {0, 1, experts - 1}:
            if at >= experts:
                continue
            bias = torch.full((experts,), low, device="cuda")
            bias[at] = high
            for k in {1, min(2, experts), min(8, experts), min(64, experts)}:
                same(spmm_npu, x, k, score, bias)
                same(spmm_npu, x.bfloat16(), k, score, bias)
            mixed = normal((experts,), torch.float32, 3, 0.1).cuda()
            mixed[at] = high
            mixed[(at + 1) % experts] = low
            same(spmm_npu, x, min(4, experts), score, mixed)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(8, 4), (12, 3), (64, 8), (66, 33), (300, 6)])
def test_sums_of_two_that_overflow(spmm_npu, score, experts, groups):
    """A group of experts at the lowest value is above one without any, and two at the greatest are not infinite."""
    size = experts // groups
    x = normal((9, experts), torch.float32, experts).cuda()
    x[1, :size] = -INF
    x[2, : size * (groups - 1)] = -INF
    x[3] = -INF
    for value in (LOWEST, -2e38, -INF, 2e38, 3e38, INF):
        for part in (slice(None), slice(size, None), slice(size, 2 * size), slice(None, None, 2)):
            bias = torch.zeros(experts, device="cuda")
            bias[part] = value
            for top_groups in {1, 2, groups - 1}:
                same(spmm_npu, x, min(2, size * top_groups), score, bias, groups, top_groups)
        # One empty group in front of one at the lowest value.
        bias = torch.full((experts,), value, device="cuda")
        bias[:size] = -INF
        same(spmm_npu, x, 1, score, bias, groups, 1)
