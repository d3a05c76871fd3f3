"""route where all selection values are next to zero, so that fp32 does not scale
their differences to keys: the choice is that of 64 bits."""

import pytest
import torch

from expert_ops_plain import INF, normal
from test_gpu_route_bias_range import same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,k", [(2, 2), (3, 1), (8, 8), (64, 8), (64, 64), (300, 20)])
def test_scores_next_to_zero(spmm_npu, experts, k):
    """Sigmoids whose differences fp32 does not scale to keys, and biases as small."""
    for most in (-70.0, -73.5, -75.0, -80.0, -86.5, -88.0, -95.0, -104.0, -200.0):
        x = torch.full((6, experts), -100.0, dtype=torch.float64)
        x[0] = most - torch.arange(experts) % 7
        x[1] = most - 0.25 * normal((experts,), torch.float32, experts).double().abs()
        x[2, -1] = most
        x[3, 0] = most
        x[4] = most
        x[5, 1::2] = -INF
        for dtype in (torch.float32, torch.bfloat16):
            y = x.to(dtype).cuda()
            same(spmm_npu, y, k, "sigmoid", torch.zeros(experts, device="cuda"))
            tiny = normal((experts,), torch.float32, 4, 1e-35).cuda()
            same(spmm_npu, y, k, "sigmoid", tiny)
            same(spmm_npu, y, k, "sigmoid", tiny.abs() + 1e-38)
            if experts % 4 == 0 and k <= experts // 4:
                same(spmm_npu, y, k, "sigmoid", torch.zeros(experts, device="cuda"), 4, 1)
