"""route in groups without a bias: the scores in 64 bits decide, also where
different logits have the same one, and so the lowest index."""

import pytest
import torch

from expert_ops_plain import choose
from test_gpu_route import run

pytestmark = pytest.mark.gpu


def logits(experts, rows, kind, score):
    """Logits that differ and whose scores, rounded to 64 bits, are the same."""
    step = torch.randint(0, 4, (rows, experts), generator=torch.Generator().manual_seed(experts)).double()
    if kind == "next to zero":          # |x| < 2^-60: e^x is 1
        return step * 1e-20
    if kind == "beside one":            # a softmax's distances from the maximum round to the same
        x = step * 1e-20
        x[:, experts // 2] = 3.0
        return x
    if score == "softmax":              # e^-distance is zero
        x = -1000.0 - step
        x[:, experts // 2] = 3.0
        return x
    if kind == "near one":              # 1 - s is e^-x: its change over an fp32 step is below 2^-53
        return 25.5 + step * 2.0 ** -19
    return 31.0 + step


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kind", ["next to zero", "beside one", "near one", "far"])
@pytest.mark.parametrize("experts,groups,kept", [(8, 4, 4), (8, 2, 1), (16, 4, 2), (64, 8, 3), (66, 6, 6), (300, 4, 4)])
def test_equal_scores_of_different_logits(spmm_npu, experts, groups, kept, kind, score):
    x = logits(experts, 33, kind, score)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype).cuda()
        for k in {1, 2, min(5, experts // groups * kept), min(64, experts // groups * kept)}:
            want = choose(y, k, score, None, groups, kept)
            got = spmm_npu.route(y, k, score=score, groups=groups, top_groups=kept)[1].cpu()
            assert torch.equal(got, want), (got != want).any(1).nonzero().flatten().tolist()
            run(spmm_npu, y, k, score, groups=groups, top_groups=kept)
