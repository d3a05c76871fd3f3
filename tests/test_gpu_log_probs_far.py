"""log_probs of rows far from zero: maxima of any size in fp32 and bf16, parts
of a row on both sides of where distances are taken before the product with
log2(e), and spans masked by a finite value.

The bounds are those of expert_ops_plain.log_probs, but for a log probability
far below zero: (x - m) log2(e), less log2 s, times log(2) rounds four times and
has two constants of a quarter of a rounding each at most, so by 4.5 roundings
of its size, of which those bounds have 2 and the result's own.  An origin that
is off by 2^-4 adds 2^-4 of a rounding to log s, of which they have 72."""

import pytest
import torch

from expert_ops_plain import E32, check, log_probs, normal

pytestmark = pytest.mark.gpu


def run(f, x, t, top):
    leaf = x.detach().requires_grad_(True)
    logp, entropy, values, ids = f.log_probs(leaf, t, top=top)
    a, h = normal(t.shape, torch.float32, 5), normal(t.shape, torch.float32, 6)
    want = log_probs(x.detach(), t, top, a, h)
    for name, got in (("logp", logp), ("values", values)):
        more = 1.5 * E32 * want[name].abs().nan_to_num(0.0, 0.0, 0.0)
        check(got, want[name], want["err_" + name] + more, name)
    check(entropy, want["entropy"], want["err_H"], "entropy")
    assert torch.equal(ids.cpu(), want["ids"])
    (dx,) = torch.autograd.grad((logp, entropy), leaf, (a.cuda(), h.cuda()))
    check(dx, want["dx"], want["err_dx"], "dx")

SIZES = [2.0 ** 20 - 1, 2.0 ** 20, 2.0 ** 20 + 3, 3e6, 1e7, 2.0 ** 24, 1e9, 2e9, 3e9, 1e10, 1e15, 1e20, 1e30, 1e37,
         3e38]


def targets(rows, n):
    t = torch.arange(rows) * 7919 % n
    t[::5] = -1
    return t.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [10, 300, 1024, 5000, 40000])
def test_maxima_of_any_size(spmm_npu, n, dtype):
    sizes = torch.tensor([s * sign for s in SIZES for sign in (1, -1)], dtype=torch.float64)[:, None]
    rows = len(sizes)
    equal = sizes.expand(rows, n)
    near = sizes + normal((rows, n), torch.float32, n, 2.0).double()
    steps = sizes * (1 + 2.0 ** -23 * torch.randint(0, 6, (rows, n), generator=torch.Generator().manual_seed(n)))
    below = torch.where(torch.arange(n) % 3 == 0, sizes, sizes - sizes.abs() / 2)
    for x in (equal, near, steps, below):
        run(spmm_npu, x.to(dtype).cuda(), targets(rows, n), min(n, 5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 40000), (3, 70001), (40, 9000)])
def test_parts_on_both_sides(spmm_npu, rows, n, dtype):
    """Maxima of a row's parts and threads around where the origin changes."""
    gen = torch.Generator().manual_seed(n)
    for edge in (2.0 ** 20, -2.0 ** 20):
        spans = torch.randint(-6, 7, (rows, n // 2048 + 1), generator=gen).repeat_interleave(2048, 1)[:, :n]
        x = (edge + spans + normal((rows, n), torch.float32, n, 1.0).double()).to(dtype).cuda()
        run(spmm_npu, x, targets(rows, n), 4)
        # One part alone beyond it.
        x = torch.full((rows, n), edge, dtype=torch.float64) - 3
        x[:, n // 2: n // 2 + 20] += 7
        run(spmm_npu, x.to(dtype).cuda(), targets(rows, n), 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(5, 300), (5, 9000), (2, 70001), (1, 131072)])
def test_spans_masked_by_a_finite_value(spmm_npu, rows, n, dtype):
    for mask in (-1e5, -1e7, -1e9, -1e10, -1e20, -1e30, float(torch.finfo(dtype).min)):
        x = normal((rows, n), dtype, n, 2.0)
        x[:, : n // 3] = mask
        x[:, n // 2:: 2] = mask
        run(spmm_npu, x.cuda(), targets(rows, n), 3)
