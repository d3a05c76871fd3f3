"""The operators around experts refuse tensors with a forward-mode tangent, which
they would drop, and take them where forward mode is off; none of them differs
on another stream or when several streams run them at once."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(spmm_npu, requires_grad):
    def rand(*s):
        return torch.randn(*s, device="cuda").requires_grad_(requires_grad)

    x, w, y = rand(6, 16), rand(6, 2), rand(12, 16)
    bias = torch.randn(16, device="cuda")
    ids = torch.zeros(6, dtype=torch.int64, device="cuda")
    plan = spmm_npu.ExpertPlan(torch.zeros(6, 2, dtype=torch.int32, device="cuda"), 3)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: spmm_npu.embedding(dual(x), ids), lambda: spmm_npu.route(dual(x), 2),
                     lambda: spmm_npu.route(x, 2, bias=dual(bias)), lambda: plan.pack(dual(x)),
                     lambda: plan.restore(dual(y), w), lambda: plan.restore(y, dual(w)),
                     lambda: spmm_npu.log_probs(dual(x), ids)):
            with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                call()
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(spmm_npu.route(dual(x), 2)[0], spmm_npu.route(x, 2)[0])


def test_many_streams_at_once(spmm_npu):
    """The same and different calls under way together, each with workspaces of its own."""
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randn(3000, 136, generator=g, device="cuda").requires_grad_(True)
    logits = torch.randn(3, 70000, generator=g, device="cuda").bfloat16().requires_grad_(True)
    inputs = [(torch.randint(0, 3000, (20000,), generator=g, device="cuda"),
               torch.randn(20000, 136, generator=g, device="cuda"),
               torch.randint(0, 70000, (3,), generator=g, device="cuda")) for _ in range(4)]

    def step(ids, grad, targets):
        rows = spmm_npu.embedding(table, ids)
        (dtable,) = torch.autograd.grad(rows, table, grad)
        weights, experts = spmm_npu.route(rows[:, :40], 3, score="sigmoid", groups=4, top_groups=2)
        plan = spmm_npu.ExpertPlan(experts, 40)
        back = plan.restore(plan.pack(rows.detach()), weights.detach())
        out = spmm_npu.log_probs(logits, targets, top=5)
        (dlogits,) = torch.autograd.grad(out[0].sum() + out[1].sum(), logits)
        return (dtable, weights.detach(), experts, plan.place, back) + tuple(o.detach() for o in out) + (dlogits,)

    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = []
    for _ in range(3):
        for s, i in zip(streams, inputs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(*i))
    torch.cuda.synchronize()
    for k, result in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(result, want[k % 4]))


class Ends(torch.autograd.Function):
    """Gives no gradient."""

    @staticmethod
    def forward(ctx, *xs):
        return xs[0].sum()

    @staticmethod
    def backward(ctx, grad):
        return None, None


def test_no_gradient_comes_in(spmm_npu):
    x = torch.randn(5, 12, device="cuda", requires_grad=True)
    ids = torch.zeros(5, dtype=torch.int64, device="cuda")
    weights, _ = spmm_npu.route(x, 2)
    logp, entropy, _, _ = spmm_npu.log_probs(x, ids)
    for a, b in ((weights, weights), (logp, entropy)):
        (dx,) = torch.autograd.grad(Ends.apply(a, b), x, allow_unused=True)
        assert dx is None or not dx.any()
    rows = spmm_npu.embedding(x, ids)
    (dx,) = torch.autograd.grad(Ends.apply(rows, rows), x, allow_unused=True)
    assert dx is None or not dx.any()
