"""A model of the operators together, as they would be used: a table of node
features, a layer norm, a router and its experts, the graph, and the labels' log
probabilities.  Forward and all gradients against 64-bit autograd."""

import pytest
import torch

from expert_ops_plain import choose

pytestmark = pytest.mark.gpu


def graph_of(nodes, degree, dtype, g):
    edges = torch.randint(0, nodes * nodes, (nodes * degree,), generator=g).unique()
    row, col = edges // nodes, edges % nodes
    counts = torch.bincount(row, minlength=nodes)
    rowptr = torch.zeros(nodes + 1, dtype=torch.int64)
    rowptr[1:] = counts.cumsum(0)
    return rowptr, col, (1.0 / counts.clamp_min(1).double())[row].to(dtype)


# The sparse operators' own tolerances (2e-2 for fp16, 1e-4 for fp32), against the largest
# value of each result.  fp32: a dozen roundings of 2^-24 and sums of up to 400 terms.  The
# router is held in 64 bits by the choice that the operators made, as a turned pair of close
# experts would be another function.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.float16, 2e-2)])
def test_model_of_experts(spmm_npu, dtype, tol):
    nodes, count, width, k, classes = 400, 6, 64, 2, 11
    g = torch.Generator().manual_seed(0)
    rowptr, col, value = graph_of(nodes, 6, dtype, g)
    graph = spmm_npu.PackedGraph(spmm_npu.preprocess(rowptr.cuda(), col.cuda(), value.cuda(), nodes, nodes,
                                                     graph_layout=True))
    normal = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    table, scale, shift = normal(1000, width), 1 + 0.1 * normal(width), 0.1 * normal(width)
    router, experts = normal(width, count) / 4, normal(count, width, width) / 8
    head = normal(width, classes) / 8
    ids = torch.randint(0, 1000, (nodes,), generator=g)
    labels = torch.randint(-1, classes, (nodes,), generator=g)
    bias = 0.05 * torch.randn(count, generator=g)
    leaves = [t.cuda().requires_grad_(True) for t in (table, scale, shift, router, experts, head)]

    t, s, b, r, e, o = leaves
    x = spmm_npu.layer_norm(spmm_npu.embedding(t, ids.cuda(), scale=8.0), s, b)
    weights, chosen = spmm_npu.route(x @ r, k, score="sigmoid", bias=bias.cuda())
    plan = spmm_npu.ExpertPlan(chosen, count)
    h = plan.restore(spmm_npu.grouped_matmul(plan.pack(x), e, plan.offsets), weights)
    h = graph.restore(graph(graph.pack(h))) + x
    logp, entropy, values, top = spmm_npu.log_probs(h @ o, labels.cuda(), top=3)
    loss = -(logp.sum() + 0.1 * entropy.sum())
    grads = torch.autograd.grad(loss, leaves)

    wide = [v.detach().double().cpu().requires_grad_(True) for v in leaves]
    t, s, b, r, e, o = wide
    x = t[ids] * 8.0
    x = (x - x.mean(1, keepdim=True)) / (x.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * s + b
    at = chosen.cpu().long()
    score = torch.sigmoid(x @ r).gather(1, at)
    w = score / score.sum(1, keepdim=True)
    h = sum(w[:, j:j + 1] * torch.bmm(x[:, None], e[at[:, j]])[:, 0] for j in range(k))
    a = torch.zeros(nodes, nodes, dtype=torch.float64)
    a[torch.repeat_interleave(torch.arange(nodes), rowptr.diff()), col] = value.double()
    logits = (a @ h + x) @ o
    lp = torch.log_softmax(logits, 1)
    want = torch.where(labels >= 0, lp[torch.arange(nodes), labels.clamp_min(0)], 0.0)
    H = -(lp.exp() * lp).sum(1)
    dense = torch.autograd.grad(-(want.sum() + 0.1 * H.sum()), wide)

    off = lambda got, ref: float((got.detach().double().cpu() - ref.detach()).abs().max() / ref.detach().abs().max())  # noqa: E731
    for name, got, ref in zip(("logp", "entropy", "weights"), (logp, entropy, weights), (want, H, w)):
        assert off(got, ref) <= tol, name
    for name, got, ref in zip(("table", "scale", "shift", "router", "experts", "head"), grads, dense):
        assert off(got, ref) <= tol, name
    if dtype == torch.float32:
        assert torch.equal(chosen.cpu(), choose((x @ r).detach().float(), k, "sigmoid", bias, 1, 1))
        assert off(values, lp.topk(3, dim=1).values) <= tol


def test_rows_without_an_expert_pass_through(spmm_npu):
    """A router that leaves some rows without experts: they come back as zeros, and
    give no gradient to the weights of any expert."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(30, 32, generator=g).cuda()
    logits = torch.randn(30, 4, generator=g).cuda()
    logits[::3] = -float("inf")
    w = torch.randn(4, 32, 32, generator=g).cuda().requires_grad_(True)
    weights, chosen = spmm_npu.route(logits, 2)
    plan = spmm_npu.ExpertPlan(chosen, 4)
    out = plan.restore(spmm_npu.grouped_matmul(plan.pack(x), w, plan.offsets), weights)
    assert not out[::3].any() and int(plan.offsets[-1]) == 40
    grad = torch.ones_like(out)
    grad[::3] = float("nan")
    (dw,) = torch.autograd.grad(out, w, grad)
    assert bool(torch.isfinite(dw).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_captured_with_its_gradients(spmm_npu, dtype):
    """A training step of the layer in one graph: every replay, with other inputs and eager
    steps in between, gives what an eager step gives."""
    g = torch.Generator().manual_seed(2)
    rows, count, width, classes = 5000, 5, 48, 3000
    normal = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    table, router, w = normal(700, width), normal(1, width, count), normal(count, width, width)
    head = normal(1, width, classes)
    every = torch.tensor([0, rows], device="cuda")
    ids = torch.zeros(rows, dtype=torch.int64, device="cuda")
    labels = torch.zeros(rows, dtype=torch.int64, device="cuda")

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (table, router, w, head)]
        t, r, e, h = leaves
        x = spmm_npu.embedding(t, ids)
        weights, experts = spmm_npu.route(spmm_npu.grouped_matmul(x, r, every), 2, renormalize=False)
        plan = spmm_npu.ExpertPlan(experts, count)
        y = plan.restore(spmm_npu.grouped_matmul(plan.pack(x), e, plan.offsets), weights)
        logp, entropy, _, top = spmm_npu.log_probs(spmm_npu.grouped_matmul(y, h, every), labels, top=2)
        return (logp.detach(), entropy.detach(), top) + torch.autograd.grad((logp, entropy), leaves, (up, up))

    up = torch.randn(rows, generator=g).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        ids.copy_(torch.randint(-1, 700, (rows,), generator=g) if k % 2 else torch.full((rows,), 3))
        labels.copy_(torch.randint(-1, classes, (rows,), generator=g))
        table.copy_(normal(700, width))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
