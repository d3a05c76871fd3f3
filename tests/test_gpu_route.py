"""route against a choice by sorting and weights and gradients in 64 bits
(expert_ops_plain.route says what the bounds count)."""

import numpy as np
import pytest
import torch

from expert_ops_plain import DTYPES, INF, check, choose, normal, route, undecided

pytestmark = pytest.mark.gpu


def run(f, x, top_k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0, seed=0):
    leaf = x.detach().requires_grad_(True)
    weights, experts = f.route(leaf, top_k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                               renormalize=renormalize, scale=scale)
    assert weights.dtype == torch.float32 and experts.dtype == torch.int32
    assert weights.shape == experts.shape == x.shape[:-1] + (top_k,)
    flat = x.detach().reshape(-1, x.size(-1))
    top_groups = groups if top_groups is None else top_groups
    want = choose(flat, top_k, score, bias, groups, top_groups)
    got = experts.reshape(want.shape).cpu()
    # Groups whose sums are equal but for their rounding may come in either order.
    turned = (got != want).any(1) & undecided(flat, score, bias, groups, top_groups)
    assert torch.equal(got[~turned], want[~turned]), f"{int((got != want).sum())} of {want.numel()} choices differ"
    want = got
    g = normal(want.shape, torch.float32, seed + 99)
    ref = route(flat, want, score, renormalize, scale, g)
    check(weights.reshape(want.shape), ref["w"], ref["err_w"], "weights")
    (dx,) = torch.autograd.grad(weights, leaf, g.cuda().view(weights.shape))
    assert dx.dtype == x.dtype and dx.shape == x.shape
    check(dx.reshape(flat.shape), ref["dx"], ref["err_dx"], "dlogits")
    # Without a gradient wanted, the same.
    again = f.route(x.detach(), top_k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                    renormalize=renormalize, scale=scale)
    assert torch.equal(again[0], weights) and torch.equal(again[1], experts)
    return weights.detach(), experts


SIZES = [(1, 1, 1), (1, 64, 4), (5, 2, 2), (33, 3, 1), (70, 12, 2), (19, 16, 16), (50, 17, 5), (129, 64, 8), (40, 65, 3),
         (65, 200, 10), (31, 256, 8), (9, 257, 33), (7, 512, 64), (4, 1000, 16), (3, 1024, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rows,experts,k", SIZES)
def test_choices_weights_gradients(spmm_npu, rows, experts, k, score, dtype):
    x = normal((rows, experts), dtype, rows + experts).cuda()
    bias = normal((experts,), torch.float32, 5, 0.3).cuda()
    run(spmm_npu, x, k, score, renormalize=True)
    run(spmm_npu, x, k, score, renormalize=False, scale=2.5)
    run(spmm_npu, x, k, score, bias=bias, renormalize=True, scale=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(8, 8, 3, 3), (12, 4, 2, 5), (64, 8, 4, 8), (64, 64, 9, 9),
                                                         (66, 3, 1, 20), (160, 8, 3, 6), (256, 8, 4, 8), (256, 32, 5, 40),
                                                         (1024, 64, 10, 64), (30, 2, 2, 7), (20, 20, 20, 20)])
def test_groups(spmm_npu, experts, groups, top_groups, k, score, dtype):
    x = normal((21, experts), dtype, experts + groups).cuda()
    bias = normal((experts,), torch.float32, 6, 0.2).cuda()
    run(spmm_npu, x, k, score, bias=bias, groups=groups, top_groups=top_groups)
    run(spmm_npu, x, k, score, groups=groups, top_groups=top_groups, renormalize=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1, 3, 4, 8, 12, 16, 20, 32, 64, 128, 252])
def test_every_shape_of_groups(spmm_npu, size, dtype):
    """Groups of few and many pieces on few and many lanes, biases of -inf and masked logits among them."""
    for groups in (2, 3, 4, 5, 8, 16, 17, 32, 63, 64):
        experts = groups * size
        if experts > 1024:
            continue
        x = normal((9, experts), dtype, experts).cuda()
        x[1, ::3] = -INF
        x[2, : experts - size] = -INF
        bias = normal((experts,), torch.float32, groups, 0.2).cuda()
        top_groups = max(1, groups // 3)
        k = min(5, top_groups * size)
        run(spmm_npu, x, k, "sigmoid", bias=bias, groups=groups, top_groups=top_groups)
        bias[::7] = -INF
        run(spmm_npu, x, k, "sigmoid", bias=bias, groups=groups, top_groups=top_groups)
        run(spmm_npu, x, k, "softmax", bias=bias)
        run(spmm_npu, x, k, "softmax", groups=groups, top_groups=top_groups)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_index(spmm_npu, score):
    for experts in (5, 64, 300):
        x = torch.from_numpy(np.random.default_rng(3).integers(-1, 2, (40, experts)).astype(np.float32)).cuda()
        x[0] = 0.25
        x[1, ::2], x[1, 1::2] = 0.0, -0.0
        for dtype in DTYPES:
            k = min(8, experts)
            run(spmm_npu, x.to(dtype), k, score)
            run(spmm_npu, x.to(dtype), k, score, bias=torch.zeros(experts, device="cuda"), renormalize=False)
        if experts % 4 == 0:
            run(spmm_npu, x, 4, score, groups=4, top_groups=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_masked_experts(spmm_npu, score, renormalize):
    for experts, k, groups in ((6, 4, 1), (64, 8, 1), (64, 8, 8), (300, 20, 4)):
        x = normal((30, experts), torch.float32, 8).cuda()
        x[torch.from_numpy(np.random.default_rng(9).random((30, experts)) < 0.8).cuda()] = -INF
        x[0] = -INF                      # none left
        x[1] = -INF
        x[1, experts - 1] = 3.0          # one left
        x[2, 0] = 200.0                  # one far above
        x[3] = -300.0                    # scores that vanish in fp32
        x[5] = -95.0                     # and beside some that do not
        x[5, ::2] = -78.0
        x[4] = torch.finfo(torch.float32).min  # the type's lowest value is a logit as any other
        bias = normal((experts,), torch.float32, 10, 0.1).cuda()
        bias[experts // 2] = -INF
        for dtype in DTYPES:
            y = x.to(dtype) if dtype != torch.float16 else x.clamp_min(-60000).masked_fill(x == -INF, -INF).to(dtype)
            w, e = run(spmm_npu, y, k, score, groups=groups, top_groups=groups, renormalize=renormalize)
            assert bool((e[0] == -1).all()) and not w[0].any() and int(e[1, 0]) == experts - 1
            kept = max(1, groups // 2)
            if experts // groups * kept >= k:
                run(spmm_npu, y, k, score, bias=bias, groups=groups, top_groups=kept, renormalize=renormalize)


def test_bias_of_minus_infinity_closes_an_expert(spmm_npu):
    x = normal((50, 12), torch.bfloat16, 11).cuda()
    bias = torch.zeros(12, device="cuda")
    bias[3] = -INF
    for score in ("softmax", "sigmoid"):
        _, e = run(spmm_npu, x, 11, score, bias=bias)
        assert not bool((e == 3).any())
        _, e = run(spmm_npu, x, 12, score, bias=bias)
        assert bool((e[:, 11] == -1).all())


def test_a_nan_is_chosen_and_seen(spmm_npu):
    x = normal((4, 40), torch.float32, 12).cuda()
    x[1, 7] = float("nan")
    x[2, 9] = INF
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(40, device="cuda")):
            w, e = spmm_npu.route(x, 3, score=score, bias=bias)
            assert bool(torch.isnan(w[1]).any()) and bool(torch.isfinite(w[[0, 3]]).all())
            if score == "sigmoid" or bias is None:
                assert int(e[1, 0]) == 7 and int(e[2, 0]) == 9
            assert bool(((e >= 0) & (e < 40)).all())


def test_close_pairs_under_a_bias(spmm_npu):
    """Pairs whose sums differ by less than fp32 tells apart."""
    x = torch.zeros(64, 8, device="cuda")
    x[:, 1] = torch.linspace(-1e-6, 1e-6, 64).cuda()
    bias = torch.tensor([0.1, 0.1, -5.0, -5, -5, -5, -5, -5], device="cuda")
    for score in ("softmax", "sigmoid"):
        run(spmm_npu, x, 2, score, bias=bias)
        run(spmm_npu, x, 1, score, bias=bias, groups=4, top_groups=1)


def test_shapes_strides_and_empty(spmm_npu):
    big = normal((6, 5, 40), torch.float16, 13).cuda()
    run(spmm_npu, big, 3)
    run(spmm_npu, big[:, :, 5:29], 3, "sigmoid", renormalize=False)
    run(spmm_npu, big.transpose(0, 1), 2, renormalize=False)
    run(spmm_npu, big[0, 0], 4)
    run(spmm_npu, big.permute(2, 0, 1)[..., :5], 2)
    empty = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w, e = spmm_npu.route(empty, 2)
    assert w.shape == e.shape == (0, 2) and torch.autograd.grad(w.sum(), empty)[0].shape == (0, 8)


def test_many_rows(spmm_npu):
    x = normal((70001, 24), torch.bfloat16, 14).cuda()
    w, e = spmm_npu.route(x, 2, renormalize=False)
    p = torch.softmax(x.double(), 1)
    at = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(e.long(), at)
    assert float((w.double() - p.gather(1, at)).abs().max()) < 1e-6


def test_graph_replays_and_another_stream(spmm_npu):
    x, bias = normal((500, 64), torch.float32, 15).cuda(), normal((64,), torch.float32, 16, 0.1).cuda()
    g = normal((500, 6), torch.float32, 17).cuda()

    def step():
        leaf = x.detach().requires_grad_(True)
        w, e = spmm_npu.route(leaf, 6, score="sigmoid", bias=bias, groups=8, top_groups=4)
        return w.detach(), e, torch.autograd.grad(w, leaf, g)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.copy_(normal((500, 64), torch.float32, 30 + k).cuda())
        bias.add_(0.01 * k)
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(spmm_npu):
    x = torch.ones(4, 8, device="cuda")
    for call, text in ((lambda: spmm_npu.route(x.double(), 2), "FP16, BF16 and FP32"),
                       (lambda: spmm_npu.route(torch.tensor(1.0, device="cuda"), 1), "at least one dimension"),
                       (lambda: spmm_npu.route(x, 2, bias=torch.ones(7, device="cuda")), "bias must be a 1D"),
                       (lambda: spmm_npu.route(x, 2, bias=torch.ones(8, device="cuda").half()), "bias must be FP32"),
                       (lambda: spmm_npu.route(x, 2, bias=torch.ones(8)), "same device"),
                       (lambda: spmm_npu.route(x, 2, bias=torch.ones(8, device="cuda", requires_grad=True)), "no gradient"),
                       (lambda: spmm_npu.route(torch.ones(2, 1025, device="cuda"), 2), "1 to 1024 experts"),
                       (lambda: spmm_npu.route(torch.ones(2, 0, device="cuda"), 1), "1 to 1024 experts")):
        with pytest.raises(RuntimeError, match=text):
            call()
    for call, text in ((lambda: spmm_npu.route(x, 0), "top_k"), (lambda: spmm_npu.route(x, 9), "top_k"),
                       (lambda: spmm_npu.route(x, -1), "top_k"), (lambda: spmm_npu.route(x, 1 << 40), "top_k"),
                       (lambda: spmm_npu.route(x, 2, groups=3), "groups"),
                       (lambda: spmm_npu.route(x, 2, groups=4, top_groups=5), "top_groups"),
                       (lambda: spmm_npu.route(x, 2, scale=0.0), "scale")):
        with pytest.raises(ValueError, match=text):
            call()
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(spmm_npu.route(leaf, 2)[0].square().sum(), leaf, create_graph=True)
    assert not spmm_npu.route(leaf, 2)[1].requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
def test_choices_that_32_bits_do_not_decide(spmm_npu, dtype):
    """Many equal and nearly equal selection values, at the border of the choice
    and behind it; scores that 64 bits do not tell apart (1 and 0)."""
    rng = np.random.default_rng(21)
    for experts, groups, kept in ((16, 4, 2), (48, 1, 1), (64, 8, 3), (256, 8, 4), (300, 6, 2), (700, 1, 1)):
        levels = torch.from_numpy(rng.integers(0, 4, (37, experts)).astype(np.float32))
        fine = torch.from_numpy(rng.integers(0, 4, (37, experts)).astype(np.float32)) * 2.0 ** -9
        for x in (levels * 0.5, levels * 0.25 + fine, levels * 20.0 - 10.0, levels * -300.0, 50.0 + levels):
            x = x.to(dtype).cuda()
            coarse = torch.from_numpy(rng.integers(0, 3, experts).astype(np.float32)).cuda() * 0.25
            tiny = torch.from_numpy(rng.standard_normal(experts).astype(np.float32)).cuda() * 1e-7
            for score in ("softmax", "sigmoid"):
                for bias in (None, torch.zeros(experts, device="cuda"), coarse, tiny, 1000.0 + coarse):
                    if bias is not None or groups > 1:
                        run(spmm_npu, x, 5, score, bias=bias, groups=groups, top_groups=kept)


def test_more_rows_than_one_launch(spmm_npu):
    rows = (1 << 24) + 5
    x = torch.zeros(rows, 2, device="cuda", dtype=torch.float16)
    x[1::3, 1] = 1.0
    x[-1, 1] = 2.0
    w, e = spmm_npu.route(x, 1, renormalize=False)
    assert torch.equal(e[:, 0].long(), (x[:, 1] > 0).long())
    p = torch.softmax(x.double(), 1).amax(1)
    assert float((w[:, 0].double() - p).abs().max()) < 1e-6 and abs(float(w[-1, 0]) - float(p[-1])) < 1e-6
