"""log_probs against 64 bits (expert_ops_plain.log_probs says what the bounds
count); likeliest classes exactly."""

import numpy as np
import pytest
import torch

from expert_ops_plain import DTYPES, INF, check, log_probs, normal

pytestmark = pytest.mark.gpu


def run(f, x, targets, top, seed=0):
    rows_shape = x.shape[:-1]
    leaf = x.detach().requires_grad_(True)
    logp, entropy, values, ids = f.log_probs(leaf, targets, top=top)
    flat, t = x.detach().reshape(-1, x.size(-1)), targets.reshape(-1)
    a, h = normal(t.shape, torch.float32, seed + 5), normal(t.shape, torch.float32, seed + 6)
    want = log_probs(flat, t, top, a, h)
    assert logp.shape == entropy.shape == rows_shape and values.shape == ids.shape == rows_shape + (top,)
    assert logp.dtype == entropy.dtype == values.dtype == torch.float32 and ids.dtype == torch.int32
    check(logp.reshape(-1), want["logp"], want["err_logp"], "logp")
    check(entropy.reshape(-1), want["entropy"], want["err_H"], "entropy")
    assert torch.equal(ids.cpu().reshape(want["ids"].shape), want["ids"])
    check(values.reshape(want["values"].shape), want["values"], want["err_values"], "top")
    (dx,) = torch.autograd.grad((logp, entropy), leaf, (a.cuda().view(rows_shape), h.cuda().view(rows_shape)))
    assert dx.dtype == x.dtype and dx.shape == x.shape
    check(dx.reshape(flat.shape), want["dx"], want["err_dx"], "dx")
    again = f.log_probs(x.detach(), targets, top=top)
    assert all(torch.equal(p, q) for p, q in zip(again, (logp, entropy, values, ids)))


def make(rows, n, dtype, seed=0, spread=2.0):
    x = normal((rows, n), dtype, 100 * seed + n + rows, spread).cuda()
    t = torch.from_numpy(np.random.default_rng(seed + n).integers(-1, n + 1, rows)).cuda()
    return x, t


SIZES = [(1, 1, 1), (1, 2, 2), (3, 5, 5), (70, 8, 3), (33, 17, 8), (300, 47, 1), (64, 64, 16), (19, 100, 64), (50, 257, 4),
         (9, 512, 0), (21, 1000, 9), (5, 2048, 64), (4, 2049, 5), (7, 4099, 16), (3, 20011, 64), (2, 70001, 8),
         (1, 131072, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,top", SIZES)
def test_values_and_gradients(spmm_npu, rows, n, top, dtype):
    x, t = make(rows, n, dtype)
    run(spmm_npu, x, t, top)
    run(spmm_npu, x, t.clamp(0, n - 1).int(), min(top, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [10, 300, 5000, 40000])
def test_masked_rows(spmm_npu, n, dtype):
    x, t = make(6, n, dtype, seed=1)
    x[torch.from_numpy(np.random.default_rng(2).random((6, n)) < 0.5).cuda()] = -INF
    x[0] = -INF                                 # nothing left
    x[1] = -INF
    x[1, n - 1] = 1.0                           # one class left
    x[2] = torch.finfo(dtype).min               # all at the type's lowest value
    x[3] = torch.finfo(dtype).min               # a few above it
    x[3, [0, n // 2]] = 2.0
    t = torch.tensor([0, n - 1, n - 1, n // 2, 5, -100], device="cuda")
    run(spmm_npu, x, t, min(n, 7))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pieces", [1, 3, 7, 12, 15, 27, 50, 90, 200])
def test_many_rows(spmm_npu, pieces, dtype):
    """Enough rows for fewer lanes and several pieces a lane, with ties and masks."""
    piece = 16 // dtype.itemsize
    n = pieces * piece - (pieces % 2) * (piece // 2)
    x, t = make(17001, n, dtype, seed=pieces)
    x[::7] = (x[::7] * 2).round()
    x[3::11, ::3] = -INF
    run(spmm_npu, x, t, min(n, 6))


@pytest.mark.parametrize("n", [40, 3000, 9000, 70000])
def test_ties_go_to_the_lowest_index(spmm_npu, n):
    for dtype in DTYPES:
        x = torch.from_numpy(np.random.default_rng(4).integers(-2, 3, (5, n)).astype(np.float32)).cuda().to(dtype)
        x[0] = 1.5                              # all equal: more than the buffer of candidates
        x[1] = 0.0
        x[1, 1::2] = -0.0
        x[2] = -1.0
        x[2, n - 3:] = 4.0
        t = torch.tensor([0, 1, n - 1, 3, -1], device="cuda")
        run(spmm_npu, x, t, 16)
        run(spmm_npu, x[:1], t[:1], 5)


def test_far_and_near_values(spmm_npu):
    """Offsets that fp32 sums with, spreads that leave one class, and peaked rows with a small entropy."""
    for n in (50, 6000):
        for dtype in DTYPES:
            x, t = make(5, n, dtype, seed=3)
            x[0] += 1000.0
            x[1] = x[1] * 40
            x[2, 7] = 60.0
            x[3, 3] = 12.0
            run(spmm_npu, x, t, 3)


def test_nan_and_infinity(spmm_npu):
    for n in (30, 3000, 9000):
        x, t = make(4, n, torch.float32, seed=4)
        x[1, n // 3] = float("nan")
        x[2, n // 2] = INF
        t = torch.tensor([0, 1, 2, 3], device="cuda")
        logp, entropy, values, ids = spmm_npu.log_probs(x, t, top=4)
        assert bool(torch.isnan(logp[1:3]).all()) and bool(torch.isnan(entropy[1:3]).all())
        assert bool(torch.isfinite(logp[[0, 3]]).all()) and bool(torch.isnan(values[1]).all())
        assert not bool((ids[1] == n // 3).any()) and int(ids[2, 0]) == n // 2
        assert bool(((ids >= 0) & (ids < n)).all())
        leaf = x.requires_grad_(True)
        (dx,) = torch.autograd.grad(spmm_npu.log_probs(leaf, t)[0].sum(), leaf)
        assert bool(torch.isnan(dx[1:3]).any(1).all()) and bool(torch.isfinite(dx[[0, 3]]).all())


def test_one_gradient_alone(spmm_npu):
    x, t = make(9, 130, torch.float32, seed=5)
    t = t.clamp(0, 129)
    leaf = x.requires_grad_(True)
    logp, entropy, _, _ = spmm_npu.log_probs(leaf, t)
    both = torch.autograd.grad((logp, entropy), leaf, (torch.ones_like(logp), torch.zeros_like(logp)), retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(logp.sum(), leaf, retain_graph=True)[0], both)
    want = log_probs(x.detach(), t, 0, torch.zeros(9), torch.ones(9))
    check(torch.autograd.grad(entropy.sum(), leaf)[0], want["dx"], want["err_dx"], "entropy alone")


def test_shapes_and_strides(spmm_npu):
    big = normal((6, 5, 90), torch.bfloat16, 6).cuda()
    t = torch.arange(30, device="cuda").view(6, 5)
    run(spmm_npu, big, t, 2)
    run(spmm_npu, big[:, :, 7:58], t, 3)
    run(spmm_npu, big.transpose(0, 1), t.t(), 1)
    run(spmm_npu, big[0, 0], t[0, 3], 2)
    wide = normal((3, 9010), torch.float16, 7).cuda()
    run(spmm_npu, wide[:, 5:9006], torch.tensor([0, 9000, 4], device="cuda"), 6)
    for rows, n in ((0, 10), (0, 9000)):
        leaf = torch.zeros(rows, n, device="cuda", requires_grad=True)
        out = spmm_npu.log_probs(leaf, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=2)
        assert out[0].shape == (0,) and out[2].shape == out[3].shape == (0, 2)
        assert torch.autograd.grad(out[0].sum(), leaf)[0].shape == (rows, n)


@pytest.mark.parametrize("rows,n", [(400, 70), (3, 50000), (40, 9000)])
def test_graph_replays_and_another_stream(spmm_npu, rows, n):
    x, t = make(rows, n, torch.bfloat16, seed=8)

    def step():
        leaf = x.detach().requires_grad_(True)
        out = spmm_npu.log_probs(leaf, t, top=3)
        grads = torch.autograd.grad((out[0], out[1]), leaf, (torch.ones_like(out[0]), torch.ones_like(out[1])))
        return tuple(o.detach() for o in out) + grads

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        x.copy_(normal((rows, n), torch.bfloat16, 60 + k, 2.0).cuda())
        t.copy_(torch.roll(t, 1))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals(spmm_npu):
    x, t = torch.ones(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call, text in ((lambda: spmm_npu.log_probs(x.double(), t), "FP16, BF16 and FP32"),
                       (lambda: spmm_npu.log_probs(x, t.float()), "int32 or int64"),
                       (lambda: spmm_npu.log_probs(x, t[:3]), "one entry for each row"),
                       (lambda: spmm_npu.log_probs(x, t[:, None]), "one entry for each row"),
                       (lambda: spmm_npu.log_probs(x, t.cpu()), "must be a GPU tensor"),
                       (lambda: spmm_npu.log_probs(x[0, 0], t[0]), "at least one dimension"),
                       (lambda: spmm_npu.log_probs(x[:, :0], t), "classes")):
        with pytest.raises(RuntimeError, match=text):
            call()
    for top in (-1, 9, 65):
        with pytest.raises(ValueError, match="top"):
            spmm_npu.log_probs(x, t, top=top)
    leaf = x.clone().requires_grad_(True)
    out = spmm_npu.log_probs(leaf, t, top=2)
    assert out[0].requires_grad and out[1].requires_grad and not out[2].requires_grad and not out[3].requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(out[0].square().sum(), leaf, create_graph=True)


def test_more_elements_and_rows_than_32_bits_or_one_launch(spmm_npu):
    """2^22 + 3 rows of 2056: over 2^33 bytes, and more rows than one launch of the wide kernel takes."""
    rows, n = (1 << 22) + 3, 2056
    x = torch.zeros(rows, n, device="cuda", dtype=torch.float16)
    x[-1, n - 1] = 3.0
    x[(1 << 22) - 1, 5] = 2.0
    t = torch.full((rows,), n - 1, dtype=torch.int32, device="cuda")
    logp, entropy, values, ids = spmm_npu.log_probs(x, t, top=1)
    even = -float(np.log(n))
    assert abs(float(logp[0]) - even) < 1e-5 and float((logp[: (1 << 22) - 1] - logp[0]).abs().max()) == 0.0
    assert abs(float(logp[-1]) - (3.0 - float(np.log(n - 1 + np.exp(3.0))))) < 1e-5
    assert int(ids[-1, 0]) == n - 1 and int(ids[(1 << 22) - 1, 0]) == 5 and int(ids[-2, 0]) == 0
    assert abs(float(logp[(1 << 22) - 1]) + float(np.log(n - 1 + np.exp(2.0)))) < 1e-5
