"""embedding and its gradient against sums in 64 bits.

A row is its value times the scale, two fp32 roundings (the scale's and the
product's) and the result's.  The gradient of a table row named n times is a sum
of n fp32 terms, off by at most n e sum|terms|, times the scale."""

import numpy as np
import pytest
import torch

from expert_ops_plain import DTYPES, E32, check, normal, scale_of

pytestmark = pytest.mark.gpu


def run(f, weight, ids, scale, grad=None):
    """Output, and with `grad` the table's gradient, checked against 64 bits."""
    rows = weight.size(0)
    out = f.embedding(weight.requires_grad_(grad is not None), ids, scale=scale)
    assert out.shape == ids.shape + weight.shape[1:] and out.dtype == weight.dtype
    w, at = weight.detach().double().cpu(), ids.cpu().long().reshape(-1)
    inside = (at >= 0) & (at < rows)
    want = torch.zeros(at.numel(), w.size(1), dtype=torch.float64)
    want[inside] = w[at[inside]] * scale
    check(out.reshape(want.shape), want, 2 * E32 * want.abs(), "out")
    if grad is None:
        return out
    (dw,) = torch.autograd.grad(out, weight, grad)
    g = grad.double().cpu().reshape(want.shape)
    total, size, count = torch.zeros_like(w), torch.zeros_like(w), torch.zeros(rows, 1, dtype=torch.float64)
    total.index_add_(0, at[inside], g[inside])
    size.index_add_(0, at[inside], g[inside].abs())
    count.index_add_(0, at[inside], torch.ones(int(inside.sum()), 1, dtype=torch.float64))
    assert dw.shape == weight.shape and dw.dtype == weight.dtype
    check(dw, total * scale, ((count + 2) * E32 * size * abs(scale)), "dweight")
    assert not dw[(count[:, 0] == 0).to(dw.device)].any()
    return out, dw


def ids_of(kind, count, table, seed=0):
    rng = np.random.default_rng(seed + count + 7 * table)
    if kind == "zipf":
        ids = np.minimum((np.exp(rng.random(count) * np.log(table + 1)) - 1).astype(np.int64), table - 1)
        ids = rng.permutation(table)[ids]
    elif kind == "uniform":
        ids = rng.integers(0, table, count)
    elif kind == "absent":
        ids = rng.integers(-2, table + 2, count)
    elif kind == "same":
        ids = np.full(count, table - 1)
    else:
        ids = np.arange(count) % table
    return torch.from_numpy(ids).cuda()


SIZES = [(1, 1, 1), (1, 5, 8), (3, 2, 7), (64, 10, 33), (257, 1000, 128), (1000, 3, 96), (31, 4096, 520),
         (33, 70000, 16), (2000, 300, 1024), (4096, 4097, 40), (4097, 4095, 40), (20011, 3001, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,table,width", SIZES)
def test_rows_and_gradient(spmm_npu, count, table, width, dtype):
    weight = normal((table, width), dtype, 1).cuda()
    grad = normal((count, width), dtype, 2).cuda()
    for kind in ("zipf", "absent"):
        run(spmm_npu, weight, ids_of(kind, count, table), scale_of(width), grad)
        run(spmm_npu, weight.detach(), ids_of(kind, count, table).int(), 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["same", "order", "uniform"])
def test_long_and_short_runs(spmm_npu, kind, dtype):
    """One id for all positions (one run over all ranges), each its own, and a few."""
    for count, table, width in ((5000, 5000, 72), (9001, 40, 264), (32, 4, 8), (64, 2, 8), (65, 64, 8)):
        run(spmm_npu, normal((table, width), dtype, 3).cuda(), ids_of(kind, count, table), 0.5,
            normal((count, width), dtype, 4).cuda())


def test_tables_over_one_and_two_digits(spmm_npu):
    """Sorts of one, two and three digits, at the borders between them."""
    for table in (2046, 2047, 2048, 2049, (1 << 22) - 1, (1 << 22) + 5):
        ids = ids_of("absent", 6000, table)
        ids[:3] = torch.tensor([0, table - 1, table], device="cuda")
        run(spmm_npu, normal((table, 4), torch.float16, 5).cuda(), ids, 1.0, normal((6000, 4), torch.float16, 6).cuda())


def test_shapes_strides_and_types(spmm_npu):
    big = normal((50, 64), torch.bfloat16, 7).cuda()
    grad = normal((4, 3, 5, 20), torch.bfloat16, 8).cuda()
    ids = ids_of("uniform", 60, 50).view(4, 3, 5)
    for weight in (big[:, 3:23], big[::2, 40:60].clone()[:25], big.t()[:20].t()):
        index = ids % weight.size(0)
        run(spmm_npu, weight.detach(), index, -1.5, grad)
        run(spmm_npu, weight.detach(), index.transpose(0, 2), 2.0, grad.permute(2, 1, 0, 3))
    weight = big[:, :20].detach()
    run(spmm_npu, weight, ids % 50, 1.0, grad.new_ones(1, 1, 1, 20).expand(4, 3, 5, 20))
    run(spmm_npu, weight, torch.tensor(7, device="cuda"), 1.0, grad[0, 0, 0])


def test_empty_extents(spmm_npu):
    for count, table, width in ((0, 5, 4), (3, 0, 4), (3, 5, 0), (0, 0, 0)):
        weight = torch.ones(table, width, device="cuda", requires_grad=True)
        out = spmm_npu.embedding(weight, torch.zeros(count, dtype=torch.int64, device="cuda"))
        assert out.shape == (count, width) and (table > 0 or not out.any())
        (dw,) = torch.autograd.grad(out, weight, torch.ones_like(out))
        assert dw.shape == (table, width) and float(dw.sum()) == (count * width if table else 0)
    two = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    weight = torch.ones(4, 0, device="cuda", requires_grad=True)
    out = spmm_npu.embedding(weight, two)
    assert out.shape == (2, 3, 0) and torch.autograd.grad(out, weight, torch.ones_like(out))[0].shape == (4, 0)


def test_repeats_exactly_and_on_another_stream(spmm_npu):
    weight = normal((700, 136), torch.float32, 9).cuda().requires_grad_(True)
    ids, grad = ids_of("zipf", 30000, 700), normal((30000, 136), torch.float32, 10).cuda()
    first = torch.autograd.grad(spmm_npu.embedding(weight, ids), weight, grad)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = torch.autograd.grad(spmm_npu.embedding(weight, ids), weight, grad)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    # An offset view of the gradient and its values elsewhere in memory give the same bits.
    shifted = torch.zeros(30000, 139, device="cuda")
    shifted[:, 1:137] = grad
    third = torch.autograd.grad(spmm_npu.embedding(weight, ids), weight, shifted[:, 1:137])[0]
    assert torch.equal(first, third)


def test_graph_replays(spmm_npu):
    weight = normal((300, 64), torch.bfloat16, 11).cuda()
    grad = normal((5000, 64), torch.bfloat16, 12).cuda()
    ids = ids_of("zipf", 5000, 300)

    def step():
        leaf = weight.detach().requires_grad_(True)
        out = spmm_npu.embedding(leaf, ids, scale=8.0)
        return out.detach(), torch.autograd.grad(out, leaf, grad)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = step()
    for k in range(4):
        ids.copy_(ids_of("absent" if k % 2 else "zipf", 5000, 300, seed=k))
        weight.copy_(normal((300, 64), torch.bfloat16, 20 + k).cuda())
        graph.replay()
        want = step()
        assert torch.equal(out, want[0]) and torch.equal(dw, want[1])


def test_infinities_and_nan_stay_in_their_rows(spmm_npu):
    weight = torch.ones(6, 16, device="cuda", dtype=torch.float16)
    weight[2], weight[4] = float("inf"), float("nan")
    leaf = weight.requires_grad_(True)
    ids = torch.tensor([0, 2, 4, 9, -1], device="cuda")
    out = spmm_npu.embedding(leaf, ids)
    assert bool(torch.isinf(out[1]).all()) and bool(torch.isnan(out[2]).all()) and not out[3:].any()
    grad = torch.ones(5, 16, device="cuda", dtype=torch.float16)
    grad[1], grad[3] = float("nan"), float("inf")  # of row 2, and of none
    (dw,) = torch.autograd.grad(out, leaf, grad)
    assert bool(torch.isnan(dw[2]).all()) and bool((dw[[0, 4]] == 1).all()) and not dw[[1, 3, 5]].any()


def test_refusals(spmm_npu):
    w, ids = torch.ones(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for weight, index, text in ((w[0], ids, "2D Tensor"), (w.double(), ids, "FP16, BF16 and FP32"),
                                (w, ids.float(), "int32 or int64"), (w, ids.cpu(), "must be a GPU tensor"),
                                (w, ids.bool(), "int32 or int64")):
        with pytest.raises(RuntimeError, match=text):
            spmm_npu.embedding(weight, index)
    with pytest.raises(ValueError, match="scale must be finite"):
        spmm_npu.embedding(w, ids, scale=float("inf"))
    out = spmm_npu.embedding(w.requires_grad_(True), ids)
    (g,) = torch.autograd.grad(out.sum(), w, create_graph=False)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(spmm_npu.embedding(w, ids).square().sum(), w, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w.detach(), torch.ones_like(w))
        with pytest.raises(RuntimeError, match="forward-mode"):
            spmm_npu.embedding(dual, ids)


@pytest.mark.parametrize("count,table,width,dtype", [(262144, 3000, 512, torch.bfloat16), (140001, 70000, 512, torch.float16),
                                                     (300000, 100, 128, torch.float32), (1200001, 5000, 4, torch.float16)])
def test_many_ids(spmm_npu, count, table, width, dtype):
    """Longer ranges of positions, runs over hundreds of them, several rounds of the sort's tiles;
    against 64-bit sums on the GPU, bounds as above."""
    g = torch.Generator(device="cuda").manual_seed(count)
    weight = torch.randn(table, width, generator=g, device="cuda").to(dtype).requires_grad_(True)
    grad = torch.randn(count, width, generator=g, device="cuda").to(dtype)
    for kind in ("zipf", "uniform"):
        ids = ids_of(kind, count, table)
        out = spmm_npu.embedding(weight, ids, scale=0.25)
        assert torch.equal(out, (weight.detach().float()[ids] * 0.25).to(dtype))
        (dw,) = torch.autograd.grad(out, weight, grad)
        total = torch.zeros(table, width, dtype=torch.float64, device="cuda").index_add_(0, ids, grad.double())
        size = torch.zeros(table, width, dtype=torch.float64, device="cuda").index_add_(0, ids, grad.double().abs())
        named = torch.bincount(ids, minlength=table).double()[:, None]
        check(dw, total * 0.25, ((named + 2) * E32 * size * 0.25).cpu(), kind)
        assert torch.equal(dw, torch.autograd.grad(spmm_npu.embedding(weight, ids, scale=0.25), weight, grad)[0])


def test_tables_of_more_than_2_31_elements(spmm_npu):
    rows, width = (1 << 21) + 7, 1032
    weight = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    weight[-1], weight[-2], weight[3] = 3.0, 2.0, 1.0
    ids = torch.tensor([rows - 1, 3, rows - 2, rows, 0, rows - 1], device="cuda")
    leaf = weight.requires_grad_(True)
    out = spmm_npu.embedding(leaf, ids)
    assert out[:, 0].tolist() == [3.0, 1.0, 2.0, 0.0, 0.0, 3.0] and out[:, -1].tolist() == out[:, 0].tolist()
    (dw,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert dw[[rows - 1, rows - 2, 3, 0], -1].tolist() == [2.0, 1.0, 1.0, 1.0]
    assert float(dw.float().sum(1).sum()) == 5 * width
