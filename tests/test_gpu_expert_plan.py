"""ExpertPlan: its sort by hand, packed rows bit for bit, and the sums and
gradients against 64 bits: a sum of k terms is off by (k + 1) e sum|terms|, a
product of two rows by (width / 32 + 64) e sum|terms|, each result rounds once."""

import numpy as np
import pytest
import torch

from expert_ops_plain import DTYPES, E32, check, normal, plan

pytestmark = pytest.mark.gpu


def choices(rows, k, count, seed=0, dropped=0.1):
    rng = np.random.default_rng(seed + rows + 13 * k + 101 * count)
    ids = np.minimum((count * rng.random((rows, k)) ** 2).astype(np.int64), count - 1)
    out = rng.random((rows, k)) < dropped
    ids[out] = rng.choice([-1, count, count + 5, -(1 << 40), 1 << 33], out.sum())
    return torch.from_numpy(ids)


def run(f, ids, count, x, y, w, grad):
    rows, k = ids.shape
    width = x.size(1)
    p = f.ExpertPlan(ids.cuda(), count)
    offsets, place = plan(ids, count)
    assert torch.equal(p.offsets.cpu(), offsets) and torch.equal(p.place.cpu().reshape(-1), place)
    assert p.place.shape == (rows, k) and p.offsets.dtype == p.place.dtype == torch.int32
    kept = ((ids >= 0) & (ids < count)).view(rows, k, 1)
    at = place.long()
    x, y, w = (t.detach().requires_grad_(True) for t in (x, y, w))
    packed = p.pack(x)
    want = torch.zeros(rows * k, width, dtype=x.dtype)
    want[at] = (x.detach().cpu()[:, None, :] * kept).reshape(rows * k, width)
    assert packed.dtype == x.dtype and torch.equal(packed.detach().cpu(), want)
    out = p.restore(y, w)
    yd = torch.where(kept, y.detach().double().cpu()[at].view(rows, k, width), 0.0)
    wd = torch.where(kept, w.detach().double().cpu()[:, :, None], 0.0)
    check(out, (yd * wd).sum(1), (k + 1) * E32 * (yd * wd).abs().sum(1), "out")
    dpacked = y.detach()
    (dx,) = torch.autograd.grad(packed, x, dpacked)
    check(dx, yd.sum(1), (k + 1) * E32 * yd.abs().sum(1), "dx")
    dy, dw = torch.autograd.grad(out, (y, w), grad)
    gd = grad.double().cpu()[:, None, :]
    wanted = torch.zeros(rows * k, width, dtype=torch.float64)
    wanted[at] = (wd * gd).reshape(rows * k, width)
    check(dy, wanted, E32 * wanted.abs(), "dy")
    check(dw, (yd * gd).sum(2), (width / 32 + 64) * E32 * (yd * gd).abs().sum(2), "dw")
    # Each gradient alone.
    assert torch.equal(torch.autograd.grad(p.restore(y, w.detach()), y, grad)[0], dy)
    assert torch.equal(torch.autograd.grad(p.restore(y.detach(), w), w, grad)[0], dw)


SIZES = [(1, 1, 1, 1), (1, 4, 8, 16), (13, 2, 8, 512), (7, 3, 5, 33), (100, 1, 12, 128), (33, 8, 64, 70), (300, 5, 256, 9),
         (64, 64, 100, 24), (5, 2, 2048, 1032), (17, 7, 3, 2100), (2049, 2, 7, 40), (1500, 6, 300, 65)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,count,width", SIZES)
def test_against_plain(spmm_npu, rows, k, count, width, dtype):
    ids = choices(rows, k, count)
    run(spmm_npu, ids, count, normal((rows, width), dtype, 1).cuda(), normal((rows * k, width), dtype, 2).cuda(),
        normal((rows, k), torch.float32, 3).cuda(), normal((rows, width), dtype, 4).cuda())


@pytest.mark.parametrize("dropped", [0.0, 1.0])
def test_all_or_no_choices_kept(spmm_npu, dropped):
    ids = choices(90, 3, 6, dropped=dropped)
    run(spmm_npu, ids, 6, normal((90, 48), torch.bfloat16, 1).cuda(), normal((270, 48), torch.bfloat16, 2).cuda(),
        normal((90, 3), torch.float32, 3).cuda(), normal((90, 48), torch.bfloat16, 4).cuda())


@pytest.mark.parametrize("count", [1, 2, 63, 64, 2047, 2048])
def test_sort_of_many_choices(spmm_npu, count):
    """More choices than a tile of the sort, of int32 and int64 ids."""
    ids = choices(9000, 3, count, dropped=0.05)
    offsets, place = plan(ids, count)
    for t in (ids.clamp(-1, count).int().cuda(), ids.cuda(), ids.t().contiguous().t().cuda()):
        p = spmm_npu.ExpertPlan(t, count)
        assert torch.equal(p.offsets.cpu(), offsets) and torch.equal(p.place.cpu().reshape(-1), place)
    one = spmm_npu.ExpertPlan(ids[:, 0].cuda(), count)
    offsets, place = plan(ids[:, 0], count)
    assert one.place.shape == (9000, 1) and torch.equal(one.place.cpu()[:, 0], place)
    assert torch.equal(one.offsets.cpu(), offsets)


@pytest.mark.parametrize("count,few", [(1, 128), (255, 128), (256, 127), (2048, 15)])
def test_sort_of_few_and_many_tiles(spmm_npu, count, few):
    """From one key beyond a launch's to one beyond the most of the few tiles, in 1 to 4 rounds a wave."""
    for n in (4097, 1024 * few, 1024 * few + 1, 2048 * few, 2048 * few + 1, 3000 * few, 4096 * few, 4096 * few + 1):
        ids = choices(n, 1, count, seed=n, dropped=0.05)
        offsets, place = plan(ids, count)
        p = spmm_npu.ExpertPlan(ids.cuda(), count)
        assert torch.equal(p.offsets.cpu(), offsets) and torch.equal(p.place.cpu().reshape(-1), place)


def test_strided_tensors(spmm_npu):
    ids = choices(60, 2, 4)
    big = normal((130, 100), torch.float16, 5).cuda()
    grad = normal((48, 60), torch.float16, 6).cuda().t()
    w = normal((2, 60), torch.float32, 7).cuda().t()
    run(spmm_npu, ids, 4, big[:60, 3:51], big[5:125, 50:98], w, grad)
    run(spmm_npu, ids, 4, big.t()[:60, :48], big[:120, ::2][:, :48], w, big[0, :48].expand(60, 48))


def test_empty_extents(spmm_npu):
    for rows, width in ((0, 8), (4, 0), (0, 0)):
        p = spmm_npu.ExpertPlan(torch.zeros(rows, 2, dtype=torch.int32, device="cuda"), 3)
        assert p.offsets.cpu().tolist() == [0, 2 * rows, 2 * rows, 2 * rows]
        x = torch.ones(rows, width, device="cuda", requires_grad=True)
        y = torch.ones(2 * rows, width, device="cuda", requires_grad=True)
        w = torch.ones(rows, 2, device="cuda", requires_grad=True)
        packed, out = p.pack(x), p.restore(y, w)
        assert packed.shape == y.shape and out.shape == x.shape
        grads = torch.autograd.grad((packed, out), (x, y, w), (torch.ones_like(packed), torch.ones_like(out)))
        assert all(g.shape == t.shape for g, t in zip(grads, (x, y, w))) and not grads[2].any()


def test_nothing_of_a_dropped_choice_is_seen(spmm_npu):
    """NaN and infinities in packed rows and weights of no expert."""
    ids = torch.tensor([[0, -1], [-1, -1], [1, 0]])
    p = spmm_npu.ExpertPlan(ids.cuda(), 2)
    y = torch.ones(6, 20, device="cuda")
    y[3:] = float("nan")
    w = torch.tensor([[2.0, float("nan")], [float("inf"), float("nan")], [3.0, 5.0]], device="cuda")
    y, w = y.requires_grad_(True), w.requires_grad_(True)
    out = p.restore(y, w)
    assert out[:, 0].tolist() == [2.0, 0.0, 8.0]
    dy, dw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert dw.tolist() == [[20.0, 0.0], [0.0, 0.0], [20.0, 20.0]]
    assert dy[:, 0].tolist() == [2.0, 5.0, 3.0, 0.0, 0.0, 0.0]
    x = torch.full((3, 20), float("inf"), device="cuda", requires_grad=True)
    packed = p.pack(x)
    assert not packed[3:].any() and bool(torch.isinf(packed[:3]).all())
    g = torch.ones(6, 20, device="cuda")
    g[3:] = float("nan")
    assert torch.autograd.grad(packed, x, g)[0][:, 0].tolist() == [1.0, 0.0, 2.0]


def test_plan_is_checked(spmm_npu):
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    p = spmm_npu.ExpertPlan(ids, 3)
    x, y, w = torch.ones(4, 8, device="cuda"), torch.ones(8, 8, device="cuda"), torch.ones(4, 2, device="cuda")
    for call, text in ((lambda: spmm_npu.ExpertPlan(ids.float(), 3), "int32 or int64"),
                       (lambda: spmm_npu.ExpertPlan(ids[None], 3), "1D or 2D"),
                       (lambda: spmm_npu.ExpertPlan(ids, 0), "1 to 2048 experts"),
                       (lambda: spmm_npu.ExpertPlan(ids, 4096), "1 to 2048 experts"),
                       (lambda: spmm_npu.ExpertPlan(ids, -3), "1 to 2048 experts"),
                       (lambda: spmm_npu.ExpertPlan(ids[:, :0], 3), "1 to 64 choices"),
                       (lambda: spmm_npu.ExpertPlan(torch.zeros(2, 65, dtype=torch.int32, device="cuda"), 3),
                        "1 to 64 choices"),
                       (lambda: p.pack(x[:3]), "4 rows"), (lambda: p.pack(x[0]), "2D Tensor"),
                       (lambda: p.pack(x.double()), "FP16, BF16 and FP32"), (lambda: p.pack(x.cpu()), "GPU tensor"),
                       (lambda: p.restore(y[:7], w), "8 packed rows"), (lambda: p.restore(y, w[:, :1]), "one entry"),
                       (lambda: p.restore(y, w.half()), "weights must be FP32"),
                       (lambda: p.restore(y, w.cpu()), "same device")):
        with pytest.raises(RuntimeError, match=text):
            call()
    leaf = y.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(p.restore(leaf, w).square().sum(), leaf, create_graph=True)


def test_graph_replays(spmm_npu):
    ids, x = choices(700, 2, 9).clamp(-1, 9).cuda(), normal((700, 72), torch.bfloat16, 8).cuda()
    w, g = normal((700, 2), torch.float32, 9).cuda(), normal((700, 72), torch.bfloat16, 10).cuda()

    def step():
        lx, lw = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        p = spmm_npu.ExpertPlan(ids, 9)
        out = p.restore(p.pack(lx), lw)
        return (p.offsets, p.place, out.detach()) + torch.autograd.grad(out, (lx, lw), g)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        ids.copy_(choices(700, 2, 9, seed=k).clamp(-1, 9).cuda())
        x.copy_(normal((700, 72), torch.bfloat16, 40 + k).cuda())
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("rows,k,count,width,dtype", [(70000, 2, 40, 520, torch.bfloat16), (300000, 3, 2000, 8, torch.float16),
                                                      (140000, 1, 3, 33, torch.float32)])
def test_many_rows(spmm_npu, rows, k, count, width, dtype):
    """Several rows a group of lanes and more than 512 tiles of the sort; against the GPU's stable sort
    and 64-bit sums, bounds as above."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = torch.randint(-1, count + 1, (rows, k), generator=g, device="cuda", dtype=torch.int32)
    key = torch.where((ids >= 0) & (ids < count), ids, torch.full_like(ids, count)).reshape(-1).long()
    place = torch.empty_like(key)
    place[key.argsort(stable=True)] = torch.arange(rows * k, device="cuda")
    p = spmm_npu.ExpertPlan(ids, count)
    assert torch.equal(p.place.reshape(-1).long(), place)
    assert torch.equal(p.offsets.long(), torch.searchsorted(key.sort().values, torch.arange(count + 1, device="cuda")))
    kept = (key < count).view(rows, k, 1)
    x = torch.randn(rows, width, generator=g, device="cuda").to(dtype).requires_grad_(True)
    y = torch.randn(rows * k, width, generator=g, device="cuda").to(dtype).requires_grad_(True)
    w = torch.randn(rows, k, generator=g, device="cuda").requires_grad_(True)
    grad = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    packed, out = p.pack(x), p.restore(y, w)
    want = (x.detach()[:, None, :] * kept).reshape(rows * k, width)
    assert torch.equal(packed.detach()[place], want)
    yd = torch.where(kept, y.detach().double()[place].view(rows, k, width), 0.0)
    wd = torch.where(kept, w.detach().double()[:, :, None], 0.0)
    check(out, (yd * wd).sum(1), ((k + 1) * E32 * (yd * wd).abs().sum(1)).cpu(), "out")
    (dx,) = torch.autograd.grad(packed, x, y.detach())
    check(dx, yd.sum(1), ((k + 1) * E32 * yd.abs().sum(1)).cpu(), "dx")
    dy, dw = torch.autograd.grad(out, (y, w), grad)
    gd = grad.double()[:, None, :]
    check(dy[place], (wd * gd).reshape(rows * k, width), (E32 * (wd * gd).abs().reshape(rows * k, width)).cpu(), "dy")
    check(dw, (yd * gd).sum(2), ((width / 32 + 64) * E32 * (yd * gd).abs().sum(2)).cpu(), "dw")


def test_packed_rows_of_more_than_2_31_elements(spmm_npu):
    rows, k, width = 1 << 20, 2, 1032
    ids = torch.tensor([[1, 0]], device="cuda").expand(rows, k)
    p = spmm_npu.ExpertPlan(ids, 2)
    x = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    x[-1], x[0] = 2.0, 1.0
    packed = p.pack(x)
    assert packed[[0, rows - 1, rows, 2 * rows - 1], -1].tolist() == [1.0, 2.0, 1.0, 2.0]
    assert float(packed[:, 0].float().sum()) == 6.0
    out = p.restore(packed, torch.tensor([[3.0, 4.0]], device="cuda").expand(rows, k))
    assert out[[0, -1], -1].tolist() == [7.0, 14.0] and not out[1:-1, 0].any()
