"""grouped_matmul forward and backward against 64-bit products, for ragged and
empty groups, rows outside all groups, odd sizes, strides and storage orders.

Tolerances: an output is rounded once (u: half a unit in the last place of its
type); the products of fp16 and bf16 values are exact in fp32 and those of fp32
values off by e = 2^-24 each, and a sum of n fp32 terms in any order is off by
at most (n + 1) e sum|terms|."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def make(rows, groups, inner, width, dtype, seed=0):
    rng = np.random.default_rng(seed + rows + 7 * inner + 13 * width)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to("cuda", dtype)  # noqa: E731
    return t(rows, inner), t(groups, inner, width), t(rows, width)


def edges_of(sizes, before=0):
    return [before, *(before + int(v) for v in np.cumsum(sizes))]


def plain(x, w, edges, dy):
    """out, dx, dw and the sums of their terms' magnitudes and term counts."""
    x, w, dy = x.double().cpu(), w.double().cpu(), dy.double().cpu()
    out, dx, dw = torch.zeros(x.size(0), w.size(2)).double(), torch.zeros_like(x), torch.zeros_like(w)
    mag = [torch.zeros_like(t) for t in (out, dx, dw)]
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        a, d = x[lo:hi], dy[lo:hi]
        for k, (p, q) in enumerate(((a, w[g]), (d, w[g].t()), (a.t(), d))):
            (out[lo:hi], dx[lo:hi], dw[g])[k].copy_(p @ q)
            (mag[0][lo:hi], mag[1][lo:hi], mag[2][g])[k].copy_(p.abs() @ q.abs())
    longest = max((hi - lo for lo, hi in zip(edges, edges[1:])), default=0)
    return (out, dx, dw), mag, (x.size(1), w.size(2), longest)


def check(got, want, mag, terms, dtype, what):
    assert got.shape == want.shape and got.dtype == dtype, what
    err = (got.double().cpu() - want).abs()
    limit = U[dtype] * want.abs() + (terms + 2) * E32 * mag * (1 + U[dtype]) + TINY[dtype]
    bad = ~(err <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / limit).max()):.3g} x the bound"


def run_all(f, x, w, edges, dy, index=torch.int32):
    off = torch.tensor(edges, dtype=index, device="cuda")
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = f(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    return y.detach(), dx, dw


CASES = [
    # sizes of the groups, inner, width
    ([1], 1, 1), ([1], 16, 16), ([3, 0, 5], 8, 8), ([0, 0, 0, 7], 33, 65), ([64, 64], 64, 64), ([63, 65, 1], 128, 130),
    ([130, 0, 257, 31], 96, 72), ([1] * 70, 48, 40), ([500, 2, 300], 333, 190), ([13], 512, 260), ([700], 40, 1024),
    ([5, 600, 1, 0, 90], 256, 256), ([200, 56], 17, 5), ([1, 0, 1, 1], 1000, 24), ([2000, 10], 7, 300), ([3000], 64, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,inner,width", CASES)
def test_products_and_gradients(spmm_npu, sizes, inner, width, dtype):
    x, w, dy = make(sum(sizes), len(sizes), inner, width, dtype)
    edges = edges_of(sizes)
    want, mag, terms = plain(x, w, edges, dy)
    for got, ref, m, n, what in zip(run_all(spmm_npu.grouped_matmul, x, w, edges, dy), want, mag, terms, ("y", "dx", "dw")):
        check(got, ref, m, n, dtype, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,inner,width", [([40, 0, 77], 64, 96), ([9, 300], 37, 51), ([200, 190, 3], 256, 512)])
def test_transposed_weights(spmm_npu, sizes, inner, width, dtype):
    """weight stored [groups, width, inner] and turned: the same results, the
    gradient in the same storage order."""
    x, w, dy = make(sum(sizes), len(sizes), inner, width, dtype)
    turned = w.transpose(1, 2).contiguous().transpose(1, 2)
    edges = edges_of(sizes)
    want, mag, terms = plain(x, w, edges, dy)
    got = run_all(spmm_npu.grouped_matmul, x, turned, edges, dy)
    assert got[2].stride(1) == 1
    for g, ref, m, n, what in zip(got, want, mag, terms, ("y", "dx", "dw")):
        check(g, ref, m, n, dtype, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_rows_outside_the_groups(spmm_npu, dtype, index):
    """They become zero in the output and in dx, and do not reach dw, even
    where they hold NaN."""
    sizes, before, after = [30, 0, 85], 70, 41
    rows = before + sum(sizes) + after
    x, w, dy = make(rows, 3, 72, 88, dtype)
    edges = edges_of(sizes, before)
    inside = slice(before, before + sum(sizes))
    want, mag, terms = plain(x[inside], w, edges_of(sizes), dy[inside])
    x[:before] = float("nan")
    dy[before + sum(sizes):] = float("nan")
    y, dx, dw = run_all(spmm_npu.grouped_matmul, x, w, edges, dy, index)
    check(y[inside], want[0], mag[0], terms[0], dtype, "y")
    check(dx[inside], want[1], mag[1], terms[1], dtype, "dx")
    check(dw, want[2], mag[2], terms[2], dtype, "dw")
    for t in (y, dx):
        assert not t[:before].any() and not t[before + sum(sizes):].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_values_stay_in_their_rows(spmm_npu, dtype):
    """A NaN or infinity reaches its own row of the output and its own row of
    dw, and no neighbouring group; columns past a row's end do not leak in."""
    sizes = [70, 50]
    x, w, dy = make(sum(sizes), 2, 45, 37, dtype)
    clean = run_all(spmm_npu.grouped_matmul, x, w, edges_of(sizes), dy)
    x[69, 44], x[70, 0] = float("nan"), float("inf")
    y, dx, dw = run_all(spmm_npu.grouped_matmul, x, w, edges_of(sizes), dy)
    assert y[69].isnan().all() and not y[70].isfinite().any()
    ordinary = [r for r in range(120) if r not in (69, 70)]
    assert torch.equal(y[ordinary], clean[0][ordinary]) and torch.equal(dx, clean[1])
    assert dw[0, 44].isnan().all() and not dw[1, 0].isfinite().any()
    assert torch.equal(dw[0, :44], clean[2][0, :44]) and torch.equal(dw[1, 1:], clean[2][1, 1:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner,width", [(40, 48), (77, 33), (256, 264)])
def test_infinities(spmm_npu, dtype, inner, width):
    """Infinite where the products say so, with their sign, also against
    factors of few digits, and NaN against zeros."""
    sizes = [40, 90]
    x, w, dy = make(sum(sizes), 2, inner, width, dtype)
    w[0, 3, :] = torch.randint(-2, 3, (width,), device="cuda").to(dtype)  # zeros, ones and twos
    x[5, 3], x[17, 3], x[100, 0] = float("inf"), float("-inf"), float("inf")
    want, _, _ = plain(x, w, edges_of(sizes), dy)
    y, dx, dw = run_all(spmm_npu.grouped_matmul, x, w, edges_of(sizes), dy)
    for got, ref in ((y, want[0]), (dw, want[2])):
        got = got.double().cpu()
        assert torch.equal(got.isnan(), ref.isnan())
        infinite = ref.isinf()
        assert infinite.any() and torch.equal(got[infinite], ref[infinite]) and got[ref.isfinite()].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner,width", [(40, 48), (129, 130), (256, 64)])
def test_views(spmm_npu, dtype, inner, width):
    """Columns of a wider x at an odd offset, an expanded and a strided
    gradient, and weights at an odd offset and apart give what contiguous
    ones give."""
    sizes = [33, 90]
    bx, _, bdy = make(123, 2, inner + 5, width + 3, dtype)
    flat = torch.randn(2 * (inner * width + 11) + 1, device="cuda").to(dtype)
    w = flat[1:].as_strided((2, inner, width), (inner * width + 11, width, 1), 1)
    x, dy = bx[:, 1:1 + inner], bdy[:, 3:3 + width]
    edges = edges_of(sizes)
    f = spmm_npu.grouped_matmul
    for g in (dy, dy[:, :1].expand(123, width), dy[:1].expand(123, width)):
        for got, want in zip(run_all(f, x, w, edges, g), run_all(f, x.contiguous(), w.contiguous(), edges, g.contiguous())):
            assert torch.equal(got, want)
    x = bx.t().contiguous().t()[:, :inner]
    assert torch.equal(run_all(f, x, w, edges, dy)[0], run_all(f, x.contiguous(), w.contiguous(), edges, dy)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,groups,inner,width", [(0, 3, 16, 16), (5, 2, 0, 8), (5, 2, 8, 0), (6, 0, 8, 8)])
def test_empty_extents(spmm_npu, rows, groups, inner, width, dtype):
    x, w, dy = make(rows, groups, inner, width, dtype)
    edges = [0] * groups + [rows if groups else 0]
    y, dx, dw = run_all(spmm_npu.grouped_matmul, x, w, edges, dy)
    assert y.shape == (rows, width) and dx.shape == x.shape and dw.shape == w.shape
    assert not y.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_one_group_of_many_rows(spmm_npu, dtype):
    """Sums over 20000 rows."""
    x, w, dy = make(20000, 1, 40, 72, dtype)
    want, mag, terms = plain(x, w, [0, 20000], dy)
    for got, ref, m, n, what in zip(run_all(spmm_npu.grouped_matmul, x, w, [0, 20000], dy), want, mag, terms, "abc"):
        check(got, ref, m, n, dtype, what)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("sizes,inner,width", [([9000, 0, 16001, 300], 264, 520), ([24999, 130, 3], 512, 264),
                                               ([700, 1000, 24001], 192, 776)])
def test_large_tiles(spmm_npu, sizes, inner, width, turned, dtype):
    """Enough rows for the 256 x 256 tiles, whose last steps, rows and columns
    are parts of one; rows before and behind the groups."""
    before, after = 300, 77
    rows = before + sum(sizes) + after
    x, w, dy = make(rows, len(sizes), inner, width, dtype)
    if turned:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    inside = slice(before, before + sum(sizes))
    want, mag, terms = plain(x[inside], w, edges_of(sizes), dy[inside])
    y, dx, dw = run_all(spmm_npu.grouped_matmul, x, w, edges_of(sizes, before), dy)
    check(y[inside], want[0], mag[0], terms[0], dtype, "y")
    check(dx[inside], want[1], mag[1], terms[1], dtype, "dx")
    check(dw, want[2], mag[2], terms[2], dtype, "dw")
    for t in (y, dx):
        assert not t[:before].any() and not t[before + sum(sizes):].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("edges,inner,width", [([100, 230], 128, 128), ([0, 64, 130, 131], 72, 40), ([19000, 19000, 19500], 256, 512),
                                               ([0, 0], 200, 136), ([5, 390], 33, 65)])
def test_few_of_many_rows_in_groups(spmm_npu, edges, inner, width, dtype):
    """Far fewer rows in the groups than the tensor has.  Memory that held NaN
    before is handed out again as the gradient's workspace."""
    x, w, dy = make(20000, len(edges) - 1, inner, width, dtype)
    want, mag, terms = plain(x, w, edges, dy)
    for size in (24, 26, 27):
        torch.full((1 << size,), float("nan"), device="cuda")
    for got, ref, m, n, what in zip(run_all(spmm_npu.grouped_matmul, x, w, edges, dy), want, mag, terms, ("y", "dx", "dw")):
        check(got, ref, m, n, dtype, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,most,inner,width", [(150, 200, 512, 512), (40, 900, 256, 264), (300, 5, 128, 128), (90, 130, 640, 321)])
def test_many_groups(spmm_npu, groups, most, inner, width, dtype):
    sizes = [int(v) for v in np.random.default_rng(groups).integers(0, most, groups)]
    x, w, dy = make(sum(sizes), groups, inner, width, dtype)
    edges = edges_of(sizes)
    want, mag, terms = plain(x, w, edges, dy)
    for got, ref, m, n, what in zip(run_all(spmm_npu.grouped_matmul, x, w, edges, dy), want, mag, terms, ("y", "dx", "dw")):
        check(got, ref, m, n, dtype, what)


def test_offsets_past_32_bits(spmm_npu):
    """x of more than 2^31 elements: its last rows are where they should be."""
    rows, inner, width = 270_000, 8192, 16
    x = torch.zeros(rows, inner, dtype=torch.float16, device="cuda")
    x[-1, -1], x[-2, 0], x[0, 1] = 2.0, 3.0, 1.0
    w = torch.randn(2, inner, width, device="cuda").half()
    y = spmm_npu.grouped_matmul(x, w, torch.tensor([0, rows - 1, rows], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[-1], 2 * w[1, -1]) and torch.equal(y[0], w[0, 1])
    assert torch.equal(y[-2], (3 * w[0, 0].float()).half()) and not y[1:-2].any()


@pytest.mark.parametrize("dtype", [torch.float32])
def test_gradient_against_differences(spmm_npu, dtype):
    """The product is linear in x and in weight, so a difference along a
    direction is exact but for rounding: fp32 terms of 64-bit differences."""
    sizes = [11, 0, 24]
    x, w, dy = make(35, 3, 20, 28, dtype)
    edges = edges_of(sizes)
    _, dx, dw = run_all(spmm_npu.grouped_matmul, x, w, edges, dy)
    value = lambda a, b: float((plain(a, b, edges, dy)[0][0] * dy.double().cpu()).sum())  # noqa: E731
    rng = np.random.default_rng(0)
    for grad, at, other in ((dx, x, lambda v: value(v, w)), (dw, w, lambda v: value(x, v))):
        v = torch.from_numpy(rng.standard_normal(tuple(at.shape))).cuda()
        slope = (other(at.double() + v) - other(at.double() - v)) / 2
        terms = grad.double() * v
        assert abs(float(terms.sum()) - slope) <= 64 * E32 * float(terms.abs().sum()) + 1e-9


def test_repeats_exactly_and_on_another_stream(spmm_npu):
    sizes = [900, 0, 1500, 77]
    x, w, dy = make(sum(sizes), 4, 128, 192, torch.bfloat16)
    first = run_all(spmm_npu.grouped_matmul, x, w, edges_of(sizes), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run_all(spmm_npu.grouped_matmul, x, w, edges_of(sizes), dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,rows", [(torch.float16, 600), (torch.bfloat16, 9), (torch.float32, 300)])
def test_graph_replays_follow_the_offsets(spmm_npu, dtype, rows):
    """The split into groups is read on the device: a captured call follows
    new offsets."""
    x, w, _ = make(rows, 3, 64, 96, dtype)
    off = torch.tensor([0, rows // 3, rows // 2, rows], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        spmm_npu.grouped_matmul(x, w, off)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = spmm_npu.grouped_matmul(x, w, off)
    for cut in ([0, 1, 5, rows], [0, 0, 0, rows], [2, rows // 2, rows - 1, rows - 1], [0, rows, rows, rows]):
        off.copy_(torch.tensor(cut, dtype=torch.int32))
        eager = spmm_npu.grouped_matmul(x, w, off)
        y.fill_(-1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_refusals(spmm_npu):
    f = spmm_npu.grouped_matmul
    x, w, _ = make(6, 2, 8, 10, torch.float16)
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    for bad, text in (((x.cpu(), w, off), "x must be a GPU tensor"),
                      ((x, w, off.cpu()), "offsets must be a GPU tensor"),
                      ((x[0], w, off), "x must be a 2D Tensor"),
                      ((x, w[0], off), "weight must be a 3D Tensor"),
                      ((x, w, off[None]), "offsets must be a 1D Tensor"),
                      ((x.double(), w.double(), off), "supports only FP16, BF16 and FP32"),
                      ((x, w.float(), off), "weight must have the dtype of x"),
                      ((x[:, :7], w, off), "x has 7 columns, but weight takes 8"),
                      ((x, w, off[:2]), "offsets must hold one entry more"),
                      ((x, w, off.float()), "must be an int32 or int64 tensor")):
        with pytest.raises(RuntimeError, match=text):
            f(*bad)
    x.requires_grad_(True)
    y = f(x, w, off)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
