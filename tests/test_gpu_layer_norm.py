"""layer_norm forward and backward against the formulas in 64 bits, and the
gradient against differences of the 64-bit forward.

Tolerances: an output is rounded once (u: half a unit in the last place of its
type), and everything before it is fp32 with e = 2^-24.  A sum of n terms in
any order is off by at most n e sum|terms|; the kernels add at most n / 32 + 64
terms one after another, so that count stands for n.  Subtracting the mean
scales the relative error of a row by 1 + |mean| rstd."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def plain(x, w, b, dy, eps):
    """y, dx, dw, db and the bounds of their errors before rounding, in 64 bits."""
    x, dy = x.double().cpu(), dy.double().cpu()
    rows, n = x.shape
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if b is None else b.double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    z = (x - mean) * rstd
    g = dy * w
    y = z * w + b
    dx = rstd * (g - g.mean(1, keepdim=True) - z * (g * z).mean(1, keepdim=True))
    dw, db = (dy * z).sum(0), dy.sum(0)
    amp = 1 + mean.abs() * rstd
    row, col = (n / 32 + 64) * E32, (rows / 32 + 64) * E32
    zerr = row * amp * (1 + z.abs())
    bounds = (zerr * w.abs() + 4 * E32 * (y.abs() + b.abs()),
              row * amp * rstd * (g.abs() + g.abs().mean(1, keepdim=True)
                                  + (1 + z.abs()) * ((g * z).abs() + g.abs()).mean(1, keepdim=True)) * 2,
              col * (dy * z).abs().sum(0) + (dy.abs() * zerr).sum(0), col * dy.abs().sum(0))
    return (y, dx, dw, db), bounds


def check(got, want, bound, dtype, what):
    assert got.shape == want.shape, what
    err = (got.double().cpu() - want).abs()
    limit = U[dtype] * want.abs() + bound * (1 + U[dtype]) + TINY[dtype]
    bad = ~(err <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / limit).max()):.3g} x the bound"


def make(rows, n, dtype, seed=0, offset=0.5):
    rng = np.random.default_rng(seed + 31 * n + rows)
    t = lambda a: torch.from_numpy(np.asarray(a, np.float32)).to("cuda", dtype)  # noqa: E731
    x = t(rng.standard_normal((rows, n)) * np.exp(0.3 * rng.standard_normal((rows, 1))) + offset)
    return x, t(1 + 0.2 * rng.standard_normal(n)), t(0.2 * rng.standard_normal(n)), t(rng.standard_normal((rows, n)))


SHAPES = [(1, 1), (1, 128), (3, 2), (5, 8), (4, 9), (17, 33), (64, 128), (1000, 64), (7, 333), (257, 96), (33, 1000),
          (5, 1024), (70, 2048), (2, 4099), (3, 8192), (2, 20011), (1, 40000), (4097, 16), (301, 520)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_forward_and_gradients(spmm_npu, rows, n, dtype):
    x, w, b, dy = make(rows, n, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = spmm_npu.layer_norm(x, w, b, 1e-5)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, leaves, dy)
    want, bounds = plain(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    for got, ref, bound, what in zip((y.detach(), *grads), want, bounds, ("y", "dx", "dw", "db")):
        check(got, ref, bound, dtype, what)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [40, 1030, 9001])
def test_fp32_parameters(spmm_npu, dtype, n):
    x, w, b, dy = make(19, n, dtype)
    w, b = w.float().requires_grad_(True), b.float().requires_grad_(True)
    y = spmm_npu.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    want, bounds = plain(x, w.detach(), b.detach(), dy, 1e-5)
    check(y.detach(), want[0], bounds[0], dtype, "y")
    check(dw, want[2], bounds[2], torch.float32, "dw")
    check(db, want[3], bounds[3], torch.float32, "db")


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_missing_parameters(spmm_npu, which):
    x, w, b, dy = make(23, 70, torch.float32)
    x.requires_grad_(True)
    w = w if which == "weight" else None
    b = b.requires_grad_(True) if which == "bias" else None
    y = spmm_npu.layer_norm(x, w, b)
    want, bounds = plain(x.detach(), w, None if b is None else b.detach(), dy, 1e-5)
    grads = torch.autograd.grad(y, [x] if b is None else [x, b], dy)
    check(y.detach(), want[0], bounds[0], torch.float32, "y")
    check(grads[0], want[1], bounds[1], torch.float32, "dx")
    if b is not None:
        check(grads[1], want[3], bounds[3], torch.float32, "db")
    plain_y = spmm_npu.layer_norm(x.detach(), w, None if b is None else b.detach())
    assert torch.equal(plain_y, y.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [31, 128, 2056, 9000])
def test_views(spmm_npu, dtype, n):
    """Rows of a wider matrix at an odd offset, a 3D input, an expanded
    gradient and a column-major input give what contiguous ones give."""
    base, w, b, dy = make(12, n + 7, dtype)
    w, b = w[:n].contiguous(), b[:n].contiguous()
    view = base[:, 3:3 + n]
    assert torch.equal(spmm_npu.layer_norm(view, w, b), spmm_npu.layer_norm(view.contiguous(), w, b))
    cube = view.contiguous().view(3, 4, n)
    assert torch.equal(spmm_npu.layer_norm(cube, w, b).view(12, n), spmm_npu.layer_norm(view, w, b))
    turned = view.t().contiguous().t()
    assert torch.equal(spmm_npu.layer_norm(turned, w, b), spmm_npu.layer_norm(view, w, b))
    assert torch.equal(spmm_npu.layer_norm(view[5], w, b), spmm_npu.layer_norm(view, w, b)[5])

    def grads(x, g):
        x = x.detach().requires_grad_(True)
        ww = w.detach().requires_grad_(True)
        return torch.autograd.grad(spmm_npu.layer_norm(x, ww, b), (x, ww), g)

    one = dy[:, :1].expand(12, n)
    for g in (one, dy[:, 2:2 + n]):
        for got, want in zip(grads(view, g), grads(view.contiguous(), g.contiguous())):
            assert torch.equal(got, want)


def test_constant_rows_large_means_and_bad_values(spmm_npu):
    n = 300
    x, w, b, dy = make(6, n, torch.float32)
    x[0] = 3.25           # no spread: y is the bias
    x[1] += 1e4           # mean far above the spread
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x.requires_grad_(True)
    y = spmm_npu.layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, dy)
    y = y.detach()
    assert torch.equal(y[0], b)
    assert y[2].isnan().all() and y[3].isnan().all() and dx[2].isnan().all() and dx[3].isnan().all()
    keep = [0, 1, 4, 5]
    want, bounds = plain(x.detach()[keep], w, b, dy[keep], 1e-5)
    check(y[keep], want[0], bounds[0], torch.float32, "y")
    check(dx[keep], want[1], bounds[1], torch.float32, "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 256, 40000])
def test_no_rows(spmm_npu, dtype, n):
    x = torch.empty(0, n, device="cuda", dtype=dtype, requires_grad=True)
    w = torch.ones(n, device="cuda", dtype=dtype, requires_grad=True)
    b = torch.zeros(n, device="cuda", dtype=dtype, requires_grad=True)
    y = spmm_npu.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, n, device="cuda", dtype=dtype))
    assert y.shape == dx.shape == (0, n) and not dw.any() and not db.any()


def test_gradient_against_differences(spmm_npu):
    """Central differences of the 64-bit forward along random directions: off
    by h^2 / 6 times the third derivative (1e-6 of the value at h = 1e-4 here)
    and the rounding of the fp32 gradient."""
    rows, n, h = 9, 50, 1e-4
    x, w, b, dy = make(rows, n, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(spmm_npu.layer_norm(x, w, b), leaves, dy)
    rng = np.random.default_rng(4)

    def value(xd, wd, bd):
        m = xd.mean(1, keepdim=True)
        z = (xd - m) / torch.sqrt(((xd - m) ** 2).mean(1, keepdim=True) + 1e-5)
        return float(((z * wd + bd) * dy.double().cpu()).sum())

    at = [t.detach().double().cpu() for t in leaves]
    for k in range(3):
        v = torch.from_numpy(rng.standard_normal(tuple(at[k].shape)))
        hi, lo = list(at), list(at)
        hi[k], lo[k] = at[k] + h * v, at[k] - h * v
        slope = (value(*hi) - value(*lo)) / (2 * h)
        got = float((grads[k].double().cpu() * v).sum())
        scale = float((grads[k].double().cpu() * v).abs().sum())
        assert abs(got - slope) <= 1e-5 * scale


def test_repeats_exactly_and_on_another_stream(spmm_npu):
    x, w, b, dy = make(5000, 136, torch.float16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = spmm_npu.layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype,rows,n", [(torch.float16, 700, 128), (torch.float32, 90, 5000)])
def test_graph_replays(spmm_npu, dtype, rows, n):
    x, w, b, dy = make(rows, n, dtype)
    y_eager = spmm_npu.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        spmm_npu.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = spmm_npu.layer_norm(x, w, b)
    for k in range(4):
        x.copy_(make(rows, n, dtype, seed=k)[0])
        y_eager = spmm_npu.layer_norm(x, w, b)
        y.fill_(-1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, y_eager)


def test_refusals(spmm_npu):
    f = spmm_npu.layer_norm
    x, w, b, dy = make(4, 16, torch.float16)
    for bad, text in (((x.cpu(), None, None), "must be a GPU tensor"),
                      ((x.double(), None, None), "supports only FP16, BF16 and FP32"),
                      ((x, w[:8], None), "weight must be a 1D Tensor of 16 elements"),
                      ((x, None, b.view(4, 4)), "bias must be a 1D Tensor"),
                      ((x, w.bfloat16(), None), "weight must have the dtype of x or be FP32"),
                      ((x, w.float(), b), "weight and bias must have the same dtype"),
                      ((x, w.cpu(), None), "weight must be on the same device"),
                      ((x[:, :0], None, None), "at least one element"),
                      ((x[0, 0], None, None), "at least one dimension")):
        with pytest.raises(RuntimeError, match=text):
            f(*bad)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps must be finite"):
            f(x, w, b, eps)
    x.requires_grad_(True)
    y = f(x, w, b)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y, x, dy, create_graph=True)
