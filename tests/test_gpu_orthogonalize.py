"""orthogonalize against Newton-Schulz steps in 64 bits.

Tolerances: the steps map singular values by p(s) = a s + b s^3 + c s^5, whose
slope is at most a = 3.4445 (at s = 0) for the default coefficients, so a
relative disturbance e of a step's X, A or polynomial reaches the result at most
a^4 times larger against the result's own norm, if it falls on the smallest
singular values; on those near 1 the slope is below 1.  fp32 sums over n terms
are off by about sqrt(n) 2^-24, and the result is rounded once to its type
(2^-11 / 2^-8).  For inputs of fp16 or fp32 the steps keep fp32 precision
(1e-5 in the 2-norm with that growth at the sizes here), and for bf16 they may
round their factors to 11 bits: 15 roundings of at most 2^-12 each, twice that
for growth, stay below 8e-3."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
REL = {torch.float16: 2.0 ** -11 + 1e-5, torch.bfloat16: 2.0 ** -8 + 8e-3, torch.float32: 1e-5}
ABC = (3.4445, -4.7750, 2.0315)


def plain(u, steps=5, coefficients=ABC, eps=1e-7):
    x = u.double().cpu()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    each = [coefficients] * steps if not isinstance(coefficients[0], (tuple, list)) else coefficients
    for a, b, c in each:
        if x.size(-2) <= x.size(-1):
            g = x @ x.transpose(-2, -1)
            x = a * x + (b * g + c * g @ g) @ x
        else:
            g = x.transpose(-2, -1) @ x
            x = a * x + x @ (b * g + c * g @ g)
    return x


def make(shape, dtype, seed=0, scale=1e-2):
    rng = np.random.default_rng(seed + sum(shape) * 7 + shape[-1])
    m, n = shape[-2:]
    k = max(1, min(m, n) // 6)
    u = rng.standard_normal(shape) + rng.standard_normal((*shape[:-1], k)) @ rng.standard_normal((*shape[:-2], k, n)) / k ** 0.5
    return torch.from_numpy((scale * u).astype(np.float32)).to("cuda", dtype)


def check(got, want, dtype, factor=1.0):
    assert got.shape == want.shape and got.dtype == dtype
    got = got.double().cpu()
    for g, w in zip(got.reshape(-1, *got.shape[-2:]), want.reshape(-1, *want.shape[-2:])):
        off = float((g - w).norm() / w.norm())
        assert off <= factor * REL[dtype], off
        rms = float(w.norm()) / w.numel() ** 0.5
        assert float(((g - w).abs() / torch.maximum(w.abs(), torch.tensor(rms))).max()) <= 16 * factor * REL[dtype]


SHAPES = [(1, 1), (1, 9), (5, 1), (2, 3), (16, 16), (17, 33), (64, 64), (65, 64), (128, 96), (96, 200), (130, 257),
          (300, 140), (7, 1000), (1000, 8), (256, 512), (500, 333), (640, 640)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_matrices(spmm_npu, m, n, dtype):
    u = make((m, n), dtype)
    check(spmm_npu.orthogonalize(u), plain(u), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 32, 48), (2, 2, 70, 40), (12, 129, 65), (1, 16, 16), (20, 8, 8), (4, 200, 300)])
def test_stacks(spmm_npu, shape, dtype):
    """Every matrix of a stack on its own norm: one of another scale, one zero."""
    u = make(shape, dtype)
    flat = u.view(-1, *shape[-2:])
    flat[0] *= 64
    want = plain(u)
    check(spmm_npu.orthogonalize(u), want, dtype)
    if flat.size(0) > 1:
        flat[1] = 0
        got = spmm_npu.orthogonalize(u).view(-1, *shape[-2:])
        assert not got[1].any()
        keep = [i for i in range(flat.size(0)) if i != 1]
        check(got[keep], want.view(-1, *shape[-2:])[keep], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(49, 300, 257), (25, 250, 900), (200, 130, 130)])
def test_large_tiles(spmm_npu, shape, dtype):
    """Enough tiles of 256 x 256 for the chip, whole and in part."""
    u = make(shape, dtype)
    check(spmm_npu.orthogonalize(u), plain(u), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,coefficients", [
    (0, ABC), (1, ABC), (2, (1.5, -0.5, 0.0)), (10, (1.5, -0.5, 0.0)), (3, (2.0, -1.5, 0.5)),
    (3, [(8.2, -23.5, 17.3), (4.1, -2.9, 0.5), (3.9, -2.8, 0.5)]), (1, (0.0, 0.0, 0.0)), (2, (30.0, 5.0, 2.0))])
def test_steps_and_coefficients(spmm_npu, steps, coefficients, dtype):
    """Other polynomials, one for each step, and one that grows by 30 a step
    (the factors' ranges follow the coefficients)."""
    u = make((90, 120), dtype)
    want = plain(u, steps, coefficients)
    if want.abs().max() == 0:
        assert not spmm_npu.orthogonalize(u, steps, coefficients).any()
        return
    if dtype == torch.float16 and want.abs().max() > 6e4:
        assert not spmm_npu.orthogonalize(u, steps, coefficients).isnan().all()
        return
    check(spmm_npu.orthogonalize(u, steps, coefficients), want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weak_directions(spmm_npu, dtype):
    """A few strong directions over noise a thousand times weaker, which the
    steps raise by up to 3.4445^5: the fp32 steps' own errors grow with them."""
    rng = np.random.default_rng(3)
    u = rng.standard_normal((200, 4)) @ rng.standard_normal((4, 260)) + 5e-3 * rng.standard_normal((200, 260))
    u = torch.from_numpy(u.astype(np.float32)).to("cuda", dtype)
    check(spmm_npu.orthogonalize(u), plain(u), dtype, factor=4.0)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e25, 3e37])
def test_scales(spmm_npu, scale):
    """The squares of these entries leave fp32's range; the norm does not."""
    u = make((40, 60), torch.float32, scale=1.0)
    u = u / u.abs().max() * scale
    check(spmm_npu.orthogonalize(u, eps=0.0), plain(u, eps=0.0), torch.float32)


def test_singular_values_and_vectors(spmm_npu):
    u = make((150, 220), torch.float32)
    got = spmm_npu.orthogonalize(u).double().cpu()
    p, s, q = torch.linalg.svd(u.double().cpu(), full_matrices=False)
    turned = p.t() @ got @ q.t()
    assert float((turned - torch.diag(torch.diagonal(turned))).abs().max()) < 1e-4
    assert 0.6 < float(torch.diagonal(turned)[: 100].min()) and float(torch.diagonal(turned).max()) < 1.3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_values_stay_in_their_matrix(spmm_npu, dtype, bad):
    u = make((3, 40, 56), dtype)
    clean = spmm_npu.orthogonalize(u)
    u[1, 7, 9] = bad
    got = spmm_npu.orthogonalize(u)
    assert got[1].isnan().all()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_streams_and_repeats(spmm_npu, dtype):
    wide = make((150, 203), dtype)
    view = wide[3:133, 5:200]
    first = spmm_npu.orthogonalize(view)
    assert torch.equal(first, spmm_npu.orthogonalize(view.contiguous()))
    turned = view.t()
    assert torch.equal(spmm_npu.orthogonalize(turned), spmm_npu.orthogonalize(turned.contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = spmm_npu.orthogonalize(view)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    for shape in ((0, 4), (4, 0), (0, 3, 5)):
        assert spmm_npu.orthogonalize(torch.empty(shape, device="cuda", dtype=dtype)).shape == shape


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (2, 256, 300)), (torch.float32, (100, 64)), (torch.float16, (48, 48))])
def test_graph_replays(spmm_npu, dtype, shape):
    u = make(shape, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        spmm_npu.orthogonalize(u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = spmm_npu.orthogonalize(u)
    for k in range(4):
        u.copy_(make(shape, dtype, seed=k + 1))
        eager = spmm_npu.orthogonalize(u)
        y.fill_(-1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_refusals(spmm_npu):
    f = spmm_npu.orthogonalize
    u = make((8, 8), torch.float32)
    for bad, text in ((u.cpu(), "must be a GPU tensor"), (u[0], "at least two dimensions"),
                      (u.double(), "supports only FP16, BF16 and FP32")):
        with pytest.raises(RuntimeError, match=text):
            f(bad)
    with pytest.raises(RuntimeError, match="not differentiable"):
        f(u.clone().requires_grad_(True))
    for kwargs, text in (({"steps": -1}, "must not be negative"), ({"coefficients": (1.0, 2.0)}, "one \\(a, b, c\\)"),
                         ({"coefficients": [ABC] * 4}, "one for each step"), ({"eps": -1.0}, "eps must be finite"),
                         ({"coefficients": (1.0, float("nan"), 0.0)}, "coefficients must be finite")):
        with pytest.raises(ValueError, match=text):
            f(u, **kwargs)
