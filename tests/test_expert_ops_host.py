"""The operators around a layer of experts on the host, without a GPU: their
entry points exist, their C ABI refuses before any device call what it cannot
run, and sizes its workspaces also for empty extents; their 64-bit gradients
agree with differences of the 64-bit forward."""

import ctypes
import os

import pytest
import torch

import expert_ops_plain as plain

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "ascend-spmm_amd", "libspmm_mi355x.so")

F16, F32, F64, BF16 = 0, 1, 2, 3
I64, I32, F64C = ctypes.c_int64, ctypes.c_int32, ctypes.c_double
FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every check precedes the launch


class EmbeddingDesc(ctypes.Structure):
    _fields_ = [("count", I64), ("table_rows", I64), ("width", I64), ("weight_stride", I64), ("grad_stride", I64),
                ("scale", F64C), ("index_type", I32), ("value_type", I32)]


class RouteDesc(ctypes.Structure):
    _fields_ = [("rows", I64), ("experts", I64), ("logits_stride", I64), ("top_k", I64), ("groups", I64),
                ("top_groups", I64), ("scale", F64C), ("score", I32), ("renormalize", I32), ("value_type", I32)]


class ExpertsDesc(ctypes.Structure):
    _fields_ = [("rows", I64), ("top_k", I64), ("experts", I64), ("width", I64), ("stride", I64), ("grad_stride", I64),
                ("value_type", I32)]


class LogProbsDesc(ctypes.Structure):
    _fields_ = [("rows", I64), ("classes", I64), ("logits_stride", I64), ("top", I64), ("index_type", I32),
                ("value_type", I32)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.fail(f"{LIB} is not built (python ascend-spmm_amd/build.py)")
    lib = ctypes.CDLL(LIB)
    lib.spmm_last_error.restype = ctypes.c_char_p
    return lib


def emb(count=8, table=10, width=16, stride=None, grad_stride=None, scale=1.0, index=1, value=F16):
    return EmbeddingDesc(count, table, width, width if stride is None else stride,
                         width if grad_stride is None else grad_stride, scale, index, value)


def test_embedding_refusals(lib):
    def run(d, ids=FAKE, out=FAKE):
        return lib.spmm_embedding_run(ctypes.byref(d), FAKE, ids, out, None)

    for d, code, text in ((emb(value=F64), 4, b"FP16, BF16 and FP32"), (emb(index=3), 4, b"int32 or int64"),
                          (emb(count=-1), 4, b"negative extent"), (emb(count=1 << 30), 4, b"below 2^30"),
                          (emb(table=1 << 30), 4, b"below 2^30"), (emb(width=1 << 22), 4, b"below 2^22"),
                          (emb(stride=15), 4, b"rows of weight overlap"), (emb(scale=float("inf")), 1, b"finite"),
                          (emb(scale=float("nan")), 1, b"finite"), (emb(scale=-1e39), 1, b"finite")):
        assert run(d) == code and text in lib.spmm_last_error()
    assert run(emb(), ids=None) == 1 and run(emb(), out=None) == 1
    assert run(emb(count=0), ids=None, out=None) == 0 and run(emb(width=0), ids=None, out=None) == 0

    def back(d, grad=FAKE, dw=FAKE, ws=FAKE, size=1 << 30):
        return lib.spmm_embedding_grad_run(ctypes.byref(d), FAKE, grad, dw, ws, ctypes.c_size_t(size), None)

    assert back(emb(grad_stride=8)) == 4 and b"rows of grad overlap" in lib.spmm_last_error()
    assert back(emb(), size=8) == 4 and b"workspace too small" in lib.spmm_last_error()
    assert back(emb(), ws=None) == 4 and back(emb(), grad=None) == 1 and back(emb(), dw=None) == 1
    assert back(emb(table=0), grad=None, dw=None, ws=None, size=0) == 0
    assert lib.spmm_embedding_run(None, FAKE, FAKE, FAKE, None) == 1


def test_embedding_workspaces(lib):
    size = ctypes.c_size_t(0)
    for count, table, width in ((0, 5, 4), (1, 1, 1), (33, 7, 5), (262144, 131072, 1024), (100, (1 << 30) - 1, 8),
                                (4097, 2048, 0)):
        assert lib.spmm_embedding_grad_workspace(ctypes.byref(emb(count, table, width)), ctypes.byref(size)) == 0
        # keys and positions twice, two rows of sums for each 32 positions, and the counts
        assert 16 * count <= size.value <= 24 * count + (count // 16 + 2) * (4 * width + 64) + (1 << 16) + 3 * count


def rt(rows=4, experts=64, stride=None, k=2, groups=1, top_groups=1, scale=1.0, score=0, renormalize=1, value=F16):
    return RouteDesc(rows, experts, experts if stride is None else stride, k, groups, top_groups, scale, score,
                     renormalize, value)


def test_route_refusals(lib):
    def run(d, x=FAKE, w=FAKE):
        return lib.spmm_route_run(ctypes.byref(d), x, None, w, FAKE, None, None)

    for d, code, text in ((rt(value=F64), 4, b"FP16, BF16 and FP32"), (rt(rows=-1), 4, b"negative extent"),
                          (rt(experts=0), 4, b"1 to 1024"), (rt(experts=1025), 4, b"1 to 1024"),
                          (rt(stride=63), 4, b"overlap"), (rt(k=0), 1, b"top_k"), (rt(k=65), 1, b"top_k"),
                          (rt(experts=3, k=4), 1, b"top_k"), (rt(groups=5), 1, b"groups"), (rt(groups=0), 1, b"groups"),
                          (rt(experts=1024, groups=128), 1, b"groups"), (rt(groups=8, top_groups=9), 1, b"top_groups"),
                          (rt(groups=8, top_groups=0), 1, b"top_groups"), (rt(groups=8, top_groups=1, k=9), 1, b"top_k"),
                          (rt(scale=0.0), 1, b"scale"), (rt(scale=float("nan")), 1, b"scale"),
                          (rt(scale=1e39), 1, b"scale"), (rt(scale=1e-39), 1, b"scale"), (rt(score=2), 1, b"score")):
        assert run(d) == code and text in lib.spmm_last_error(), lib.spmm_last_error()
    assert run(rt(), x=None) == 1 and run(rt(), w=None) == 1 and run(rt(rows=0), x=None) == 0

    def back(d, stats=None, grad=FAKE):
        return lib.spmm_route_grad_run(ctypes.byref(d), FAKE, FAKE, FAKE, stats, grad, FAKE, None)

    assert back(rt(renormalize=0)) == 1 and b"null device pointer" in lib.spmm_last_error()
    assert back(rt(), grad=None) == 1 and back(rt(rows=0), grad=None) == 0


def ex(rows=4, k=2, experts=8, width=16, stride=None, grad_stride=None, value=F16):
    return ExpertsDesc(rows, k, experts, width, width if stride is None else stride,
                       width if grad_stride is None else grad_stride, value)


def test_experts_refusals(lib):
    size = ctypes.c_size_t(0)
    for choices, experts, text in ((-1, 4, b"choices"), (1 << 31, 4, b"choices"), (4, 0, b"1 to 2048"),
                                   (4, 2049, b"1 to 2048")):
        assert lib.spmm_expert_plan_workspace(I64(choices), I64(experts), ctypes.byref(size)) == 4
        assert text in lib.spmm_last_error()
    for choices, experts in ((0, 1), (1, 2048), (100000, 64)):
        assert lib.spmm_expert_plan_workspace(I64(choices), I64(experts), ctypes.byref(size)) == 0
        assert size.value <= 4 * (choices // 256 + 3) * (experts + 1)

    def plan(index=0, ids=FAKE, choices=5000, ws=FAKE, size=1 << 20, offsets=FAKE):
        return lib.spmm_expert_plan_run(I32(index), ids, I64(choices), I64(8), offsets, FAKE, ws, ctypes.c_size_t(size),
                                        None)

    assert plan(index=2) == 4 and plan(ids=None) == 1 and plan(offsets=None) == 1
    assert plan(size=4) == 4 and b"workspace too small" in lib.spmm_last_error() and plan(ws=None) == 4

    def pack(d, x=FAKE):
        return lib.spmm_expert_pack_run(ctypes.byref(d), x, FAKE, FAKE, FAKE, None)

    for d, text in ((ex(value=F64), b"FP16, BF16 and FP32"), (ex(rows=-1), b"negative extent"), (ex(k=0), b"1 to 64"),
                    (ex(k=65), b"1 to 64"), (ex(experts=0), b"1 to 2048"), (ex(experts=2049), b"1 to 2048"),
                    (ex(rows=1 << 30), b"below 2^31"), (ex(width=1 << 22), b"below 2^22"), (ex(stride=15), b"overlap")):
        assert pack(d) == 4 and text in lib.spmm_last_error()
    assert pack(ex(), x=None) == 1 and pack(ex(rows=0), x=None) == 0 and pack(ex(width=0), x=None) == 0

    def back(d, y=FAKE, dw=FAKE):
        return lib.spmm_expert_restore_grad_run(ctypes.byref(d), y, FAKE, FAKE, FAKE, FAKE, FAKE, dw, None)

    assert back(ex(grad_stride=3)) == 4 and b"rows of grad overlap" in lib.spmm_last_error()
    assert back(ex(), y=None) == 1 and back(ex(rows=0), y=None) == 0
    assert lib.spmm_expert_restore_run(ctypes.byref(ex()), FAKE, None, FAKE, FAKE, FAKE, None) == 1
    assert lib.spmm_expert_pack_grad_run(ctypes.byref(ex()), FAKE, None, FAKE, FAKE, None) == 1


def lp(rows=4, classes=100, stride=None, top=0, index=1, value=F16):
    return LogProbsDesc(rows, classes, classes if stride is None else stride, top, index, value)


def test_log_probs_refusals(lib):
    def run(d, x=FAKE, top=FAKE, ws=FAKE, size=1 << 30):
        return lib.spmm_log_probs_run(ctypes.byref(d), x, FAKE, FAKE, FAKE, top, top, None, ws, ctypes.c_size_t(size),
                                      None)

    for d, code, text in ((lp(value=F64), 4, b"FP16, BF16 and FP32"), (lp(index=4), 4, b"int32 or int64"),
                          (lp(rows=-1), 4, b"rows"), (lp(rows=1 << 31), 4, b"rows"), (lp(classes=0), 4, b"classes"),
                          (lp(classes=1 << 31), 4, b"classes"), (lp(stride=99), 4, b"overlap"), (lp(top=-1), 1, b"top"),
                          (lp(top=65), 1, b"top"), (lp(classes=3, top=4), 1, b"top")):
        assert run(d) == code and text in lib.spmm_last_error()
    assert run(lp(), x=None) == 1 and run(lp(top=1), top=None) == 1 and run(lp(rows=0), x=None) == 0
    big = lp(rows=1, classes=131072, top=8)
    assert run(big, size=16) == 4 and b"workspace too small" in lib.spmm_last_error() and run(big, ws=None) == 4
    size = ctypes.c_size_t(0)
    for rows, classes, top in ((0, 7, 0), (1, 1, 1), (5, 4096, 64), (1, 1 << 20, 64), (4096, 131072, 4), (100, 40000, 0)):
        assert lib.spmm_log_probs_workspace(ctypes.byref(lp(rows, classes, top=top)), ctypes.byref(size)) == 0
        assert size.value <= 64 * max(rows, 1) * (12 + 8 * top) + 256

    def back(d, stats=FAKE):
        return lib.spmm_log_probs_grad_run(ctypes.byref(d), FAKE, FAKE, stats, FAKE, None, None, FAKE, None)

    assert back(lp(), stats=None) == 1 and back(lp(rows=0), stats=None) == 0 and back(lp(value=F64)) == 4


def test_surface():
    import spmm_npu

    for name in ("embedding", "route", "ExpertPlan", "log_probs"):
        assert callable(getattr(spmm_npu, name)) and name in spmm_npu.__all__
    for op in ("embedding", "route", "expert_plan", "expert_pack", "expert_restore", "log_probs"):
        assert hasattr(torch.ops.myops, op)
    x, ids = torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: spmm_npu.embedding(x, ids), lambda: spmm_npu.route(x, 2),
                 lambda: spmm_npu.ExpertPlan(ids, 2), lambda: spmm_npu.log_probs(x, ids)):
        with pytest.raises(RuntimeError, match="must be a GPU tensor"):
            call()
    with pytest.raises(ValueError, match="score must be one of"):
        spmm_npu.route(x, 2, score="tanh")


def differences(f, x, step=1e-6):
    """d f / d x by central differences."""
    out = torch.zeros_like(x)
    for i in range(x.numel()):
        hi, lo = x.clone(), x.clone()
        hi.view(-1)[i] += step
        lo.view(-1)[i] -= step
        out.view(-1)[i] = (f(hi) - f(lo)) / (2 * step)
    return out


def test_log_probs_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    x = 2 * torch.randn(4, 9, generator=g, dtype=torch.float64)
    targets = torch.tensor([0, 8, -1, 3])
    a, h = torch.randn(4, generator=g, dtype=torch.float64), torch.randn(4, generator=g, dtype=torch.float64)

    def f(v):
        out = plain.log_probs(v, targets, 0)
        return float((out["logp"] * a + out["entropy"] * h).sum())

    dx = plain.log_probs(x, targets, 0, a, h)["dx"]
    assert (dx - differences(f, x)).abs().max() < 1e-8  # step^2 and 2^-53 / step


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_against_differences(score, renormalize):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 7, generator=g, dtype=torch.float64)
    x[2, 1:] = -plain.INF  # one expert left for two choices
    chosen = plain.choose(x, 2, score, None, 1, 1)
    grad = torch.randn(3, 2, generator=g, dtype=torch.float64)

    def f(v):
        return float((plain.route(v, chosen, score, renormalize, 1.7)["w"] * grad).sum())

    dx = plain.route(x, chosen, score, renormalize, 1.7, grad)["dx"]
    steps = differences(f, x)
    steps[x == -plain.INF] = 0.0
    assert (dx - steps).abs().max() < 1e-8
