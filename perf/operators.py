"""The dense operators that a graph layer with typed nodes trains with, each as
one pass through its public entry points, beside its plain form.

* ``norm``: layer norm over the feature dimension (``layer_norm``), forward or
  a training step's forward and backward with the gradients of the input, the
  weight and the bias.
* ``grouped``: node features sorted by type, each type multiplied by its own
  weight matrix (``grouped_matmul``): ragged row groups, some of them empty.
  Forward, or forward and backward with the gradients of features and weights.
* ``orth``: a momentum-averaged update of one weight matrix, or of a stack of
  them, orthogonalised by five Newton-Schulz steps (``orthogonalize``).

``listed()`` holds twelve cases and ``draw(rng)`` makes more of the same
ranges.  A case is a plain dict of sizes and options.  Where ``own`` is false,
``run`` computes the plain form in 32 bits; where it is true, it calls the
framework.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS_NORM = 1e-5
EPS_ORTH = 1e-7
STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # One node answered online: a single row, where only latency counts.
        dict(name="norm_one_row_fp16", op="norm", train=False, rows=1, width=128, dtype="fp16"),
        # The headline matrix's node features (100000 x 128) in a training step.
        dict(name="norm_headline_train_fp16", op="norm", train=True, rows=100000, width=128, dtype="fp16"),
        # Wide features, the widest that the sparse operators take: pure bandwidth.
        dict(name="norm_wide_train_bf16", op="norm", train=True, rows=65536, width=1024, dtype="bf16"),
        # Rows and width that no vector load divides, in 32 bits.
        dict(name="norm_odd_train_fp32", op="norm", train=True, rows=16381, width=333, dtype="fp32"),
        # A handful of nodes of eight types answered online: the weights' bytes count.
        dict(name="grouped_few_rows_bf16", op="grouped", train=False, rows=13, groups=8, inner=512, width=512,
             dtype="bf16"),
        # The headline matrix's nodes in twelve types, 128 features in and out.
        dict(name="grouped_headline_train_fp16", op="grouped", train=True, rows=100000, groups=12, inner=128,
             width=128, dtype="fp16"),
        # A wide typed layer's training step: three large ragged products.
        dict(name="grouped_large_train_bf16", op="grouped", train=True, rows=65536, groups=8, inner=1024, width=2048,
             dtype="bf16"),
        # Raw input features of odd widths in 32 bits.
        dict(name="grouped_odd_train_fp32", op="grouped", train=True, rows=16381, groups=5, inner=333, width=190,
             dtype="fp32"),
        # The update of one small layer in 32 bits: launches count.
        dict(name="orth_small_fp32", op="orth", batch=1, rows=128, width=96, dtype="fp32"),
        # The updates of a typed layer's weights, one matrix for each of twelve types.
        dict(name="orth_types_bf16", op="orth", batch=12, rows=512, width=1024, dtype="bf16"),
        # A tall matrix: more rows than columns, in half precision.
        dict(name="orth_tall_fp16", op="orth", batch=1, rows=2048, width=512, dtype="fp16"),
        # The largest square weight that a user of such an optimiser holds.
        dict(name="orth_large_bf16", op="orth", batch=1, rows=4096, width=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range: as it falls, or rounded to
    a multiple of 16, as most layers' widths are."""
    n = _log_int(rng, lo, hi)
    if rng.random() < 0.5 and n >= 16:
        n = n // 16 * 16
    return n + 1 if n == 3072 else n


# Most elements of a drawn norm, and most products of the other two.
_MOST_ELEMENTS = 65536 * 1024
_MOST_GROUPED = 65536 * 1024 * 2048
_MOST_ORTH = 5 * 4 * 4096 ** 3


def draw(rng):
    op = rng.choice(["norm", "grouped", "orth"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    if op == "norm":
        while True:
            rows, width = _size(rng, 1, 262144), _size(rng, 8, 8192)
            if rows * width * BYTES[dtype] <= 2 * _MOST_ELEMENTS:
                return dict(op=op, train=rng.random() < 0.7, rows=rows, width=width, dtype=dtype)
    if op == "grouped":
        while True:
            rows, inner, width = _size(rng, 1, 131072), _size(rng, 16, 2048), _size(rng, 16, 2048)
            # 32-bit products run at a small part of the rate
            if rows * inner * width * (8 if dtype == "fp32" else 1) <= _MOST_GROUPED:
                return dict(op=op, train=rng.random() < 0.7, rows=rows, groups=rng.randint(1, 24), inner=inner,
                            width=width, dtype=dtype)
    while True:
        # In 32 bits up to 768: the plain form's own sums stay well inside that type's precision.
        most = 768 if dtype == "fp32" else 4096
        case = dict(op=op, batch=rng.choice([1, 1, 1, rng.randint(2, 16)]), rows=_size(rng, 16, most),
                    width=_size(rng, 16, most), dtype=dtype)
        if _orth_products(case) <= _MOST_ORTH:
            return case


def _orth_products(case):
    m, n = sorted((case["rows"], case["width"]))
    return case["batch"] * STEPS * (m * m * n + m ** 3 + 2 * m * m * n)


def _group_sizes(case, seed):
    """Ragged group sizes that add up to the rows: heavy-tailed shares, and with
    more than three groups one that is empty."""
    rng = random.Random(seed * 7919 + 17)
    share = [rng.lognormvariate(0.0, 0.6) for _ in range(case["groups"])]
    if case["groups"] > 3:
        share[rng.randrange(case["groups"])] = 0.0
    total, edges, done = sum(share), [0], 0.0
    for s in share:
        done += s
        edges.append(round(case["rows"] * done / total))
    edges[-1] = case["rows"]
    return [b - a for a, b in zip(edges, edges[1:])], edges


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = DTYPE[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    state = {"case": dict(case)}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # Activations: features of different scale and offset, rows of different scale.
        x = normal(rows, width)
        x.mul_(torch.exp(0.5 * normal(1, width))).add_(0.3 * normal(1, width)).mul_(torch.exp(0.3 * normal(rows, 1)))
        state["x"] = x.to(dtype)
        state["weight"] = (1.0 + 0.1 * normal(width)).to(dtype)
        state["bias"] = (0.1 * normal(width)).to(dtype)
        leaves = ("x", "weight", "bias")
        if case["train"]:
            state["grad"] = normal(rows, width).mul_(0.1).to(dtype)
    elif case["op"] == "grouped":
        sizes, edges = _group_sizes(case, int(seed))
        rows, inner, width = case["rows"], case["inner"], case["width"]
        state["sizes"] = sizes
        state["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
        state["x"] = normal(rows, inner).to(dtype)
        state["weight"] = normal(case["groups"], inner, width).div_(math.sqrt(inner)).to(dtype)
        leaves = ("x", "weight")
        if case["train"]:
            state["grad"] = normal(rows, width).mul_(0.1).to(dtype)
    else:
        batch, rows, width = case["batch"], case["rows"], case["width"]
        # A gradient: a few strong directions over noise.
        k = max(1, min(rows, width) // 8)
        u = normal(batch, rows, width)
        u.add_(torch.bmm(normal(batch, rows, k), normal(batch, k, width)).mul_(1.0 / math.sqrt(k)))
        u.mul_(1e-2)
        state["update"] = (u if batch > 1 else u[0]).to(dtype)
        leaves = ()
    if case.get("train"):
        for name in leaves:
            state[name].requires_grad_(True)
    return state


def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-spmm_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import spmm_npu

    return spmm_npu


def _run_own(state):
    f, case = _framework(), state["case"]
    if case["op"] == "norm":
        y = f.layer_norm(state["x"], state["weight"], state["bias"], EPS_NORM)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["grad"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "grouped":
        y = f.grouped_matmul(state["x"], state["weight"], state["offsets"])
        if not case["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (state["x"], state["weight"]), state["grad"])
        return {"y": y.detach(), "dx": dx, "dweight": dw}
    return {"update": f.orthogonalize(state["update"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS_ORTH)}


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS_NORM)
    unit = centred * rstd
    y = (unit * w + b).to(dtype)
    if not case["train"]:
        return {"y": y}
    dy = state["grad"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dweight": (dy * unit).sum(0).to(dtype), "dbias": dy.sum(0).to(dtype)}


def _plain_grouped(state):
    case, dtype, sizes = state["case"], state["x"].dtype, state["sizes"]
    x, w = state["x"].float().split(sizes), state["weight"].float()
    y = torch.cat([a @ b for a, b in zip(x, w)]).to(dtype)
    if not case["train"]:
        return {"y": y}
    dy = state["grad"].float().split(sizes)
    dx = torch.cat([d @ b.t() for d, b in zip(dy, w)]).to(dtype)
    dw = torch.stack([a.t() @ d for a, d in zip(x, dy)]).to(dtype)
    return {"y": y, "dx": dx, "dweight": dw}


def _plain_orth(state):
    u = state["update"]
    x = u.float()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS_ORTH)
    tall = x.size(-2) > x.size(-1)
    x = x.transpose(-2, -1).contiguous() if tall else x
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return {"update": (x.transpose(-2, -1).contiguous() if tall else x).to(u.dtype)}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "grouped": _plain_grouped, "orth": _plain_orth}[state["case"]["op"]](state)


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "norm":
        elements = case["rows"] * case["width"]
        # x in, y out; with a backward pass also the incoming gradient and dx.
        passes, vectors, flops = (4, 4, 20) if case["train"] else (2, 2, 8)
        return {"bytes": b * (passes * elements + vectors * case["width"]), "flops": flops * elements}
    if case["op"] == "grouped":
        rows, inner, width = case["rows"], case["inner"], case["width"]
        active = case["groups"] - (1 if case["groups"] > 3 else 0)
        # Only the weights of groups with rows are needed.
        matrix = rows * inner + min(active, rows) * inner * width + rows * width
        flops = 2 * rows * inner * width
        return {"bytes": b * matrix * (2 if case["train"] else 1), "flops": flops * (3 if case["train"] else 1)}
    # The Gram matrix and its square are symmetric: half of their products are enough.
    return {"bytes": 2 * b * case["batch"] * case["rows"] * case["width"], "flops": _orth_products(case)}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            x, w, b = (state[k].detach().double() for k in ("x", "weight", "bias"))
            n = case["width"]
            mean = x.sum(1) / n
            var = ((x - mean[:, None]) ** 2).sum(1) / n
            inv = 1.0 / (var + EPS_NORM) ** 0.5
            z = (x - mean[:, None]) * inv[:, None]
            y = z * w + b
            if not case["train"]:
                return {"y": y}
            dy = state["grad"].double()
            dz = dy * w
            # d var and d mean of the definition, then the chain rule.
            dvar = -0.5 * (dz * (x - mean[:, None])).sum(1) * inv ** 3
            dmean = -(dz.sum(1) * inv)
            dx = dz * inv[:, None] + (2.0 / n) * dvar[:, None] * (x - mean[:, None]) + dmean[:, None] / n
            return {"y": y, "dx": dx, "dweight": torch.einsum("rn,rn->n", dy, z), "dbias": dy.sum(0)}
        if case["op"] == "grouped":
            x, w = state["x"].detach().double(), state["weight"].detach().double()
            y = x.new_zeros(case["rows"], case["width"])
            dx, dw = torch.zeros_like(x), torch.zeros_like(w)
            dy = state["grad"].double() if case["train"] else None
            start = 0
            for i, size in enumerate(state["sizes"]):
                part = slice(start, start + size)
                start += size
                if size:
                    y[part] = x[part] @ w[i]
                    if case["train"]:
                        dx[part] = dy[part] @ w[i].t()
                        dw[i] = x[part].t() @ dy[part]
            return {"y": y, "dx": dx, "dweight": dw} if case["train"] else {"y": y}
        a, b, c = COEFFICIENTS
        u = state["update"].double()
        stack = u if u.dim() == 3 else u[None]
        out = []
        for m in stack:
            m = m / (torch.linalg.norm(m) + EPS_ORTH)
            left = m.shape[0] <= m.shape[1]
            for _ in range(STEPS):
                if left:
                    s = m @ m.t()
                    m = a * m + b * (s @ m) + c * (s @ (s @ m))
                else:
                    s = m.t() @ m
                    m = a * m + b * (m @ s) + c * ((m @ s) @ s)
            out.append(m)
        out = torch.stack(out)
        return {"update": out if u.dim() == 3 else out[0]}
