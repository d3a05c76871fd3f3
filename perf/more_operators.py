"""The operators around a layer of experts on a graph's nodes, each as one pass
through its public entry points, beside its plain form.

* ``embedding``: features of nodes that have none of their own, rows of a
  learned table (``embedding``).  Forward, or with the table's gradient.
* ``route``: the experts of each node and their weights, from a router's
  logits (``route``).  Forward, or with the logits' gradient.
* ``experts``: each node's row brought to its experts, whose row ranges
  ``grouped_matmul`` takes, and the experts' results brought back, weighted
  (``ExpertPlan``, its ``pack`` and ``restore``).  What the experts make of
  the rows is an input here.  Forward, or with all gradients.
* ``log_probs``: log probabilities of the nodes' labels, the entropy and the
  best classes (``log_probs``).  Forward, or with the logits' gradient.

``listed()`` holds twelve cases and ``draw(rng)`` makes more of the same
ranges.  A case is a plain dict of sizes and options.  Where ``own`` is false,
``run`` computes the plain form; where it is true, it calls the framework.
"""

import math
import os
import sys

import torch

own = False

DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
INF = float("inf")


def listed():
    return [
        # A handful of nodes answered online, from the headline matrix's 100000 nodes: latency.
        dict(name="embedding_few_fp16", op="embedding", train=False, count=13, table=100000, width=128, ids="popular",
             dtype="fp16"),
        # The headline matrix's nodes, each with a row of its own, in a full-graph training step.
        dict(name="embedding_each_train_fp32", op="embedding", train=True, count=100000, table=100000, width=128,
             ids="each", dtype="fp32"),
        # Sampled neighbourhoods of a power-law graph: popular nodes many times, most not at all.
        dict(name="embedding_popular_train_bf16", op="embedding", train=True, count=262144, table=131072, width=1024,
             ids="popular", dtype="bf16"),
        # One node answered online: a single row of logits.
        dict(name="route_one_row_bf16", op="route", train=False, rows=1, experts=64, k=4, score="softmax", bias=False,
             groups=1, top_groups=1, renormalize=True, masked=False, dtype="bf16"),
        # The headline matrix's nodes over a few experts, the weights as probabilities, in training.
        dict(name="route_headline_train_fp16", op="route", train=True, rows=100000, experts=12, k=2, score="softmax",
             bias=False, groups=1, top_groups=1, renormalize=False, masked=False, dtype="fp16"),
        # Many experts in groups, balanced by a bias, logits in 32 bits, in training.
        dict(name="route_groups_train_fp32", op="route", train=True, rows=65536, experts=256, k=8, score="sigmoid",
             bias=True, groups=8, top_groups=4, renormalize=True, masked=False, dtype="fp32"),
        # A handful of nodes answered online: launches count.
        dict(name="experts_few_bf16", op="experts", train=False, rows=13, experts=8, k=2, width=512, dropped=False,
             dtype="bf16"),
        # Raw input features of an odd width in 32 bits, some choices dropped for want of room.
        dict(name="experts_odd_train_fp32", op="experts", train=True, rows=16381, experts=5, k=3, width=333,
             dropped=True, dtype="fp32"),
        # A wide layer of many experts in training: pure bandwidth.
        dict(name="experts_wide_train_bf16", op="experts", train=True, rows=32768, experts=64, k=8, width=1024,
             dropped=False, dtype="bf16"),
        # The likeliest items of a large catalogue for one node: a single long row.
        dict(name="log_probs_one_row_bf16", op="log_probs", train=False, rows=1, classes=131072, top=8, masked=False,
             dtype="bf16"),
        # The headline matrix's nodes in an odd number of classes, labels for a part of them.
        dict(name="log_probs_classes_train_fp32", op="log_probs", train=True, rows=100000, classes=47, top=1,
             masked=True, dtype="fp32"),
        # A batch of nodes against a large catalogue in training: the largest.
        dict(name="log_probs_catalogue_train_bf16", op="log_probs", train=True, rows=4096, classes=131072, top=4,
             masked=False, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range: as it falls, or rounded to
    a multiple of 16, as most layers' widths are."""
    n = _log_int(rng, lo, hi)
    return n // 16 * 16 if rng.random() < 0.5 and n >= 16 else n


# Most elements of a drawn embedding's gradient with its table, of a drawn router's logits, of drawn packed rows and of
# drawn logits, in elements of 16 bits.
_MOST_EMBEDDING = (262144 + 131072) * 1024
_MOST_ROUTE = 2 * 65536 * 256
_MOST_EXPERTS = 262144 * 1024
_MOST_LOGITS = 4096 * 131072


def draw(rng):
    op = rng.choice(["embedding", "route", "experts", "log_probs"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    train, wide = rng.random() < 0.7, 2 if dtype == "fp32" else 1
    while True:
        if op == "embedding":
            count, table, width = _size(rng, 1, 524288), _size(rng, 1, 524288), _size(rng, 8, 2048)
            if (count + table) * width * wide <= _MOST_EMBEDDING:
                return dict(op=op, train=train, count=count, table=table, width=width,
                            ids=rng.choice(["popular", "popular", "uniform", "absent"]), dtype=dtype)
        elif op == "route":
            rows, groups = _size(rng, 1, 131072), rng.choice([1, 1, 2, 4, 8])
            experts = groups * max(1, _size(rng, 2, 512) // groups)
            top_groups = rng.randint(1, groups)
            k = min(rng.randint(1, 16), experts // groups * top_groups)
            if rows * experts * wide <= _MOST_ROUTE:
                return dict(op=op, train=train, rows=rows, experts=experts, k=k,
                            score=rng.choice(["softmax", "sigmoid"]), bias=groups > 1 or rng.random() < 0.3,
                            groups=groups, top_groups=top_groups, renormalize=rng.random() < 0.5,
                            masked=rng.random() < 0.3, dtype=dtype)
        elif op == "experts":
            rows, k, width = _size(rng, 1, 131072), rng.randint(1, 8), _size(rng, 8, 2048)
            experts = max(k, _size(rng, 1, 256))
            if rows * k * width * wide <= _MOST_EXPERTS:
                return dict(op=op, train=train, rows=rows, experts=experts, k=k, width=width,
                            dropped=rng.random() < 0.4, dtype=dtype)
        else:
            rows, classes = _size(rng, 1, 131072), _size(rng, 2, 262144)
            if rows * classes * wide <= _MOST_LOGITS:
                return dict(op=op, train=train, rows=rows, classes=classes,
                            top=min(classes, rng.choice([0, 0, 1, 5, 16])), masked=rng.random() < 0.4, dtype=dtype)


def _wants(state, *names):
    if state["case"]["train"]:
        for name in names:
            state[name].requires_grad_(True)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = DTYPE[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    state = {"case": dict(case)}
    if case["op"] == "embedding":
        count, table, width = case["count"], case["table"], case["width"]
        shuffled = torch.randperm(table, generator=g, device="cuda")
        if case["ids"] == "each":
            ids = shuffled[torch.arange(count, device="cuda") % table]
        elif case["ids"] == "popular":
            # The r-th most popular row about in proportion to 1 / r.
            rank = (torch.exp(uniform(count).double() * math.log(table + 1)) - 1).long().clamp(0, table - 1)
            ids = shuffled[rank]
        else:
            ids = torch.randint(0, table, (count,), generator=g, device="cuda")
        if case["ids"] == "absent":
            # Places of a padded batch that hold no node.
            ids = torch.where(uniform(count) < 0.2, torch.full_like(ids, -1), ids)
        state["ids"] = ids
        state["scale"] = math.sqrt(width)
        state["weight"] = normal(table, width).mul_(0.02).to(dtype)
        _wants(state, "weight")
        if case["train"]:
            state["grad"] = normal(count, width).mul_(0.1).to(dtype)
    elif case["op"] == "route":
        rows, experts = case["rows"], case["experts"]
        # Some experts are favoured by all rows.
        logits = normal(rows, experts).add_(0.5 * normal(1, experts))
        if case["masked"]:
            logits.masked_fill_(uniform(rows, experts) < 0.1, -INF)
        state["logits"] = logits.to(dtype)
        state["bias"] = 0.1 * normal(experts) if case["bias"] else None
        _wants(state, "logits")
        if case["train"]:
            state["grad"] = normal(rows, case["k"])
    elif case["op"] == "experts":
        rows, experts, k, width = case["rows"], case["experts"], case["k"], case["width"]
        # k different experts a row, some of them favoured by all.
        chosen = (uniform(rows, experts) + 0.3 * uniform(1, experts)).topk(k, dim=1).indices.to(torch.int32)
        if case["dropped"]:
            chosen = torch.where(uniform(rows, k) < 0.1, torch.full_like(chosen, -1), chosen)
        state["experts"] = chosen
        state["weights"] = torch.softmax(normal(rows, k), 1)
        state["x"] = normal(rows, width).to(dtype)
        state["results"] = normal(rows * k, width).to(dtype)
        _wants(state, "weights", "x", "results")
        if case["train"]:
            state["grad"] = normal(rows, width).mul_(0.1).to(dtype)
    else:
        rows, classes = case["rows"], case["classes"]
        logits = normal(rows, classes).mul_(2.0)
        targets = torch.randint(0, classes, (rows,), generator=g, device="cuda")
        # The label is likelier than the rest, as it is after some training.
        logits.scatter_add_(1, targets[:, None], 4.0 * uniform(rows, 1))
        if case["masked"]:
            # Classes that a row cannot have, and rows without a label.
            hidden = uniform(rows, classes) < 0.1
            hidden.scatter_(1, targets[:, None], False)
            logits.masked_fill_(hidden, -INF)
            targets = torch.where(uniform(rows) < 0.3, torch.full_like(targets, -100), targets)
        state["logits"] = logits.to(dtype)
        state["targets"] = targets
        _wants(state, "logits")
        if case["train"]:
            # The mean of the negative log probabilities, and a little of the entropy.
            state["grad"] = torch.full((rows,), -1.0, device="cuda") * (0.5 + uniform(rows))
            state["grad_entropy"] = -0.1 * uniform(rows)
    return state


def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-spmm_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import spmm_npu

    return spmm_npu


def _run_own(state):
    f, case = _framework(), state["case"]
    if case["op"] == "embedding":
        out = f.embedding(state["weight"], state["ids"], scale=state["scale"])
        if not case["train"]:
            return {"out": out}
        (dweight,) = torch.autograd.grad(out, (state["weight"],), state["grad"])
        return {"out": out.detach(), "dweight": dweight}
    if case["op"] == "route":
        weights, experts = f.route(state["logits"], case["k"], score=case["score"], bias=state["bias"],
                                   groups=case["groups"], top_groups=case["top_groups"],
                                   renormalize=case["renormalize"])
        if not case["train"]:
            return {"weights": weights, "experts": experts}
        (dlogits,) = torch.autograd.grad(weights, (state["logits"],), state["grad"])
        return {"weights": weights.detach(), "experts": experts, "dlogits": dlogits}
    if case["op"] == "experts":
        plan = f.ExpertPlan(state["experts"], case["experts"])
        packed = plan.pack(state["x"])
        out = plan.restore(state["results"], state["weights"])
        got = {"offsets": plan.offsets, "place": plan.place, "packed": packed.detach(), "out": out.detach()}
        if case["train"]:
            dresults, dweights = torch.autograd.grad(out, (state["results"], state["weights"]), state["grad"])
            (dx,) = torch.autograd.grad(packed, (state["x"],), dresults)
            got.update(dresults=dresults, dweights=dweights, dx=dx)
        return got
    logp, entropy, top, top_ids = f.log_probs(state["logits"], state["targets"], top=case["top"])
    got = {"logp": logp.detach(), "entropy": entropy.detach(), "top": top, "top_ids": top_ids}
    if case["train"]:
        (got["dlogits"],) = torch.autograd.grad((logp, entropy), (state["logits"],),
                                                (state["grad"], state["grad_entropy"]))
    return got


def _plain_embedding(state):
    case, weight, ids = state["case"], state["weight"], state["ids"]
    present = ((ids >= 0) & (ids < case["table"]))[:, None]
    at = ids.clamp(0, case["table"] - 1)
    got = {"out": (weight[at].float() * present * state["scale"]).to(weight.dtype)}
    if case["train"]:
        total = torch.zeros(weight.shape, device=weight.device)
        total.index_add_(0, at, state["grad"].float() * present)
        got["dweight"] = (total * state["scale"]).to(weight.dtype)
    return got


def _plain_route(state):
    case, logits, bias = state["case"], state["logits"], state["bias"]
    rows, experts, k, groups = case["rows"], case["experts"], case["k"], case["groups"]
    x = logits.float()
    closed = x == -INF
    if bias is None and groups == 1:
        value = x
    else:
        # Next to a border between two experts, 32 bits would decide by their rounding.
        wide = logits.double()
        if case["score"] == "softmax":
            value = torch.exp(wide - wide.amax(1, keepdim=True))
            value = value / value.sum(1, keepdim=True)
        else:
            value = 1.0 / (1.0 + torch.exp(-wide))
        if bias is not None:
            value = value + bias.double()
    value = value.masked_fill(closed, -INF)
    if groups > 1:
        best = value.view(rows, groups, -1).sort(2, descending=True).values[:, :, :2]
        second = best[:, :, 1:].sum(2)
        best = best[:, :, 0] + torch.where(second == -INF, torch.zeros_like(second), second)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_groups = torch.zeros(rows, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        value = value.masked_fill(~open_groups.repeat_interleave(experts // groups, 1), -INF)
    value, chosen = value.sort(dim=1, descending=True, stable=True)
    found, chosen = value[:, :k] != -INF, chosen[:, :k]

    if case["score"] == "softmax":
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - top)
        total = p.sum(1, keepdim=True)
        log_score, p = x - top - torch.log(total), torch.where(closed, torch.zeros_like(x), p / total)
    else:
        log_score = x.clamp_max(0.0) - torch.log1p(torch.exp(-x.abs()))
    mine = log_score.gather(1, chosen).masked_fill(~found, -INF)
    if case["renormalize"]:
        mine = torch.exp(mine - mine.amax(1, keepdim=True))
        weights = mine / mine.sum(1, keepdim=True)
    else:
        weights = torch.exp(mine)
    weights = torch.where(found, weights, torch.zeros_like(weights))
    got = {"weights": weights, "experts": torch.where(found, chosen, torch.full_like(chosen, -1)).to(torch.int32)}
    if case["train"]:
        grad = torch.where(found, state["grad"], torch.zeros_like(weights))
        dlog = weights * grad
        if case["renormalize"]:
            dlog = dlog - weights * dlog.sum(1, keepdim=True)
        if case["score"] == "sigmoid":
            at = x.gather(1, chosen)
            dlog = torch.where(found, dlog / (1.0 + torch.exp(at)), torch.zeros_like(dlog))
        dlogits = torch.zeros_like(x).scatter_add_(1, chosen, dlog)
        if case["score"] == "softmax" and not case["renormalize"]:
            dlogits -= p * dlog.sum(1, keepdim=True)
        got["dlogits"] = dlogits.to(logits.dtype)
    return got


def _plain_experts(state):
    case, experts, x, results, weights = (state[n] for n in ("case", "experts", "x", "results", "weights"))
    rows, k, count, width = case["rows"], case["k"], case["experts"], case["width"]
    key = experts.reshape(-1).long()
    key = torch.where((key >= 0) & (key < count), key, torch.full_like(key, count))
    by_expert = key.argsort(stable=True)
    place = torch.empty_like(by_expert).scatter_(0, by_expert, torch.arange(rows * k, device=x.device))
    sizes = torch.zeros(count + 1, dtype=torch.int64, device=x.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([sizes.new_zeros(1), sizes[:count].cumsum(0)])
    kept = (key < count).view(rows, k, 1)
    packed = x[by_expert // k].float() * (key[by_expert] < count)[:, None]
    brought = results[place].float().view(rows, k, width) * kept
    out = (brought * weights[:, :, None]).sum(1)
    got = {"offsets": offsets.to(torch.int32), "place": place.view(rows, k).to(torch.int32),
           "packed": packed.to(x.dtype), "out": out.to(x.dtype)}
    if case["train"]:
        grad = state["grad"].float()[:, None, :]
        sent = (weights[:, :, None] * grad * kept).to(x.dtype).view(rows * k, width)
        got["dresults"] = sent[by_expert]
        got["dweights"] = (brought * grad).sum(2)
        got["dx"] = sent.float().view(rows, k, width).sum(1).to(x.dtype)
    return got


def _plain_log_probs(state):
    case, logits, targets = state["case"], state["logits"], state["targets"]
    classes, top = case["classes"], case["top"]
    x = logits.float()
    labelled = (targets >= 0) & (targets < classes)
    at = targets.clamp(0, classes - 1)[:, None]
    z = x - x.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    p = e / total
    spread = torch.where(e > 0, p * z, torch.zeros_like(z)).sum(1, keepdim=True)
    entropy = lse - spread
    logp = torch.where(labelled, (z.gather(1, at) - lse)[:, 0], torch.zeros_like(lse[:, 0]))
    got = {"logp": logp, "entropy": entropy[:, 0]}
    if top:
        # One whole number a class, by value and then the lowest index first, so that ties are decided.
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (bits << 32) + torch.arange(classes - 1, -1, -1, device=x.device)
        ids = classes - 1 - (key.topk(top, dim=1).values & 0xFFFFFFFF)
        best = z.gather(1, ids) - lse
        got["top"], got["top_ids"] = best, torch.where(best == -INF, torch.full_like(ids, -1), ids).to(torch.int32)
    else:
        got["top"], got["top_ids"] = x.new_zeros(case["rows"], 0), at.new_zeros(case["rows"], 0).to(torch.int32)
    if case["train"]:
        a = torch.where(labelled, state["grad"], torch.zeros_like(logp))[:, None]
        dlogits = -p * a - torch.where(e > 0, state["grad_entropy"][:, None] * p * (z - lse + entropy),
                                       torch.zeros_like(z))
        got["dlogits"] = dlogits.scatter_add_(1, at, a).to(logits.dtype)
    return got


def run(state):
    if own:
        return _run_own(state)
    plain = {"embedding": _plain_embedding, "route": _plain_route, "experts": _plain_experts,
             "log_probs": _plain_log_probs}
    with torch.no_grad():
        return plain[state["case"]["op"]](state)


def _distinct_rows(case):
    """About how many rows of the table the ids name."""
    count, table = case["count"], case["table"]
    if case["ids"] == "each":
        return min(count, table)
    if case["ids"] == "popular":
        # Over ranks r with probability log((r + 1) / r) / log(table + 1): those expected once, and a part of the rest.
        share = count / math.log(table + 1)
        return min(table, count, share * (1.0 + max(0.0, math.log(max(table / share, 1.0)))))
    return table * (1.0 - math.exp(-count / table))


def work(case):
    b, train = BYTES[case["dtype"]], case["train"]
    if case["op"] == "embedding":
        count, table, width = case["count"], case["table"], case["width"]
        read = 8 * count + b * width * _distinct_rows(case)
        return {"bytes": read + b * width * (count + (count + table if train else 0)), "flops": 2 * count * width}
    if case["op"] == "route":
        logits, chosen = case["rows"] * case["experts"], case["rows"] * case["k"]
        return {"bytes": b * logits * (2 if train else 1) + chosen * (12 if train else 8),
                "flops": logits * (12 if train else 6)}
    if case["op"] == "experts":
        rows, width, chosen = case["rows"], case["width"], case["rows"] * case["k"]
        # x, out and the choices' rows packed and brought back; grad, dx and the results' gradient.
        elements = width * (2 * rows + 2 * chosen + (2 * rows + chosen if train else 0))
        return {"bytes": b * elements + chosen * (16 if train else 12), "flops": 2 * chosen * width * (3 if train else 1)}
    logits = case["rows"] * case["classes"]
    return {"bytes": b * logits * (2 if train else 1) + case["rows"] * (24 + 8 * case["top"]),
            "flops": logits * (12 if train else 6)}


def _exact_route(state, case):
    """The choice by sorting each row's (value, index) pairs, the weights and
    their gradient by differentiating the definition."""
    x = state["logits"].detach().double().requires_grad_(case["train"])
    rows, experts, k, groups = case["rows"], case["experts"], case["k"], case["groups"]
    log_score = torch.log_softmax(x, 1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(x)
    with torch.no_grad():
        plain = state["bias"] is None and groups == 1
        value = x.detach().clone() if plain else log_score.detach().exp()
        if state["bias"] is not None:
            value += state["bias"].double()
        value[torch.isneginf(x)] = -INF
        if groups > 1:
            parts = value.reshape(rows, groups, experts // groups)
            first, where = parts.max(2)
            others = parts.scatter(2, where[..., None], -INF)
            second = others.amax(2)
            first = first + torch.where(torch.isneginf(second), torch.zeros_like(second), second)
            kept = torch.argsort(-first, dim=1, stable=True)[:, :case["top_groups"]]
            shut = torch.ones(rows, groups, dtype=torch.bool, device=x.device)
            shut[torch.arange(rows, device=x.device)[:, None], kept] = False
            parts.masked_fill_(shut[..., None], -INF)
            value = parts.reshape(rows, experts)
        chosen = torch.argsort(-value, dim=1, stable=True)[:, :k]
        found = ~torch.isneginf(value.gather(1, chosen))
    # Choices that there are not, by a finite stand-in, so that their gradient is zero and not undefined.
    mine = torch.where(found, log_score.gather(1, chosen), torch.full_like(found, -1e300, dtype=torch.float64))
    weights = torch.softmax(mine, 1) if case["renormalize"] else mine.exp()
    weights = weights * found
    got = {"weights": weights.detach(), "experts": None}
    if case["train"]:
        (dx,) = torch.autograd.grad(weights, (x,), state["grad"].double())
        # log_softmax has no derivative where the logit is minus infinity; the definition gives zero there.
        got["dlogits"] = torch.where(torch.isneginf(x.detach()), torch.zeros_like(dx), dx)
    return got


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(state, case)
    with torch.no_grad():
        if case["op"] == "embedding":
            ids, scale = state["ids"], state["scale"]
            rows = torch.cat([state["weight"].detach().double(), state["weight"].new_zeros(1, case["width"]).double()])
            ids = torch.where(ids < 0, torch.full_like(ids, case["table"]), ids)
            got = {"out": rows.index_select(0, ids) * scale}
            if case["train"]:
                # Sums of sorted rows as differences of running sums' ends would lose digits: added by index instead.
                rows.zero_()
                rows.index_put_((ids,), state["grad"].double(), accumulate=True)
                got["dweight"] = rows[:case["table"]] * scale
            return got
        if case["op"] == "experts":
            rows, k = case["rows"], case["k"]
            experts = state["experts"].long()
            dropped = (experts < 0).reshape(-1)
            flat = torch.where(dropped, case["experts"], experts.reshape(-1))
            # The place of a choice: those of lower experts, and those before it of its own.
            order = torch.sort(flat * (rows * k) + torch.arange(rows * k, device=flat.device)).indices
            place = torch.argsort(order)
            scattered = state["x"].detach().double().repeat_interleave(k, 0)
            scattered[dropped] = 0.0
            got = {"offsets": None, "place": None, "packed": scattered[order]}
            w = state["weights"].detach().double().reshape(-1, 1).clone()
            w[dropped] = 0.0
            y = state["results"].detach().double()[place]
            got["out"] = torch.zeros(rows, case["width"], dtype=torch.float64, device=y.device)
            owner = torch.arange(rows, device=y.device).repeat_interleave(k)
            got["out"].index_add_(0, owner, w * y)
            if case["train"]:
                g = state["grad"].double()[owner]
                got["dresults"] = (w * g)[order]
                got["dweights"] = ((y * g).sum(1) * ~dropped).view(rows, k)
                got["dx"] = state["grad"].double() * w.view(rows, k).sum(1, keepdim=True)
            return got
        x, targets = state["logits"].detach().double(), state["targets"]
        log_all = x - torch.logsumexp(x, 1, keepdim=True)
        p = torch.exp(log_all)
        info = torch.nan_to_num(log_all, neginf=0.0)
        entropy = -(p * info).sum(1)
        named = targets >= 0
        logp = torch.where(named, log_all[torch.arange(len(targets), device=x.device), targets.clamp_min(0)], 0.0)
        got = {"logp": logp, "entropy": entropy, "top": log_all.topk(case["top"], dim=1).values, "top_ids": None}
        if case["train"]:
            a, h = state["grad"].double() * named, state["grad_entropy"].double()
            dx = -(a[:, None] + h[:, None] * (info + entropy[:, None])) * p
            dx[torch.arange(len(targets), device=x.device), targets.clamp_min(0)] += a
            got["dlogits"] = dx
        return got
