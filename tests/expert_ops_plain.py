"""Plain 64-bit forms of the operators around a layer of experts, and the
rounding of their types, for the tests of embedding, route, ExpertPlan and
log_probs."""

import math

import numpy as np
import torch

E32 = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# Half the distance of the smallest values: what a result near zero rounds by.
# (fp32: results below 2^-126 may become zero.)
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
INF = float("inf")


def check(got, want, bound, what):
    """|got - want| within the rounding of got's type, and `bound` before it.
    Infinities and NaN have to be where the plain form has them."""
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    got, want, dtype = got.detach().double().cpu(), want.double().cpu(), got.dtype
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    special = ~finite & ~torch.isnan(want)
    assert torch.equal(got[special], want[special]), f"{what}: infinities differ"
    bound = torch.as_tensor(bound, dtype=torch.float64).expand(want.shape)
    limit = U[dtype] * want.abs() + bound * (1 + U[dtype]) + TINY[dtype]
    bad = finite & ~((got - want).abs() <= limit)
    if bad.any():
        ratio = ((got - want).abs() / limit)[finite].max()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(ratio):.3g} x the bound")


def normal(shape, dtype, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(dtype)


# ------------------------------------------------------------- log_probs


def log_probs(x, targets, top, a=None, h=None):
    """logp, entropy, top values, top ids and (with incoming gradients a and h)
    dx, of 2D logits in 64 bits; and the parts the bounds are made of."""
    x, targets = x.double().cpu(), targets.cpu().long()
    rows, n = x.shape
    named = (targets >= 0) & (targets < n)
    at = targets.clamp(0, n - 1)
    m = x.amax(1, keepdim=True)
    empty = (m == -INF)[:, 0]
    m = torch.where(m == -INF, torch.zeros_like(m), m)
    z = x - m
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    ls = torch.log(s)
    p = torch.where(empty[:, None], torch.zeros_like(e), e / s)
    ez = torch.where(e == 0, torch.zeros_like(z), e * z)
    H = torch.where(empty, torch.zeros(rows, dtype=torch.float64), (ls - ez.sum(1, keepdim=True) / s)[:, 0])
    logp = (z - ls).gather(1, at[:, None])[:, 0]
    logp = torch.where(empty, torch.full_like(logp, -INF), logp)
    logp = torch.where(named, logp, torch.zeros_like(logp))
    # A stable sort keeps equal ones in the order of their indices; NaN is none of them.
    best = torch.where(torch.isnan(x), torch.full_like(x, -INF), x).sort(dim=1, descending=True, stable=True)
    ids, found = best.indices[:, :top], best.values[:, :top] > -INF
    values = torch.where(found, (z - ls).gather(1, ids), torch.full_like(found, -INF, dtype=torch.float64))
    ids = torch.where(found, ids, torch.full_like(ids, -1)).to(torch.int32)
    out = dict(logp=logp, entropy=H, values=values, ids=ids)
    if a is not None:
        ga = torch.where(named & ~empty, a.double().cpu(), torch.zeros_like(logp))[:, None]
        gh = h.double().cpu()[:, None]
        lp = torch.where(p == 0, torch.zeros_like(z), z - ls)
        dx = -p * (ga + gh * (lp + H[:, None]))
        dx.scatter_add_(1, at[:, None], ga)
        out["dx"] = dx
    # Bounds.  z rounds by |z| e; e^z by that, by the rounded product with log2(e) and the
    # constant (16-bit logits: 1.5 |z| e) and 4 e of the exponential.  s adds its terms at
    # most n / 32 + 64 one after another, and a thread that meets a new maximum scales what
    # it has: the shifts add up to at most the spread of the terms that count.
    az = torch.where(p == 0, torch.zeros_like(z), z.abs()).clamp_max(104.0)
    spread = az.amax(1, keepdim=True)
    term = (2.5 * az + 4) * E32
    depth = (n / 32 + 72) * E32 + 2.5 * spread * E32
    rel_s = (p * term).sum(1, keepdim=True) + depth
    err_ls = rel_s + 2 * E32 * torch.where(empty[:, None], torch.zeros_like(ls), ls).abs()
    t = (p * az).sum(1, keepdim=True)
    err_H = (err_ls + (p * az * (term + 2 * E32)).sum(1, keepdim=True) + t * (depth + rel_s + 2 * E32)
             + E32 * H[:, None].abs())
    err_lp = az * E32 + err_ls + E32 * (az + ls.abs().nan_to_num(0.0, 0.0, 0.0))
    out["err_H"] = err_H[:, 0]
    zt = z.gather(1, at[:, None])[:, 0].abs().nan_to_num(0.0, 0.0, 0.0)
    out["err_logp"] = 2 * zt * E32 + err_ls[:, 0] + E32 * ls[:, 0].abs().nan_to_num(0.0, 0.0, 0.0)
    out["err_values"] = (2 * values.abs().nan_to_num(0.0, 0.0, 0.0) * E32 + 2 * err_ls)
    if a is not None:
        inner = ga.abs() + gh.abs() * (lp.abs() + H[:, None].abs())
        rel_p = err_lp + 1.5 * lp.abs() * E32 + 4 * E32
        out["err_dx"] = (p * (rel_p * inner + gh.abs() * (err_lp + err_H) + 4 * E32 * inner)
                         + 2 * E32 * (out["dx"].abs() + p * inner) + 2.0 ** -126 * inner)
    return out


# ----------------------------------------------------------------- route


def choose(x, top_k, score, bias, groups, top_groups):
    """Chosen experts [rows, top_k], -1 where none is left, by sorting (value,
    index) of each row in 64 bits."""
    x = x.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    rows, n = x.shape
    out = np.full((rows, top_k), -1, np.int32)

    def key(v):  # NaN above all
        return -INF if v != v else -v

    for r in range(rows):
        with np.errstate(all="ignore"):
            if b is None and groups == 1:
                v = x[r].copy()
            else:
                if score == "softmax":
                    v = np.exp(x[r] - np.fmax.reduce(x[r]))
                    v = v / v.sum()
                else:
                    v = 1.0 / (1.0 + np.exp(-x[r]))
                if b is not None:
                    v = np.where(np.isneginf(b), -np.inf, v + b)
            v[np.isneginf(x[r])] = -np.inf
        if groups > 1:
            size, totals = n // groups, []
            for g in range(groups):
                part = sorted((v[g * size + i] for i in range(size)), key=key)[:2]
                if part[0] == -np.inf:
                    totals.append(-np.inf)
                else:
                    totals.append(part[0] + (part[1] if size > 1 and part[1] != -np.inf else 0.0))
            kept = sorted(range(groups), key=lambda g: (key(totals[g]), g))[:top_groups]
            for g in range(groups):
                if g not in kept:
                    v[g * size:(g + 1) * size] = -np.inf
        order = sorted((i for i in range(n) if v[i] != -np.inf), key=lambda i: (key(v[i]), i))[:top_k]
        out[r, :len(order)] = order
    return torch.from_numpy(out)


def undecided(x, score, bias, groups, top_groups):
    """Rows in which two groups at the border of the choice have sums within
    2^-50 of each other.  Such a sum is of four numbers, s_i + b_i and s_j + b_j:
    where another group has the same scores with the biases exchanged, the two
    are equal, and each is off by up to four roundings of 2^-53 of at most its
    size (two additions, their sum, the scores' own): 64 bits leave either
    first."""
    if groups == 1:
        return torch.zeros(x.size(0), dtype=torch.bool)
    v = x.double().cpu()
    v = torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)
    v = v if bias is None else v + bias.double().cpu()
    v = torch.where(x.cpu() == -INF, torch.full_like(v, -INF), v)
    two = v.view(x.size(0), groups, -1).sort(2, descending=True).values[:, :, :2]
    total = torch.where(two == -INF, torch.zeros_like(two), two).sum(2)
    total = total.sort(1, descending=True).values
    if top_groups == groups:
        return torch.zeros(x.size(0), dtype=torch.bool)
    gap = total[:, top_groups - 1] - total[:, top_groups]
    return gap <= 2.0 ** -50 * total[:, 0].abs().clamp_min(1.0)


def route(x, chosen, score, renormalize, scale, g=None):
    """Weights of the chosen experts, their bound, and (with the incoming
    gradient g) dx and its bound, in 64 bits."""
    x = x.double().cpu()
    rows, n = x.shape
    found, at = chosen >= 0, chosen.clamp_min(0).long()
    m = x.amax(1, keepdim=True)
    z = torch.where(m == -INF, torch.full_like(x, -INF), x - m)
    if score == "softmax":
        e = torch.exp(z)
        s = e.sum(1, keepdim=True)
        p = torch.where(s == 0, torch.zeros_like(e), e / s)
        log_score = torch.where(e == 0, torch.full_like(z, -INF), z - torch.log(s))
        log_score = torch.where((x > -INF) & (e == 0), z - torch.log(s), log_score)
        az = torch.where(p == 0, torch.zeros_like(z), z.abs())
        rel_s = (p * (az + 4)).sum(1, keepdim=True) * E32 + (n / 16 + 16) * E32
        own = z.abs().nan_to_num(0.0, 0.0, 0.0)
        err_l = 2 * own * E32 + rel_s + 4 * E32 * torch.log(s).abs().nan_to_num(0.0, 0.0, 0.0)
    else:
        log_score = torch.nn.functional.logsigmoid(x)
        err_l = 4 * E32 * log_score.abs().nan_to_num(0.0, 0.0, 0.0) + 3 * E32
    mine = torch.where(found, log_score.gather(1, at), torch.full_like(found, -INF, dtype=torch.float64))
    err = torch.where(found, err_l.gather(1, at), torch.zeros_like(mine))
    if renormalize:
        top = mine.amax(1, keepdim=True)
        u = torch.where(found, torch.exp(mine - torch.where(top == -INF, torch.zeros_like(top), top)),
                        torch.zeros_like(mine))
        total = u.sum(1, keepdim=True)
        u = torch.where(total == 0, torch.zeros_like(u), u / total)
        rel = 2 * err.amax(1, keepdim=True) + err
        rel = rel + (u * rel).sum(1, keepdim=True) + (chosen.shape[1] + 10) * E32
    else:
        u = torch.where(found, torch.exp(mine), torch.zeros_like(mine))
        rel = err + 6 * E32
    w = scale * u
    out = dict(w=w, err_w=w * (rel + 2 * E32))
    if g is not None:
        g = torch.where(found, g.double().cpu(), torch.zeros_like(w))
        k = chosen.shape[1]
        if renormalize:
            mean = (u * g).sum(1, keepdim=True)
            err_mean = (u * g.abs() * (rel + (k + 4) * E32)).sum(1, keepdim=True)
            dl = w * (g - mean)
            err_dl = w * ((g - mean).abs() * (rel + 4 * E32) + err_mean + E32 * (g.abs() + mean.abs()))
        else:
            dl = w * g
            err_dl = dl.abs() * (rel + 4 * E32)
        total = dl.sum(1, keepdim=True)
        err_total = err_dl.sum(1, keepdim=True) + (k + 2) * E32 * dl.abs().sum(1, keepdim=True)
        if score == "sigmoid":
            back = torch.sigmoid(-x).gather(1, at)
            dl, err_dl = dl * back, err_dl * back + (dl * back).abs() * 8 * E32
        dl, err_dl = torch.where(found, dl, torch.zeros_like(dl)), torch.where(found, err_dl, torch.zeros_like(dl))
        dx = torch.zeros_like(x).scatter_add_(1, at, dl)
        err_dx = torch.zeros_like(x).scatter_add_(1, at, err_dl)
        if score == "softmax" and not renormalize:
            dx = dx - p * total
            err_dx = err_dx + p * (err_total + total.abs() * (err_l.nan_to_num(0.0, 0.0, 0.0) + 8 * E32)) + 2 * E32 * dx.abs()
        out.update(dx=dx, err_dx=err_dx)
    return out


# ---------------------------------------------------------------- experts


def plan(experts, count):
    """offsets and place, by hand."""
    ids = experts.reshape(-1).cpu().tolist()
    buckets = [[] for _ in range(count + 1)]
    for i, e in enumerate(ids):
        buckets[e if 0 <= e < count else count].append(i)
    offsets, place, at = [0], [0] * len(ids), 0
    for b, bucket in enumerate(buckets):
        for i in bucket:
            place[i] = at
            at += 1
        if b < count:
            offsets.append(at)
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(place, dtype=torch.int32)


def scale_of(width):
    return math.sqrt(width)
