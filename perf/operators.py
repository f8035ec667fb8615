"""Timed cases of the expert-routing operators and of the plain layer norm, their plain forms in
elementary torch operations and their definitions in 64 bits.

The operators are those of a mixture-of-experts node MLP: the layer norm of the invariants that a
router reads, the choice of the experts (top-k with softmax weights), the nodes' rows sorted by expert
and back, and the experts' per-degree channel maps on the sorted rows.

With ``own`` false ``run`` computes the plain forms, with ``own`` true it calls the package.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LN_EPS = 1e-5


def _package():
    """The package, imported only where its operators are called."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-eq_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_eq
    return flash_eq


# ---- cases -------------------------------------------------------------------------------------------

def listed():
    return [
        # a toy graph's router input: 64 channels' norms of degrees 0..2, one training call, latency
        dict(name="norm_toy", kind="norm", rows=100, width=192, dtype="f32", train=True),
        # the same invariants of a 50k-node chain
        dict(name="norm_nodes", kind="norm", rows=50000, width=192, dtype="f32", train=True),
        # 128 channels' norms of degrees 0..6 on every edge of the high-degree layer, bfloat16
        dict(name="norm_edges_bf16", kind="norm", rows=160000, width=896, dtype="bf16", train=True),
        # the choice among a few experts for a toy graph
        dict(name="topk_toy", kind="topk", rows=100, experts=8, k=2, dtype="f32", normalize=True, train=True),
        # many nodes over many experts, probabilities not renormalised, an odd number of rows
        dict(name="topk_nodes", kind="topk", rows=200003, experts=64, k=4, dtype="f32", normalize=False, train=True),
        # one expert per node of a toy graph: four components of 32 channels
        dict(name="rows_toy", kind="rows", rows=100, planes=4, width=32, experts=4, k=1, dtype="f32", unrouted=0.0),
        # two experts per node of a training batch, degrees 0..2 of 64 channels; a tenth of the rows is
        # padding of the batch and goes to no expert
        dict(name="rows_nodes", kind="rows", rows=20000, planes=9, width=64, experts=8, k=2, dtype="f32", unrouted=0.1),
        # high-degree features in bfloat16, four of many experts, an odd number of rows
        dict(name="rows_l6_bf16", kind="rows", rows=5003, planes=49, width=128, experts=64, k=4, dtype="bf16",
             unrouted=0.0),
        # inference of a single node by two of its experts
        dict(name="linear_one_node", kind="linear", slots=2, lmax=2, cin=64, cout=128, experts=8, dtype="f32", train=False),
        # the widening map of a training batch: 20k nodes by two experts, degrees 0..2
        dict(name="linear_nodes", kind="linear", slots=40000, lmax=2, cin=64, cout=128, experts=8, dtype="f32", train=True),
        # high-degree features in bfloat16, an odd number of rows
        dict(name="linear_l6_bf16", kind="linear", slots=20011, lmax=6, cin=128, cout=128, experts=16, dtype="bf16",
             train=True),
        # a map of scalars (an invariant head), wide channels, many experts with ragged counts
        dict(name="linear_wide_bf16", kind="linear", slots=8191, lmax=0, cin=512, cout=1024, experts=64, dtype="bf16",
             train=True),
    ]


def _log_int(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    kind = rng.choice(["norm", "topk", "rows", "linear"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "norm":
        width = _log_int(rng, 1, 8192)
        case = dict(kind=kind, rows=_log_int(rng, 1, 160000), width=width, dtype=dtype, train=rng.random() < 0.7)
        size = "rows"
    elif kind == "topk":
        experts = _log_int(rng, 2, 256)
        case = dict(kind=kind, rows=_log_int(rng, 1, 400000), experts=experts, k=rng.randint(1, min(8, experts)), dtype=dtype,
                    normalize=rng.random() < 0.5, train=rng.random() < 0.7)
        size = "rows"
    elif kind == "rows":
        planes = rng.choice([1, 4, 9, 16, 25, 36, 49])
        experts = _log_int(rng, 1, 128)
        case = dict(kind=kind, rows=_log_int(rng, 1, 100000), planes=planes,
                    width=_log_int(rng, 1, 1152 if planes == 1 else 128), experts=experts, k=rng.randint(1, min(4, experts)),
                    dtype=dtype, unrouted=rng.choice([0.0, 0.0, 0.1, 0.5]))
        size = "rows"
    else:
        lmax = rng.choice([0, 0, 1, 2, 3, 4, 6])
        most = 1024 if lmax == 0 else 160
        case = dict(kind=kind, slots=_log_int(rng, 1, 100000), lmax=lmax, cin=_log_int(rng, 4, most),
                    cout=_log_int(rng, 4, most), experts=_log_int(rng, 1, 64), dtype=dtype, train=rng.random() < 0.7)
        size = "slots"
    # no more than the largest listed case of the kind: in bytes, in operations
    top = [work(c) for c in listed() if c["kind"] == kind]
    while case[size] > 1 and any(work(case)[key] > max(t[key] for t in top) for key in ("bytes", "flops")):
        case[size] = case[size] * 2 // 3
    return case


def _degrees(case):
    return list(range(case["lmax"] + 1))


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        n, w = case["rows"] * case["width"], case["width"]
        if not case["train"]:
            return dict(bytes=2 * size * n + 2 * size * w, flops=8 * n)
        return dict(bytes=4 * size * n + 4 * size * w, flops=22 * n)
    if kind == "topk":
        n, x, k = case["rows"], case["experts"], case["k"]
        out = 12 * n * k + 4 * x
        if not case["train"]:
            return dict(bytes=size * n * x + out, flops=n * x * (4 + k))
        return dict(bytes=2 * size * n * x + out + 4 * n * k + 4 * x, flops=n * x * (10 + k))
    if kind == "rows":
        row = size * case["planes"] * case["width"]
        t, s = case["rows"], case["rows"] * case["k"]
        ints = 8 * s + 8 * s + 4 * case["experts"] + 4
        return dict(bytes=ints + 4 * t * row + 4 * s * row + 8 * s,
                    flops=s * case["planes"] * case["width"] * 6)
    d, s, x = (case["lmax"] + 1) ** 2, case["slots"], case["experts"]
    ci, co, reps = case["cin"], case["cout"], case["lmax"] + 1
    weights = size * x * (reps * ci * co + co)
    once = 2 * d * s * ci * co
    if not case["train"]:
        return dict(bytes=size * d * s * (ci + co) + min(1.0, s / x) * weights, flops=once)
    return dict(bytes=2 * size * d * s * (ci + co) + 2 * weights, flops=3 * once)


# ---- inputs ------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 9973 + 41)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uneven_experts(g, rows, experts, k):
    """k different experts for every row, some experts chosen far more often than others."""
    liking = _randn(g, experts) + 1.5 * _randn(g, rows, experts)
    return torch.sort(liking, dim=1, descending=True, stable=True).indices[:, :k].contiguous()


def _inputs(case, seed):
    """What the seed determines: the same for ``run`` and ``exact``."""
    g = _generator(seed)
    dt = _DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "norm":
        r, w = case["rows"], case["width"]
        # Euclidean norms of a few components: positive, of different scale from row to row
        x = (_randn(g, r, w) ** 2 + _randn(g, r, w) ** 2).sqrt_() * (0.5 + torch.rand(r, 1, generator=g, device="cuda"))
        return dict(x=x.to(dt), weight=(1 + 0.1 * _randn(g, w)).to(dt), bias=(0.1 * _randn(g, w)).to(dt),
                    gy=_randn(g, r, w).to(dt) if case["train"] else None)
    if kind == "topk":
        r, x = case["rows"], case["experts"]
        logits = (_randn(g, x) + 1.5 * _randn(g, r, x)).to(dt)
        return dict(logits=logits, gw=_randn(g, r, case["k"]), gmean=_randn(g, x))
    if kind == "rows":
        t, d, w, k = case["rows"], case["planes"], case["width"], case["k"]
        ids = _uneven_experts(g, t, case["experts"], k)
        pad = int(case["unrouted"] * t)
        if pad:                                         # the batch's padding: its last rows
            ids[t - pad:] = -1
        weights = torch.rand(t, k, generator=g, device="cuda") + 0.1
        return dict(ids=ids, x=_randn(g, d, t, w).to(dt), ys=_randn(g, d, t * k, w).to(dt), gy=_randn(g, d, t, w).to(dt),
                    gxs=_randn(g, d, t * k, w).to(dt), weights=weights / weights.sum(1, keepdim=True))
    d, s, reps = (case["lmax"] + 1) ** 2, case["slots"], case["lmax"] + 1
    ci, co, x = case["cin"], case["cout"], case["experts"]
    ids = _uneven_experts(g, s, x, 1)
    return dict(ids=ids, x=_randn(g, d, s, ci).to(dt), weight=(_randn(g, x, reps, co, ci) / math.sqrt(ci)).to(dt),
                bias=(0.1 * _randn(g, x, co, 1)).to(dt), gy=_randn(g, d, s, co).to(dt) if case["train"] else None)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    kind = case["kind"]
    if own:
        fe = s["fe"] = _package()
        if kind == "norm":
            s["norm"] = fe.InvariantLayerNorm(case["width"], epsilon=LN_EPS).to(device="cuda", dtype=_DTYPES[case["dtype"]])
            with torch.no_grad():
                s["norm"].weight.copy_(s["weight"])
                s["norm"].bias.copy_(s["bias"])
            s["x"].requires_grad_(case["train"])
        elif kind == "topk":
            s["logits"].requires_grad_(case["train"])
        elif kind == "rows":
            for name in ("x", "ys", "weights"):
                s[name].requires_grad_()
        else:                                           # the plan is made once for all of a layer's maps
            s["plan"] = fe.ExpertPlan(s["ids"], case["experts"])
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(case["train"])
    elif kind == "linear":                              # the sorted rows' ranges, on the host
        s["counts"] = torch.bincount(s["ids"].view(-1), minlength=case["experts"]).tolist()
    return s


# ---- one pass ----------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return dict(norm=_own_norm, topk=_own_topk, rows=_own_rows, linear=_own_linear)[kind](s)
    return dict(norm=_plain_norm, topk=_plain_topk, rows=_plain_rows, linear=_plain_linear)[kind](s)


def _own_norm(s):
    if not s["case"]["train"]:
        with torch.no_grad():
            return dict(y=s["norm"](s["x"]))
    y = s["norm"](s["x"])
    gx, gw, gb = torch.autograd.grad(y, [s["x"], s["norm"].weight, s["norm"].bias], s["gy"])
    return dict(y=y.detach(), gx=gx, gw=gw, gb=gb)


def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    dt = s["x"].dtype
    c = x - x.mean(1, keepdim=True)
    rstd = 1.0 / ((c * c).mean(1, keepdim=True) + LN_EPS).sqrt()
    xh = c * rstd
    y = (xh * w + b).to(dt)
    if not s["case"]["train"]:
        return dict(y=y)
    g = s["gy"].float()
    h = g * w
    gx = rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
    return dict(y=y, gx=gx.to(dt), gw=(g * xh).sum(0).to(dt), gb=g.sum(0).to(dt))


def _own_topk(s):
    case = s["case"]
    if not case["train"]:
        with torch.no_grad():
            ids, weights, mean = s["fe"].expert_topk(s["logits"], case["k"], normalize=case["normalize"])
        return dict(ids=ids, weights=weights, mean=mean)
    ids, weights, mean = s["fe"].expert_topk(s["logits"], case["k"], normalize=case["normalize"])
    (gl,) = torch.autograd.grad([weights, mean], [s["logits"]], [s["gw"], s["gmean"]])
    return dict(ids=ids, weights=weights.detach(), mean=mean.detach(), gl=gl)


def _plain_topk(s):
    case = s["case"]
    l = s["logits"].float()
    e = (l - l.amax(1, keepdim=True)).exp()
    p = e / e.sum(1, keepdim=True)
    ids = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :case["k"]].contiguous()
    chosen = p.gather(1, ids)
    total = chosen.sum(1, keepdim=True)
    weights = chosen / total if case["normalize"] else chosen
    out = dict(ids=ids, weights=weights, mean=(p.double().sum(0) / p.shape[0]).float())
    if case["train"]:
        g, m = s["gw"], s["gmean"]
        gp = m / p.shape[0] + torch.zeros_like(p)
        if case["normalize"]:
            g = (g - (g * weights).sum(1, keepdim=True)) / total
        gp.scatter_add_(1, ids, g)
        out["gl"] = (p * (gp - (p * gp).sum(1, keepdim=True))).to(s["logits"].dtype)
    return out


def _own_rows(s):
    plan = s["fe"].ExpertPlan(s["ids"], s["case"]["experts"])
    xs = plan.dispatch(s["x"])
    y = plan.combine(s["ys"], s["weights"])
    gx, gys, gw = torch.autograd.grad([xs, y], [s["x"], s["ys"], s["weights"]], [s["gxs"], s["gy"]])
    return dict(order=plan.order, positions=plan.positions, offsets=plan.offsets, xs=xs.detach(), y=y.detach(), gx=gx,
                gys=gys, gw=gw)


def _plain_rows(s):
    case = s["case"]
    dt, n, k = s["x"].dtype, case["experts"], case["k"]
    ids = s["ids"].reshape(-1)
    routed = (ids >= 0) & (ids < n)
    key = torch.where(routed, ids, torch.full_like(ids, n))
    key, order = torch.sort(key, stable=True)
    offsets = (key[None, :] < torch.arange(n + 1, device=key.device)[:, None]).sum(1)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device=order.device)
    node = order // k
    live = (key < n).float()[:, None]
    live_slot = routed.float().view(-1, k, 1)
    w = s["weights"]
    positions = positions.view(-1, k)
    xs = s["x"].float()[:, node] * live
    picked = s["ys"].float()[:, positions]                              # (planes, rows, k, width)
    y = (picked * (w[..., None] * live_slot)).sum(2)
    gy = s["gy"].float()
    gw = (picked * gy[:, :, None]).sum((0, 3)) * live_slot[..., 0]
    gys = gy[:, node] * (w.reshape(-1)[order][:, None] * live)
    gx = (s["gxs"].float()[:, positions] * live_slot).sum(2)
    return dict(order=order.int(), positions=positions.int(), offsets=offsets.int(), xs=xs.to(dt), y=y.to(dt), gx=gx.to(dt),
                gys=gys.to(dt), gw=gw)


def _own_linear(s):
    case = s["case"]
    lvals = _degrees(case)
    if not case["train"]:
        with torch.no_grad():
            return dict(y=s["fe"].expert_linear(s["x"], s["weight"], s["plan"], lvals, s["bias"]))
    y = s["fe"].expert_linear(s["x"], s["weight"], s["plan"], lvals, s["bias"])
    gx, gw, gb = torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["gy"])
    return dict(y=y.detach(), gx=gx, gw=gw, gb=gb)


def _plain_linear(s):
    case = s["case"]
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    dt = s["x"].dtype
    train = case["train"]
    y = torch.empty(x.shape[0], x.shape[1], case["cout"], device=x.device)
    if train:
        gy = s["gy"].float()
        gx, gw, gb = torch.empty_like(x), torch.zeros_like(w), torch.zeros_like(b)
    a = 0
    for e, count in enumerate(s["counts"]):
        z = a + count
        if count:
            for l in range(case["lmax"] + 1):
                for d in range(l * l, (l + 1) * (l + 1)):
                    torch.mm(x[d, a:z], w[e, l].t(), out=y[d, a:z])
                    if train:
                        torch.mm(gy[d, a:z], w[e, l], out=gx[d, a:z])
                        gw[e, l] += torch.mm(gy[d, a:z].t(), x[d, a:z])
            y[0, a:z] += b[e, :, 0]
            if train:
                gb[e, :, 0] = gy[0, a:z].sum(0)
        a = z
    if not train:
        return dict(y=y.to(dt))
    return dict(y=y.to(dt), gx=gx.to(dt), gw=gw.to(dt), gb=gb.to(dt))


# ---- the definitions in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return dict(norm=_exact_norm, topk=_exact_topk, rows=_exact_rows, linear=_exact_linear)[case["kind"]](case, s)


def _leaf(t):
    return t.double().requires_grad_()


def _exact_norm(case, s):
    """By autograd from y = (x - E x) / sqrt(Var x + eps) * w + b, in pieces of rows."""
    w, b = _leaf(s["weight"]), _leaf(s["bias"])
    ys, gxs, gw, gb = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for a in range(0, case["rows"], 16384):
        x = _leaf(s["x"][a:a + 16384])
        mu = x.sum(1, keepdim=True) / case["width"]
        var = (x ** 2).sum(1, keepdim=True) / case["width"] - mu ** 2
        y = (x - mu) * (var.clamp(min=0) + LN_EPS) ** -0.5 * w + b
        ys.append(y.detach())
        if case["train"]:
            d = torch.autograd.grad(y, [x, w, b], s["gy"][a:a + 16384].double())
            gxs.append(d[0])
            gw += d[1]
            gb += d[2]
    if not case["train"]:
        return dict(y=torch.cat(ys))
    return dict(y=torch.cat(ys), gx=torch.cat(gxs), gw=gw.detach(), gb=gb.detach())


def _exact_topk(case, s):
    """The choice on the host, one maximum after another; values and gradients by autograd."""
    values = s["logits"].float().cpu().numpy().astype(np.float64)
    left, rows = values.copy(), np.arange(case["rows"])
    picks = []
    for _ in range(case["k"]):
        best = left.argmax(1)                           # the first of equal maxima
        picks.append(best)
        left[rows, best] = -np.inf
    ids = torch.from_numpy(np.stack(picks, 1)).to(s["logits"].device)
    l = _leaf(s["logits"])
    p = torch.softmax(l, 1)
    weights = torch.softmax(l.gather(1, ids), 1) if case["normalize"] else p.gather(1, ids)
    mean = p.mean(0)
    out = dict(ids=ids, weights=weights.detach(), mean=mean.detach())
    if case["train"]:
        out["gl"] = torch.autograd.grad((weights * s["gw"].double()).sum() + (mean * s["gmean"].double()).sum(), l)[0]
    return out


def _exact_rows(case, s):
    """The order on the host; the moves and their gradients by autograd over one row of slots after another."""
    n, k, t = case["experts"], case["k"], case["rows"]
    dev = s["x"].device
    flat = s["ids"].cpu().numpy().reshape(-1)
    key = np.where((flat < 0) | (flat >= n), n, flat)
    order = np.argsort(key, kind="stable")
    positions = np.argsort(order, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(n + 1))
    slots = torch.from_numpy(positions.reshape(t, k)).to(dev)
    routed = torch.from_numpy((key < n).reshape(t, k)).to(dev)
    w = s["weights"].double()
    xs = torch.zeros(s["ys"].shape, dtype=torch.float64, device=dev)
    gys = torch.zeros_like(xs)
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device=dev)
    gx, gw = torch.zeros_like(y), torch.zeros_like(w)
    for d in range(case["planes"]):
        x, ys, gy, gxs = (s[name][d].double() for name in ("x", "ys", "gy", "gxs"))
        for j in range(k):
            live = routed[:, j].nonzero()[:, 0]
            at = slots[live, j]
            xs[d, at] = x[live]
            y[d, live] += w[live, j, None] * ys[at]
            gx[d, live] += gxs[at]
            gys[d, at] = w[live, j, None] * gy[live]
            gw[live, j] += (gy[live] * ys[at]).sum(1)
    as_int = lambda a, shape: torch.from_numpy(a.astype(np.int32).reshape(shape)).to(dev)
    return dict(order=as_int(order, -1), positions=as_int(positions, (t, k)), offsets=as_int(offsets, -1), xs=xs, y=y, gx=gx,
                gys=gys, gw=gw)


def _exact_linear(case, s):
    """Every expert's rows by a mask over the sorted experts, by autograd."""
    expert = torch.sort(s["ids"].view(-1)).values
    w, b = _leaf(s["weight"]), _leaf(s["bias"])
    shape = (s["x"].shape[0], case["slots"])
    y = torch.zeros(*shape, case["cout"], dtype=torch.float64, device=w.device)
    gx = torch.zeros(*shape, case["cin"], dtype=torch.float64, device=w.device)
    gw, gb = torch.zeros_like(w), torch.zeros_like(b)
    for e in range(case["experts"]):
        rows = (expert == e).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        for l in range(case["lmax"] + 1):
            comps = torch.arange(l * l, (l + 1) ** 2, device=w.device)
            x = _leaf(s["x"][comps][:, rows])
            out = torch.matmul(x.reshape(-1, case["cin"]), w[e, l].t()).view(len(comps), rows.numel(), case["cout"])
            if l == 0:
                out = out + b[e, :, 0]
            y[comps[:, None], rows] = out.detach()
            if case["train"]:
                leaves = [x, w] + ([b] if l == 0 else [])
                d = torch.autograd.grad(out, leaves, s["gy"][comps][:, rows].double())
                gx[comps[:, None], rows] = d[0]
                gw += d[1]
                if l == 0:
                    gb += d[2]
    if not case["train"]:
        return dict(y=y)
    return dict(y=y, gx=gx, gw=gw.detach(), gb=gb.detach())
