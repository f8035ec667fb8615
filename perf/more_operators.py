"""Timed cases of the operators that fine-tune a trained transformer, their plain forms in elementary torch
operations and their definitions in 64 bits.

* attention: the edge attention's weights with a learned bias for each head and bucket of distances, and dropout of the weights;
* dropout: whole irreps of features dropped by a counter-based generator whose mask is never stored;
* adapter: a linear map shared by all rows beside low-rank maps of which every row has its own (one for each task,
  structure or request of a batch).

With ``own`` false ``run`` computes the plain forms, with ``own`` true it calls the package.

The generator is Philox 4 x 32 with ten rounds (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011).  The key
is the seed; block b has the counter (b mod 2^32, b / 2^32, 0, 0), and its four words make eight numbers of 16 bits, the
lower half of a word first.  Unit u of a tensor has number u mod 8 of block u / 8 and is dropped where that is below
round(65536 p); what is kept is multiplied by 65536 / (65536 - round(65536 p)).
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAX_DIST = 10.0
ADAPTER_SCALE = 2.0


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
        # a toy graph's training step, latency: 500 random edges of 100 nodes, degrees 0 and 1 of 32 channels
        dict(name="attention_toy", kind="attention", nodes=100, degree=5, edges="random", lmax=1, mult=32, heads=8, dtype="f32",
             cm=False, buckets=32, cutoff=False, p=0.1, train=True),
        # a transformer block's training batch: 20k nodes with 32 neighbours each, component-major as the block keeps it; the
        # last bucket is beyond the cutoff
        dict(name="attention_block", kind="attention", nodes=20000, degree=32, edges="neighbours", lmax=2, mult=64, heads=8,
             dtype="f32", cm=True, buckets=100, cutoff=True, p=0.1, train=True),
        # inference over a chain of 50k nodes, whose neighbours have near numbers
        dict(name="attention_chain_infer", kind="attention", nodes=50000, degree=24, edges="chain", lmax=2, mult=64, heads=8,
             dtype="f32", cm=True, buckets=32, cutoff=False, p=0.0, train=False),
        # high-degree features in bfloat16, an odd number of nodes and of neighbours
        dict(name="attention_l6_bf16", kind="attention", nodes=5003, degree=31, edges="neighbours", lmax=6, mult=128, heads=8,
             dtype="bf16", cm=False, buckets=100, cutoff=False, p=0.25, train=True),
        # a toy graph's features, latency
        dict(name="dropout_toy", kind="dropout", rows=100, lmax=1, mult=32, dtype="f32", cm=False, p=0.1, train=True),
        # the residual branch of 50k nodes, degrees 0 to 2: one decision for all components of an irrep
        dict(name="dropout_nodes", kind="dropout", rows=50000, lmax=2, mult=64, dtype="f32", cm=False, p=0.1, train=True),
        # invariants of every edge of the high-degree layer, element by element
        dict(name="dropout_edges_bf16", kind="dropout", rows=160000, lmax=0, mult=896, dtype="bf16", cm=False, p=0.2, train=True),
        # inference of a single node with its adapter
        dict(name="adapter_one_node", kind="adapter", rows=1, lmax=2, cin=64, cout=128, adapters=8, rank=8, dtype="f32", none=0.0,
             train="no"),
        # 64 requests of one row each, most with an adapter of their own, through a wide map
        dict(name="adapter_requests_bf16", kind="adapter", rows=64, lmax=0, cin=512, cout=1024, adapters=64, rank=16,
             dtype="bf16", none=0.1, train="no"),
        # a training batch of 20k nodes from eight tasks, degrees 0 to 2, the shared map trained too
        dict(name="adapter_nodes", kind="adapter", rows=20000, lmax=2, cin=64, cout=128, adapters=8, rank=16, dtype="f32",
             none=0.0, train="all"),
        # high-degree features in bfloat16, an odd number of rows, the shared map frozen
        dict(name="adapter_l6_bf16", kind="adapter", rows=20011, lmax=6, cin=128, cout=128, adapters=16, rank=16, dtype="bf16",
             none=0.0, train="adapters"),
        # a map of scalars with wide channels and many adapters; a tenth of the rows has none
        dict(name="adapter_wide_bf16", kind="adapter", rows=8191, lmax=0, cin=512, cout=1024, adapters=64, rank=32, dtype="bf16",
             none=0.1, train="adapters"),
    ]


def _log_int(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "dropout", "adapter", "adapter"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "attention":
        heads = rng.choice([1, 2, 3, 4, 8, 16])
        lmax = rng.choice([0, 1, 2, 2, 3, 4, 6])
        case = dict(kind=kind, nodes=_log_int(rng, 1, 50000), degree=rng.randint(1, 32),
                    edges=rng.choice(["random", "neighbours", "chain"]), lmax=lmax,
                    mult=heads * max(1, _log_int(rng, 4, 128) // heads), heads=heads, dtype=dtype, cm=rng.random() < 0.5,
                    buckets=_log_int(rng, 1, 512), cutoff=rng.random() < 0.3, p=rng.choice([0.0, 0.1, 0.25, 0.5]),
                    train=rng.random() < 0.7)
        size = "nodes"
    elif kind == "dropout":
        lmax = rng.choice([0, 0, 1, 2, 3, 4, 6])
        case = dict(kind=kind, rows=_log_int(rng, 1, 160000), lmax=lmax, mult=_log_int(rng, 1, 1024 if lmax == 0 else 128),
                    dtype=dtype, cm=rng.random() < 0.5, p=rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]), train=rng.random() < 0.7)
        size = "rows"
    else:
        lmax = rng.choice([0, 0, 1, 2, 3, 4, 6])
        most = 1024 if lmax == 0 else 160
        adapters = _log_int(rng, 1, 64)
        case = dict(kind=kind, rows=_log_int(rng, 1, 100000), lmax=lmax, cin=_log_int(rng, 4, most), cout=_log_int(rng, 4, most),
                    adapters=adapters, rank=_log_int(rng, 1, min(64, 2048 // adapters)), dtype=dtype,
                    none=rng.choice([0.0, 0.0, 0.1, 0.5]), train=rng.choice(["no", "adapters", "adapters", "all"]))
        size = "rows"
    # no more than the largest listed case of the kind: in bytes, in operations
    top = [work(c) for c in listed() if c["kind"] == kind]
    while case[size] > 1 and any(work(case)[key] > max(t[key] for t in top) for key in ("bytes", "flops")):
        case[size] = case[size] * 2 // 3
    return case


def _dim(case):
    return (case["lmax"] + 1) ** 2


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "attention":
        n, e, h = case["nodes"], case["nodes"] * case["degree"], case["heads"]
        row = case["mult"] * _dim(case)
        # the table, two indices and the distance of every edge, buckets and weights
        once = size * 2 * n * row + e * (16 + 4 + 4 + size * h) + size * case["buckets"] * h
        dots = 2 * e * row + 12 * e * h
        if not case["train"]:
            return dict(bytes=once, flops=dots)
        # the weights' gradient read, the table's and the bias's written; a dot's two gradients
        return dict(bytes=once + size * 2 * n * row + size * e * h + size * case["buckets"] * h, flops=3 * dots)
    if case["kind"] == "dropout":
        n = case["rows"] * case["mult"] * _dim(case)
        once = 2 * size * n
        return dict(bytes=2 * once if case["train"] else once, flops=2 * n if case["train"] else n)
    d, r, x = _dim(case), case["rows"], case["adapters"]
    ci, co, k, reps = case["cin"], case["cout"], case["rank"], case["lmax"] + 1
    shared = size * (reps * ci * co + co)
    low = size * min(x, r) * reps * k * (ci + co)
    rows = size * d * r
    flops, thin = 2 * d * r * ci * co, 2 * d * r * k * (ci + co)
    if case["train"] == "no":
        return dict(bytes=rows * (ci + co) + shared + low + 4 * r, flops=flops + thin)
    every = case["train"] == "all"
    low_grads = size * x * reps * k * (ci + co)
    # both directions' rows, the weights once, their gradients; the reduced rows are formed again by what needs them
    return dict(bytes=2 * rows * (ci + co) + shared * (2 if every else 1) + low + low_grads + 4 * r,
                flops=flops * (3 if every else 2) + 3 * thin)


# ---- inputs ------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7547 + 29)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _seed(g):
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), generator=g, device="cuda")


def _inputs(case, seed):
    """What the seed determines: the same for ``run`` and ``exact``."""
    g = _generator(seed)
    dt = _DTYPES[case["dtype"]]
    if case["kind"] == "attention":
        n, h, b, mult, dim = case["nodes"], case["heads"], case["buckets"], case["mult"], _dim(case)
        e = n * case["degree"]
        if case["edges"] == "random":                       # any order, nodes without edges among them
            dst = torch.randint(0, n, (e,), generator=g, device="cuda")
        else:
            dst = torch.arange(n, device="cuda").repeat_interleave(case["degree"])
        if case["edges"] == "chain":
            src = (dst + torch.randint(-case["degree"], case["degree"] + 1, (e,), generator=g, device="cuda")) % n
        else:
            src = torch.randint(0, n, (e,), generator=g, device="cuda")
        bounds = torch.linspace(0, MAX_DIST, b + 1, device="cuda")[1:-1].contiguous()
        dist = torch.rand(e, generator=g, device="cuda") * (MAX_DIST * 1.05)
        if b > 1:                                           # some edges exactly at a border
            at = torch.arange(0, e, 17, device="cuda")
            dist[at] = bounds[at % (b - 1)]
        bias = 0.5 * _randn(g, b, h)
        if case["cutoff"]:
            bias[-1] = float("-inf")
        shape = (dim, n, 2 * mult) if case["cm"] else (n, 2 * mult, dim)
        qk = _randn(g, *shape).to(dt)
        scale = torch.full((), math.log((mult // h * dim) ** -0.5), device="cuda")
        return dict(src=src, dst=dst, bounds=bounds, dist=dist, bias=bias.to(dt), qk=qk, log_scale=scale, seed=_seed(g),
                    gw=_randn(g, e, h).to(dt) if case["train"] else None)
    if case["kind"] == "dropout":
        r, mult, dim = case["rows"], case["mult"], _dim(case)
        shape = (dim, r, mult) if case["cm"] else (r, mult, dim)
        return dict(x=_randn(g, *shape).to(dt), seed=_seed(g), gy=_randn(g, *shape).to(dt) if case["train"] else None)
    d, r, x, reps = _dim(case), case["rows"], case["adapters"], case["lmax"] + 1
    ci, co, k = case["cin"], case["cout"], case["rank"]
    # structures of a batch lie together; some adapters have far more rows than others
    liking = torch.softmax(1.5 * _randn(g, x), 0)
    ids = torch.multinomial(liking, r, replacement=True, generator=g)
    if r > 64:
        ids = torch.sort(ids).values.roll(r // 3)
    pad = int(case["none"] * r)
    if pad:
        ids[r - pad:] = -1
    train = case["train"] != "no"
    return dict(ids=ids, x=_randn(g, d, r, ci).to(dt), weight=(_randn(g, reps, co, ci) / math.sqrt(ci)).to(dt),
                bias=(0.1 * _randn(g, co, 1)).to(dt), down=(_randn(g, x, reps, k, ci) / math.sqrt(ci)).to(dt),
                up=(_randn(g, x, reps, co, k) / math.sqrt(k)).to(dt), gy=_randn(g, d, r, co).to(dt) if train else None)


def _degrees(case):
    return list(range(case["lmax"] + 1))


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    kind = case["kind"]
    if own:
        fe = s["fe"] = _package()
        if kind == "attention":
            s["graph"] = fe.Graph(s["src"], s["dst"], case["nodes"])
            leaves = ("qk", "bias", "log_scale") if case["train"] else ()
        elif kind == "dropout":
            leaves = ("x",) if case["train"] else ()
        else:                                               # made once for all maps of a model
            s["plan"] = fe.ExpertPlan(s["ids"], case["adapters"])
            leaves = dict(no=(), adapters=("x", "down", "up"), all=("x", "down", "up", "weight", "bias"))[case["train"]]
        for name in leaves:
            s[name].requires_grad_()
        s["leaves"] = [s[name] for name in leaves]
    return s


# ---- one pass ----------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return dict(attention=_own_attention, dropout=_own_dropout, adapter=_own_adapter)[kind](s)
    return dict(attention=_plain_attention, dropout=_plain_dropout, adapter=_plain_adapter)[kind](s)


def _own_attention(s):
    fe, case = s["fe"], s["case"]

    def weights():
        buckets = fe.distance_buckets(s["dist"], s["bounds"])
        return buckets, fe.edge_attention_weights(
            s["qk"], s["graph"], case["heads"], s["log_scale"], component_major=case["cm"], bias=s["bias"], buckets=buckets,
            dropout=case["p"], seed=s["seed"])

    if not case["train"]:
        with torch.no_grad():
            buckets, w = weights()
        return dict(buckets=buckets, w=w)
    buckets, w = weights()
    gqk, gbias, gscale = torch.autograd.grad(w, s["leaves"], s["gw"])
    return dict(buckets=buckets, w=w.detach(), gqk=gqk, gbias=gbias, gscale=gscale)


def _own_dropout(s):
    fe, case = s["fe"], s["case"]
    args = (s["x"], case["p"], s["seed"], _degrees(case), case["cm"])
    if not case["train"]:
        with torch.no_grad():
            return dict(y=fe.feature_dropout(*args))
    y = fe.feature_dropout(*args)
    (gx,) = torch.autograd.grad(y, s["leaves"], s["gy"])
    return dict(y=y.detach(), gx=gx)


def _own_adapter(s):
    fe, case = s["fe"], s["case"]
    args = (s["x"], s["weight"], s["down"], s["up"], s["plan"], _degrees(case), s["bias"], ADAPTER_SCALE)
    if case["train"] == "no":
        with torch.no_grad():
            return dict(y=fe.adapter_linear(*args))
    y = fe.adapter_linear(*args)
    grads = torch.autograd.grad(y, s["leaves"], s["gy"])
    return dict(zip(("gx", "gdown", "gup", "gweight", "gbias"), grads), y=y.detach())


def _times(a, b):
    """The high and low 32 bits of the products of 32-bit numbers, held in 64 (a product's upper bits may wrap)."""
    p = a * b
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _plain_words(seed, blocks, device):
    """The generator's words (blocks, 4)."""
    b = torch.arange(blocks, device=device)
    c0, c1, c2, c3 = b & 0xFFFFFFFF, b >> 32, torch.zeros_like(b), torch.zeros_like(b)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):                                     # the generator's rounds
        h0, l0 = _times(c0, 0xD2511F53)
        h1, l1 = _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], 1)


def _plain_factors(seed, units, p):
    """0 or 1 / (1 - p) for every unit."""
    t = int(round(p * 65536))
    w = _plain_words(seed, (units + 7) // 8, seed.device)
    numbers = torch.stack([w & 0xFFFF, w >> 16], 2).view(-1)[:units]
    return (numbers >= t).float() * (65536.0 / (65536 - t))


def _plain_attention(s):
    case = s["case"]
    n, h, mult, dim = case["nodes"], case["heads"], case["mult"], _dim(case)
    e, dh, dt = s["src"].shape[0], mult // h * dim, s["qk"].dtype
    src, dst = s["src"], s["dst"]
    buckets = (s["bounds"][None, :] <= s["dist"][:, None]).sum(1)
    qk = s["qk"].float()
    if case["cm"]:
        qk = qk.permute(1, 2, 0)
    q, k = qk[:, :mult].reshape(n, h, dh)[dst], qk[:, mult:].reshape(n, h, dh)[src]
    scale = s["log_scale"].exp()
    dots = scale * (q * k).sum(-1)
    logits = dots + s["bias"].float()[buckets]
    at = dst[:, None].expand(e, h)
    top = torch.full((n, h), float("-inf"), device=qk.device).scatter_reduce(0, at, logits, "amax")
    top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
    w = (logits - top[dst]).exp()
    w = w / (torch.zeros(n, h, device=qk.device).index_add_(0, dst, w) + 1e-8)[dst]
    factors = _plain_factors(s["seed"], e * h, case["p"]).view(e, h) if case["p"] > 0 else None
    out = dict(buckets=buckets.int(), w=(w if factors is None else w * factors).to(dt))
    if not case["train"]:
        return out
    g = s["gw"].float() if factors is None else s["gw"].float() * factors
    gl = w * (g - torch.zeros(n, h, device=qk.device).index_add_(0, dst, w * g)[dst])
    gq = torch.zeros(n, h, dh, device=qk.device).index_add_(0, dst, (scale * gl)[..., None] * k)
    gk = torch.zeros(n, h, dh, device=qk.device).index_add_(0, src, (scale * gl)[..., None] * q)
    gqk = torch.cat([gq.view(n, mult, dim), gk.view(n, mult, dim)], 1)
    out["gqk"] = (gqk.permute(2, 0, 1).contiguous() if case["cm"] else gqk).to(dt)
    out["gbias"] = torch.zeros(case["buckets"], h, device=qk.device, dtype=torch.float64).index_add_(0, buckets, gl.double()).to(dt)
    out["gscale"] = (gl * dots).double().sum().float()
    return out


def _irreps(case):
    """The irrep of every component."""
    degree = torch.arange(_dim(case), device="cuda")
    return degree.double().sqrt().long()                    # exact: components l^2 .. (l + 1)^2 - 1 belong to degree l


def _plain_dropout(s):
    case = s["case"]
    r, mult, reps = case["rows"], case["mult"], case["lmax"] + 1
    factors = _plain_factors(s["seed"], r * mult * reps, case["p"]).view(r, mult, reps)[..., _irreps(case)]
    if case["cm"]:
        factors = factors.permute(2, 0, 1)
    out = dict(y=(s["x"].float() * factors).to(s["x"].dtype))
    if case["train"]:
        out["gx"] = (s["gy"].float() * factors).to(s["x"].dtype)
    return out


def _plain_adapter(s):
    """All rows through all adapters' maps at once, of which every row keeps its own."""
    case = s["case"]
    dt, train = s["x"].dtype, case["train"]
    adapters, k, rep = case["adapters"], case["rank"], _irreps(case)
    ci, co, dim, rows, reps = case["cin"], case["cout"], _dim(case), case["rows"], case["lmax"] + 1
    x, w = s["x"].float(), s["weight"].float()[rep]                         # (dim, rows, ci), (dim, co, ci)
    down = s["down"].float().permute(1, 0, 2, 3).reshape(reps, adapters * k, ci)[rep]      # (dim, adapters k, ci)
    up = s["up"].float().permute(1, 0, 3, 2).reshape(reps, adapters * k, co)[rep]          # (dim, adapters k, co)
    mine = (s["ids"][:, None] == torch.arange(adapters, device=x.device)).float().repeat_interleave(k, 1) * ADAPTER_SCALE
    low = torch.bmm(x, down.transpose(1, 2).contiguous()) * mine            # (dim, rows, adapters k)
    y = torch.bmm(x, w.transpose(1, 2).contiguous()) + torch.bmm(low, up)
    y[0] += s["bias"].float()[:, 0]
    out = dict(y=y.to(dt))
    if train == "no":
        return out
    g = s["gy"].float()
    glow = torch.bmm(g, up.transpose(1, 2).contiguous()) * mine
    out["gx"] = (torch.bmm(g, w) + torch.bmm(glow, down)).to(dt)
    of = (rep[None, :] == torch.arange(reps, device=x.device)[:, None]).float()            # (reps, dim)
    gdown = torch.bmm(glow.transpose(1, 2).contiguous(), x).view(dim, -1)
    out["gdown"] = (of @ gdown).view(reps, adapters, k, ci).permute(1, 0, 2, 3).contiguous().to(dt)
    gup = torch.bmm(g.transpose(1, 2).contiguous(), low).view(dim, -1)
    out["gup"] = (of @ gup).view(reps, co, adapters, k).permute(2, 0, 1, 3).contiguous().to(dt)
    if train == "all":
        gw = torch.bmm(g.transpose(1, 2).contiguous(), x).view(dim, -1)
        out["gweight"] = (of @ gw).view(reps, co, ci).to(dt)
        out["gbias"] = g[0].sum(0)[:, None].to(dt)
    return out


# ---- the definitions in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return dict(attention=_exact_attention, dropout=_exact_dropout, adapter=_exact_adapter)[case["kind"]](case, s)


def _leaf(t):
    return t.detach().double().requires_grad_()


def _exact_kept(seed, units, p, device):
    """Factors of the units, the generator on the host in pieces."""
    key = int(seed.item()) & (2 ** 64 - 1)
    limit = int(math.floor(p * 65536 + 0.5))
    factors = np.empty((units + 7) // 8 * 8)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for a in range(0, factors.size // 8, 1 << 16):
        blocks = np.arange(a, min(a + (1 << 16), factors.size // 8), dtype=np.uint64)
        x = [blocks & low, blocks >> half, np.zeros_like(blocks), np.zeros_like(blocks)]
        for i in range(10):
            k = [np.uint64((key + i * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((key >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)]
            u, v = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
            x = [(v >> half) ^ x[1] ^ k[0], v & low, (u >> half) ^ x[3] ^ k[1], u & low]
        numbers = np.stack(x, 1).astype("<u4").view("<u2")
        factors[8 * a:8 * (a + len(blocks))] = np.where(numbers.reshape(-1) < limit, 0.0, 65536.0 / (65536 - limit))
    return torch.from_numpy(factors[:units]).to(device)


def _exact_attention(case, s):
    """By autograd, one head after another."""
    n, h, mult, dim = case["nodes"], case["heads"], case["mult"], _dim(case)
    e, hc, dev = s["src"].shape[0], mult // h, s["qk"].device
    buckets = torch.from_numpy(np.searchsorted(s["bounds"].cpu().numpy(), s["dist"].cpu().numpy(), side="right")).to(dev)
    qk, bias, log_scale = _leaf(s["qk"]), _leaf(s["bias"]), _leaf(s["log_scale"])
    rows = qk.permute(1, 2, 0) if case["cm"] else qk
    kept = _exact_kept(s["seed"], e * h, case["p"], dev).view(e, h) if case["p"] > 0 else torch.ones(e, h, device=dev)
    out = torch.empty(e, h, dtype=torch.float64, device=dev)
    grads = [torch.zeros_like(t) for t in (qk, bias, log_scale)]
    with torch.set_grad_enabled(case["train"]):
        for j in range(h):
            q = rows[:, j * hc:(j + 1) * hc].reshape(n, hc * dim).index_select(0, s["dst"])
            k = rows[:, mult + j * hc:mult + (j + 1) * hc].reshape(n, hc * dim).index_select(0, s["src"])
            z = (q * k).sum(1) * torch.exp(log_scale) + bias[:, j].index_select(0, buckets)
            live = (z > float("-inf")).nonzero()[:, 0]
            z, to = z[live], s["dst"][live]
            top = torch.full((n,), float("-inf"), dtype=torch.float64, device=dev)
            top = top.scatter_reduce(0, to, z.detach(), "amax")
            u = torch.exp(z - top[to])
            total = torch.zeros(n, dtype=torch.float64, device=dev).scatter_add(0, to, u)
            w = torch.zeros(e, dtype=torch.float64, device=dev).scatter(0, live, u / (total[to] + 1e-8)) * kept[:, j]
            out[:, j] = w.detach()
            if case["train"]:
                for total_grad, d in zip(grads, torch.autograd.grad(w, [qk, bias, log_scale], s["gw"][:, j].double())):
                    total_grad += d
    found = dict(buckets=buckets.int(), w=out)
    if case["train"]:
        found.update(zip(("gqk", "gbias", "gscale"), grads))
    return found


def _exact_dropout(case, s):
    r, mult, reps = case["rows"], case["mult"], case["lmax"] + 1
    kept = _exact_kept(s["seed"], r * mult * reps, case["p"], s["x"].device).view(r, mult, reps)
    whole = torch.cat([kept[:, :, l:l + 1].expand(r, mult, 2 * l + 1) for l in range(reps)], 2)
    if case["cm"]:
        whole = whole.permute(2, 0, 1)
    out = dict(y=s["x"].double() * whole)
    if case["train"]:
        out["gx"] = s["gy"].double() * whole
    return out


def _exact_adapter(case, s):
    """Adapter by adapter and degree by degree, by autograd."""
    train = case["train"]
    names = [] if train == "no" else ["x", "down", "up"] if train == "adapters" else ["x", "down", "up", "weight", "bias"]
    t = {k: s[k].detach().double() for k in ("x", "down", "up", "weight", "bias")}
    grads = {k: torch.zeros_like(t[k]) for k in names}
    y = torch.empty(_dim(case), case["rows"], case["cout"], dtype=torch.float64, device=s["x"].device)
    for a in range(-1, case["adapters"]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        for l in range(case["lmax"] + 1):
            comps = torch.arange(l * l, (l + 1) ** 2, device=rows.device)
            x, w = t["x"][comps][:, rows].requires_grad_(), t["weight"][l].clone().requires_grad_()
            leaves = dict(x=x, weight=w)
            m = w
            if a >= 0:
                leaves["down"], leaves["up"] = t["down"][a, l].clone().requires_grad_(), t["up"][a, l].clone().requires_grad_()
                m = w + ADAPTER_SCALE * torch.mm(leaves["up"], leaves["down"])
            out = torch.mm(x.reshape(-1, case["cin"]), m.t()).view(len(comps), rows.numel(), case["cout"])
            if l == 0:
                leaves["bias"] = t["bias"][:, 0].clone().requires_grad_()
                out = out + leaves["bias"]
            y[comps[:, None], rows] = out.detach()
            wanted = [k for k in names if k in leaves]
            if not wanted:
                continue
            found = torch.autograd.grad(out, [leaves[k] for k in wanted], s["gy"][comps][:, rows].double())
            for k, d in zip(wanted, found):
                if k == "x":
                    grads[k][comps[:, None], rows] = d
                elif k == "weight":
                    grads[k][l] += d
                elif k == "bias":
                    grads[k][:, 0] += d
                else:
                    grads[k][a, l] += d
    return dict({"g" + k: v for k, v in grads.items()}, y=y)
