"""Dropout and biased edge attention (csrc/dropout.hip, edge_attention.hip) against the float64 oracle on the same
inputs.

u = 2^-24 (float32), HALF(t) half a step of the stored type t.  Float32 sums of n terms are off by at most n u of their
absolute terms; exp by 2 u and u times its exponent's size."""
import pytest
import torch

import flash_eq as fe
from oracle import finetune as OF

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, tol):
    got = got.detach()
    err = (got.double().cpu() - want.detach()).abs()
    bad = ~(err <= tol + TINY[got.dtype])
    assert not bad.any(), (float((err - tol).max()), int(bad.sum()), tuple(got.shape))


def seed_of(dev, value):
    return torch.tensor([value], dtype=torch.int64, device=dev)


# ---- dropout -----------------------------------------------------------------------------

def check_dropout(dev, shape, lvals, cm, p, dtype, seed, base=None):
    g = gen(seed)
    x, gy = torch.randn(*shape, generator=g).to(dtype), torch.randn(*shape, generator=g).to(dtype)
    want, gwant = (OF.dropout(t.double(), p, 1234567 - seed, lvals, cm) for t in (x, gy))
    xx = x.to(dev) if base is None else base(x.to(dev))
    xx.requires_grad_()
    y = fe.feature_dropout(xx, p, seed_of(dev, 1234567 - seed), lvals, cm)
    (gx,) = torch.autograd.grad(y, xx, gy.to(dev))
    assert y.shape == xx.shape and y.dtype == dtype
    for got, ref in ((y, want), (gx, gwant)):
        assert torch.equal(got.detach().cpu() == 0, ref == 0)                   # the same units
        within(got, ref, (HALF[dtype] + 2 * U) * ref.abs())                     # the scale, the product, the stored type
    with torch.no_grad():
        assert torch.equal(fe.feature_dropout(xx, p, seed_of(dev, 1234567 - seed), lvals, cm), y)


LVALS = [[0], [0, 1], [0, 1, 2], [1], [0, 0, 1, 3], [2, 2], list(range(7)), [0] * 5, [0] * 32, [15], [6, 6, 6, 6, 6, 6, 6, 6, 6, 5]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cm", [False, True])
@pytest.mark.parametrize("lvals", LVALS)
def test_dropout_irreps(dev, lvals, cm, dtype):
    dim = sum(2 * l + 1 for l in lvals)
    for rows, mult, p in ((1, 1, 0.5), (3, 5, 0.25), (37, 7, 0.1), (64, 16, 0.9)):
        shape = (dim, rows, mult) if cm else (rows, mult, dim)
        check_dropout(dev, shape, lvals, cm, p, dtype, rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2049, 20011])
def test_dropout_elements(dev, n, dtype):
    check_dropout(dev, (n,), None, False, 0.3, dtype, n)


def test_dropout_of_several_tiles(dev):
    check_dropout(dev, (411, 9, 9), [0, 1, 2], False, 0.2, torch.float32, 1)
    check_dropout(dev, (9, 411, 9), [0, 1, 2], True, 0.2, torch.bfloat16, 2)


def test_dropout_shares_at_the_ends(dev):
    x = torch.randn(50, 4, 4, generator=gen(0)).to(dev)
    x[0] = NAN
    x[1] = INF
    s = seed_of(dev, 5)
    assert torch.equal(fe.feature_dropout(x[1:], 0.0, s, [0, 1]), x[1:])
    assert torch.equal(fe.feature_dropout(x, 1.0, s, [0, 1]), torch.zeros_like(x))
    y = fe.feature_dropout(x, 0.5, s, [0, 1])
    f = OF.factors(5, 50 * 4 * 2, 0.5).view(50, 4, 2)[..., [0, 1, 1, 1]].to(dev)
    assert (y[f == 0] == 0).all() and y[0][f[0] > 0].isnan().all() and y[1][f[1] > 0].isinf().all()
    assert torch.equal(fe.feature_dropout(x[1:], 2.0 ** -18, s), x[1:])           # less than half a 65536th


def test_dropout_views_and_no_rows(dev):
    check_dropout(dev, (33, 6, 4), [0, 1], False, 0.4, torch.float32, 3, lambda t: t.permute(2, 0, 1).contiguous().permute(1, 2, 0))
    check_dropout(dev, (33, 6, 4), [0, 1], False, 0.4, torch.bfloat16, 4,          # two bytes off every vector
                  lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape).detach())
    check_dropout(dev, (4, 33, 7), [0, 1], True, 0.4, torch.float16, 5,
                  lambda t: torch.cat([t.new_zeros(3), t.reshape(-1)])[3:].view(t.shape).detach())
    check_dropout(dev, (5, 6, 3, 4), [0, 1], False, 0.4, torch.float32, 6)
    x = torch.zeros(0, 4, 4, device=dev, requires_grad=True)
    y = fe.feature_dropout(x, 0.5, seed_of(dev, 1), [0, 1])
    assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


def test_dropout_units_past_32_bits(dev):
    """The last elements of a table of more than 2^32 of them (bfloat16: 8.6 GB): their numbers are those of their
    units, formed on the host."""
    n = 2 ** 32 + 24
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    y = fe.feature_dropout(x, 0.5, seed_of(dev, 77))
    words = [w for b in range(2 ** 29 - 1, 2 ** 29 + 3) for w in OF.philox((b, 0, 0, 0), (77, 0))]
    want = [2.0 * (v >= 32768) for w in words for v in (w & 0xFFFF, w >> 16)]
    assert y[-32:].tolist() == want
    del x, y
    torch.cuda.empty_cache()


def test_dropout_expanded_gradient_second_backward_and_changed_seed(dev):
    x = torch.randn(40, 3, 4, generator=gen(1)).to(dev).requires_grad_()
    s = seed_of(dev, 3)
    y = fe.feature_dropout(x, 0.5, s, [0, 1])
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)                    # an expanded gradient
    assert torch.equal(gx.detach().cpu().double(), OF.dropout(torch.ones(40, 3, 4, dtype=torch.float64), 0.5, 3, [0, 1]))
    with pytest.raises(RuntimeError, match="no second derivative"):
        gx.sum().backward()
    y = fe.feature_dropout(x, 0.5, s, [0, 1])
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_seeds(dev):
    torch.manual_seed(5)
    a = [fe.dropout_seed(dev).item() for _ in range(4)]
    torch.manual_seed(5)
    assert a == [fe.dropout_seed(dev).item() for _ in range(4)] and len(set(a)) == 4


# ---- edge attention ----------------------------------------------------------------------

def sums(n, idx, v):
    """v summed by index, those outside [0, n) left out."""
    inside = (idx >= 0) & (idx < n)
    return torch.zeros(n, *v.shape[1:], dtype=v.dtype).index_add_(0, idx[inside], v[inside])


def check_attention(dev, src, dst, nodes, heads, mult, dim, dtype, *, cm=False, edge_form=False, buckets=0, p=0.0, decay=0.0, seed=0,
                    bias_type=None, wide=False, bias_edit=None, leaves=("qk", "log_scale", "bias", "dist")):
    g = gen(seed + 100)
    E, Dh, H = src.shape[0], mult // heads * dim, heads
    if edge_form:
        tables = [torch.randn(E, H, Dh, generator=g).to(dtype) for _ in range(2)]
    else:
        tables = [torch.randn(*((dim, nodes, 2 * mult) if cm else (nodes, 2 * mult, dim)), generator=g).to(dtype)]
    ls = torch.tensor(float(torch.log(torch.tensor(1.5 * Dh ** -0.5))))
    bias = bucket = dist = None
    if buckets:
        bias = torch.randn(buckets, H, generator=g).to(bias_type or dtype)
        if bias_edit:
            bias_edit(bias)
        bucket = torch.randint(-1, buckets + 1, (E,), generator=g)              # some outside the table
        if wide and E:
            bucket[0] = 2 ** 32
    if decay:
        dist = torch.rand(E, generator=g) * 10
    gw = torch.randn(E, H, generator=g).to(dtype)

    # the oracle
    t64 = [t.double().requires_grad_() for t in tables]
    ls64 = ls.double().requires_grad_()
    b64 = bias.double().requires_grad_() if buckets else None
    d64 = dist.double().requires_grad_() if decay else None
    q, k = t64 if edge_form else OF.node_qk(t64[0], H, src, dst, cm)
    q, k = (t.detach().requires_grad_() for t in (q, k))
    w = OF.edge_attention(q, k, dst, nodes, ls64, d64, decay, b64, bucket, p, seed + 17)
    plain = OF.edge_attention(q, k, dst, nodes, ls64, d64, decay, b64, bucket).detach()
    named = {"q": q, "k": k, "log_scale": ls64, "bias": b64, "dist": d64}
    named = {n: t for n, t in named.items() if t is not None}
    grads = dict(zip(named, torch.autograd.grad(w, list(named.values()), gw.double(), allow_unused=True)))
    grads = {n: torch.zeros_like(named[n]) if v is None else v for n, v in grads.items()}

    # the framework
    tt = [t.to(dev).requires_grad_("qk" in leaves) for t in tables]
    lsd = ls.to(dev).requires_grad_("log_scale" in leaves)
    bd = bias.to(dev).requires_grad_("bias" in leaves) if buckets else None
    dd = dist.to(dev).requires_grad_("dist" in leaves) if decay else None
    graph = fe.Graph(src.to(dev), dst.to(dev), nodes)
    args = dict(distances=dd, decay=decay, bias=bd, buckets=(bucket if wide else bucket.int()).to(dev) if buckets else None, dropout=p,
                seed=seed_of(dev, seed + 17) if p else None)

    def run():
        if edge_form:
            return fe.edge_attention_weights_qk(tt[0], tt[1], graph, lsd, **args)
        return fe.edge_attention_weights(tt[0], graph, H, lsd, component_major=cm, **args)

    got = run()
    assert got.shape == (E, H) and got.dtype == dtype
    wanted = [t for t in (*tt, lsd, bd, dd) if t is not None and t.requires_grad]
    found = {id(t): v for t, v in zip(wanted, torch.autograd.grad(got, wanted, gw.to(dev)))} if wanted else {}

    # bounds: the dot product's, the logit's, the weight's relative one, the logit gradient's
    qd, kd = q.detach(), k.detach()
    scale = float(ls64.detach().exp())
    size = scale * (qd * kd).abs().sum(-1)
    z = scale * (qd * kd).sum(-1)
    extra = torch.zeros_like(z)
    if buckets:
        known = (bucket >= 0) & (bucket < buckets)
        b = torch.where(known[:, None], b64.detach()[bucket.clamp(0, buckets - 1)], torch.zeros_like(z))
        extra = extra + b
    if decay:
        extra = extra - d64.detach()[:, None] / decay
    live = (extra > -INF) & ((dst >= 0) & (dst < nodes))[:, None]
    total = torch.where(live, z + extra, torch.zeros_like(z))
    fine = torch.where(live, extra, torch.zeros_like(z))
    ez = torch.where(live, U * ((2 * Dh + 8) * size + 4 * z.abs() + 8 * fine.abs() + 4 * total.abs()), torch.zeros_like(z))
    safe = dst.clamp(0, nodes - 1)
    at = safe[:, None].expand(E, H)
    low = torch.full((nodes, H), -1e300, dtype=torch.float64)
    top = low.scatter_reduce(0, at, torch.where(live, total, torch.full_like(total, -1e300)), "amax") if E else low
    worst = torch.zeros(nodes, H, dtype=torch.float64).scatter_reduce(0, at, ez, "amax") if E else low
    deg = sums(nodes, dst, torch.ones(E, 1, dtype=torch.float64)) if E else torch.zeros(nodes, 1, dtype=torch.float64)
    span = torch.where(live, (top[safe] - total).clamp(0, 110), torch.zeros_like(total))
    rel = ez + worst[safe] + U * (2 * span + deg[safe] + 32)
    floor = 2.0 ** -120                       # below the smallest normal number exp may flush to 0
    f = OF.factors(seed + 17, E * H, p).view(E, H) if p else torch.ones(E, H, dtype=torch.float64)
    within(got, w, (rel + HALF[dtype] + 2 * U) * w.detach().abs() + floor)
    assert torch.equal(got.detach().cpu()[~live], torch.zeros(int((~live).sum()), dtype=dtype))
    gg = gw.double() * f
    dot = sums(nodes, dst, plain * gg)[safe] if E else gg
    mass = sums(nodes, dst, plain * gg.abs())[safe] if E else gg
    gz = plain * (gg - dot)
    ego = sums(nodes, dst, plain * gg.abs() * (rel + (deg[safe] + 8) * U))[safe] if E else gg
    egz = plain * ((rel + 6 * U) * (gg.abs() + mass) + ego) + floor * (1 + gg.abs() + mass)
    half = HALF[dtype]
    gdeg = deg[safe][:, :, None]
    tq = scale * (egz[..., None] * kd.abs() + (gdeg + 8) * U * (gz[..., None] * kd).abs())
    odeg = sums(nodes, src, torch.ones(E, 1, dtype=torch.float64))[src.clamp(0, nodes - 1)][:, :, None] if E else gdeg
    tk = scale * (egz[..., None] * qd.abs() + (odeg + 8) * U * (gz[..., None] * qd).abs())
    if edge_form:
        pairs = [(tt[0], grads["q"], tq), (tt[1], grads["k"], tk)]
    else:
        def table(a, b):
            a, b = (sums(nodes, i, v).view(nodes, mult, dim) for i, v in ((dst, a), (src, b)))
            both = torch.cat([a, b], 1)
            return both.permute(2, 0, 1) if cm else both
        pairs = [(tt[0], table(grads["q"], grads["k"]), table(tq, tk))]
    for leaf, want, tol in pairs:
        if leaf.requires_grad:
            within(found[id(leaf)], want, tol + half * want.abs())
    if lsd.requires_grad:
        most = float(deg.max()) if E else 0.0
        tol = (egz * size + gz.abs() * size * U * (2 * Dh + most + 40)).sum()
        within(found[id(lsd)], grads["log_scale"], tol + U * grads["log_scale"].abs())
    if buckets and bd.requires_grad:
        count = sums(buckets, bucket, torch.ones(E, 1, dtype=torch.float64))
        tol = sums(buckets, bucket, egz) + (count + 16) * U * sums(buckets, bucket, gz.abs())
        within(found[id(bd)], grads["bias"], tol + HALF[bd.dtype] * grads["bias"].abs())
    if decay and dd.requires_grad:
        tol = (egz + (H + 6) * U * gz.abs()).sum(1) / decay
        within(found[id(dd)], grads["dist"], tol)
    with torch.no_grad():
        assert torch.equal(run(), got)
    return got


def random_graph(seed, nodes, edges):
    g = gen(seed)
    return torch.randint(0, nodes, (edges,), generator=g), torch.randint(0, nodes, (edges,), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,mult,dim", [(1, 1, 1), (1, 3, 4), (2, 6, 9), (3, 9, 4), (4, 32, 4), (8, 64, 9), (8, 8, 49), (16, 32, 1),
                                            (17, 34, 4), (1, 40, 49), (5, 35, 9), (33, 33, 3), (2, 160, 49)])
def test_attention_heads(dev, heads, mult, dim, dtype):
    src, dst = random_graph(heads, 23, 150)
    for cm in (False, True):
        check_attention(dev, src, dst, 23, heads, mult, dim, dtype, cm=cm, buckets=7, seed=heads)
    if mult * dim < 400:
        check_attention(dev, src, dst, 23, heads, mult, dim, dtype, edge_form=True, buckets=7, p=0.25, seed=heads)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long_heads(dev, dtype):
    """Heads of several slices."""
    src, dst = random_graph(2, 9, 40)
    for cm in (False, True):
        check_attention(dev, src, dst, 9, 1, 131, 49, dtype, cm=cm, buckets=3, p=0.1)
    check_attention(dev, src, dst, 9, 2, 512, 9, dtype, buckets=3)


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5])
@pytest.mark.parametrize("nodes,edges", [(1, 1), (1, 300), (2, 5), (300, 40), (40, 2000), (7, 3000)])
def test_attention_graphs(dev, nodes, edges, p):
    src, dst = random_graph(nodes, nodes, edges)
    check_attention(dev, src, dst, nodes, 4, 16, 4, torch.float32, buckets=20, p=p, decay=3.0, seed=edges)
    check_attention(dev, src, dst, nodes, 2, 16, 4, torch.bfloat16, cm=True, buckets=1, p=p, seed=edges)


def test_attention_without_a_bias_decay_alone_and_types(dev):
    src, dst = random_graph(3, 20, 100)
    check_attention(dev, src, dst, 20, 4, 16, 9, torch.float32)
    check_attention(dev, src, dst, 20, 4, 16, 9, torch.float32, decay=2.0, p=0.3)
    check_attention(dev, src, dst, 20, 4, 16, 9, torch.bfloat16, buckets=6, bias_type=torch.float32, wide=True)
    check_attention(dev, src, dst, 20, 4, 16, 9, torch.float32, buckets=6, bias_type=torch.float16, wide=True)


@pytest.mark.parametrize("leaves", [("qk",), ("bias",), ("log_scale",), ("dist",), ("bias", "dist"), ()])
def test_attention_gradients_one_by_one(dev, leaves):
    src, dst = random_graph(4, 20, 100)
    for edge_form in (False, True):
        check_attention(dev, src, dst, 20, 4, 16, 9, torch.float32, buckets=6, decay=2.0, p=0.2, leaves=leaves, edge_form=edge_form)


def test_attention_edges_outside_the_graph(dev):
    src, dst = random_graph(5, 20, 200)
    src[::7], src[3] = -1, 20
    dst[::11], dst[4] = 20, -3
    for cm in (False, True):
        check_attention(dev, src, dst, 20, 4, 16, 9, torch.float32, cm=cm, buckets=6, p=0.2, decay=1.5)
    check_attention(dev, src, dst, 20, 4, 16, 9, torch.float32, edge_form=True, buckets=6)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_forbidden_buckets(dev, dtype):
    src, dst = random_graph(6, 60, 150)          # few edges a node: some have forbidden ones alone

    def edit(b):
        b[0] = -INF
        b[1, 0] = -INF
        b[2] = torch.finfo(b.dtype).min          # masked by the type's lowest value instead
        b[3] = -INF
    for cm in (False, True):
        check_attention(dev, src, dst, 60, 2, 8, 4, dtype, cm=cm, buckets=5, bias_edit=edit, p=0.25)
    check_attention(dev, src, dst, 60, 2, 8, 4, dtype, buckets=5, bias_edit=lambda b: b.fill_(-INF))
    check_attention(dev, src, dst, 60, 2, 8, 4, dtype, edge_form=True, buckets=5, bias_edit=edit)


def test_attention_nan_and_infinity_in_masked_places(dev):
    """What a forbidden edge's key, a dropped or zero weight's gradient and a query without edges hold reaches nothing."""
    g = gen(7)
    nodes, E, H = 30, 200, 2
    src, dst = torch.randint(0, nodes - 2, (E,), generator=g), torch.randint(0, nodes - 1, (E,), generator=g)
    bucket = torch.randint(0, 3, (E,), generator=g)
    bucket[src == 5] = 3                                             # every edge from node 5 is forbidden
    bias = torch.randn(4, H, generator=g)
    bias[3] = -INF
    qk = torch.randn(nodes, 8, 4, generator=g)
    gw = torch.randn(E, H, generator=g)
    graph = fe.Graph(src.to(dev), dst.to(dev), nodes)
    ls = torch.zeros((), device=dev)

    def run(qk, gw):
        a, b, s = qk.to(dev).requires_grad_(), bias.to(dev).requires_grad_(), ls.clone().requires_grad_()
        w = fe.edge_attention_weights(a, graph, H, s, bias=b, buckets=bucket.to(dev), dropout=0.25, seed=seed_of(dev, 3))
        return (w, *torch.autograd.grad(w, [a, b, s], gw.to(dev)))

    clean = run(qk, gw)
    bad, gbad = qk.clone(), gw.clone()
    bad[5, 4:] = NAN
    bad[nodes - 1, :4] = INF                                         # no edge reaches the last node
    bad[nodes - 1, 4:] = NAN                                         # none leaves the last two
    gbad[bucket == 3] = NAN
    f = OF.factors(3, E * H, 0.25).view(E, H)
    gbad[f == 0] = INF
    for a, b in zip(clean, run(bad, gbad)):
        assert torch.equal(a, b)
    bad = qk.clone()
    bad[2, 0, 0] = NAN                                               # a query in use: its node's first head, and its keys' gradients
    w = run(bad, gw)[0].cpu()
    hit = dst == 2
    kept = f > 0
    assert w[hit, 0][kept[hit, 0]].isnan().all() and torch.equal(w[~hit], clean[0].cpu()[~hit]) and torch.equal(w[:, 1], clean[0].cpu()[:, 1])


def test_attention_views_and_expanded_gradients(dev):
    src, dst = random_graph(8, 20, 100)
    graph = fe.Graph(src.int().to(dev), dst.int().to(dev), 20)
    g = gen(8)
    base = torch.randn(20, 16, 9, generator=g).to(dev)
    bias, bucket = torch.randn(6, 4, generator=g).to(dev), torch.randint(0, 6, (100,), generator=g).to(dev)
    ls = torch.zeros((), device=dev)

    def run(qk, b, k, cm=False, gw=None):
        qk, b = qk.detach().requires_grad_(), b.detach().requires_grad_()
        w = fe.edge_attention_weights(qk, graph, 4, ls, component_major=cm, bias=b, buckets=k)
        return (w.detach(), *torch.autograd.grad(w, [qk, b], torch.ones_like(w[:1, :1]).expand_as(w) if gw is None else gw))

    want = run(base, bias, bucket)
    strided = base.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    wide = torch.randn(6, 8, device=dev)
    wide[:, ::2] = bias
    offset = torch.cat([base.new_zeros(1), base.reshape(-1)])[1:].view(base.shape)
    for got in (run(strided, wide[:, ::2], bucket), run(offset, bias, bucket.repeat_interleave(2)[::2]),
                run(base, bias, bucket, gw=torch.ones(4, 100, device=dev).t())):
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    got = run(base.permute(2, 0, 1), bias, bucket, cm=True)          # other vectors, another order of the sums
    # a dot product of 36 terms (log_scale 0) is off by 80 u of its absolute terms, a weight by twice that, either way
    most = base.abs().max().item()
    size = base.abs().sum((1, 2)).max().item() / 8 * most
    assert ((got[0] - want[0]).abs() <= 4 * 80 * U * size * want[0]).all()
    # gradients of ones: grad_z = w (1 - sum w) is rounding alone, at most w (110 u + 1e-8) for up to 100 edges; the weights
    # into a node sum to 1, those out of one to at most its edges, and a bucket's to at most its edges
    out = torch.bincount(src).max().item()
    for a, b, terms in ((got[1].permute(1, 2, 0), want[1], most * out), (got[2], want[2], torch.bincount(bucket).max().item())):
        assert (a - b).abs().max() <= 2 * terms * (110 * U + 1e-8)


def test_attention_no_edges(dev):
    empty = torch.zeros(0, dtype=torch.int64, device=dev)
    graph = fe.Graph(empty, empty, 4)
    qk = torch.randn(4, 8, 4, device=dev, requires_grad=True)
    bias, ls = torch.randn(3, 2, device=dev, requires_grad=True), torch.zeros((), device=dev, requires_grad=True)
    w = fe.edge_attention_weights(qk, graph, 2, ls, bias=bias, buckets=empty, dropout=0.5, seed=seed_of(dev, 1))
    assert w.shape == (0, 2)
    for t, v in zip((qk, bias, ls), torch.autograd.grad(w.sum(), [qk, bias, ls])):
        assert torch.equal(v, torch.zeros_like(t))


@pytest.mark.parametrize("buckets,heads", [(1, 1), (100, 8), (512, 3), (1000, 16), (4096, 1), (4096, 5), (300, 70)])
def test_attention_bias_sizes(dev, buckets, heads):
    src, dst = random_graph(buckets, 50, 4000)
    check_attention(dev, src, dst, 50, heads, heads, 4, torch.float32, buckets=buckets, leaves=("bias",))


def test_attention_bias_gradient_of_one_bucket(dev):
    """All edges in one bucket."""
    src, dst = random_graph(9, 50, 5000)
    g = gen(9)
    qk = torch.randn(50, 8, 4, generator=g).to(dev)
    bias = torch.zeros(64, 4, device=dev, requires_grad=True)
    gw = torch.randn(5000, 4, generator=g).to(dev)
    w = fe.edge_attention_weights(qk, fe.Graph(src.to(dev), dst.to(dev), 50), 4, torch.zeros((), device=dev), bias=bias,
                                  buckets=torch.full((5000,), 7, dtype=torch.int32, device=dev))
    (gb,) = torch.autograd.grad(w, bias, gw)
    keep = torch.arange(64, device=dev) != 7
    assert (gb[keep] == 0).all()
    # a constant added to all logits changes nothing: the sum vanishes but for rounding, whose scale its terms set
    ww, gg = w.detach().double(), gw.double()
    assert (gb[7].double().abs() <= 5000 * U * 8 * (ww * gg.abs()).sum(0) + 1e-12).all()


def test_attention_changed_buffers_and_second_backward(dev):
    src, dst = random_graph(10, 20, 60)
    graph = fe.Graph(src.to(dev), dst.to(dev), 20)
    qk = torch.randn(20, 8, 4, device=dev, requires_grad=True)
    ls = torch.zeros((), device=dev)
    w = fe.edge_attention_weights(qk, graph, 2, ls)
    (g,) = torch.autograd.grad(w.sum(), qk, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()
    w = fe.edge_attention_weights(qk, graph, 2, ls)
    w.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        w.sum().backward()
    w = fe.edge_attention_weights(qk, graph, 2, ls)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()
    w = fe.edge_attention_weights(qk, graph, 2, ls, dropout=0.5, seed=seed_of(dev, 1))     # its weights are its own
    (w * 2).sum().backward()


def test_attention_is_deterministic(dev):
    src, dst = random_graph(11, 500, 20000)
    g = gen(11)
    qk = torch.randn(500, 32, 9, generator=g).to(dev).requires_grad_()
    bias = torch.randn(40, 4, generator=g).to(dev).requires_grad_()
    ls = torch.zeros((), device=dev, requires_grad=True)
    bucket = torch.randint(0, 40, (20000,), generator=g).to(dev)
    gw = torch.randn(20000, 4, generator=g).to(dev)
    graph = fe.Graph(src.to(dev), dst.to(dev), 500)
    runs = []
    for _ in range(3):
        w = fe.edge_attention_weights(qk, graph, 4, ls, bias=bias, buckets=bucket, dropout=0.1, seed=seed_of(dev, 5))
        runs.append((w.detach(), *torch.autograd.grad(w, [qk, bias, ls], gw)))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)


def test_buckets(dev):
    g = gen(12)
    for n in (0, 1, 2, 31, 32, 99, 4095):
        bounds = torch.sort(torch.rand(n, generator=g) * 10).values
        dist = torch.rand(3000, generator=g) * 12 - 1
        if n:
            dist[::3] = bounds[torch.randint(0, n, (1000,), generator=g)]      # exactly at a border
        dist[5], dist[7], dist[11] = NAN, INF, -INF
        got = fe.distance_buckets(dist.to(dev), bounds.to(dev))
        want = torch.searchsorted(bounds, dist, right=True)
        want[5] = 0
        assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)
    assert fe.distance_buckets(torch.zeros(0, device=dev), torch.zeros(3, device=dev)).shape == (0,)


# ---- streams and graphs ------------------------------------------------------------------

def test_step_on_another_stream(dev):
    src, dst = random_graph(13, 100, 1000)
    g = gen(13)
    qk0, bias = torch.randn(100, 32, 9, generator=g).to(dev), torch.randn(8, 4, generator=g).to(dev)
    bucket = torch.randint(0, 8, (1000,), generator=g).to(dev)
    graph = fe.Graph(src.to(dev), dst.to(dev), 100)

    def step():
        qk, b = qk0.clone().requires_grad_(), bias.clone().requires_grad_()
        x = fe.feature_dropout(qk, 0.2, seed_of(dev, 8), [0, 1, 2])
        w = fe.edge_attention_weights(x, graph, 4, torch.zeros((), device=dev), bias=b, buckets=bucket, dropout=0.1, seed=seed_of(dev, 9))
        return torch.autograd.grad(w.square().sum(), [qk, b])

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_step_draws_new_masks(dev):
    """A captured step draws another seed on every replay; each replay gives what an eager step with its seed does."""
    src, dst = random_graph(14, 100, 1000)
    g = gen(14)
    qk = torch.randn(100, 32, 9, generator=g).to(dev).requires_grad_()
    bias = torch.randn(8, 4, generator=g).to(dev).requires_grad_()
    bucket = torch.randint(0, 8, (1000,), generator=g).to(dev)
    graph = fe.Graph(src.to(dev), dst.to(dev), 100)
    graph.csr(), graph.csr_src()
    ls = torch.zeros((), device=dev)
    seen = torch.zeros(1, dtype=torch.int64, device=dev)

    def step(seed=None):
        s = fe.dropout_seed(dev) if seed is None else seed
        if seed is None:
            seen.copy_(s)
        w = fe.edge_attention_weights(fe.feature_dropout(qk, 0.2, s, [0, 1, 2]), graph, 4, ls, bias=bias, buckets=bucket, dropout=0.1, seed=s)
        loss = w.square().sum(1)
        loss.backward(torch.ones_like(loss))
        return w

    from flash_eq.capture import capture_step
    cuda_graph, w = capture_step(step, [qk, bias])
    seeds = []
    for _ in range(4):
        cuda_graph.replay()
        torch.cuda.synchronize()
        seeds.append(seen.item())
        got = [t.detach().clone() for t in (w, qk.grad, bias.grad)]
        q2, b2 = qk.detach().clone().requires_grad_(), bias.detach().clone().requires_grad_()
        s = seed_of(dev, seeds[-1])
        ww = fe.edge_attention_weights(fe.feature_dropout(q2, 0.2, s, [0, 1, 2]), graph, 4, ls, bias=b2, buckets=bucket, dropout=0.1, seed=s)
        loss = ww.square().sum(1)
        for a, b in zip(got, (ww.detach(), *torch.autograd.grad(loss, [q2, b2], torch.ones_like(loss)))):
            assert torch.equal(a, b)
    assert len(set(seeds)) == 4


# ---- large tables, several threads ---------------------------------------------------------

@pytest.mark.parametrize("cm", [False, True])
def test_attention_offsets_past_32_bits(dev, cm):
    """The last nodes of a table of more than 4 GB (float32, 9 components, 64 channels).  Queries and keys are 0 and +-1
    and a node has two edges either way, so every sum is one of whole numbers or of two terms and has the same bits
    in a small table of these nodes alone."""
    n, far, heads = 2_000_003, 500, 4
    first = n - far
    i = torch.arange(far)
    src, dst = torch.cat([i, i]), torch.cat([(i + 1) % far, (i + 2) % far])
    g = gen(21)
    small = torch.randint(-1, 2, (far, 64, 9), generator=g).float()
    bias = torch.randn(5, heads, generator=g)
    bucket = torch.randint(0, 5, (2 * far,), generator=g).int().to(dev)
    gw = torch.randn(2 * far, heads, generator=g).to(dev)
    ls = torch.tensor(0.125).log().to(dev)

    def run(qk, s, d, nodes):
        qk.requires_grad_()
        b = bias.to(dev).requires_grad_()
        graph = fe.Graph(s.to(dev), d.to(dev), nodes)
        w = fe.edge_attention_weights(qk, graph, heads, ls, component_major=cm, bias=b, buckets=bucket, dropout=0.25, seed=seed_of(dev, 4))
        return w.detach(), *torch.autograd.grad(w, [qk, b], gw)

    at = small.to(dev)
    big = torch.zeros((9, n, 64) if cm else (n, 64, 9), device=dev)
    if cm:
        big[:, first:] = at.permute(2, 0, 1)
    else:
        big[first:] = at
    w, gq, gb = run(big, src + first, dst + first, n)
    w1, gq1, gb1 = run(at.permute(2, 0, 1).contiguous() if cm else at, src, dst, far)
    near, rest = (gq[:, first:], gq[:, :first]) if cm else (gq[first:], gq[:first])
    assert torch.equal(w, w1) and torch.equal(near, gq1) and torch.equal(gb, gb1)
    assert not rest.any() and gq1.any()
    del big, gq, near, rest
    torch.cuda.empty_cache()


def test_calls_of_several_threads(dev):
    """Threads with streams of their own at once: each gets what it gets alone."""
    import threading
    src, dst = random_graph(15, 300, 4000)
    g = gen(15)
    qk0, bias = torch.randn(300, 32, 9, generator=g).to(dev), torch.randn(8, 4, generator=g).to(dev)
    bucket = torch.randint(0, 8, (4000,), generator=g).to(dev)
    graph = fe.Graph(src.to(dev), dst.to(dev), 300)
    graph.csr(), graph.csr_src()
    ls = torch.zeros((), device=dev)
    plan = fe.ExpertPlan(torch.randint(0, 3, (300,), generator=g).to(dev), 3)
    maps = [torch.randn(*s, generator=g).to(dev) for s in ((3, 32, 32), (3, 3, 4, 32), (3, 3, 32, 4))]

    def step(n):
        leaves = [t.clone().requires_grad_() for t in (qk0, bias, *maps)]
        x = fe.feature_dropout(leaves[0], 0.2, seed_of(dev, n), [0, 1, 2])
        y = fe.adapter_linear(x.permute(2, 0, 1), *leaves[2:], plan, [0, 1, 2])
        w = fe.edge_attention_weights(y, graph, 4, ls, component_major=True, bias=leaves[1], buckets=bucket, dropout=0.1, seed=seed_of(dev, n + 9))
        return torch.autograd.grad(w.square().sum(), leaves)

    want = [step(n) for n in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[n] = step(n)
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # for the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_captured_steps_replayed_in_turn(dev):
    """Two captured steps, replayed in turn and one after the other, each with the eager result."""
    from flash_eq.capture import capture_step
    g = gen(16)
    ls = torch.zeros((), device=dev)
    steps = []
    for nodes, edges in ((100, 900), (250, 4000)):
        src, dst = random_graph(nodes, nodes, edges)
        qk, bias = torch.randn(nodes, 32, 9, generator=g).to(dev).requires_grad_(), torch.randn(8, 4, generator=g).to(dev).requires_grad_()
        bucket = torch.randint(0, 8, (edges,), generator=g).to(dev)
        graph = fe.Graph(src.to(dev), dst.to(dev), nodes)
        graph.csr(), graph.csr_src()
        seed = seed_of(dev, nodes)

        def step(qk=qk, bias=bias, bucket=bucket, graph=graph, seed=seed):
            w = fe.edge_attention_weights(qk, graph, 4, ls, bias=bias, buckets=bucket, dropout=0.1, seed=seed)
            loss = w.square().sum(1)
            loss.backward(torch.ones_like(loss))
            return w

        q2, b2 = qk.detach().clone().requires_grad_(), bias.detach().clone().requires_grad_()
        w = fe.edge_attention_weights(q2, graph, 4, ls, bias=b2, buckets=bucket, dropout=0.1, seed=seed)
        loss = w.square().sum(1)
        want = [w.detach().clone(), *torch.autograd.grad(loss, [q2, b2], torch.ones_like(loss))]
        del w, loss, q2, b2
        cuda_graph, out = capture_step(step, [qk, bias])
        steps.append((cuda_graph, out, qk, bias, want, step))       # the graph reads the step's tensors
    for order in ((0, 1), (1, 0), (0, 0, 1), (1, 1)):
        for i in order:
            steps[i][0].replay()
        torch.cuda.synchronize()
        for i in set(order):
            _, out, qk, bias, want, _ = steps[i]
            assert all(torch.equal(a.detach(), b) for a, b in zip((out, qk.grad, bias.grad), want))
