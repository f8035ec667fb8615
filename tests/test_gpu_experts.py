"""Expert routing kernels (csrc/expert_route.hip, expert_rows.hip, expert_linear.hip) against the float64
oracle on the same inputs.

u = 2^-24 (float32), h(t) half a step of the stored type t.  Whole numbers and moved rows are exact.
Float32 sums of n terms are off by at most n u of their absolute terms; the matrix cores' sums are
counted twice (2 n u), for the steps inside an instruction."""
import pytest
import torch

import flash_eq as fe
from oracle import experts as OE

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, tol):
    err = (got.detach().double().cpu() - want).abs()
    bad = ~(err <= tol + TINY[got.dtype])
    assert not bad.any(), (float((err - tol).max()), int(bad.sum()), tuple(got.shape))


# ---- top-k -----------------------------------------------------------------------------

def check_topk(dev, logits, k, normalize, seed=0):
    g = gen(seed)
    rows, experts = logits.shape
    l64 = logits.double().cpu().requires_grad_()
    ids = OE.topk_ids(l64.detach(), k)
    w, mean = OE.topk_weights(l64, ids, normalize)
    gw, gm = torch.randn(rows, k, generator=g), torch.randn(experts, generator=g)
    (gl,) = torch.autograd.grad((w * gw.double()).sum() + (mean * gm.double()).sum(), [l64])

    ll = logits.detach().requires_grad_()
    ids2, w2, mean2 = fe.expert_topk(ll, k, normalize)
    assert ids2.dtype == torch.int64 and w2.dtype == mean2.dtype == torch.float32
    assert torch.equal(ids2.cpu(), ids)
    (gl2,) = torch.autograd.grad([w2, mean2], [ll], [gw.to(dev), gm.to(dev)])
    # the exponent l - max is off by u |l - max|; exp by 2 u; sums over the experts by 24 u (16 a lane, 6 levels)
    x = l64.detach()
    top = x.masked_fill(torch.isinf(x), -1e30).amax(1, keepdim=True)
    span = (x - top).abs().masked_fill(torch.isinf(x), 0.0).clamp(max=110)    # below, exp is 0 in float32
    rel = U * (40 + span.amax(1, keepdim=True))
    floor = 2.0 ** -125           # below the smallest normal number exp may flush to 0
    within(w2, w.detach(), rel * w.detach() + floor)
    p = OE.softmax(x)
    # a lane adds at most rows / 4 values and 1024 workgroups' sums are added by a fixed tree
    within(mean2, mean.detach(), ((rel + U * (96 + rows / 4)) * p).sum(0) / max(rows, 1) + floor)
    routed = torch.zeros_like(x)
    scale = (w.detach() if normalize else p.gather(1, ids.clamp(min=0)) * (ids >= 0))
    dot = (scale * gw.double().abs()).sum(1, keepdim=True)
    routed.scatter_add_(1, ids.clamp(min=0), scale * (gw.double().abs() + dot) * (ids >= 0))
    if not normalize:
        routed = routed + p * dot
    gma = gm.double().abs() / max(rows, 1)
    tol = HALF[logits.dtype] * gl.abs() + (4 * rel + U * 64) * (routed + p * (gma + (p * gma).sum(1, keepdim=True))) + floor
    within(gl2, gl, tol)
    with torch.no_grad():
        for a, b in zip(fe.expert_topk(logits, k, normalize), (ids2, w2, mean2)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (5, 2, 1), (9, 7, 7), (100, 8, 2), (64, 16, 4), (33, 64, 8),
                                            (17, 100, 3), (9, 256, 5), (5, 512, 2), (4, 513, 4), (3, 1000, 64),
                                            (3, 1024, 1), (3001, 8, 2), (50, 9, 2), (41, 61, 9), (19, 65, 4), (23, 201, 6),
                                            (12, 515, 8), (5, 1021, 33)])
def test_topk_sizes(dev, rows, experts, k, dtype):
    logits = (2 * torch.randn(rows, experts, generator=gen(rows + experts))).to(dev, dtype)
    for normalize in (True, False):
        check_topk(dev, logits, k, normalize)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_topk_masks_and_ties(dev, dtype, normalize):
    g = gen(1)
    l = torch.randn(12, 10, generator=g)
    l[0] = -INF                                  # nothing left
    l[1, 1:] = -INF                              # less left than chosen
    l[2, ::2] = -INF
    l[3] = 0.0                                   # all equal
    l[4] = torch.tensor([0.0, -0.0] * 5)
    l[5] = torch.finfo(dtype).min                # masked by the type's lowest value instead
    l[6, 3:] = torch.finfo(dtype).min
    l[7, 0], l[7, 9] = torch.finfo(dtype).max, torch.finfo(dtype).min
    l[8] = torch.round(l[8])                     # some equal
    l[9] *= 50
    check_topk(dev, l.to(dev, dtype), 3, normalize)
    check_topk(dev, l.to(dev, dtype), 10, normalize)


def test_topk_nan_and_infinity_stay_in_their_rows(dev):
    l = torch.randn(40, 24, generator=gen(2)).to(dev)
    a = l.clone().requires_grad_()
    ids, w, _ = fe.expert_topk(a, 3)
    gw = torch.randn(40, 3, generator=gen(3)).to(dev)
    (ga,) = torch.autograd.grad([w], [a], [gw])
    b = l.clone()
    b[4, 20], b[9, 2], b[9, 7], b[30, 5] = NAN, NAN, NAN, INF
    b.requires_grad_()
    ids2, w2, _ = fe.expert_topk(b, 3)
    (gb,) = torch.autograd.grad([w2], [b], [gw])
    assert ids2[4, 0] == 20 and ids2[9, :2].tolist() == [2, 7] and ids2[30, 0] == 5
    assert torch.isnan(w2[4]).any() and torch.isnan(w2[9]).any()
    keep = [r for r in range(40) if r not in (4, 9, 30)]
    for x, y in ((ids, ids2), (w, w2), (ga, gb)):
        assert torch.equal(x[keep], y[keep])


def test_topk_gradients_one_by_one_shapes_and_no_rows(dev):
    l = torch.randn(6, 5, 12, generator=gen(4)).to(dev)
    ids, w, mean = fe.expert_topk(l, 2)
    ids2, w2, mean2 = fe.expert_topk(l.view(30, 12), 2)
    assert ids.shape == w.shape == (6, 5, 2)
    assert torch.equal(ids.view(30, 2), ids2) and torch.equal(w.view(30, 2), w2) and torch.equal(mean, mean2)
    t = l.view(30, 12).t().contiguous().t()      # not contiguous
    assert torch.equal(fe.expert_topk(t, 2)[1], w2)
    for normalize in (True, False):
        a = l.view(30, 12).clone().requires_grad_()
        ids, w, mean = fe.expert_topk(a, 2, normalize)
        gw, gm = torch.randn(30, 2, generator=gen(5)).to(dev), torch.randn(12, generator=gen(6)).to(dev)
        (both,) = torch.autograd.grad([w, mean], [a], [gw, gm], retain_graph=True)
        (one,) = torch.autograd.grad([w], [a], [gw], retain_graph=True)
        (two,) = torch.autograd.grad([mean], [a], [gm])
        assert (one + two - both).abs().max() < 1e-6 * both.abs().max()
    e = torch.empty(0, 12, device=dev, requires_grad=True)
    ids, w, mean = fe.expert_topk(e, 2)
    assert ids.shape == (0, 2) and not mean.any()
    (ge,) = torch.autograd.grad([w, mean], [e], [torch.empty(0, 2, device=dev), torch.ones(12, device=dev)])
    assert ge.shape == (0, 12)


@pytest.mark.parametrize("experts", [5, 24, 67, 530])
def test_topk_of_unaligned_logits(dev, experts):
    for dtype in TYPES:
        l = torch.randn(31, experts, generator=gen(experts)).to(dev, dtype)
        apart = torch.cat([l.new_zeros(1), l.reshape(-1)])[1:].view(l.shape)
        both = []
        for t in (l, apart):
            t = t.detach().requires_grad_()
            ids, w, mean = fe.expert_topk(t, 3, False)
            both.append((ids, w, mean, torch.autograd.grad(w.square().sum() + mean.square().sum(), [t])[0]))
        for a, b in zip(*both):
            assert torch.equal(a, b)


def test_topk_gradient_against_differences(dev):
    l = torch.randn(3, 6, generator=gen(7), dtype=torch.float64)
    gw = torch.randn(3, 2, generator=gen(8), dtype=torch.float64)

    def loss(v):
        _, w, mean = fe.expert_topk(v.float().to(dev), 2, False)
        return (w.double().cpu() * gw).sum() + mean.double().cpu()[0]

    a = l.float().to(dev).requires_grad_()
    _, w, mean = fe.expert_topk(a, 2, False)
    ((w * gw.float().to(dev)).sum() + mean[0]).backward()
    step = 2.0 ** -7
    for i in range(3):
        for j in range(6):
            d = torch.zeros_like(l)
            d[i, j] = step
            diff = (loss(l + d) - loss(l - d)) / (2 * step)
            # third derivatives of a softmax are below 1 per unit of weight; float32 values are off by 2^-22 each
            assert abs(diff - a.grad[i, j].item()) < step ** 2 * gw.abs().sum() + 2.0 ** -20 / step


# ---- plan and rows ---------------------------------------------------------------------

def some_ids(g, rows, k, experts, bad=0.1):
    """Random experts; a tenth of the slots outside the experts' range, near and far."""
    ids = torch.randint(0, experts, (rows, k), generator=g)
    outside = torch.tensor([-1, experts, 2 ** 40, -2 ** 62])[torch.randint(0, 4, (rows, k), generator=g)]
    return torch.where(torch.rand(rows, k, generator=g) < bad, outside, ids)


@pytest.mark.parametrize("rows,k,experts", [(0, 2, 4), (1, 1, 1), (5, 1, 3), (100, 2, 8), (64, 1, 64), (333, 3, 65),
                                            (4096, 2, 8), (8193, 1, 5), (1000, 64, 9), (3000, 4, 1024), (2049, 8, 100),
                                            (30011, 2, 16), (700, 2, 1024), (4095, 2, 960), (4095, 2, 962), (70000, 2, 1023),
                                            (9000, 1, 255), (9000, 1, 256)])
def test_plan_is_exact(dev, rows, k, experts):
    ids = some_ids(gen(rows + k), rows, k, experts)
    order, positions, offsets = OE.plan(ids, experts)
    plan = fe.ExpertPlan(ids.to(dev), experts)
    assert torch.equal(plan.order.cpu().long(), order)
    assert torch.equal(plan.positions.cpu().long(), positions)
    assert torch.equal(plan.offsets.cpu().long(), offsets)


def test_plan_of_one_expert_none_and_small_integer_types(dev):
    for value, n in ((3, 5000), (-1, 5000), (7, 20)):
        plan = fe.ExpertPlan(torch.full((n, 2), value, device=dev), 7)
        want = 2 * n if 0 <= value < 7 else 0
        assert plan.offsets[-1].item() == want and torch.equal(plan.order.cpu(), torch.arange(2 * n, dtype=torch.int32))
    ids = torch.tensor([2, 0, 1, 0])
    for t in (torch.int32, torch.int16, torch.int8, torch.uint8):
        plan = fe.ExpertPlan(ids.to(dev, t), 3)
        assert plan.order.tolist() == [1, 3, 2, 0] and plan.positions.shape == (4, 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,rows,k,width,experts", [
    ((), 1, 1, 1, 1), ((), 7, 2, 3, 4), ((9,), 50, 2, 64, 8), ((2, 3), 33, 3, 20, 5), ((49,), 20, 4, 128, 16),
    ((4,), 100, 5, 33, 8), ((), 300, 8, 576, 12), ((1,), 65, 1, 1152, 3), ((3,), 41, 9, 6, 10),
    ((4,), 30, 2, 5, 3), ((9,), 12, 3, 13, 4), ((16,), 11, 4, 259, 5)])
def test_rows_and_their_gradients(dev, lead, rows, k, width, experts, dtype):
    g = gen(rows * k + width)
    ids = some_ids(g, rows, k, experts)
    ids[0] = -1                                  # a row without any expert
    x = torch.randn(*lead, rows, width, generator=g).to(dtype)
    ys = torch.randn(*lead, rows * k, width, generator=g).to(dtype)
    w = torch.randn(rows, k, generator=g)
    gxs, gy = torch.randn(*lead, rows * k, width, generator=g).to(dtype), torch.randn(*lead, rows, width, generator=g).to(dtype)
    x64, ys64, w64 = (t.double().requires_grad_() for t in (x, ys, w))
    xs_r = OE.dispatch(x64, ids, experts)
    y_r = OE.combine(ys64, w64, ids, experts)
    gx_r, gys_r, gw_r = torch.autograd.grad([xs_r, y_r], [x64, ys64, w64], [gxs.double(), gy.double()])

    plan = fe.ExpertPlan(ids.to(dev), experts)
    xl, yl, wl = (t.to(dev).requires_grad_() for t in (x, ys, w))
    xs = plan.dispatch(xl)
    y = plan.combine(yl, wl)
    gx, gys, gw = torch.autograd.grad([xs, y], [xl, yl, wl], [gxs.to(dev), gy.to(dev)])
    assert torch.equal(xs.detach().cpu().double(), xs_r.detach())           # moved, not computed
    absolute = OE.combine(ys.double().abs(), w.double().abs(), ids, experts)
    within(y, y_r.detach(), HALF[dtype] * y_r.detach().abs() + U * (k + 1) * absolute)
    ones = torch.ones(rows, k, dtype=torch.float64)
    within(gx, gx_r, HALF[dtype] * gx_r.abs() + U * k * OE.combine(gxs.double().abs(), ones, ids, experts))
    within(gys, gys_r, (HALF[dtype] + U) * gys_r.abs())
    # a lane's run: its planes times its 8 (16-bit) or 4 elements a vector, one for odd widths, then 6 + 16 more
    a64, b64 = ys.double().abs().requires_grad_(), torch.ones(rows, k, dtype=torch.float64, requires_grad=True)
    (mass,) = torch.autograd.grad(OE.combine(a64, b64, ids, experts), [b64], gy.double().abs())
    planes = x.numel() // (rows * width)
    within(gw, gw_r, U * (gw_r.abs() + (planes + 8 * (width // 64 + 1) * (planes // 4 + 1) + 32) * mass))


def test_rows_strides_weight_types_and_unaligned_views(dev):
    g = gen(11)
    ids = some_ids(g, 30, 2, 4).to(dev)
    plan = fe.ExpertPlan(ids, 4)
    x = torch.randn(30, 9, 16, generator=g).to(dev).permute(1, 0, 2)        # node-major, seen component-major
    assert torch.equal(plan.dispatch(x), plan.dispatch(x.contiguous()))
    flat = torch.randn(9 * 30 * 16 + 1, generator=g).to(dev)[1:].view(9, 30, 16)   # 4-byte aligned
    assert torch.equal(plan.dispatch(flat), plan.dispatch(flat.clone()))
    half = torch.randn(30 * 16 + 1, generator=g).to(dev, torch.bfloat16)[1:].view(30, 16)
    assert torch.equal(plan.dispatch(half), plan.dispatch(half.clone()))
    ys = torch.randn(9 * 60 * 16 + 1, generator=g).to(dev)[1:].view(9, 60, 16)
    w = torch.rand(30, 2, generator=g).to(dev)
    for t in TYPES:
        wt = w.to(t).requires_grad_()
        y = plan.combine(ys, wt)
        assert torch.equal(y, plan.combine(ys.clone(), wt.detach().float()))
        (gw,) = torch.autograd.grad(y.sum(), [wt])
        assert gw.dtype == t
    one = fe.ExpertPlan(ids[:, 0].contiguous(), 4)
    assert torch.equal(one.combine(ys[0, :30], w[:, 0]), one.combine(ys[0, :30], w[:, :1]))


def test_the_same_expert_twice_and_unrouted_garbage(dev):
    """A row may name an expert twice; what stands in the places without an expert is never read."""
    ids = torch.tensor([[1, 1], [0, -1], [-1, -1], [2, 0]], device=dev)
    plan = fe.ExpertPlan(ids, 3)
    x = torch.randn(4, 5, generator=gen(12)).to(dev)
    xs = plan.dispatch(x)
    n = plan.offsets[-1].item()
    assert n == 5 and not xs[n:].any()
    w = torch.tensor([[0.25, 0.5], [2.0, NAN], [INF, NAN], [1.0, 1.0]], device=dev)
    ys = xs.clone()
    ys[n:] = NAN
    ys.requires_grad_()
    wl = w.clone().requires_grad_()
    y = plan.combine(ys, wl)
    want = torch.stack([0.75 * x[0], 2 * x[1], 0 * x[2], 2 * x[3]])
    assert torch.allclose(y, want, atol=1e-6) and not y[2].any()
    gys, gw = torch.autograd.grad(y, [ys, wl], torch.ones_like(y))
    assert not gys[n:].any() and torch.isfinite(gys).all()
    assert gw[1, 1] == 0 and not gw[2].any() and torch.isfinite(gw).all()
    xl = x.clone().requires_grad_()
    g = torch.randn(8, 5, generator=gen(13)).to(dev)
    g[n:] = NAN
    (gx,) = torch.autograd.grad(plan.dispatch(xl), [xl], g)
    assert torch.isfinite(gx).all() and not gx[2].any()


def test_rows_without_elements(dev):
    plan = fe.ExpertPlan(torch.empty(0, 2, dtype=torch.int64, device=dev), 3)
    assert plan.offsets.tolist() == [0] * 4
    x = torch.empty(4, 0, 8, device=dev, requires_grad=True)
    w = torch.empty(0, 2, device=dev, requires_grad=True)
    y = plan.combine(plan.dispatch(x), w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.empty(4, 0, 8, device=dev))
    assert y.shape == gx.shape == (4, 0, 8) and gw.shape == (0, 2)


# ---- the experts' maps -----------------------------------------------------------------

def check_linear(dev, lvals, counts, unrouted, cin, cout, dtype, bias=True, seed=0):
    g = gen(seed)
    experts = len(counts)
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((unrouted,), -1)]).long()
    ids = ids[torch.randperm(ids.numel(), generator=g)]
    slots, dim = ids.numel(), sum(2 * l + 1 for l in lvals)
    x = torch.randn(dim, slots, cin, generator=g).to(dtype)
    w = torch.randn(experts, len(lvals), cout, cin, generator=g).to(dtype)
    ns = sum(l == 0 for l in lvals)
    b = torch.randn(experts, cout, ns, generator=g).to(dtype) if bias and ns else None
    gy = torch.randn(dim, slots, cout, generator=g).to(dtype)
    plan = fe.ExpertPlan(ids.to(dev), experts)
    n = plan.offsets[-1].item()
    gyd = gy.clone()
    x[:, n:], gyd[:, n:] = NAN, NAN              # the rows without an expert are not read
    xl, wl = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    bl = b.to(dev).requires_grad_() if b is not None else None
    leaves = [t for t in (xl, wl, bl) if t is not None]
    y = fe.expert_linear(xl, wl, plan, lvals, bl)
    got = torch.autograd.grad(y, leaves, gyd.to(dev))
    with torch.no_grad():
        assert torch.equal(fe.expert_linear(xl, wl, plan, lvals, bl), y)

    def reference(f):
        x64, w64 = f(x.nan_to_num().double()).requires_grad_(), f(w.double()).requires_grad_()
        b64 = f(b.double()).requires_grad_() if b is not None else None
        y64 = OE.linear(x64, w64, plan.offsets.cpu(), lvals, b64)
        return (y64.detach(), *torch.autograd.grad(y64, [t for t in (x64, w64, b64) if t is not None], f(gy.double())))
    want, mass = reference(lambda t: t.clone()), reference(torch.abs)
    terms = [2 * cin + 2, 2 * cout, None, None]
    rows = 2 * (max([1, *counts]) * (2 * max(lvals) + 1)) + 64              # terms of a weight's gradient
    for i, (a, r, m) in enumerate(zip((y, *got), want, mass)):
        within(a, r, HALF[dtype] * r.abs() + U * (terms[i] or rows) * m)
    assert not y[:, n:].any() and not got[0][:, n:].any()
    for i, leaf in enumerate(leaves):            # each gradient without the others
        args = [t.detach().requires_grad_(t is leaf) if t is not None else None for t in (xl, wl, bl)]
        (one,) = torch.autograd.grad(fe.expert_linear(*args[:2], plan, lvals, args[2]), [args[i]], gyd.to(dev))
        within(one, want[1 + i], HALF[dtype] * want[1 + i].abs() + U * (terms[1 + i] or rows) * mass[1 + i])
        assert i or not one[:, n:].any()


CHANNELS = [(64, 128), (128, 64), (8, 8), (33, 7), (1, 1), (160, 200), (12, 260), (300, 20), (301, 133), (131, 9),
            (22, 26), (9, 98), (32, 64), (30, 70), (48, 61), (72, 9), (5, 129), (136, 72), (129, 65)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cin,cout", CHANNELS)
def test_linear_channels(dev, cin, cout, dtype):
    check_linear(dev, (0, 1), [30, 0, 200, 5], 9, cin, cout, dtype, seed=cin + cout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lvals", [(0,), (1,), (0, 0), (2, 0, 1, 0), (0, 1, 2, 3, 4, 5, 6)])
def test_linear_irreps(dev, lvals, dtype):
    check_linear(dev, lvals, [17, 140], 0, 32, 48, dtype, seed=len(lvals))
    check_linear(dev, lvals, [17, 140], 3, 32, 48, dtype, bias=False, seed=len(lvals))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts,unrouted", [([1], 0), ([0], 0), ([0, 0, 0], 5), ([0, 1], 0), ([128], 0), ([129, 127], 0),
                                             ([1] * 64, 0), ([3] * 65, 2), ([0] * 100 + [40] + [2] * 99, 1), ([900, 1, 1], 0),
                                             ([2] * 1024, 0)])
def test_linear_counts(dev, counts, unrouted, dtype):
    check_linear(dev, (0, 1), counts, unrouted, 24, 40, dtype, seed=len(counts))


def test_linear_many_chunks(dev):
    """Experts of several weight-gradient chunks beside ones of one and none."""
    check_linear(dev, (0, 1), [5000, 100, 0, 2000, 129], 50, 16, 24, torch.float32, seed=3)
    check_linear(dev, (0,), [3000, 64, 1500], 0, 64, 64, torch.bfloat16, seed=4)
    check_linear(dev, (0, 0), [30000, 1], 3, 34, 51, torch.float32, seed=5)      # more than eight chunks an expert
    check_linear(dev, (0,), [9000, 40000], 0, 32, 32, torch.float16, seed=6)


def test_linear_views_and_two_dimensions(dev):
    g = gen(5)
    plan = fe.ExpertPlan(torch.tensor([1, 0, 1, 1], device=dev), 2)
    x = torch.randn(4, 9, generator=g).to(dev)
    w = torch.randn(2, 1, 5, 9, generator=g).to(dev)
    y = fe.expert_linear(x, w, plan)
    assert y.shape == (4, 5) and torch.equal(y, fe.expert_linear(x[None], w, plan)[0])
    t = torch.randn(9, 4, generator=g).to(dev).t()          # strided
    assert torch.equal(fe.expert_linear(t, w, plan), fe.expert_linear(t.contiguous(), w, plan))
    flat = torch.randn(4 * 16 + 1, generator=g).to(dev)[1:].view(4, 16)     # 4-byte aligned
    w16 = torch.randn(2, 1, 8, 16, generator=g).to(dev)
    assert torch.equal(fe.expert_linear(flat, w16, plan), fe.expert_linear(flat.clone(), w16, plan))


@pytest.mark.parametrize("cin,cout", [(5, 6), (24, 40), (41, 30), (150, 136), (137, 9)])
def test_linear_of_unaligned_tables(dev, cin, cout):
    """Every table one element further on: as far from the formula as aligned ones, and zeros behind the last row."""
    for dtype in TYPES:
        g = gen(cin)
        ids = some_ids(g, 70, 1, 3)
        plan = fe.ExpertPlan(ids.to(dev), 3)
        n = plan.offsets[-1].item()

        def apart(*shape):
            return torch.randn(torch.Size(shape).numel() + 1, generator=g).to(dtype)[1:].view(shape)
        x, w, b, gy = apart(4, 70, cin), apart(3, 2, cout, cin), apart(3, cout, 1), apart(4, 70, cout)
        # moved to the device with the element before them
        far = [torch.cat([t.new_zeros(1), t.reshape(-1)]).to(dev)[1:].view(t.shape) for t in (x, w, b, gy)]
        leaves = [t.requires_grad_() for t in far[:3]]
        y = fe.expert_linear(*leaves[:2], plan, (0, 1), leaves[2])
        got = (y, *torch.autograd.grad(y, leaves, far[3]))

        def reference(f):
            l64 = [f(t.double()).requires_grad_() for t in (x, w, b)]
            y64 = OE.linear(*l64[:2], plan.offsets.cpu(), (0, 1), l64[2])
            return (y64.detach(), *torch.autograd.grad(y64, l64, f(gy.double())))
        want, mass = reference(lambda t: t.clone()), reference(torch.abs)
        for a, r, m, terms in zip(got, want, mass, (2 * cin + 2, 2 * cout, 700, 700)):
            within(a, r, HALF[dtype] * r.abs() + U * terms * m)
        assert not y[:, n:].any() and not got[1][:, n:].any()


def test_linear_infinity_stays_in_its_row_and_expert(dev):
    g = gen(6)
    ids = torch.arange(300, device=dev) % 3
    plan = fe.ExpertPlan(ids, 3)
    x = torch.randn(4, 300, 20, generator=g).to(dev)
    w = torch.randn(3, 2, 12, 20, generator=g).to(dev)
    gy = torch.randn(4, 300, 12, generator=g).to(dev)

    def step(x):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = fe.expert_linear(xl, wl, plan, (0, 1))
        return (y.detach(), *torch.autograd.grad(y, [xl, wl], gy))
    y, gx, gw = step(x)
    x2 = x.clone()
    x2[1, 150, 3], x2[0, 10, 0] = INF, NAN       # rows of experts 1 and 0
    y2, gx2, gw2 = step(x2)
    assert torch.equal(gx, gx2)
    want = torch.sign(w[1, 1, :, 3]) * INF       # infinity times the weight
    assert torch.equal(y2[1, 150], want) and torch.isnan(y2[0, 10]).all()
    y2[1, 150], y2[0, 10] = y[1, 150], y[0, 10]
    assert torch.equal(y, y2)
    assert torch.equal(gw[2], gw2[2]) and torch.equal(gw[0, 1], gw2[0, 1]) and torch.equal(gw[1, 0], gw2[1, 0])


def test_refusals(dev):
    x, ids = torch.randn(6, 8, device=dev), torch.zeros(6, 2, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="top_k must be 1 to 8"):
        fe.expert_topk(x, 9)
    with pytest.raises(TypeError, match="float64"):
        fe.expert_topk(x.double(), 2)
    with pytest.raises(TypeError, match="ids must be integers"):
        fe.ExpertPlan(ids.float(), 3)
    with pytest.raises(ValueError, match="num_experts must be"):
        fe.ExpertPlan(ids, 0)
    with pytest.raises(ValueError, match="ids must be"):
        fe.ExpertPlan(ids[None], 3)
    plan = fe.ExpertPlan(ids, 3)
    with pytest.raises(ValueError, match="x must be"):
        plan.dispatch(x[:5])
    with pytest.raises(ValueError, match="ys must be"):
        plan.combine(x, torch.ones(6, 2, device=dev))
    with pytest.raises(ValueError, match="weights must be"):
        plan.combine(torch.randn(12, 8, device=dev), torch.ones(6, device=dev))
    with pytest.raises(fe.CUDANotAvailableError):
        plan.dispatch(x.cpu())
    with pytest.raises(TypeError, match="weights"):
        plan.combine(torch.randn(12, 8, device=dev), torch.ones(6, 2, device=dev, dtype=torch.float64))
    xs, w = torch.randn(1, 12, 8, device=dev), torch.randn(3, 1, 4, 8, device=dev)
    for args, text in (((xs, w[:2], plan), "weight must be"), ((xs[:, :11], w, plan), "x must be"),
                       ((xs, w, plan, (0, 1)), "weight must be"), ((xs, w, plan, (0,), torch.zeros(3, 4, 2, device=dev)), "bias must be"),
                       ((xs, w, plan, ()), "lvals must be"), ((xs, w[:, :, :0], plan), "no channels")):
        with pytest.raises(ValueError, match=text):
            fe.expert_linear(*args)
    with pytest.raises(TypeError, match="different dtypes"):
        fe.expert_linear(xs, w.half(), plan)


def test_broadcast_inputs_and_gradients(dev):
    """Expanded inputs give what their copies give, and their sources the copies' gradients summed."""
    g = gen(14)
    plan = fe.ExpertPlan(some_ids(g, 40, 2, 3).to(dev), 3)
    x, ys = torch.randn(1, 40, 8, generator=g).to(dev), torch.randn(4, 1, 8, generator=g).to(dev)
    w, lw = torch.rand(1, 2, generator=g).to(dev), torch.randn(3, 1, 6, 8, generator=g).to(dev)
    l = torch.randn(1, 3, generator=g).to(dev)
    calls = [(lambda a: plan.dispatch(a), x, (4, 40, 8)),
             (lambda a: plan.combine(a, w.expand(40, 2)), ys, (4, 80, 8)),
             (lambda a: plan.combine(ys.expand(4, 80, 8), a), w, (40, 2)),
             (lambda a: fe.expert_linear(ys.expand(4, 80, 8), a, plan, (0, 1)), lw, (3, 2, 6, 8)),
             (lambda a: fe.expert_linear(a, lw.expand(3, 2, 6, 8), plan, (0, 1)), ys, (4, 80, 8)),
             (lambda a: fe.expert_topk(a, 2)[1], l, (40, 3))]
    for call, small, shape in calls:
        a = small.clone().requires_grad_()
        b = small.expand(shape).contiguous().requires_grad_()
        ya, yb = call(a.expand(shape)), call(b)
        assert torch.equal(ya, yb)
        gy = torch.ones(1, device=dev).expand(ya.shape)              # as of a sum, stride 0
        (ga,), (gb,) = torch.autograd.grad(ya, [a], gy), torch.autograd.grad(yb, [b], gy.contiguous())
        assert torch.allclose(ga, gb.sum_to_size(small.shape), rtol=1e-5, atol=1e-6 * max(1.0, gb.abs().max().item()))


def test_a_plan_is_for_reading(dev):
    """Places that a kernel would write to are those of the sort, or the call is refused; copies are plans too."""
    import copy
    import pickle
    ids = torch.tensor([[0, 1], [2, 0], [-1, 1]], device=dev)
    x, w = torch.randn(3, 8, device=dev, requires_grad=True), torch.ones(3, 2, device=dev, requires_grad=True)
    lw = torch.randn(3, 1, 8, 8, device=dev, requires_grad=True)
    plan = fe.ExpertPlan(ids, 3)
    with pytest.raises(AttributeError):
        plan.positions = plan.positions.long()
    for other in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        assert torch.equal(other.order, plan.order) and torch.equal(other.dispatch(x), plan.dispatch(x))
    xs = plan.dispatch(x)
    ys = fe.expert_linear(xs, lw, plan)
    y = plan.combine(ys, w)
    plan.offsets[-1] += 1
    with pytest.raises(RuntimeError, match="offsets of an ExpertPlan have been modified"):
        plan.dispatch(x)
    with pytest.raises(RuntimeError, match="have been modified"):
        fe.expert_linear(xs, lw, plan)
    for out, leaf in ((y, w), (ys, lw), (xs, x)):
        with pytest.raises(RuntimeError, match="have been modified"):
            torch.autograd.grad(out.sum(), [leaf], retain_graph=True)
    plan = fe.ExpertPlan(ids, 3)
    plan.positions.clamp_(max=2)
    with pytest.raises(RuntimeError, match="positions of an ExpertPlan have been modified"):
        plan.combine(ys, w)
    with torch.inference_mode():
        plan = fe.ExpertPlan(ids, 3)
        assert plan.combine(plan.dispatch(x), w).shape == (3, 8)


def test_derivatives_that_there_are_not(dev):
    """Inputs changed before the backward, second derivatives and forward mode raise; none gives a wrong gradient."""
    ids = torch.tensor([[0, 1], [1, 0]], device=dev)
    plan = fe.ExpertPlan(ids, 2)
    calls = [(lambda l: fe.expert_topk(l, 2, False)[1], [(5, 4)]),
             (lambda x: plan.dispatch(x), [(2, 6)]),
             (lambda ys, w: plan.combine(ys, w), [(4, 6), (2, 2)]),
             (lambda x, w: fe.expert_linear(x, w, plan), [(4, 6), (2, 1, 3, 6)])]
    for k, (call, shapes) in enumerate(calls):
        for i in range(len(shapes)):
            args = [torch.randn(s, generator=gen(i)).to(dev).requires_grad_() for s in shapes]
            out = call(*args)
            grads = torch.autograd.grad(out.square().sum(), args, create_graph=True)
            with pytest.raises(RuntimeError, match="no second derivative"):
                grads[i].sum().backward()
            if k != 1:                           # dispatch keeps none of its input
                out = call(*args)
                with torch.no_grad():
                    args[i].add_(1.0)
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    out.sum().backward()
            with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                duals = [torch.autograd.forward_ad.make_dual(a.detach(), torch.ones_like(a)) if j == i else a.detach()
                         for j, a in enumerate(args)]
                call(*duals)
    l = torch.randn(5, 4, device=dev, requires_grad=True)
    chosen, w, _ = fe.expert_topk(l, 2)
    chosen.clamp_(max=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.square().sum().backward()


def test_past_32_bit_offsets(dev):
    """Rows whose elements lie behind the first 2^31, read and written at their places."""
    rows, width = 2 ** 20 + 5, 1030                  # two slots a row: 2.2e9 elements in expert order
    g = gen(17)
    ids = torch.zeros(rows, 2, dtype=torch.int64, device=dev)
    ids[:, 1], ids[0], ids[-1, 1] = 1, 1, -1
    plan = fe.ExpertPlan(ids, 2)
    x = torch.zeros(rows, width, device=dev, dtype=torch.bfloat16)
    x[0], x[-1] = torch.randn(2, width, generator=g).to(dev, torch.bfloat16)
    xs = plan.dispatch(x)
    slots = 2 * rows
    places = plan.positions[[0, -1]].tolist()        # row 0 behind the expert 0's, the last slot unrouted
    assert places[1][1] == slots - 1 and places[0][0] == rows - 1
    assert torch.equal(xs[rows - 1], x[0]) and torch.equal(xs[rows], x[0]) and torch.equal(xs[rows - 2], x[-1])
    assert not xs[-1].any() and not xs[slots // 2 + 9].any()
    w = torch.ones(rows, 2, device=dev)
    xs[slots - 2] = 1.0                              # row rows - 2's second slot, in the last places
    y = plan.combine(xs, w)
    assert torch.equal(y[0], (2 * x[0].float()).bfloat16()) and torch.equal(y[-1], x[-1])
    assert (y[-2] == 1).all() and not y[-3].any()
    del xs, y
    lw = torch.randn(2, 1, 8, 1030, generator=g).to(dev, torch.bfloat16)
    big = torch.zeros(slots, width, device=dev, dtype=torch.bfloat16)
    big[slots - 2], big[3] = x[0], x[-1]
    out = fe.expert_linear(big, lw, plan)
    small = fe.ExpertPlan(torch.tensor([0, 1], device=dev), 2)
    want = fe.expert_linear(torch.stack([x[-1], x[0]]), lw, small)
    assert torch.equal(out[3], want[0]) and torch.equal(out[slots - 2], want[1]) and not out[slots - 1].any()
    del big
    gy = torch.zeros(slots, 8, device=dev, dtype=torch.bfloat16)
    gy[slots - 2], gy[3] = 1.0, 2.0
    lx = torch.zeros(slots, width, device=dev, dtype=torch.bfloat16)
    lx[slots - 2], lx[3] = x[0], x[-1]
    lx.requires_grad_()
    gx, gw = torch.autograd.grad(fe.expert_linear(lx, lw.requires_grad_(), plan), [lx, lw], gy)
    sx = torch.stack([x[-1], x[0]]).requires_grad_()
    gx2, gw2 = torch.autograd.grad(fe.expert_linear(sx, lw, small), [sx, lw], gy[[3, slots - 2]])
    assert torch.equal(gx[3], gx2[0]) and torch.equal(gx[slots - 2], gx2[1]) and torch.equal(gw, gw2)


def test_topk_past_32_bit_offsets(dev):
    rows, experts = 2 ** 25 + 7, 64                  # 2.1e9 logits
    l = torch.zeros(rows, experts, device=dev, dtype=torch.float16)
    tail = torch.randn(9, experts, generator=gen(18)).to(dev, torch.float16)
    l[-9:] = tail
    l.requires_grad_()
    ids, w, _ = fe.expert_topk(l, 2)
    t = tail.clone().requires_grad_()
    ids2, w2, _ = fe.expert_topk(t, 2)
    assert torch.equal(ids[-9:], ids2) and torch.equal(w[-9:], w2) and (ids[0] == torch.tensor([0, 1], device=dev)).all()
    gw = torch.zeros_like(w)
    gw[-9:, 0] = 1.0
    (gl,) = torch.autograd.grad(w, [l], gw)
    (gt,) = torch.autograd.grad(w2, [t], gw[-9:].clone())
    assert torch.equal(gl[-9:], gt) and not gl[:9].any()


# ---- a run of them together ------------------------------------------------------------

@pytest.mark.parametrize("top_k", [1, 2])
def test_expert_mlp_matches_the_oracle(dev, top_k):
    torch.manual_seed(5)
    rp = fe.Repr([0, 1, 2], 32)
    mlp = fe.EquivariantExpertMLP(rp, 6, top_k=top_k).to(dev)
    with torch.no_grad():
        for b in (mlp.up.bias, mlp.down.bias, mlp.act.linear.bias):
            b.normal_(generator=torch.Generator(device=dev).manual_seed(1))
    x = torch.randn(403, 32, 9, generator=gen(6))
    xl = x.to(dev).requires_grad_()
    terms = []
    y = mlp(xl, balance=terms)
    (own,) = terms
    gy = torch.randn(403, 32, 9, generator=gen(7))
    params = dict(mlp.named_parameters())
    grads = torch.autograd.grad((y * gy.to(dev)).sum() + own, [xl, *params.values()])

    x64 = x.double().requires_grad_()
    p64 = {k: v.detach().double().cpu().requires_grad_() for k, v in params.items()}
    inv = torch.stack([(x64[..., a:b] ** 2).sum(-1) for a, b in ((0, 1), (1, 4), (4, 9))], -1) + 1e-8
    logits = OE.layer_norm(inv.sqrt().flatten(-2), p64["router.lnorm.weight"], p64["router.lnorm.bias"]) \
        @ p64["router.linear.weight"].t()
    ids = OE.topk_ids(logits.detach(), top_k)
    # float32 logits of this size are off by less than 1e-5: no choice lies that close to another
    top = logits.detach().sort(1, descending=True).values
    assert (top[:, top_k - 1] - top[:, top_k]).min() > 1e-5
    w, mean = OE.topk_weights(logits, ids, True)
    _, _, offsets = OE.plan(ids, 6)
    balance = 6 * ((offsets[1:] - offsets[:-1]).double() * mean).sum() / ids.numel()
    names = dict(up_w="up.weight", up_b="up.bias", gate_w="act.linear.weight", gate_b="act.linear.bias",
                 down_w="down.weight", down_b="down.bias")
    y64 = OE.expert_mlp(x64, ids, w, {k: p64[v] for k, v in names.items()}, (0, 1, 2), 1e-8)
    want = torch.autograd.grad((y64 * gy.double()).sum() + balance, [x64, *p64.values()])
    rel = lambda a, b: ((a.detach().double().cpu() - b).abs().max() / b.abs().max()).item()
    assert rel(y, y64.detach()) < 1e-5 and rel(own, balance.detach()) < 1e-5
    for name, a, b in zip(["x", *params], grads, want):
        if top_k == 1 and name.startswith("router"):     # one weight of 1: only the balance is left, tiny
            assert (a.detach().double().cpu() - b).abs().max() < 1e-5
        else:
            assert rel(a, b) < 2e-5, name


def test_expert_block_is_equivariant_and_trains(dev):
    """A transformer with expert MLPs: rotated inputs give the rotated output (the choice reads invariants),
    and every parameter has a gradient."""
    torch.manual_seed(2)
    rp = fe.Repr([0, 1], 16)
    model = fe.EquivariantTransformer(rp, rp, rp, num_layers=2, num_heads=4, layer_scale_init=0.3, num_experts=4,
                                      experts_per_node=2).to(dev)
    g = gen(3)
    xyz = torch.randn(120, 3, generator=g) * 3
    d = torch.cdist(xyz, xyz) + torch.eye(120) * 1e9
    src = d.topk(8, largest=False).indices.reshape(-1)
    dst = torch.arange(120).repeat_interleave(8)
    graph = fe.Graph(src.to(dev), dst.to(dev), 120)
    x = torch.randn(120, 16, 4, generator=g)
    axis, angle = fe.random_rotation()
    D = fe.WignerD(rp).rot(axis, angle)
    R = fe.WignerD(fe.Repr([1])).rot(axis, angle, cartesian=True)
    y = model(xyz.to(dev), x.to(dev), graph)
    y2 = model((xyz @ R.t()).to(dev), (x @ D.t()).to(dev), graph)
    err = ((y2 - y @ D.t().to(dev)).abs().max() / y.abs().max()).item()
    assert err < 1e-2, err           # the bar of the model's other equivariance tests
    terms = []
    y = model(xyz.to(dev), x.to(dev), graph, balance=terms)
    assert len(terms) == 2
    loss = y.pow(2).mean() + 0.01 * sum(terms)
    loss.backward()
    missing = [k for k, p in model.named_parameters() if p.grad is None]
    assert not missing, missing
    for layer in model.layers:
        for p in (layer.experts.up.weight, layer.experts.down.weight, layer.experts.router.linear.weight):
            assert torch.isfinite(p.grad).all() and p.grad.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_precision_block_and_mlp(dev, dtype):
    torch.manual_seed(4)
    rp = fe.Repr([0, 1], 16)
    mlp = fe.EquivariantExpertMLP(rp, 4, 2).to(dev, dtype)
    x = torch.randn(50, 16, 4, generator=gen(8)).to(dev, dtype).requires_grad_()
    terms = []
    y = mlp(x, terms)
    (gx,) = torch.autograd.grad(y.sum() + terms[0], [x])
    assert y.dtype == gx.dtype == dtype and torch.isfinite(y).all() and torch.isfinite(gx).all()
    block = fe.EquivariantTransformerBlock(rp, rp, num_heads=2, num_experts=4).to(dev, dtype)
    graph = fe.Graph.random(50, 300, device=dev)
    vec = torch.randn(300, 3, generator=gen(9)).to(dev)
    (P,) = fe.WignerDBasis([rp]).to(dev)(vec)
    out = block(P.to(dtype), P.to(dtype), x, vec.norm(dim=-1).to(dtype), graph, balance=terms)
    assert out.dtype == dtype and torch.isfinite(out).all()
    assert len(terms) == 2 and torch.isfinite(terms[1])
    with pytest.raises(TypeError, match="float64"):
        fe.EquivariantExpertMLP(rp, 4, 2).to(dev).double()(x.double())


def test_captured_training_step(dev):
    """The whole mixture in a graph: replays on new inputs give the eager step's bits."""
    from flash_eq.capture import capture_step
    torch.manual_seed(6)
    rp = fe.Repr([0, 1], 32)
    mlp = fe.EquivariantExpertMLP(rp, 8, 2).to(dev)
    x = torch.randn(5000, 32, 4, generator=gen(1)).to(dev).requires_grad_()      # 10000 slots: the plan's tiled form
    gy = torch.randn(5000, 32, 4, generator=gen(2)).to(dev)
    leaves = [x, *mlp.parameters()]

    def step():
        terms = []
        loss = (mlp(x, terms) * gy).sum((1, 2)).mean() + terms[0]
        loss.backward()
        return loss

    graph, loss = capture_step(step, leaves)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(5000, 32, 4, generator=gen(30 + k)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.grad.clone() for t in leaves]
        terms = []
        y = (mlp(x, terms) * gy).sum((1, 2)).mean() + terms[0]
        want = torch.autograd.grad(y, leaves)
        for a, b in zip(got, want):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6 * b.abs().max().item())
        torch.cuda.synchronize()


def test_another_stream_and_the_same_bits(dev):
    g = gen(9)
    ids = some_ids(g, 900, 2, 8).to(dev)
    x = torch.randn(9, 900, 64, generator=g).to(dev)
    w = torch.randn(8, 3, 64, 64, generator=g).to(dev).requires_grad_()
    probs = torch.rand(900, 2, generator=g).to(dev).requires_grad_()

    def step():
        plan = fe.ExpertPlan(ids, 8)
        y = plan.combine(fe.expert_linear(plan.dispatch(x), w, plan, (0, 1, 2)), probs)
        return (y.detach(), *torch.autograd.grad(y.square().sum(), [w, probs]))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, other, step()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_graphs_two_threads_and_an_empty_input(dev):
    """Captured steps replayed in turn, with eager work between, and threads on streams of their own: each call's
    results are its own."""
    import threading
    from flash_eq.capture import capture_step
    torch.manual_seed(8)
    rp = fe.Repr([0, 1], 16)
    mlps = [fe.EquivariantExpertMLP(rp, n, 2).to(dev) for n in (4, 9)]
    xs = [torch.randn(n, 16, 4, generator=gen(n)).to(dev).requires_grad_() for n in (700, 5001)]

    def eager(i):
        terms = []
        loss = mlps[i](xs[i], terms).square().sum((1, 2)).mean() + terms[0]
        return loss, [xs[i], *mlps[i].parameters()]

    def step_of(i):
        def step():
            loss, _ = eager(i)
            loss.backward()
            return loss
        return step
    graphs = [capture_step(step_of(i), eager(i)[1]) for i in range(2)]
    for k in range(3):
        for x in xs:
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, generator=gen(60 + k)))
        for graph, _ in graphs:
            graph.replay()
        for i in range(2):
            torch.cuda.synchronize()
            loss, leaves = eager(i)
            for leaf, want in zip(leaves, torch.autograd.grad(loss, leaves)):
                assert torch.allclose(leaf.grad, want, rtol=1e-5, atol=1e-6 * want.abs().max().item())
        torch.cuda.synchronize()

    want = [torch.autograd.grad(*eager(i)) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = torch.autograd.grad(*eager(i))
                torch.cuda.current_stream().synchronize()
                wrong.extend(i for a, b in zip(got, want[i]) if not torch.allclose(a, b, rtol=1e-5, atol=1e-6 * b.abs().max().item()))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

    terms = []
    e = torch.empty(0, 16, 4, device=dev, requires_grad=True)
    y = mlps[0](e, terms)
    grads = torch.autograd.grad(y.sum() + terms[0], [e, *mlps[0].parameters()], allow_unused=True)
    assert y.shape == (0, 16, 4) and terms[0] == 0 and not any(g.any() for g in grads if g is not None)


def test_a_module_is_copied_and_saved_after_a_call(dev):
    import copy
    mlp = fe.EquivariantExpertMLP(fe.Repr([0, 1], 8), 4, 2).to(dev)
    x = torch.randn(30, 8, 4, generator=gen(1)).to(dev)
    terms = []
    y = mlp(x, terms)
    assert torch.equal(copy.deepcopy(mlp)(x), y) and torch.equal(mlp(x), y)


@pytest.mark.parametrize("gating", [True, False])
@pytest.mark.parametrize("lvals,mult", [([0, 1, 2], 32), ([0], 8), ([0, 0, 1], 5), ([1, 2], 6), ([0, 1], 1)])
def test_one_expert_is_the_dense_mlp(dev, lvals, mult, gating):
    """With one expert (weight 1) the mixture is linear, gating, linear with that expert's weights, in 64 bits."""
    torch.manual_seed(10)
    rp = fe.Repr(lvals, mult)
    hidden = fe.Repr(lvals, 2 * mult)
    mlp = fe.EquivariantExpertMLP(rp, 1, top_k=1, use_gating=gating).to(dev)
    up, down = fe.EquivariantLinear(rp, hidden).double(), fe.EquivariantLinear(hidden, rp).double()
    act = fe.EquivariantGating(hidden).double() if gating else torch.nn.Identity()
    with torch.no_grad():
        for dense, own in ((up, mlp.up), (down, mlp.down)):
            dense.weight.copy_(own.weight[0].reshape(dense.weight.shape))
            assert (dense.bias is None) == (own.bias is None)
            if own.bias is not None:
                own.bias.normal_(generator=torch.Generator(device=dev).manual_seed(2))
                dense.bias.copy_(own.bias[0].reshape(dense.bias.shape))
        if gating:
            act.load_state_dict({k: v.double().cpu() for k, v in mlp.act.state_dict().items()})
    x = torch.randn(77, mult, rp.dim(), generator=gen(mult))
    gy = torch.randn(77, mult, rp.dim(), generator=gen(mult + 1))
    xl = x.to(dev).requires_grad_()
    y = mlp(xl)
    (gx,) = torch.autograd.grad(y, [xl], gy.to(dev))
    x64 = x.double().requires_grad_()
    with fe.utils.epsilon_dtype(torch.float32):          # the gating's norms as in float32
        y64 = down(act(up(x64)))
    (gx64,) = torch.autograd.grad(y64, [x64], gy.double())
    rel = lambda a, b: ((a.detach().double().cpu() - b).abs().max() / b.abs().max()).item()
    # sums of up to 2 mult terms twice and a gate: 64 steps of float32 at the largest value are 4e-6
    assert rel(y, y64.detach()) < 1e-5 and rel(gx, gx64) < 2e-5


# ---- gradients at places without an expert ---------------------------------------------

@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts,k", [(5, 2), (9, 4), (70, 12)])
def test_topk_gradient_at_places_without_an_expert_is_not_read(dev, experts, k, dtype, normalize):
    """Whatever gradient meets the constant weight 0 of a place without an expert, infinity and NaN too: the others
    are those of a 0 there."""
    l = torch.randn(6, experts, generator=gen(experts)).to(dev, dtype)
    l[0] = -INF
    l[1, 1:] = -INF
    l[2, k // 2:] = -INF
    l.requires_grad_()
    ids, w, _ = fe.expert_topk(l, k, normalize)
    gw = torch.randn(6, k, generator=gen(k)).to(dev)
    got = []
    for garbage in (0.0, INF, -INF, NAN):
        g = torch.where(ids < 0, torch.full_like(gw, garbage), gw)
        got.append(torch.autograd.grad([w], [l], [g], retain_graph=True)[0])
    assert (ids < 0).any() and torch.isfinite(got[0]).all()
    for other in got[1:]:
        assert torch.equal(other, got[0])


def test_a_second_backward_names_what_was_freed(dev):
    plan = fe.ExpertPlan(torch.tensor([[0, 1], [1, 0]], device=dev), 2)
    w = torch.randn(2, 1, 3, 6, device=dev, requires_grad=True)
    for call in (lambda a: plan.combine(a, torch.ones(2, 2, device=dev)), lambda a: fe.expert_linear(a, w, plan),
                 lambda a: fe.expert_topk(a, 2)[1], lambda a: fe.ops.layer_norm(a)):
        y = call(torch.randn(4, 6, device=dev, requires_grad=True)).sum()
        y.backward()
        with pytest.raises(RuntimeError, match="backward through the graph a second time"):
            y.backward()


def test_plans_made_in_inference_mode_are_for_reading(dev):
    """Changes in place are refused there as elsewhere, of copies too; unchanged plans serve in and out of the mode."""
    import copy
    x, w = torch.randn(3, 8, device=dev), torch.ones(3, 2, device=dev)
    lw = torch.randn(3, 1, 8, 8, device=dev)
    for inside in (True, False):
        with torch.inference_mode():
            ids = torch.tensor([[0, 1], [2, 0], [-1, 1]], device=dev)
            plan = fe.ExpertPlan(ids, 3)
            copied = copy.deepcopy(plan)
            late = fe.ExpertPlan(ids.int(), 3)
            ys = fe.expert_linear(plan.dispatch(x), lw, copied)
            assert torch.equal(late.combine(ys, w), plan.combine(ys, w))
        a = x.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(plan.dispatch(a).sum(), [a])[0][2], torch.ones(8, device=dev))
        for p in (plan, copied):
            with torch.inference_mode(inside):
                p.positions.clamp_(max=2)
            for mode in (True, False):
                with torch.inference_mode(mode), pytest.raises(RuntimeError, match="positions of an ExpertPlan have been modified"):
                    p.dispatch(x)
        with torch.inference_mode(inside):
            late.offsets[-1] += 1
            with pytest.raises(RuntimeError, match="offsets of an ExpertPlan have been modified"):
                fe.expert_linear(ys, lw, late)


# ---- the 16-bit mixture ----------------------------------------------------------------

def check_half_mlp(dev, dtype, gating, scale):
    """Values and gradients against the float64 formulas on the same 16-bit values, with the module's choice.

    Norms (Frobenius, |.|) bound the errors.  A table stored in the type is off by h |table|, its half step with room
    for the float32 sums; a map multiplies errors by at most its largest singular value; with the gate's matrix L,
    lambda = |L|, and rows of irrep norms n of at most N, the gate u s(L n) by 1 + lambda N / 4 (|s'| <= 1/4), and its
    derivative's own error has, relative to the gradient that comes in, h lambda N / 4 from s, and
    h lambda N (1/4 + lambda N / 10 + 1/2) from <u, g>, s' (|s''| < 1/10) and u / n."""
    torch.manual_seed(11)
    rp, k, lvals = fe.Repr([0, 1, 2], 16), 2, (0, 1, 2)
    mlp = fe.EquivariantExpertMLP(rp, 4, k, use_gating=gating).to(dev, dtype)
    on_dev = torch.Generator(device=dev).manual_seed(1)
    names = ["up.weight", "up.bias", "down.weight", "down.bias"] + ["act.linear.weight", "act.linear.bias"] * gating
    params = [dict(mlp.named_parameters())[n] for n in names]
    with torch.no_grad():
        for b in params[1::2]:
            b.normal_(generator=on_dev)
    x = (scale * torch.randn(60, 16, 9, generator=gen(12))).to(dtype)
    gy = torch.randn(60, 16, 9, generator=gen(13)).to(dtype)
    xl = x.to(dev).requires_grad_()
    with torch.no_grad():
        ids, w, mean = mlp.router(xl)
    assert w.dtype == mean.dtype == torch.float32
    y = mlp(xl)
    got = dict(zip(["y", "x"] + names, (y, *torch.autograd.grad(y, [xl, *params], gy.to(dev)))))
    assert all(t.dtype == dtype for t in got.values())

    x64, gy64 = x.double().requires_grad_(), gy.double().permute(2, 0, 1)
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in mlp.named_parameters()}
    irreps = ((0, 1), (1, 4), (4, 9))
    norms = lambda t, eps: torch.stack([(t[a:b] ** 2).sum(0) + eps for a, b in irreps], -1).sqrt()
    ids = ids.cpu()
    invariants = norms(x64.permute(2, 0, 1), 1e-5).flatten(-2)
    logits = OE.layer_norm(invariants, p["router.lnorm.weight"], p["router.lnorm.bias"]) @ p["router.linear.weight"].t()
    w64, _ = OE.topk_weights(logits, ids, True)
    assert (w.double().cpu() - w64).abs().max() < 1e-5       # float32 logits are off by less
    _, _, offsets = OE.plan(ids, 4)
    xs = OE.dispatch(x64.permute(2, 0, 1), ids, 4)
    u = OE.linear(xs, p["up.weight"], offsets, lvals, p["up.bias"])
    a, n = u, torch.zeros(1, 1, dtype=torch.float64)
    if gating:
        n = norms(u, 1e-5)
        gate = torch.sigmoid(n.flatten(-2) @ p["act.linear.weight"].t() + p["act.linear.bias"]).view(n.shape)
        a = torch.cat([u[i:j] * gate[..., r] for r, (i, j) in enumerate(irreps)])
        n = n.flatten(-2)
    s = OE.linear(a, p["down.weight"], offsets, lvals, p["down.bias"])
    y64 = OE.combine(s, w64, ids, 4)
    *gp, gx, gxs, gu, ga, gs, gw = (t.detach() for t in torch.autograd.grad(
        y64, [*(p[m] for m in names), x64, xs, u, a, s, w64], gy64, retain_graph=True))
    jac = sum(torch.autograd.grad(w64[:, i].sum(), x64, retain_graph=True)[0].flatten(1).norm(dim=1) ** 2 for i in range(k))

    f = lambda t: t.detach().norm().item()
    top = lambda t: torch.linalg.matrix_norm(t.detach(), ord=2).max().item()
    h, root = HALF[dtype] + 2.0 ** -18, ids.numel() ** 0.5
    up, down, lam = top(p["up.weight"]), top(p["down.weight"]), top(p["act.linear.weight"]) if gating else 0.0
    N = n.detach().norm(dim=-1).max().item()
    lip = 1 + lam * N / 4
    e_u = h * f(u)
    e_a = lip * e_u + h * f(a)
    e_s = down * e_a + h * f(s)
    e_y = e_s + 2e-5 * f(s) + h * f(y64)                     # weights of a row: together at most 1
    e_gs = h * f(gs) + 2e-5 * f(gy64)
    e_ga = down * e_gs + h * f(ga)
    e_gu = lip * e_ga + h * lam * N * (1 + lam * N / 10) * f(ga) + h * f(gu)
    e_gxs = up * e_gu + h * f(gxs)
    rows = OE.combine(gxs, torch.ones_like(w64), ids, 4).permute(1, 2, 0)
    e_rows = k ** 0.5 * e_gxs + h * f(rows)
    e_router = jac.max().sqrt().item() * (gy64.permute(1, 0, 2).flatten(1).norm(dim=1).max().item() * e_s + 2.0 ** -14 * f(gw)) \
        + h * f(gx - rows)
    e_q = N / 4 * e_ga + h * N * (1 / 4 + lam * N / 10) * f(ga)
    bounds = dict(zip(["y", "x"] + names, (
        e_y, e_rows + e_router + h * (f(rows) + f(gx - rows) + f(gx)),
        e_gu * f(xs) + h * f(gp[0]), root * e_gu + h * f(gp[1]),
        e_gs * (f(a) + e_a) + f(gs) * e_a + h * f(gp[2]), root * e_gs + h * f(gp[3]))))
    if gating:
        q = N / 4 * f(ga)
        bounds["act.linear.weight"] = (e_q + q * h) * f(n) + h * f(gp[4])
        bounds["act.linear.bias"] = root * e_q + h * f(gp[5])
    want = dict(zip(["y", "x"] + names, (y64.permute(1, 2, 0), gx, *gp)))
    for name, bound in bounds.items():
        err = f(got[name].double().cpu() - want[name])
        assert err <= bound + TINY[dtype] * got[name].numel(), (name, err, bound, f(want[name]))


@pytest.mark.parametrize("gating", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_precision_mlp_values(dev, dtype, gating):
    check_half_mlp(dev, dtype, gating, 1.0)


@pytest.mark.parametrize("gating", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_precision_mlp_of_large_features(dev, dtype, gating):
    """Features whose squares a float16 does not hold."""
    check_half_mlp(dev, dtype, gating, 300.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_another_activation_is_called(dev, dtype):
    """A module put in the place of the gating gets (slots, hidden, dim) features; here it scales by a power of two."""
    class Scale(torch.nn.Module):
        def forward(self, st):
            assert st.shape[1:] == (16, 4)
            return 4 * st
    torch.manual_seed(12)
    mlp = fe.EquivariantExpertMLP(fe.Repr([0, 1], 8), 3, 2, use_gating=False).to(dev, dtype)
    x = torch.randn(20, 8, 4, generator=gen(14)).to(dev, dtype)
    y = mlp(x)                                   # biases are zero
    mlp.act = Scale()
    assert y.any() and torch.equal(mlp(x), 4 * y)


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_and_subclasses_without_the_balance_argument(dev, dtype):
    """Only a call that asks for the balancing terms passes the list on."""
    class Block(fe.EquivariantTransformerBlock):
        def forward(self, P, Q, node_features, distances, graph, edge_features=None):
            return super().forward(P, Q, node_features, distances, graph, edge_features)

    class Model(fe.EquivariantTransformer):
        def forward(self, coordinates, node_features, graph):
            return super().forward(coordinates, node_features, graph)
    torch.manual_seed(13)
    rp = fe.Repr([0, 1], 16)
    model = Model(rp, rp, rp, num_layers=2, num_heads=2).to(dev, dtype)
    graph = fe.Graph.random(40, 200, device=dev)
    xyz = torch.randn(40, 3, generator=gen(15)).to(dev, dtype)
    x = torch.randn(40, 16, 4, generator=gen(16)).to(dev, dtype)
    want = fe.EquivariantTransformer.forward(model, xyz, x, graph) if dtype == torch.float32 else None
    for i in range(2):
        block = Block(rp, rp, num_heads=2).to(dev, dtype)
        block.load_state_dict(model.layers[i].state_dict())
        model.layers[i] = block
    y = model(xyz, x, graph)
    assert y.dtype == dtype and torch.isfinite(y).all() and (want is None or torch.equal(y, want))
    with pytest.raises(TypeError, match="balance"):
        fe.EquivariantTransformer.forward(model, xyz.float(), x.float(), graph, balance=[])


def test_the_most_slots(dev):
    """2^30 slots of one channel: the sort, the move and the maps at the last places and the first."""
    slots = 2 ** 30
    ids = torch.zeros(slots, dtype=torch.int8, device=dev)
    ids[0], ids[5], ids[-1], ids[-2] = 1, -1, 1, 1
    plan = fe.ExpertPlan(ids, 2)
    del ids
    assert plan.offsets.tolist() == [0, slots - 4, slots - 1]
    assert plan.order[[0, 4, slots - 4, slots - 3, slots - 2, slots - 1]].tolist() == [1, 6, 0, slots - 2, slots - 1, 5]
    assert plan.positions[[0, 1, 5, 6, slots - 1], 0].tolist() == [slots - 4, 0, slots - 1, 4, slots - 2]
    x = torch.zeros(slots, 1, device=dev, dtype=torch.bfloat16)
    x[0], x[1], x[5], x[-1] = 2.0, 3.0, NAN, 5.0
    xs = plan.dispatch(x)
    del x
    at = [0, 1, slots - 4, slots - 3, slots - 2, slots - 1]
    assert xs[at, 0].tolist() == [3, 0, 2, 0, 5, 0]
    xs[-1] = NAN
    xs.requires_grad_()
    w = torch.tensor([[[[1.0]]], [[[4.0]]]], device=dev, dtype=torch.bfloat16, requires_grad=True)
    y = fe.expert_linear(xs, w, plan)
    assert y[at, 0].tolist() == [3, 0, 8, 0, 20, 0] and not y[2:-4].any()
    gy = torch.zeros_like(y)
    gy[at] = torch.tensor([1, 2, 3, 4, 5, NAN], device=dev, dtype=torch.bfloat16)[:, None]
    gx, gw = torch.autograd.grad(y, [xs, w], gy)
    assert gx[at, 0].tolist() == [1, 2, 12, 16, 20, 0] and not gx[2:-4].any()
    assert gw.flatten().tolist() == [3, 31]


def test_weight_gradient_of_many_rows_and_a_very_large_weight(dev):
    """More than 2^30 elements of a weight whose gradient is summed from many chunks of rows."""
    from flash_eq import _native as N
    c, slots = 33001, 74000
    x, gy = (torch.zeros(1, slots, c, device=dev, dtype=torch.bfloat16) for _ in range(2))
    plan = fe.ExpertPlan(torch.zeros(slots, 1, dtype=torch.int64, device=dev), 1)
    rows = torch.arange(0, slots, 4000, device=dev)          # 19 rows, in every chunk
    x[0, rows[:, None], torch.tensor([0, 17, c - 1], device=dev)] = torch.tensor([1.0, 2.0, 3.0], device=dev, dtype=torch.bfloat16)
    gy[0, rows[:, None], torch.tensor([1, 99, c - 1], device=dev)] = torch.tensor([1.0, 4.0, 8.0], device=dev, dtype=torch.bfloat16)
    w = torch.zeros(1, 1, c, c, device=dev, dtype=torch.bfloat16, requires_grad=True)
    lvals = (N.ctypes.c_int32 * 1)(0)
    assert N.lib().feq_expert_linear_bwd_workspace(lvals, 1, 1, slots, c, c, 0) >= 18 * 4 * c * c
    y = fe.expert_linear(x, w, plan)
    (gw,) = torch.autograd.grad(y, [w], gy)
    out, inp = [0, 1, 99, c - 1], [0, 1, 17, c - 1]
    got = gw[0, 0][out][:, inp].float().cpu()
    want = 19 * torch.tensor([0.0, 1, 4, 8])[:, None] * torch.tensor([1.0, 0, 2, 3])
    assert torch.equal(got, want) and gw.count_nonzero().item() == 9


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lvals", [(0,), (0, 1)])
def test_linear_of_many_large_uneven_experts(dev, lvals, dtype):
    """Weights that outweigh the rows take longer chunks (512 and more tiles of 128 columns both ways over the
    experts and irreps): tiles in both directions, experts of no, one and several chunks, rows without an expert."""
    from flash_eq import _native as N
    cin, cout = 300, 520
    counts = [(7 * e) % 23 for e in range(64)]
    counts[40], counts[63], counts[9] = 2500, 700, 0
    assert -(-cin // 128) * -(-cout // 128) * 64 >= 512 and 0 in counts
    arr = (N.ctypes.c_int32 * len(lvals))(*lvals)
    assert N.lib().feq_expert_linear_bwd_workspace(arr, len(lvals), 64, sum(counts) + 37, cin, cout, 1) > 4 * cin * cout
    check_linear(dev, lvals, counts, 37, cin, cout, dtype, seed=21)


def hooked_calls(dev):
    """(call, its leaves) of every operator that keeps tensors for its backward."""
    g = gen(22)
    plan = fe.ExpertPlan(torch.tensor([[0, 1], [1, 0], [1, 1]], device=dev), 2)
    leaf = lambda *s: torch.randn(*s, generator=g).to(dev).requires_grad_()
    return [(lambda x, w: fe.ops.layer_norm(x, w), (leaf(5, 24), leaf(24))),
            (lambda l: fe.expert_topk(l, 2)[1], (leaf(5, 24),)),
            (lambda ys, w: plan.combine(ys, w), (leaf(4, 6, 24), leaf(3, 2))),
            (lambda x, w: fe.expert_linear(x, w, plan, (0, 1)), (leaf(4, 6, 24), leaf(2, 2, 7, 24)))]


def test_saved_tensors_come_back_in_any_layout(dev):
    """A hook may hand out a saved tensor's values with other strides."""
    turn = lambda t: t.permute(*range(t.dim() - 1, -1, -1))
    for call, leaves in hooked_calls(dev):
        gy = torch.randn(call(*leaves).shape, generator=gen(23)).to(dev)
        want = torch.autograd.grad(call(*leaves), leaves, gy)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: turn(t).contiguous(), turn):
            y = call(*leaves)
        for a, b in zip(torch.autograd.grad(y, leaves, gy), want):
            assert torch.equal(a, b)
        with torch.autograd.graph.save_on_cpu():
            y = call(*leaves)
        for a, b in zip(torch.autograd.grad(y, leaves, gy), want):
            assert torch.equal(a, b)


def test_saved_tensors_of_another_kind_are_refused(dev):
    """What a hook hands out has the kept tensor's shape, type and device, or the backward raises."""
    others = [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.double() if t.is_floating_point() else t.int(),
              lambda t: t.reshape(-1)]
    for other in others:
        for call, leaves in hooked_calls(dev):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
                y = call(*leaves)
            with pytest.raises(RuntimeError, match="a saved-tensor hook returned a"):
                y.sum().backward()


def test_two_threads_take_one_graph_backward(dev):
    """One frees what the other may be reading: each ends with the gradient or with the error of a second backward."""
    import threading
    for call, leaves in hooked_calls(dev):
        want = torch.autograd.grad(call(*leaves).sum(), leaves)
        torch.cuda.synchronize()
        for _ in range(20):
            y = call(*leaves).sum()
            ends = []

            def work():
                try:
                    ends.append(all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves), want)))
                except RuntimeError as e:
                    ends.append("a second time" in str(e))
            threads = [threading.Thread(target=work) for _ in range(2)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            assert ends == [True, True]


@pytest.mark.parametrize("lout,mult", [([0, 1, 2], 32), ([0, 1], 20)])
def test_a_block_of_one_expert_is_the_dense_block(dev, lout, mult):
    """Values and all gradients of the whole block, its residual and layer scales included."""
    torch.manual_seed(14)
    rin, rout = fe.Repr([0, 1], mult), fe.Repr(lout, mult)
    args = dict(num_heads=4, layer_scale_init=0.3)
    dense = fe.EquivariantTransformerBlock(rin, rout, **args).to(dev)
    mixed = fe.EquivariantTransformerBlock(rin, rout, num_experts=1, experts_per_node=1, **args).to(dev)
    state = {k: v for k, v in dense.state_dict().items() if not k.startswith("mlp_")}
    own = mixed.experts.state_dict()
    for name in ("up", "down"):
        own[f"{name}.weight"] = getattr(dense, f"mlp_{name}").weight.detach().view(own[f"{name}.weight"].shape)
        own[f"{name}.bias"] = torch.randn(own[f"{name}.bias"].shape, generator=gen(24)).to(dev)
        with torch.no_grad():
            getattr(dense, f"mlp_{name}").bias.copy_(own[f"{name}.bias"].view(getattr(dense, f"mlp_{name}").bias.shape))
    own.update({f"act.{k}": v for k, v in dense.mlp_act.state_dict().items()})
    mixed.load_state_dict({**state, **{f"experts.{k}": v for k, v in own.items()}})
    graph = fe.Graph.random(300, 2400, device=dev)
    vec = torch.randn(2400, 3, generator=gen(25)).to(dev)
    P, Q = fe.WignerDBasis([rin, rout]).to(dev)(vec)
    x = torch.randn(300, mult, rin.dim(), generator=gen(26)).to(dev).requires_grad_()
    gy = torch.randn(300, mult, rout.dim(), generator=gen(27)).to(dev)
    got = []
    for block in (dense, mixed):
        y = block(P, Q, x, vec.norm(dim=-1), graph)
        names = [k for k, _ in block.named_parameters() if "router" not in k]
        grads = torch.autograd.grad(y, [x] + [block.get_parameter(k) for k in names], gy)
        got.append(dict(zip(["y", "x"] + [k.replace("experts.", "mlp_") for k in names], (y.detach(), *grads))))
    assert got[0].keys() == got[1].keys()
    for k, a in got[0].items():
        b = got[1][k].view(a.shape)
        assert (a - b).abs().max() <= 2e-5 * a.abs().max(), k       # the bar of the mixture against 64 bits


def test_deterministic_algorithms(dev):
    """The setting, which fills new tensors in place, changes nothing and refuses nothing."""
    torch.manual_seed(15)
    mlp = fe.EquivariantExpertMLP(fe.Repr([0, 1], 8), 4, 2).to(dev)
    x = torch.randn(50, 8, 4, generator=gen(28)).to(dev).requires_grad_()
    leaves = [x, *mlp.parameters()]
    step = lambda: torch.autograd.grad(mlp(x).square().sum(), leaves)
    want = step()
    torch.use_deterministic_algorithms(True)
    try:
        got = step()
        with torch.inference_mode():
            y = mlp(x)
    finally:
        torch.use_deterministic_algorithms(False)
    assert torch.equal(y, mlp(x))
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6 * b.abs().max().item())


def test_gating_and_mixture_under_autocast(dev):
    """The kernels around the gating's products read float32: autocast leaves them so, forward and backward."""
    torch.manual_seed(16)
    rp = fe.Repr([0, 1], 24)
    gating, mlp = fe.EquivariantGating(rp).to(dev), fe.EquivariantExpertMLP(rp, 1, 1).to(dev)
    x = torch.randn(70, 24, 4, generator=gen(29)).to(dev).requires_grad_()
    gy = torch.randn(70, 24, 4, generator=gen(30)).to(dev)
    for module in (gating, mlp):
        leaves = [x] + [p for k, p in module.named_parameters() if "router" not in k]
        y = module(x)
        want = (y, *torch.autograd.grad(y, leaves, gy))
        for dtype in (torch.bfloat16, torch.float16):
            with torch.autocast("cuda", dtype=dtype):
                y = module(x)
                outside = torch.autograd.grad(y, leaves[:1], gy, retain_graph=True)
            got = (y, *torch.autograd.grad(y, leaves, gy))
            assert torch.equal(outside[0], got[1])
            for a, b in zip(got, want):
                assert a.dtype == torch.float32 and torch.equal(a, b)


@pytest.mark.parametrize("cin,cout,dtype", [(65536, 9, torch.bfloat16), (40, 65536, torch.float32),
                                            (65535, 130, torch.float32), (136, 65533, torch.bfloat16)])
def test_linear_of_the_most_channels(dev, cin, cout, dtype):
    check_linear(dev, (0, 1), [9, 0, 140], 2, cin, cout, dtype, seed=31)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("lead,rows,k,width,experts", [((65535,), 3, 2, 3, 4), ((3, 5), 37, 64, 9, 100), ((), 3, 64, 4099, 64),
                                                       ((300,), 2, 7, 130, 9)])
def test_rows_of_the_most_planes_and_choices(dev, lead, rows, k, width, experts, dtype):
    test_rows_and_their_gradients(dev, lead, rows, k, width, experts, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_captured_half_precision_step(dev, dtype):
    """Router and gating in float32 inside, recorded as the rest; replays on new inputs give the eager step's values."""
    from flash_eq.capture import capture_step
    torch.manual_seed(17)
    mlp = fe.EquivariantExpertMLP(fe.Repr([0, 1], 16), 4, 2).to(dev, dtype)
    x = torch.randn(900, 16, 4, generator=gen(32)).to(dev, dtype).requires_grad_()
    gy = torch.randn(900, 16, 4, generator=gen(33)).to(dev, dtype)
    leaves = [x, *mlp.parameters()]

    def loss_of():
        terms = []
        return (mlp(x, terms) * gy).float().sum((1, 2)).mean() + terms[0]

    def step():
        loss = loss_of()
        loss.backward()
        return loss
    graph, _ = capture_step(step, leaves)
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(900, 16, 4, generator=gen(50 + k)))
        graph.replay()
        torch.cuda.synchronize()
        for leaf, want in zip(leaves, torch.autograd.grad(loss_of(), leaves)):
            assert torch.isfinite(leaf.grad).all()
            # one step of the type, and what float32 sums in another order make of it
            assert torch.allclose(leaf.grad.float(), want.float(), rtol=2 * HALF[dtype], atol=HALF[dtype] * want.abs().max().item())
        torch.cuda.synchronize()
