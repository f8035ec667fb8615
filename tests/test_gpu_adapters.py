"""Low-rank adapters beside a shared map (csrc/adapter_linear.hip) against the float64 oracle on the same inputs.

u = 2^-24, HALF(t) half a step of the stored type t.  The matrix cores' float32 sums of n terms are counted as 2 n u of their
absolute terms.  A reduced row of a 16-bit type enters the second product as two numbers of that type: SPLIT(t) of its row's
largest value is lost (two halves of a step)."""
import pytest
import torch

import flash_eq as fe
from oracle import finetune as OF

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SPLIT = {torch.float32: 0.0, torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -16}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, tol):
    got = got.detach()
    err = (got.double().cpu() - want.detach()).abs()
    bad = ~(err <= tol + TINY[got.dtype])
    assert not bad.any(), (float((err - tol).max()), int(bad.sum()), tuple(got.shape))


def by_adapter(ids, adapters, rep, nreps, z, v):
    """(adapters, irreps, z's columns, v's columns): sums over rows and planes of z v."""
    out = torch.zeros(adapters, nreps, z.shape[-1], v.shape[-1], dtype=torch.float64)
    for a in range(adapters):
        at = (ids == a).nonzero()[:, 0]
        for d, r in enumerate(rep):
            out[a, r] += z[d, at].t() @ v[d, at]
    return out


def reduced(x, first, ids, rep, scale):
    """scale first[a] x of every row, zeros without an adapter; first (adapters, irreps, rank, columns)."""
    out = torch.zeros(*x.shape[:2], first.shape[2], dtype=torch.float64)
    for a in range(first.shape[0]):
        at = (ids == a).nonzero()[:, 0]
        for d, r in enumerate(rep):
            out[d, at] = scale * (x[d, at] @ first[a, r].t())
    return out


def check(dev, rows, lvals, ci, co, adapters, rank, dtype, *, none=0.0, bias=True, scale=0.7, seed=0, ids=None, edit=None, train=True,
          flat=False, views=None, leaves=("x", "weight", "down", "up", "bias"), weight2d=False):
    g = gen(seed + rows)
    rep = OF.irreps(lvals).tolist()
    dim, n, ns = len(rep), len(lvals), sum(l == 0 for l in lvals)
    x = torch.randn(dim, rows, ci, generator=g)
    t = dict(x=x, weight=torch.randn(n, co, ci, generator=g) / ci ** 0.5, down=torch.randn(adapters, n, rank, ci, generator=g) / ci ** 0.5,
             up=torch.randn(adapters, n, co, rank, generator=g) / rank ** 0.5)
    if bias and ns:
        t["bias"] = torch.randn(co, ns, generator=g)
    t = {k: v.to(dtype) for k, v in t.items()}
    if edit:
        edit(t)
    if ids is None:
        ids = torch.randint(0, adapters, (rows,), generator=g)
        ids[torch.rand(rows, generator=g) < none] = -1
    gy = torch.randn(dim, rows, co, generator=g).to(dtype)

    f = {k: v.double().requires_grad_() for k, v in t.items()}
    y = OF.adapter_linear(f["x"], f["weight"], f["down"], f["up"], ids, lvals, f.get("bias"), scale)
    names = [k for k in leaves if k in t]
    grads = dict(zip(f, torch.autograd.grad(y, list(f.values()), gy.double(), allow_unused=True)))
    grads = {k: torch.zeros_like(f[k]) if v is None else v for k, v in grads.items()}

    on = {k: v.to(dev) for k, v in t.items()}
    if views:
        on = {k: views(v) for k, v in on.items()}
    gyd = gy.to(dev)
    if flat:
        on["x"], gyd = on["x"][0], gyd[0]
    if weight2d:
        on["weight"] = on["weight"].view(n * co, ci)
    on = {k: v.detach().requires_grad_(k in names and train) for k, v in on.items()}
    plan = fe.ExpertPlan(ids.to(dev), adapters)

    def run():
        return fe.adapter_linear(on["x"], on["weight"], on["down"], on["up"], plan, lvals, on.get("bias"), scale)

    got = run()
    assert got.dtype == dtype and got.shape == (*on["x"].shape[:-1], co)
    a = {k: v.detach().abs() for k, v in f.items()}
    low, high = reduced(a["x"], a["down"], ids, rep, abs(scale)), reduced(gy.double().abs(), a["up"].transpose(2, 3), ids, rep, abs(scale))
    # a reduced value's error; what it does to the result
    el, eh = (2 * ci + 6) * U * low, (2 * co + 6) * U * high
    sl, sh = el + SPLIT[dtype] * low.amax(-1, keepdim=True), eh + SPLIT[dtype] * high.amax(-1, keepdim=True)

    def spread(v, second):
        """second[a] v of every row; second (adapters, irreps, columns, rank)."""
        return reduced(v, second, ids, rep, 1.0)
    base = OF.adapter_linear(a["x"], a["weight"], a["down"], a["up"], torch.full_like(ids, -1), lvals, a.get("bias"), 0.0)
    tol = (2 * ci + 2 * rank + 8) * U * (base + spread(low, a["up"])) + spread(sl, a["up"]) + HALF[dtype] * y.detach().abs()
    yy = got.detach().view(y.shape)
    within(yy, y, tol)
    if train and names:
        found = dict(zip(names, torch.autograd.grad(got, [on[k] for k in names], gyd)))
        tols = {}
        gbase = torch.stack([gy[d].double().abs() @ a["weight"][r] for d, r in enumerate(rep)]) if rows else torch.zeros(dim, 0, ci).double()
        tols["x"] = (2 * co + 2 * rank + 8) * U * (gbase + spread(high, a["down"].transpose(2, 3))) + spread(sh, a["down"].transpose(2, 3))
        terms = 2 * (rows * max(2 * l + 1 for l in lvals) + 8) * U
        ax, ag = a["x"], gy.double().abs()
        tols["down"] = by_adapter(ids, adapters, rep, n, eh, ax) + terms * by_adapter(ids, adapters, rep, n, high, ax)
        tols["up"] = by_adapter(ids, adapters, rep, n, ag, el) + terms * by_adapter(ids, adapters, rep, n, ag, low)
        tols["weight"] = terms * by_adapter(torch.zeros(rows, dtype=torch.int64), 1, rep, n, ag, ax)[0]
        if "bias" in t:
            tols["bias"] = 2 * (rows + 8) * U * torch.stack([ag[d].sum(0) for d, r in enumerate(rep) if lvals[r] == 0], 1)
        for k in names:
            want = grads[k]
            within(found[k].view(want.shape), want, tols[k] + HALF[dtype] * want.abs())
    with torch.no_grad():
        assert torch.equal(run(), got)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,lvals,ci,co,adapters,rank", [
    (1, [0], 1, 1, 1, 1), (1, [0, 1, 2], 64, 128, 8, 8), (3, [0], 4, 9, 2, 3), (17, [0, 1], 8, 8, 3, 16), (100, [0, 1, 2], 32, 64, 4, 17),
    (33, [1], 7, 5, 2, 1), (64, [0], 64, 64, 64, 33), (257, [0, 0, 1], 30, 34, 5, 4), (130, [0, 1], 128, 128, 2, 64), (40, [0], 127, 129, 7, 5),
    (50, [0, 1], 65, 33, 4, 9), (200, [0], 20, 300, 3, 48), (12, list(range(7)), 16, 24, 3, 16), (300, [0], 96, 40, 1, 20)])
def test_narrow_maps(dev, rows, lvals, ci, co, adapters, rank, dtype):
    check(dev, rows, lvals, ci, co, adapters, rank, dtype, none=0.2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,lvals,ci,co,adapters,rank", [
    (1, [0], 129, 130, 1, 1), (64, [0], 512, 256, 64, 16), (130, [0], 200, 64, 3, 33), (129, [0, 1], 160, 150, 4, 8), (300, [0], 131, 1, 5, 64),
    (77, [0, 0], 256, 7, 9, 4), (257, [0], 136, 300, 2, 20), (20, [1], 133, 133, 6, 3), (500, [0], 144, 128, 100, 12)])
def test_wide_maps(dev, rows, lvals, ci, co, adapters, rank, dtype):
    check(dev, rows, lvals, ci, co, adapters, rank, dtype, none=0.1)
    check(dev, rows, lvals, co, ci, adapters, rank, dtype, none=0.1, seed=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dev, dtype):
    """Several chunks an adapter."""
    check(dev, 5003, [0, 1], 24, 40, 3, 6, dtype, none=0.1)
    check(dev, 9001, [0], 12, 8, 1, 5, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_orders_of_the_rows(dev, dtype):
    g = gen(1)
    n = 300
    same = torch.full((n,), 2)
    for ids in (same, torch.full((n,), -1), torch.sort(torch.randint(0, 4, (n,), generator=g)).values, torch.arange(n) % 4,
                torch.randint(-3, 9, (n,), generator=g), torch.randint(0, 4, (n,), generator=g).int()):
        check(dev, n, [0, 1], 32, 48, 4, 8, dtype, ids=ids)
        check(dev, n, [0], 160, 136, 4, 8, dtype, ids=ids)


def test_limits_of_adapters_and_rank(dev):
    check(dev, 2000, [0], 16, 16, 1024, 2, torch.float32)
    check(dev, 2000, [0], 144, 16, 1024, 2, torch.bfloat16)
    check(dev, 50, [0] * 32, 8, 8, 2, 4, torch.float32)
    check(dev, 20, [6] * 9 + [5], 8, 8, 2, 4, torch.bfloat16)        # 128 components


@pytest.mark.parametrize("leaves", [("x",), ("down",), ("up",), ("down", "up"), ("weight",), ("bias",), ("x", "weight"), ("up", "bias")])
def test_gradients_one_by_one(dev, leaves):
    for ci, co in ((32, 48), (160, 136)):
        check(dev, 150, [0, 1], ci, co, 3, 8, torch.float32, leaves=leaves)


def test_shapes_and_views(dev):
    check(dev, 70, [0], 32, 48, 3, 8, torch.float32, flat=True)
    check(dev, 70, [0, 1], 32, 48, 3, 8, torch.float32, weight2d=True)
    check(dev, 70, [1, 2], 32, 48, 3, 8, torch.float32)              # no scalars, no bias
    check(dev, 70, [0, 1], 32, 48, 3, 8, torch.float32, bias=False, scale=-2.5)
    check(dev, 70, [0, 1], 32, 48, 3, 8, torch.float32, scale=0.0)
    for dtype in TYPES:
        off = lambda v: torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)
        check(dev, 70, [0, 1], 32, 48, 3, 8, dtype, views=off)
        check(dev, 70, [0], 160, 136, 3, 8, dtype, views=off)
        check(dev, 70, [0, 1], 32, 48, 3, 8, dtype, views=lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2))


def test_no_rows(dev):
    plan = fe.ExpertPlan(torch.zeros(0, dtype=torch.int64, device=dev), 3)
    t = [torch.randn(4, 0, 8, device=dev), torch.randn(2, 6, 8, device=dev), torch.randn(3, 2, 4, 8, device=dev),
         torch.randn(3, 2, 6, 4, device=dev), torch.randn(6, 1, device=dev)]
    t = [v.requires_grad_() for v in t]
    y = fe.adapter_linear(t[0], t[1], t[2], t[3], plan, [0, 1], t[4])
    assert y.shape == (4, 0, 6)
    for v, gv in zip(t, torch.autograd.grad(y.sum(), t)):
        assert torch.equal(gv, torch.zeros_like(v))


@pytest.mark.parametrize("ci,co", [(32, 48), (160, 136)])
def test_float16_reduced_rows_out_of_range(dev, ci, co):
    """Reduced rows far past float16's largest value and below its smallest, whose results it holds."""
    def large(t):
        t["down"] *= 30000.0
        t["x"] *= 50
        t["up"] /= 30000.0

    def small(t):
        t["down"] /= 2000.0
        t["x"] /= 2000
        t["up"] *= 5000.0
    for edit in (large, small):
        check(dev, 90, [0, 1], ci, co, 3, 8, torch.float16, edit=edit, train=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ci,co", [(32, 48), (17, 19), (160, 136)])
def test_nan_and_infinity_stay_in_their_rows(dev, ci, co, dtype):
    g = gen(5)
    n, rank = 100, 6
    ids = torch.randint(-1, 4, (n,), generator=g)
    t = [torch.randn(4, n, ci, generator=g), torch.randn(2, co, ci, generator=g), torch.randn(4, 2, rank, ci, generator=g),
         torch.randn(4, 2, co, rank, generator=g)]
    t = [v.to(dev, dtype) for v in t]
    gy = torch.randn(4, n, co, generator=g).to(dev, dtype)

    def run(x, down, up):
        plan = fe.ExpertPlan(ids.to(dev), 4)
        x, down, up = (v.clone().requires_grad_() for v in (x, down, up))
        y = fe.adapter_linear(x, t[1], down, up, plan, [0, 1])
        return (y.detach(), *torch.autograd.grad(y, [x, down, up], gy))

    clean = run(t[0], t[2], t[3])
    x = t[0].clone()
    row = int((ids == 1).nonzero()[0])
    free = int((ids == -1).nonzero()[0])
    x[:, row, 3], x[0, free, 0] = INF, NAN
    y, gx, gd, gu = run(x, t[2], t[3])
    others = [i for i in range(n) if i not in (row, free)]
    assert torch.equal(y[:, others], clean[0][:, others]) and torch.equal(gx, clean[1])
    assert not y[:, row].isfinite().any() and y[0, free].isnan().all() and torch.equal(y[1:, free], clean[0][1:, free])
    for got, want in ((gd, clean[2]), (gu, clean[3])):               # adapter 1 alone
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and not got[1].isfinite().all()
    down, up = t[2].clone(), t[3].clone()
    down[2], up[2] = NAN, INF                                         # another adapter's rows see nothing of it
    y, gx, gd, gu = run(t[0], down, up)
    keep = ids.to(dev) != 2
    assert torch.equal(y[:, keep], clean[0][:, keep]) and torch.equal(gx[:, keep], clean[1][:, keep])
    assert torch.equal(gd[[0, 1, 3]], clean[2][[0, 1, 3]]) and torch.equal(gu[[0, 1, 3]], clean[3][[0, 1, 3]])


def test_deterministic_changed_plan_and_second_backward(dev):
    g = gen(6)
    ids = torch.randint(0, 5, (3000,), generator=g).to(dev)
    x, w = torch.randn(4, 3000, 64, generator=g).to(dev), torch.randn(2, 96, 64, generator=g).to(dev)
    d, u = torch.randn(5, 2, 16, 64, generator=g).to(dev), torch.randn(5, 2, 96, 16, generator=g).to(dev)
    leaves = [v.requires_grad_() for v in (x, w, d, u)]
    plan = fe.ExpertPlan(ids, 5)
    runs = []
    for _ in range(3):
        y = fe.adapter_linear(x, w, d, u, plan, [0, 1])
        runs.append((y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)
    y = fe.adapter_linear(x, w, d, u, plan, [0, 1])
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        gx.sum().backward()
    y = fe.adapter_linear(x, w, d, u, plan, [0, 1])
    plan.order.add_(0)
    with pytest.raises(RuntimeError, match="modified in place"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="modified in place"):
        fe.adapter_linear(x, w, d, u, plan, [0, 1])


@pytest.mark.parametrize("ci,co", [(64, 96), (160, 136)])
def test_captured_step(dev, ci, co):
    from flash_eq.capture import capture_step
    g = gen(7)
    ids = torch.randint(-1, 5, (2000,), generator=g).to(dev)
    t = [torch.randn(4, 2000, ci, generator=g), torch.randn(2, co, ci, generator=g), torch.randn(5, 2, 16, ci, generator=g),
         torch.randn(5, 2, co, 16, generator=g)]
    t = [v.to(dev).requires_grad_() for v in t]

    def step():
        y = fe.adapter_linear(t[0], t[1], t[2], t[3], fe.ExpertPlan(ids, 5), [0, 1])
        y.backward(torch.ones_like(y))
        return y

    graph, y = capture_step(step, t)
    for _ in range(3):
        for v in t:
            v.grad.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        got = [y.detach().clone()] + [v.grad.clone() for v in t]
        new = [v.detach().clone().requires_grad_() for v in t]
        z = fe.adapter_linear(new[0], new[1], new[2], new[3], fe.ExpertPlan(ids, 5), [0, 1])
        for a, b in zip(got, (z.detach(), *torch.autograd.grad(z, new, torch.ones_like(z)))):
            assert torch.equal(a, b)
        with torch.no_grad():
            t[0].mul_(0.5)


@pytest.mark.parametrize("rows,lvals,ci,co,rank", [(1_050_005, [0], 2048, 16, 12), (350_003, list(range(7)), 128, 128, 8)])
def test_offsets_past_32_bits(dev, rows, lvals, ci, co, rank):
    """The ends of tables of more than 4 GB.  All values are 0 and +-1 (a reduced row's sums are below 2^16: two bfloat16 numbers
    hold them), and gradients reach 30 rows at either end, so sums are of whole numbers below 2^24 and exact."""
    g = gen(5)
    rep, n, ends = OF.irreps(lvals).tolist(), len(lvals), 30
    dim = len(rep)

    def signs(*s):
        return torch.randint(-1, 2, s, generator=g).to(torch.bfloat16)
    w, down, up = signs(n, co, ci), signs(2, n, rank, ci), signs(2, n, co, rank)
    x_at, gy_at = signs(dim, 2 * ends, ci), signs(dim, 2 * ends, co)
    ids = torch.randint(0, 2, (rows,), generator=g)
    x, gy = (torch.zeros(dim, rows, c, dtype=torch.bfloat16, device=dev) for c in (ci, co))
    for full, part in ((x, x_at), (gy, gy_at)):
        full[:, :ends], full[:, -ends:] = part[:, :ends].to(dev), part[:, ends:].to(dev)
    f = [t.double().requires_grad_() for t in (x_at, w, down, up)]
    y64 = OF.adapter_linear(*f, torch.cat([ids[:ends], ids[-ends:]]), lvals, None, 1.0)
    want = torch.autograd.grad(y64, f, gy_at.double())
    leaves = [x.requires_grad_(), *(t.to(dev).requires_grad_() for t in (w, down, up))]
    y = fe.adapter_linear(*leaves, fe.ExpertPlan(ids.to(dev), 2), lvals)
    grads = torch.autograd.grad(y, leaves, gy)
    both = torch.cat([y.detach()[:, :ends], y.detach()[:, -ends:]], 1)
    assert torch.equal(both.cpu(), y64.detach().to(torch.bfloat16)) and not y.detach()[:, ends:-ends].any()
    gx = torch.cat([grads[0][:, :ends], grads[0][:, -ends:]], 1)
    assert torch.equal(gx.cpu(), want[0].to(torch.bfloat16)) and not grads[0][:, ends:-ends].any()
    for a, b in zip(grads[1:], want[1:]):
        assert torch.equal(a.cpu().view(b.shape), b.to(torch.bfloat16))
    del x, gy, y, grads, leaves, both, gx
    torch.cuda.empty_cache()
