"""The tiled product of the adapters (csrc/adapter_linear.hip, k_ad_mm) against the float64 oracle.  It serves reductions above
128 columns whose blocks of 128 rows and columns, over all planes, are 128 or more; fewer go to k_ad_few, which the sizes of
``test_gpu_adapters.py`` reach.  Bounds: that file's."""
import pytest
import torch

import flash_eq as fe
from test_gpu_adapters import INF, NAN, TYPES, check, gen

pytestmark = pytest.mark.gpu


def tiled(rows, lvals, k, n):
    """Whether a product of k reduction columns and n results' takes 128-row tiles."""
    return k > 128 and -(-rows // 128) * -(-n // 128) * sum(2 * l + 1 for l in lvals) >= 128


HIGH = list(range(7))                                              # 49 planes


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,lvals,ci,co,adapters,rank", [
    (300, HIGH, 136, 160, 5, 16), (333, HIGH, 131, 150, 1, 3), (300, HIGH, 257, 300, 12, 64), (385, HIGH, 144, 129, 100, 20),
    (8200, [0], 256, 130, 7, 33), (2100, [0, 1], 160, 136, 3, 1)])
def test_both_directions_tiled(dev, rows, lvals, ci, co, adapters, rank, dtype):
    assert tiled(rows, lvals, ci, co) and tiled(rows, lvals, co, ci)
    check(dev, rows, lvals, ci, co, adapters, rank, dtype, none=0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,lvals,wide,narrow,adapters,rank", [
    (400, HIGH, 200, 7, 100, 33), (390, HIGH, 136, 64, 6, 16), (2100, [0, 1, 2], 130, 1, 4, 5), (16300, [0], 192, 33, 9, 8)])
def test_one_direction_tiled(dev, rows, lvals, wide, narrow, adapters, rank, dtype):
    """Results of at most 64 columns, rows of fewer than 16 bytes among them: the forward, then grad_x."""
    assert tiled(rows, lvals, wide, narrow)
    check(dev, rows, lvals, wide, narrow, adapters, rank, dtype, none=0.1)
    check(dev, rows, lvals, narrow, wide, adapters, rank, dtype, none=0.1, seed=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_orders_of_the_rows_tiled(dev, dtype):
    """Blocks of one adapter, of none, of many, and some of both."""
    g, n = gen(2), 2100
    assert tiled(n, [0, 1], 160, 136) and tiled(n, [0, 1], 136, 160)
    for ids in (torch.full((n,), 2), torch.full((n,), -1), torch.arange(n) // 130 % 4, torch.randint(-3, 9, (n,), generator=g)):
        check(dev, n, [0, 1], 160, 136, 4, 8, dtype, ids=ids)


@pytest.mark.parametrize("leaves", [("x",), ("down",), ("up",), ("down", "up"), ("weight",), ("bias",), ("x", "weight"), ("up", "bias")])
def test_gradients_one_by_one_tiled(dev, leaves):
    check(dev, 2100, [0, 1], 160, 136, 3, 8, torch.bfloat16, leaves=leaves, none=0.1)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_tiled(dev, dtype):
    """Tables an element off every vector, and transposed ones."""
    check(dev, 2100, [0, 1], 160, 136, 3, 8, dtype, views=lambda v: torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape))
    check(dev, 2100, [0, 1], 160, 136, 3, 8, dtype, views=lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2), scale=-2.5)


def test_float16_reduced_rows_out_of_range_tiled(dev):
    def large(t):
        t["down"] *= 30000.0
        t["x"] *= 50
        t["up"] /= 30000.0

    def small(t):
        t["down"] /= 2000.0
        t["x"] /= 2000
        t["up"] *= 5000.0
    for edit in (large, small):
        check(dev, 2100, [0, 1], 160, 136, 3, 8, torch.float16, edit=edit, train=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinity_stay_in_their_rows_tiled(dev, dtype):
    """A tile's rows have several adapters or none: what one adapter's maps or one row holds reaches no other row."""
    g, n, ci, co, rank = gen(5), 2100, 136, 160, 6
    ids = torch.randint(-1, 4, (n,), generator=g)
    t = [torch.randn(4, n, ci, generator=g), torch.randn(2, co, ci, generator=g), torch.randn(4, 2, rank, ci, generator=g),
         torch.randn(4, 2, co, rank, generator=g)]
    t = [v.to(dev, dtype) for v in t]
    gy = torch.randn(4, n, co, generator=g).to(dev, dtype)

    def run(x, down, up, gy=gy):
        plan = fe.ExpertPlan(ids.to(dev), 4)
        x, down, up = (v.clone().requires_grad_() for v in (x, down, up))
        y = fe.adapter_linear(x, t[1], down, up, plan, [0, 1])
        return (y.detach(), *torch.autograd.grad(y, [x, down, up], gy))

    clean = run(t[0], t[2], t[3])
    row, free = int((ids == 1).nonzero()[0]), int((ids == -1).nonzero()[0])
    others = [i for i in range(n) if i not in (row, free)]
    x = t[0].clone()
    x[:, row, 3], x[0, free, 0] = INF, NAN
    y, gx, gd, gu = run(x, t[2], t[3])
    assert torch.equal(y[:, others], clean[0][:, others]) and torch.equal(gx, clean[1])
    assert not y[:, row].isfinite().any() and y[0, free].isnan().all() and torch.equal(y[1:, free], clean[0][1:, free])
    for got, want in ((gd, clean[2]), (gu, clean[3])):               # adapter 1 alone
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and not got[1].isfinite().all()
    bad = gy.clone()
    bad[:, row, 3], bad[0, free, 0] = INF, NAN
    y, gx, gd, gu = run(t[0], t[2], t[3], bad)
    assert torch.equal(y, clean[0]) and torch.equal(gx[:, others], clean[1][:, others]) and not gx[:, row].isfinite().any()
    for got, want in ((gd, clean[2]), (gu, clean[3])):
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and not got[1].isfinite().all()
    down, up = t[2].clone(), t[3].clone()
    down[2], up[2] = NAN, INF                                         # another adapter's rows see nothing of it
    y, gx, gd, gu = run(t[0], down, up)
    keep = ids.to(dev) != 2
    assert torch.equal(y[:, keep], clean[0][:, keep]) and torch.equal(gx[:, keep], clean[1][:, keep])
    assert torch.equal(gd[[0, 1, 3]], clean[2][[0, 1, 3]]) and torch.equal(gu[[0, 1, 3]], clean[3][[0, 1, 3]])
