"""The expert-routing oracle against per-row loops, closed forms and differences (float64)."""
import math

import pytest
import torch

from oracle import experts as OE


def _g(seed):
    return torch.Generator().manual_seed(seed)


def test_layer_norm_closed_form():
    x = torch.tensor([[1.0, 3.0], [-2.0, -2.0]], dtype=torch.float64)
    y = OE.layer_norm(x, eps=0.5)
    s = 1 / math.sqrt(1.5)
    assert torch.allclose(y, torch.tensor([[-s, s], [0.0, 0.0]], dtype=torch.float64), atol=1e-15)


def test_layer_norm_gradients():
    g = _g(1)
    x = torch.randn(4, 6, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(6, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(6, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(OE.layer_norm, (x, w, b), eps=1e-6, atol=1e-8)


def test_topk_ties_masks_and_nan():
    inf, nan = float("inf"), float("nan")
    l = torch.tensor([[1.0, 2.0, 2.0, 0.0], [-inf, 5.0, -inf, -inf], [-inf] * 4, [0.0, nan, 9.0, nan],
                      [0.0, -0.0, 0.0, -0.0]], dtype=torch.float64)
    assert OE.topk_ids(l, 3).tolist() == [[1, 2, 0], [1, -1, -1], [-1, -1, -1], [1, 3, 2], [0, 1, 2]]
    w, mean = OE.topk_weights(l[:3], OE.topk_ids(l[:3], 3), True)
    assert w[1].tolist() == [1.0, 0.0, 0.0] and w[2].tolist() == [0.0] * 3
    e = [math.exp(v) for v in (1.0, 2.0, 2.0, 0.0)]
    assert torch.allclose(w[0], torch.tensor([e[1], e[2], e[0]], dtype=torch.float64) / (e[0] + e[1] + e[2]))
    assert torch.allclose(mean, torch.tensor([e[0], e[1] + sum(e), e[2], e[3]], dtype=torch.float64) / sum(e) / 3)


@pytest.mark.parametrize("normalize", [True, False])
def test_topk_weight_gradients(normalize):
    l = torch.randn(5, 7, generator=_g(2), dtype=torch.float64, requires_grad=True)
    ids = OE.topk_ids(l.detach(), 3)
    assert torch.autograd.gradcheck(lambda t: OE.topk_weights(t, ids, normalize), (l,), eps=1e-6, atol=1e-8)


def test_plan_and_moves_match_loops():
    g = _g(3)
    ids = torch.randint(-1, 6, (9, 3), generator=g)          # 5 and -1: no expert of 5
    x = torch.randn(2, 9, 4, generator=g, dtype=torch.float64)
    ys = torch.randn(2, 27, 4, generator=g, dtype=torch.float64)
    w = torch.rand(9, 3, generator=g, dtype=torch.float64)
    order, positions, offsets = OE.plan(ids, 5)
    at, xs, y = 0, torch.zeros(2, 27, 4, dtype=torch.float64), torch.zeros(2, 9, 4, dtype=torch.float64)
    for e in range(6):
        assert int(offsets[e]) == at
        for slot in range(27):
            v = int(ids.view(-1)[slot])
            if (v if 0 <= v < 5 else 5) != e:
                continue
            assert int(order[at]) == slot and int(positions.view(-1)[slot]) == at
            if e < 5:
                xs[:, at] = x[:, slot // 3]
                y[:, slot // 3] += w.view(-1)[slot] * ys[:, at]
            at += 1
    assert at == 27
    assert torch.equal(OE.dispatch(x, ids, 5), xs)
    assert torch.allclose(OE.combine(ys, w, ids, 5), y, atol=1e-14)


def test_linear_matches_loop():
    g = _g(4)
    lvals, offsets = (0, 1, 0), torch.tensor([0, 2, 2, 5])
    x = torch.randn(5, 7, 3, generator=g, dtype=torch.float64)
    w = torch.randn(3, 3, 2, 3, generator=g, dtype=torch.float64)
    b = torch.randn(3, 2, 2, generator=g, dtype=torch.float64)
    y = OE.linear(x, w, offsets, lvals, b)
    irrep, col = [0, 1, 1, 1, 2], [0, None, None, None, 1]
    for d in range(5):
        for p in range(7):
            e = 0 if p < 2 else 2
            want = torch.zeros(2, dtype=torch.float64) if p >= 5 else w[e, irrep[d]] @ x[d, p]
            if p < 5 and col[d] is not None:
                want = want + b[e, :, col[d]]
            assert torch.allclose(y[d, p], want, atol=1e-14)
