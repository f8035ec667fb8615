"""What a call of the adapters keeps until its backward."""
import pytest
import torch

import flash_eq as fe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trained", [("down",), ("x", "weight"), ("up",)])
def test_reduced_rows_are_kept_for_the_gradient_of_up_alone(dev, trained):
    rows, ci, co, rank = 1 << 16, 160, 24, 16
    g = torch.Generator().manual_seed(1)
    t = dict(x=torch.randn(1, rows, ci, generator=g), weight=torch.randn(1, co, ci, generator=g),
             down=torch.randn(2, 1, rank, ci, generator=g), up=torch.randn(2, 1, co, rank, generator=g))
    t = {k: v.to(dev).requires_grad_(k in trained) for k, v in t.items()}
    plan = fe.ExpertPlan(torch.zeros(rows, dtype=torch.int64, device=dev), 2)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    y = fe.adapter_linear(t["x"], t["weight"], t["down"], t["up"], plan)
    kept = torch.cuda.memory_allocated(dev) - before - y.numel() * 4
    assert (kept >= rows * rank * 4) == ("up" in trained) and (kept == 0 or "up" in trained)
    grads = torch.autograd.grad(y, [t[k] for k in trained], torch.ones_like(y))

    def gradient(k, of):
        """In float64; of the absolute values: the sum of the gradient's absolute terms."""
        d = {n: of(v.detach().double()).requires_grad_(n == k) for n, v in t.items()}
        w = d["weight"][0] + d["up"][0, 0] @ d["down"][0, 0]
        return torch.autograd.grad((d["x"][0] @ w.t()).sum(), d[k])[0]
    for k, got in zip(trained, grads):
        # products and sums of that many terms in float32, the matrix cores' counted twice
        tol = 2 * (rows + ci + co + rank + 8) * 2.0 ** -24 * gradient(k, torch.abs)
        assert ((got.double() - gradient(k, lambda v: v)).abs() <= tol).all(), k
