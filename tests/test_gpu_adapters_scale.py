"""Small scales of the adapters in float16, whose rows of reduced values are multiplied by powers of two on their way into the second
product: the shared map's part of the result must not leave float32 with them."""
import pytest
import torch

from test_gpu_adapters import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-6, 1e-12, -1e-24, 1e-36, 1e-44])
@pytest.mark.parametrize("rows,lvals,ci,co,rank", [
    (90, [0, 1], 32, 48, 8),            # streamed, one backward kernel
    (90, [0, 1], 32, 48, 40),           # streamed, three rank tiles
    (90, [0, 1], 160, 136, 8),          # few rows
    (2100, [0, 1], 160, 136, 8)])       # tiles
def test_small_scales(dev, rows, lvals, ci, co, rank, scale):
    def larger(t):
        t["x"] *= 30                    # results of about 100 and gradients of about 3
    check(dev, rows, lvals, ci, co, 3, rank, torch.float16, scale=scale, edit=larger, none=0.1)
