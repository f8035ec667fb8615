"""Low-rank adapters of many rows at once beside a shared channel map.

``EquivariantLinear`` (``linear.py:242-268`` of the reference, which has no counterpart of the adapters) with, for
every row, the low-rank map of its adapter added: one model for several data sets, tasks or requests, whose rows share
a batch.  Argument checks and autograd are ``csrc/torch_nodes.cpp``, the kernels ``csrc/adapter_linear.hip``.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _native as N
from .experts import ExpertPlan

MAX_RANK = 64


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor, plan: ExpertPlan,
                   lvals: Sequence[int] = (0,), bias: Optional[torch.Tensor] = None, scale: float = 1.0) -> torch.Tensor:
    """weight x + scale up[a] (down[a] x) (+ bias on the scalars), a the adapter of the row, for every irrep.

    x (dim, rows, cin), component-major, with dim the components of ``lvals`` (or (rows, cin) for the scalars alone,
    lvals (0,)), the rows in any order; ``plan``: ``ExpertPlan(ids, adapters)`` of the rows' adapters (rows,), made once
    for all maps of a model, a row whose id lies outside having none.  weight (irreps, cout, cin), or (irreps cout, cin)
    as ``EquivariantLinear``'s; down (adapters, irreps, rank, cin), up (adapters, irreps, cout, rank), rank at most 64;
    bias (cout, scalar irreps) or None; all of one dtype (float32, float16 or bfloat16), sums in float32.  Returns (dim,
    rows, cout).  Gradients reach x, weight, down, up and bias; an adapter without rows gets zeros."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f"plan must be an ExpertPlan, got {type(plan).__name__}")
    return N.nodes().adapter_linear(x, weight, down, up, bias, plan.order, plan.offsets, plan.num_rows, plan.top_k, lvals, scale)
