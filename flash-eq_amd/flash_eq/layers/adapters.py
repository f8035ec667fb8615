"""Low-rank adapters of ``EquivariantLinear`` maps: one trained model for several data sets, tasks or requests.

``add_adapters(model, n, rank)`` gives every ``EquivariantLinear`` of a model ``n`` adapters; a call with ``adapters`` (the
nodes' adapter ids, or the plan made of them) adds to every map, for each node, the low-rank map of its adapter
(``flash_eq/adapters.py``).  A new adapter changes nothing: its ``up`` maps are zero.  No counterpart in the reference.
"""
from __future__ import annotations

import math
from typing import List, Optional, Union

import torch
import torch.nn as nn

from ..adapters import MAX_RANK, adapter_linear
from ..experts import MAX_EXPERTS, ExpertPlan
from ..representations import Repr

Adapters = Union[torch.Tensor, ExpertPlan]


class LinearAdapters(nn.Module):
    """The adapters of one ``EquivariantLinear``: per adapter and irrep ``down`` (rank, in_mult), random, and ``up``
    (out_mult, rank), zero; their product is scaled by ``alpha`` / rank (1 without ``alpha``)."""

    def __init__(self, in_repr: Repr, out_repr: Repr, num_adapters: int, rank: int = 8, alpha: Optional[float] = None) -> None:
        super().__init__()
        if not 1 <= num_adapters <= MAX_EXPERTS:
            raise ValueError(f"num_adapters must be 1 to {MAX_EXPERTS}, got {num_adapters}")
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"rank must be 1 to {MAX_RANK}, got {rank}")
        self.num_adapters = num_adapters
        self.rank = rank
        self.scale = 1.0 if alpha is None else alpha / rank
        if not math.isfinite(self.scale):
            raise ValueError(f"alpha must be finite, got {alpha}")
        n, bound = in_repr.nreps(), in_repr.mult ** -0.5
        self.down = nn.Parameter(torch.empty(num_adapters, n, rank, in_repr.mult).uniform_(-bound, bound))
        self.up = nn.Parameter(torch.zeros(num_adapters, n, out_repr.mult, rank))
        self._lv = tuple(int(l) for l in in_repr.lvals.tolist())

    def forward(self, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], plan: ExpertPlan) -> torch.Tensor:
        """The shared map with the rows' adapters, on component-major x (dim, rows, in_mult)."""
        if plan.num_experts != self.num_adapters:
            raise ValueError(f"a plan for {plan.num_experts} adapters, the layer has {self.num_adapters}")
        return adapter_linear(x, weight, self.down, self.up, plan, self._lv, bias, self.scale)

    def extra_repr(self) -> str:
        return f"num_adapters={self.num_adapters}, rank={self.rank}, scale={self.scale}"


def add_adapters(module: nn.Module, num_adapters: int, rank: int = 8, alpha: Optional[float] = None) -> List[nn.Parameter]:
    """Gives every ``EquivariantLinear`` of ``module`` ``num_adapters`` adapters and returns their parameters, on the maps'
    device and in their type (the maps themselves are left as they are: freeze them to train the adapters alone)."""
    from .linear import EquivariantLinear
    found = [m for m in module.modules() if isinstance(m, EquivariantLinear)]
    if not found:
        raise ValueError("the module has no EquivariantLinear")
    params: List[nn.Parameter] = []
    for linear in found:
        params += linear.add_adapters(num_adapters, rank, alpha)
    return params


def adapter_plan(module: nn.Module, adapters: Optional[Adapters]) -> Optional[ExpertPlan]:
    """The plan of the nodes' adapter ids (a plan itself, or None, as it is)."""
    if adapters is None or isinstance(adapters, ExpertPlan):
        return adapters
    count = next((m.num_adapters for m in module.modules() if isinstance(m, LinearAdapters)), None)
    if count is None:
        raise ValueError("adapters were given to a module that has none (add_adapters)")
    return ExpertPlan(adapters, count)


def wanted(**options) -> dict:
    """The keywords of a call that are given: modules and subclasses without the others stay callable, and a hook that
    returns a new input leaves them alone."""
    return {k: v for k, v in options.items() if v is not None}
