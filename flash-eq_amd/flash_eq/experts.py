"""Routing of rows to experts: the choice, the sort by expert and back, the experts' maps.

The pieces of a mixture-of-experts node MLP (``layers/experts.py``); the reference has one
dense MLP for all nodes (``transformer.py:187-206``) and no counterpart.  Everything runs on GPU
tensors in float32, float16 or bfloat16 with float32 sums, on the current stream, without a host
synchronisation: an expert's number of rows stays on the device.  Argument checks, autograd and
the launches are ``csrc/torch_nodes.cpp``; the kernels ``csrc/expert_*.hip``.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _native as N

MAX_EXPERTS = 1024
MAX_TOP_K = 64


def expert_topk(logits: torch.Tensor, top_k: int,
                normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``top_k`` experts of the largest logits of every row.

    logits (..., experts), at most 1024 experts and 64 choices.  Returns ids (..., top_k) int64,
    largest first and equal logits by the lowest index (a NaN counts as the largest); weights (...,
    top_k) float32, the softmax over all experts at the chosen ones, divided by their sum with
    ``normalize``; and the mean over the rows of the softmax (experts,) float32, for a balancing loss.
    An expert whose logit is -inf is never chosen: its place holds id -1, which ``ExpertPlan`` leaves
    unrouted, and weight 0.  Gradients of the weights and the mean reach the logits."""
    return N.nodes().expert_topk(logits, top_k, normalize)


class ExpertPlan:
    """The slots (row t, choice k) of ``ids`` (rows, top_k) sorted by expert.

    ids: the experts of every row (``expert_topk``), any integer type; an id outside
    [0, num_experts) leaves the slot without an expert.  At most 1024 experts, 64 choices a row and
    2^30 slots.  Slot t * top_k + k:

    * ``order`` (slots,) int32: the slot at every place, experts in order, an expert's slots in
      theirs, slots without an expert last;
    * ``positions`` (rows, top_k) int32: the place of every slot;
    * ``offsets`` (num_experts + 1,) int32: every expert's first place; the last one is the number
      of slots with an expert.

    They and the sizes are for reading: kernels write where they point, and a plan whose positions or offsets
    have been modified in place is refused.  ``dispatch`` copies rows to their places, ``combine`` sums them
    back with weights."""

    def __init__(self, ids: torch.Tensor, num_experts: int) -> None:
        self._order, self._positions, self._offsets = N.nodes().expert_plan(ids, num_experts)

    @property
    def num_experts(self) -> int:
        return self._offsets.shape[0] - 1

    @property
    def num_rows(self) -> int:
        return self._positions.shape[0]

    @property
    def top_k(self) -> int:
        return self._positions.shape[1]

    @property
    def num_slots(self) -> int:
        return self._positions.numel()

    @property
    def order(self) -> torch.Tensor:
        return self._order

    @property
    def positions(self) -> torch.Tensor:
        return self._positions

    @property
    def offsets(self) -> torch.Tensor:
        return self._offsets

    def __getstate__(self) -> dict:
        # a copy counts changes from its own beginning: one of a changed plan would be taken
        for name in ("order", "positions", "offsets"):
            if getattr(self, name)._version != 0:
                raise RuntimeError(f"the {name} of an ExpertPlan have been modified in place")
        return self.__dict__

    def __setstate__(self, state: dict) -> None:
        # of a copy or a pickle, whose tensors were filled in place
        copy = N.nodes().plan_copy
        self.__dict__.update({k: copy(v) if isinstance(v, torch.Tensor) else v for k, v in state.items()})

    def dispatch(self, x: torch.Tensor) -> torch.Tensor:
        """x (..., rows, width) to (..., slots, width): every place its slot's row, zeros at the
        places without an expert.  The gradient of a row is the sum over its places, in the order of
        its choices."""
        return N.nodes().expert_dispatch(x, self._positions, self._offsets)

    def combine(self, ys: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """ys (..., slots, width) to (..., rows, width): the sum over a row's choices of weight times
        the row at the choice's place, over the choices with an expert (none: zeros).  weights (rows,
        top_k), float32, float16 or bfloat16.  Gradients for both."""
        return N.nodes().expert_combine(ys, weights, self._positions, self._offsets)

    def __repr__(self) -> str:
        return f"ExpertPlan(rows={self.num_rows}, top_k={self.top_k}, num_experts={self.num_experts})"


def expert_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, lvals: Sequence[int] = (0,),
                  bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every expert's channel map of its rows: ``EquivariantLinear`` with a weight per expert, on
    component-major rows in expert order (``ExpertPlan.dispatch``).

    x (dim, slots, cin) with dim the components of ``lvals`` (or (slots, cin) for the scalars
    alone, lvals (0,)); weight (experts, irreps, cout, cin); bias (experts, cout, scalar irreps) or
    None, added to the scalar irreps; all of one dtype (float32, float16 or bfloat16).  Returns (dim,
    slots, cout); zeros in the rows without an expert, which enter no gradient."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f"plan must be an ExpertPlan, got {type(plan).__name__}")
    return N.nodes().expert_linear(x, weight, bias, plan.offsets, plan.num_slots, lvals)
