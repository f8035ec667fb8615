"""Mixture of experts over nodes: router, per-expert linear maps, the experts' MLP.

The block's node MLP (``transformer.py:187-206`` of the reference: linear, gating, linear) with a
weight per expert.  A router chooses ``top_k`` experts of every node from its invariants (the
norms of its irreps), so the choice does not depend on the frame and the mixture stays
equivariant.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
import torch.nn as nn

from ..experts import MAX_EXPERTS, MAX_TOP_K, ExpertPlan, expert_linear, expert_topk
from ..representations import Repr
from ..utils import epsilon_dtype
from ._precision import half_dtype, run_float32, up_all
from .gating import EquivariantGating
from .norm import InvariantLayerNorm, RepNorm


class ExpertRouter(nn.Module):
    """The experts of every node: layer norm of its invariants, a linear map to one logit per
    expert, the ``top_k`` largest with softmax weights (``expert_topk``).

    float16 and bfloat16 features and parameters go through it in float32 (the squares of float16 features
    pass its range from 256 on, and logits of 16 bits tie)."""

    def __init__(self, repr: Repr, num_experts: int, top_k: int = 2, normalize: bool = True) -> None:
        super().__init__()
        if not 1 <= num_experts <= MAX_EXPERTS:
            raise ValueError(f"num_experts must be 1 to {MAX_EXPERTS}, got {num_experts}")
        if not 1 <= top_k <= min(num_experts, MAX_TOP_K):
            raise ValueError(f"top_k must be 1 to num_experts (at most {MAX_TOP_K}), got {top_k} of {num_experts}")
        self.num_experts = num_experts
        self.top_k = top_k
        self.normalize = normalize
        width = repr.nreps() * repr.mult
        self.norm = RepNorm(repr)
        self.lnorm = InvariantLayerNorm(width)
        self.linear = nn.Linear(width, num_experts, bias=False)
        nn.init.xavier_uniform_(self.linear.weight)

    def forward(self, st: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(nodes, mult, dim) to ids (nodes, top_k), weights (nodes, top_k), mean probabilities."""
        half = half_dtype(st)
        if half is not None:
            with epsilon_dtype(half):
                return torch.func.functional_call(self, up_all(self.named_parameters()), (st.float(),))
        invariants = self.norm(st).flatten(-2, -1)
        return expert_topk(self.linear(self.lnorm(invariants)), self.top_k, self.normalize)

    def balance(self, plan: ExpertPlan, mean: torch.Tensor) -> torch.Tensor:
        """num_experts * sum over the experts of (share of the routed slots) * (mean probability): 1 for
        an even load, num_experts when one expert takes all.  Its gradient goes through the means."""
        counts = (plan.offsets[1:] - plan.offsets[:-1]).to(mean.dtype)
        return self.num_experts * (counts * mean).sum() / plan.offsets[-1].clamp(min=1)

    def extra_repr(self) -> str:
        return f"num_experts={self.num_experts}, top_k={self.top_k}, normalize={self.normalize}"


class EquivariantExpertLinear(nn.Module):
    """``EquivariantLinear`` with a weight and bias per expert, on component-major rows in expert
    order: (dim, slots, in_mult) to (dim, slots, out_mult)."""

    def __init__(self, in_repr: Repr, out_repr: Repr, num_experts: int, bias: bool = True) -> None:
        super().__init__()
        if not torch.equal(in_repr.lvals, out_repr.lvals):
            raise ValueError(
                "EquivariantExpertLinear cannot modify the degrees of a representation. "
                f"Got input lvals={in_repr.lvals.tolist()}, output lvals={out_repr.lvals.tolist()}")
        self.in_repr = in_repr
        self.out_repr = out_repr
        self.num_experts = num_experts
        self.weight = nn.Parameter(torch.empty(num_experts, in_repr.nreps(), out_repr.mult, in_repr.mult))
        for e in range(num_experts):         # as EquivariantLinear's (irreps * out_mult, in_mult) weight
            nn.init.xavier_uniform_(self.weight.data[e].view(-1, in_repr.mult))
        nscalar, _ = in_repr.find_scalar()
        self.bias: nn.Parameter | None
        if nscalar > 0 and bias:
            self.bias = nn.Parameter(torch.zeros(num_experts, out_repr.mult, nscalar))
        else:
            self.bias = None
        self._lv = tuple(int(l) for l in in_repr.lvals.tolist())

    def forward(self, x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
        return expert_linear(x, self.weight, plan, self._lv, self.bias)

    def extra_repr(self) -> str:
        return f"in_repr={self.in_repr}, out_repr={self.out_repr}, num_experts={self.num_experts}"


class EquivariantExpertMLP(nn.Module):
    """The gated node MLP as a mixture of experts: (nodes, mult, dim) to the same.

    Every node's row goes to its ``top_k`` experts (``ExpertRouter``), through their maps up, the
    gating (shared by the experts) and their maps down, and the results are summed with the
    router's weights.  float16 and bfloat16 features keep their type between these steps; router and gating
    run in float32 inside.  ``forward(x, balance=terms)`` appends the router's balancing term to the list
    ``terms``, for the training loss (the module keeps nothing of a call, so no graph outlives it)."""

    def __init__(self, repr: Repr, num_experts: int, top_k: int = 2, mlp_ratio: int = 2, use_gating: bool = True,
                 normalize: bool = True) -> None:
        super().__init__()
        hidden = Repr(lvals=repr.lvals, mult=repr.mult * mlp_ratio)
        self.repr = repr
        self.router = ExpertRouter(repr, num_experts, top_k, normalize)
        self.up = EquivariantExpertLinear(repr, hidden, num_experts)
        self.act: nn.Module = EquivariantGating(hidden) if use_gating else nn.Identity()
        self.down = EquivariantExpertLinear(hidden, repr, num_experts)

    def forward(self, x: torch.Tensor, balance: Optional[List[torch.Tensor]] = None) -> torch.Tensor:
        if x.dim() != 3 or x.shape[1:] != (self.repr.mult, self.repr.dim()):
            raise ValueError(f"node features must be (nodes, {self.repr.mult}, {self.repr.dim()}), got {tuple(x.shape)}")
        ids, weights, mean = self.router(x)
        plan = ExpertPlan(ids, self.router.num_experts)
        if balance is not None:
            balance.append(self.router.balance(plan, mean))
        # component-major (dim, nodes, mult): the layout of the maps and the gating
        h = self.up(plan.dispatch(x.permute(2, 0, 1).contiguous()), plan)
        if isinstance(self.act, EquivariantGating) and self.act.kernels_ok(h):
            h = self.act.forward_cm(h)
        elif type(self.act) is not nn.Identity:
            nodes, half = h.permute(1, 2, 0), half_dtype(h)
            nodes = self.act(nodes) if half is None else run_float32(self.act, half, (nodes,), {})
            h = nodes.permute(2, 0, 1).contiguous()
        return plan.combine(self.down(h, plan), weights).permute(1, 2, 0).contiguous()

    def extra_repr(self) -> str:
        return f"{self.repr}"
