"""Routing of rows to experts: the choice, the sort by expert and back, the experts' maps.

The pieces of a mixture-of-experts node MLP (``layers/experts.py``); the reference has one
dense MLP for all nodes (``transformer.py:187-206``) and no counterpart.  Everything runs on GPU
tensors in float32, float16 or bfloat16 with float32 sums, on the current stream, without a host
synchronisation: an expert's number of rows stays on the device.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .ops import _c, _lvals_i32, _same_device, element_type

MAX_EXPERTS = 1024
MAX_TOP_K = 64
_INDEX_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---- the choice of the experts ---------------------------------------------------------

class ExpertTopKFn(torch.autograd.Function):
    """``feq_expert_topk_fwd`` / ``_bwd`` on logits (rows, experts)."""

    @staticmethod
    def run(logits, top_k: int, normalize: bool):
        rows, experts = logits.shape
        dev = logits.device
        lc = logits.detach().contiguous()
        ids = torch.empty(rows, top_k, dtype=torch.int64, device=dev)
        weights = torch.empty(rows, top_k, dtype=torch.float32, device=dev)
        mean = torch.empty(experts, dtype=torch.float32, device=dev)
        lib = N.lib()
        ws = N.workspace(lib.feq_expert_topk_workspace(rows, experts), dev)
        with N.on_device(dev):
            rc = lib.feq_expert_topk_fwd(N.ptr(lc), rows, experts, N.DTYPES[lc.dtype], top_k, int(normalize),
                                         N.ptr(ids), N.ptr(weights), N.ptr(mean), N.ptr(ws), ws.numel(),
                                         N.stream_ptr(dev))
        N.check(rc, "feq_expert_topk_fwd")
        return lc, ids, weights, mean

    @staticmethod
    def forward(ctx, logits, top_k, normalize):
        lc, ids, weights, mean = ExpertTopKFn.run(logits, top_k, normalize)
        ctx.save_for_backward(lc, ids, weights)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, weights, mean

    @staticmethod
    @once_differentiable
    def backward(ctx, _gids, gw, gmean):
        lc, ids, weights = ctx.saved_tensors
        if gw is None and gmean is None:
            return None, None, None
        gw = gw.float().contiguous() if gw is not None else None
        gmean = gmean.float().contiguous() if gmean is not None else None
        rows, experts = lc.shape
        dev = lc.device
        gl = torch.empty_like(lc)
        with N.on_device(dev):
            rc = N.lib().feq_expert_topk_bwd(N.ptr(lc), N.ptr(ids), N.ptr(weights), N.ptr(gw), N.ptr(gmean), rows,
                                             experts, N.DTYPES[lc.dtype], ids.shape[1], int(ctx.normalize), N.ptr(gl),
                                             N.stream_ptr(dev))
        N.check(rc, "feq_expert_topk_bwd")
        return gl, None, None


def expert_topk(logits: torch.Tensor, top_k: int,
                normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``top_k`` experts of the largest logits of every row.

    logits (..., experts).  Returns ids (..., top_k) int64, largest first and equal logits by the
    lowest index (a NaN counts as the largest); weights (..., top_k) float32, the softmax over all
    experts at the chosen ones, divided by their sum with ``normalize``; and the mean over the rows of
    the softmax (experts,) float32, for a balancing loss.  An expert whose logit is -inf is never
    chosen: its place holds id -1, which ``ExpertPlan`` leaves unrouted, and weight 0.  Gradients of
    the weights and the mean reach the logits."""
    element_type(logits, "logits")
    if logits.dim() < 1:
        raise ValueError("logits must be (..., experts)")
    experts = logits.shape[-1]
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be 1 to {MAX_EXPERTS}, got {experts}")
    if not 1 <= top_k <= min(experts, MAX_TOP_K):
        raise ValueError(f"top_k must be 1 to {min(experts, MAX_TOP_K)} of {experts} experts, got {top_k}")
    flat = logits.reshape(-1, experts)
    if _wants_grad(logits):
        ids, weights, mean = ExpertTopKFn.apply(flat, int(top_k), bool(normalize))
    else:
        _, ids, weights, mean = ExpertTopKFn.run(flat, int(top_k), bool(normalize))
    if logits.dim() != 2:
        ids, weights = (t.view(*logits.shape[:-1], top_k) for t in (ids, weights))
    return ids, weights, mean


# ---- rows into expert order and back ---------------------------------------------------

def _combine(plan: "ExpertPlan", ys: torch.Tensor, weights: Optional[torch.Tensor]) -> torch.Tensor:
    planes, width = plan._planes(ys, "ys", plan.num_slots)
    y = torch.empty(*ys.shape[:-2], plan.num_rows, width, dtype=ys.dtype, device=ys.device)
    if y.numel():
        dev = ys.device
        with N.on_device(dev):
            rc = N.lib().feq_expert_combine(N.ptr(ys), planes, plan.num_rows, plan.top_k, width, N.DTYPES[ys.dtype],
                                            N.ptr(plan.positions), plan._placed(), N.ptr(weights),
                                            N.DTYPES[weights.dtype] if weights is not None else 0, N.ptr(y),
                                            N.stream_ptr(dev))
        N.check(rc, "feq_expert_combine")
    return y


class DispatchFn(torch.autograd.Function):
    """xs[d, positions[t, k]] = x[d, t] (``feq_expert_dispatch``); its gradient sums a row's places
    in the order of its choices (``feq_expert_combine`` without weights)."""

    @staticmethod
    def run(plan, x):
        planes, width = plan._planes(x, "x", plan.num_rows)
        xc = x.detach().contiguous()
        xs = torch.empty(*x.shape[:-2], plan.num_slots, width, dtype=x.dtype, device=x.device)
        if xs.numel():
            dev = x.device
            with N.on_device(dev):
                rc = N.lib().feq_expert_dispatch(N.ptr(xc), planes, plan.num_rows, plan.top_k, width,
                                                 N.DTYPES[x.dtype], N.ptr(plan.positions), plan._placed(), N.ptr(xs),
                                                 N.stream_ptr(dev))
            N.check(rc, "feq_expert_dispatch")
        return xs

    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return DispatchFn.run(plan, x)

    @staticmethod
    @once_differentiable
    def backward(ctx, gxs):
        return _combine(ctx.plan, gxs.contiguous(), None), None


class CombineFn(torch.autograd.Function):
    """y[d, t] = sum_k weights[t, k] ys[d, positions[t, k]] (``feq_expert_combine`` / ``_bwd``)."""

    @staticmethod
    def forward(ctx, ys, weights, plan):
        yc, wc = ys.detach().contiguous(), weights.detach().contiguous()
        ctx.save_for_backward(yc, wc)
        ctx.plan = plan
        return _combine(plan, yc, wc)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        ys, weights = ctx.saved_tensors
        plan = ctx.plan
        need_y, need_w, _ = ctx.needs_input_grad
        planes, width = plan._planes(ys, "ys", plan.num_slots)
        dev = ys.device
        gys = torch.empty_like(ys) if need_y else None
        gw = torch.empty_like(weights) if need_w else None
        if ys.numel():
            g = gy.contiguous()
            with N.on_device(dev):
                rc = N.lib().feq_expert_combine_bwd(N.ptr(g), N.ptr(ys), planes, plan.num_rows, plan.top_k, width,
                                                    N.DTYPES[ys.dtype], N.ptr(plan.positions), plan._placed(),
                                                    N.ptr(weights), N.DTYPES[weights.dtype], N.ptr(gys), N.ptr(gw),
                                                    N.stream_ptr(dev))
            N.check(rc, "feq_expert_combine_bwd")
        elif gw is not None:
            gw.zero_()
        return gys, gw, None


class ExpertPlan:
    """The slots (row t, choice k) of ``ids`` (rows, top_k) sorted by expert.

    ids: the experts of every row (``expert_topk``), any integer type; an id outside
    [0, num_experts) leaves the slot without an expert.  Slot t * top_k + k:

    * ``order`` (slots,) int32: the slot at every place, experts in order, an expert's slots in
      theirs, slots without an expert last;
    * ``positions`` (rows, top_k) int32: the place of every slot;
    * ``offsets`` (num_experts + 1,) int32: every expert's first place; the last one is the number
      of slots with an expert.

    ``dispatch`` copies rows to their places, ``combine`` sums them back with weights."""

    def __init__(self, ids: torch.Tensor, num_experts: int) -> None:
        N.require_cuda_tensor(ids, "ids")
        if ids.dtype not in _INDEX_TYPES:
            raise TypeError(f"ids must be integers, got {ids.dtype}")
        if ids.dim() not in (1, 2):
            raise ValueError(f"ids must be (rows, top_k) or (rows,), got shape {tuple(ids.shape)}")
        if not 1 <= num_experts <= MAX_EXPERTS:
            raise ValueError(f"num_experts must be 1 to {MAX_EXPERTS}, got {num_experts}")
        top_k = ids.shape[1] if ids.dim() == 2 else 1
        if not 1 <= top_k <= MAX_TOP_K:
            raise ValueError(f"top_k must be 1 to {MAX_TOP_K}, got {top_k}")
        self.num_experts = int(num_experts)
        self.num_rows = ids.shape[0]
        self.top_k = top_k
        self.num_slots = self.num_rows * top_k
        if self.num_slots > 2 ** 30:
            raise ValueError(f"more than 2^30 slots: {self.num_slots}")
        dev = self.device = ids.device
        flat = ids.detach().to(torch.int64).contiguous()
        self.order = torch.empty(self.num_slots, dtype=torch.int32, device=dev)
        self.positions = torch.empty(self.num_rows, top_k, dtype=torch.int32, device=dev)
        self.offsets = torch.empty(self.num_experts + 1, dtype=torch.int32, device=dev)
        lib = N.lib()
        need = lib.feq_expert_plan_workspace(self.num_slots, self.num_experts)
        ws = N.workspace(need, dev) if need else None
        with N.on_device(dev):
            rc = lib.feq_expert_plan(N.ptr(flat), self.num_slots, self.num_experts, N.ptr(self.order),
                                     N.ptr(self.positions), N.ptr(self.offsets), N.ptr(ws), need, N.stream_ptr(dev))
        N.check(rc, "feq_expert_plan")

    def _placed(self) -> int:
        """The address of the number of slots with an expert."""
        return self.offsets.data_ptr() + 4 * self.num_experts

    def _planes(self, t: torch.Tensor, name: str, rows: int) -> Tuple[int, int]:
        element_type(t, name)
        if t.device != self.device:
            raise ValueError(f"tensors on different devices: {self.device} and {t.device}")
        if t.dim() < 2 or t.shape[-2] != rows:
            raise ValueError(f"{name} must be (..., {rows}, width), got shape {tuple(t.shape)}")
        planes = 1
        for n in t.shape[:-2]:
            planes *= n
        return planes, t.shape[-1]

    def dispatch(self, x: torch.Tensor) -> torch.Tensor:
        """x (..., rows, width) to (..., slots, width): every place its slot's row, zeros at the
        places without an expert.  The gradient of a row is the sum over its places, in the order of
        its choices."""
        self._planes(x, "x", self.num_rows)
        return DispatchFn.apply(x, self) if _wants_grad(x) else DispatchFn.run(self, x)

    def combine(self, ys: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """ys (..., slots, width) to (..., rows, width): the sum over a row's choices of weight times
        the row at the choice's place, over the choices with an expert (none: zeros).  weights (rows,
        top_k), float32, float16 or bfloat16.  Gradients for both."""
        self._planes(ys, "ys", self.num_slots)
        element_type(weights, "weights")
        if weights.dim() == 1 and self.top_k == 1:
            weights = weights.unsqueeze(1)
        if weights.shape != (self.num_rows, self.top_k):
            raise ValueError(f"weights must be ({self.num_rows}, {self.top_k}), got shape {tuple(weights.shape)}")
        _same_device(ys, weights)
        if _wants_grad(ys, weights):
            return CombineFn.apply(ys, weights, self)
        return _combine(self, ys.detach().contiguous(), weights.detach().contiguous())

    def __repr__(self) -> str:
        return f"ExpertPlan(rows={self.num_rows}, top_k={self.top_k}, num_experts={self.num_experts})"


# ---- the experts' maps -----------------------------------------------------------------

@lru_cache(maxsize=256)
def _bias_columns(lvals: Tuple[int, ...]) -> Tuple[int, ...]:
    """Per irrep: its column among the scalar irreps, -1 for the others."""
    cols, j = [], 0
    for l in lvals:
        cols.append(j if l == 0 else -1)
        j += l == 0
    return tuple(cols)


class ExpertLinearFn(torch.autograd.Function):
    """``feq_expert_linear_fwd`` / ``_bwd_x`` / ``_bwd_w``."""

    @staticmethod
    def run(x, weight, bias, plan, lvals):
        dim, slots, cin = x.shape
        cout = weight.shape[2]
        dev = x.device
        xc, wc, bc = x.detach().contiguous(), weight.detach().contiguous(), _c(bias)
        y = torch.empty(dim, slots, cout, dtype=x.dtype, device=dev)
        with N.on_device(dev):
            rc = N.lib().feq_expert_linear_fwd(_lvals_i32(lvals), len(lvals), plan.num_experts, slots, cin, cout,
                                               N.DTYPES[x.dtype], N.ptr(xc), N.ptr(wc), N.ptr(plan.offsets), N.ptr(bc),
                                               bc.shape[2] if bc is not None else 0, _lvals_i32(_bias_columns(lvals)),
                                               N.ptr(y), N.stream_ptr(dev))
        N.check(rc, "feq_expert_linear_fwd")
        return y, xc, wc

    @staticmethod
    def forward(ctx, x, weight, bias, plan, lvals):
        y, xc, wc = ExpertLinearFn.run(x, weight, bias, plan, lvals)
        ctx.save_for_backward(xc, wc)
        ctx.plan, ctx.lvals = plan, lvals
        ctx.nbias = bias.shape[2] if bias is not None else 0
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, w = ctx.saved_tensors
        plan, lvals = ctx.plan, ctx.lvals
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dim, slots, cin = x.shape
        experts, nreps, cout, _ = w.shape
        dev = x.device
        code = N.DTYPES[x.dtype]
        g = gy.contiguous()
        lib = N.lib()
        lv = _lvals_i32(lvals)
        gx = gw = gb = None
        with N.on_device(dev):
            if need_x:
                gx = torch.empty_like(x)
                N.check(lib.feq_expert_linear_bwd_x(lv, nreps, experts, slots, cin, cout, code, N.ptr(g), N.ptr(w),
                                                    N.ptr(plan.offsets), N.ptr(gx), N.stream_ptr(dev)),
                        "feq_expert_linear_bwd_x")
            if need_w or need_b:
                nb = ctx.nbias if need_b else 0
                gw = torch.empty_like(w)
                gb = torch.empty(experts, cout, nb, dtype=x.dtype, device=dev) if need_b else None
                ws = N.workspace(lib.feq_expert_linear_bwd_w_workspace(nreps, experts, slots, cin, cout, nb), dev)
                N.check(lib.feq_expert_linear_bwd_w(lv, nreps, experts, slots, cin, cout, code, N.ptr(g), N.ptr(x),
                                                    N.ptr(plan.offsets), nb, _lvals_i32(_bias_columns(lvals)),
                                                    N.ptr(gw), N.ptr(gb), N.ptr(ws), ws.numel(), N.stream_ptr(dev)),
                        "feq_expert_linear_bwd_w")
        return gx, gw if need_w else None, gb, None, None


def expert_linear(x: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan, lvals: Sequence[int] = (0,),
                  bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every expert's channel map of its rows: ``EquivariantLinear`` with a weight per expert, on
    component-major rows in expert order (``ExpertPlan.dispatch``).

    x (dim, slots, cin) with dim the components of ``lvals`` (or (slots, cin) for the scalars
    alone, lvals (0,)); weight (experts, irreps, cout, cin); bias (experts, cout, scalar irreps) or
    None, added to the scalar irreps; all of one dtype (float32, float16 or bfloat16).  Returns (dim,
    slots, cout); zeros in the rows without an expert, which enter no gradient."""
    lvals = tuple(int(l) for l in lvals)
    if not lvals or min(lvals) < 0:
        raise ValueError(f"lvals must be non-negative degrees, got {lvals}")
    for t, name in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is not None:
            element_type(t, name)
            if t.dtype != x.dtype:
                raise TypeError(f"x and {name} of different dtypes: {x.dtype} and {t.dtype}")
    _same_device(x, weight, bias, plan.offsets)
    dim = sum(2 * l + 1 for l in lvals)
    flat = x.dim() == 2 and lvals == (0,)
    x3 = x.unsqueeze(0) if flat else x
    if weight.dim() != 4 or weight.shape[0] != plan.num_experts or weight.shape[1] != len(lvals):
        raise ValueError(f"weight must be ({plan.num_experts}, {len(lvals)}, cout, cin), got shape {tuple(weight.shape)}")
    cout, cin = weight.shape[2:]
    if x3.dim() != 3 or x3.shape != (dim, plan.num_slots, cin):
        raise ValueError(f"x must be ({dim}, {plan.num_slots}, {cin}), got shape {tuple(x.shape)}")
    if cin < 1 or cout < 1:
        raise ValueError(f"weight has no channels: shape {tuple(weight.shape)}")
    nscalar = sum(l == 0 for l in lvals)
    if bias is not None and (nscalar == 0 or bias.shape != (plan.num_experts, cout, nscalar)):
        raise ValueError(f"bias must be ({plan.num_experts}, {cout}, {nscalar}), one column per scalar irrep, "
                         f"got shape {tuple(bias.shape)}")
    if _wants_grad(x, weight, bias):
        y = ExpertLinearFn.apply(x3, weight, bias, plan, lvals)
    else:
        y = ExpertLinearFn.run(x3, weight, bias, plan, lvals)[0]
    return y.squeeze(0) if flat else y
