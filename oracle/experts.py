"""Mixture-of-experts routing and the plain layer norm (oracle, float64).

No counterpart in the reference; the formulas are those of ``include/flasheq.h``.  Values and
gradients come from autograd through these forms.  Pinned by ``tests/test_oracle_experts.py``: per-row
and per-slot loops, closed forms and differences.
"""
from __future__ import annotations

import torch


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    mu = x.mean(-1, keepdim=True)
    var = ((x - mu) ** 2).mean(-1, keepdim=True)
    y = (x - mu) / torch.sqrt(var + eps)
    if weight is not None:
        y = y * weight
    return y if bias is None else y + bias


def topk_ids(logits, k):
    """The k largest of every row, equal ones by the lowest index, NaN the largest, -inf as -1."""
    key = torch.where(torch.isnan(logits), torch.full_like(logits, float("inf")), logits)
    nan = torch.isnan(logits)
    ids = torch.full((logits.shape[0], k), -1, dtype=torch.int64)
    for r in range(logits.shape[0]):
        order = sorted(range(logits.shape[1]), key=lambda i: (not bool(nan[r, i]), -float(key[r, i]), i))
        for j, i in enumerate(order[:k]):
            if float(key[r, i]) != float("-inf"):
                ids[r, j] = i
    return ids


def softmax(logits):
    """Softmax whose rows of -inf alone are 0."""
    dead = torch.isinf(logits).all(-1, keepdim=True) & (logits < 0).all(-1, keepdim=True)
    p = torch.softmax(logits.masked_fill(dead, 0.0), -1)
    return p.masked_fill(dead, 0.0)


def topk_weights(logits, ids, normalize):
    """Weights at the chosen ids (0 at -1) and the mean probability of every expert."""
    p = softmax(logits)
    live = ids >= 0
    safe = ids.clamp(min=0)
    if normalize:
        chosen = logits.gather(1, safe).masked_fill(~live, float("-inf"))
        w = softmax(chosen)
    else:
        w = p.gather(1, safe).masked_fill(~live, 0.0)
    mean = p.sum(0) / max(logits.shape[0], 1)
    return w, mean


def plan(ids, num_experts):
    """(order, positions, offsets) of the slots sorted by expert, the unrouted ones last."""
    flat = ids.reshape(-1)
    key = torch.where((flat < 0) | (flat >= num_experts), torch.full_like(flat, num_experts), flat)
    order = torch.argsort(key, stable=True)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel())
    offsets = torch.tensor([int((key < e).sum()) for e in range(num_experts + 1)])
    return order, positions.view(ids.shape), offsets


def dispatch(x, ids, num_experts):
    order, _, offsets = plan(ids, num_experts)
    k = ids.shape[1]
    n = int(offsets[-1])
    xs = torch.zeros(*x.shape[:-2], order.numel(), x.shape[-1], dtype=x.dtype)
    return xs.index_copy(-2, torch.arange(n), x.index_select(-2, order[:n] // k))


def combine(ys, weights, ids, num_experts):
    order, _, offsets = plan(ids, num_experts)
    k = ids.shape[1]
    n = int(offsets[-1])
    rows = ys.index_select(-2, torch.arange(n)) * weights.reshape(-1)[order[:n]].unsqueeze(-1)
    y = torch.zeros(*ys.shape[:-2], ids.shape[0], ys.shape[-1], dtype=ys.dtype)
    return y.index_add(-2, order[:n] // k, rows)


def linear(x, weight, offsets, lvals, bias=None):
    """x (dim, slots, cin), weight (experts, irreps, cout, cin), bias (experts, cout, scalars)."""
    dim, slots, _ = x.shape
    planes, d, j = [], 0, 0
    off = [int(v) for v in offsets]
    for r, l in enumerate(lvals):
        for _ in range(2 * l + 1):
            parts = []
            for e in range(weight.shape[0]):
                y = x[d, off[e]:off[e + 1]] @ weight[e, r].t()
                if l == 0 and bias is not None:
                    y = y + bias[e, :, j]
                parts.append(y)
            parts.append(torch.zeros(slots - off[-1], weight.shape[2], dtype=x.dtype))
            planes.append(torch.cat(parts))
            d += 1
        j += l == 0
    assert d == dim
    return torch.stack(planes)


def expert_mlp(x, ids, weights, p, lvals, eps):
    """EquivariantExpertMLP behind its router: x (nodes, mult, dim); p: up_w, up_b, gate_w, gate_b, down_w,
    down_b; the gating sigmoid(Linear(irrep norms)) per irrep and channel."""
    experts = p["up_w"].shape[0]
    _, _, offsets = plan(ids, experts)
    h = linear(dispatch(x.permute(2, 0, 1), ids, experts), p["up_w"], offsets, lvals, p["up_b"])
    comps, a = [], 0
    for l in lvals:
        comps.append((a, a + 2 * l + 1))
        a += 2 * l + 1
    norms = torch.stack([(h[a:b] ** 2).sum(0) for a, b in comps], -1)        # (slots, mult, irreps)
    lin = torch.sqrt(norms + eps).flatten(-2) @ p["gate_w"].t() + p["gate_b"]
    gate = torch.sigmoid(lin).view(norms.shape)
    h = torch.cat([h[a:b] * gate[..., i] for i, (a, b) in enumerate(comps)])
    y = combine(linear(h, p["down_w"], offsets, lvals, p["down_b"]), weights, ids, experts)
    return y.permute(1, 2, 0)
