"""Fine-tuning operators (oracle, float64): counter-based dropout, biased edge attention, low-rank adapters.

No counterpart in the reference; the formulas are those of ``include/flasheq.h``.  Values and gradients come from
autograd through these forms.  Pinned by ``tests/test_oracle_finetune.py``: the generator's published known answers,
loops, closed forms and differences.
"""
from __future__ import annotations

import torch

MASK = 0xFFFFFFFF


def philox(counter, key):
    """Four words from four counter words and two key words (Salmon et al., SC 2011), ten rounds, by Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & MASK, (a >> 32) ^ c[3] ^ k[1], a & MASK]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return c


def factors(seed, units, p):
    """The dropout's factor of units 0 .. units - 1 (float64)."""
    seed &= (1 << 64) - 1
    limit = int(p * 65536 + 0.5)
    out = []
    for b in range((units + 7) // 8):
        for w in philox((b & MASK, b >> 32, 0, 0), (seed & MASK, seed >> 32)):
            out += [w & 0xFFFF, w >> 16]
    scale = 65536.0 / (65536 - limit) if limit < 65536 else 0.0
    return torch.tensor([0.0 if v < limit else scale for v in out[:units]], dtype=torch.float64)


def irreps(lvals):
    """The irrep of every component."""
    return torch.tensor([r for r, l in enumerate(lvals) for _ in range(2 * l + 1)])


def dropout(x, p, seed, lvals=None, component_major=False):
    """0 where dropped, whatever x holds."""
    if lvals is None:
        f = factors(seed, x.numel(), p).view(x.shape)
    else:
        rep, n = irreps(lvals), x.numel() // sum(2 * l + 1 for l in lvals)
        f = factors(seed, n * len(lvals), p).view(n, len(lvals))[:, rep]          # (row-channels, dim)
        f = f.t().reshape(x.shape) if component_major else f.reshape(x.shape)
    return torch.where(f == 0, torch.zeros_like(x), x * f)


def buckets(dist, bounds):
    return torch.tensor([sum(1 for b in bounds.tolist() if b <= r) for r in dist.tolist()], dtype=torch.int64)


def edge_attention(q, k, dst, num_nodes, log_scale, dist=None, decay=0.0, bias=None, bucket=None, p=0.0, seed=0):
    """q, k (edges, heads, head dim) of every edge; the weights (edges, heads)."""
    E, H, _ = q.shape
    z = (q * k).sum(-1) * log_scale.exp()
    if decay > 0:
        z = z - dist[:, None] / decay
    forbidden = torch.zeros(E, H, dtype=torch.bool)
    if bias is not None:
        known = (bucket >= 0) & (bucket < bias.shape[0])
        b = torch.where(known[:, None], bias[bucket.clamp(0, bias.shape[0] - 1)], torch.zeros_like(z))
        forbidden = b.detach() == float("-inf")
        z = z + torch.where(forbidden, torch.zeros_like(b), b)
    cols = []
    for n in range(num_nodes):
        at = (dst == n).nonzero()[:, 0]
        for h in range(H):
            live = at[~forbidden[at, h]]
            if live.numel():
                u = torch.exp(z[live, h] - z[live, h].detach().max())
                cols.append((live * H + h, u / (u.sum() + 1e-8)))
    w = torch.zeros(E * H, dtype=z.dtype)
    if cols:
        w = w.index_put((torch.cat([c[0] for c in cols]),), torch.cat([c[1] for c in cols]))
    if p > 0:
        f = factors(seed, E * H, p)
        w = torch.where(f == 0, torch.zeros_like(w), w * f)
    return w.view(E, H)


def rows_at(table, idx):
    """table[idx], zeros where an index lies outside."""
    inside = (idx >= 0) & (idx < table.shape[0])
    rows = table[idx.clamp(0, table.shape[0] - 1)]
    return torch.where(inside.view(-1, *[1] * (table.dim() - 1)), rows, torch.zeros_like(rows))


def node_qk(qk, heads, src, dst, component_major=False):
    """(edges, heads, head dim) queries and keys from the table of the nodes."""
    if component_major:
        qk = qk.permute(1, 2, 0)
    n, two, dim = qk.shape
    q = qk[:, :two // 2].reshape(n, heads, -1)
    k = qk[:, two // 2:].reshape(n, heads, -1)
    return rows_at(q, dst), rows_at(k, src)


def adapter_linear(x, weight, down, up, ids, lvals, bias=None, scale=1.0):
    """x (dim, rows, cin), weight (irreps, cout, cin), down (adapters, irreps, rank, cin), up (adapters, irreps, cout, rank)."""
    rep = irreps(lvals)
    scalars = [r for r, l in enumerate(lvals) if l == 0]
    y = torch.stack([x[d] @ weight[r].t() for d, r in enumerate(rep.tolist())])
    low = torch.zeros_like(y)
    for a in range(down.shape[0]):
        at = (ids == a).nonzero()[:, 0]
        if at.numel():
            own = torch.stack([(x[d, at] @ down[a, r].t()) @ up[a, r].t() for d, r in enumerate(rep.tolist())])
            low = low.index_copy(1, at, own)
    y = y + scale * low
    if bias is not None:
        column = torch.zeros(len(rep), weight.shape[1], dtype=y.dtype)
        for j, r in enumerate(scalars):
            column = column + (rep == r).to(y.dtype)[:, None] * bias[:, j]
        y = y + column[:, None]
    return y
