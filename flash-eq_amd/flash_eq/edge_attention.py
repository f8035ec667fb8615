"""Attention weights of edges with a learned bias for each head and bucket of distances, and dropout.

The edge attention of the reference (``attention.py:92-141``) has a fixed distance decay and PyTorch's dropout; here the
logits get a learned table's entry for the edge's bucket (a relative position bias), and the weights' dropout is
formed inside the kernels (``dropout.py``).  Argument checks and autograd are ``csrc/torch_nodes.cpp``, the kernels
``csrc/edge_attention.hip``.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native as N
from .graph import Graph

MAX_BUCKETS = 4096


def distance_buckets(distances: torch.Tensor, boundaries: torch.Tensor) -> torch.Tensor:
    """The bucket (edges,) int32 of every distance: the number of ``boundaries`` (ascending) that are at most the
    distance, so n boundaries make n + 1 buckets.  Both float32.  A NaN has bucket 0.  No gradient."""
    return N.nodes().distance_buckets(distances, boundaries)


def edge_attention_weights(qk: torch.Tensor, graph: Graph, num_heads: int, log_scale: torch.Tensor, *,
                           component_major: bool = False, distances: Optional[torch.Tensor] = None, decay: float = 0.0,
                           bias: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                           dropout: float = 0.0, seed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights (edges, heads) of every edge over the edges into its destination:

        softmax(exp(log_scale) <Q[dst], K[src]> - distances / decay + bias[buckets])

    with the reference's 1e-8 in the denominator, then dropout of the weights with share ``dropout`` from ``seed`` (one
    int64, ``dropout_seed``; unit: edge x heads + head).

    qk (nodes, 2 mult, dim), or (dim, nodes, 2 mult) with ``component_major``: the queries in channels [0, mult), the
    keys in the rest, ``num_heads`` dividing mult.  log_scale: one number.  bias (buckets, heads), at most 4096 buckets;
    buckets (edges,) int32 or int64, an edge whose bucket lies outside gets no bias.  decay 0: none.  float32, float16
    or bfloat16, the bias and log_scale of any of them; sums are float32, the result has qk's dtype.

    A bias of -inf forbids a bucket: its edges have weight 0 and pass no gradient, whatever their keys hold, and a node
    that no other edge reaches has weights 0.  A NaN or +inf among a node's other logits makes its head's weights NaN.
    Gradients reach qk, log_scale, bias and distances.  Edges whose source lies outside the graph see keys of 0, those
    whose destination does have weight 0."""
    perm, offsets = graph.csr()
    perm_s, offsets_s = graph.csr_src()
    return N.nodes().edge_attention(qk, None, graph.src, graph.dst, perm, offsets, perm_s, offsets_s, graph.num_nodes,
                                    graph.num_edges, num_heads, log_scale, component_major, distances, decay, bias, buckets,
                                    dropout, seed)


def edge_attention_weights_qk(Q: torch.Tensor, K: torch.Tensor, graph: Graph, log_scale: torch.Tensor, *,
                              distances: Optional[torch.Tensor] = None, decay: float = 0.0,
                              bias: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                              dropout: float = 0.0, seed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``edge_attention_weights`` of the edges' own queries and keys (edges, heads, head dim)."""
    perm, offsets = graph.csr()
    return N.nodes().edge_attention(Q, K, None, None, perm, offsets, None, None, graph.num_nodes, graph.num_edges,
                                    Q.shape[1] if Q.dim() == 3 else 0, log_scale, False, distances, decay, bias, buckets,
                                    dropout, seed)
