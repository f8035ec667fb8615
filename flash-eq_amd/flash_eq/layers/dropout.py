"""Dropout of equivariant features: whole irreps, with masks that are never stored (``flash_eq/dropout.py``).

The reference drops attention weights alone (``attention.py:56-60``)."""
from __future__ import annotations

import torch
import torch.nn as nn

from ..dropout import dropout_seed, feature_dropout
from ..representations import Repr


class EquivariantDropout(nn.Module):
    """In training every irrep of every channel is 0 with probability ``p``, all its components together, and the others
    are multiplied by 1 / (1 - p).  Each call draws its seed from PyTorch's generator of the features' device."""

    def __init__(self, repr: Repr, p: float = 0.1) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be between 0 and 1, got {p}")
        self.repr = repr
        self.p = p
        self._lv = tuple(int(l) for l in repr.lvals.tolist())

    def forward(self, x: torch.Tensor, component_major: bool = False) -> torch.Tensor:
        """x (..., mult, dim), or (dim, ..., mult) with ``component_major``."""
        if not self.training or self.p == 0.0:
            return x
        return feature_dropout(x, self.p, dropout_seed(x.device), self._lv, component_major)

    def extra_repr(self) -> str:
        return f"{self.repr}, p={self.p}"
