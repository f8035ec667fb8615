"""Dropout of whole irreps from a counter-based generator.

The mask is a function of the seed and of the place alone: it is formed again in the backward and never
stored, and is the same for node-major and component-major tables.  The kernel is ``csrc/dropout.hip``, the
generator ``csrc/philox.h``.  The reference has PyTorch's dropout on the attention weights alone
(``attention.py:56-60``) and no counterpart.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _native as N


def dropout_seed(device) -> torch.Tensor:
    """A new seed (one int64) on the GPU from PyTorch's generator of that device: ``torch.manual_seed`` fixes the
    sequence, and a captured call draws another seed on every replay."""
    return torch.empty(1, dtype=torch.int64, device=device).random_()


def feature_dropout(x: torch.Tensor, p: float, seed: torch.Tensor, lvals: Optional[Sequence[int]] = None,
                    component_major: bool = False) -> torch.Tensor:
    """x with a share ``p`` of its units set to 0 and the others multiplied by 1 / (1 - p).

    ``lvals``: the degrees of x's irreps; x is (..., mult, dim), or (dim, ..., mult) with ``component_major``, and a
    unit is an irrep of a channel, whose components are dropped together (the result stays equivariant).  None: a unit
    is an element, whatever x's shape.  ``seed``: one int64 on x's device (``dropout_seed``); one seed, one mask, so a
    call for other features takes another.  float32, float16 or bfloat16; at most 32 irreps and 128 components.

    The share that is dropped is ``p`` to the nearest 65536th, from 0 to 1.  What is dropped is 0 whatever it held; its
    gradient too."""
    return N.nodes().feature_dropout(x, p, seed, lvals, component_major)
