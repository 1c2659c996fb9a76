"""Gated linear layer: ``y = act(x Wg^T + bg) * (x Wu^T + bu)`` in one kernel.

The first half of a gated feed-forward block (GEGLU, SwiGLU): both
projections, the activation and the product, with the second half,
``linear_act(y, w_down, b_down, residual)``, next to it in rocps/ops/linear.py.
``weight`` holds Wg's F rows and then Wu's F rows, so that it is the weight of
one ``nn.Linear(K, 2 * F)``, and ``bias`` likewise.

The kernel reads x once for both projections and keeps their sums of the same
columns in the same lanes, so neither projection is written to memory but
where the backward pass needs it.  Types, strides, ``checkpoint="8bit"`` and
the CPU path are as in rocps/ops/linear.py.  The backward pass:

    dg = dy * u * act'(g)     du = dy * act(g)     (rounded to the type)
    dx = [dg du] W            dW = [dg du]^T x     db = column sums
"""

from __future__ import annotations

from typing import Optional

import torch

from rocps.ops.linear import _ACTS, layer

__all__ = ["gated_linear"]

_GATES = {name: a for name, a in _ACTS.items() if name is not None}


def gated_linear(x: torch.Tensor, weight: torch.Tensor,
                 bias: Optional[torch.Tensor] = None, *,
                 activation: str = "silu",
                 checkpoint: Optional[str] = None) -> torch.Tensor:
    """x (..., K), weight (2 F, K), bias (2 F,) -> (..., F), all of one type on
    one device; ``activation`` "silu", "gelu" (tanh form) or "relu"."""
    return layer("gated_linear", _GATES, x, weight, bias, None, activation,
                 checkpoint, True)
