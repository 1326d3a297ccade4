"""Root-mean-square norm as a module: of a layer's input, or a residual stream with the input added."""

from __future__ import annotations

import torch
from torch.nn.parameter import Parameter

from ..dispatch import ops
from .moe_config import MoEConfig


class RMSNorm(torch.nn.Module):
    """``forward(x)`` is the normalised x, ``forward(x, residual)`` is ``(y, x + residual)`` with
    y the normalised sum. ``weight`` is ``[hidden_size]``, ones at first."""

    def __init__(self, config: MoEConfig, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = float(eps)
        self.weight = Parameter(torch.ones(config.hidden_size, dtype=config.params_dtype))

    def forward(self, hidden_states, residual=None):
        return ops.rms_norm(hidden_states, self.weight, self.eps, residual=residual)


__all__ = ["RMSNorm"]
