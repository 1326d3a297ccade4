"""Dropout whose mask is a function of a key and the position of an element.

``CounterDropout`` stands in for ``torch.nn.Dropout``: it draws a key (a seed and
an offset) from PyTorch's generator of the device for each forward and calls the
``dropout`` op, which keeps no mask. So ``torch.manual_seed`` governs it, activation
checkpointing (which restores the generator) recomputes the same mask, and a
captured graph draws a new key in each replay.
"""

from __future__ import annotations

import torch

from ..dispatch import ops


class CounterDropout(torch.nn.Module):
    def __init__(self, p: float = 0.5) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability must be in [0, 1], got {p}")
        self.p = float(p)

    @property
    def active(self) -> bool:
        return self.training and self.p > 0.0

    @staticmethod
    def draw_key(device) -> torch.Tensor:
        """A key (int64 ``[2]``) from the device's default generator, without a host sync."""
        return torch.empty((2,), dtype=torch.int64, device=device).random_()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.active:
            return x
        return ops.dropout(x, self.p, self.draw_key(x.device))

    def extra_repr(self) -> str:
        return f"p={self.p}"


__all__ = ["CounterDropout"]
