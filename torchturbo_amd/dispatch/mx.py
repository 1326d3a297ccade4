"""Rows in 8 bits, as the norm and the activations give them and the 4-bit products take them.

The microscaling format (OCP MX): 32 consecutive elements of a row share a power of
two, kept as a byte ``c`` of value ``2^(c - 127)`` (255: the group is NaN); elements
are E4M3.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

GROUP = 32


@dataclass(eq=False, slots=True)
class MxRows:
    # [..., K] float8_e4m3fn.
    codes: torch.Tensor
    # [..., K / 32] uint8: the exponent of each group, offset by 127.
    scales: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def view(self, *lead: int) -> "MxRows":
        """The same rows with other leading dimensions."""
        return MxRows(self.codes.view(*lead, self.codes.shape[-1]),
                      self.scales.view(*lead, self.scales.shape[-1]))


@dataclass(eq=False, slots=True)
class NormRows:
    """What ``rms_norm_mx`` gives."""

    # The normalised rows in 8 bits.
    rows: MxRows
    # [..., H] the same in the input's dtype, where asked for.
    y: torch.Tensor | None
    # [..., H] input + residual, where there is one.
    sum: torch.Tensor | None


__all__ = ["GROUP", "MxRows", "NormRows"]
