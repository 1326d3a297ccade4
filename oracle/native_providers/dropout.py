"""Counter-based dropout (CPU oracle).

Element (row, column) of a tensor (all dimensions but the last together the row)
takes 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
numbers: as easy as 1, 2, 3", SC 2011): key = the key's seed, counter = (column / 8,
row, the key's offset), bits 16 (column % 2) of word (column % 8) / 2. It is
dropped when they are below ``round(p 2^16)`` (at least 1, at most 65535, for p
strictly between 0 and 1), and otherwise multiplied by the inverse of the kept
share.

Pinned by: the published known-answer vectors of Philox4x32-10, see
``tests/test_dense_ops.py``. No reference counterpart.
"""

from __future__ import annotations

import numpy as np
import torch

from torchturbo_amd.dispatch import OpImpl, OpImplKind, register_op

_LOW = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key):
    """Ten rounds on arrays of 32-bit words (as uint64): counter c0 .. c3, key k0, k1."""
    c0, c1, c2, c3 = (np.asarray(c, dtype=np.uint64) for c in counter)
    k0, k1 = (int(k) for k in key)
    shift = np.uint64(32)
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c0, np.uint64(0xCD9E8D57) * c2
        c0, c1, c2, c3 = ((p1 >> shift) ^ c1 ^ np.uint64(k0), p1 & _LOW,
                          (p0 >> shift) ^ c3 ^ np.uint64(k1), p0 & _LOW)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c0, c1, c2, c3


def threshold_of(p: float) -> int:
    return int(p) * 65536 if p in (0.0, 1.0) else min(max(round(p * 65536), 1), 65535)


def factors(rows: int, cols: int, p: float, key, first_row: int = 0) -> torch.Tensor:
    """fp64 [rows, cols]: 0, or the inverse of the kept share (rows first_row ...)."""
    seed, offset = (int(v) % (1 << 64) for v in key.tolist())
    groups = (cols + 7) // 8
    c0 = np.broadcast_to(np.arange(groups, dtype=np.uint64), (rows, groups))
    c1 = np.broadcast_to(np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None],
                         (rows, groups))
    words = philox4x32((c0, c1, np.full_like(c0, offset & 0xFFFFFFFF), np.full_like(c0, offset >> 32)),
                       (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.empty((rows, groups, 8), dtype=np.int64)
    for j in range(8):
        bits[:, :, j] = (words[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF)
    t = threshold_of(p)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    kept = bits.reshape(rows, groups * 8)[:, :cols] >= t
    return torch.from_numpy(np.ascontiguousarray(kept)).double() * scale


def dropout(x: torch.Tensor, p: float, key: torch.Tensor) -> torch.Tensor:
    if threshold_of(p) == 0:
        return x
    cols = x.shape[-1]
    f = factors(x.numel() // max(cols, 1), cols, p, key).view(x.shape)
    # A dropped element is 0 whatever it held; a kept one is multiplied in fp32 (fp64).
    wide = x if x.dtype == torch.float64 else x.float()
    return torch.where(f > 0, wide * f.to(wide.dtype), torch.zeros_like(wide)).to(x.dtype)


@register_op(op_name="dropout", impl_name="torch_counter_dropout",
             kind=OpImplKind.NATIVE, priority=0, devices=())
class TorchDropout(OpImpl):
    def __call__(self, x, p, key):
        return dropout(x, p, key)
