"""HIP dropout from a counter-based generator, with a mask that is never stored.

``dropout(x, p, key)`` keeps or clears an element by 16 bits of Philox4x32-10
(Salmon et al., SC 2011) of ``key`` (a seed and an offset, int64 ``[2]`` on the
device) and the element's position: the last dimension is the column, all others
together the row. Kept elements are multiplied by the inverse of the share that
is kept, cleared ones are 0 whatever they held. The backward makes the mask again
from the key, so nothing but the key is kept, and a call with the same key, shape
and ``p`` gives the same mask (activation checkpointing, a replayed graph).

``p`` is taken in steps of 2^-16 (at least one step unless it is 0, and less than
all unless it is 1); ``p = 0`` returns ``x``.
"""

from __future__ import annotations

import torch

from ... import _lib as L
from ...dispatch import OpImpl, OpImplKind, register_op
from ...runtime import TurboDevice
from . import PRIORITY
from ._functions import require_cuda
from .available import hip_available

MAX_ROWS = 1 << 32


def drop_threshold(p) -> int:
    """How many of 65536 equal shares ``p`` drops (``ValueError`` outside [0, 1])."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    if p in (0.0, 1.0):
        return int(p) * 65536
    return min(max(round(p * 65536), 1), 65535)


def check_key(key, device: torch.device) -> torch.Tensor:
    """``key`` as a contiguous int64 ``[2]`` on ``device``, or ``ValueError``."""
    if not isinstance(key, torch.Tensor) or key.dtype != torch.int64 or key.shape != (2,):
        raise ValueError("dropout needs a key: an int64 tensor of shape [2] (seed, offset)")
    if key.device != device:
        raise ValueError(f"the dropout key is on {key.device}, expected {device}")
    return key.contiguous()


def _drop(x, threshold, key):
    y = torch.empty_like(x)
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    L.call("tt_dropout", L.ptr(x), L.dtype_code(x.dtype), rows, cols, threshold, L.ptr(key),
           L.ptr(y), L.stream(x.device))
    return y


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, threshold, key):
        ctx.save_for_backward(key)
        ctx.threshold = threshold
        return _drop(x.contiguous(), threshold, key)

    @staticmethod
    def backward(ctx, dy):
        (key,) = ctx.saved_tensors
        if torch.is_grad_enabled():  # a product with a fixed factor: differentiable again
            return Dropout.apply(dy, ctx.threshold, key), None, None
        return _drop(dy.contiguous(), ctx.threshold, key), None, None


@register_op(op_name="dropout", impl_name="hip_dropout", kind=OpImplKind.CUSTOM,
             priority=PRIORITY, devices=(TurboDevice.CUDA,))
class HipDropout(OpImpl):
    def available(self) -> bool:
        return hip_available()

    def __call__(self, x, p, key):
        threshold = drop_threshold(p)
        if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"dropout takes f32, bf16 or f16 tensors, got {x.dtype}")
        if x.dim() == 0:
            raise ValueError("dropout needs at least one dimension")
        if x.shape[-1] and x.numel() // x.shape[-1] >= MAX_ROWS:
            raise ValueError(f"dropout takes fewer than {MAX_ROWS} rows")
        if threshold == 0:
            return x
        key = check_key(key, x.device)
        require_cuda(x)
        return Dropout.apply(x, threshold, key)
