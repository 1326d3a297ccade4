"""HIP root-mean-square norm with the residual's addition.

* ``rms_norm(x, weight, eps, residual)``: ``y = h (mean(h^2) + eps)^(-1/2) weight``
  of ``h = x + residual`` over the last dimension; with a residual ``(y, h)``, else
  ``y``. Gradients flow to x, residual and weight from y and h.
* ``rms_norm_mx``: the same forward with y in 8 bits (``NormRows``), for the products
  with 4-bit weights, and y itself where a router reads it. Without gradients. The rows
  are those of the unrounded y, or with ``rounded`` of y as it is given back: what
  ``quantize_mxfp8(y)`` gives, so that it does not matter who quantises.

x and residual share one dtype (f32, bf16 or f16), the weight may have another of the
three. The statistics and the product are formed in fp32 from the unrounded sum; y and
h are rounded once. The backward reads the rounded h, so that one copy of it serves the
residual stream and the gradient.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ... import _lib as L
from ...dispatch import MxRows, NormRows, OpImpl, OpImplKind, register_op
from ...dispatch.mx import GROUP
from ...runtime import TurboDevice
from . import PRIORITY
from .available import hip_available
from .linear import FLOATS, _autograd_sees, _rows
from .mx import _device


def _forward(x, weight, eps, residual, with_y, with_rstd, with_mx, rounded=False):
    """(y, sum, rstd, codes, scales) of rows [T, H]; None for a part not wanted."""
    (t, h), dev = x.shape, x.device
    y = torch.empty_like(x) if with_y else None
    total = None if residual is None else torch.empty_like(x)
    rstd = torch.empty((t,), dtype=torch.float32, device=dev) if with_rstd else None
    codes = scales = None
    if with_mx:
        codes = torch.empty((t, h), dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty((t, h // GROUP), dtype=torch.uint8, device=dev)
    L.call("tt_rms_norm_fwd_rounded" if rounded else "tt_rms_norm_fwd", L.ptr(x), L.ptr(residual),
           L.ptr(weight), L.dtype_code(weight.dtype), L.dtype_code(x.dtype), t, h, eps, L.ptr(y),
           L.ptr(total), L.ptr(rstd), L.ptr(codes), L.ptr(scales), L.stream(dev))
    return y, total, rstd, codes, scales


class RmsNorm(torch.autograd.Function):
    """``(x [T, H], weight, residual or None, eps) -> (y, h or None)``."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, total, rstd, _, _ = _forward(x, weight, eps, residual, True, True, False)
        ctx.save_for_backward(x if total is None else total, weight, rstd)
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gsum):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if gy is None:
            return gsum if need_x else None, None, gsum if need_r else None, None
        gy = gy.to(h.dtype).contiguous()
        gsum = None if gsum is None else gsum.to(h.dtype).contiguous()
        dx = torch.empty_like(h) if need_x or need_r else None
        dw = torch.empty_like(weight) if need_w else None
        if h.numel() == 0:
            return dx, None if dw is None else dw.zero_(), dx if need_r else None, None
        size = L.load().tt_rms_norm_bwd_workspace(*h.shape) if need_w else 0
        ws = torch.empty((size,), dtype=torch.uint8, device=h.device) if size else None
        L.call("tt_rms_norm_bwd", L.ptr(h), L.ptr(weight), L.dtype_code(weight.dtype), L.ptr(rstd),
               L.ptr(gy), L.ptr(gsum), L.dtype_code(h.dtype), *h.shape, L.ptr(dx), L.ptr(dw),
               L.ptr(ws), size, L.stream(h.device))
        return dx if need_x else None, dw, dx if need_r else None, None


def _operands(op, x, weight, residual):
    if x.dim() == 0:
        raise ValueError(f"{op} needs at least one dimension")
    if x.dtype not in FLOATS or weight.dtype not in FLOATS:
        raise ValueError(f"{op} takes f32, bf16 or f16 tensors, got {x.dtype} and {weight.dtype}")
    if tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"{op}: the weight must have shape [{x.shape[-1]}], got "
                         f"{list(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{op}: the residual must be {x.dtype} {list(x.shape)}, got "
                         f"{residual.dtype} {list(residual.shape)}")
    if x.shape[-1] >= 1 << 31:
        raise ValueError(f"{op} takes fewer than 2^31 features")
    _device(x, weight, residual)
    h = x.shape[-1]
    return _rows(x, h), weight.contiguous(), None if residual is None else _rows(residual, h)


@register_op(op_name="rms_norm", impl_name="hip_rms_norm", kind=OpImplKind.CUSTOM,
             priority=PRIORITY, devices=(TurboDevice.CUDA,))
class HipRmsNorm(OpImpl):
    def available(self) -> bool:
        return hip_available()

    def __call__(self, x, weight, eps=1e-6, *, residual=None):
        x2, w, r = _operands("rms_norm", x, weight, residual)
        if _autograd_sees(x2, w, r):
            y, h = RmsNorm.apply(x2, w, r, float(eps))
        else:
            y, h = _forward(x2, w, float(eps), r, True, False, False)[:2]
        if x.dim() != 2:
            y, h = y.view(x.shape), None if h is None else h.view(x.shape)
        return y if residual is None else (y, h)


@register_op(op_name="rms_norm_mx", impl_name="hip_rms_norm_mx", kind=OpImplKind.CUSTOM,
             priority=PRIORITY, devices=(TurboDevice.CUDA,))
class HipRmsNormMx(OpImpl):
    def available(self) -> bool:
        return hip_available()

    def __call__(self, x, weight, eps=1e-6, *, residual=None, with_y=False, rounded=False):
        if x.dim() and x.shape[-1] % GROUP:
            raise ValueError(f"rms_norm_mx: the features must be whole groups of {GROUP}, got "
                             f"{x.shape[-1]}")
        x2, w, r = _operands("rms_norm_mx", x, weight, residual)
        if _autograd_sees(x2, w, r):
            raise RuntimeError("rms_norm_mx has no gradient: call it under torch.no_grad(), or "
                               "rms_norm in its place")
        y, h, _, codes, scales = _forward(x2, w, float(eps), r, with_y, False, True, rounded)
        rows = MxRows(codes, scales)
        if x.dim() == 2:
            return NormRows(rows, y, h)
        return NormRows(rows.view(*x.shape[:-1]), y.view(x.shape) if with_y else None,
                        None if h is None else h.view(x.shape))
