"""Root-mean-square norm with the residual's addition, in 64 bits."""

from __future__ import annotations

import torch

from torchturbo_amd.dispatch import NormRows, OpImpl, OpImplKind, register_op

from .mx import quantize_mxfp8


def norm(x, weight, eps, residual=None):
    """(y, h) in 64 bits, unrounded and differentiable."""
    h = x.double() if residual is None else x.double() + residual.double()
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double(), h


@register_op(op_name="rms_norm", impl_name="torch_rms_norm", kind=OpImplKind.NATIVE, priority=0,
             devices=())
class TorchRmsNorm(OpImpl):
    def __call__(self, x, weight, eps=1e-6, *, residual=None):
        y, h = norm(x, weight, eps, residual)
        return y.to(x.dtype) if residual is None else (y.to(x.dtype), h.to(x.dtype))


@register_op(op_name="rms_norm_mx", impl_name="torch_rms_norm_mx", kind=OpImplKind.NATIVE,
             priority=0, devices=())
class TorchRmsNormMx(OpImpl):
    def __call__(self, x, weight, eps=1e-6, *, residual=None, with_y=False, rounded=False):
        y, h = norm(x, weight, eps, residual)
        return NormRows(quantize_mxfp8(y.to(x.dtype) if rounded else y),
                        y.to(x.dtype) if with_y else None,
                        None if residual is None else h.to(x.dtype))
