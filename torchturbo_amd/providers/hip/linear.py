"""HIP dense products with what follows them in their epilogue.

* ``linear_act(x, weight, bias, activation_func, gated)``:
  ``act(x W^T + b)``, or with ``gated`` and a weight ``[2 N, K]`` (the gate's rows
  first) ``act(a[..., :N]) * a[..., N:]`` of ``a = x W^T + b``.
* ``linear_residual(x, weight, bias, residual, row_scale, dropout_p, dropout_key)``:
  ``residual + row_scale * dropout(x W^T + b)``, one ``row_scale`` per row; the
  dropout is that of the ``dropout`` op on the product.

``x`` is ``[..., K]``, ``weight`` ``[out, in]`` as in ``torch.nn.Linear``; x,
weight and residual share one dtype (f32, bf16 or f16), bias and row_scale may
have another of the three. Sums, bias, activation and scale are formed in fp32 and
rounded once. The activation's backward keeps its input ``a`` in fp32: rounded to
16 bits it would add an error of its own to every gradient, for 2 % of a training
pass. They are the two halves of a shared expert
(``models/modules/moe/moe_layer.py:175-182``).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ... import _lib as L
from ...dispatch import OpImpl, OpImplKind, register_op
from ...runtime import TurboDevice
from . import PRIORITY
from ._functions import require_cuda
from .available import hip_available
from .dropout import check_key, drop_threshold

FLOATS = (torch.float32, torch.bfloat16, torch.float16)
ACTIVATIONS = {None: 0, F.silu: 1, F.gelu: 2}
ACT, GATED, RESIDUAL = range(3)


def _scratch(size, device):
    return torch.empty((size,), dtype=torch.uint8, device=device) if size else None


def _code(t):
    return 0 if t is None else L.dtype_code(t.dtype)


def act_fwd(x, w, bias, act, gated, pre):
    """y [M, N] of x [M, K]; ``pre``: fp32 [M, N or 2 N] that takes the activation's input."""
    m, k = x.shape
    n = w.shape[0] // 2 if gated else w.shape[0]
    dev, code = x.device, L.dtype_code(x.dtype)
    y = torch.empty((m, n), dtype=x.dtype, device=dev)
    size = L.load().tt_linear_workspace(GATED if gated else ACT, code, m, k, n)
    ws = _scratch(size, dev)
    L.call("tt_linear_act_fwd", L.ptr(x), L.ptr(w), L.ptr(bias), _code(bias), code, m, k, n, act,
           gated, L.ptr(pre), L.ptr(y), L.ptr(ws), size, L.stream(dev))
    return y


def residual_fwd(x, w, bias, residual, scale, threshold, key):
    m, k = x.shape
    n = w.shape[0]
    dev, code = x.device, L.dtype_code(x.dtype)
    y = torch.empty((m, n), dtype=x.dtype, device=dev)
    size = L.load().tt_linear_workspace(RESIDUAL, code, m, k, n)
    ws = _scratch(size, dev)
    L.call("tt_linear_residual_fwd", L.ptr(x), L.ptr(w), L.ptr(bias), _code(bias), L.ptr(residual),
           L.ptr(scale), _code(scale), code, m, k, n, threshold, L.ptr(key), L.ptr(y), L.ptr(ws),
           size, L.stream(dev))
    return y


class LinearAct(torch.autograd.Function):
    """``(x [M, K], w, bias, act, gated) -> y [M, N]``."""

    @staticmethod
    def forward(ctx, x, w, bias, act, gated):
        pre = None
        if act or gated:
            pre = torch.empty((x.shape[0], w.shape[0]), dtype=torch.float32, device=x.device)
        y = act_fwd(x, w, bias, act, gated, pre)
        ctx.save_for_backward(x, w, bias, pre)
        ctx.cfg = (act, gated)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, bias, pre = ctx.saved_tensors
        act, gated = ctx.cfg
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = dy.to(x.dtype).contiguous()
        (m, n), k, dev, code = dy.shape, x.shape[1], x.device, L.dtype_code(x.dtype)
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty_like(w) if need_w else None
        dbias = torch.empty_like(bias) if need_b else None
        size = L.load().tt_linear_act_bwd_workspace(code, m, k, n, act, gated)
        ws = _scratch(size, dev)
        L.call("tt_linear_act_bwd", L.ptr(dy), L.ptr(x), L.ptr(w), L.ptr(pre), code, m, k, n, act,
               gated, L.ptr(dx), L.ptr(dw), L.ptr(dbias), _code(dbias), L.ptr(ws), size,
               L.stream(dev))
        return dx, dw, dbias, None, None


class LinearResidual(torch.autograd.Function):
    """``(x [M, K], w, bias, residual [M, N], scale [M], threshold, key) -> y [M, N]``."""

    @staticmethod
    def forward(ctx, x, w, bias, residual, scale, threshold, key):
        y = residual_fwd(x, w, bias, residual, scale, threshold, key)
        ctx.save_for_backward(x, w, bias, scale, key)
        ctx.threshold = threshold
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, bias, scale, key = ctx.saved_tensors
        need_x, need_w, need_b, need_r, need_s = ctx.needs_input_grad[:5]
        d_residual = dy if need_r else None
        if not (need_x or need_w or need_b or need_s):
            return None, None, None, d_residual, None, None, None
        dy = dy.to(x.dtype).contiguous()
        t = ctx.threshold
        (m, n), k, dev, code = dy.shape, x.shape[1], x.device, L.dtype_code(x.dtype)
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty_like(w) if need_w else None
        dbias = torch.empty_like(bias) if need_b else None
        ds = torch.empty_like(scale) if need_s else None
        size = L.load().tt_linear_residual_bwd_workspace(code, m, k, n, scale is not None, t != 0)
        ws = _scratch(size, dev)
        L.call("tt_linear_residual_bwd", L.ptr(dy), L.ptr(x), L.ptr(w), L.ptr(bias), _code(bias),
               L.ptr(scale), _code(scale), code, m, k, n, t, L.ptr(key), L.ptr(dx), L.ptr(dw),
               L.ptr(dbias), L.ptr(ds), L.ptr(ws), size, L.stream(dev))
        return dx, dw, dbias, d_residual, ds, None, None


def _operands(op, x, weight, bias):
    """Checks shared by both products."""
    dtype, w_shape, features = x.dtype, weight.shape, x.shape[-1] if x.dim() else -1
    if features < 0 or len(w_shape) != 2:
        raise ValueError(f"{op} expects x [..., in] and weight [out, in]")
    if dtype not in FLOATS or weight.dtype is not dtype:
        raise ValueError(f"{op}: x and weight must both be f32, bf16 or f16, got {dtype} and "
                         f"{weight.dtype}")
    if w_shape[1] != features:
        raise ValueError(f"{op}: x has {features} features, weight expects {w_shape[1]}")
    if bias is not None and (bias.dtype not in FLOATS or bias.shape != w_shape[:1]):
        raise ValueError(f"{op}: the bias must be a float tensor of shape [{w_shape[0]}], got "
                         f"{bias.dtype} {list(bias.shape)}")
    if x.numel() >= (1 << 31) * max(features, 1):
        raise ValueError(f"{op} takes fewer than 2^31 rows")


def _autograd_sees(*tensors) -> bool:
    """Whether the call has to go through its autograd function: for gradients, and for the
    tangents and function transforms that the function refuses and a native call on addresses
    would lose (a dual tensor does not require gradients)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return (torch.autograd.forward_ad._current_level >= 0
            or torch._C._are_functorch_transforms_active())


def _rows(t, width):
    """[..., width] as contiguous rows (their number from the other dimensions alone)."""
    if t.dim() == 2:
        return t.contiguous()
    count = 1
    for d in t.shape[:-1]:
        count *= d
    return t.reshape(count, width).contiguous()


@register_op(op_name="linear_act", impl_name="hip_linear_act", kind=OpImplKind.CUSTOM,
             priority=PRIORITY, devices=(TurboDevice.CUDA,))
class HipLinearAct(OpImpl):
    def available(self) -> bool:
        return hip_available()

    def __call__(self, x, weight, bias=None, *, activation_func=None, gated=False):
        if activation_func not in ACTIVATIONS:
            raise ValueError("linear_act only supports no activation, F.silu and F.gelu")
        _operands("linear_act", x, weight, bias)
        if gated and weight.shape[0] % 2:
            raise ValueError("linear_act: a gated weight needs an even number of rows")
        require_cuda(x, weight, bias)
        act, gated = ACTIVATIONS[activation_func], bool(gated)
        n = weight.shape[0] // 2 if gated else weight.shape[0]
        x2, w = _rows(x, x.shape[-1]), weight.contiguous()
        b = None if bias is None else bias.contiguous()
        if _autograd_sees(x2, w, b):
            y = LinearAct.apply(x2, w, b, act, gated)
        else:
            y = act_fwd(x2, w, b, act, gated, None)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], n)


@register_op(op_name="linear_residual", impl_name="hip_linear_residual", kind=OpImplKind.CUSTOM,
             priority=PRIORITY, devices=(TurboDevice.CUDA,))
class HipLinearResidual(OpImpl):
    def available(self) -> bool:
        return hip_available()

    def __call__(self, x, weight, bias=None, residual=None, row_scale=None, *, dropout_p=0.0,
                 dropout_key=None):
        threshold = drop_threshold(dropout_p)
        _operands("linear_residual", x, weight, bias)
        n = weight.shape[0]
        shape = (*x.shape[:-1], n)
        if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
            raise ValueError(f"linear_residual: the residual must be {x.dtype} {list(shape)}, got "
                             f"{residual.dtype} {list(residual.shape)}")
        if row_scale is not None:
            if row_scale.dtype not in FLOATS or tuple(row_scale.shape) not in (
                    tuple(x.shape[:-1]), (*x.shape[:-1], 1)):
                raise ValueError(f"linear_residual: row_scale must be a float tensor of shape "
                                 f"{list(x.shape[:-1])} (or with a last dimension of 1), got "
                                 f"{row_scale.dtype} {list(row_scale.shape)}")
        key = check_key(dropout_key, x.device) if threshold else None
        require_cuda(x, weight, bias, residual, row_scale)
        x2, w = _rows(x, x.shape[-1]), weight.contiguous()
        b = None if bias is None else bias.contiguous()
        r = None if residual is None else _rows(residual, n)
        s = None if row_scale is None else row_scale.reshape(-1).contiguous()
        if _autograd_sees(x2, w, b, r, s):
            y = LinearResidual.apply(x2, w, b, r, s, threshold, key)
        else:
            y = residual_fwd(x2, w, b, r, s, threshold, key)
        return y if x.dim() == 2 else y.view(shape)
