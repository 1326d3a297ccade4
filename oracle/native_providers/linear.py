"""Dense products with their epilogue (CPU oracle).

``linear_act``: ``act(x W^T + b)``, gated: ``act`` of the first half of the features
times the second half. ``linear_residual``: ``residual + row_scale * dropout(x W^T +
b)``. Every step in the widest of the operands' dtype and fp32, rounded once at the end, with
PyTorch's autograd of the same composition as the backward; called with fp64
tensors they are the fp64 reference of the HIP kernels.

Pinned by: the textbook product on integer values and central differences in fp64,
see ``tests/test_dense_ops.py``. The reference forms both from separate torch calls
(``src/torchturbo/models/modules/moe/moe_layer.py:175-182``).
"""

from __future__ import annotations

import torch

from torchturbo_amd.dispatch import OpImpl, OpImplKind, register_op

from .dropout import dropout


def _wide(t):
    return t if t is None or t.dtype == torch.float64 else t.float()


def linear_act(x, weight, bias=None, *, activation_func=None, gated=False):
    a = _wide(x) @ _wide(weight).t()
    if bias is not None:
        a = a + _wide(bias)
    act = activation_func if activation_func is not None else (lambda v: v)
    if gated:
        gate, up = a.chunk(2, dim=-1)
        return (act(gate) * up).to(x.dtype)
    return act(a).to(x.dtype)


def linear_residual(x, weight, bias=None, residual=None, row_scale=None, *, dropout_p=0.0,
                    dropout_key=None):
    y = _wide(x) @ _wide(weight).t()
    if bias is not None:
        y = y + _wide(bias)
    if dropout_p:
        y = dropout(y, dropout_p, dropout_key)
    if row_scale is not None:
        y = y * _wide(row_scale).reshape(*y.shape[:-1], 1)
    if residual is not None:
        y = _wide(residual) + y
    return y.to(x.dtype)


@register_op(op_name="linear_act", impl_name="torch_linear_act",
             kind=OpImplKind.NATIVE, priority=0, devices=())
class TorchLinearAct(OpImpl):
    def __call__(self, x, weight, bias=None, *, activation_func=None, gated=False):
        return linear_act(x, weight, bias, activation_func=activation_func, gated=gated)


@register_op(op_name="linear_residual", impl_name="torch_linear_residual",
             kind=OpImplKind.NATIVE, priority=0, devices=())
class TorchLinearResidual(OpImpl):
    def __call__(self, x, weight, bias=None, residual=None, row_scale=None, *, dropout_p=0.0,
                 dropout_key=None):
        return linear_residual(x, weight, bias, residual, row_scale, dropout_p=dropout_p,
                               dropout_key=dropout_key)
