"""Microscaling formats and the products over them in 64 bits, from the formats' definition.

Nothing is shared with the kernels: values are rounded by dividing by their own step, codes
are read field by field.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from torchturbo_amd.dispatch import MxRows, OpImpl, OpImplKind, register_op

GROUP = 32


def power(exponent: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones_like(exponent, dtype=torch.float64), exponent.to(torch.int32))


def scale_values(scales: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) in 64 bits, NaN for 255."""
    v = power(scales.to(torch.int32) - 127)
    return torch.where(scales == 255, torch.full_like(v, float("nan")), v)


def _shared(x: torch.Tensor, top: int):
    """(groups in 64 bits, E8M0 bytes [..., K / 32], groups that are not finite)."""
    v = x.double().unflatten(-1, (-1, GROUP))
    finite = torch.isfinite(v).all(-1)
    amax = torch.where(finite, v.abs().amax(-1), torch.ones((), dtype=torch.float64))
    exponent = torch.frexp(amax).exponent - 1
    byte = torch.where(amax > 0, (exponent - top + 127).clamp(0, 254), 0)
    return v, torch.where(finite, byte, 255), finite


def _nearest(u: torch.Tensor, fraction: int, least: int, most: float) -> torch.Tensor:
    """``u`` with ``fraction`` bits behind its leading one (exponents from ``least``), half to even."""
    exponent = torch.where(u == 0, least, torch.frexp(u).exponent - 1).clamp(min=least)
    step = power(exponent - fraction)
    return (torch.round(u / step) * step).clamp(-most, most)


MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def e2m1_values(codes: torch.Tensor) -> torch.Tensor:
    """Values [..., K] of packed codes [..., K / 2] in 64 bits."""
    both = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    table = torch.tensor([*MAGNITUDES, *(-m for m in MAGNITUDES)], dtype=torch.float64)
    return table[both]


def quantize_mxfp4(weight: torch.Tensor):
    v, byte, finite = _shared(weight, 2)
    q = _nearest(v / power(byte - 127).unsqueeze(-1), 1, 0, 6.0)
    code = torch.zeros_like(q, dtype=torch.int64)
    for i, m in enumerate(MAGNITUDES):
        code = torch.where(q.abs() == m, i, code)
    code = code + 8 * (q < 0)
    code = torch.where(finite.unsqueeze(-1), code, 0).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), byte.to(torch.uint8)


def dequantize_mxfp4(codes, scales, dtype=torch.bfloat16):
    v = e2m1_values(codes).unflatten(-1, (-1, GROUP)) * scale_values(scales).unsqueeze(-1)
    return v.flatten(-2).to(dtype)


def quantize_mxfp8(x: torch.Tensor) -> MxRows:
    v, byte, finite = _shared(x, 8)
    q = _nearest(v / power(byte - 127).unsqueeze(-1), 3, -6, 448.0)
    q = torch.where(finite.unsqueeze(-1), q, torch.full_like(q, float("nan")))
    return MxRows(q.flatten(-2).float().to(torch.float8_e4m3fn), byte.to(torch.uint8))


def dequantize_mxfp8(rows: MxRows, dtype=torch.bfloat16):
    v = rows.codes.float().double().unflatten(-1, (-1, GROUP))
    return (v * scale_values(rows.scales).unsqueeze(-1)).flatten(-2).to(dtype)


def values_of(x) -> torch.Tensor:
    return dequantize_mxfp8(x, torch.float64) if isinstance(x, MxRows) else x.double()


def epilogue(a, activation_func, gated, probs=None):
    act = activation_func or (lambda v: v)
    if gated:
        gate, up = a.chunk(2, -1)
        a = act(gate) * up
    else:
        a = act(a)
    return a if probs is None else a * probs.reshape(-1, 1).double()


def linear(x, codes, scales, activation_func=None, gated=False) -> torch.Tensor:
    """``linear_mxfp4`` in 64 bits, unrounded."""
    w = dequantize_mxfp4(codes, scales, torch.float64)
    return epilogue(values_of(x) @ w.t(), activation_func, gated)


def grouped(x, codes, scales, counts, probs=None, gated=False, row_map=None) -> torch.Tensor:
    """``grouped_matmul_mxfp4`` in 64 bits, unrounded."""
    v = values_of(x)
    if row_map is not None:
        v = v[row_map.long()]
    parts = v.split([int(c) for c in counts])
    y = torch.cat([p @ dequantize_mxfp4(codes[e], scales[e], torch.float64).t()
                   for e, p in enumerate(parts)])
    return epilogue(y, F.silu if gated else None, gated, probs)


def _rounded(y, like, mx_out):
    if mx_out:
        return quantize_mxfp8(y)
    return y.to(torch.bfloat16 if isinstance(like, MxRows) else like.dtype)


@register_op(op_name="linear_mxfp4", impl_name="torch_linear_mxfp4", kind=OpImplKind.NATIVE,
             priority=0, devices=())
class TorchLinearMxfp4(OpImpl):
    def __call__(self, x, codes, scales, *, activation_func=None, gated=False, mx_out=False):
        return _rounded(linear(x, codes, scales, activation_func, gated), x, mx_out)


@register_op(op_name="grouped_matmul_mxfp4", impl_name="torch_grouped_matmul_mxfp4",
             kind=OpImplKind.NATIVE, priority=0, devices=())
class TorchGroupedMatmulMxfp4(OpImpl):
    def __call__(self, x, codes, scales, tokens_per_expert, *, probs=None, gated=False,
                 row_map=None, mx_out=False):
        return _rounded(grouped(x, codes, scales, tokens_per_expert, probs, gated, row_map), x,
                        mx_out)


@register_op(op_name="quantize_mxfp4", impl_name="torch_quantize_mxfp4", kind=OpImplKind.NATIVE,
             priority=0, devices=())
class TorchQuantizeMxfp4(OpImpl):
    def __call__(self, weight):
        return quantize_mxfp4(weight)


@register_op(op_name="dequantize_mxfp4", impl_name="torch_dequantize_mxfp4",
             kind=OpImplKind.NATIVE, priority=0, devices=())
class TorchDequantizeMxfp4(OpImpl):
    def __call__(self, codes, scales, dtype=torch.bfloat16):
        return dequantize_mxfp4(codes, scales, dtype)


@register_op(op_name="quantize_mxfp8", impl_name="torch_quantize_mxfp8", kind=OpImplKind.NATIVE,
             priority=0, devices=())
class TorchQuantizeMxfp8(OpImpl):
    def __call__(self, x):
        return quantize_mxfp8(x)


@register_op(op_name="dequantize_mxfp8", impl_name="torch_dequantize_mxfp8",
             kind=OpImplKind.NATIVE, priority=0, devices=())
class TorchDequantizeMxfp8(OpImpl):
    def __call__(self, rows, dtype=torch.bfloat16):
        return dequantize_mxfp8(rows, dtype)
