"""Experts and shared expert with 4-bit weights (MXFP4), frozen.

Weights are kept in ``[out, in]`` orientation as E2M1 codes, two to a byte, with one power of two
per 32 elements of a row: a quarter of bf16's bytes and a sixteenth more. They are quantised from
16-bit weights (:meth:`Mxfp4GroupedMLP.quantize`) or copied from a checkpoint in the same format.
The products read them as they are (``linear_mxfp4``, ``grouped_matmul_mxfp4``).

With ``rows_in_8_bits`` the rows that the products read are E4M3 in the same groups, when no
gradients are asked for: twice the matrix rate, half the bytes, and 2^-4 of rounding per
element. Gradients flow to the input and the probabilities through bf16 rows either way: adapters or
layers below train while the experts stay as they are.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..dispatch import MxRows, ops
from ..dispatch.mx import GROUP
from .moe_config import MoEConfig


def _grads(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Mxfp4Weights(torch.nn.Module):
    """Buffers ``q1, s1, q2, s2`` of the two weights ``[..., rows1, hidden]``, ``[..., hidden, ffn]``."""

    def __init__(self, lead, rows1, hidden, ffn) -> None:
        super().__init__()
        if hidden % GROUP or ffn % GROUP:
            raise ValueError(f"MXFP4 weights need hidden and ffn sizes divisible by {GROUP}.")
        for i, (rows, cols) in enumerate(((rows1, hidden), (hidden, ffn)), 1):
            self.register_buffer(f"q{i}", torch.zeros(*lead, rows, cols // 2, dtype=torch.uint8))
            self.register_buffer(f"s{i}", torch.zeros(*lead, rows, cols // GROUP, dtype=torch.uint8))

    @torch.no_grad()
    def load_quantized(self, q1, s1, q2, s2) -> None:
        """Copy codes and scales (uint8, or torch's ``float4_e2m1fn_x2`` and ``float8_e8m0fnu``)."""
        checked = []
        for name, t in (("q1", q1), ("s1", s1), ("q2", q2), ("s2", s2)):
            own = getattr(self, name)
            if t.dtype not in (torch.uint8, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu):
                raise ValueError(f"{name} must be uint8, float4_e2m1fn_x2 or float8_e8m0fnu, got "
                                 f"{t.dtype}")
            t = t if t.dtype == torch.uint8 else t.view(torch.uint8)
            if t.shape != own.shape:
                raise ValueError(f"{name} has shape {list(t.shape)}, expected {list(own.shape)}")
            checked.append((own, t))
        for own, t in checked:
            own.copy_(t)

    def _quantize(self, which: int, weight) -> None:
        codes, scales = ops.quantize_mxfp4(weight)
        getattr(self, f"q{which}").copy_(codes)
        getattr(self, f"s{which}").copy_(scales)


class Mxfp4GroupedMLP(_Mxfp4Weights):
    """SwiGLU experts with 4-bit weights: ``q1 [E, 2F, H / 2]`` (gate rows, then up rows), ``q2 [E, H,
    F / 2]``, in the place of ``GroupedMLP``."""

    def __init__(self, num_local_experts: int, use_te: bool, config: MoEConfig,
                 layer_number: int | None = None, rows_in_8_bits: bool = False) -> None:
        if not (config.gated_linear_unit and config.activation_func is F.silu):
            raise ValueError("Mxfp4GroupedMLP implements SwiGLU experts only.")
        if config.moe_apply_probs_on_input:
            raise ValueError("Mxfp4GroupedMLP applies probabilities to the activations only.")
        limits = getattr(config, "moe_swiglu_limit", None)
        if limits is not None and layer_number is not None and 0 <= layer_number < len(limits) \
                and limits[layer_number]:
            raise ValueError("Mxfp4GroupedMLP implements SwiGLU without a limit only.")
        super().__init__((num_local_experts,), 2 * config.moe_ffn_hidden_size, config.hidden_size,
                         config.moe_ffn_hidden_size)
        self.config = config
        self.num_local_experts = num_local_experts
        self.rows_in_8_bits = bool(rows_in_8_bits)

    @torch.no_grad()
    def quantize(self, weight1, weight2) -> None:
        """Quantise ``GroupedMLP``'s weights (``[E*H, 2F]`` and ``[E*F, H]``, any view of them)."""
        E, H = self.num_local_experts, self.config.hidden_size
        w1 = weight1.reshape(E, H, -1).transpose(1, 2)
        w2 = weight2.reshape(E, -1, H).transpose(1, 2)
        if w1.shape[1] != self.q1.shape[1] or w2.shape[2] != 2 * self.q2.shape[2]:
            raise ValueError(f"weights {list(weight1.shape)} and {list(weight2.shape)} do not fit "
                             f"{E} experts of {H} and {2 * self.q2.shape[2]} features")
        self._quantize(1, w1.contiguous())
        self._quantize(2, w2.contiguous())

    def forward(self, permuted_local_hidden_states, tokens_per_expert, permuted_probs):
        x, probs = permuted_local_hidden_states, permuted_probs.reshape(-1)
        if isinstance(x, MxRows) or not _grads(x, probs):
            return self.inference(x, tokens_per_expert, probs), None
        h = ops.grouped_matmul_mxfp4(x, self.q1, self.s1, tokens_per_expert, probs=probs, gated=True)
        return ops.grouped_matmul_mxfp4(h, self.q2, self.s2, tokens_per_expert), None

    def inference(self, x, tokens_per_expert, probs, row_map=None):
        """The experts' output without gradients; rows of ``x`` (bf16 or ``MxRows``) taken through
        ``row_map`` where given."""
        eight = self.rows_in_8_bits
        if eight and not isinstance(x, MxRows):
            x = ops.quantize_mxfp8(x)
        h = ops.grouped_matmul_mxfp4(x, self.q1, self.s1, tokens_per_expert, probs=probs, gated=True,
                                     row_map=row_map, mx_out=eight)
        return ops.grouped_matmul_mxfp4(h, self.q2, self.s2, tokens_per_expert)


class Mxfp4SharedExpertMLP(_Mxfp4Weights):
    """The expert that every token takes, with 4-bit weights: ``act(x W1^T) W2^T`` as
    ``SharedExpertMLP`` without bias and dropout."""

    def __init__(self, config: MoEConfig, rows_in_8_bits: bool = False) -> None:
        ffn = config.moe_shared_expert_intermediate_size
        if not ffn or ffn < 0:
            raise ValueError("Mxfp4SharedExpertMLP needs config.moe_shared_expert_intermediate_size.")
        if config.activation_func not in (F.silu, F.gelu):
            raise ValueError("Activation function must be silu or gelu when using "
                             "Mxfp4SharedExpertMLP.")
        super().__init__((), ffn * (2 if config.gated_linear_unit else 1), config.hidden_size, ffn)
        self.config = config
        self.rows_in_8_bits = bool(rows_in_8_bits)

    @torch.no_grad()
    def quantize(self, weight1, weight2) -> None:
        """Quantise ``SharedExpertMLP``'s weights (``[2F or F, H]`` and ``[H, F]``)."""
        shapes = [[*q.shape[:-1], 2 * q.shape[-1]] for q in (self.q1, self.q2)]
        if [list(weight1.shape), list(weight2.shape)] != shapes:
            raise ValueError(f"weights {list(weight1.shape)} and {list(weight2.shape)} do not fit "
                             f"{shapes[0]} and {shapes[1]}")
        self._quantize(1, weight1)
        self._quantize(2, weight2)

    def forward(self, hidden_states):
        cfg = self.config
        eight = self.rows_in_8_bits and not _grads(hidden_states)
        x = ops.quantize_mxfp8(hidden_states) if eight else hidden_states
        h = ops.linear_mxfp4(x, self.q1, self.s1, activation_func=cfg.activation_func,
                             gated=cfg.gated_linear_unit, mx_out=eight)
        # Products of rows in 8 bits are bf16 whatever the input was.
        return ops.linear_mxfp4(h, self.q2, self.s2).to(hidden_states.dtype)


__all__ = ["Mxfp4GroupedMLP", "Mxfp4SharedExpertMLP"]
