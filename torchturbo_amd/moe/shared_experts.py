"""The expert that every token takes: a dense MLP added to the routed experts' output.

The reference leaves it to the Hugging Face block (a ``down(act(gate(x)) * up(x))``
of three linears) and adds it in a pass of its own, with a sigmoid gate per token
where the model has one (``src/torchturbo/models/modules/moe/moe_layer.py:175-182``).
Here it is two products with everything else in their epilogues: ``linear_act``
(gate and up as one weight, activation and their product), and ``linear_residual``
(the down projection, dropout, the token's gate and the routed experts' output).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.nn.parameter import Parameter

from ..dispatch import ops
from .dropout import CounterDropout
from .module import attached
from .moe_config import MoEConfig


class SharedExpertMLP(torch.nn.Module):
    """``residual + row_scale * dropout(act(x W1^T + b1) W2^T + b2)``.

    ``weight1`` is ``[2 F, H]`` (the gate's rows, then the up projection's) or
    ``[F, H]`` without ``config.gated_linear_unit``, ``weight2`` ``[H, F]``; F is
    ``config.moe_shared_expert_intermediate_size``. State dicts with
    ``gate_proj`` / ``up_proj`` / ``down_proj`` entries load as they are.
    """

    def __init__(self, config: MoEConfig, bias: bool = False, dropout: float = 0.0) -> None:
        super().__init__()
        ffn = config.moe_shared_expert_intermediate_size
        if not ffn or ffn < 0:
            raise ValueError("SharedExpertMLP needs config.moe_shared_expert_intermediate_size.")
        if config.activation_func not in (F.silu, F.gelu):
            raise ValueError("Activation function must be silu or gelu when using SharedExpertMLP.")
        self.config = config
        dtype, rows = config.params_dtype, ffn * (2 if config.gated_linear_unit else 1)
        self.weight1 = Parameter(torch.empty(rows, config.hidden_size, dtype=dtype))
        self.weight2 = Parameter(torch.empty(config.hidden_size, ffn, dtype=dtype))
        if bias:
            self.bias1 = Parameter(torch.zeros(rows, dtype=dtype))
            self.bias2 = Parameter(torch.zeros(config.hidden_size, dtype=dtype))
        else:
            self.register_parameter("bias1", None)
            self.register_parameter("bias2", None)
        self.dropout = CounterDropout(dropout)
        if config.perform_initialization:
            config.init_method(self.weight1)
            config.init_method(self.weight2)

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        for kind, first, second in (("weight", "weight1", "weight2"), ("bias", "bias1", "bias2")):
            parts = ("gate_proj", "up_proj") if self.config.gated_linear_unit else ("up_proj",)
            names = [f"{prefix}{p}.{kind}" for p in parts]
            if all(n in state_dict for n in names):
                state_dict[prefix + first] = torch.cat([state_dict.pop(n) for n in names])
            if f"{prefix}down_proj.{kind}" in state_dict:
                state_dict[prefix + second] = state_dict.pop(f"{prefix}down_proj.{kind}")
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def forward(self, hidden_states, residual=None, row_scale=None):
        h = ops.linear_act(hidden_states, self.weight1, self.bias1,
                           activation_func=self.config.activation_func,
                           gated=self.config.gated_linear_unit)
        drop = self.dropout
        if not self._dropout_in_epilogue(drop):
            y = drop(ops.linear_residual(h, self.weight2, self.bias2))
            if row_scale is not None:
                y = y * row_scale.reshape(*y.shape[:-1], 1)
            return (y if residual is None else residual + y).to(hidden_states.dtype)
        p, key = 0.0, None
        if drop.active:
            p, key = drop.p, drop.draw_key(hidden_states.device)
        return ops.linear_residual(h, self.weight2, self.bias2, residual, row_scale, dropout_p=p,
                                   dropout_key=key)

    @staticmethod
    def _dropout_in_epilogue(drop) -> bool:
        """Whether ``linear_residual`` may make the mask in place of a call of ``drop``: nothing
        is attached to it, and the HIP product's mask is that of the ``dropout`` op chosen."""
        if type(drop) is not CounterDropout or attached(drop, "draw_key"):
            return False
        return (not drop.active or ops.selected_impl_name("dropout") == "hip_dropout"
                or ops.selected_impl_name("linear_residual") != "hip_linear_residual")


__all__ = ["SharedExpertMLP"]
