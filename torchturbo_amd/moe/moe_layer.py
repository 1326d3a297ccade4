"""MoE layer: router -> dispatcher -> experts -> combine.

Mirrors ``MoELayer`` (``src/torchturbo/models/modules/moe/moe_layer.py:94-183``):
same constructor, ``forward(hidden_states, input_ids=None) -> (output,
logits)`` and shared-expert handling. ``forward_with_logits`` runs the same
path from router logits supplied by the caller (the benchmark feeds synthetic
logits of a given distribution, as the reference's configurations state).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch
import torch.distributed as dist
import torch.nn.functional as F

from ..dispatch import op_resolves, ops
from .experts import Fp8GroupedMLP, GroupedMLP
from .module import ModuleSpec, attached, build_module
from .moe_config import MoEConfig
from .mxfp4 import Mxfp4GroupedMLP
from .norm import RMSNorm
from .router import TopKRouter
from .shared_experts import SharedExpertMLP
from .token_dispatcher import MoEAlltoAllTokenDispatcher


@dataclass
class MoESubmodules:
    experts: Union[ModuleSpec, type] = None
    shared_experts: Union[ModuleSpec, type] = None
    # Norm of the layer's input (RMSNorm); the reference leaves it to the decoder layer.
    norm: Union[ModuleSpec, type] = None


@dataclass
class MoERuntimeInputs:
    padding_mask: torch.Tensor | None = None
    accumulate_tokens_per_expert: bool = True


def _group_size_rank(group) -> tuple[int, int]:
    if group is None or not dist.is_available() or not dist.is_initialized():
        return 1, 0
    return dist.get_world_size(group), dist.get_rank(group)


class BaseMoELayer(torch.nn.Module):
    def __init__(self, config: MoEConfig, ep_group, layer_number: Optional[int] = None):
        super().__init__()
        ep_size, ep_rank = _group_size_rank(ep_group)
        self.config = config
        self.expert_parallel_size = ep_size
        assert config.num_moe_experts % ep_size == 0
        self.num_local_experts = config.num_moe_experts // ep_size
        offset = ep_rank * self.num_local_experts
        self.use_shared_expert = config.moe_shared_expert_intermediate_size is not None
        self.local_expert_indices = [offset + i for i in range(self.num_local_experts)]
        self.router = None
        self.experts = None
        self.shared_experts = None
        self.shared_expert = None
        self.shared_expert_gate = None
        self.token_dispatcher = None
        self.layer_number = layer_number
        self._runtime_inputs = MoERuntimeInputs()

    def set_runtime_inputs(self, inputs: MoERuntimeInputs) -> None:
        self._runtime_inputs = inputs


class MoELayer(BaseMoELayer):
    """Mixture-of-experts layer without token dropping."""

    # Whether the layer normalises its input: only where its submodules ask for a norm (a `norm` that
    # they did not ask for is a subclass's own).
    _norms_input = False

    def __init__(self, config: MoEConfig, ep_group=None, submodules: Optional[MoESubmodules] = None,
                 use_te: bool = False, layer_number: Optional[int] = None, sp_group=None):
        self.use_te = use_te
        self.submodules = submodules
        super().__init__(config=config, ep_group=ep_group, layer_number=layer_number)
        self.router = TopKRouter(config=config, layer_number=layer_number, sp_group=sp_group)
        if config.moe_token_dispatcher_type != "alltoall":
            raise ValueError(
                f"Unsupported token dispatcher type: {config.moe_token_dispatcher_type}")
        self.token_dispatcher = MoEAlltoAllTokenDispatcher(
            self.num_local_experts, self.local_expert_indices, config=config, ep_group=ep_group)
        self.experts = build_module(submodules.experts, self.num_local_experts, use_te, config,
                                    layer_number=layer_number)
        if self.use_shared_expert:
            self.shared_experts = build_module(submodules.shared_experts, config=config)
        norm = build_module(getattr(submodules, "norm", None), config=config)
        self._norms_input = norm is not None
        if self._norms_input or not hasattr(type(self), "norm"):
            self.norm = norm

    def _gathering_experts(self, tokens, expert_indices) -> bool:
        """Whether the permutation and unpermutation can be folded into the
        experts' GEMMs (HIP providers for the three ops, plain ``GroupedMLP``
        experts; shapes in ``providers.hip.fused_experts.eligible``)."""
        if type(self.experts) is not GroupedMLP or self.config.moe_apply_probs_on_input:
            return False
        if expert_indices is None or not tokens.is_cuda:
            return False
        try:
            chosen = (ops.selected_impl_name("moe_permutation"),
                      ops.selected_impl_name("grouped_matmul"),
                      ops.selected_impl_name("moe_unpermutation"))
        except RuntimeError:
            return False
        if chosen != ("hip_moe_mask_permutation", "hip_grouped_matmul",
                      "hip_moe_mask_unpermutation"):
            return False
        from ..providers.hip import fused_experts
        return fused_experts.eligible(tokens, self.experts.weight1, expert_indices.shape[1],
                                      self.num_local_experts)

    def _inference_experts(self, hidden_states, probs, expert_indices):
        """The experts' output for a small batch without gradients, in one native call where
        the HIP providers serve the ops it stands for (the conditions are in
        ``providers.hip.fused_experts.inference_eligible``); None otherwise."""
        if torch.is_grad_enabled() or not hidden_states.is_cuda:
            return None
        tokens = hidden_states.view(-1, hidden_states.shape[-1])
        e = self.experts
        fp8 = type(e) is Fp8GroupedMLP
        if not fp8 and type(e) is not GroupedMLP:
            return None
        cfg = e.config
        if not fp8 and (not cfg.gated_linear_unit or cfg.moe_apply_probs_on_input
                        or cfg.activation_func not in (F.silu, F.gelu)):
            return None
        if type(self.token_dispatcher) is not MoEAlltoAllTokenDispatcher:
            return None
        plain = fp8 or e._fused_swiglu
        wanted = (("moe_permutation", "hip_moe_mask_permutation"),
                  ("grouped_matmul_fp8", "hip_grouped_matmul_fp8") if fp8 else
                  ("grouped_matmul", "hip_grouped_matmul"),
                  ("swiglu_probs", "hip_swiglu_probs") if plain else
                  ("gated_activation_probs", "hip_gated_activation_probs"),
                  ("moe_unpermutation", "hip_moe_mask_unpermutation"))
        try:
            if any(ops.selected_impl_name(op) != impl for op, impl in wanted):
                return None
        except RuntimeError:
            return None
        from ..providers.hip import fused_experts
        weights = (e.q1, e.q2) if fp8 else (e.weight1, e.weight2)
        scales = (e.s1, e.s2) if fp8 else None
        if not fused_experts.inference_eligible(e, weights, scales, tokens, probs, expert_indices,
                                                self.num_local_experts, cfg.moe_ffn_hidden_size):
            return None
        output, counts = fused_experts.experts_forward(
            tokens, probs, expert_indices, self.num_local_experts, cfg.moe_ffn_hidden_size,
            weights, scales, F.silu if fp8 else cfg.activation_func,
            0.0 if fp8 else e.swiglu_limit,
            False if fp8 else cfg.moe_swiglu_clamp_gate_after_activation)
        d = self.token_dispatcher
        d.tokens_per_expert = counts
        d.hidden_shape, d.hidden_shape_before_permute = hidden_states.shape, tokens.shape
        return output.view(hidden_states.shape)

    def _mxfp4_inference(self, hidden_states) -> bool:
        """Whether 4-bit experts may read the tokens' rows through the routing index: no gradients,
        nothing attached to the experts, and the HIP providers for the ops this stands in for."""
        if (torch.is_grad_enabled() or not hidden_states.is_cuda
                or type(self.experts) is not Mxfp4GroupedMLP or attached(self.experts, "inference")
                or type(self.token_dispatcher) is not MoEAlltoAllTokenDispatcher
                or self.num_local_experts != self.config.num_moe_experts):
            return False
        wanted = (("moe_permutation", "hip_moe_mask_permutation"),
                  ("moe_unpermutation", "hip_moe_mask_unpermutation"),
                  ("grouped_matmul_mxfp4", "hip_grouped_matmul_mxfp4"))
        try:
            return all(ops.selected_impl_name(op) == impl for op, impl in wanted)
        except RuntimeError:
            return False

    def _mxfp4_experts(self, hidden_states, probs, expert_indices, rows):
        """The output of 4-bit experts without gradients, their rows gathered by the products
        (``rows``: the tokens in 8 bits, or None); None where the conditions do not hold."""
        if expert_indices is None or not self._mxfp4_inference(hidden_states):
            return None
        from ..providers.hip import fused_experts
        output, counts = fused_experts.mxfp4_forward(
            self.experts, hidden_states.view(-1, hidden_states.shape[-1]), rows, probs,
            expert_indices)
        if output is None:
            return None
        d = self.token_dispatcher
        d.tokens_per_expert = counts
        d.hidden_shape = hidden_states.shape
        d.hidden_shape_before_permute = (hidden_states.numel() // hidden_states.shape[-1],
                                         hidden_states.shape[-1])
        return output.view(hidden_states.shape)

    def _normalised(self, hidden_states, residual):
        """(normalised input, the same in 8 bits or None, input + residual or None)."""
        norm = self.norm if self._norms_input else None
        if norm is None:
            if residual is not None:
                raise ValueError("MoELayer takes a residual only with a norm (MoESubmodules.norm)")
            return hidden_states, None, None
        if (type(norm) is RMSNorm and not attached(norm) and self._mxfp4_inference(hidden_states)
                and self.experts.rows_in_8_bits and op_resolves("rms_norm_mx")
                and ops.selected_impl_name("rms_norm_mx") == "hip_rms_norm_mx"
                and ops.selected_impl_name("rms_norm") == "hip_rms_norm"):
            # The router's rows and the experts' in one pass: the rows that the experts would
            # quantise themselves, so that a hook or a check does not change the output.
            out = ops.rms_norm_mx(hidden_states, norm.weight, norm.eps, residual=residual,
                                  with_y=True, rounded=True)
            return out.y, out.rows, out.sum
        if residual is None:
            return norm(hidden_states), None, None
        y, total = norm(hidden_states, residual)
        return y, None, total

    def _combined(self, hidden_states, probs, routing_map, expert_indices, rows):
        # Subclasses that override the call know no rows, unless there are some.
        more = () if rows is None else (rows,)
        return self._experts_and_combine(hidden_states, probs, routing_map, expert_indices, *more)

    def _experts_and_combine(self, hidden_states, probs, routing_map, expert_indices, rows=None):
        flat = hidden_states.view(-1, hidden_states.shape[-1])
        if self._gathering_experts(flat, expert_indices):
            # One GPU, every expert local: the GEMMs gather the token rows
            # themselves (same results, no packed copies).
            from ..providers.hip import fused_experts
            tokens, counts = fused_experts.grouped_mlp_tokens(self.experts, flat, probs,
                                                              routing_map, expert_indices)
            self.token_dispatcher.tokens_per_expert = counts
            output = tokens.view(hidden_states.shape).to(hidden_states.dtype)
        else:
            output = self._inference_experts(hidden_states, probs, expert_indices)
            if output is None:
                output = self._mxfp4_experts(hidden_states, probs, expert_indices, rows)
            if output is None:
                output = self._dispatched_experts(hidden_states, probs, routing_map,
                                                  expert_indices)
        if self.shared_expert is not None:
            if self._adds_itself(self.shared_expert):
                gate = F.sigmoid(self.shared_expert_gate(hidden_states))
                if gate.shape == (*hidden_states.shape[:-1], 1):
                    # The token's gate and the sum in the expert's last product.
                    output = self.shared_expert(hidden_states, output, gate)
                else:
                    output = output + gate * self.shared_expert(hidden_states)
            else:
                # Any other module runs before its gate (moe_layer.py:175-182): hooks and random
                # draws keep their order.
                shared = self.shared_expert(hidden_states)
                output = output + F.sigmoid(self.shared_expert_gate(hidden_states)) * shared
        if self.shared_experts is not None:
            if self._adds_itself(self.shared_experts):
                output = self.shared_experts(hidden_states, output)
            else:
                output = output + self.shared_experts(hidden_states)
        return output

    @staticmethod
    def _adds_itself(expert) -> bool:
        """Whether ``expert`` takes the sum (and a token's gate) into its last product. With
        something attached it is called as any module is: hooks see its own output."""
        return type(expert) is SharedExpertMLP and not attached(expert)

    def _dispatched_experts(self, hidden_states, probs, routing_map, expert_indices):
        d = self.token_dispatcher
        tokens, expert_probs = d.dispatch_preprocess(hidden_states, routing_map, probs,
                                                     expert_indices=expert_indices)
        tokens, expert_probs = d.token_dispatch(tokens, expert_probs)
        tokens, tokens_per_expert, expert_probs = d.dispatch_postprocess(tokens, expert_probs)
        tokens, bias = self.experts(tokens, tokens_per_expert, expert_probs)
        assert bias is None
        tokens = d.combine_preprocess(tokens)
        tokens = d.token_combine(tokens)
        tokens = d.combine_postprocess(tokens)
        return tokens.to(hidden_states.dtype)

    def forward(self, hidden_states, input_ids=None, residual=None):
        """``(output, logits)``; with a norm and a ``residual`` stream ``(output, logits, hidden_states
        + residual)``, the output being that of the normalised sum."""
        hidden_states, rows, total = self._normalised(hidden_states, residual)
        probs, routing_map, expert_indices, logits = self.router(
            hidden_states, input_ids, self._runtime_inputs.padding_mask,
            self._runtime_inputs.accumulate_tokens_per_expert)
        logits = logits.view(-1, logits.shape[-1])
        output = self._combined(hidden_states, probs, routing_map, expert_indices, rows)
        return (output, logits) if residual is None else (output, logits, total)

    def forward_with_logits(self, hidden_states, logits, input_ids=None):
        """Same path with caller-supplied router logits [T, E]."""
        hidden_states, rows, _ = self._normalised(hidden_states, None)
        probs, routing_map, expert_indices = self.router.routing(
            logits, input_ids, self._runtime_inputs.padding_mask,
            self._runtime_inputs.accumulate_tokens_per_expert)
        return self._combined(hidden_states, probs, routing_map, expert_indices, rows)
