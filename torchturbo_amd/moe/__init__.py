"""MoE layer stack (router, EP=1 token dispatcher, grouped experts, shared expert)."""

from .dropout import CounterDropout
from .experts import Fp8GroupedMLP, GroupedMLP
from .fp8_checkpoint import SafetensorsCheckpoint, load_fp8_experts
from .lora import GroupedLoRALinear, GroupedMLPLoRA
from .module import ModuleSpec, build_module
from .moe_config import MoEConfig, get_base_moe_config
from .moe_layer import MoELayer, MoERuntimeInputs, MoESubmodules
from .mxfp4 import Mxfp4GroupedMLP, Mxfp4SharedExpertMLP
from .norm import RMSNorm
from .router import MoEAuxLossAutoScaler, RouterGatingLinearFunction, TopKRouter
from .shared_experts import SharedExpertMLP
from .token_dispatcher import MoEAlltoAllTokenDispatcher

__all__ = [
    "CounterDropout",
    "Fp8GroupedMLP",
    "GroupedLoRALinear",
    "GroupedMLP",
    "GroupedMLPLoRA",
    "MoEAlltoAllTokenDispatcher",
    "MoEAuxLossAutoScaler",
    "MoEConfig",
    "MoELayer",
    "MoERuntimeInputs",
    "MoESubmodules",
    "ModuleSpec",
    "Mxfp4GroupedMLP",
    "Mxfp4SharedExpertMLP",
    "RMSNorm",
    "RouterGatingLinearFunction",
    "SafetensorsCheckpoint",
    "SharedExpertMLP",
    "TopKRouter",
    "build_module",
    "get_base_moe_config",
    "load_fp8_experts",
]
