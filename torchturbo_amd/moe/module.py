"""Module spec helpers (``src/torchturbo/models/modules/moe/module.py:20-107``)."""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Any

import torch


@dataclass
class ModuleSpec:
    module: type
    params: dict = field(default_factory=dict)
    submodules: Any = None


def build_module(spec_or_module, *args, **kwargs):
    if spec_or_module is None:
        return None
    if isinstance(spec_or_module, ModuleSpec):
        params = dict(spec_or_module.params)
        params.update(kwargs)
        if spec_or_module.submodules is not None:
            params["submodules"] = spec_or_module.submodules
        return spec_or_module.module(*args, **params)
    if isinstance(spec_or_module, type):
        return spec_or_module(*args, **kwargs)
    return spec_or_module


def attached(module, *methods: str) -> bool:
    """Whether calling ``module`` runs more than its class's ``forward``: hooks of its own or
    of all modules, or one of ``methods`` replaced on the instance. Fused operators that
    stand in for the call step back then."""
    every = torch.nn.modules.module
    hooks = (module._forward_hooks, module._forward_pre_hooks, module._backward_hooks,
             module._backward_pre_hooks, every._global_forward_hooks,
             every._global_forward_pre_hooks, every._global_backward_hooks,
             every._global_backward_pre_hooks)
    return any(hooks) or any(n in vars(module) for n in ("forward", *methods))
