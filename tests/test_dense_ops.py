"""Dense products with an epilogue, counter-based dropout and the modules over them, on
the CPU: the oracle's own pins, the refusals of the HIP providers and of the C entry
points (checked before anything reaches a GPU), and the module logic with the oracle's
providers."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle.native_providers import dropout as o_dropout
from oracle.native_providers import linear as o_linear
from torchturbo_amd import _lib as L
from torchturbo_amd.dispatch import OpPolicy, ops
from torchturbo_amd.moe import (CounterDropout, GroupedMLP, GroupedMLPLoRA, MoEConfig, MoELayer,
                                MoESubmodules, ModuleSpec, SharedExpertMLP)
from torchturbo_amd.providers.hip.dropout import HipDropout, drop_threshold
from torchturbo_amd.providers.hip.linear import HipLinearAct, HipLinearResidual
from torchturbo_amd.providers.hip.lora import HipLoRAResidual
from torchturbo_amd.runtime import CpuRuntime


# ---------------------------------------------------------------------------
# The oracle
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("counter, key, words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_published_vectors(counter, key, words):
    got = o_dropout.philox4x32([np.uint64(c) for c in counter], key)
    assert tuple(int(w) for w in got) == words


def test_oracle_mask_is_the_positions():
    """A tensor's first rows and columns take the mask that the smaller tensor takes."""
    key = torch.tensor([-5, 1 << 40])
    big = o_dropout.factors(37, 53, 0.3, key)
    assert torch.equal(big[:11, :9], o_dropout.factors(11, 9, 0.3, key))
    assert abs((big == 0).double().mean().item() - 0.3) < 0.05
    assert not torch.equal(big, o_dropout.factors(37, 53, 0.3, key + 1))


def test_oracle_products_are_exact_on_integers():
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-4, 5, (5, 3, 12), generator=g).float()
    w, b = (torch.randint(-4, 5, s, generator=g).float() for s in ((8, 12), (8,)))
    r = torch.randint(-4, 5, (5, 3, 8), generator=g).float()
    s = torch.tensor([0.0, 0.5, -2.0]).repeat(5, 1)
    plain = torch.einsum("abk,nk->abn", x, w) + b
    assert torch.equal(o_linear.linear_act(x, w, b), plain)
    assert torch.equal(o_linear.linear_residual(x, w, b, r, s), r + s[..., None] * plain)
    assert torch.equal(o_linear.linear_act(x, w, b, activation_func=F.silu, gated=True),
                       F.silu(plain[..., :4]) * plain[..., 4:])


@pytest.mark.parametrize("act, gated", [(None, False), (F.silu, True), (F.gelu, True),
                                        (F.gelu, False)])
def test_oracle_gradients_by_differences(act, gated):
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 5), (8, 5), (8,)))
    w2, b2 = (torch.randn(s, generator=g, dtype=torch.float64)
              for s in ((6, 4 if gated else 8), (6,)))
    r, s = (torch.randn(v, generator=g, dtype=torch.float64) for v in ((3, 6), (3, 1)))
    key = torch.tensor([3, 4])
    leaves = [t.requires_grad_() for t in (x, w, b, w2, b2, r, s)]

    def both(x, w, b, w2, b2, r, s):
        h = o_linear.linear_act(x, w, b, activation_func=act, gated=gated)
        return o_linear.linear_residual(h, w2, b2, r, s, dropout_p=0.25, dropout_key=key)

    assert torch.autograd.gradcheck(both, leaves)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_drop_threshold():
    assert [drop_threshold(p) for p in (0, 1, 0.5, 1e-9, 1 - 1e-9, 0.1)] == \
        [0, 65536, 32768, 1, 65535, 6554]
    assert all(drop_threshold(p) == o_dropout.threshold_of(p)
               for p in (0.0, 1.0, 0.05, 0.1, 0.3, 1e-7))
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="dropout probability"):
            drop_threshold(p)
    with pytest.raises(ValueError, match="dropout probability"):
        CounterDropout(1.5)


KEY = torch.tensor([1, 2])


@pytest.mark.parametrize("call, message", [
    (lambda x, w: HipLinearAct()(x, w.half()), "x and weight must both be"),
    (lambda x, w: HipLinearAct()(x.double(), w.double()), "x and weight must both be"),
    (lambda x, w: HipLinearAct()(x[:, :5], w), "x has 5 features"),
    (lambda x, w: HipLinearAct()(x, w[0]), r"expects x \[..., in\]"),
    (lambda x, w: HipLinearAct()(x, w, torch.zeros(5)), r"the bias must be .* \[6\]"),
    (lambda x, w: HipLinearAct()(x, w, torch.zeros(6, dtype=torch.int32)), "the bias must be"),
    (lambda x, w: HipLinearAct()(x, w[:5], gated=True), "even number of rows"),
    (lambda x, w: HipLinearAct()(x, w, activation_func=F.relu), "only supports"),
    (lambda x, w: HipLinearAct()(x, w), "HIP kernels need device tensors"),
    (lambda x, w: HipLinearResidual()(x, w, None, torch.zeros(4, 5)), "the residual must be"),
    (lambda x, w: HipLinearResidual()(x, w, None, torch.zeros(4, 6).half()), "the residual must be"),
    (lambda x, w: HipLinearResidual()(x, w, None, torch.zeros(1, 6)), "the residual must be"),
    (lambda x, w: HipLinearResidual()(x, w, None, None, torch.zeros(4, 6)), "row_scale must be"),
    (lambda x, w: HipLinearResidual()(x, w, None, None, torch.zeros(1)), "row_scale must be"),
    (lambda x, w: HipLinearResidual()(x, w, dropout_p=0.5), "needs a key"),
    (lambda x, w: HipLinearResidual()(x, w, dropout_p=0.5, dropout_key=KEY.int()), "needs a key"),
    (lambda x, w: HipLinearResidual()(x, w, dropout_p=2.0), "dropout probability"),
    (lambda x, w: HipLinearResidual()(x, w), "HIP kernels need device tensors"),
    (lambda x, w: HipDropout()(x.double(), 0.5, KEY), "takes f32, bf16 or f16"),
    (lambda x, w: HipDropout()(x[0, 0], 0.5, KEY), "at least one dimension"),
    (lambda x, w: HipDropout()(x, 0.5, KEY[:1]), "needs a key"),
    (lambda x, w: HipDropout()(x, 0.5, None), "needs a key"),
    (lambda x, w: HipDropout()(x, 0.5, KEY), "HIP kernels need device tensors"),
    (lambda x, w: HipLoRAResidual()(x, x, w, w, KEY, 1.0, dropout_p=-1), "dropout probability"),
])
def test_refusals_of_the_providers(call, message):
    with pytest.raises(ValueError, match=message):
        call(torch.zeros(4, 8), torch.zeros(6, 8))


def null(name, **given):
    """A call of a C entry point with null pointers and sizes that would be taken but for ``given``."""
    sizes = {"m": 4, "k": 8, "n": 8, "dtype": L.TT_BF16, "act": 1, "gated": 1, "t": 0, "bias": None,
             "bias_dt": L.TT_F32, "scale": None, "scale_dt": L.TT_F32, "key": None, "ds": None,
             "bytes": 1 << 40}
    s = {**sizes, **given}
    args = {
        "tt_linear_act_fwd": lambda: (None, None, s["bias"], s["bias_dt"], s["dtype"], s["m"],
                                      s["k"], s["n"], s["act"], s["gated"], None, None, None, 0,
                                      None),
        "tt_linear_act_bwd": lambda: (None, None, None, None, s["dtype"], s["m"], s["k"], s["n"],
                                      s["act"], s["gated"], None, None, s["bias"], s["bias_dt"],
                                      None, s["bytes"], None),
        "tt_linear_residual_fwd": lambda: (None, None, s["bias"], s["bias_dt"], None, s["scale"],
                                           s["scale_dt"], s["dtype"], s["m"], s["k"], s["n"],
                                           s["t"], s["key"], None, None, 0, None),
        "tt_linear_residual_bwd": lambda: (None, None, None, s["bias"], s["bias_dt"], s["scale"],
                                           s["scale_dt"], s["dtype"], s["m"], s["k"], s["n"],
                                           s["t"], s["key"], None, None, None, s["ds"], None,
                                           s["bytes"], None),
        "tt_dropout": lambda: (None, s["dtype"], s["m"], s["n"], s["t"], s["key"], None, None),
        "tt_lora_down_dropout": lambda: (None, None, s["dtype"], s["m"], s["k"], 4, 2, None, s["t"],
                                         s["key"], None, None),
        "tt_lora_up_dropout": lambda: (None, None, s["dtype"], s["m"], s["k"], 4, 2, None, s["t"],
                                       s["key"], None, None),
        "tt_lora_wgrad_dropout": lambda: (None, None, s["dtype"], s["m"], s["k"], 4, 2, None,
                                          s["t"], s["key"], None, None),
    }[name]()
    L.call(name, *args)


P = ctypes.c_void_p(16)


@pytest.mark.parametrize("name, given, message", [
    ("tt_linear_act_fwd", {"dtype": L.TT_F64}, "must be f32, bf16 or f16"),
    ("tt_linear_act_fwd", {"m": -1}, "bad sizes"),
    ("tt_linear_act_fwd", {"n": 1 << 30}, "bad sizes"),
    ("tt_linear_act_fwd", {"act": 3}, "unknown activation"),
    ("tt_linear_act_fwd", {"bias": P, "bias_dt": L.TT_F8E4M3}, "the bias must be"),
    ("tt_linear_act_bwd", {"act": -1}, "unknown activation"),
    ("tt_linear_act_bwd", {"bias": P, "bias_dt": L.TT_F64}, "the bias must be"),
    ("tt_linear_act_bwd", {"bytes": 100}, "workspace is too small"),
    ("tt_linear_residual_fwd", {"t": 65537}, "threshold must be"),
    ("tt_linear_residual_fwd", {"t": 5}, "dropout without a key"),
    ("tt_linear_residual_fwd", {"scale": P, "scale_dt": L.TT_F64}, "the row scale must be"),
    ("tt_linear_residual_bwd", {"t": 5}, "dropout without a key"),
    ("tt_linear_residual_bwd", {"t": -1}, "threshold must be"),
    ("tt_linear_residual_bwd", {"t": 5, "key": P, "bytes": 100}, "workspace is too small"),
    ("tt_linear_residual_bwd", {"ds": P}, "needs a row scale"),
    ("tt_dropout", {"dtype": L.TT_F64}, "must be f32, bf16 or f16"),
    ("tt_dropout", {"m": 1 << 32}, "bad sizes"),
    ("tt_dropout", {"t": 65537}, "threshold must be"),
    ("tt_dropout", {"t": 5}, "null pointer"),
    ("tt_lora_down_dropout", {"t": 0}, "threshold must be"),
    ("tt_lora_up_dropout", {"t": 5}, "dropout without a key"),
    ("tt_lora_wgrad_dropout", {"t": 5, "k": 9, "key": P}, "multiples of 8"),
])
def test_refusals_of_the_entry_points(name, given, message):
    with pytest.raises(ValueError, match=message):
        null(name, **given)


def test_empty_calls_of_the_entry_points_launch_nothing():
    null("tt_linear_act_fwd", m=0)
    null("tt_linear_residual_fwd", n=0)
    null("tt_linear_act_bwd", n=0)  # nor here, with no gradient asked for
    null("tt_linear_residual_bwd")
    null("tt_dropout", n=0)
    null("tt_lora_down_dropout", m=0, t=5, key=P)


# ---------------------------------------------------------------------------
# Modules
# ---------------------------------------------------------------------------
def shared_config(gated=True, act=F.silu, **more):
    return MoEConfig(hidden_size=16, num_moe_experts=4, moe_ffn_hidden_size=8, moe_router_topk=2,
                     gated_linear_unit=gated, activation_func=act,
                     moe_shared_expert_intermediate_size=12, **more)


@pytest.mark.parametrize("gated, act, bias", [(True, F.silu, False), (True, F.gelu, True),
                                              (False, F.gelu, True)])
def test_shared_expert_is_the_dense_mlp(process_ops, gated, act, bias):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    torch.manual_seed(3)
    mlp = SharedExpertMLP(shared_config(gated, act), bias=bias)
    names = ["up_proj", "down_proj"] + (["gate_proj"] if gated else [])
    hf = {}
    for n in names:
        rows, cols = (16, 12) if n == "down_proj" else (12, 16)
        hf[n + ".weight"] = torch.randn(rows, cols)
        if bias:
            hf[n + ".bias"] = torch.randn(rows)
    mlp.load_state_dict(hf)
    x = torch.randn(2, 5, 16)

    def lin(n, v):
        return F.linear(v, hf[n + ".weight"], hf.get(n + ".bias"))

    h = act(lin("gate_proj", x)) * lin("up_proj", x) if gated else act(lin("up_proj", x))
    torch.testing.assert_close(mlp(x), lin("down_proj", h))
    r, s = torch.randn(2, 5, 16), torch.rand(2, 5, 1)
    torch.testing.assert_close(mlp(x, r, s), r + s * lin("down_proj", h))


def test_shared_expert_arguments(process_ops):
    with pytest.raises(ValueError, match="moe_shared_expert_intermediate_size"):
        SharedExpertMLP(MoEConfig(hidden_size=8, activation_func=F.silu))
    with pytest.raises(ValueError, match="silu or gelu"):
        SharedExpertMLP(shared_config(act=F.relu))


def test_shared_expert_dropout_follows_the_generator(process_ops):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    torch.manual_seed(4)
    mlp = SharedExpertMLP(shared_config(), dropout=0.4)
    x, r = torch.randn(7, 16), torch.randn(7, 16)
    torch.manual_seed(5)
    a, b = mlp(x, r), mlp(x, r)
    torch.manual_seed(5)
    assert torch.equal(mlp(x, r), a) and not torch.equal(a, b)
    assert 0 < (a == r).sum() < a.numel()  # dropped elements leave the residual
    mlp.eval()
    torch.testing.assert_close(mlp(x, r), r + mlp(x))


class _Plain(torch.nn.Module):
    """The same expert as its own module: the layer's earlier path."""

    def __init__(self, mlp):
        super().__init__()
        self.mlp = mlp

    def forward(self, x):
        return self.mlp(x)


@pytest.mark.parametrize("gate_width", [1, 16])
def test_layer_adds_the_shared_expert(process_ops, gate_width):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    torch.manual_seed(6)
    cfg = shared_config()
    layer = MoELayer(cfg, None, MoESubmodules(experts=ModuleSpec(module=GroupedMLP),
                                              shared_experts=ModuleSpec(module=SharedExpertMLP)))
    layer.shared_expert = SharedExpertMLP(cfg)
    layer.shared_expert_gate = torch.nn.Linear(16, gate_width, bias=False)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(std=0.2)
    x = torch.randn(3, 5, 16)
    got, _ = layer(x)
    grads = torch.autograd.grad(got.square().sum(), list(layer.parameters()))
    one, two = layer.shared_expert, layer.shared_experts
    layer.shared_expert, layer.shared_experts = _Plain(one), _Plain(two)
    want, _ = layer(x)
    torch.testing.assert_close(got, want)
    for a, b in zip(grads, torch.autograd.grad(want.square().sum(), list(layer.parameters()))):
        torch.testing.assert_close(a, b)


def test_counter_dropout_module(process_ops):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    drop = CounterDropout(0.25)
    x = torch.randn(64, 40)
    torch.manual_seed(1)
    y, z = drop(x), drop(x)
    torch.manual_seed(1)
    assert torch.equal(drop(x), y) and not torch.equal(y, z)
    kept = y != 0
    torch.testing.assert_close(y[kept], x[kept] / 0.75, rtol=1e-5, atol=0)
    drop.eval()
    assert drop(x) is x
    assert CounterDropout(0.0)(x) is x and "p=0.25" in repr(drop)


def test_lora_counter_dropout_is_opt_in(process_ops):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    cfg = MoEConfig(hidden_size=8, moe_ffn_hidden_size=6, gated_linear_unit=True,
                    activation_func=F.silu)
    torch.manual_seed(2)
    base = GroupedMLP(2, False, cfg)
    with torch.no_grad():
        for p in base.parameters():
            p.normal_(std=0.3)
    plain = GroupedMLPLoRA(base, "default", r=2, lora_dropout=0.3)
    assert type(plain.lora_dropout["default"]) is torch.nn.Dropout
    lora = GroupedMLPLoRA(base, "default", r=2, lora_dropout=0.3, counter_dropout=True,
                          init_lora_weights="gaussian")
    assert type(lora.lora_dropout["default"]) is CounterDropout
    with torch.no_grad():
        for n, p in lora.named_parameters():
            if "lora_B" in n:
                p.normal_()
    x, counts, probs = torch.randn(9, 8), torch.tensor([4, 5]), torch.rand(9)
    torch.manual_seed(7)
    got, _ = lora(x, counts, probs)
    torch.manual_seed(7)
    keys = [CounterDropout.draw_key("cpu") for _ in range(2)]

    def residual(v, a, b, key):
        d = ops.dropout(v, 0.3, key)
        return ops.grouped_matmul(ops.grouped_matmul(d, a.weight, counts), b.weight,
                                  counts) * lora.scaling["default"]

    w1, w2 = base.weight1.view(2, 8, -1), base.weight2.view(2, 6, 8)
    h = ops.grouped_matmul(x, w1, counts) + residual(x, lora.lora_A["default"],
                                                     lora.lora_B["default"], keys[0])
    act = base.activation_func_with_probs(h, probs)
    want = ops.grouped_matmul(act, w2, counts) + residual(act, lora.lora_A2["default"],
                                                          lora.lora_B2["default"], keys[1])
    torch.testing.assert_close(got, want)
    lora.eval()
    assert torch.equal(lora(x, counts, probs)[0], lora(x, counts, probs)[0])


# ---------------------------------------------------------------------------
# What autograd has to see
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(5))
def test_tangents_and_transforms_are_refused(monkeypatch, which, grad):
    """A dual tensor does not require gradients: a native call on its address would lose
    the tangent without a word, so the operators raise, as all others of the package do."""
    from torchturbo_amd.providers.hip import linear as hip_linear

    # The native calls stubbed, everything before them as it is.
    monkeypatch.setattr(hip_linear, "require_cuda", lambda *t: None)
    monkeypatch.setattr(hip_linear, "act_fwd", lambda x, w, *a: torch.zeros(x.shape[0], w.shape[0]))
    monkeypatch.setattr(hip_linear, "residual_fwd",
                        lambda x, w, *a: torch.zeros(x.shape[0], w.shape[0]))
    leaves = [torch.ones(s) for s in ((4, 8), (6, 8), (6,), (4, 6), (4, 1))]
    calls = [lambda v: HipLinearResidual()(*v)]
    if which < 3:
        calls.append(lambda v: HipLinearAct()(*v[:3]))
    fwd = torch.autograd.forward_ad
    for call in calls:
        def of(t):
            return call([t if i == which else v for i, v in enumerate(leaves)])

        with torch.set_grad_enabled(grad):
            assert of(leaves[which]).shape == (4, 6)
            with fwd.dual_level():
                assert of(leaves[which]).shape == (4, 6)  # no tangent: nothing to lose
                with pytest.raises(NotImplementedError, match="jvp"):
                    of(fwd.make_dual(leaves[which], torch.ones_like(leaves[which])))
            with pytest.raises(RuntimeError, match="autograd.Function"):
                torch.func.jvp(of, (leaves[which],), (torch.ones_like(leaves[which]),))


# ---------------------------------------------------------------------------
# What a caller attaches to the modules
# ---------------------------------------------------------------------------
def shared_layer(expert):
    torch.manual_seed(6)
    cfg = shared_config()
    layer = MoELayer(cfg, None, MoESubmodules(experts=ModuleSpec(module=GroupedMLP)))
    layer.shared_expert = expert(cfg)
    layer.shared_expert_gate = torch.nn.Linear(16, 1, bias=False)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(std=0.2)
    return layer


def test_another_shared_expert_runs_before_its_gate(process_ops):
    """The order of the reference: that of hooks, and of random draws in either of the two."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    layer = shared_layer(lambda cfg: torch.nn.Sequential(torch.nn.Linear(16, 16),
                                                         torch.nn.Dropout(0.5)))
    layer.shared_expert_gate = torch.nn.Sequential(torch.nn.Dropout(0.5), torch.nn.Linear(16, 1))
    seen = []
    layer.shared_expert.register_forward_hook(lambda *a: seen.append("expert"))
    layer.shared_expert_gate.register_forward_hook(lambda *a: seen.append("gate"))
    x = torch.randn(3, 5, 16)
    torch.manual_seed(1)
    got, _ = layer(x)
    assert seen == ["expert", "gate"]
    expert, gate = layer.shared_expert, layer.shared_expert_gate
    layer.shared_expert = None
    routed, _ = layer(x)
    torch.manual_seed(1)
    shared = expert(x)
    assert torch.equal(got, routed + F.sigmoid(gate(x)) * shared)


class _FusedOps:
    """Stands in for the process dispatcher where the HIP operators are chosen."""

    def __init__(self, **chosen):
        self.chosen = {"lora_residual": "hip_lora_residual", "dropout": "hip_dropout",
                       "grouped_matmul": "hip_grouped_matmul",
                       "linear_residual": "hip_linear_residual", **chosen}
        self.calls = []

    def selected_impl_name(self, op):
        return self.chosen[op]

    def lora_residual(self, base, x, a, b, counts, scale, **dropout):
        self.calls.append(("lora_residual", sorted(dropout)))
        return base

    def dropout(self, x, p, key):
        self.calls.append(("dropout", p))
        return x


def _hook(drop):
    drop.register_forward_hook(lambda *a: None)


def _pre_hook(drop):
    drop.register_forward_pre_hook(lambda *a: None)


def _backward_hook(drop):
    drop.register_full_backward_hook(lambda *a: None)


def _replaced(drop):
    drop.forward = type(drop).forward.__get__(drop)


class _OnGpu:
    is_cuda, device = True, torch.device("cpu")


@pytest.mark.filterwarnings("ignore:For backward hooks to be called")
@pytest.mark.parametrize("attach, chosen, fused", [
    (None, {}, True), (_hook, {}, False), (_pre_hook, {}, False), (_backward_hook, {}, False),
    (_replaced, {}, False), (None, {"dropout": "other"}, False),
    (None, {"lora_residual": "other"}, False)])
def test_lora_calls_a_dropout_that_something_is_attached_to(monkeypatch, attach, chosen, fused):
    """The fused operator makes the mask itself only where calling the module would do
    nothing else: hooks run, and another implementation that was chosen is called."""
    from torchturbo_amd.moe import dropout as m_dropout
    from torchturbo_amd.moe import lora as m_lora

    fake = _FusedOps(**chosen)
    monkeypatch.setattr(m_lora, "ops", fake)
    monkeypatch.setattr(m_dropout, "ops", fake)
    monkeypatch.setattr(m_lora, "op_resolves", lambda name: True)
    cfg = MoEConfig(hidden_size=8, moe_ffn_hidden_size=6, gated_linear_unit=True,
                    activation_func=F.silu)
    lora = GroupedMLPLoRA(GroupedMLP(2, False, cfg), "default", r=2, lora_dropout=0.3,
                          counter_dropout=True)
    drop = lora.lora_dropout["default"]
    x, counts = _OnGpu(), torch.tensor([4, 5])
    if attach is not None:
        attach(drop)
    lora._add_residual(torch.zeros(1), x, counts, "default", lora.lora_A, lora.lora_B)
    if fused:
        assert fake.calls == [("lora_residual", ["dropout_key", "dropout_p"])]
    else:
        assert fake.calls == [("dropout", 0.3), ("lora_residual", [])]


@pytest.mark.parametrize("attach", [_hook, _pre_hook, _backward_hook, _replaced, "module"])
@pytest.mark.parametrize("scaled", [True, False])
def test_shared_expert_calls_a_dropout_that_something_is_attached_to(process_ops, monkeypatch,
                                                                     attach, scaled):
    """The same values as with the mask made in the product's epilogue."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    torch.manual_seed(4)
    mlp = SharedExpertMLP(shared_config(), dropout=0.4)
    x, r, s = torch.randn(7, 16), torch.randn(7, 16), torch.rand(7) if scaled else None
    torch.manual_seed(5)
    want = mlp(x, r, s)
    calls, forward = [], CounterDropout.forward
    monkeypatch.setattr(CounterDropout, "forward",
                        lambda self, v: calls.append(v.shape) or forward(self, v))
    if attach == "module":
        mlp.dropout = torch.nn.Sequential(mlp.dropout)
    else:
        attach(mlp.dropout)
    torch.manual_seed(5)
    torch.testing.assert_close(mlp(x, r, s), want)
    assert calls == [(7, 16)]
    torch.manual_seed(5)
    torch.testing.assert_close(mlp(x), want - r if s is None else (want - r) / s[:, None],
                               rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("chosen, calls", [
    ({}, [("linear_residual", True)]),
    ({"dropout": "other"}, [("linear_residual", False), ("dropout", 0.4)]),
    # Another product brings a dropout of its own.
    ({"dropout": "other", "linear_residual": "other"}, [("linear_residual", True)])])
def test_shared_expert_uses_the_dropout_that_was_chosen(monkeypatch, chosen, calls):
    from torchturbo_amd.moe import dropout as m_dropout
    from torchturbo_amd.moe import shared_experts as m_shared

    fake = _FusedOps(**chosen)
    fake.linear_act = lambda x, w, b, **how: x @ w[:12].t()

    def linear_residual(x, w, b, residual=None, row_scale=None, *, dropout_p=0.0, dropout_key=None):
        fake.calls.append(("linear_residual", dropout_p > 0))
        return x @ w.t()

    fake.linear_residual = linear_residual
    for module in (m_dropout, m_shared):
        monkeypatch.setattr(module, "ops", fake)
    mlp = SharedExpertMLP(shared_config(), dropout=0.4)
    mlp(torch.randn(7, 16), torch.randn(7, 16))
    assert fake.calls == calls
    fake.calls.clear()
    mlp.eval()  # nothing to drop: one product, whatever is chosen
    mlp(torch.randn(7, 16), torch.randn(7, 16))
    assert fake.calls == [("linear_residual", False)]


@pytest.mark.parametrize("name", ["shared_expert", "shared_experts"])
@pytest.mark.parametrize("attach", ["hook", "pre_hook", "replaced"])
def test_what_is_attached_to_a_shared_expert_sees_the_expert_alone(process_ops, name, attach):
    """Its input, and its output without the gate and the routed experts, as with any module."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    layer = shared_layer(SharedExpertMLP)
    expert = layer.shared_expert
    if name == "shared_experts":
        layer.shared_expert, layer.shared_experts = None, expert
    x = torch.randn(3, 5, 16)
    want, own = layer(x)[0], expert(x)
    seen = []
    if attach == "hook":
        expert.register_forward_hook(lambda m, args, out: seen.append((args, out)))
    elif attach == "pre_hook":
        expert.register_forward_pre_hook(lambda m, args: seen.append((args, own)))
    else:
        forward = expert.forward
        expert.forward = lambda v: seen.append(((v,), forward(v))) or seen[-1][1]
    torch.testing.assert_close(layer(x)[0], want)
    (args, out), = seen
    assert len(args) == 1 and torch.equal(args[0], x)
    torch.testing.assert_close(out, own)


# ---------------------------------------------------------------------------
# Pointers of the entry points
# ---------------------------------------------------------------------------
def pointers(name, given, **sizes):
    """A call of a C entry point whose pointers are NULL but for those ``given`` (an address
    that no kernel ever gets: every such call is refused)."""
    s = {"m": 4, "k": 8, "n": 8, "t": 0, "act": 1, "gated": 1, "bytes": 1 << 40, **sizes}
    size = (L.TT_BF16, s["m"], s["k"], s["n"])
    given = given if isinstance(given, dict) else dict.fromkeys(given, 4096)
    g = {n: ctypes.c_void_p(v) for n, v in given.items()}.get
    L.call(name, *{
        "tt_linear_act_fwd": lambda: (g("x"), g("w"), g("bias"), 0, *size, s["act"], s["gated"],
                                      g("pre"), g("y"), g("ws"), s["bytes"], None),
        "tt_linear_act_bwd": lambda: (g("dy"), g("x"), g("w"), g("pre"), *size, s["act"],
                                      s["gated"], g("dx"), g("dw"), g("db"), 0, g("ws"),
                                      s["bytes"], None),
        "tt_linear_residual_fwd": lambda: (g("x"), g("w"), g("bias"), 0, g("res"), g("scale"), 0,
                                           *size, s["t"], g("key"), g("y"), g("ws"), s["bytes"],
                                           None),
        "tt_linear_residual_bwd": lambda: (g("dy"), g("x"), g("w"), g("bias"), 0, g("scale"), 0,
                                           *size, s["t"], g("key"), g("dx"), g("dw"), g("db"),
                                           g("ds"), g("ws"), s["bytes"], None),
    }[name]())


@pytest.mark.parametrize("name, given, missing", [
    ("tt_linear_act_fwd", "w y ws", "x"),
    ("tt_linear_act_fwd", "x y ws", "w"),
    ("tt_linear_act_fwd", "x w ws", "y"),
    ("tt_linear_act_fwd", "x w y", "the workspace"),
    ("tt_linear_act_bwd", "x w pre dx dw ws", "dy"),
    ("tt_linear_act_bwd", "dy x w dx ws", "pre"),
    ("tt_linear_act_bwd", "dy db ws", "pre"),
    ("tt_linear_act_bwd", "dy x pre dx ws", "w"),
    ("tt_linear_act_bwd", "dy w pre dw ws", "x"),
    ("tt_linear_act_bwd", "dy x w pre dx dw", "the workspace"),
    ("tt_linear_residual_fwd", "w y ws", "x"),
    ("tt_linear_residual_fwd", "x y ws res scale bias", "w"),
    ("tt_linear_residual_fwd", "x w ws", "y"),
    ("tt_linear_residual_fwd", "x w y", "the workspace"),
    ("tt_linear_residual_bwd", "x w dx dw ws", "dy"),
    ("tt_linear_residual_bwd", "db ws", "dy"),
    ("tt_linear_residual_bwd", "dy x dx ws", "w"),
    ("tt_linear_residual_bwd", "dy x scale dw ws", "w"),
    ("tt_linear_residual_bwd", "dy x scale ds ws", "w"),
    ("tt_linear_residual_bwd", "dy w dw ws", "x"),
    ("tt_linear_residual_bwd", "dy w scale ds ws", "x"),
    ("tt_linear_residual_bwd", "dy x w dx db", "the workspace"),
])
def test_null_pointers_are_refused(name, given, missing):
    with pytest.raises(ValueError, match=rf"null pointer \({missing}\)"):
        pointers(name, given.split())


@pytest.mark.parametrize("name, given", [
    ("tt_linear_act_fwd", "x w y"), ("tt_linear_residual_fwd", "x w y"),
    ("tt_linear_act_bwd", "dy x w pre dx"), ("tt_linear_residual_bwd", "dy x w dx")])
def test_a_workspace_off_its_alignment_is_refused(name, given):
    with pytest.raises(ValueError, match="aligned to 256 bytes"):
        pointers(name, {**{n: 4096 for n in given.split()}, "ws": 4096 + 16})


def test_calls_that_ask_for_no_gradient_launch_nothing():
    pointers("tt_linear_act_bwd", [])
    pointers("tt_linear_residual_bwd", ["scale", "key"], t=7)


@pytest.mark.parametrize("name", ["tt_lora_down_dropout", "tt_lora_up_dropout",
                                  "tt_lora_wgrad_dropout"])
@pytest.mark.parametrize("missing", range(4))
def test_null_pointers_of_the_adapters_are_refused(name, missing):
    at = [None if i == missing else ctypes.c_void_p(4096) for i in range(4)]
    with pytest.raises(ValueError, match="null pointer"):
        L.call(name, at[0], at[1], L.TT_BF16, 4, 8, 4, 2, at[2], 5, P, at[3], None)


@pytest.mark.parametrize("m, base, transposed, taken", [
    (0, None, 0, True), (0, P, 0, True), (0, None, 1, True), (0, P, 1, False),
    (4, None, 0, False), (4, P, 1, False)])
def test_base_of_the_up_projection(m, base, transposed, taken):
    """A base in the gradient's form is refused, of an empty call too, whose base may
    be NULL in the forward's."""
    args = ("tt_lora_up", P, P, base, L.TT_BF16, m, 8, 4, transposed, 1.0, 2, P, P, None)
    if taken:
        L.call(*args)
    else:
        with pytest.raises(ValueError, match="forward form only"):
            L.call(*args)


# ---------------------------------------------------------------------------
# Which kernel runs a product
# ---------------------------------------------------------------------------
def test_sizes_of_the_gpu_tests_take_the_kernels_they_name():
    from test_gpu_linear import BF, HF, WIDE, plan

    for op, T, K, N, plans in WIDE:
        for dtype in (BF, HF):
            assert " ".join(plan(op, i, T, K, N, dtype) for i in range(3)) == plans, (op, T, K, N)
    # A weight of more than 4 GiB goes to the tiles however few the rows are.
    assert plan("residual", 0, 3, 32768, 69640) == "T64/1"
    assert plan("residual", 0, 3, 8192, 8192) == plan("gated", 0, 1, 7168, 2048) == "ROWS/1"


def test_plan_query():
    query = L.load().tt_linear_plan
    f32, bf = L.TT_F32, L.TT_BF16
    assert query(2, 0, f32, 512, 256, 512, 1) % 256 == 0
    # An address off 16 bytes, or a size off eight elements: the kernels of any alignment.
    assert query(0, 0, bf, 200, 128, 128, 1) % 256 == 2 and query(0, 0, bf, 200, 128, 128, 0) % 256 == 6
    assert query(0, 0, bf, 200, 127, 128, 1) % 256 == 6
    for bad in ((3, 0, bf, 4, 8, 8), (-1, 0, bf, 4, 8, 8), (0, 3, bf, 4, 8, 8), (0, -1, bf, 4, 8, 8),
                (0, 0, L.TT_F64, 4, 8, 8), (0, 0, bf, -1, 8, 8), (0, 0, bf, 0, 8, 8),
                (0, 1, bf, 4, 0, 8), (0, 2, bf, 4, 8, 0)):
        assert query(*bad, 1) == -1


@pytest.mark.parametrize("name, given", [("tt_linear_act_fwd", "x w y"),
                                         ("tt_linear_residual_fwd", "x w y")])
def test_more_tiles_than_a_launch_has_are_refused(name, given):
    """A launch ends below 2^32 threads, 2^24 blocks of 256."""
    with pytest.raises(ValueError, match="grid too large"):
        pointers(name, given.split(), m=(1 << 30) + 1, k=4, bytes=0)


@pytest.mark.parametrize("name, rows, rank", [("tt_lora_down_dropout", 1 << 29, 64),
                                              ("tt_lora_up_dropout", 1 << 30, 4)])
def test_more_blocks_of_the_adapters_than_a_launch_has_are_refused(name, rows, rank):
    at = ctypes.c_void_p(4096)
    with pytest.raises(ValueError, match="grid too large"):
        L.call(name, at, at, L.TT_BF16, rows, 8, rank, 2, at, 5, P, at, None)
