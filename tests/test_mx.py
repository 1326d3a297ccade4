"""4-bit weights, rows in 8 bits and the norm on the CPU: the oracle's own pins, the refusals of the HIP
providers and of the C entry points (checked before anything reaches a GPU), and the modules with
the oracle's providers."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.nn.functional as F

from oracle.native_providers import mx as o_mx
from oracle.native_providers import norm as o_norm
from torchturbo_amd import _lib as L
from torchturbo_amd.dispatch import MxRows, OpPolicy, ops
from torchturbo_amd.moe import (GroupedMLP, MoEConfig, MoELayer, MoESubmodules, ModuleSpec,
                                Mxfp4GroupedMLP, Mxfp4SharedExpertMLP, RMSNorm, SharedExpertMLP)
from torchturbo_amd.providers.hip.mx import (HipDequantizeMxfp4, HipDequantizeMxfp8,
                                             HipGroupedMatmulMxfp4, HipLinearMxfp4,
                                             HipQuantizeMxfp4, HipQuantizeMxfp8, _device)
from torchturbo_amd.providers.hip.norm import HipRmsNorm, HipRmsNormMx
from torchturbo_amd.runtime import CpuRuntime

BF16 = torch.bfloat16


# ---------------------------------------------------------------------------
# The oracle
# ---------------------------------------------------------------------------
def test_oracle_codes_of_the_formats():
    """Each code's value by the formats' fields; scales; the packing's order."""
    values = o_mx.e2m1_values(torch.arange(256, dtype=torch.uint8))
    for byte in range(256):
        for half, code in enumerate((byte & 15, byte >> 4)):
            e, m = (code >> 1) & 3, code & 1
            want = (m / 2 if e == 0 else (1 + m / 2) * 2 ** (e - 1)) * (-1) ** (code >> 3)
            assert values[2 * byte + half] == want
    s = o_mx.scale_values(torch.tensor([0, 127, 130, 254, 255], dtype=torch.uint8))
    assert s[:4].tolist() == [2.0 ** -127, 1.0, 8.0, 2.0 ** 127] and s[4].isnan()


def test_oracle_rounding():
    """Ties go to the even code, what exceeds the largest value stays there, and the scale is that of
    the largest magnitude's exponent."""
    v = torch.zeros(32)
    v[:12] = torch.tensor([4.0, 5.0, 7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5.01, -0.2, 0.26])
    codes, scales = o_mx.quantize_mxfp4(v)
    assert scales.tolist() == [127]
    assert o_mx.dequantize_mxfp4(codes, scales, torch.float32)[:12].tolist() == \
        [4.0, 4.0, 6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, -6.0, 0.0, 0.5]
    v[:12] = torch.tensor([256.0, 511.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 449.0, 1.0, 0, 0, 0, 0])
    rows = o_mx.quantize_mxfp8(v)
    assert rows.scales.tolist() == [127]
    assert rows.codes.float()[:8].tolist() == [256.0, 448.0, 16.0, 20.0, 0.0, 2.0 ** -8, 448.0, 1.0]
    x = torch.randn(5, 96, generator=torch.Generator().manual_seed(0)) * 3.0
    for _ in range(2):  # values of the format are kept
        codes, scales = o_mx.quantize_mxfp4(x)
        again = o_mx.dequantize_mxfp4(codes, scales, torch.float32)
        assert _ == 0 or torch.equal(again, x)
        assert ((again - x).abs() <= x.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) / 4).all()
        x = again
    assert torch.equal(o_mx.quantize_mxfp8(x.float()).codes.float().view(-1),
                       x.unflatten(-1, (-1, 32)).div(o_mx.scale_values(
                           o_mx.quantize_mxfp8(x).scales).unsqueeze(-1)).float().view(-1))


def test_oracle_special_values():
    x = torch.zeros(4, 32)
    x[1, 3], x[2, 4], x[3, 5] = float("nan"), float("inf"), 2.0 ** -140
    codes, scales = o_mx.quantize_mxfp4(x)
    assert scales.view(-1).tolist() == [0, 255, 255, 0]
    v = o_mx.dequantize_mxfp4(codes, scales, torch.float32)
    assert not v[0].any() and v[1:3].isnan().all() and not v[3].any()
    rows = o_mx.quantize_mxfp8(x)
    assert rows.scales.view(-1).tolist() == [0, 255, 255, 0]
    assert o_mx.dequantize_mxfp8(rows)[1:3].isnan().all()


@pytest.mark.parametrize("residual", [False, True])
def test_oracle_norm_gradients_by_differences(residual):
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(3, 7, generator=g, dtype=torch.float64).requires_grad_() for _ in range(2))
    w = torch.randn(7, generator=g, dtype=torch.float64).requires_grad_()
    leaves = [x, w] + ([r] if residual else [])
    assert torch.autograd.gradcheck(lambda *a: o_norm.norm(a[0], a[1], 1e-3, *a[2:]), leaves)
    y, h = o_norm.norm(x, w, 0.0)
    assert torch.allclose((y / w).square().mean(-1), torch.ones(3, dtype=torch.float64))


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
X = torch.zeros(4, 64, dtype=BF16)
Q, S = torch.zeros(6, 32, dtype=torch.uint8), torch.zeros(6, 2, dtype=torch.uint8)
QE, SE = Q.expand(3, 6, 32), S.expand(3, 6, 2)
R8 = MxRows(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8))
W = torch.ones(64)


@pytest.mark.parametrize("call, message", [
    (lambda: HipLinearMxfp4()(X.half(), Q, S), "takes bf16 rows"),
    (lambda: HipLinearMxfp4()(X.tolist(), Q, S), "takes bf16 rows"),
    (lambda: HipLinearMxfp4()(X[:, :32], Q, S), "x has 32 features, weight expects 64"),
    (lambda: HipLinearMxfp4()(X, Q.int(), S), "codes must be uint8"),
    (lambda: HipLinearMxfp4()(X, Q, S.float()), "scales must be uint8"),
    (lambda: HipLinearMxfp4()(X, Q[0], S[0]), "expects codes of 2 dimensions"),
    (lambda: HipLinearMxfp4()(X, Q[:, :8], S[:, :1]), "whole groups of 32"),
    (lambda: HipLinearMxfp4()(X, Q, S[:, :1]), "need scales"),
    (lambda: HipLinearMxfp4()(X, Q[:5], S[:5], gated=True), "even number of rows"),
    (lambda: HipLinearMxfp4()(X, Q, S, mx_out=True), "whole groups of 32, got 6"),
    (lambda: HipLinearMxfp4()(X, Q, S, activation_func=F.relu), "only supports"),
    (lambda: HipLinearMxfp4()(MxRows(R8.codes, R8.scales[:, :1]), Q, S), "rows in 8 bits are"),
    (lambda: HipLinearMxfp4()(MxRows(X, R8.scales), Q, S), "rows in 8 bits are"),
    (lambda: HipLinearMxfp4()(X, Q, S), "HIP kernels need device tensors"),
    (lambda: HipLinearMxfp4()(R8, Q, S), "HIP kernels need device tensors"),
    (lambda: HipGroupedMatmulMxfp4()(X, Q, S, [4]), "expects codes of 3 dimensions"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE[:0], SE[:0], []), "at least one expert"),
    (lambda: HipGroupedMatmulMxfp4()(X[None], QE, SE, [4, 0, 0]), "packed rows"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE, SE, [4, 0, 0], probs=torch.ones(3)), r"shape \[4\]"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE, SE, [4, 0, 0], probs=torch.ones(4).int()), "probs must be"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE, SE, [4, 0, 0], row_map=torch.zeros(4)), "row_map must be"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE[:, :5], SE[:, :5], [4, 0, 0], gated=True), "even number"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE, SE, [4, 0, 0], mx_out=True), "whole groups"),
    (lambda: HipGroupedMatmulMxfp4()(X, QE, SE, [4, 0, 0]), "HIP kernels need device tensors"),
    (lambda: HipQuantizeMxfp4()(X[:, :40]), "whole groups of 32"),
    (lambda: HipQuantizeMxfp4()(X.double()), "takes f32, bf16 or f16"),
    (lambda: HipQuantizeMxfp8()(torch.zeros(())), "whole groups of 32"),
    (lambda: HipQuantizeMxfp8()(X), "HIP kernels need device tensors"),
    (lambda: HipDequantizeMxfp4()(Q, S, torch.float64), "gives f32, bf16 or f16"),
    (lambda: HipDequantizeMxfp4()(Q, S[:, :1]), "need scales"),
    (lambda: HipDequantizeMxfp4()(torch.zeros((), dtype=torch.uint8), S), "dimensions"),
    (lambda: HipDequantizeMxfp8()(X), "takes MxRows"),
    (lambda: HipDequantizeMxfp8()(R8), "HIP kernels need device tensors"),
    (lambda: HipRmsNorm()(X, W[:63]), r"the weight must have shape \[64\]"),
    (lambda: HipRmsNorm()(X.double(), W), "takes f32, bf16 or f16"),
    (lambda: HipRmsNorm()(X, W.int()), "takes f32, bf16 or f16"),
    (lambda: HipRmsNorm()(X[0, 0], W), "at least one dimension"),
    (lambda: HipRmsNorm()(X, W, residual=X[:2]), "the residual must be"),
    (lambda: HipRmsNorm()(X, W, residual=X.float()), "the residual must be"),
    (lambda: HipRmsNorm()(X, W), "HIP kernels need device tensors"),
    (lambda: HipRmsNormMx()(X[:, :40], W[:40]), "whole groups of 32, got 40"),
    (lambda: HipRmsNormMx()(X, W), "HIP kernels need device tensors"),
])
def test_refusals(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_tensors_of_another_gpu_than_the_current_one(monkeypatch):
    class Elsewhere:
        device = torch.device("cuda", 1)

        def get_device(self):
            return 1

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="cuda:1, which is not the current device"):
        _device(Elsewhere(), None, Elsewhere())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    assert _device(Elsewhere(), None, Elsewhere()) == Elsewhere.device


def test_rows_in_8_bits_have_no_gradient():
    """Codes that ask for one (or a transform that follows them) are refused before any product."""
    rows = MxRows(R8.codes.clone().requires_grad_(), R8.scales)
    calls = (lambda r: HipLinearMxfp4()(r, Q, S),
             lambda r: HipGroupedMatmulMxfp4()(r, QE, SE, [4, 0, 0]))
    for call in calls:
        with pytest.raises(RuntimeError, match="rows in 8 bits have no gradient"):
            call(rows)
        with torch.autograd.forward_ad.dual_level(), torch.no_grad(), \
                pytest.raises(RuntimeError, match="rows in 8 bits have no gradient"):
            call(R8)


AT = ctypes.c_void_p(4096)  # an address that no kernel ever gets: every such call is refused
ODD = ctypes.c_void_p(4104)


def _product(**over):
    a = dict(x=AT, xs=None, map=None, src=16, q=AT, s=AT, M=16, K=64, N=32, E=1, counts=None, gated=0,
             act=0, probs=None, pdt=0, y=AT, ys=None, ws=None, size=0, stream=None)
    a.update(over)
    return "tt_mx_product", tuple(a.values())


def _dgrad(**over):
    a = dict(dy=AT, q=AT, s=AT, M=16, K=64, N=32, E=1, counts=None, dx=AT, stream=None)
    a.update(over)
    return "tt_mx_dgrad", tuple(a.values())


def _norm(**over):
    a = dict(x=AT, r=None, w=AT, wdt=0, dt=1, T=4, H=64, eps=1e-6, y=AT, sum=None, rstd=None, codes=None,
             scales=None, stream=None)
    a.update(over)
    return "tt_rms_norm_fwd", tuple(a.values())


def _norm_bwd(**over):
    a = dict(h=AT, w=AT, wdt=0, rstd=AT, gy=AT, gs=None, dt=1, T=4, H=64, dx=AT, dw=AT, ws=AT,
             size=1 << 20, stream=None)
    a.update(over)
    return "tt_rms_norm_bwd", tuple(a.values())


@pytest.mark.parametrize("call, message", [
    (_product(K=48), "whole groups"),
    (_product(M=-1), "bad sizes"),
    (_product(E=0), "bad sizes"),
    (_product(E=2), "need their counts"),
    (_product(act=3), "activation"),
    (_product(probs=AT, pdt=4), "probabilities"),
    (_product(N=40, ys=AT), "whole groups of 32 columns"),
    (_product(y=None), "NULL output"),
    (_product(x=None), "NULL tensor"),
    (_product(s=None), "NULL tensor"),
    (_product(x=ODD), "16-byte aligned"),
    (_product(q=ODD), "16-byte aligned"),
    (_product(ys=AT, y=ctypes.c_void_p(4100)), "8-byte aligned"),
    (_product(map=AT, src=0), "row map of no rows"),
    (_product(K=1 << 31), "sizes past"),
    (_product(M=1 << 31), "sizes past"),
    (_dgrad(K=48), "whole groups"),
    (_dgrad(N=-1), "bad sizes"),
    (_dgrad(E=2), "need their counts"),
    (_dgrad(dx=None), "NULL tensor"),
    (_dgrad(dy=None), "NULL tensor"),
    (_dgrad(q=ODD), "16-byte aligned"),
    (_dgrad(N=1 << 24), "sizes past"),
    (_norm(dt=4), "must be f32"),
    (_norm(wdt=3), "must be f32"),
    (_norm(T=-1), "bad sizes"),
    (_norm(x=None), "NULL tensor"),
    (_norm(codes=AT), "or neither"),
    (_norm(codes=AT, scales=AT, H=40), "whole groups"),
    (_norm(codes=ctypes.c_void_p(4100), scales=AT), "8-byte aligned"),
    (_norm(sum=AT), "needs a residual"),
    (_norm_bwd(T=0), "the caller's"),
    (_norm_bwd(gy=None), "NULL tensor"),
    (_norm_bwd(size=8), "workspace too small"),
    (("tt_mxfp4_quantize", (AT, 4, 4, 64, AT, AT, None)), "must be f32"),
    (("tt_mxfp4_quantize", (AT, 1, 4, 40, AT, AT, None)), "whole groups"),
    (("tt_mxfp4_quantize", (None, 1, 4, 64, AT, AT, None)), "NULL tensor"),
    (("tt_mxfp8_quantize", (AT, 1, 4, 64, ctypes.c_void_p(4100), AT, None)), "8-byte aligned"),
    (("tt_mxfp4_quantize", (AT, 1, 1 << 31, 1 << 12, AT, AT, None)), "too many|too large"),
    (("tt_mxfp4_dequantize", (AT, AT, -1, 64, AT, 1, None)), "whole groups"),
    (("tt_mxfp8_dequantize", (AT, AT, 4, 64, None, 1, None)), "NULL tensor"),
])
def test_entry_points_refuse_before_any_launch(call, message):
    name, args = call
    with pytest.raises(ValueError, match=message):
        L.call(name, *args)


def test_entry_points_of_nothing_do_nothing():
    for name, args in (_product(M=0), _product(N=0, x=None), _dgrad(M=0), _dgrad(K=0), _norm(T=0),
                       _norm(H=0), ("tt_mxfp4_quantize", (None, 1, 0, 64, None, None, None)),
                       ("tt_mxfp8_dequantize", (None, None, 4, 0, None, 1, None))):
        L.call(name, *args)
    size = L.load().tt_mx_product_workspace
    assert size(1, 7168, 2048, 0, 1) == 0 and size(128, 7168, 2048, 1, 1) == 0
    # 128 x 4096 outputs in 64 x 128 tiles, the reduction of 7168 in four parts.
    assert size(128, 7168, 2048, 0, 1) == 4 * 128 * 4096 * 4
    assert L.load().tt_rms_norm_bwd_workspace(0, 64) == 0


# ---------------------------------------------------------------------------
# Modules
# ---------------------------------------------------------------------------
def _config(**over):
    kw = dict(hidden_size=64, num_moe_experts=4, moe_ffn_hidden_size=96, gated_linear_unit=True,
              activation_func=F.silu, moe_router_topk=2, params_dtype=torch.float32)
    kw.update(over)
    return MoEConfig(**kw)


def _filled(module, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in module.parameters():
            p.copy_(torch.randn(p.shape, generator=g) * 0.1)
    return module


def test_experts_are_grouped_mlp_with_the_quantised_weights(process_ops):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    cfg = _config()
    plain = _filled(GroupedMLP(4, False, cfg))
    experts = Mxfp4GroupedMLP(4, False, cfg)
    experts.quantize(plain.weight1, plain.weight2)
    with torch.no_grad():
        w1 = o_mx.dequantize_mxfp4(experts.q1, experts.s1, torch.float32)  # [E, 2F, H]
        w2 = o_mx.dequantize_mxfp4(experts.q2, experts.s2, torch.float32)
        error = (w1.transpose(1, 2).reshape_as(plain.weight1) - plain.weight1).norm()
        assert error < 0.15 * plain.weight1.norm()
        plain.weight1.copy_(w1.transpose(1, 2).reshape_as(plain.weight1))
        plain.weight2.copy_(w2.transpose(1, 2).reshape_as(plain.weight2))
    g = torch.Generator().manual_seed(1)
    x, probs, counts = torch.randn(20, 64, generator=g), torch.rand(20, generator=g), torch.tensor([5, 0, 12, 3])
    outs = []
    for module in (plain, experts):
        leaves = [x.clone().requires_grad_(), probs.clone().requires_grad_()]
        y, bias = module(leaves[0], counts, leaves[1])
        assert bias is None
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))])
    for a, b in zip(*outs):  # one in 64 bits, one in 32
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    with torch.no_grad():
        assert torch.equal(experts(x, counts, probs)[0], experts.inference(x, counts, probs))
        experts.rows_in_8_bits = True
        y8 = experts(x, counts, probs)[0]
        assert y8.dtype == BF16
        # Two roundings of 2^-4 at most and bf16's, averaged over 64 and 96 features.
        assert (y8.double() - outs[1][0]).norm() < 0.08 * outs[1][0].norm()
        rows = ops.quantize_mxfp8(x)
        assert torch.equal(experts(rows, counts, probs)[0], y8)
    y, _ = experts(x.clone().requires_grad_(), counts, probs)  # gradients: plain rows
    assert torch.equal(y.detach(), outs[1][0])


def test_module_refusals_and_state(process_ops):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    for over, message in (({"activation_func": F.gelu}, "SwiGLU"), ({"hidden_size": 72}, "divisible by 32"),
                          ({"moe_ffn_hidden_size": 40}, "divisible by 32"),
                          ({"moe_apply_probs_on_input": True}, "probabilities")):
        with pytest.raises(ValueError, match=message):
            Mxfp4GroupedMLP(4, False, _config(**over))
    with pytest.raises(ValueError, match="limit"):
        Mxfp4GroupedMLP(4, False, _config(moe_swiglu_limit=[7.0]), layer_number=0)
    with pytest.raises(ValueError, match="intermediate_size"):
        Mxfp4SharedExpertMLP(_config())
    experts = Mxfp4GroupedMLP(4, False, _config())
    with pytest.raises(ValueError, match="do not fit"):
        experts.quantize(torch.zeros(4 * 64, 64), torch.zeros(4 * 32, 64))
    with pytest.raises(ValueError, match="q1 must be uint8"):
        experts.load_quantized(experts.q1.int(), experts.s1, experts.q2, experts.s2)
    with pytest.raises(ValueError, match="s2 has shape"):
        experts.load_quantized(experts.q1, experts.s1, experts.q2, experts.s2[:2])
    codes, scales = o_mx.quantize_mxfp4(torch.randn(4, 192, 64))
    experts.load_quantized(codes.view(torch.float4_e2m1fn_x2), scales.view(torch.float8_e8m0fnu),
                           experts.q2, experts.s2)
    assert torch.equal(experts.q1, codes) and torch.equal(experts.s1, scales)
    other = Mxfp4GroupedMLP(4, False, _config())
    other.load_state_dict(experts.state_dict())
    assert torch.equal(other.q1, codes) and not list(experts.parameters())
    assert experts.to(BF16).q1.dtype == torch.uint8


@pytest.mark.parametrize("act, gated", [(F.silu, True), (F.gelu, False)])
def test_shared_expert(process_ops, act, gated):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    cfg = _config(moe_shared_expert_intermediate_size=128, activation_func=act, gated_linear_unit=gated)
    plain, small = _filled(SharedExpertMLP(cfg)), Mxfp4SharedExpertMLP(cfg)
    small.quantize(plain.weight1.detach(), plain.weight2.detach())
    with torch.no_grad():
        plain.weight1.copy_(o_mx.dequantize_mxfp4(small.q1, small.s1, torch.float32))
        plain.weight2.copy_(o_mx.dequantize_mxfp4(small.q2, small.s2, torch.float32))
    x = torch.randn(3, 5, 64, generator=torch.Generator().manual_seed(2))
    assert torch.allclose(small(x), plain(x), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("residual", [False, True])
def test_layer_with_a_norm(process_ops, residual):
    """Its output is that of the layer without on the normalised input, and the stream the sum."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    cfg = _config(moe_shared_expert_intermediate_size=128)
    subs = dict(experts=ModuleSpec(module=Mxfp4GroupedMLP),
                shared_experts=ModuleSpec(module=Mxfp4SharedExpertMLP))
    layer = MoELayer(cfg, None, submodules=MoESubmodules(**subs, norm=ModuleSpec(RMSNorm, {"eps": 1e-5})))
    bare = MoELayer(cfg, None, submodules=MoESubmodules(**subs))
    src = _filled(GroupedMLP(4, False, cfg))
    layer.experts.quantize(src.weight1, src.weight2)
    sw = _filled(SharedExpertMLP(cfg), 3)
    layer.shared_experts.quantize(sw.weight1.detach(), sw.weight2.detach())
    with torch.no_grad():
        layer.norm.weight.uniform_(0.5, 1.5)
    state = layer.state_dict()
    assert "norm.weight" in state
    bare.load_state_dict({k: v for k, v in state.items() if not k.startswith("norm")})
    g = torch.Generator().manual_seed(4)
    x, r = torch.randn(2, 6, 64, generator=g), torch.randn(2, 6, 64, generator=g)
    if residual:
        out, logits, total = layer(x, residual=r)
        y, h = ops.rms_norm(x, layer.norm.weight, 1e-5, residual=r)
        assert torch.equal(total, h)
    else:
        (out, logits), y = layer(x), ops.rms_norm(x, layer.norm.weight, 1e-5)
    want, want_logits = bare(y)
    assert torch.equal(out, want) and torch.equal(logits, want_logits)
    assert torch.equal(layer.forward_with_logits(x, logits), bare.forward_with_logits(
        ops.rms_norm(x, layer.norm.weight, 1e-5), logits))
    with pytest.raises(ValueError, match="only with a norm"):
        bare(x, residual=r)
    calls = []
    handle = layer.norm.register_forward_hook(lambda *a: calls.append(1))
    layer(x)
    handle.remove()
    assert calls == [1]


def test_rounded_rows_of_the_norm(process_ops):
    """The rows that ``quantize_mxfp8`` gives for the output; not asked for, a provider without them serves."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(40, 64, generator=g).to(BF16), torch.rand(64, generator=g).to(BF16)
    out = ops.rms_norm_mx(x, w, with_y=True, rounded=True)
    want = ops.quantize_mxfp8(ops.rms_norm(x, w))
    assert torch.equal(out.y, ops.rms_norm(x, w))
    assert torch.equal(out.rows.codes.float(), want.codes.float())
    assert torch.equal(out.rows.scales, want.scales)
    plain = ops.rms_norm_mx(x, w).rows
    assert (plain.codes.float() != want.codes.float()).any()  # the unrounded y's differ here and there
    with pytest.raises(ValueError, match="NULL tensor"):
        L.call("tt_rms_norm_fwd_rounded", *_norm(x=None)[1])


def test_shared_expert_refuses_weights_of_other_shapes(process_ops):
    """Also those that would fill every row by broadcasting; nothing is written then."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    small = Mxfp4SharedExpertMLP(_config(moe_shared_expert_intermediate_size=128))
    w1, w2 = torch.randn(256, 64), torch.randn(64, 128)
    small.quantize(w1, w2)
    state = {k: v.clone() for k, v in small.state_dict().items()}
    for a, b in ((w1[:1], w2[:1]), (w1[:1], w2), (w1, w2[:1]), (w1, w2[:, :64]), (w1[:128], w2),
                 (w1[None], w2), (w1[0], w2), (w1, w2.t())):
        with pytest.raises(ValueError, match=r"do not fit \[256, 64\] and \[64, 128\]"):
            small.quantize(-a, -b)
        assert all(torch.equal(v, state[k]) for k, v in small.state_dict().items())


def test_a_refused_checkpoint_leaves_the_weights(process_ops):
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    experts = Mxfp4GroupedMLP(4, False, _config())
    state = {k: v.clone() for k, v in experts.state_dict().items()}
    ones = [torch.ones_like(t) for t in (experts.q1, experts.s1, experts.q2, experts.s2)]
    for bad in (ones[3][:2], ones[3].int()):
        with pytest.raises(ValueError, match="s2"):
            experts.load_quantized(*ones[:3], bad)
        assert all(torch.equal(v, state[k]) for k, v in experts.state_dict().items())
    experts.load_quantized(*ones)
    assert all((v == 1).all() for v in experts.state_dict().values())


def test_8_bit_conversions_do_not_cut_a_gradient():
    """Gradients, tangents and transforms are refused before any GPU is looked for; what none follows
    reaches the device's check."""
    x = torch.randn(4, 64)
    calls = ((HipQuantizeMxfp8(), x, lambda v: v), (HipDequantizeMxfp8(), R8.codes,
                                                    lambda v: MxRows(v, R8.scales)))
    for op, plain, form in calls:
        leaf = plain.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            op(form(leaf))
        for v in (plain, leaf.detach()):
            with pytest.raises(ValueError, match="need device tensors"):
                op(form(v))
        with torch.no_grad(), pytest.raises(ValueError, match="need device tensors"):
            op(form(leaf))
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(ValueError, match="need device tensors"):
                op(form(plain))
            dual = torch.autograd.forward_ad.make_dual(plain, torch.ones_like(plain))
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                op(form(dual))
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.vmap(lambda v: HipQuantizeMxfp8()(v).codes)(x[None])
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.jvp(lambda v: HipQuantizeMxfp8()(v).codes.float(), (x,), (x,))


def test_a_subclass_keeps_what_it_calls_norm(process_ops):
    """A norm that no submodule spec asked for is the subclass's own: the layer does not apply it."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    subs = MoESubmodules(experts=ModuleSpec(module=GroupedMLP))

    class Normed(MoELayer):
        def __init__(self, cfg):
            super().__init__(cfg, None, submodules=subs)
            self.norm = RMSNorm(cfg)

        def forward(self, x, input_ids=None):
            return super().forward(self.norm(x), input_ids)

    class Measured(MoELayer):
        def norm(self, x):
            return x.norm()

    plain = _filled(MoELayer(_config(), None, submodules=subs))
    x = torch.randn(6, 64, generator=torch.Generator().manual_seed(8))
    normed = Normed(_config())
    normed.load_state_dict(plain.state_dict(), strict=False)
    with torch.no_grad():
        normed.norm.weight.uniform_(0.5, 1.5)
        want, logits = plain(normed.norm(x))
        assert all(torch.equal(a, b) for a, b in zip(normed(x), (want, logits)))
        measured = Measured(_config(), None, submodules=subs)
        measured.load_state_dict(plain.state_dict())
        assert measured.norm(x) == x.norm()
        assert torch.equal(measured(x)[0], plain(x)[0]) and plain.norm is None
    with pytest.raises(ValueError, match="only with a norm"):
        MoELayer.forward(normed, x, residual=x)


def test_a_subclass_that_combines_by_itself(process_ops):
    """An override with the arguments that the layer had before there were rows in 8 bits serves a layer
    without them."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    subs = MoESubmodules(experts=ModuleSpec(module=GroupedMLP))

    class Halved(MoELayer):
        def _experts_and_combine(self, hidden_states, probs, routing_map, expert_indices):
            return super()._experts_and_combine(hidden_states, probs, routing_map, expert_indices) / 2

    plain = _filled(MoELayer(_config(), None, submodules=subs))
    halved = Halved(_config(), None, submodules=subs)
    halved.load_state_dict(plain.state_dict())
    x = torch.randn(6, 64, generator=torch.Generator().manual_seed(9))
    with torch.no_grad():
        want, logits = plain(x)
        assert torch.equal(halved(x)[0], want / 2)
        assert torch.equal(halved.forward_with_logits(x, logits), want / 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, BF16])
def test_shared_expert_with_8_bit_rows_keeps_the_dtype(process_ops, dtype):
    """Its products give bf16; the output is in the input's dtype, as SharedExpertMLP's, and so is the
    layer's."""
    process_ops(CpuRuntime(), OpPolicy.NATIVE, oracle=True)
    cfg = _config(moe_shared_expert_intermediate_size=128, params_dtype=dtype)
    eight = {"rows_in_8_bits": True}
    layer = MoELayer(cfg, None, submodules=MoESubmodules(
        experts=ModuleSpec(Mxfp4GroupedMLP, eight), shared_experts=ModuleSpec(Mxfp4SharedExpertMLP, eight)))
    layer.shared_experts.quantize(torch.randn(256, 64), torch.randn(64, 128))
    x = torch.randn(6, 64, generator=torch.Generator().manual_seed(10)).to(dtype)
    with torch.no_grad():
        shared = layer.shared_experts(x)
        assert shared.dtype == dtype and shared.any() and torch.equal(shared.to(BF16).to(dtype), shared)
        assert layer(x)[0].dtype == dtype


def test_no_workspace_for_reductions_that_are_not_split():
    """Split reductions are multiples of 128: other sizes ask for no scratch, which no kernel would touch."""
    size = L.load().tt_mx_product_workspace
    for K in (7136, 7104, 7200):
        assert size(128, K, 2048, 0, 1) == size(128, K, 2048, 0, 0) == 0
    assert size(128, 7040, 2048, 0, 1) > 0


def test_counts_of_another_gpu_are_refused(monkeypatch):
    """The kernels read the counts where they are: those of another GPU than the rows' are refused."""
    from torchturbo_amd.providers.hip import mx as provider

    def launched(*a, **k):
        raise AssertionError("launched")

    monkeypatch.setattr(provider, "_device", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(provider, "device_counts", lambda c, *a, **k: c)  # device counts come back as they are
    monkeypatch.setattr(provider, "product", launched)
    counts = torch.tensor([4, 0, 0], device="meta")  # on a device that is not cuda:0
    with pytest.raises(ValueError, match="tokens_per_expert is on meta, the rows on cuda:0"):
        HipGroupedMatmulMxfp4()(X, QE, SE, counts)
