"""The layer with 4-bit experts, their shared expert and the norm, as a decoder would run them, on the GPU.

Against 64 bits: every stage's bf16 rounding is 2^-8 of its value at most and E4M3's 2^-4; over the
hundreds of terms of each product they average out, so the norm of the error stays below the sum
of the stages' steps over sqrt(3) (uniform errors), taken here without that root.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle.native_providers import mx as o_mx
from oracle.native_providers import norm as o_norm
from tests.conftest import assert_bf16_close
from torchturbo_amd import checks
from torchturbo_amd.dispatch import OpPolicy, ops
from torchturbo_amd.moe import (GroupedMLP, MoEConfig, MoELayer, MoESubmodules, ModuleSpec,
                                Mxfp4GroupedMLP, Mxfp4SharedExpertMLP, RMSNorm)
from torchturbo_amd.runtime import CudaRuntime

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
H, F_, E, K = 256, 128, 8, 2


def _layer(eight=False, norm=True, shared=True, experts=Mxfp4GroupedMLP):
    cfg = MoEConfig(hidden_size=H, num_moe_experts=E, moe_ffn_hidden_size=F_, gated_linear_unit=True,
                    activation_func=F.silu, moe_router_topk=K, params_dtype=BF16,
                    moe_router_dtype="fp32",
                    moe_shared_expert_intermediate_size=192 if shared else None)
    params = {"rows_in_8_bits": eight} if experts is Mxfp4GroupedMLP else {}
    layer = MoELayer(cfg, None, submodules=MoESubmodules(
        experts=ModuleSpec(experts, params),
        shared_experts=ModuleSpec(Mxfp4SharedExpertMLP, {"rows_in_8_bits": eight}) if shared else None,
        norm=ModuleSpec(RMSNorm) if norm else None)).to(DEV)
    g = torch.Generator().manual_seed(0)
    w1, w2 = torch.randn(E * H, 2 * F_, generator=g) * 0.1, torch.randn(E * F_, H, generator=g) * 0.1
    with torch.no_grad():
        layer.router.weight.copy_(torch.randn(E, H, generator=g) * 0.3)
        if experts is Mxfp4GroupedMLP:
            layer.experts.quantize(w1.to(BF16).to(DEV), w2.to(BF16).to(DEV))
        if norm:
            layer.norm.weight.copy_(1 + 0.2 * torch.randn(H, generator=g))
        if shared:
            layer.shared_experts.quantize(torch.randn(384, H, generator=g).to(BF16).to(DEV) * 0.1,
                                          torch.randn(H, 192, generator=g).to(BF16).to(DEV) * 0.1)
    return layer


def _tokens(shape, seed=1):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


@pytest.mark.parametrize("tokens", [1, 7, 64, 700])
@pytest.mark.parametrize("eight", [False, True])
def test_gathered_rows_are_the_dispatched_ones(process_ops, tokens, eight):
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(eight, norm=False)
    x = _tokens((tokens, H))
    with torch.no_grad():
        gathered, logits = layer(x)
        counts = layer.token_dispatcher.tokens_per_expert.clone()
        seen = []
        handle = layer.experts.register_forward_hook(lambda m, a, o: seen.append(a[0].shape))
        dispatched, logits2 = layer(x)
        handle.remove()
    assert seen == [(tokens * K, H)]
    assert torch.equal(gathered, dispatched) and torch.equal(logits, logits2)
    assert torch.equal(counts, layer.token_dispatcher.tokens_per_expert)


@pytest.mark.parametrize("tokens", [1, 33, 600])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_block_against_64_bits(process_ops, tokens, eight, residual):
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(eight)
    x, r = _tokens((tokens, H)), _tokens((tokens, H), 2) if residual else None
    with torch.no_grad():
        out = layer(x, residual=r)
        y, h = o_norm.norm(x.cpu(), layer.norm.weight.cpu(), 1e-6, None if r is None else r.cpu())
        # The routing that the layer took, from its own rows.
        probs, _, ids, _ = layer.router((layer.norm(x) if r is None else layer.norm(x, r)[0]))
    if residual:
        assert torch.equal(out[2].cpu(), h.to(BF16))
    e, s = layer.experts, layer.shared_experts
    ids, probs = ids.cpu(), probs.double().cpu()
    want = torch.zeros(tokens, H, dtype=torch.float64)
    for i in range(E):
        t, _ = (ids == i).nonzero(as_tuple=True)
        a = o_mx.linear(y[t], e.q1[i].cpu(), e.s1[i].cpu(), F.silu, True) * probs[t, i].unsqueeze(1)
        want[t] += o_mx.linear(a, e.q2[i].cpu(), e.s2[i].cpu())
    want += o_mx.linear(o_mx.linear(y, s.q1.cpu(), s.s1.cpu(), F.silu, True), s.q2.cpu(), s.s2.cpu())
    got = out[0].double().cpu()
    # y, the activations and the sums; with 8 bits the rows twice.
    steps = 4 * 2.0 ** -8 + (2 * 2.0 ** -4 if eight else 0.0)
    assert (got - want).norm() <= steps * want.norm()


def test_gradients_are_those_of_the_dequantised_experts(process_ops):
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer, plain = _layer(shared=False), _layer(shared=False, experts=GroupedMLP)
    e = layer.experts
    with torch.no_grad():
        w1 = ops.dequantize_mxfp4(e.q1, e.s1)
        w2 = ops.dequantize_mxfp4(e.q2, e.s2)
        plain.experts.weight1.copy_(w1.transpose(1, 2).reshape(E * H, 2 * F_))
        plain.experts.weight2.copy_(w2.transpose(1, 2).reshape(E * F_, H))
        plain.router.weight.copy_(layer.router.weight)
        plain.norm.weight.copy_(layer.norm.weight)
    grads = []
    for m in (layer, plain):
        x, r = _tokens((300, H)).requires_grad_(), _tokens((300, H), 2).requires_grad_()
        out, _, total = m(x, residual=r)
        loss_grad = _tokens((300, H), 3)
        grads.append([out.detach(), *torch.autograd.grad([out, total], [x, r, m.norm.weight, m.router.weight],
                                                          [loss_grad, loss_grad])])
    for a, b, name in zip(*grads, ("out", "dx", "dr", "dw", "drouter")):
        assert_bf16_close(a, b, what=name)


def test_decode_step_in_a_graph(process_ops):
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(True)
    x, r = _tokens((4, H)), _tokens((4, H), 2)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                layer(x, residual=r)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = layer(x, residual=r)
        for seed in range(4):
            x.copy_(_tokens((4, H), 10 + seed))
            r.copy_(_tokens((4, H), 20 + seed))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, layer(x, residual=r)))


def test_two_streams_at_once(process_ops):
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(True)
    xs = [_tokens((500, H), s) for s in range(4)]
    with torch.no_grad():
        want = [layer(x)[0] for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in xs]
        got = []
        for x, s in zip(xs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append([layer(x)[0] for _ in range(3)])
        torch.cuda.synchronize()
    assert all(torch.equal(a, w) for many, w in zip(got, want) for a in many)


def test_empty_batch(process_ops):
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    for eight in (False, True):
        layer = _layer(eight)
        with torch.no_grad():
            out, _, total = layer(_tokens((0, H)), residual=_tokens((0, H)))
        assert out.shape == total.shape == (0, H)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_column_major_tokens(process_ops, eight, norm):
    """A dense [T, H] whose tokens lie along the fast dimension: the output is that of its copy."""
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(eight, norm=norm)
    x = _tokens((65, H))
    turned = x.t().contiguous().t()
    assert not turned.is_contiguous() and torch.equal(turned, x)
    # Given logits: a library product of the turned tokens may round them another way.
    logits = torch.randn(65, E, generator=torch.Generator().manual_seed(3)).to(DEV)
    with torch.no_grad():
        out, want = (layer.forward_with_logits(t, logits) for t in (turned, x))
    assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [1, 7, 64, 700])
@pytest.mark.parametrize("residual", [False, True])
def test_the_norms_rows_are_those_of_its_output(process_ops, tokens, residual):
    """With rows in 8 bits: a hook on the experts or on the norm, or checks of the inputs, send the layer
    another way; its output stays the same."""
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(True)
    x, r = _tokens((tokens, H)), _tokens((tokens, H), 2) if residual else None
    with torch.no_grad():
        want = layer(x, residual=r)
        others = []
        for module in (layer.experts, layer.norm):
            handle = module.register_forward_hook(lambda *a: None)
            others.append(layer(x, residual=r))
            handle.remove()
        with checks.checking():
            others.append(layer(x, residual=r))
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(want, other))


@pytest.mark.parametrize("eight", [False, True])
def test_every_token_against_64_bits(process_ops, eight):
    """The bound of the block's norm for each token by itself: a token that took another's rows or experts
    would be off by its whole norm. Roundings are uniform errors, so that a token's error comes to
    1 / sqrt(3) of the sum of its steps and less, and with 256 features hardly varies."""
    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    layer = _layer(eight)
    x, r = _tokens((600, H)), _tokens((600, H), 2)
    with torch.no_grad():
        got = layer(x, residual=r)[0].double().cpu()
        probs, _, ids, _ = layer.router(layer.norm(x, r)[0])
    y, _ = o_norm.norm(x.cpu(), layer.norm.weight.cpu(), 1e-6, r.cpu())
    e, s = layer.experts, layer.shared_experts
    ids, probs = ids.cpu(), probs.double().cpu()
    want = o_mx.linear(o_mx.linear(y, s.q1.cpu(), s.s1.cpu(), F.silu, True), s.q2.cpu(), s.s2.cpu())
    for i in range(E):
        t, _ = (ids == i).nonzero(as_tuple=True)
        a = o_mx.linear(y[t], e.q1[i].cpu(), e.s1[i].cpu(), F.silu, True) * probs[t, i].unsqueeze(1)
        want[t] += o_mx.linear(a, e.q2[i].cpu(), e.s2[i].cpu())
    steps = 4 * 2.0 ** -8 + (2 * 2.0 ** -4 if eight else 0.0)
    error = (got - want).norm(dim=1) / want.norm(dim=1)
    print(f"largest {error.max():.4f}, mean {error.mean():.4f}, bound {steps:.4f}")
    assert (error <= steps).all()
