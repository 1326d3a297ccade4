"""HIP root-mean-square norm against the oracle in 64 bits.

Tolerances. With u the half step of the dtype (2^-8 bf16, 2^-11 f16, 2^-24 f32): a stored value
is off by u of itself. The fp32 arithmetic before it: a sum of n squares in chains of at most n / 64
and a tree is off by at most (n / 64 + 10) 2^-24 relative (all terms are positive), half of that in
its root, and four more roundings: below (n / 128 + 9) 2^-24 =: f of the value. The backward adds
the rounded h (u of each element, in xh and in the mean); every sum there has terms of both signs,
whose errors count relative to the sum of their magnitudes.
"""

from __future__ import annotations

import pytest
import torch

from oracle.native_providers import mx as o_mx
from oracle.native_providers import norm as o_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _inputs(shape, dtype, residual, seed=0, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * torch.rand(shape[:-1] + (1,), generator=g).exp()).to(dtype)
    r = torch.randn(shape, generator=g).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(shape[-1], generator=g)).to(wdtype or dtype)
    return x, r, w


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _within(got, want, bound, what):
    got = got.double().cpu()
    bad = (got - want).abs() > bound
    assert not bad.any(), (what, int(bad.sum()), (got - want)[bad][:4], bound.expand_as(want)[bad][:4])


def _fp32(n):
    return (n / 128 + 9) * 2.0 ** -24


SHAPES = [((1, 8), "bf16"), ((1, 7168), "bf16"), ((3, 1), "f32"), ((5, 33), "bf16"), ((7, 512), "f16"),
          ((9, 513), "f16"), ((4, 5, 1000), "bf16"), ((300, 2048), "bf16"), ((17, 2056), "f32"),
          ((6, 4096), "f32"), ((5, 8192), "bf16"), ((3, 8200), "f16"), ((2, 16384), "bf16"),
          ((2, 16385), "f32"), ((2, 20480), "bf16"), ((9000, 64), "bf16"), ((2100, 7168), "bf16"),
          ((0, 64), "bf16"), ((4, 0), "bf16")]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.mark.parametrize("shape, dtype", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward(hip_ops, shape, dtype, residual):
    dt = DTYPES[dtype]
    x, r, w = _inputs(shape, dt, residual)
    xd, rd, wd = _dev(x, r, w)
    out = hip_ops.rms_norm(xd, wd, 1e-5, residual=rd)
    y, h = o_norm.norm(x, w, 1e-5, r)
    if residual:
        assert out[1].shape == x.shape and out[1].dtype == dt
        _within(out[1], h, HALF[dt] * h.abs() + 1e-30, "sum")
        out = out[0]
    assert out.shape == x.shape and out.dtype == dt
    # f16 results below its normal range are off by half of its smallest step.
    _within(out, y, (HALF[dt] + 2 * _fp32(shape[-1])) * y.abs() + 2.0 ** -25, "y")


@pytest.mark.parametrize("shape, dtype", [s for s in SHAPES if s[0][-1]])
@pytest.mark.parametrize("residual", [False, True])
def test_backward(hip_ops, shape, dtype, residual):
    dt, n = DTYPES[dtype], shape[-1]
    x, r, w = _inputs(shape, dt, residual, seed=1)
    g = torch.Generator().manual_seed(2)
    gy = torch.randn(shape, generator=g).to(dt)
    gs = torch.randn(shape, generator=g).to(dt)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, r) if t is not None]
    out = hip_ops.rms_norm(leaves[0], leaves[1], 1e-5, residual=leaves[2] if residual else None)
    outs, grads = (list(out), [gy.to(DEV), gs.to(DEV)]) if residual else ([out], [gy.to(DEV)])
    got = torch.autograd.grad(outs, leaves, grads)
    wide = [t.double().requires_grad_() for t in (x, w, r) if t is not None]
    y, h = o_norm.norm(wide[0], wide[1], 1e-5, wide[2] if residual else None)
    want = torch.autograd.grad([y, h] if residual else [y], wide,
                               [gy.double(), gs.double()] if residual else [gy.double()])
    u, f = HALF[dt], _fp32(n)
    h = h.detach()
    rho = torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    xh, a = h * rho, gy.double() * w.double()
    hu = u if residual else 0.0  # the backward's h is rounded
    mean = (a * xh).abs().mean(-1, keepdim=True)
    inner = rho * xh.abs() * mean
    bound = u * want[0].abs() + (2 * hu + 8 * f) * inner + 8 * f * (rho * a.abs() + gs.double().abs()) + 2.0 ** -25
    _within(got[0], want[0], bound, "d_x")
    if residual:
        assert torch.equal(got[0], got[2])
    terms = (gy.double() * xh).reshape(-1, n).abs().sum(0)
    rows = terms.new_tensor(float(max(x.numel() // n, 1)))
    chain = (rows / 8 + 16) * 2.0 ** -24  # rows of a block, then of an eighth of the blocks
    _within(got[1], want[1], u * want[1].abs() + (hu + 4 * f + chain) * terms + 2.0 ** -25, "d_w")


def test_gradient_by_differences(hip_ops):
    """fp32: the directional derivative against central differences of the 64-bit forward."""
    x, r, w = _inputs((3, 96), torch.float32, True, seed=3)
    g = torch.Generator().manual_seed(4)
    gy, gs = torch.randn(3, 96, generator=g).double(), torch.randn(3, 96, generator=g).double()
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, r)]
    got = torch.autograd.grad(list(hip_ops.rms_norm(*leaves[:2], 1e-5, residual=leaves[2])), leaves,
                              [gy.float().to(DEV), gs.float().to(DEV)])

    def value(x, w, r):
        y, h = o_norm.norm(x, w, 1e-5, r)
        return ((y * gy.float().double()).sum() + (h * gs.float().double()).sum()).item()

    base = [t.double() for t in (x, w, r)]
    for i in range(3):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        plus, minus = ([b + s * eps * d if j == i else b for j, b in enumerate(base)] for s in (1, -1))
        slope = (value(*plus) - value(*minus)) / (2 * eps)
        assert abs((got[i].double().cpu() * d).sum().item() - slope) <= 1e-4 * max(1.0, abs(slope))


@pytest.mark.parametrize("which", ["y", "sum"])
def test_one_of_the_two_gradients(hip_ops, which):
    x, r, w = _inputs((6, 160), torch.bfloat16, True)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, r)]
    out = hip_ops.rms_norm(*leaves[:2], residual=leaves[2])
    g = torch.randn(6, 160, device=DEV).bfloat16()
    if which == "sum":
        dx, dr = torch.autograd.grad(out[1], [leaves[0], leaves[2]], g)
        assert torch.equal(dx, g) and torch.equal(dr, g)
    else:
        zero = torch.zeros_like(g)
        with_zero = torch.autograd.grad(list(hip_ops.rms_norm(*leaves[:2], residual=leaves[2])),
                                        leaves, [g, zero])
        alone = torch.autograd.grad(out[0], leaves, g)
        assert all(torch.equal(a, b) for a, b in zip(alone, with_zero))


def test_weight_of_another_dtype_strides_and_views(hip_ops):
    x, _, w = _inputs((40, 264), torch.bfloat16, False, wdtype=torch.float32)
    xd, wd = _dev(x, w)
    y = hip_ops.rms_norm(xd, wd)
    strided = torch.empty(264, 40, dtype=x.dtype, device=DEV).t().copy_(xd)
    assert torch.equal(hip_ops.rms_norm(strided, wd), y)
    store = torch.empty(40 * 264 + 3, dtype=x.dtype, device=DEV)
    shifted = store[3:].view(40, 264).copy_(xd)  # 6 bytes past a 16-byte boundary
    assert torch.equal(hip_ops.rms_norm(shifted, wd), y)
    wide = torch.empty(40, 528, dtype=x.dtype, device=DEV)[:, ::2].copy_(xd)
    assert torch.equal(hip_ops.rms_norm(wide, wd), y)


def test_nan_stays_in_its_row(hip_ops):
    x, _, w = _inputs((8, 2048), torch.bfloat16, False)
    clean = hip_ops.rms_norm(*_dev(x, w))
    bad = x.clone()
    bad[3, 77], bad[5, 0] = float("nan"), float("inf")
    y = hip_ops.rms_norm(*_dev(bad, w))
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[keep], clean[keep]) and y[3].isnan().all()
    assert y[5, 0].isnan() and (y[5, 1:] == 0).all()
    zero = hip_ops.rms_norm(torch.zeros(2, 64, device=DEV), torch.ones(64, device=DEV))
    assert torch.equal(zero, torch.zeros_like(zero))


MX_SHAPES = [((1, 32), "bf16"), ((3, 96), "f32"), ((1, 7168), "bf16"), ((33, 2048), "f16"),
             ((5, 2080), "bf16"), ((2, 3, 8192), "bf16"), ((2, 16416), "f32"), ((0, 64), "bf16"),
             ((2500, 2048), "bf16")]


@pytest.mark.parametrize("shape, dtype", MX_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rows_in_8_bits(hip_ops, shape, dtype, residual):
    """A code is the value's nearest, or, where the fp32 value lies within its error of a border
    between two, the other: the values stay within half a step and that error."""
    dt = DTYPES[dtype]
    x, r, w = _inputs(shape, dt, residual)
    xd, rd, wd = _dev(x, r, w)
    out = hip_ops.rms_norm_mx(xd, wd, 1e-5, residual=rd, with_y=True)
    plain = hip_ops.rms_norm(xd, wd, 1e-5, residual=rd)
    if residual:
        assert torch.equal(out.y, plain[0]) and torch.equal(out.sum, plain[1])
    else:
        assert torch.equal(out.y, plain) and out.sum is None
    codes, scales = out.rows.codes.cpu(), out.rows.scales.cpu()
    assert codes.shape == x.shape and scales.shape == (*x.shape[:-1], x.shape[-1] // 32)
    if x.numel() == 0:
        return
    y, _ = o_norm.norm(x, w, 1e-5, r)
    want = o_mx.quantize_mxfp8(y)
    f = 2 * _fp32(shape[-1])
    groups = y.unflatten(-1, (-1, 32))
    # A byte differs only where the largest magnitude lies within its error of a power of two.
    amax = groups.abs().amax(-1)
    edge = torch.minimum((amax / 2.0 ** torch.floor(torch.log2(amax)) - 1).abs(),
                         (amax / 2.0 ** torch.ceil(torch.log2(amax)) - 1).abs()) <= f
    assert ((scales == want.scales) | edge).all()
    got = o_mx.dequantize_mxfp8(out.rows.__class__(codes, scales), torch.float64)
    step = o_mx.power(scales.int() - 127).unsqueeze(-1)
    exponent = torch.log2((groups / step).abs().clamp(min=2.0 ** -6)).floor()
    half = 2.0 ** (exponent - 4) * step
    top = 448 * step
    bound = torch.maximum(half, groups.abs() - top) + 2 * f * groups.abs()
    _within(got, y, bound.flatten(-2), "rows")
    same = scales == want.scales
    differ = (codes.view(torch.uint8) != want.codes.view(torch.uint8)).unflatten(-1, (-1, 32))
    # Fewer than one in 500 values lies that near to a border (steps are 2^-4 of a value wide).
    assert differ[same].double().mean() <= 0.002 + 0.001 * (dtype == "f32")


def test_rows_without_y_and_refusals(hip_ops):
    x, _, w = _inputs((4, 64), torch.bfloat16, False)
    xd, wd = _dev(x, w)
    out = hip_ops.rms_norm_mx(xd, wd)
    assert out.y is None and out.sum is None
    with pytest.raises(RuntimeError, match="no gradient"):
        hip_ops.rms_norm_mx(xd.requires_grad_(), wd)
    with torch.no_grad():
        hip_ops.rms_norm_mx(xd, wd)


def test_graph_replay(hip_ops):
    x, r, w = _dev(*_inputs((512, 2048), torch.bfloat16, True))
    gy, gs = torch.randn_like(x), torch.randn_like(x)

    def step(x, r, w):
        leaves = [t.detach().requires_grad_() for t in (x, w, r)]
        out = hip_ops.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        rows = hip_ops.rms_norm_mx(x, w, residual=r).rows
        return [*(o.detach() for o in out), *torch.autograd.grad(list(out), leaves, [gy, gs]),
                rows.codes.view(torch.uint8), rows.scales]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, r, w)
    for seed in range(3):
        nx, nr, nw = _dev(*_inputs((512, 2048), torch.bfloat16, True, seed=seed + 10))
        x.copy_(nx), r.copy_(nr), w.copy_(nw)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step(x, r, w)))


@pytest.mark.parametrize("shape, dtype", MX_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("with_y", [False, True])
def test_rounded_rows_are_the_quantisers(hip_ops, shape, dtype, residual, with_y):
    """To the bit: the codes and scales of y as it is stored."""
    x, r, w = _dev(*_inputs(shape, DTYPES[dtype], residual))
    out = hip_ops.rms_norm_mx(x, w, 1e-5, residual=r, with_y=with_y, rounded=True)
    y = hip_ops.rms_norm(x, w, 1e-5, residual=r)
    if residual:
        assert torch.equal(out.sum, y[1])
        y = y[0]
    assert torch.equal(out.y, y) if with_y else out.y is None
    want = o_mx.quantize_mxfp8(y.cpu())
    assert torch.equal(out.rows.codes.cpu().view(torch.uint8), want.codes.view(torch.uint8))
    assert torch.equal(out.rows.scales.cpu(), want.scales)


@pytest.mark.parametrize("rows", [1, 33])
def test_weight_gradient_of_more_features_than_a_launch_has_threads_for(hip_ops, rows):
    """2^27 features: one block of 1024 threads per 32 of them, or a thread for each in every part, would be
    2^32 threads and more. Rows of +-1 have rstd 1, so with gradients of small whole numbers all is
    exact."""
    n = 1 << 27
    g = torch.Generator(device=DEV).manual_seed(rows)
    w = torch.ones(n, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    x = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
    gy = torch.empty_like(x)
    want = torch.zeros(n, device=DEV)
    for r in range(rows):
        x[r] = torch.randint(0, 2, (n,), generator=g, device=DEV, dtype=torch.int8) * 2 - 1
        gy[r] = torch.randint(-3, 4, (n,), generator=g, device=DEV, dtype=torch.int8)
        want += x[r].float() * gy[r].float()
    y = hip_ops.rms_norm(x, w, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(y.detach(), x))
    dw, = torch.autograd.grad(y, w, gy)
    assert torch.equal(dw, want.to(torch.bfloat16))  # at most 99: exact


def test_a_tensor_as_its_own_residual(hip_ops):
    """Both of its gradients add up: h = 2 x, so dx is twice the sum's gradient."""
    x, _, w = _inputs((6, 160), torch.float32, False)
    leaf, wd = x.to(DEV).requires_grad_(), w.to(DEV)
    y, h = hip_ops.rms_norm(leaf, wd, residual=leaf)
    y.sum().add(h.sum()).backward()  # gradients of stride zero
    other = (2 * x).to(DEV).requires_grad_()
    want = hip_ops.rms_norm(other, wd)
    dx, = torch.autograd.grad(want, other, torch.ones_like(want))
    assert torch.equal(y, want) and torch.equal(h, other)
    # 1 added within the kernel, or here: each rounds once, before the exact doubling.
    bound = 2.0 ** -23 * (dx.abs() + 1) * 2
    assert ((leaf.grad - 2 * (dx + 1)).abs() <= bound).all()
