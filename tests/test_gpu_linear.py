"""Dense products with an epilogue (``linear_act``, ``linear_residual``), counter-based
dropout and LoRA with it on the GPU, against the oracle's compositions in fp64.

Tolerances: with u half a step of the tensor's type (eps / 2, relative) and gamma(R) =
(R + 8) 2^-24 for an fp32 sum of R products, an output may be off by u |y| plus the sum's
gamma times the sum of the products' magnitudes; every operand rounded on the way adds
u times the magnitude of what it enters. The activations themselves are within 2^-20 of
what they are made of (hardware exp2 and reciprocal, a few steps of fp32)."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle.native_providers import dropout as o_dropout
from oracle.native_providers import linear as o_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
ACT_EPS = 2.0 ** -20
SLOPE = 1.13  # the largest |act'| and |act''| of SiLU and GELU are below this


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def gamma(r):
    return (r + 8) * 2.0 ** -24


def tiny(dtype):
    """Half the spacing of the smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def make(shape, seed, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - tol
    assert torch.isfinite(got).all() and (over <= 0).all(), \
        f"{what}: {over.max().item():.3e} over, {(over > 0).sum().item()} of {over.numel()}"


def wide(*tensors):
    return [None if t is None else t.detach().double() for t in tensors]


def check_act(ops, x, w, b, act, gated, backward=True):
    u, K = unit(x.dtype), x.shape[-1]
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = ops.linear_act(*leaves, activation_func=act, gated=gated)
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, activation_func=act, gated=gated), y)
    X, W, B = wide(x.reshape(-1, K), w, b)
    T, N = X.shape[0], y.shape[-1]
    a = X @ W.t()
    mag = X.abs() @ W.abs().t()
    if b is not None:
        a, mag = a + B, mag + B.abs()
    ea = gamma(K) * mag  # of the fp32 sums
    f = act or (lambda v: v)
    if gated:
        p, q, ep, eq = a[:, :N], a[:, N:], ea[:, :N], ea[:, N:]
    else:
        p, q, ep, eq = a, torch.ones_like(a), ea, torch.zeros_like(ea)
    p = p.detach().requires_grad_()
    fp = f(p)
    slope = torch.autograd.grad(fp.sum(), p)[0] if act else torch.ones_like(p)
    p, fp = p.detach(), fp.detach()
    want = fp * q
    fa = ACT_EPS * (1 + p.abs()) if act else 0.0  # of the activation and its slope
    tol = u * want.abs() + 1.01 * (q.abs() * (SLOPE * ep + fa) + (fp.abs() + 1) * eq) + tiny(x.dtype)
    within(y.reshape(T, N), want, tol, "y")
    if not backward:
        return
    dy = make(tuple(y.shape), 77, x.dtype)
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, wanted, dy)
    G = dy.reshape(T, N).double()
    second = SLOPE if act else 0.0
    dp = G * q * slope
    edp = G.abs() * (q.abs() * (second * ep + fa) + 1.2 * eq)
    if gated:
        dq, edq = G * fp, G.abs() * (SLOPE * ep + fa)
        da, eda = torch.cat([dp, dq], 1), torch.cat([edp, edq], 1)
    else:
        da, eda = dp, edp
    ebias = eda + 2.0 ** -22 * da.abs()
    # 16 bits: rounded before the products.
    eda = 1.01 * ebias + u * da.abs() + tiny(x.dtype)
    R = da.shape[1]
    dx, dw = da @ W, da.t() @ X
    within(grads[0].reshape(T, K), dx,
           u * dx.abs() + 1.01 * (eda @ W.abs() + gamma(R) * (da.abs() @ W.abs())) + tiny(x.dtype), "dx")
    within(grads[1], dw,
           u * dw.abs() + 1.01 * (eda.t() @ X.abs() + gamma(T) * (da.abs().t() @ X.abs())) + tiny(x.dtype),
           "dw")
    if b is not None:
        db = da.sum(0)
        within(grads[2], db, unit(b.dtype) * db.abs() + 1.01 * (ebias.sum(0) + gamma(T) * da.abs().sum(0)) +
               tiny(b.dtype), "db")


def check_residual(ops, x, w, b, r, s, p=0.0, key=None, backward=True):
    u, K = unit(x.dtype), x.shape[-1]
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, r, s)]
    y = ops.linear_residual(*leaves, dropout_p=p, dropout_key=key)
    with torch.no_grad():
        assert torch.equal(ops.linear_residual(x, w, b, r, s, dropout_p=p, dropout_key=key), y)
    X, W, B, Rs, S = wide(x.reshape(-1, K), w, b, r, s)
    T, N = X.shape[0], w.shape[0]
    S = torch.ones(T, 1, dtype=torch.float64, device=DEV) if s is None else S.reshape(T, 1)
    f = torch.ones(T, N, dtype=torch.float64, device=DEV)
    if p:
        f = o_dropout.factors(T, N, p, key.cpu()).to(DEV)
    a, mag = X @ W.t(), X.abs() @ W.abs().t()
    if b is not None:
        a, mag = a + B, mag + B.abs()
    want = S * f * a
    total = want if r is None else want + Rs.reshape(T, N)
    tol = (u * total.abs() + 1.01 * (S * f).abs() * (gamma(K) * mag + 2.0 ** -22 * a.abs()) +
           2.0 ** -23 * total.abs() + tiny(x.dtype))
    within(y.reshape(T, N), total, tol, "y")
    if not backward:
        return
    dy = make(tuple(y.shape), 78, x.dtype)
    wanted = [t for t in leaves if t is not None]
    names = [n for n, t in zip("xwbrs", leaves) if t is not None]
    grads = dict(zip(names, torch.autograd.grad(y, wanted, dy)))
    G = dy.reshape(T, N).double()
    g = G * f
    gw, gwm = g @ W, g.abs() @ W.abs()
    dx = S * gw
    within(grads["x"].reshape(T, K), dx,
           u * dx.abs() + 1.01 * (S.abs() * (gamma(N) * gwm + 2.0 ** -22 * gw.abs())) + tiny(x.dtype), "dx")
    # The rows enter the weight's gradient times their scale, rounded where there is one.
    xs = S * X
    exs = 0.0 if s is None else u * xs.abs() + tiny(x.dtype)
    dw = g.t() @ xs
    inner = g.abs().t() @ (xs.abs() * 1.01)
    within(grads["w"], dw, u * dw.abs() + 1.01 * (g.abs().t() @ (exs + 0 * xs) +
           (gamma(T) + 2.0 ** -22) * inner) + tiny(x.dtype), "dw")
    if r is not None:
        assert torch.equal(grads["r"], dy)
    if b is not None:
        db = (S * g).sum(0)
        within(grads["b"], db, unit(b.dtype) * db.abs() + 1.01 * (gamma(T) + 2.0 ** -22) *
               (S * g).abs().sum(0) + tiny(b.dtype), "db")
    if s is not None:
        ds, m = (X * gw).sum(1), (X.abs() * gwm).sum(1)
        if b is not None:
            ds, m = ds + g @ B, m + g.abs() @ B.abs()
        within(grads["s"].reshape(-1), ds, unit(s.dtype) * ds.abs() +
               1.01 * (gamma(N) + gamma(K) + 2.0 ** -22) * m + tiny(s.dtype), "ds")


# One token, odd sizes, sizes around tiles of 64, 128 and 256, reductions that are no
# multiple of 64, long reductions over few outputs, few rows over many columns.
SIZES = [(1, 64, 16), (1, 1024, 264), (3, 72, 40), (5, 33, 17), (17, 4096, 64), (64, 136, 520),
         (65, 200, 72), (130, 515, 257), (257, 1032, 264), (300, 64, 1032), (512, 512, 512),
         (1030, 320, 136), (2500, 40, 24), (777, 2048, 384)]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("T, K, N", SIZES)
@pytest.mark.parametrize("act, gated, bias", [(F.silu, True, False), (F.gelu, True, True),
                                              (F.gelu, False, True), (None, False, True)])
def test_linear_act(hip_ops, T, K, N, dtype, act, gated, bias):
    x, w = make((T, K), 1, dtype), make((2 * N if gated else N, K), 2, dtype, K ** -0.5)
    b = make((w.shape[0],), 3, FP if dtype == HF else dtype, 0.3) if bias else None
    check_act(hip_ops, x, w, b, act, gated)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("T, K, N", SIZES)
@pytest.mark.parametrize("bias, res, scale, p", [(False, True, False, 0.0), (True, True, True, 0.0),
                                                 (True, False, True, 0.3), (False, True, False, 0.5)])
def test_linear_residual(hip_ops, T, K, N, dtype, bias, res, scale, p):
    x, w = make((T, K), 4, dtype), make((N, K), 5, dtype, K ** -0.5)
    b = make((N,), 6, dtype, 0.3) if bias else None
    r = make((T, N), 7, dtype) if res else None
    s = make((T, 1), 8, FP if dtype == BF else dtype) if scale else None
    key = torch.tensor([T * 12345678901, -K], device=DEV) if p else None
    check_residual(hip_ops, x, w, b, r, s, p, key)


# Enough tiles of 256 for the largest kernels: in the forward, in the gradient of x and
# in the gradient of the weight.
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T, K, N", [(3850, 136, 3400), (3850, 3400, 136), (140, 3400, 3848)])
def test_largest_tiles(hip_ops, T, K, N, dtype):
    x, w, b = make((T, K), 1, dtype), make((N, K), 2, dtype, K ** -0.5), make((N,), 3, dtype, 0.3)
    check_act(hip_ops, x, w, b, F.gelu, False)
    check_act(hip_ops, x, make((N + N % 16, K), 4, dtype, K ** -0.5), None, F.silu, True)
    key = torch.tensor([K, N], device=DEV)
    check_residual(hip_ops, x, w, b, make((T, N), 5, dtype), make((T, 1), 6, dtype), 0.2, key)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_empty_sizes(hip_ops, dtype):
    for T, K, N in ((0, 16, 8), (4, 0, 8), (4, 16, 0), (0, 0, 0)):
        x, w = make((T, K), 1, dtype), make((2 * N, K), 2, dtype)
        b, r, s = make((2 * N,), 3, dtype), make((T, 2 * N), 4, dtype), make((T,), 5, dtype)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = hip_ops.linear_act(x, w, b, activation_func=F.silu, gated=True)
        assert y.shape == (T, N)
        if T and N:  # K = 0: the bias alone
            torch.testing.assert_close(y, (F.silu(b.float()[:N]) * b.float()[N:]).to(dtype).expand(T, N))
        for t, g in zip(leaves, torch.autograd.grad(y, leaves, torch.ones_like(y))):
            assert g.shape == t.shape and (T and N or not g.any())
        more = leaves + [t.requires_grad_() for t in (r, s)]
        y = hip_ops.linear_residual(x, w, b, r, s)
        assert y.shape == (T, 2 * N)
        for t, g in zip(more, torch.autograd.grad(y, more, torch.ones_like(y))):
            assert g.shape == t.shape


@pytest.mark.parametrize("T, K, N", [(0, 2048, 2048), (0, 2049, 2051), (2048, 0, 2056), (5, 2049, 2051)])
def test_reductions_of_nearly_nothing_over_many_tiles(hip_ops, T, K, N):
    # 256 and more tiles of 128 x 128, each with at most five products to an element.
    x, w = make((T, K), 1, BF), make((2 * N, K), 2, BF)
    if T and K:
        check_act(hip_ops, x, w, None, F.silu, True)
        return
    x.requires_grad_()
    w.requires_grad_()
    y = hip_ops.linear_act(x, w, activation_func=F.silu, gated=True)
    assert y.shape == (T, N) and not y.any()
    for t, g in zip((x, w), torch.autograd.grad(y, (x, w), torch.ones_like(y))):
        assert g.shape == t.shape and not g.any()
    y = hip_ops.linear_residual(x, w)
    assert y.shape == (T, 2 * N) and not y.any()
    for t, g in zip((x, w), torch.autograd.grad(y, (x, w), torch.ones_like(y))):
        assert g.shape == t.shape and not g.any()


def test_strides_alignment_and_dimensions(hip_ops):
    """Transposed, sliced, expanded and unaligned operands and leading dimensions give the
    contiguous, aligned call's values."""
    x, w, b = make((6, 40, 128), 1, BF), make((128, 128), 2, BF, 0.1), make((128,), 3, BF)
    r, s = make((6, 40, 128), 4, BF), make((6, 40, 1), 5, BF)
    want = hip_ops.linear_residual(x, w, b, r, s)
    act = hip_ops.linear_act(x, w, b, activation_func=F.gelu, gated=True)
    assert want.shape == (6, 40, 128) and act.shape == (6, 40, 64)

    def moved(t, how):
        if how == "transposed":
            return t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t
        if how == "sliced":
            return torch.cat([t, t], -1)[..., :t.shape[-1]]
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:]
        return flat.copy_(t.reshape(-1)).view(t.shape)

    for how in ("transposed", "sliced", "unaligned"):
        ops = [moved(t, how) for t in (x, w, b, r, s)]
        got = hip_ops.linear_residual(*ops)
        got_act = hip_ops.linear_act(*ops[:3], activation_func=F.gelu, gated=True)
        if how == "unaligned":  # other kernels, another order of the sums
            torch.testing.assert_close(got, want, rtol=2 ** -7, atol=1e-3)
            torch.testing.assert_close(got_act, act, rtol=2 ** -7, atol=1e-3)
        else:
            assert torch.equal(got, want) and torch.equal(got_act, act)
    one = hip_ops.linear_act(x[0, 0], w, b)
    assert one.shape == (128,)
    torch.testing.assert_close(one, hip_ops.linear_act(x, w, b)[0, 0], rtol=2 ** -7, atol=1e-3)
    wide_row = x[:1, :1].expand(6, 40, 128)
    assert torch.equal(hip_ops.linear_act(wide_row, w, b),
                       hip_ops.linear_act(wide_row.contiguous(), w, b))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T, K, N", [(20, 72, 40), (300, 200, 264), (70, 33, 31), (300, 1032, 72)])
def test_not_finite_values_stay_in_their_rows(hip_ops, T, K, N, dtype):
    """NaN and infinities of one token, or of one feature's weights, reach nothing else:
    tiles read past the ends of rows and reductions, and what they read counts for nothing."""
    x, w = make((T, K), 1, dtype), make((2 * N, K), 2, dtype, 0.1)
    r, s = make((T, 2 * N), 3, dtype), make((T, 1), 4, dtype)
    bad_x, bad_w = x.clone(), w.clone()
    bad_x[T // 2], bad_x[-1] = float("inf"), float("nan")
    bad_w[3], bad_w[-1] = float("nan"), float("inf")
    rows = torch.ones(T, dtype=torch.bool, device=DEV)
    rows[T // 2] = rows[-1] = False
    cols = torch.ones(2 * N, dtype=torch.bool, device=DEV)
    cols[3] = cols[-1] = False
    clean, dirty = hip_ops.linear_residual(x, w, None, r, s), hip_ops.linear_residual(bad_x, bad_w, None, r, s)
    assert torch.equal(dirty[rows][:, cols], clean[rows][:, cols])
    assert not torch.isfinite(dirty[~rows]).any() and not torch.isfinite(dirty[:, ~cols]).any()
    # Gradients: a row of dy that is NaN reaches its own row of dx alone.
    dy = make((T, 2 * N), 5, dtype)
    bad = dy.clone()
    bad[T // 2] = float("nan")
    leaf = x.clone().requires_grad_()
    good, = torch.autograd.grad(hip_ops.linear_act(leaf, w), leaf, dy)
    got, = torch.autograd.grad(hip_ops.linear_act(leaf, w), leaf, bad)
    keep = torch.arange(T, device=DEV) != T // 2
    assert torch.equal(got[keep], good[keep]) and got[~keep].isnan().all()


def test_gradients_by_differences(hip_ops):
    """fp32: the derivative along a direction against the difference of two calls. With a
    step of 2^-6 along unit-sized directions the difference's cubic term is below 1e-3 of
    the derivative's scale, and the fp32 sums add below 1e-3."""
    T, K, N = 37, 48, 40
    x, w, b = make((T, K), 1, FP), make((2 * N, K), 2, FP, K ** -0.5), make((2 * N,), 3, FP)
    w2, b2 = make((24, N), 4, FP, N ** -0.5), make((24,), 5, FP)
    r, s, dy = make((T, 24), 6, FP), make((T, 1), 7, FP), make((T, 24), 8, FP)
    key = torch.tensor([11, 12], device=DEV)
    leaves = [x, w, b, w2, b2, r, s]

    def loss(v):
        h = hip_ops.linear_act(v[0], v[1], v[2], activation_func=F.silu, gated=True)
        y = hip_ops.linear_residual(h, *v[3:], dropout_p=0.25, dropout_key=key)
        return y, (y.double() * dy.double()).sum()

    for t in leaves:
        t.requires_grad_()
    grads = torch.autograd.grad(loss(leaves)[0], leaves, dy)
    for i, t in enumerate(leaves):
        d = make(tuple(t.shape), 20 + i, FP)
        d /= d.norm()
        step = 2.0 ** -6
        with torch.no_grad():
            up = loss([v + step * d if j == i else v for j, v in enumerate(leaves)])[1]
            down = loss([v - step * d if j == i else v for j, v in enumerate(leaves)])[1]
        diff, want = ((up - down) / (2 * step)).item(), (grads[i].double() * d.double()).sum().item()
        scale = grads[i].double().norm().item()
        assert abs(diff - want) <= 4e-3 * scale + 1e-3, (i, diff, want, scale)


def test_parts_of_the_gradient(hip_ops):
    """Each gradient asked for alone is the one of the full backward."""
    T, K, N = 140, 128, 72
    x, w, b = make((T, K), 1, BF), make((N, K), 2, BF, 0.1), make((N,), 3, BF)
    r, s, dy = make((T, N), 4, BF), make((T, 1), 5, BF), make((T, N), 6, BF)
    key = torch.tensor([1, 2], device=DEV)
    full = [t.clone().requires_grad_() for t in (x, w, b, r, s)]
    y = hip_ops.linear_residual(*full, dropout_p=0.1, dropout_key=key)
    want = torch.autograd.grad(y, full, dy)
    for i in range(5):
        part = [t.clone() for t in (x, w, b, r, s)]
        part[i].requires_grad_()
        y = hip_ops.linear_residual(*part, dropout_p=0.1, dropout_key=key)
        got, = torch.autograd.grad(y, part[i], dy)
        assert torch.equal(got, want[i]), i
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        g, = torch.autograd.grad(hip_ops.linear_act(full[0], w), full[0], dy, create_graph=True)
        torch.autograd.grad(g.sum(), full[0])


def test_offsets_past_32_bits(hip_ops):
    """Tensors of more than 2^31 elements and 4 GiB: the last rows of the output and of
    the gradients are those of a call on these rows alone, and the weight's gradient, whose
    operand no 32-bit offset spans, is the sum over slices of the rows."""
    T, K, N, last = 72000, 64, 32768, 200
    x, w = make((T, K), 1, BF), make((N, K), 2, BF, 0.1)
    g = torch.Generator(device=DEV).manual_seed(3)
    dy = torch.empty((T, N), dtype=BF, device=DEV).normal_(generator=g)
    s = torch.rand((T, 1), generator=g, device=DEV).to(BF)
    leaves = [t.requires_grad_() for t in (x, w, s)]
    y = hip_ops.linear_residual(x, w, None, dy, s)
    dx, dw, ds = torch.autograd.grad(y, leaves, dy)
    part = [x[-last:].detach().requires_grad_(), w, s[-last:].detach().requires_grad_()]
    yp = hip_ops.linear_residual(part[0], w, None, dy[-last:], part[2])
    dxp, dsp = torch.autograd.grad(yp, [part[0], part[2]], dy[-last:])
    # The same roundings to 16 bits at the end of fp32 sums of at most N products.
    for a, b in ((y[-last:], yp), (dx[-last:], dxp), (ds[-last:], dsp)):
        assert (a.double() - b.double()).norm() <= 2 * unit(BF) * b.double().norm()
    want = torch.zeros((N, K), dtype=torch.float64, device=DEV)
    for at in range(0, T, 9000):
        rows = (s[at:at + 9000].float() * x[at:at + 9000].float()).to(BF).detach()
        want += (dy[at:at + 9000].float().t() @ rows.float()).double()
    assert (dw.double() - want).norm() <= 2 * unit(BF) * want.norm()


# ---------------------------------------------------------------------------
# Dropout
# ---------------------------------------------------------------------------
def test_few_rows_with_a_weight_past_32_bits(hip_ops):
    """Columns of a weight of more than 4 GiB against a call on their rows of it alone."""
    T, K, N = 3, 32768, 69640
    x = make((T, K), 1, BF)
    g = torch.Generator(device=DEV).manual_seed(4)
    w = torch.empty((N, K), dtype=BF, device=DEV).normal_(0.0, 0.01, generator=g)
    assert w.numel() * 2 > 1 << 32
    y = hip_ops.linear_residual(x, w)
    for at in (0, 65528, N - 200):
        part = hip_ops.linear_residual(x, w[at:at + 200])
        want = part.double()
        # Roundings to 16 bits at the end of fp32 sums of K products.
        assert (y[:, at:at + 200].double() - want).norm() <= 2 * unit(BF) * want.norm()
    exact = x.double() @ w[-200:].double().t()
    assert (y[:, -200:].double() - exact).norm() <= 2 * unit(BF) * exact.norm()


def test_fp32_rows_further_apart_than_32_bits(hip_ops):
    # 64 rows of a tile span more than 4 GiB; whole numbers, so that every sum is exact.
    K = (1 << 24) + 1001
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randint(-1, 2, (2, K), generator=g, device=DEV).float().requires_grad_()
    w = torch.randint(-1, 2, (3, K), generator=g, device=DEV).float().requires_grad_()
    dy = torch.tensor([[1.0, -2.0, 3.0], [0.0, 4.0, -5.0]], device=DEV)
    y = hip_ops.linear_residual(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        for i in range(2):
            for j in range(3):
                assert y[i, j].item() == (x[i].double() * w[j].double()).sum().item()
            assert torch.equal(dx[i], sum(dy[i, j] * w[j] for j in range(3)))
        for j in range(3):
            assert torch.equal(dw[j], sum(dy[i, j] * x[i] for i in range(2)))


def test_dropout_past_32_bits(hip_ops):
    rows, cols = 1 << 20, 4104
    x = torch.ones((rows, cols), dtype=BF, device=DEV)
    key = torch.tensor([77, 78], device=DEV)
    y = hip_ops.dropout(x, 0.5, key)
    f = o_dropout.factors(3, cols, 0.5, key.cpu(), rows - 3)
    assert torch.equal(y[-3:].double().cpu(), f)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (9,), (130, 1024), (2, 4104), (3, 5, 13),
                                   (70000, 3), (2, 3, 4, 2056)])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0, 1e-7])
def test_dropout(hip_ops, shape, dtype, p):
    x = make(shape, 1, dtype).requires_grad_()
    dy = make(shape, 2, dtype)
    key = torch.tensor([0x7FFF00FF12345678, -0x1234567800000001], device=DEV)
    y = hip_ops.dropout(x, p, key)
    dx, = torch.autograd.grad(y, x, dy)
    # The product with the fp32 factor rounded once: the oracle's, bit for bit.
    assert torch.equal(y.cpu(), o_dropout.dropout(x.detach().cpu(), p, key.cpu()))
    assert torch.equal(dx.cpu(), o_dropout.dropout(dy.cpu(), p, key.cpu()))


def test_dropout_of_other_layouts_and_values(hip_ops):
    key = torch.tensor([5, 6], device=DEV)
    x = make((24, 96), 1, BF)
    want = hip_ops.dropout(x, 0.4, key)
    assert torch.equal(hip_ops.dropout(x.t().contiguous().t(), 0.4, key), want)
    assert torch.equal(hip_ops.dropout(torch.cat([x, x], 1)[:, :96], 0.4, key), want)
    flat = torch.empty(x.numel() + 1, dtype=BF, device=DEV)[1:].view(24, 96).copy_(x)
    assert torch.equal(hip_ops.dropout(flat, 0.4, key), want)
    assert hip_ops.dropout(x, 0.0, None) is x
    assert hip_ops.dropout(x[:0], 0.4, key).shape == (0, 96)
    assert hip_ops.dropout(x[:, :0], 0.4, key).shape == (24, 0)
    bad = torch.full_like(x, float("inf"))
    bad[::2] = float("nan")
    got = hip_ops.dropout(bad, 0.4, key)
    kept = o_dropout.factors(24, 96, 0.4, key.cpu()).to(DEV) > 0
    assert torch.equal(got != 0, kept) and not got[~kept].any() and not torch.isfinite(got[kept]).any()
    # The key changes the mask; changing it in place between the passes is noticed.
    assert not torch.equal(hip_ops.dropout(x, 0.4, key + 1), want)
    leaf = x.clone().requires_grad_()
    y = hip_ops.dropout(leaf, 0.4, key)
    key += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_is_differentiable_twice(hip_ops):
    key = torch.tensor([5, 6], device=DEV)
    x = make((8, 16), 1, FP).requires_grad_()
    g, = torch.autograd.grad(hip_ops.dropout(x, 0.5, key).square().sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), x)
    f = o_dropout.factors(8, 16, 0.5, key.cpu()).to(DEV)
    torch.testing.assert_close(h.double(), 2 * f * f)


# ---------------------------------------------------------------------------
# LoRA with dropout
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("counts, K, N, r", [([5], 64, 32, 4), ([0, 37, 0, 200, 1], 136, 264, 16),
                                             ([70, 0, 130], 512, 128, 24), ([300, 41], 200, 72, 64),
                                             ([0, 0], 64, 64, 8), ([1] * 40, 768, 96, 32)])
def test_lora_residual_with_dropout(hip_ops, counts, K, N, r, dtype):
    M, E, s, p = sum(counts), len(counts), 2.0, 0.3
    base, x = make((M, N), 1, dtype), make((M, K), 2, dtype)
    a, b = make((E, K, r), 3, FP, K ** -0.5), make((E, r, N), 4, FP, 0.2)
    dy = make((M, N), 5, dtype)
    key = torch.tensor([M * 987654321, K], device=DEV)
    leaves = [t.requires_grad_() for t in (base, x, a, b)]
    y = hip_ops.lora_residual(*leaves, torch.tensor(counts, device=DEV), s, dropout_p=p,
                              dropout_key=key)
    grads = torch.autograd.grad(y, leaves, dy)
    f = o_dropout.factors(M, K, p, key.cpu()).to(DEV)
    Bs, X, A, B, G = wide(base, x, a, b, dy)
    u, at = unit(dtype), 0
    assert torch.equal(grads[0], dy)
    for e, n in enumerate(counts):
        part = slice(at, at + n)
        at += n
        xs, g = X[part] * f[part], s * G[part]
        h, hm = xs @ A[e], xs.abs() @ A[e].abs()
        d, dm = h @ B[e], hm @ B[e].abs()
        want = Bs[part] + s * d
        # The product, its multiple and the sum are each rounded to 16 bits.
        tol = u * (want.abs() + 2.02 * s * d.abs()) + 1.01 * s * (gamma(K) + gamma(r)) * dm
        within(y[part], want, tol + tiny(dtype), "y")
        dh, dhm = g @ B[e].t(), g.abs() @ B[e].abs().t()
        dx, dxm = (dh @ A[e].t()) * f[part], (dhm @ A[e].abs().t()) * f[part]
        within(grads[1][part], dx, u * dx.abs() + 1.01 * (gamma(N) + gamma(r)) * dxm + tiny(dtype), "dx")
        within(grads[2][e], xs.t() @ dh, 1.01 * (gamma(N) + gamma(n)) * (xs.abs().t() @ dhm), "da")
        within(grads[3][e], h.t() @ g, 1.01 * (gamma(K) + gamma(n)) * (hm.t() @ g.abs()), "db")


def test_lora_dropout_drops_what_is_not_finite(hip_ops):
    M, K, N, r, p = 50, 64, 32, 8, 0.5
    key = torch.tensor([8, 9], device=DEV)
    f = o_dropout.factors(M, K, p, key.cpu()).to(DEV)
    x = torch.where(f > 0, make((M, K), 1, BF).double(), torch.full((), float("nan"), device=DEV).double())
    a, b = make((1, K, r), 2, FP), make((1, r, N), 3, FP)
    leaves = [t.requires_grad_() for t in (x.to(BF), a, b)]
    y = hip_ops.lora_residual(make((M, N), 4, BF), *leaves, torch.tensor([M], device=DEV), 1.0,
                              dropout_p=p, dropout_key=key)
    for t in (y, *torch.autograd.grad(y.float().sum(), leaves)):
        assert torch.isfinite(t).all()


# ---------------------------------------------------------------------------
# Streams, graphs and the run of them together
# ---------------------------------------------------------------------------
def test_two_streams_at_once(hip_ops):
    """Calls on two streams share nothing (each has a workspace of its own)."""
    x, w = make((17, 4096), 1, BF), make((64, 4096), 2, BF, 0.02)
    x2 = make((17, 4096), 3, BF)
    want = [hip_ops.linear_residual(v, w) for v in (x, x2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = [[], []]
    for _ in range(20):
        for i, (st, v) in enumerate(zip(streams, (x, x2))):
            with torch.cuda.stream(st):
                out[i].append(hip_ops.linear_residual(v, w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in out[i])


def test_captured_and_replayed(hip_ops):
    """A training step of both products with dropout in a graph: each replay, with eager
    work in between, gives the eager results of the inputs and key it finds."""
    T, K, Fi = 96, 128, 72
    w1, w2 = make((2 * Fi, K), 1, BF, 0.1), make((K, Fi), 2, BF, 0.1)
    b1, b2 = make((2 * Fi,), 3, BF), make((K,), 4, BF)
    x, s, dy = make((T, K), 5, BF), make((T, 1), 6, BF), make((T, K), 7, BF)
    key = torch.tensor([1, 2], device=DEV)

    def step(x, key):
        leaves = [t.detach().requires_grad_() for t in (x, w1, b1, w2, b2, s)]
        h = hip_ops.linear_act(*leaves[:3], activation_func=F.silu, gated=True)
        y = hip_ops.linear_residual(h, leaves[3], leaves[4], leaves[0], leaves[5], dropout_p=0.2,
                                    dropout_key=key)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, key)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x, key)
    for i in range(4):
        x.copy_(make((T, K), 30 + i, BF))
        key.copy_(torch.tensor([i, 99 - i]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step(x.clone(), key.clone())):
            assert torch.equal(a, b), i


def test_shared_expert_and_adapters_in_the_layer(process_ops):
    """A layer with a gated shared expert and experts with adapters under dropout: forward
    and gradients against the same layer composed of the oracle's operators on the CPU in
    fp64, from the keys that the generator gave."""
    from torchturbo_amd.dispatch import OpPolicy, ops
    from torchturbo_amd.moe import (CounterDropout, GroupedMLP, GroupedMLPLoRA, MoEConfig, MoELayer,
                                    MoESubmodules, ModuleSpec, SharedExpertMLP)
    from torchturbo_amd.runtime import CudaRuntime

    process_ops(CudaRuntime(), OpPolicy.CUSTOM)
    T, H, E, Fi, Fs = 200, 128, 8, 64, 96
    cfg = MoEConfig(hidden_size=H, num_moe_experts=E, moe_ffn_hidden_size=Fi, moe_router_topk=2,
                    gated_linear_unit=True, activation_func=F.silu, params_dtype=BF,
                    moe_shared_expert_intermediate_size=Fs)
    torch.manual_seed(0)
    with torch.device(DEV):
        layer = MoELayer(cfg, None, MoESubmodules(experts=ModuleSpec(module=GroupedMLP)))
        layer.shared_expert = SharedExpertMLP(cfg, bias=True, dropout=0.25)
        layer.shared_expert_gate = torch.nn.Linear(H, 1, bias=False, dtype=BF)
    with torch.no_grad():
        for i, prm in enumerate(layer.parameters()):
            prm.copy_(make(tuple(prm.shape), 50 + i, BF, 0.1))
    layer.experts = GroupedMLPLoRA(layer.experts, "default", r=4, lora_alpha=8, lora_dropout=0.3,
                                   counter_dropout=True)
    with torch.no_grad():
        for i, name in enumerate(("lora_A", "lora_B", "lora_A2", "lora_B2")):
            prm = getattr(layer.experts, name)["default"].weight
            prm.copy_(make(tuple(prm.shape), 80 + i, FP, 0.1))
    x, logits, dy = make((T, H), 90, BF), make((T, E), 91, FP), make((T, H), 92, BF)
    leaf = x.clone().requires_grad_()
    torch.manual_seed(123)
    out = layer.forward_with_logits(leaf, logits)
    names = [n for n, prm in layer.named_parameters() if "router" not in n]
    params = [dict(layer.named_parameters())[n] for n in names]
    grads = dict(zip(["x"] + names, torch.autograd.grad(out, [leaf] + params, dy)))
    torch.manual_seed(123)
    k1, k2, k3 = (CounterDropout.draw_key(DEV).cpu() for _ in range(3))

    # The same in fp64 on the CPU.
    X = x.double().cpu().requires_grad_()
    P = {n: prm.detach().double().cpu().requires_grad_() for n, prm in zip(names, params)}
    top = torch.topk(logits.double().cpu(), 2, dim=1)
    probs = torch.softmax(top.values, 1)
    order = [(e, t, j) for e in range(E) for t in range(T) for j in range(2) if top.indices[t, j] == e]
    tok = torch.tensor([t for _, t, _ in order])
    pr = torch.stack([probs[t, j] for _, t, j in order])
    loads = [sum(1 for e, _, _ in order if e == i) for i in range(E)]
    rows = X[tok]

    def grouped(v, w):
        return torch.cat([p @ w[e] for e, p in enumerate(v.split(loads))])

    def adapted(v, w, a, b, key):
        d = v * o_dropout.factors(*v.shape, 0.3, key)
        return grouped(v, w) + 2.0 * grouped(grouped(d, P[f"experts.{a}.default.weight"]),
                                             P[f"experts.{b}.default.weight"])

    h = adapted(rows, P["experts.base_layer.weight1"].view(E, H, 2 * Fi), "lora_A", "lora_B", k1)
    act = F.silu(h[:, :Fi]) * h[:, Fi:] * pr[:, None]
    y = adapted(act, P["experts.base_layer.weight2"].view(E, Fi, H), "lora_A2", "lora_B2", k2)
    total = torch.zeros_like(X).index_add(0, tok, y)
    sh = o_linear.linear_act(X, P["shared_expert.weight1"], P["shared_expert.bias1"],
                             activation_func=F.silu, gated=True)
    gate = torch.sigmoid(X @ P["shared_expert_gate.weight"].t())
    want = o_linear.linear_residual(sh, P["shared_expert.weight2"], P["shared_expert.bias2"], total,
                                    gate, dropout_p=0.25, dropout_key=k3)
    wg = dict(zip(["x"] + names, torch.autograd.grad(want, [X] + list(P.values()), dy.double().cpu())))

    # About a dozen 16-bit roundings lie on the longest path (u = 2^-8 each, adding up as
    # squares for sums of many terms): 4 u of the result's norm.
    def near(a, b, what):
        d = (a.double().cpu() - b).norm() / b.norm()
        assert d < 4 * 2.0 ** -8, (what, d)

    near(out, want.detach(), "out")
    for n in wg:
        near(grads[n], wg[n], n)


# ---------------------------------------------------------------------------
# Ends of tiles
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("K", [40, 72, 200, 1032])
def test_scale_gradient_counts_its_columns_alone(hip_ops, K):
    """Finite operands with a finite gradient: a tile's columns past K hold sums of one row of
    dy with the weight's next row, here past the largest fp32 number, and count for nothing."""
    T, N = 70, 48
    x, w = make((T, K), 1, BF), make((N, K), 2, BF)
    s, dy = make((T, 1), 3, BF), make((T, N), 4, BF)
    w[0], w[1, :32], dy[5, 0], dy[5, 1] = 0.0, 4.0, 3e38, 0.0
    leaf = s.clone().requires_grad_()
    ds, = torch.autograd.grad(hip_ops.linear_residual(x, w, None, None, leaf), leaf, dy)
    X, W, G = wide(x, w, dy)
    want, mag = (X * (G @ W)).sum(1), (X.abs() * (G.abs() @ W.abs())).sum(1)
    assert want.abs().max() < 1e6
    within(ds.reshape(-1), want, unit(BF) * want.abs() +
           1.01 * (gamma(N) + gamma(K) + 2.0 ** -22) * mag, "ds")


# ---------------------------------------------------------------------------
# Sizes that take the wide tiles
# ---------------------------------------------------------------------------
KERNELS = "F32 ROWS T64 T128 T256x128 T256 ODD64 ODD128".split()  # TT_LINEAR_KERNEL_...
OPS = {"act": 0, "gated": 1, "residual": 2}


def plan(op, which, T, K, N, dtype=BF, aligned=True):
    """Kernel / parts of a product: which 0 the forward, 1 the gradient of x, 2 of w."""
    from torchturbo_amd import _lib as L

    v = L.load().tt_linear_plan(OPS[op], which, L.dtype_code(dtype), T, K, N, int(aligned))
    return f"{KERNELS[v % 256]}/{v // 256}"


# Operation, sizes and the plans of its three products: every wide kernel in every layout, whole
# and split, with rows, columns and reductions that end inside a tile.
WIDE = [
    ("gated", 3850, 2056, 3400, "T256/1 T256/1 T256/1"),
    ("residual", 3850, 2056, 3400, "T256/1 T256/1 T256x128/1"),
    ("act", 3850, 2056, 3400, "T256/1 T256/1 T256x128/1"),
    ("residual", 1542, 5016, 1552, "T256x128/2 T256/1 T256/1"),
    ("gated", 257, 1440, 5472, "T256x128/1 T64/4 T128/1"),
    ("gated", 202, 4592, 2080, "T256x128/4 T128/4 T128/1"),
    ("gated", 4411, 72, 4424, "T128/1 T256x128/8 T256x128/4"),
    ("gated", 1869, 2184, 552, "T128/1 T256x128/1 T128/1"),
    ("residual", 5484, 1096, 712, "T256x128/1 T128/1 T128/4"),
    ("residual", 135, 4616, 5488, "T256x128/4 T64/1 T128/1"),
    ("residual", 131, 5448, 4984, "T64/1 T256x128/4 T128/1"),
    ("residual", 838, 4680, 1120, "T128/4 T256x128/1 T128/1"),
    ("residual", 4743, 136, 5528, "T128/1 T64/1 T256x128/4"),
    ("act", 1000, 5632, 2048, "T256x128/4 T256x128/1 T128/1"),
    ("gated", 2051, 2051, 2051, "ODD128/1 ODD128/1 ODD128/1"),
    ("residual", 2051, 2051, 2051, "ODD128/1 ODD128/1 ODD128/1"),
    ("act", 4001, 1201, 1703, "ODD128/1 ODD128/1 ODD64/1"),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("op, T, K, N, plans", WIDE)
def test_wide_tiles(hip_ops, op, T, K, N, plans, dtype):
    assert " ".join(plan(op, i, T, K, N, dtype) for i in range(3)) == plans
    x = make((T, K), 1, dtype)
    if op == "residual":
        w, b = make((N, K), 2, dtype, K ** -0.5), make((N,), 3, dtype, 0.3)
        r, s = make((T, N), 4, dtype), make((T, 1), 5, dtype)
        key = torch.tensor([T * 123456789, -K], device=DEV)
        check_residual(hip_ops, x, w, b, r, s, 0.2, key)
        check_residual(hip_ops, x, w, None, r, None)
        check_residual(hip_ops, x, w, None, None, s.float())
    else:
        rows = 2 * N if op == "gated" else N
        w, b = make((rows, K), 2, dtype, K ** -0.5), make((rows,), 3, dtype, 0.3)
        check_act(hip_ops, x, w, None, F.silu, op == "gated")
        check_act(hip_ops, x, w, b, F.gelu if op == "gated" else None, op == "gated")


@pytest.mark.parametrize("T, K, N, gated, residual", [
    (2048, 2048, 2048, "ODD128/1 ODD128/1 ODD128/1", "ODD128/1 ODD128/1 ODD128/1"),
    (1030, 2056, 2104, "ODD128/1 ODD64/1 ODD128/1", "ODD64/1 ODD64/1 ODD128/1")])
def test_wide_tiles_of_unaligned_operands(hip_ops, T, K, N, gated, residual):
    for op, plans in (("gated", gated), ("residual", residual)):
        assert " ".join(plan(op, i, T, K, N, aligned=False) for i in range(3)) == plans

    def off(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].copy_(t.reshape(-1)).view(t.shape)

    x, w = off(make((T, K), 1, BF)), off(make((2 * N, K), 2, BF, K ** -0.5))
    assert x.data_ptr() % 16 and w.data_ptr() % 16
    check_act(hip_ops, x, w, None, F.silu, True)
    r, s = off(make((T, N), 4, BF)), make((T, 1), 5, BF)
    check_residual(hip_ops, x, off(w[:N]), None, r, s, 0.2, torch.tensor([1, 2], device=DEV))


def test_few_rows_of_the_largest_weights(hip_ops):
    """The most that the kernel of few rows streams: above about 620 MB the tiles are taken."""
    for T, K, N, gated in ((1, 41168, 7560, False), (1, 55680, 2784, True)):
        assert plan("gated" if gated else "residual", 0, T, K, N) == "ROWS/1"
        x = make((T, K), 1, BF)
        g = torch.Generator(device=DEV).manual_seed(4)
        w = torch.empty((N * (1 + gated), K), dtype=BF, device=DEV).normal_(0.0, K ** -0.5, generator=g)
        if gated:
            check_act(hip_ops, x, w, None, F.silu, True, backward=False)
        else:
            check_residual(hip_ops, x, w, None, make((T, N), 5, BF), None, backward=False)


def test_more_rows_than_one_launch_of_a_wave_each(hip_ops):
    """2^26 rows and some more: the scale's gradient takes a wave per row, and a launch ends
    below 2^32 threads. The last rows against a call on them alone."""
    T, K, N, last = (1 << 26) + 5, 8, 8, 300
    g = torch.Generator(device=DEV).manual_seed(6)

    def normal(*shape):
        return torch.empty(shape, dtype=BF, device=DEV).normal_(generator=g)

    x, w, b, s, dy = normal(T, K), normal(N, K), normal(N), normal(T, 1), normal(T, N)
    s.requires_grad_()
    ds, = torch.autograd.grad(hip_ops.linear_residual(x, w, b, None, s), s, dy)
    part = s[-last:].detach().requires_grad_()
    want, = torch.autograd.grad(hip_ops.linear_residual(x[-last:], w, b, None, part), part, dy[-last:])
    # fp32 sums of 8 + 8 products, rounded once: at most the order of the sums differs.
    X, W, B, G = wide(x[-last:], w, b, dy[-last:])
    mag = (X.abs() * (G.abs() @ W.abs())).sum(1) + G.abs() @ B.abs()
    exact = (X * (G @ W)).sum(1) + G @ B
    tol = unit(BF) * exact.abs() + 1.01 * (gamma(N) + gamma(K)) * mag
    within(ds[-last:].reshape(-1), exact, tol, "ds")
    within(want.reshape(-1), exact, tol, "ds of the last rows")


def test_dropout_of_more_rows_than_its_launch_has(hip_ops):
    rows, cols = (1 << 22) + 3, 1032  # four rows to a block of threads at a time
    x = torch.ones((rows, cols), dtype=BF, device=DEV)
    key = torch.tensor([79, 80], device=DEV)
    y = hip_ops.dropout(x, 0.5, key)
    for at in (0, (1 << 22) - 2, rows - 3):
        f = o_dropout.factors(3, cols, 0.5, key.cpu(), at)
        assert torch.equal(y[at:at + 3].double().cpu(), f), at
