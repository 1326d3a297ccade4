"""Performance cases of the 4-bit expert path and of the norm before it, through ``ops``.

Weights are E2M1 in groups of 32 along the reduction, each group with a power of
two (an E8M0 byte); rows are bf16, or E4M3 with the same groups. Each case is a
dict of plain values; ``prepare`` makes its inputs on the GPU, ``run`` makes one
pass, ``exact`` gives the same outputs in 64 bits. The kinds:

* ``norm``: ``ops.rms_norm`` with the residual's addition, and its backward;
* ``norm_mx``: ``ops.rms_norm_mx``, the same with the normalised rows in 8 bits too;
* ``quantize``: weights to 4 bits and back (``ops.quantize_mxfp4``, ``ops.dequantize_mxfp4``);
* ``linear``: ``ops.linear_mxfp4``, a dense product with 4-bit weights;
* ``experts``: ``ops.grouped_matmul_mxfp4``, the product of every expert's rows.

``train`` cases return the output and every gradient, the others run forward
without gradients; ``mx`` cases take rows in 8 bits; ``mx_out`` cases give such
rows, returned as the values they stand for. With ``own`` false, ``run`` computes
the same from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 32
EPS = 1e-6


def _case(name, kind, rows, k, n, **more):
    """``k``: features of a row; ``n``: the output's features (of one half where gated)."""
    case = {"name": name, "kind": kind, "rows": rows, "k": k, "n": n, "dtype": "bf16",
            "train": False, "residual": False, "mx": False, "mx_out": False, "gated": False,
            "act": "none", "experts": 0}
    case.update(more)
    return case


def listed():
    return [
        # Norm before the experts of one decoding token: the router's rows and the experts'.
        _case("norm_mx_decode_1", "norm_mx", 1, 7168, 0, residual=True),
        # The same for a prompt of 4096 tokens.
        _case("norm_mx_prefill_4k", "norm_mx", 4096, 7168, 0, residual=True),
        # Norm of the headline layer in training, with the residual stream.
        _case("norm_train_16k", "norm", 16384, 2048, 0, residual=True, train=True),
        # A shared expert's gate and up weights, when a checkpoint is loaded.
        _case("quantize_shared", "quantize", 0, 7168, 4096, experts=1),
        # 32 experts' gate and up weights.
        _case("quantize_experts", "quantize", 0, 7168, 4096, experts=32),
        # Shared expert's gate and up for one decoding token: a stream of weights.
        _case("linear_decode_1", "linear", 1, 7168, 2048, act="silu", gated=True),
        # Its down projection for a batch of decoding sequences, rows in 8 bits.
        _case("linear_decode_24_mx", "linear", 24, 2048, 7168, mx=True),
        # Gate and up of a wide layer for a prompt, rows in 8 bits.
        _case("linear_prefill_4k_mx", "linear", 4096, 4096, 14336, mx=True, act="silu", gated=True),
        # A frozen projection under adapters, ragged batch: forward and the rows' gradient.
        _case("linear_train_1531", "linear", 1531, 5632, 2048, train=True),
        # 16 decoding tokens, 8 of 128 experts each: gate, up, SwiGLU and probabilities.
        _case("experts_decode_128", "experts", 128, 2048, 768, experts=128, gated=True),
        # A prompt of 4096 tokens, 8 of 64 experts each, rows in 8 bits in and out.
        _case("experts_prefill_32k_mx", "experts", 32768, 7168, 2048, experts=64, gated=True,
              mx=True, mx_out=True),
        # The headline layer's first product with frozen experts: forward and the rows' gradient.
        _case("experts_train_131k", "experts", 131072, 2048, 1536, experts=128, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_mx", "quantize", "linear", "linear", "linear", "experts",
                       "experts", "experts"])
    while True:
        if kind == "norm":
            case = _case("", kind, _log(rng, 1, 32768), _log(rng, 33, 16384), 0,
                         residual=rng.random() < 0.6, train=rng.random() < 0.6,
                         dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
            if case["rows"] * case["k"] > 1 << 27:
                continue
        elif kind == "norm_mx":
            case = _case("", kind, _log(rng, 1, 32768), GROUP * _log(rng, 2, 448), 0,
                         residual=rng.random() < 0.6, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
            if case["rows"] * case["k"] > 1 << 27:
                continue
        elif kind == "quantize":
            case = _case("", kind, 0, GROUP * _log(rng, 2, 448), _log(rng, 33, 8192),
                         experts=rng.choice([1, 4, 8, 16]),
                         dtype=rng.choice(["bf16", "bf16", "f32"]))
            if case["experts"] * case["k"] * case["n"] > 1 << 28:
                continue
        else:
            experts = rng.choice([8, 32, 60, 128]) if kind == "experts" else 0
            train = rng.random() < 0.3
            mx = not train and rng.random() < 0.5
            gated = not train and rng.random() < 0.6
            mx_out = mx and rng.random() < 0.4
            odd = rng.random() < 0.25 and not mx_out
            n = _log(rng, 33, 2049) if odd else GROUP * _log(rng, 2, 256)
            act = "none"
            if kind == "linear" and not train:
                act = rng.choice(["silu", "gelu"]) if gated else rng.choice(["none", "none", "silu"])
            case = _case("", kind, _log(rng, 1, 16384 if kind == "linear" else 65536),
                         GROUP * _log(rng, 2, 256), n, experts=experts, train=train, mx=mx,
                         mx_out=mx_out, gated=gated, act=act)
            if work(case)["flops"] > 1e12 or max(experts, 1) * case["k"] * n > 1 << 30:
                continue
        del case["name"]
        return case


# ---------------------------------------------------------------------------
# The formats, in 32 bits
# ---------------------------------------------------------------------------
def _group_scale(v, top):
    """(E8M0 bytes [..., K / 32, 1], 2^-(byte - 127)) of ``v`` [..., K / 32, 32]: the group's
    largest exponent less the element type's, ``top``."""
    amax = v.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(amax).exponent.to(torch.int32) - 1
    byte = torch.where(amax > 0, (exponent - top + 127).clamp(0, 254), torch.zeros_like(exponent))
    return byte, ((254 - byte) << 23).view(torch.float32)


def _power(byte):
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _to_e2m1(v):
    """``v`` [..., 32 g] as (E2M1 values, E8M0 bytes [..., g, 1]), both before packing."""
    v = v.unflatten(-1, (-1, GROUP))
    byte, inverse = _group_scale(v, 2)
    q = (v * inverse).clamp(-6.0, 6.0)
    step = torch.where(q.abs() >= 4, 2.0, torch.where(q.abs() >= 2, 1.0, 0.5))
    return torch.round(q / step) * step, byte


def _to_e4m3(v):
    v = v.unflatten(-1, (-1, GROUP))
    byte, inverse = _group_scale(v, 8)
    return (v * inverse).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), byte


def _pack(q):
    """E2M1 values [..., K] as bytes [..., K / 2], the lower index in the low four bits."""
    a = q.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code + (q < 0).to(torch.uint8) * 8
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _weights(codes, scales):
    """fp32 values [..., N, K] of packed codes [..., N, K / 2] and E8M0 bytes [..., N, K / 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    both = torch.stack([codes & 15, codes >> 4], dim=-1).to(torch.int32)
    values = table[both].flatten(-2).unflatten(-1, (-1, GROUP))
    return (values * _power(scales).unsqueeze(-1)).flatten(-2)


def _rows(codes, scales):
    """fp32 values of E4M3 rows [..., K] with E8M0 bytes [..., K / 32]."""
    values = codes.float().unflatten(-1, (-1, GROUP))
    return (values * _power(scales).unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(shape, g, std, dtype):
    return torch.empty(shape, device=DEV).normal_(0.0, std, generator=g).to(dtype)


def _hidden(rows, k, g, dtype):
    """Hidden states as a model has them: rows of their own size, a few features far larger."""
    x = torch.empty((rows, k), device=DEV).normal_(generator=g)
    x *= torch.empty((rows, 1), device=DEV).normal_(generator=g).mul_(0.5).exp_()
    x[:, torch.randperm(k, generator=g, device=DEV)[: k // 200]] *= 12.0
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T, K, N, kind, dtype = (case[v] for v in ("rows", "k", "n", "kind", "dtype"))
    dtype = DTYPES[dtype]
    E = case["experts"]
    state = {"case": case}
    if kind in ("norm", "norm_mx"):
        state["x"] = _hidden(T, K, g, dtype)
        state["residual"] = _hidden(T, K, g, dtype) if case["residual"] else None
        state["weight"] = _normal((K,), g, 0.1, torch.float32).add_(1.0).to(dtype)
        if case["train"]:
            state["grad"] = _normal((T, K), g, 1.0, dtype)
            state["grad_sum"] = _normal((T, K), g, 1.0, dtype) if case["residual"] else None
        return state
    width = 2 * N if case["gated"] else N
    if kind == "quantize":
        w = torch.empty((E, N, K), dtype=dtype, device=DEV)
        for e in range(E):
            w[e] = _normal((N, K), g, 0.02, dtype)
        state["w"] = w
        return state
    codes = torch.empty((max(E, 1), width, K // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((max(E, 1), width, K // GROUP), dtype=torch.uint8, device=DEV)
    for e in range(max(E, 1)):
        q, byte = _to_e2m1(_normal((width, K), g, 0.02, torch.float32))
        codes[e], scales[e] = _pack(q.flatten(-2)), byte.squeeze(-1).to(torch.uint8)
    state["codes"], state["scales"] = (codes, scales) if E else (codes[0], scales[0])
    x = _normal((T, K), g, 1.0, torch.float32)
    if case["mx"]:
        q, byte = _to_e4m3(x)
        state["x"] = (q.flatten(-2), byte.squeeze(-1).to(torch.uint8))
    else:
        state["x"] = x.to(dtype)
    if kind == "experts":
        # Loads of the experts as a skewed router gives them; some may have no rows.
        share = torch.empty(E, device=DEV).exponential_(generator=g)
        taken = torch.multinomial(share, T, replacement=True, generator=g)
        state["counts"] = torch.bincount(taken, minlength=E)
        state["loads"] = state["counts"].tolist()
        state["probs"] = torch.rand(T, generator=g, device=DEV) if case["gated"] else None
    if case["train"]:
        state["grad"] = _normal((T, N), g, 1.0, dtype)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _activate(act, a):
    if act == "silu":
        return a / (1.0 + torch.exp(-a))
    if act == "gelu":
        return 0.5 * a * (1.0 + torch.erf(a * math.sqrt(0.5)))
    return a


def _plain_norm(x, residual, weight):
    h = x if residual is None else x + residual
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * weight, h


def _plain_epilogue(case, a, probs):
    act = "silu" if case["kind"] == "experts" and case["gated"] else case["act"]
    if case["gated"]:
        gate, up = a.chunk(2, dim=-1)
        a = _activate(act, gate) * up
    else:
        a = _activate(act, a)
    return a if probs is None else a * probs.unsqueeze(-1)


def _plain_product(state, x):
    if state["case"]["kind"] == "linear":
        return x @ _weights(state["codes"], state["scales"]).t()
    parts = x.split(state["loads"])
    return torch.cat([v @ _weights(state["codes"][e], state["scales"][e]).t()
                      for e, v in enumerate(parts)])


def _run_plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        q, byte = _to_e2m1(state["w"].float())
        return {"w": (q * _power(byte)).flatten(-2).to(torch.bfloat16)}
    if kind in ("norm", "norm_mx"):
        dtype = state["x"].dtype
        x, weight = state["x"].float(), state["weight"].float()
        residual = None if state["residual"] is None else state["residual"].float()
        if not case["train"]:
            y, h = _plain_norm(x, residual, weight)
            result = {"y": y.to(dtype)}
            if residual is not None:
                result["sum"] = h.to(dtype)
            if kind == "norm_mx":
                q, byte = _to_e4m3(y)
                result["rows"] = (q.float() * _power(byte)).flatten(-2).to(torch.bfloat16)
            return result
        leaves = [v.requires_grad_() for v in (x, weight, residual) if v is not None]
        y, h = _plain_norm(x, residual, weight)
        outs, grads = [y], [state["grad"].float()]
        if residual is not None:
            outs, grads = [y, h], [*grads, state["grad_sum"].float()]
        d = torch.autograd.grad(outs, leaves, grads)
        result = {"y": y.detach().to(dtype), "d_x": d[0].to(dtype), "d_weight": d[1].to(dtype)}
        if residual is not None:
            result["sum"], result["d_residual"] = h.detach().to(dtype), d[2].to(dtype)
        return result
    x = _rows(*state["x"]) if case["mx"] else state["x"].float()
    if case["train"]:
        x.requires_grad_()
        y = _plain_product(state, x)
        dx, = torch.autograd.grad(y, x, state["grad"].float())
        return {"y": y.detach().to(torch.bfloat16), "d_x": dx.to(torch.bfloat16)}
    y = _plain_epilogue(case, _plain_product(state, x), state.get("probs"))
    if case["mx_out"]:
        q, byte = _to_e4m3(y)
        y = (q.float() * _power(byte)).flatten(-2)
    return {"y": y.to(torch.bfloat16)}


def _call_product(ops, state, x):
    case = state["case"]
    if case["kind"] == "linear":
        act = {"silu": F.silu, "gelu": F.gelu, "none": None}[case["act"]]
        return ops.linear_mxfp4(x, state["codes"], state["scales"], activation_func=act,
                                gated=case["gated"], mx_out=case["mx_out"])
    return ops.grouped_matmul_mxfp4(x, state["codes"], state["scales"], state["counts"],
                                    probs=state["probs"], gated=case["gated"],
                                    mx_out=case["mx_out"])


def _run_own(state):
    from torchturbo_amd import init_ops
    from torchturbo_amd.dispatch import MxRows

    case, kind = state["case"], state["case"]["kind"]
    ops = init_ops()
    if kind == "quantize":
        return {"w": ops.dequantize_mxfp4(*ops.quantize_mxfp4(state["w"]))}
    if kind == "norm_mx":
        out = ops.rms_norm_mx(state["x"], state["weight"], EPS, residual=state["residual"],
                              with_y=True)
        result = {"y": out.y, "rows": ops.dequantize_mxfp8(out.rows)}
        if state["residual"] is not None:
            result["sum"] = out.sum
        return result
    if kind == "norm":
        names = [n for n in ("x", "weight", "residual") if state[n] is not None]
        leaves = {n: state[n].detach().requires_grad_(case["train"]) for n in names}
        out = ops.rms_norm(leaves["x"], leaves["weight"], EPS, residual=leaves.get("residual"))
        y, h = out if state["residual"] is not None else (out, None)
        result = {"y": y.detach()}
        if h is not None:
            result["sum"] = h.detach()
        if case["train"]:
            outs = [v for v in (y, h) if v is not None]
            grads = [v for v in (state["grad"], state["grad_sum"]) if v is not None]
            d = torch.autograd.grad(outs, list(leaves.values()), grads)
            result.update({"d_" + n: v for n, v in zip(names, d)})
        return result
    if case["train"]:
        x = state["x"].detach().requires_grad_()
        y = _call_product(ops, state, x)
        dx, = torch.autograd.grad(y, x, state["grad"])
        return {"y": y.detach(), "d_x": dx}
    with torch.no_grad():
        y = _call_product(ops, state, MxRows(*state["x"]) if case["mx"] else state["x"])
        return {"y": ops.dequantize_mxfp8(y) if case["mx_out"] else y}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def _two_to(exponent):
    """2^exponent of whole numbers, in 64 bits."""
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rounded(v, bits, least, most, top):
    """``v`` in groups of 32 that share a power of two, each value rounded to ``bits`` fraction
    bits (half to even), exponents from ``least`` on, at most ``most``; the values."""
    shape = v.shape
    v = v.reshape(*shape[:-1], -1, GROUP)
    amax = v.abs().amax(-1, keepdim=True)
    scale = _two_to((torch.floor(torch.log2(amax.clamp(min=2.0 ** -140))) - top).clamp(min=-127))
    u = v / scale
    exponent = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** least)))
    step = _two_to(exponent - bits)
    return (torch.clamp(torch.round(u / step) * step, -most, most) * scale).reshape(shape)


def _exact_weights(codes, scales):
    c = torch.empty((*codes.shape[:-1], codes.shape[-1] * 2), dtype=torch.int64, device=codes.device)
    c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
    exponent, half, sign = (c // 2) % 4, (c % 2).double() / 2, 1.0 - 2.0 * (c // 8)
    value = sign * torch.where(exponent == 0, half, (1 + half) * _two_to(exponent - 1))
    return value * _two_to(scales.long() - 127).repeat_interleave(GROUP, -1)


def _exact_act(act, a):
    if act == "silu":
        return a * torch.sigmoid(a)
    if act == "gelu":
        return 0.5 * a * torch.erfc(-a / math.sqrt(2.0))
    return a


def exact(case, seed):
    s = prepare(case, seed)
    kind, N = case["kind"], case["n"]
    if kind == "quantize":
        w = torch.empty_like(s["w"], dtype=torch.float32)
        for e in range(case["experts"]):
            w[e] = _rounded(s["w"][e].double(), 1, 0, 6.0, 2)
        return {"w": w}  # each is a 32-bit value
    if kind in ("norm", "norm_mx"):
        h, w = s["x"].double(), s["weight"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        rho = (h.pow(2).sum(-1, keepdim=True) / case["k"] + EPS).pow(-0.5)
        y = h * rho * w
        result = {"y": y}
        if s["residual"] is not None:
            result["sum"] = h
        if kind == "norm_mx":
            result["rows"] = _rounded(y, 3, -6, 448.0, 8)
        if case["train"]:
            g = s["grad"].double()
            a = g * w
            dh = rho * a - h * rho.pow(3) * (a * h).sum(-1, keepdim=True) / case["k"]
            if s["residual"] is not None:
                dh = dh + s["grad_sum"].double()
                result["d_residual"] = dh
            result["d_x"], result["d_weight"] = dh, (g * h * rho).sum(0)
        return result
    if case["mx"]:
        codes, scales = s["x"]
        x = codes.double() * _two_to(scales.long() - 127).repeat_interleave(GROUP, -1)
    else:
        x = s["x"].double()
    dx = torch.empty_like(x) if case["train"] else None
    y = torch.empty((x.shape[0], N), dtype=torch.float64, device=DEV)
    act = "silu" if kind == "experts" and case["gated"] else case["act"]
    at = 0
    for e, count in enumerate(s["loads"] if kind == "experts" else [x.shape[0]]):
        part = slice(at, at + count)
        at += count
        w = (_exact_weights(s["codes"][e], s["scales"][e]) if kind == "experts" else
             _exact_weights(s["codes"], s["scales"]))
        a = x[part] @ w.t()
        if case["gated"]:
            y[part] = _exact_act(act, a[:, :N]) * a[:, N:]
        else:
            y[part] = _exact_act(act, a)
        if case["train"]:
            dx[part] = s["grad"][part].double() @ w
    if s.get("probs") is not None:
        y *= s["probs"].double()[:, None]
    if case["mx_out"]:
        y = _rounded(y, 3, -6, 448.0, 8)
    return {"y": y, "d_x": dx} if case["train"] else {"y": y}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    T, K, N, E = case["rows"], case["k"], case["n"], case["experts"]
    b = 4 if case["dtype"] == "f32" else 2
    small = 1.0 + 1.0 / GROUP  # bytes of a value in 8 bits with its share of the scale
    if case["kind"] == "quantize":
        # The weights in; codes and scales out and in again; the values out.
        return {"bytes": E * N * K * (b + 2 * (0.5 + 1.0 / GROUP) + 2.0), "flops": 4.0 * E * N * K}
    if case["kind"] in ("norm", "norm_mx"):
        streams = 4.0 if case["residual"] else 2.0  # x, residual, sum, y
        bytes_ = T * K * b * streams
        if case["kind"] == "norm_mx":
            bytes_ += T * K * (2 * small + 2.0)  # rows out, in again, and their values
        if case["train"]:
            bytes_ += T * K * b * (4.0 if case["residual"] else 3.0)  # gradients, sum, d_x
        return {"bytes": bytes_, "flops": T * K * (12.0 if case["train"] else 4.0)}
    width = 2 * N if case["gated"] else N
    experts = min(E, T) if E else 1
    weights = experts * width * K * (0.5 + 1.0 / GROUP)
    row_in = K * (small if case["mx"] else 2.0)
    row_out = N * (2 * small + 2.0 if case["mx_out"] else 2.0)
    times = 2.0 if case["train"] else 1.0
    return {"bytes": times * (weights + T * (row_in + row_out)),
            "flops": times * 2.0 * T * K * width}
