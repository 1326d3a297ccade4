"""Performance cases of the layer's dense products and of counter-based dropout, through ``ops``.

Each case is a dict of plain values; ``prepare`` makes its inputs on the GPU,
``run`` makes one pass, ``exact`` gives the same outputs in 64 bits. The kinds:

* ``act``: ``ops.linear_act``, a product with bias, activation and (gated) the
  product of its two halves: the first half of a shared expert;
* ``residual``: ``ops.linear_residual``, a product with bias, dropout, a scale
  for each row and a residual: its second half, added to the routed experts;
* ``dropout``: ``ops.dropout``, with a mask that is computed from a key and the
  position, and again in the backward;
* ``lora``: ``ops.lora_residual`` with such a dropout on its rows.

``train`` cases return the output and every gradient, the others run forward
without gradients. With ``own`` false, ``run`` computes the same from elementary
torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, kind, tokens, k, n, **more):
    """``n``: the output's features (of one half where gated)."""
    case = {"name": name, "kind": kind, "tokens": tokens, "k": k, "n": n, "dtype": "bf16",
            "train": False, "act": "none", "gated": False, "bias": False, "scale": False,
            "p": 0.0, "experts": 0, "rank": 0}
    case.update(more)
    return case


def listed():
    return [
        # Shared expert's gate and up of a decode step: the smallest call, one weight stream.
        _case("act_decode_1", "act", 1, 7168, 2048, act="silu", gated=True),
        # The same in training, a micro batch of 4096 tokens.
        _case("act_train_4k", "act", 4096, 7168, 2048, act="silu", gated=True, train=True),
        # The largest: a wide gated layer over a long batch.
        _case("act_train_8x14k", "act", 8192, 4096, 14336, act="silu", gated=True, train=True),
        # A ragged batch of a small model in f16, GELU and bias.
        _case("act_ragged_f16", "act", 1531, 1024, 704, act="gelu", gated=True, bias=True,
              dtype="f16", train=True),
        # A unit-sized model in fp32, without a gate.
        _case("act_toy_f32", "act", 512, 256, 512, act="gelu", bias=True, dtype="f32", train=True),
        # Shared expert's down projection for a batch of decoding sequences.
        _case("residual_decode_24", "residual", 24, 2048, 7168),
        # The same for a prompt, with the shared expert's gate and a bias.
        _case("residual_prefill_1000", "residual", 1000, 5632, 2048, scale=True, bias=True),
        # The down projection in training, gated for each token.
        _case("residual_train_4k", "residual", 4096, 2048, 7168, scale=True, train=True),
        # With dropout of the expert's output, odd batch.
        _case("residual_drop_777", "residual", 777, 704, 1024, bias=True, p=0.1, train=True),
        # Rows of the adapters of one decode-sized step: latency.
        _case("dropout_24", "dropout", 24, 0, 2048, p=0.05, dtype="f16", train=True),
        # Packed rows of the headline layer: bandwidth.
        _case("dropout_131k", "dropout", 131072, 0, 2048, p=0.1, train=True),
        # Adapters of 128 experts with dropout, 2048 tokens of 8 experts each.
        _case("lora_16k_r16", "lora", 16384, 2048, 1536, experts=128, rank=16, p=0.05, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["act", "act", "act", "residual", "residual", "residual", "dropout", "lora"])
    while True:
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
        if kind == "dropout":
            case = _case("", kind, _log(rng, 1, 131072), 0, _log(rng, 7, 8192), dtype=dtype,
                         train=True, p=rng.choice([0.05, 0.1, 0.3, 0.5]))
            if case["tokens"] * case["n"] > (1 << 28):
                continue
        elif kind == "lora":
            case = _case("", kind, _log(rng, 64, 16384), 64 * _log(rng, 8, 40),
                         32 * _log(rng, 12, 64), dtype=rng.choice(["bf16", "f16"]), train=True,
                         experts=rng.choice([8, 32, 60, 128]), rank=rng.choice([4, 8, 16, 32, 64]),
                         p=rng.choice([0.05, 0.1, 0.3]))
        else:
            odd = rng.random() < 0.25  # sizes that no vector load fits
            size = (lambda: _log(rng, 33, 2049)) if odd else (lambda: 8 * _log(rng, 8, 1024))
            case = _case("", kind, _log(rng, 1, 16384), size(), size(), dtype=dtype,
                         train=rng.random() < 0.5, bias=rng.random() < 0.5)
            if kind == "act":
                case["act"] = rng.choice(["silu", "silu", "gelu", "none"])
                case["gated"] = case["act"] != "none" and rng.random() < 0.7
            else:
                case["scale"] = rng.random() < 0.5
                if case["train"] and rng.random() < 0.3:
                    case["p"] = rng.choice([0.05, 0.1, 0.5])
            flops = work(case)["flops"]
            if flops > (1e11 if odd or dtype == "f32" else 2e12):
                continue
        del case["name"]
        return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(shape, g, std, dtype):
    return torch.empty(shape, device=DEV).normal_(0.0, std, generator=g).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T, K, N, dtype = case["tokens"], case["k"], case["n"], DTYPES[case["dtype"]]
    state = {"case": case}
    if case["p"]:
        # The dropout's key, drawn for each step: a seed and an offset.
        state["key"] = torch.randint(-(1 << 62), 1 << 62, (2,), generator=g, device=DEV)
    if case["train"]:
        state["grad"] = _normal((T, N), g, 1.0, dtype)
    if case["kind"] == "dropout":
        state["x"] = _normal((T, N), g, 1.0, dtype)
        return state
    state["x"] = _normal((T, K), g, 1.0, dtype)
    if case["kind"] == "lora":
        E, r = case["experts"], case["rank"]
        # Loads of the experts as a skewed router gives them; some may have no rows.
        weights = torch.empty(E, device=DEV).exponential_(generator=g)
        taken = torch.multinomial(weights, T, replacement=True, generator=g)
        state["counts"] = torch.bincount(taken, minlength=E)
        state["loads"] = state["counts"].tolist()
        state["base"] = _normal((T, N), g, 1.0, dtype)
        state["a"] = _normal((E, K, r), g, 1.0 / math.sqrt(K), torch.float32)
        state["b"] = _normal((E, r, N), g, 0.02, torch.float32)
        return state
    rows = 2 * N if case["gated"] else N
    state["w"] = _normal((rows, K), g, 0.02, dtype)
    state["bias"] = _normal((rows,), g, 0.1, dtype) if case["bias"] else None
    if case["kind"] == "residual":
        state["residual"] = _normal((T, N), g, 1.0, dtype)
        state["scale"] = (torch.sigmoid(_normal((T, 1), g, 1.0, torch.float32)).to(dtype)
                          if case["scale"] else None)
    return state


NAMES = {"act": ("x", "w", "bias"), "residual": ("x", "w", "bias", "residual", "scale"),
         "dropout": ("x",), "lora": ("x", "a", "b")}
SCALING = 2.0  # alpha / r of the adapters


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _keep(key, rows, cols):
    """The 16-bit random number of each element [rows, cols]: Philox4x32-10 (Salmon, Moraes,
    Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with the key's first entry as
    its key and the counter (column / 8, row, the key's second entry)."""
    low = 0xFFFFFFFF
    groups = (cols + 7) // 8
    c0 = torch.arange(groups, device=DEV).expand(rows, groups)
    c1 = torch.arange(rows, device=DEV).unsqueeze(1).expand(rows, groups)
    k0, k1 = key[0] & low, (key[0] >> 32) & low
    c2, c3 = key[1] & low, (key[1] >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64
        c0, c2 = ((p1 >> 32) & low) ^ c1 ^ k0, ((p0 >> 32) & low) ^ c3 ^ k1
        c1, c3 = p1 & low, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    parts = [v for c in (c0, c1, c2, c3) for v in (c & 0xFFFF, c >> 16)]
    return torch.stack([v.to(torch.int32) for v in parts], dim=2).view(rows, -1)[:, :cols]


def _plain_dropout(x, p, key):
    drop = min(max(round(p * 65536), 1), 65535)
    keep = _keep(key, *x.shape) >= drop
    return torch.where(keep, x * (65536.0 / (65536 - drop)), torch.zeros((), device=DEV))


def _activate(case, a):
    if case["act"] == "silu":
        return a / (1.0 + torch.exp(-a))
    if case["act"] == "gelu":
        return 0.5 * a * (1.0 + torch.erf(a * math.sqrt(0.5)))
    return a


def _plain(state, leaves):
    case, kind = state["case"], state["case"]["kind"]
    x = leaves["x"]
    if kind == "dropout":
        return _plain_dropout(x, case["p"], state["key"])
    if kind == "lora":
        rows = _plain_dropout(x, case["p"], state["key"])
        parts = rows.split(state["loads"])
        delta = [v @ leaves["a"][e] @ leaves["b"][e] for e, v in enumerate(parts)]
        return state["base"].float() + torch.cat(delta) * SCALING
    y = x @ leaves["w"].t()
    if leaves["bias"] is not None:
        y = y + leaves["bias"]
    if kind == "act":
        if case["gated"]:
            gate, up = y.chunk(2, dim=1)
            return _activate(case, gate) * up
        return _activate(case, y)
    if case["p"]:
        y = _plain_dropout(y, case["p"], state["key"])
    if leaves["scale"] is not None:
        y = y * leaves["scale"]
    return leaves["residual"] + y


def _call(state, leaves):
    from torchturbo_amd import init_ops

    case, kind = state["case"], state["case"]["kind"]
    ops = init_ops()
    if kind == "dropout":
        return ops.dropout(leaves["x"], case["p"], state["key"])
    if kind == "lora":
        return ops.lora_residual(state["base"], leaves["x"], leaves["a"], leaves["b"],
                                 state["counts"], SCALING, dropout_p=case["p"],
                                 dropout_key=state["key"])
    if kind == "act":
        act = {"silu": F.silu, "gelu": F.gelu, "none": None}[case["act"]]
        return ops.linear_act(leaves["x"], leaves["w"], leaves["bias"], activation_func=act,
                              gated=case["gated"])
    return ops.linear_residual(leaves["x"], leaves["w"], leaves["bias"], leaves["residual"],
                               leaves["scale"], dropout_p=case["p"], dropout_key=state.get("key"))


def run(state):
    case = state["case"]
    given = {n: state[n] for n in NAMES[case["kind"]]}
    leaves = {n: None if v is None else v.detach() if own else v.detach().float()
              for n, v in given.items()}
    compute = _call if own else _plain
    if not case["train"]:
        with torch.no_grad():
            return {"y": compute(state, leaves).to(state["x"].dtype)}
    wanted = [n for n, v in leaves.items() if v is not None]
    for n in wanted:
        leaves[n].requires_grad_()
    y = compute(state, leaves)
    grads = torch.autograd.grad(y, [leaves[n] for n in wanted], state["grad"].to(y.dtype))
    result = {"y": y.detach().to(state["x"].dtype)}
    for n, v in zip(wanted, grads):
        result["d_" + n] = v.to(given[n].dtype)
    return result


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def _product32(constant, v):
    """High and low 32 bits of ``constant * v``, of 16-bit limbs."""
    ch, cl, vh, vl = constant >> 16, constant & 0xFFFF, v >> 16, v & 0xFFFF
    low, mid1, mid2 = cl * vl, ch * vl, cl * vh
    carry = (low >> 16) + (mid1 & 0xFFFF) + (mid2 & 0xFFFF)
    high = ch * vh + (mid1 >> 16) + (mid2 >> 16) + (carry >> 16)
    return high, ((carry & 0xFFFF) << 16) | (low & 0xFFFF)


def _factor(case, key, rows, cols):
    """Dropout's factor of each element, 0 or the inverse of the kept share."""
    seed, offset = (int(v) % (1 << 64) for v in key.tolist())
    group = torch.arange((cols + 7) // 8, device=DEV).repeat(rows, 1)
    row = torch.arange(rows, device=DEV).repeat_interleave(group.shape[1]).view_as(group)
    ctr = [group, row, torch.full_like(row, offset % (1 << 32)), torch.full_like(row, offset >> 32)]
    words = [seed % (1 << 32), seed >> 32]
    for _ in range(10):
        h0, l0 = _product32(0xD2511F53, ctr[0])
        h1, l1 = _product32(0xCD9E8D57, ctr[2])
        ctr = [h1 ^ ctr[1] ^ words[0], l1, h0 ^ ctr[3] ^ words[1], l0]
        words = [(words[0] + 0x9E3779B9) % (1 << 32), (words[1] + 0xBB67AE85) % (1 << 32)]
    drop = min(max(round(case["p"] * 65536), 1), 65535)
    out = torch.empty((rows, group.shape[1] * 8), dtype=torch.float64, device=DEV)
    for j in range(8):
        half = (ctr[j // 2] >> 16) if j % 2 else ctr[j // 2] % 65536
        out[:, j::8] = (half >= drop) * (65536.0 / (65536 - drop))
    return out[:, :cols]


def _derivative(case, a):
    """(act(a), act'(a))."""
    if case["act"] == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1.0 + a * (1.0 - s))
    if case["act"] == "gelu":
        cdf = 0.5 * torch.erfc(-a / math.sqrt(2.0))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)
    return a, torch.ones_like(a)


def exact(case, seed):
    s = prepare(case, seed)
    train, kind, N = case["train"], case["kind"], case["n"]
    x = s["x"].double()
    g = s["grad"].double() if train else None
    if kind == "dropout":
        f = _factor(case, s["key"], *x.shape)
        return {"y": x * f, "d_x": g * f}
    if kind == "lora":
        f = _factor(case, s["key"], *x.shape)
        rows, y, dx = x * f, s["base"].double(), torch.zeros_like(x)
        da, db = s["a"].double().zero_(), s["b"].double().zero_()
        at = 0
        for e, count in enumerate(s["loads"]):
            part = slice(at, at + count)
            a, b = s["a"][e].double(), s["b"][e].double()
            y[part] += SCALING * (rows[part] @ a) @ b
            back = SCALING * g[part] @ b.t()
            dx[part] = (back @ a.t()) * f[part]
            da[e], db[e] = rows[part].t() @ back, SCALING * (rows[part] @ a).t() @ g[part]
            at += count
        return {"y": y, "d_x": dx, "d_a": da, "d_b": db}
    w = s["w"].double()
    a = x @ w.t()
    if s["bias"] is not None:
        a += s["bias"].double()
    result = {}
    if kind == "act":
        if case["gated"]:
            value, slope = _derivative(case, a[:, :N])
            result["y"] = value * a[:, N:]
            da = torch.cat([g * a[:, N:] * slope, g * value], dim=1) if train else None
        else:
            result["y"], slope = _derivative(case, a)
            da = g * slope if train else None
    else:
        scale = s["scale"].double() if s["scale"] is not None else 1.0
        f = _factor(case, s["key"], *a.shape) if case["p"] else 1.0
        result["y"] = s["residual"].double() + a * f * scale
        da = g * f * scale if train else None
        if train:
            result["d_residual"] = g
            if s["scale"] is not None:
                result["d_scale"] = (g * f * a).sum(1, keepdim=True)
    if train:
        result["d_x"], result["d_w"] = da @ w, da.t() @ x
        if s["bias"] is not None:
            result["d_bias"] = da.sum(0)
    return result


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    T, K, N = case["tokens"], case["k"], case["n"]
    b = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "dropout":
        return {"bytes": 4.0 * T * N * b, "flops": 2.0 * T * N}
    if case["kind"] == "lora":
        E, r = case["experts"], case["rank"]
        # x, the base and the gradient in, y and the rows' gradient out; adapters and theirs.
        return {"bytes": T * (2.0 * K + 3.0 * N) * b + 2.0 * E * r * (K + N) * 4,
                "flops": 6.0 * T * r * (K + N)}
    rows = 2 * N if case["gated"] else N
    residual = T * N * b if case["kind"] == "residual" else 0
    bytes_ = (T * K + rows * K + T * N) * b + residual
    flops = 2.0 * T * K * rows
    if case["train"]:
        return {"bytes": 2.0 * bytes_, "flops": 3.0 * flops}
    return {"bytes": float(bytes_), "flops": flops}
