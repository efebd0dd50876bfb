"""The operators of a pre-norm gated feed-forward block and its update, as they are measured: layer norm (forward and
backward), the gated linear layer h = act(x Wg + bg) * (x Wu + bu) (forward and backward) and the AdamW step over many
tensors, with states in 32 or 8 bits.  `run` computes them in plain torch operations, or, where `own` is true, through
this package's public calls."""
import math

import torch

own = False

BLOCK = 256       # values that share a scale in an 8-bit state
EPS = 1e-5        # layer norm
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.95, 1e-8, 0.1
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def listed():
    return [
        # one token's norm while text is generated: latency alone
        {"name": "norm_one_token", "op": "norm", "rows": 1, "cols": 4096, "type": "bf16", "train": False},
        # a ragged batch of an odd width
        {"name": "norm_odd", "op": "norm", "rows": 1000, "cols": 257, "type": "f32", "train": True},
        # the 512-row batch of the three-layer MLP
        {"name": "norm_batch", "op": "norm", "rows": 512, "cols": 1024, "type": "f32", "train": True},
        # a training step's tokens at the wide MLP's width
        {"name": "norm_wide", "op": "norm", "rows": 8192, "cols": 4096, "type": "bf16", "train": True},
        # one token through the gated layer: the weights' bytes
        {"name": "gated_one_token", "op": "gated", "tokens": 1, "d": 4096, "f": 8192, "type": "bf16", "act": "silu",
         "bias": False, "transpose_w": False, "train": False},
        # a small ragged batch on full-precision weights stored [out, in]
        {"name": "gated_small_f32", "op": "gated", "tokens": 33, "d": 784, "f": 1000, "type": "f32", "act": "gelu",
         "bias": True, "transpose_w": True, "train": True},
        # the 512-row batch in full precision
        {"name": "gated_batch_f32", "op": "gated", "tokens": 512, "d": 1024, "f": 4096, "type": "f32", "act": "silu",
         "bias": True, "transpose_w": False, "train": True},
        # ragged tokens and an odd inner width, whose rows start off 16-byte boundaries
        {"name": "gated_odd_bf16", "op": "gated", "tokens": 1000, "d": 1000, "f": 2731, "type": "bf16",
         "act": "gelu_tanh", "bias": True, "transpose_w": False, "train": True},
        # a training step's tokens at the wide MLP's width: the matrix products' rate
        {"name": "gated_wide_bf16", "op": "gated", "tokens": 8192, "d": 4096, "f": 8192, "type": "bf16", "act": "silu",
         "bias": False, "transpose_w": False, "train": True},
        # the tensors of the 784-256-10 MLP: one small launch
        {"name": "adamw_small", "op": "adamw", "kind": "mlp", "d": 784, "f": 256, "layers": 1, "out": 10, "bits": 32,
         "grad": "f32"},
        # the tensors of the wide MLP
        {"name": "adamw_wide", "op": "adamw", "kind": "mlp", "d": 4096, "f": 4096, "layers": 3, "out": 1000, "bits": 32,
         "grad": "f32"},
        # two gated blocks trained in bf16: 8-bit states, and the bf16 copy that the next step's products read
        {"name": "adamw_blocks_8bit", "op": "adamw", "kind": "block", "d": 4096, "f": 8192, "layers": 2, "out": 0,
         "bits": 8, "grad": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "gated", "adamw"))
    if op == "norm":
        cols = _log(rng, 8, 8192)
        return {"op": op, "rows": _log(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols,
                "type": rng.choice(("f32", "bf16")), "train": rng.random() < 0.8}
    if op == "gated":
        return {"op": op, "tokens": _log(rng, 1, 8192), "d": _log(rng, 32, 4096), "f": _log(rng, 32, 8192),
                "type": rng.choice(("f32", "bf16", "bf16")), "act": rng.choice(ACTS), "bias": rng.random() < 0.5,
                "transpose_w": rng.random() < 0.5, "train": rng.random() < 0.75}
    if rng.random() < 0.5:
        return {"op": op, "kind": "mlp", "d": _log(rng, 16, 4096), "f": _log(rng, 16, 4096),
                "layers": rng.randint(1, 6), "out": _log(rng, 10, 1000), "bits": rng.choice((8, 32)),
                "grad": rng.choice(("f32", "bf16"))}
    return {"op": op, "kind": "block", "d": _log(rng, 64, 4096), "f": _log(rng, 64, 8192), "layers": rng.randint(1, 2),
            "out": 0, "bits": rng.choice((8, 32)), "grad": rng.choice(("f32", "bf16"))}


def _shapes(case):
    """The tensors that an AdamW case updates."""
    if case["kind"] == "mlp":
        dims = [case["d"]] + [case["f"]] * case["layers"] + [case["out"]]
        return [s for a, b in zip(dims, dims[1:]) for s in ((a, b), (b,))]
    d, f = case["d"], case["f"]
    return [(d,), (d,), (d, 2 * f), (f, d)] * case["layers"]


def _offsets(case):
    """Each tensor's first element in the flat buffers, and their length: every tensor starts on a block of its own."""
    at, offs = 0, []
    for s in _shapes(case):
        offs.append(at)
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return offs, at


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    if case["op"] == "norm":
        t, r, c = TYPES[case["type"]], case["rows"], case["cols"]
        # the residual stream: rows of different size, with an offset
        size = torch.rand(r, 1, device="cuda", generator=gen) * 4 + 0.1
        x = (randn(r, c) * size + randn(r, 1)).to(t)
        return {"case": dict(case), "x": x, "dy": randn(r, c, scale=0.1, dtype=t), "weight": 1 + randn(c, scale=0.2),
                "bias": randn(c, scale=0.2)}
    if case["op"] == "gated":
        t, m, d, f = TYPES[case["type"]], case["tokens"], case["d"], case["f"]
        shape = (2 * f, d) if case["transpose_w"] else (d, 2 * f)
        return {"case": dict(case), "x": randn(m, d, dtype=t), "w": randn(*shape, scale=d ** -0.5, dtype=t),
                "bias": randn(2 * f, scale=0.1, dtype=t) if case["bias"] else None,
                "dh": randn(m, f, scale=0.1, dtype=t)}
    offs, n = _offsets(case)
    live = torch.zeros(n, device="cuda", dtype=torch.bool)
    for o, s in zip(offs, _shapes(case)):
        live[o:o + math.prod(s)] = True
    zero = torch.zeros((), device="cuda")

    def flat(scale):  # zero between the tensors
        return torch.where(live, randn(n, scale=scale), zero)

    # the middle of a run: gradients of different size along each tensor, moments that have met such gradients
    size = torch.exp(randn(n // BLOCK, 1, scale=0.5)).expand(-1, BLOCK).reshape(-1)
    st = {"case": dict(case), "step": 100, "p": flat(0.02), "g": (flat(1e-3) * size).to(TYPES[case["grad"]]),
          "copy": torch.zeros(n, device="cuda", dtype=torch.bfloat16) if case["kind"] == "block" else None}
    m, v = flat(3e-4) * size, (flat(1e-3) * size).square() + torch.where(live, size.square() * 1e-8, zero)
    if case["bits"] == 32:
        return {**st, "m": m, "v": v}
    st["m"], st["m_scale"] = _encode(m)
    st["v"], st["v_scale"] = _encode(v.sqrt())
    return st


def _encode(x):
    """8-bit floating-point values (4 exponent bits, 3 of mantissa) and one power of two for each block, which takes
    the block's largest value into [128, 256).  A value above zero stays above zero."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -119)
    scale = (top.view(torch.int32) & 0x7F800000).view(torch.float32) * 2.0 ** -7
    y = x / scale
    y = torch.where((y > 0) & (y < 2.0 ** -9), 2.0 ** -9, y)
    y = torch.where((y < 0) & (y > -(2.0 ** -9)), -(2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _decode(q, scale):
    return (q.float().view(-1, BLOCK) * scale.view(-1, 1)).view(-1)


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    if name == "relu":
        return torch.where(g > 0, g, 0.0), (g > 0).to(g.dtype)
    s = 1 / (1 + torch.exp(-g))
    return s, s * (1 - s)


def run(state):
    return {"norm": _norm, "gated": _gated, "adamw": _adamw}[state["case"]["op"]](state)


def _norm(st):
    x, w, b, dy, train = st["x"], st["weight"], st["bias"], st["dy"], st["case"]["train"]
    if own:
        from moonxi_net_b200 import ops
        if not train:
            return {"y": ops.layer_norm(x, w, b, EPS)[0]}
        y, mean, rstd = ops.layer_norm(x, w, b, EPS, stats=True)
        dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    t = x.dtype
    x = x.float()
    mean = x.mean(1, keepdim=True)
    x = x - mean
    rstd = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    xhat = x * rstd
    y = (xhat * w + b).to(t)
    if not train:
        return {"y": y}
    dy = dy.float()
    dxhat = dy * w
    dx = rstd * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(t), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _gated(st):
    c, x, w, bias, dh = st["case"], st["x"], st["w"], st["bias"], st["dh"]
    tw = c["transpose_w"]
    if own:
        from moonxi_net_b200 import ops
        if not c["train"]:
            return {"h": ops.gated_linear(x, w, bias, act=c["act"], transpose_w=tw)[0]}
        h, pre = ops.gated_linear(x, w, bias, act=c["act"], transpose_w=tw, save=True)
        dx, dw, db = ops.gated_linear_backward(dh, pre, x, w, act=c["act"], transpose_w=tw, want_bias=bias is not None)
        return {"h": h, "dx": dx, "dw": dw, "dbias": db}
    t, f = x.dtype, c["f"]
    x, w = x.float(), w.float()
    w = w.t() if tw else w
    pre = x @ w
    if bias is not None:
        pre = pre + bias.float()
    g, u = pre[:, :f], pre[:, f:]
    a, da = _act(c["act"], g)
    h = (a * u).to(t)
    if not c["train"]:
        return {"h": h}
    dh = dh.float()
    dpre = torch.cat((dh * u * da, dh * a), 1)
    dx = (dpre @ w.t()).to(t)
    dw = (dpre.t() @ x if tw else x.t() @ dpre).to(t)
    return {"h": h, "dx": dx, "dw": dw, "dbias": dpre.sum(0).to(t) if bias is not None else None}


def _adamw(st):
    c = st["case"]
    keys = ("p", "m", "v", "copy") if c["bits"] == 32 else ("p", "m", "m_scale", "v", "v_scale", "copy")
    if own:
        if "opt" not in st:
            st["opt"], st["grads"] = _optimizer(st)
        st["opt"].step(st["grads"])
        return {k: st[k] for k in keys}
    st["step"] += 1
    p, g = st["p"], st["g"].float()
    m = st["m"] if c["bits"] == 32 else _decode(st["m"], st["m_scale"])
    v = st["v"] if c["bits"] == 32 else _decode(st["v"], st["v_scale"]).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = torch.sqrt(v)
    denom = root * (1 / math.sqrt(1 - BETA2 ** st["step"])) + ADAM_EPS
    p.copy_(p * (1 - LR * DECAY) - (m * (LR / (1 - BETA1 ** st["step"]))) / denom)
    if c["bits"] == 32:
        st["m"].copy_(m)
        st["v"].copy_(v)
    else:
        for key, x in (("m", m), ("v", root)):
            q, scale = _encode(x)
            st[key].copy_(q)
            st[key + "_scale"].copy_(scale)
    if st["copy"] is not None:
        st["copy"].copy_(p)
    return {k: st[k] for k in keys}


def _optimizer(st):
    """The optimizer over the case's tensors, on the moments that the state holds, and the tensors' gradients."""
    from moonxi_net_b200 import nn
    c = st["case"]
    offs, _ = _offsets(c)

    def views(buf, per=1):
        return [buf[o // per:o // per + -(-math.prod(s) // per)] for o, s in zip(offs, _shapes(c))]

    m, v = views(st["m"]), views(st["v"])
    if c["bits"] == 8:
        state = list(zip(m, views(st["m_scale"], BLOCK), v, views(st["v_scale"], BLOCK)))
    else:
        state = list(zip(m, v))
    opt = nn.AdamW(views(st["p"]), lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=c["bits"],
                   copies=None if st["copy"] is None else views(st["copy"]), state=state, step_count=st["step"])
    return opt, views(st["g"])


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["cols"], 4 if case["type"] == "f32" else 2
        w = 4 * case["cols"]
        # forward: x in, y out; backward: x and dy in, dx out, one row of each gradient
        return {"bytes": n * b * (5 if case["train"] else 2) + w * (5 if case["train"] else 2),
                "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "gated":
        m, d, f, b = case["tokens"], case["d"], case["f"], 4 if case["type"] == "f32" else 2
        x, w, h, bias = m * d * b, 2 * d * f * b, m * f * b, 2 * f * b if case["bias"] else 0
        if not case["train"]:
            return {"bytes": x + w + h + bias, "flops": 4 * m * d * f}
        return {"bytes": 2 * x + 2 * w + 2 * h + 2 * bias, "flops": 12 * m * d * f}
    n = sum(math.prod(s) for s in _shapes(case))
    per = 8 + (4 if case["grad"] == "f32" else 2) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    return {"bytes": n * (per + (2 if case["kind"] == "block" else 0)), "flops": 15 * n}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        x, dy, w, b = (st[k].double() for k in ("x", "dy", "weight", "bias"))
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / (var + EPS).sqrt() * w + b
        if not case["train"]:
            return {"y": y.detach()}
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "gated":
        x, w, dh = (st[k].double().requires_grad_(k != "dh") for k in ("x", "w", "dh"))
        bias = torch.zeros(2 * case["f"], device="cuda") if st["bias"] is None else st["bias"]
        bias = bias.double().requires_grad_(True)
        gate, up = torch.addmm(bias, x, w.t() if case["transpose_w"] else w).chunk(2, 1)
        fn = torch.nn.functional
        act = {"silu": fn.silu, "gelu": fn.gelu, "gelu_tanh": lambda z: fn.gelu(z, approximate="tanh"),
               "relu": fn.relu, "sigmoid": torch.sigmoid}[case["act"]]
        h = act(gate) * up
        if not case["train"]:
            return {"h": h.detach()}
        dx, dw, db = torch.autograd.grad(h, (x, w, bias), dh)
        return {"h": h.detach(), "dx": dx, "dw": dw, "dbias": db if case["bias"] else None}
    t = st["step"] + 1
    p, g, m, v = (st[k].double() for k in ("p", "g", "m", "v"))
    if case["bits"] == 8:
        m = m * st["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * st["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m, v = torch.lerp(g, m, BETA1), torch.lerp(g ** 2, v, BETA2)
    p = p - LR * DECAY * p
    p = p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    copy = p if case["kind"] == "block" else None
    if case["bits"] == 32:
        return {"p": p, "m": m, "v": v, "copy": copy}
    # which of two neighbours an 8-bit value or a scale becomes is decided in 32 bits: no value in 64
    return {"p": p, "m": None, "m_scale": None, "v": None, "v_scale": None, "copy": copy}
