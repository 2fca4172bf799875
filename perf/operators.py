"""The operators of a transformer's dense layers, as calls to measure.

Four operators: a linear layer with its bias, activation and residual, its
backward pass, a gated feed-forward block's two projections with the
activation and the product, and its backward pass.

    linear            z = x W^T + b,  y = act(z) + r
    linear_backward   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum of dz's rows
    gated             g = x Wg^T,  u = x Wu^T,  h = act(g) u
    gated_backward    dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x

With ``own`` false :func:`run` computes them from elementary torch operations
in 32 bits; with ``own`` true it calls ``eas.ops``.
"""

import math

import torch

own = False

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MOST_FLOPS = 2.0 * 8192 ** 3


def _case(op, dtype, m, n, k, act, **more):
    """One case: m tokens, n outputs (of each projection, for a gated block), k inputs."""
    case = {"op": op, "dtype": dtype, "m": m, "n": n, "k": k, "act": act, "pad": 0}
    if op == "linear":
        case.update(bias=False, residual=False, save=False)
    elif op == "linear_backward":
        case.update(bias=False)
    elif op == "gated":
        case.update(save=False)
    case.update(more)
    return case


def listed():
    cases = {
        # one token through a projection with a bias: the smallest call of a decoding step
        "linear_token": _case("linear", "f16", 1, 4096, 4096, "none", bias=True),
        # a batch of sequences, one token each, back onto the residual stream
        "linear_tokens": _case("linear", "bf16", 24, 4096, 8192, "none", residual=True),
        # a ragged batch whose rows start on no 16-byte boundary, everything in the epilogue
        "linear_unaligned": _case("linear", "f16", 1031, 1001, 1044, "gelu", bias=True, residual=True),
        # a long prompt or a training batch through a wide layer, forward
        "linear_prompt": _case("linear", "bf16", 8192, 8192, 8192, "gelu_tanh", bias=True),
        # a training step's backward pass of a layer with an activation
        "linear_train": _case("linear_backward", "bf16", 4096, 8192, 4096, "gelu", bias=True),
        # the same of a small layer on a ragged batch, without an activation
        "linear_train_ragged": _case("linear_backward", "f16", 777, 1000, 2088, "none", bias=True),
        # one token through a gated block
        "gated_token": _case("gated", "f16", 1, 8192, 4096, "silu"),
        # 64 sequences decoded together
        "gated_tokens": _case("gated", "bf16", 64, 8192, 4096, "silu"),
        # a long prompt
        "gated_prompt": _case("gated", "bf16", 8192, 8192, 4096, "silu"),
        # a training step's forward pass, with what the backward pass needs stored; inputs that
        # are columns of a wider tensor
        "gated_save_ragged": _case("gated", "f16", 1500, 2731, 1024, "gelu_tanh", save=True, pad=1024),
        # a training step's backward pass
        "gated_train": _case("gated_backward", "bf16", 4096, 8192, 4096, "silu"),
        # the same of a small block on a ragged batch
        "gated_train_ragged": _case("gated_backward", "f16", 613, 1375, 512, "gelu"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        step = rng.choice((1, 8, 8, 64, 128))
        return max(1, v) if v < step else v - v % step

    op = rng.choice(("linear", "linear", "linear_backward", "gated", "gated", "gated_backward"))
    n, k = size(64, 8192), size(64, 8192)
    per_token = {"linear": 2.0, "linear_backward": 4.0, "gated": 4.0, "gated_backward": 8.0}[op] * n * k
    m = size(1, 8192)
    m = max(1, min(m, int(MOST_FLOPS / per_token)))
    case = _case(op, rng.choice(("f16", "bf16")), m, n, k, rng.choice(ACTS[1:] if "gated" in op else ACTS),
                 pad=rng.choice((0, 0, 8, 64, 3)))
    for flag in ("bias", "residual", "save"):
        if flag in case:
            case[flag] = rng.random() < 0.5
    return case


def _pairs(op):
    return 2 if op.startswith("gated") else 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    m, n, k = case["m"], case["n"], case["k"]
    pad = case["pad"]

    def normal(rows, cols, scale, wider=0):
        t = torch.randn(rows, cols + wider, device="cuda", generator=gen).mul_(scale).to(dtype)
        return t[:, :cols]

    def empty(rows, cols):
        return torch.empty(rows, cols, device="cuda", dtype=dtype)

    op = case["op"]
    state = {"op": op, "act": case["act"], "x": normal(m, k, 1.0, pad)}
    state["w"] = [normal(n, k, k ** -0.5) for _ in range(_pairs(op))]
    if op == "linear":
        state["bias"] = normal(1, n, 0.5)[0] if case["bias"] else None
        state["residual"] = normal(m, n, 1.0) if case["residual"] else None
        state["y"] = empty(m, n)
        state["pre"] = empty(m, n) if case["save"] else None
    elif op == "gated":
        state["y"] = empty(m, n)
        state["pre"] = [empty(m, n), empty(m, n)] if case["save"] else [None, None]
    else:
        state["dy"] = normal(m, n, 0.1)
        state["pre"] = [normal(m, n, 1.0) for _ in range(_pairs(op))]
        state["dx"] = empty(m, k)
        state["dw"] = [empty(n, k) for _ in range(_pairs(op))]
        if op == "linear_backward":
            state["db"] = torch.empty(n, device="cuda", dtype=dtype) if case["bias"] else None
    return state


def _act(name, z):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return z


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if name in ("silu", "sigmoid"):
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s)) if name == "silu" else s * (1.0 - s)
    return torch.ones_like(z)


def _own(s):
    import eas

    op, act = s["op"], s["act"]
    if op == "linear":
        eas.ops.linear(s["x"], s["w"][0], s["y"], bias=s["bias"], residual=s["residual"], act=act, pre=s["pre"],
                       _sync=False)
        return {"y": s["y"]} if s["pre"] is None else {"y": s["y"], "pre": s["pre"]}
    if op == "gated":
        gate, up = s["pre"]
        eas.ops.gated(s["x"], s["w"][0], s["w"][1], s["y"], act=act, gate=gate, up=up, _sync=False)
        return {"h": s["y"]} if gate is None else {"h": s["y"], "gate": gate, "up": up}
    if op == "linear_backward":
        eas.ops.linear_backward(s["dy"], s["x"], s["w"][0], dx=s["dx"], dw=s["dw"][0], dbias=s["db"], act=act,
                                pre=s["pre"][0], _sync=False)
        out = {"dx": s["dx"], "dw": s["dw"][0]}
        return out if s["db"] is None else dict(out, db=s["db"])
    eas.ops.gated_backward(s["dy"], s["x"], s["w"][0], s["w"][1], s["pre"][0], s["pre"][1], dx=s["dx"],
                           dw_gate=s["dw"][0], dw_up=s["dw"][1], act=act, _sync=False)
    return {"dx": s["dx"], "dw_gate": s["dw"][0], "dw_up": s["dw"][1]}


def run(state):
    if own:
        return _own(state)
    op, act, dtype = state["op"], state["act"], state["x"].dtype
    x = state["x"].float()
    w = [t.float() for t in state["w"]]
    if op == "linear":
        z = x @ w[0].T
        if state["bias"] is not None:
            z = z + state["bias"].float()
        y = _act(act, z)
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return {"y": y.to(dtype)} if state["pre"] is None else {"y": y.to(dtype), "pre": z.to(dtype)}
    if op == "gated":
        g, u = x @ w[0].T, x @ w[1].T
        h = (_act(act, g) * u).to(dtype)
        return {"h": h} if state["pre"][0] is None else {"h": h, "gate": g.to(dtype), "up": u.to(dtype)}
    dy = state["dy"].float()
    z = state["pre"][0].float()
    if op == "linear_backward":
        dz = dy * _act_grad(act, z)
        out = {"dx": (dz @ w[0]).to(dtype), "dw": (dz.T @ x).to(dtype)}
        return out if state["db"] is None else dict(out, db=dz.sum(0).to(dtype))
    dg = dy * state["pre"][1].float() * _act_grad(act, z)
    du = dy * _act(act, z)
    return {"dx": (dg @ w[0] + du @ w[1]).to(dtype), "dw_gate": (dg.T @ x).to(dtype), "dw_up": (du.T @ x).to(dtype)}


def work(case):
    m, n, k = case["m"], case["n"], case["k"]
    op = case["op"]
    if op == "linear":
        numbers = m * k + n * k + m * n * (1 + case["residual"] + case["save"]) + n * case["bias"]
        return {"bytes": 2 * numbers, "flops": 2 * m * n * k}
    if op == "gated":
        return {"bytes": 2 * (m * k + 2 * n * k + m * n * (3 if case["save"] else 1)), "flops": 4 * m * n * k}
    if op == "linear_backward":
        saved = 0 if case["act"] == "none" else m * n
        return {"bytes": 2 * (m * n + saved + 2 * m * k + 2 * n * k + n * case["bias"]), "flops": 4 * m * n * k}
    return {"bytes": 2 * (3 * m * n + 2 * m * k + 4 * n * k), "flops": 8 * m * n * k}


def exact(case, seed):
    """The definitions in 64 bits; derivatives by what the functions are made of, not by run's formulas."""
    s = prepare(case, seed)
    double = {key: s[key].double() for key in ("x", "dy") if key in s}
    x, w = double["x"], [t.double() for t in s["w"]]

    def phi(z):  # the normal distribution's density
        return torch.exp(-z.square() / 2) / (2 * math.pi) ** 0.5

    def value_and_slope(z):
        name = case["act"]
        if name == "none":
            return z, torch.ones_like(z)
        if name == "relu":
            return z.clamp(min=0), torch.sign(z).clamp(min=0)
        if name == "gelu":
            cdf = torch.erfc(-z / 2 ** 0.5) / 2
            return z * cdf, cdf + z * phi(z)
        if name == "gelu_tanh":  # 1/2 (1 + tanh q) is the logistic function of 2 q
            q = (z + 0.044715 * z ** 3) * (8 / math.pi) ** 0.5
            p = torch.sigmoid(q)
            return z * p, p + z * p * torch.sigmoid(-q) * (1 + 0.134145 * z.square()) * (8 / math.pi) ** 0.5
        p, rest = torch.sigmoid(z), torch.sigmoid(-z)
        return (z * p, p + z * p * rest) if name == "silu" else (p, p * rest)

    op = case["op"]
    if op == "linear":
        z = torch.einsum("mk,nk->mn", x, w[0])
        if s["bias"] is not None:
            z += s["bias"].double()[None]
        y = value_and_slope(z)[0]
        if s["residual"] is not None:
            y = s["residual"].double() + y
        return {"y": y, "pre": z} if case["save"] else {"y": y}
    if op == "gated":
        g, u = (torch.einsum("mk,nk->mn", x, t) for t in w)
        h = u * value_and_slope(g)[0]
        return {"h": h, "gate": g, "up": u} if case["save"] else {"h": h}
    value, slope = value_and_slope(s["pre"][0].double())
    if op == "linear_backward":
        dz = slope * double["dy"]
        out = {"dx": torch.einsum("mn,nk->mk", dz, w[0]), "dw": torch.einsum("mn,mk->nk", dz, x)}
        return dict(out, db=torch.einsum("mn->n", dz)) if case["bias"] else out
    du = value * double["dy"]
    dg = slope * double["dy"] * s["pre"][1].double()
    dx = torch.einsum("mn,nk->mk", dg, w[0])
    dx += torch.einsum("mn,nk->mk", du, w[1])
    return {"dx": dx, "dw_gate": torch.einsum("mn,mk->nk", dg, x), "dw_up": torch.einsum("mn,mk->nk", du, x)}
