"""The dense operators of ``eas.ops`` in 64 bits, from their definitions, with the error that each result may have.

Error model of one result, elementwise (u = half a step of the 16-bit type, relative):

* a sum of K products in f32 is off by at most g(K) S, with S the sum of the absolute products and g(K) = (K + 16) 2^-24
  (a chain of K roundings to nearest; the matrix instructions round once per 16 products and so stay below it);
* an activation is a function with |slope| <= 1.13, evaluated with a relative error of at most 2^-15: its exponential is
  off by 2 + 1.17 |z| units of 2^-24 where it matters (|z| < 100);
* rounding to the type: u |value|, or half the smallest subnormal.
"""

import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -120}
SLOPE = 1.13
EVAL = 2.0 ** -15


def gamma(k):
    return (k + 16) * 2.0 ** -24


def act(name, z):
    """(act(z), act'(z)) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s, r = torch.sigmoid(c * (z + 0.044715 * z ** 3)), torch.sigmoid(-c * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * r * c * (1 + 3 * 0.044715 * z * z)
    s, r = torch.sigmoid(z), torch.sigmoid(-z)
    if name == "silu":
        return z * s, s + z * s * r
    if name == "sigmoid":
        return s, s * r
    raise ValueError(name)


def rounded(value, err, dtype):
    """(value, allowed error) of a result that is off by ``err`` before its rounding."""
    return value, err + U[dtype] * (value.abs() + err) + TINY[dtype]


def _product(a, b):
    """a b^T, and its error in f32."""
    return a @ b.T, gamma(a.shape[1]) * (a.abs() @ b.abs().T)


def linear(x, w, bias=None, residual=None, name="none"):
    """{"y": (value, error), "pre": ...} before rounding to 16 bits is added (see ``rounded``)."""
    dt = x.dtype
    z, ez = _product(x.double(), w.double())
    if bias is not None:
        z = z + bias.double()
        ez = ez + 2.0 ** -23 * (z.abs() + bias.double().abs())
    y, _ = act(name, z)
    ey = SLOPE * ez + (EVAL * y.abs() if name != "none" else 0)
    if residual is not None:
        y = y + residual.double()
        ey = ey + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return {"y": rounded(y, ey, dt), "pre": rounded(z, ez, dt)}


def gated(x, wg, wu, name="silu"):
    dt = x.dtype
    g, eg = _product(x.double(), wg.double())
    u, eu = _product(x.double(), wu.double())
    a, _ = act(name, g)
    ea = SLOPE * eg + EVAL * a.abs()
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + 2.0 ** -23 * h.abs()
    return {"h": rounded(h, eh, dt), "gate": rounded(g, eg, dt), "up": rounded(u, eu, dt)}


def _grads(dzs, ws, x, dt):
    """dx and the dW of dz given as (value, error before its own rounding to 16 bits)."""
    x = x.double()
    out, dx, edx = [], 0, 0
    for (dz, e), w in zip(dzs, ws):
        dz, e = rounded(dz, e, dt)
        w = w.double()
        big = dz.abs() + e
        dx = dx + dz @ w
        edx = edx + e @ w.abs() + gamma(2 * dz.shape[1]) * (big @ w.abs())
        out.append(rounded(dz.T @ x, e.T @ x.abs() + gamma(dz.shape[0]) * (big.T @ x.abs()), dt))
    return rounded(dx, edx, dt), out


def linear_backward(dy, x, w, pre=None, name="none"):
    dt = x.dtype
    dz = dy.double()
    e = torch.zeros_like(dz)
    if name != "none":
        dz = dz * act(name, pre.double())[1]
    if name not in ("none", "relu"):
        # the slope is a sum of terms that can cancel: its error is relative to them, 1 + |z| at most
        e = EVAL * dy.double().abs() * (1 + pre.double().abs().clamp(max=8))
    db = rounded(dz.sum(0), (e + gamma(dz.shape[0]) * dz.abs()).sum(0), dt)
    dx, (dw,) = _grads([(dz, e)], [w], x, dt)
    return {"dx": dx, "dw": dw, "dbias": db}


def gated_backward(dh, x, wg, wu, gate, up, name="silu"):
    dt = x.dtype
    dh, g, u = dh.double(), gate.double(), up.double()
    v, d = act(name, g)
    dg, du = dh * u * d, dh * v
    eg = EVAL * dh.abs() * u.abs() * (1 + g.abs().clamp(max=8))
    eu = EVAL * dh.abs() * v.abs()
    dx, (dwg, dwu) = _grads([(dg, eg), (du, eu)], [wg, wu], x, dt)
    return {"dx": dx, "dw_gate": dwg, "dw_up": dwu}


def check(got, want, what=""):
    value, tol = want
    off = (got.double() - value).abs()
    bad = ~(off <= tol)
    if bool(bad.any()):
        i = int(torch.where(bad.reshape(-1), off.reshape(-1) / tol.reshape(-1).clamp(min=1e-300), 0).argmax())
        at = tuple(int(v) for v in torch.unravel_index(torch.tensor(i), value.shape))
        raise AssertionError(f"{what}: {int(bad.sum())} of {value.numel()} values are off; worst at {at}: got "
                             f"{float(got[at])}, expected {float(value[at])} +- {float(tol[at])}")
