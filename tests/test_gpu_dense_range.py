"""GPU: gradients whose inner values (dz, dg, du) leave f16's range, or its full precision, while the results do not.

Powers of two leave sparse integers exact at every step, so those results must be equal (and are chosen to be values of f16 themselves).  Other values are compared with the
definition in 64 bits: an inner value is rounded at a power-of-two scale 2^e that brings the largest of them below 2^15, so it
is off by at most 2^-11 of itself or half the smallest subnormal, 2^-25, at that scale."""

import math

import pytest
import torch

import dense_oracle as oracle
import eas

pytestmark = pytest.mark.gpu

F16 = torch.float16
# both kernels of few rows' gradients, single-CTA tiles whole and split, pairs; even and odd widths
SHAPES = [(1, 8, 8), (3, 5, 7), (5, 264, 40), (64, 136, 200), (300, 520, 264), (613, 1375, 512), (40, 72, 16400),
          (1024, 1536, 320), (2304, 2080, 136), (8000, 600, 2000)]


@pytest.fixture(autouse=True)
def _ready(cuda_rt):
    yield
    cuda_rt.synchronize()
    torch.cuda.synchronize()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def sparse(g, rows, cols, per_row, scale=1.0):
    p = min(1.0, per_row / max(cols, 1))
    v = torch.randint(0, 2, (rows, cols), device="cuda", generator=g) * 2.0 - 1
    return (v * (torch.rand(rows, cols, device="cuda", generator=g) < p) * scale).half()


def normal(g, rows, cols, scale=1.0):
    return (torch.randn(rows, cols, device="cuda", generator=g) * scale).half()


def gated_backward(dh, x, wg, wu, gate, up, act):
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    eas.ops.gated_backward(dh, x, wg, wu, gate, up, dx=dx, dw_gate=dwg, dw_up=dwu, act=act)
    alone = torch.empty_like(wu)
    eas.ops.gated_backward(dh, x, wg, wu, gate, up, dw_up=alone, act=act)
    assert torch.equal(alone.view(torch.int16), dwu.view(torch.int16))
    return dx, dwg, dwu


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dh_log,up_log,w_log,x_log", [(0, 0, 0, 0), (-12, -12, 12, 12), (9, 9, -12, -12), (-24, 2, 8, 8),
                                                       (15, 15, -20, -20)])
def test_gated_exact_at_any_scale(shape, dh_log, up_log, w_log, x_log):
    """Inner values of 2^(dh_log + up_log): far below and above what f16 holds."""
    m, n, k = shape
    g = gen(m + n + k)
    dh, up, gate = sparse(g, m, n, 5, 2.0 ** dh_log), sparse(g, m, n, n, 2.0 ** up_log), sparse(g, m, n, n // 2 + 1, 2.0 ** up_log)
    x, wg, wu = sparse(g, m, k, 6, 2.0 ** x_log), sparse(g, n, k, 6, 2.0 ** w_log), sparse(g, n, k, 6, 2.0 ** w_log)
    dg, du = dh.double() * up.double() * (gate.double() > 0), dh.double() * gate.double().clamp(min=0)
    want = dg @ wg.double() + du @ wu.double(), dg.T @ x.double(), du.T @ x.double()
    for got, v in zip(gated_backward(dh, x, wg, wu, gate, up, "relu"), want):
        assert torch.equal(v.half().double(), v)      # the results are values of f16
        assert torch.equal(got.double(), v)


def exponent(*inner):
    """e of the scale 2^e for inner values that need one."""
    top = max(float(v[v.isfinite()].abs().max()) for v in inner)
    return 14 - math.floor(math.log2(top))


def backward_oracle(dzs, ws, x, e):
    """dx and the dW with their errors (see dense_oracle), for inner values (value, error) rounded at scale 2^e."""
    x = x.double()
    dx, edx, out = 0, 0, []
    for (dz, err), w in zip(dzs, ws):
        err = err + oracle.U[F16] * (dz.abs() + err) + 2.0 ** (-25 - e)
        big = dz.abs() + err
        dx = dx + dz @ w.double()
        edx = edx + err @ w.double().abs() + oracle.gamma(2 * dz.shape[1]) * (big @ w.double().abs())
        out.append(oracle.rounded(dz.T @ x, err.T @ x.abs() + oracle.gamma(dz.shape[0]) * (big.T @ x.abs()), F16))
    return oracle.rounded(dx, edx, F16), out


def inner_of_gated(dh, gate, up, act):
    d64, g64, u64 = dh.double(), gate.double(), up.double()
    v, d = oracle.act(act, g64)
    dg, du = d64 * u64 * d, d64 * v
    return (dg, oracle.EVAL * d64.abs() * u64.abs() * (1 + g64.abs().clamp(max=8))), (du, oracle.EVAL * d64.abs() * v.abs())


@pytest.mark.parametrize("act", ["silu", "gelu", "none"])
@pytest.mark.parametrize("shape", [(64, 136, 200), (300, 521, 264), (613, 1375, 512)])
@pytest.mark.parametrize("dh_scale,up_scale,other", [(300.0, 300.0, 1e-4), (1e-5, 1.0, 1.0), (1e-3, 1e-3, 10.0)])
def test_gated_values_at_any_scale(shape, act, dh_scale, up_scale, other):
    m, n, k = shape
    g = gen(m + n + k)
    dh, up, gate = normal(g, m, n, dh_scale), normal(g, m, n, up_scale), normal(g, m, n)
    x, wg, wu = normal(g, m, k, other), normal(g, n, k, other), normal(g, n, k, other)
    dg, du = inner_of_gated(dh, gate, up, act)
    dx, dws = backward_oracle((dg, du), (wg, wu), x, exponent(dg[0], du[0]))
    got = gated_backward(dh, x, wg, wu, gate, up, act)
    assert all(v.isfinite().all() for v in got)
    for v, w, name in zip(got, (dx, *dws), ("dx", "dw_gate", "dw_up")):
        oracle.check(v, w, name)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("shape", [(5, 264, 40), (300, 521, 264), (1024, 1536, 320)])
@pytest.mark.parametrize("scale", [3e-8, 1e-5, 60000.0])
def test_linear_values_at_any_scale(shape, act, scale):
    """Gradients near f16's smallest and largest values: an activation's slope takes dz out of what it holds well."""
    m, n, k = shape
    g = gen(m + n + k)
    dy, pre = (torch.rand(m, n, device="cuda", generator=g) * scale).half(), normal(g, m, n, 2.0)
    x, w = normal(g, m, k, 100.0 if scale < 1 else 1e-4), normal(g, n, k, 10.0 if scale < 1 else 1e-4)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda", dtype=F16)
    eas.ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, act=act, pre=pre)
    dz = dy.double() * oracle.act(act, pre.double())[1]
    err = oracle.EVAL * dy.double().abs() * (1 + pre.double().abs().clamp(max=8))
    e = exponent(dz) if scale < 1 else min(exponent(dz), 0)     # large values keep scale 1 while they fit
    want_dx, (want_dw,) = backward_oracle([(dz, err)], [w], x, e)
    oracle.check(dx, want_dx, "dx")
    oracle.check(dw, want_dw, "dw")
    want, tol = oracle.rounded(dz.sum(0), (err + oracle.gamma(m) * dz.abs()).sum(0), F16)
    past = want - tol > 65520                  # dbias is a sum of such values itself, and may be past f16
    assert (db[past] == float("inf")).all()
    inside = want + tol < 65520
    oracle.check(db[inside], (want[inside], tol[inside]), "dbias")


def test_small_gradients_beside_large_ones():
    """A few rows far above the others: the others keep their precision."""
    m, n, k = 600, 520, 200
    g = gen(7)
    dh, up, gate = normal(g, m, n, 2.0 ** -18), normal(g, m, n), normal(g, m, n)
    dh[::100] = normal(g, m // 100, n, 0.05)
    x, wg, wu = normal(g, m, k), normal(g, n, k), normal(g, n, k)
    x[::100] = 0                      # those rows are in dx alone
    dg, du = inner_of_gated(dh, gate, up, "silu")
    dx, dws = backward_oracle((dg, du), (wg, wu), x, exponent(dg[0], du[0]))
    for v, w, name in zip(gated_backward(dh, x, wg, wu, gate, up, "silu"), (dx, *dws), ("dx", "dw_gate", "dw_up")):
        oracle.check(v, w, name)


@pytest.mark.parametrize("n", [520, 521])
def test_infinite_gradients_stay_where_they_are(n):
    """An infinity or a NaN reaches its own row of dx and its own outputs' rows of dW, and no scale is taken from it."""
    m, k = 200, 72
    g = gen(n)
    dh, up, gate = normal(g, m, n, 300.0), normal(g, m, n, 300.0), normal(g, m, n)
    x, wg, wu = normal(g, m, k, 1e-4), normal(g, n, k, 1e-4), normal(g, n, k, 1e-4)
    clean = gated_backward(dh, x, wg, wu, gate, up, "silu")
    bad = dh.clone()
    bad[3, 17], bad[90, 400] = float("inf"), float("nan")
    dx, dwg, dwu = gated_backward(bad, x, wg, wu, gate, up, "silu")
    keep, cols = [i for i in range(m) if i not in (3, 90)], [i for i in range(n) if i not in (17, 400)]
    assert not dx[[3, 90]].isfinite().any() and torch.equal(dx[keep], clean[0][keep])
    for got, was in ((dwg, clean[1]), (dwu, clean[2])):
        assert not got[[17, 400]].isfinite().any()
        assert got[cols].isfinite().all()
    dh = torch.full_like(dh, float("inf"))
    assert not any(v.isfinite().any() for v in gated_backward(dh, x, wg, wu, gate, up, "silu"))


def test_no_gradient():
    m, n, k = 100, 264, 72
    g = gen(0)
    x, wg, wu, gate, up = normal(g, m, k), normal(g, n, k), normal(g, n, k), normal(g, m, n), normal(g, m, n)
    for v in gated_backward(torch.zeros(m, n, device="cuda", dtype=F16), x, wg, wu, gate, up, "gelu"):
        assert (v == 0).all()


@pytest.mark.parametrize("shape", [(64, 136, 200), (613, 1375, 512), (2304, 2080, 136)])
def test_each_replay_takes_its_own_scale(shape):
    """A captured call, replayed with gradients of other sizes, gives the bits of the same call made directly."""
    m, n, k = shape
    g = gen(m)
    up, gate = normal(g, m, n), normal(g, m, n)
    x, wg, wu = normal(g, m, k), normal(g, n, k), normal(g, n, k)
    dh = torch.empty(m, n, device="cuda", dtype=F16)
    outs = [torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)]

    def run():
        eas.ops.gated_backward(dh, x, wg, wu, gate, up, dx=outs[0], dw_gate=outs[1], dw_up=outs[2], _sync=False)

    dh.copy_(normal(g, m, n))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for scale in (1.0, 1e-6, 1e-3, 2e4, 1.0, 0.0):
        dh.copy_(normal(g, m, n, scale))
        run()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.nan_to_num(1e4), v.nan_to_num(1e4)) for o, v in zip(outs, want))


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
@pytest.mark.parametrize("m", [3, 200])
def test_pre_activations_past_f16(act, m):
    """A pre-activation of -70000 is stored as -inf: the layer's value is 0 (sigmoid's too), and so are the gradients
    through it; to the right the slope is 1 (sigmoid 0)."""
    n, k = 72, 40
    g = gen(m)
    x, w = torch.ones(m, k, device="cuda", dtype=F16), torch.zeros(n, k, device="cuda", dtype=F16)
    bias = normal(g, 1, n)[0]
    w[5, 0], w[5, 1], w[9, 0], w[9, 1] = -60000, -10000, 60000, 10000
    y, pre = torch.empty(m, n, device="cuda", dtype=F16), torch.empty(m, n, device="cuda", dtype=F16)
    eas.ops.linear(x, w, y, bias=bias, act=act, pre=pre)
    assert (pre[:, 5] == -float("inf")).all() and (pre[:, 9] == float("inf")).all() and (y[:, 5] == 0).all()
    dy = normal(g, m, n)
    db, dx, dw = torch.empty_like(bias), torch.empty_like(x), torch.empty_like(w)
    small = normal(g, n, k)
    eas.ops.linear_backward(dy, x, small, dx=dx, dw=dw, dbias=db, act=act, pre=pre)
    right = torch.zeros_like(db[9]) if act == "sigmoid" else dy[:, 9].double().sum().half()
    assert db[5] == 0 and abs(float(db[9]) - float(right)) <= 2.0 ** -10 * abs(float(right)) and db.isfinite().all()
    assert dx.isfinite().all() and dw.isfinite().all() and (dw[5] == 0).all()
    nan = pre.clone()
    nan[:, 5] = float("nan")
    eas.ops.linear_backward(dy, x, small, dbias=db, act=act, pre=nan)
    assert db[5].isnan() and int(db.isnan().sum()) == 1
    # gated: the gate's value is 0 there, whatever the up projection
    dg, du = torch.empty_like(small), torch.empty_like(small)
    gate, up = pre.clone(), normal(g, m, n)
    gate[:, 9] = 1
    eas.ops.gated_backward(dy, x, small, small, gate, up, dx=dx, dw_gate=dg, dw_up=du, act=act)
    assert dx.isfinite().all() and (dg[5] == 0).all() and (du[5] == 0).all()
