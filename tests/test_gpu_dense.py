"""GPU: eas.ops (linear, gated and their backward passes) against the definitions in 64 bits.

Two kinds of inputs: sparse small integers, whose every intermediate and result is exact in f32 and in the 16-bit type, so
the results must be equal whatever the order of the sums; and normal values, compared under the error model of
``dense_oracle``."""

import pytest
import torch

import dense_oracle as oracle
import eas
from dense_shapes import BIG, SHAPES, VARIANTS

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
ACTS = list(eas.ops.ACTIVATIONS)
EXACT = [(s, t) for s in SHAPES + BIG for t in TYPES] + [(s, TYPES[i % 2]) for i, s in enumerate(VARIANTS)]


@pytest.fixture(autouse=True)
def _ready(cuda_rt):
    yield
    torch.cuda.synchronize()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, rows, cols, dtype, scale=1.0, pad=0, front=0):
    """Normal values as ``cols`` columns of a matrix ``pad + front`` columns wider."""
    t = (torch.randn(rows, front + cols + pad, device="cuda", generator=g) * scale).to(dtype)
    return t[:, front:front + cols]


def sparse(g, rows, cols, dtype, per_row, pad=0):
    """-1, 0, 1 with about ``per_row`` nonzero values in a row."""
    p = min(1.0, per_row / max(cols, 1))
    v = torch.randint(0, 2, (rows, cols + pad), device="cuda", generator=g) * 2.0 - 1
    v = v * (torch.rand(rows, cols + pad, device="cuda", generator=g) < p)
    return v.to(dtype)[:, :cols]


class Guarded:
    """An output inside a larger buffer of a marker value, to see what is written around it."""

    MARK = 77.0

    def __init__(self, rows, cols, dtype, pad=0, front=0):
        self.whole = torch.full((rows + 2, front + cols + pad), self.MARK, device="cuda", dtype=dtype)
        self.t = self.whole[1:1 + rows, front:front + cols]
        self.rows, self.cols, self.front = rows, cols, front

    def intact(self):
        w = self.whole.clone()
        w[1:1 + self.rows, self.front:self.front + self.cols] = self.MARK
        return bool((w == self.MARK).all())


def vector(t):
    return t[0]


@pytest.mark.parametrize("shape,dtype", EXACT)
def test_linear_exact(shape, dtype):
    m, n, k = shape
    g = gen(m * 7 + n * 3 + k)
    x, w = sparse(g, m, k, dtype, 10), sparse(g, n, k, dtype, 10)
    bias, res = vector(sparse(g, 1, n, dtype, n)), sparse(g, m, n, dtype, n)
    z = x.double() @ w.double().T + bias.double()
    assert z.abs().max() <= 250
    y, pre = Guarded(m, n, dtype), Guarded(m, n, dtype)
    eas.ops.linear(x, w, y.t, bias=bias, residual=res, act="relu", pre=pre.t)
    assert torch.equal(pre.t.double(), z)
    assert torch.equal(y.t.double(), z.clamp(min=0) + res.double())
    assert y.intact() and pre.intact()
    plain = Guarded(m, n, dtype)
    eas.ops.linear(x, w, plain.t)
    assert torch.equal(plain.t.double(), x.double() @ w.double().T) and plain.intact()


@pytest.mark.parametrize("shape,dtype", EXACT)
def test_gated_exact(shape, dtype):
    m, n, k = shape
    gr = gen(m * 5 + n + k)
    x, wg, wu = sparse(gr, m, k, dtype, 6), sparse(gr, n, k, dtype, 6), sparse(gr, n, k, dtype, 6)
    gz, uz = x.double() @ wg.double().T, x.double() @ wu.double().T
    assert (gz * uz).abs().max() <= 250
    h, gate, up = Guarded(m, n, dtype), Guarded(m, n, dtype), Guarded(m, n, dtype)
    eas.ops.gated(x, wg, wu, h.t, act="relu", gate=gate.t, up=up.t)
    assert torch.equal(gate.t.double(), gz) and torch.equal(up.t.double(), uz)
    assert torch.equal(h.t.double(), gz.clamp(min=0) * uz)
    assert h.intact() and gate.intact() and up.intact()
    alone = Guarded(m, n, dtype)
    eas.ops.gated(x, wg, wu, alone.t, act="relu")
    assert torch.equal(alone.t, h.t) and alone.intact()


@pytest.mark.parametrize("shape,dtype", EXACT)
def test_linear_backward_exact(shape, dtype):
    m, n, k = shape
    g = gen(m + n * 11 + k)
    dy, x, w = sparse(g, m, n, dtype, 10), sparse(g, m, k, dtype, 10), sparse(g, n, k, dtype, 10)
    pre = normal(g, m, n, dtype)
    dz = dy.double() * (pre.double() > 0)
    want = {"dx": dz @ w.double(), "dw": dz.T @ x.double(), "dbias": dz.sum(0)}
    assert all(v.abs().max() <= 250 for v in want.values())
    dx, dw, db = Guarded(m, k, dtype), Guarded(n, k, dtype), Guarded(1, n, dtype)
    eas.ops.linear_backward(dy, x, w, dx=dx.t, dw=dw.t, dbias=db.t[0], act="relu", pre=pre)
    assert torch.equal(dx.t.double(), want["dx"])
    assert torch.equal(dw.t.double(), want["dw"])
    assert torch.equal(db.t[0].double(), want["dbias"])
    assert dx.intact() and dw.intact() and db.intact()
    # each output alone, without an activation
    dz = dy.double()
    dx, dw, db = Guarded(m, k, dtype), Guarded(n, k, dtype), Guarded(1, n, dtype)
    eas.ops.linear_backward(dy, x, w, dx=dx.t)
    eas.ops.linear_backward(dy, x, w, dw=dw.t)
    eas.ops.linear_backward(dy, x, w, dbias=db.t[0])
    assert torch.equal(dx.t.double(), dz @ w.double()) and dx.intact()
    assert torch.equal(dw.t.double(), dz.T @ x.double()) and dw.intact()
    assert torch.equal(db.t[0].double(), dz.sum(0)) and db.intact()


@pytest.mark.parametrize("shape,dtype", EXACT)
def test_gated_backward_exact(shape, dtype):
    m, n, k = shape
    g = gen(m + n + k * 13)
    dh, x = sparse(g, m, n, dtype, 5), sparse(g, m, k, dtype, 6)
    wg, wu = sparse(g, n, k, dtype, 6), sparse(g, n, k, dtype, 6)
    gate, up = sparse(g, m, n, dtype, n // 2 + 1), sparse(g, m, n, dtype, n)
    dg, du = dh.double() * up.double() * (gate.double() > 0), dh.double() * gate.double().clamp(min=0)
    want = {"dx": dg @ wg.double() + du @ wu.double(), "dw_gate": dg.T @ x.double(), "dw_up": du.T @ x.double()}
    assert all(v.abs().max() <= 250 for v in want.values())
    outs = {"dx": Guarded(m, k, dtype), "dw_gate": Guarded(n, k, dtype), "dw_up": Guarded(n, k, dtype)}
    eas.ops.gated_backward(dh, x, wg, wu, gate, up, act="relu", **{name: o.t for name, o in outs.items()})
    for name, o in outs.items():
        assert torch.equal(o.t.double(), want[name]), name
        assert o.intact(), name
    for name in outs:   # each output alone
        o = Guarded(*outs[name].t.shape, dtype)
        eas.ops.gated_backward(dh, x, wg, wu, gate, up, act="relu", **{name: o.t})
        assert torch.equal(o.t, outs[name].t) and o.intact(), name


NORMAL = [(1, 264, 520), (40, 72, 16400), (7, 130, 1044), (24, 520, 264), (130, 264, 1000), (300, 520, 200), (777, 1000, 264)]


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORMAL)
def test_values(shape, dtype, name):
    """Every activation, forward and backward, on normal values (the pre-activations reach +-4)."""
    m, n, k = shape
    g = gen(m + n + k)
    x, w, wu = normal(g, m, k, dtype), normal(g, n, k, dtype, k ** -0.5), normal(g, n, k, dtype, k ** -0.5)
    bias, res, dy = vector(normal(g, 1, n, dtype)), normal(g, m, n, dtype), normal(g, m, n, dtype, 0.1)
    y, pre, h, gate, up = (torch.empty(m, n, device="cuda", dtype=dtype) for _ in range(5))
    dx = torch.empty(m, k, device="cuda", dtype=dtype)
    dw, dw2 = torch.empty_like(w), torch.empty_like(w)
    db = torch.empty(n, device="cuda", dtype=dtype)

    eas.ops.linear(x, w, y, bias=bias, residual=res, act=name, pre=pre)
    want = oracle.linear(x, w, bias, res, name)
    oracle.check(y, want["y"], "y")
    oracle.check(pre, want["pre"], "pre")

    eas.ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, act=name, pre=pre)
    want = oracle.linear_backward(dy, x, w, pre, name)
    for got, key in ((dx, "dx"), (dw, "dw"), (db, "dbias")):
        oracle.check(got, want[key], key)

    eas.ops.gated(x, w, wu, h, act=name, gate=gate, up=up)
    want = oracle.gated(x, w, wu, name)
    for got, key in ((h, "h"), (gate, "gate"), (up, "up")):
        oracle.check(got, want[key], key)

    eas.ops.gated_backward(dy, x, w, wu, gate, up, dx=dx, dw_gate=dw, dw_up=dw2, act=name)
    want = oracle.gated_backward(dy, x, w, wu, gate, up, name)
    for got, key in ((dx, "dx"), (dw, "dw_gate"), (dw2, "dw_up")):
        oracle.check(got, want[key], key)


@pytest.mark.parametrize("pad,front", [(8, 0), (64, 8), (1, 0), (2, 3), (0, 4)])
@pytest.mark.parametrize("m", [1, 12, 40, 260])
def test_row_pitches(m, pad, front):
    """Operands and results as columns of wider matrices, at 16-byte and at other alignments."""
    n, k, dtype = 136, 200, torch.float16
    g = gen(m + pad)
    x, w, wu = (normal(g, r, k, dtype, s, pad, front) for r, s in ((m, 1.0), (n, k ** -0.5), (n, k ** -0.5)))
    res, dy = normal(g, m, n, dtype, 1.0, pad, front), normal(g, m, n, dtype, 0.1, pad, front)
    y, pre, gate, up = (Guarded(m, n, dtype, pad, front) for _ in range(4))
    dx = Guarded(m, k, dtype, pad, front)
    dw, dw2 = Guarded(n, k, dtype, pad, front), Guarded(n, k, dtype, pad, front)
    eas.ops.linear(x, w, y.t, residual=res, act="silu", pre=pre.t)
    want = oracle.linear(x, w, None, res, "silu")
    oracle.check(y.t, want["y"])
    oracle.check(pre.t, want["pre"])
    eas.ops.linear_backward(dy, x, w, dx=dx.t, dw=dw.t, act="silu", pre=pre.t)
    want = oracle.linear_backward(dy, x, w, pre.t, "silu")
    oracle.check(dx.t, want["dx"])
    oracle.check(dw.t, want["dw"])
    eas.ops.linear_backward(dy, x, w, dx=dx.t, dw=dw.t)
    want = oracle.linear_backward(dy, x, w)
    oracle.check(dx.t, want["dx"])
    oracle.check(dw.t, want["dw"])
    eas.ops.gated(x, w, wu, y.t, gate=gate.t, up=up.t)
    want = oracle.gated(x, w, wu)
    for got, key in ((y, "h"), (gate, "gate"), (up, "up")):
        oracle.check(got.t, want[key])
    eas.ops.gated_backward(dy, x, w, wu, gate.t, up.t, dx=dx.t, dw_gate=dw.t, dw_up=dw2.t)
    want = oracle.gated_backward(dy, x, w, wu, gate.t, up.t)
    for got, key in ((dx, "dx"), (dw, "dw_gate"), (dw2, "dw_up")):
        oracle.check(got.t, want[key])
    assert all(o.intact() for o in (y, pre, gate, up, dx, dw, dw2))


@pytest.mark.parametrize("m", [3, 150])
def test_orders_and_broadcasts(m):
    """Inputs of other orders (transposed, expanded, many leading dimensions) are taken as they are."""
    n, k, dtype = 72, 96, torch.bfloat16
    g = gen(m)
    x = normal(g, k, m, dtype).T
    w = normal(g, k, n, dtype, 0.1).T
    res = vector(normal(g, 1, n, dtype)).expand(m, n)
    y = torch.empty(m, n, device="cuda", dtype=dtype)
    eas.ops.linear(x, w, y, residual=res)
    oracle.check(y, oracle.linear(x, w, None, res)["y"])
    x1 = normal(g, 1, k, dtype).expand(m, k)
    eas.ops.linear(x1, w, y, bias=vector(normal(g, 1, n, dtype))[:1].expand(n))
    assert torch.equal(y, y[:1].expand(m, n))
    x3 = normal(g, 6 * m, k, dtype).view(2, 3, m, k)
    y3 = torch.empty(2, 3, m, n, device="cuda", dtype=dtype)
    eas.ops.linear(x3, w, y3)
    oracle.check(y3.view(-1, n), oracle.linear(x3.view(-1, k), w)["y"])
    eas.ops.linear(x3.transpose(0, 1), w, y3.view(3, 2, m, n))   # leading dimensions out of order: copied
    oracle.check(y3.view(-1, n), oracle.linear(x3.transpose(0, 1).reshape(-1, k), w)["y"])
    y1 = torch.empty(n, device="cuda", dtype=dtype)
    eas.ops.linear(x3[0, 0, 0], w, y1)
    oracle.check(y1[None], oracle.linear(x3[0, 0, :1], w)["y"])
    with pytest.raises(ValueError, match="unit stride"):
        eas.ops.linear(x, w, torch.empty(n, m, device="cuda", dtype=dtype).T)
    with pytest.raises(ValueError, match="unit stride"):
        eas.ops.linear(x, w, torch.empty(1, n, device="cuda", dtype=dtype).expand(m, n))
    with pytest.raises(ValueError, match="leading dimensions"):
        eas.ops.linear(x3.transpose(0, 1), w, y3.transpose(0, 1))


@pytest.mark.parametrize("m", [1, 5, 20, 50, 300])
def test_special_values_stay_in_their_rows(m):
    """NaN and infinities reach exactly the results whose sums they are in."""
    n, k, dtype = 200, 136, torch.float16
    g = gen(m)
    x, w, wu = normal(g, m, k, dtype), normal(g, n, k, dtype, 0.1), normal(g, n, k, dtype, 0.1)
    y, h, clean = (torch.empty(m, n, device="cuda", dtype=dtype) for _ in range(3))
    eas.ops.linear(x, w, clean)
    r = m // 2
    bad = x.clone()
    bad[r, k - 1] = float("nan")
    eas.ops.linear(bad, w, y)
    eas.ops.gated(bad, w, wu, h, act="relu")
    assert y[r].isnan().all() and h[r].isnan().all()
    keep = [i for i in range(m) if i != r]
    assert torch.equal(y[keep], clean[keep]) and not h[keep].isnan().any()
    bad[r, k - 1] = float("inf")
    wp = w.clone()
    wp[:, k - 1] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 0.25, -0.25).half()
    eas.ops.linear(bad, wp, y, act="relu")
    want = torch.where(torch.arange(n, device="cuda") % 2 == 0, float("inf"), 0.0).half()
    assert torch.equal(y[r], want)
    eas.ops.linear(bad, wp, y, act="sigmoid")
    assert torch.equal(y[r], (want > 0).half())
    # values past the type's range become infinite, as the type rounds
    big = torch.full_like(x, 240.0)
    eas.ops.linear(big, torch.full_like(w, 240.0), y)
    assert (y == float("inf")).all()
    # a NaN in one row of dz is in all of dW's columns sums but only in that row of dx
    dy = normal(g, m, n, dtype)
    dy[r, 3] = float("nan")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda", dtype=dtype)
    eas.ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db)
    assert dx[r].isnan().all() and not dx[keep].isnan().any()
    assert dw[3].isnan().all() and int(dw.isnan().any(1).sum()) == 1
    assert db[3].isnan() and int(db.isnan().sum()) == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 7), (1, 300, 64), (2, 17, 65), (3, 70, 1025), (5, 4099, 130), (7, 33, 127),
                                   (8, 600, 4095), (8, 2, 4999), (4, 21, 9001), (3, 2100, 1025), (1, 33000, 65),
                                   (2, 520, 4100), (9, 70, 33), (40, 300, 201), (130, 72, 63)])
def test_rows_at_any_address(m, n, k, dtype):
    """Operands whose rows start anywhere, with NaN all around them, give the bits that aligned copies give."""
    g = gen(m * n + k)

    def placed(t, front, pitch):
        rows, cols = t.shape
        mem = torch.full((front + (rows - 1) * pitch + cols,), float("nan"), device="cuda", dtype=dtype)
        view = mem.as_strided((rows, cols), (pitch, 1), front)
        view.copy_(t)
        return view

    x, w, wu = normal(g, m, k, dtype), normal(g, n, k, dtype, 0.1), normal(g, n, k, dtype, 0.1)
    res, dy, z = normal(g, m, n, dtype), normal(g, m, n, dtype), normal(g, m, n, dtype)
    new = lambda *shape: torch.full(shape, 7.0, device="cuda", dtype=dtype)

    def run(x, w, wu, res, dy, z):
        y, h, dx, dw, db = new(m, n), new(m, n), new(m, k), new(n, k), new(n)
        eas.ops.linear(x, w, y, residual=res, act="silu")
        eas.ops.gated(x, w, wu, h)
        eas.ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, act="gelu", pre=z)
        dx2, dg, du, db2 = new(m, k), new(n, k), new(n, k), new(n)
        eas.ops.gated_backward(dy, x, w, wu, z, res, dx=dx2, dw_gate=dg, dw_up=du)
        eas.ops.linear_backward(dy, x, w, dbias=db2)
        return y, h, dx, dw, db, dx2, dg, du, db2

    pitch_k, pitch_n = -(-k // 8) * 8, -(-n // 8) * 8
    want = run(*(placed(t, 0, p) for t, p in ((x, pitch_k), (w, pitch_k), (wu, pitch_k), (res, pitch_n), (dy, pitch_n),
                                              (z, pitch_n))))
    assert all(t.isfinite().all() for t in want)
    for front, extra in ((1, 0), (7, 1), (4, 3), (3, 6), (0, 1), (6, 13)):
        odd = [placed(t, (front + 3 * i) % 8, t.shape[1] + extra + i) for i, t in enumerate((x, w, wu, res, dy, z))]
        for a, b in zip(run(*odd), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("m", [2, 40, 300])
def test_special_values_stay_in_their_columns(m, name):
    """A NaN in one output's weights or bias is in that column alone, whatever the columns beside it share."""
    n, k, dtype = 264, 72, torch.bfloat16
    g = gen(m)
    x, w, wu = normal(g, m, k, dtype), normal(g, n, k, dtype, 0.1), normal(g, n, k, dtype, 0.1)
    bias = vector(normal(g, 1, n, dtype))
    y, clean, h, hc = (torch.empty(m, n, device="cuda", dtype=dtype) for _ in range(4))
    eas.ops.linear(x, w, clean, bias=bias, act=name)
    eas.ops.gated(x, w, wu, hc, act=name)
    for c in (0, 5, 130, n - 1):
        bad = bias.clone()
        bad[c] = float("nan")
        eas.ops.linear(x, w, y, bias=bad, act=name)
        wb = w.clone()
        wb[c, 3] = float("nan")
        eas.ops.gated(x, wb, wu, h, act=name)
        keep = [i for i in range(n) if i != c]
        assert y[:, c].isnan().all() and torch.equal(y[:, keep], clean[:, keep])
        assert h[:, c].isnan().all() and torch.equal(h[:, keep], hc[:, keep])
    for big in (3e38, 1e20, -1e20, -3e38):   # far values beside near ones
        bad = bias.clone()
        bad[2::4] = big
        eas.ops.linear(x, w, y, bias=bad, act=name)
        keep = [i for i in range(n) if i % 4 != 2]
        assert torch.equal(y[:, keep], clean[:, keep])
        far = oracle.act(name, bad[2::4].double())[0].nan_to_num(0.0)
        far = torch.where(bad[2::4].double() < -1e4, torch.zeros_like(far), far) if name != "none" else far
        assert torch.allclose(y[:, 2::4].double(), far.expand(m, -1), rtol=2.0 ** -7, atol=1e-30)


def test_far_pre_activations():
    """Slopes and values where the exponentials under- and overflow."""
    dtype = torch.bfloat16
    z = torch.tensor([-3e38, -1e20, -1e4, -200.0, -100.0, -89.0, -88.0, -60.0, -20.0, -6.0, -1e-30, 0.0, 1e-30, 6.0, 20.0,
                      60.0, 88.0, 89.0, 100.0, 200.0, 1e4, 1e20, 3e38], device="cuda", dtype=dtype)
    n = z.numel()
    dy = torch.ones(1, n, device="cuda", dtype=dtype)
    x = torch.ones(1, 8, device="cuda", dtype=dtype)
    w = torch.zeros(n, 8, device="cuda", dtype=dtype)
    for name in ACTS[1:]:
        db = torch.empty(n, device="cuda", dtype=dtype)
        eas.ops.linear_backward(dy, x, w, dbias=db, act=name, pre=z[None])
        d = oracle.act(name, z.double().clamp(-1e4, 1e4))[1]
        assert torch.allclose(db.double(), d, rtol=2.0 ** -7, atol=1e-30), name
        y = torch.empty(1, n, device="cuda", dtype=dtype)
        eas.ops.linear(x, w, y, bias=z, act=name)
        v = oracle.act(name, z.double())[0].nan_to_num(0.0)
        v = torch.where(z.double() < -1e4, torch.zeros_like(v), v)
        assert torch.allclose(y[0].double(), v, rtol=2.0 ** -7, atol=1e-30), name


def test_no_rows():
    """Zero tokens: nothing is launched forward; gradients that are sums over tokens are zero."""
    n, k, dtype = 40, 24, torch.float16
    x, y = torch.empty(0, k, device="cuda", dtype=dtype), torch.empty(0, n, device="cuda", dtype=dtype)
    w = torch.ones(n, k, device="cuda", dtype=dtype)
    eas.ops.linear(x, w, y)
    eas.ops.gated(x, w, w.clone(), y)
    dw, dw2, db = Guarded(n, k, dtype, 8), Guarded(n, k, dtype, 3), Guarded(1, n, dtype)
    eas.ops.linear_backward(y, x, w, dx=x.clone(), dw=dw.t, dbias=db.t[0], act="gelu", pre=y.clone())
    assert (dw.t == 0).all() and (db.t == 0).all() and dw.intact() and db.intact()
    eas.ops.gated_backward(y, x, w, w.clone(), y, y, dw_gate=dw.t, dw_up=dw2.t)
    assert (dw2.t == 0).all() and dw2.intact()
    x0 = torch.empty(3, 0, 2, k, device="cuda", dtype=dtype)
    eas.ops.linear(x0, w, torch.empty(3, 0, 2, n, device="cuda", dtype=dtype))


@pytest.mark.parametrize("m", [1, 20, 80, 600])
def test_in_place_residual_and_repeatability(m):
    n, k, dtype = 264, 520, torch.bfloat16
    g = gen(m)
    x, w, res = normal(g, m, k, dtype), normal(g, n, k, dtype, 0.05), normal(g, m, n, dtype)
    y = torch.empty_like(res)
    eas.ops.linear(x, w, y, residual=res, act="gelu")
    stream = res.clone()
    eas.ops.linear(x, w, stream, residual=stream, act="gelu")
    assert torch.equal(stream, y)
    for _ in range(3):
        again = torch.empty_like(y)
        eas.ops.linear(x, w, again, residual=res, act="gelu")
        assert torch.equal(again, y)
    grads = []
    for _ in range(2):
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda", dtype=dtype)
        eas.ops.linear_backward(res, x, w, dx=dx, dw=dw, dbias=db, act="silu", pre=y)
        grads.append((dx, dw, db))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def _block(x, wg, wu, wd, dy, sync=True):
    """A gated block on the residual stream, forward and backward, as a training step runs it."""
    m, k = x.shape
    n, dt = wg.shape[0], x.dtype
    new = lambda *s: torch.empty(*s, device="cuda", dtype=dt)  # noqa: E731
    h, gate, up, y = new(m, n), new(m, n), new(m, n), new(m, k)
    dh, dwd, dx, dwg, dwu = new(m, n), new(k, n), new(m, k), new(n, k), new(n, k)
    eas.ops.gated(x, wg, wu, h, gate=gate, up=up, _sync=sync)
    eas.ops.linear(h, wd, y, residual=x, _sync=sync)
    eas.ops.linear_backward(dy, h, wd, dx=dh, dw=dwd, _sync=sync)
    eas.ops.gated_backward(dh, x, wg, wu, gate, up, dx=dx, dw_gate=dwg, dw_up=dwu, _sync=sync)
    return {"h": h, "gate": gate, "up": up, "y": y, "dh": dh, "dwd": dwd, "dx": dx, "dwg": dwg, "dwu": dwu}


def _block_inputs(m, n, k, dtype, seed=0):
    g = gen(seed)
    return (normal(g, m, k, dtype), normal(g, n, k, dtype, k ** -0.5), normal(g, n, k, dtype, k ** -0.5),
            normal(g, k, n, dtype, n ** -0.5), normal(g, m, k, dtype, 0.1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 8, 48, 333])
def test_block_step_by_step(m, dtype):
    """The operators one after another, each checked on what the one before it gave."""
    x, wg, wu, wd, dy = _block_inputs(m, 520, 264, dtype)
    o = _block(x, wg, wu, wd, dy)
    want = oracle.gated(x, wg, wu)
    for key in ("h", "gate", "up"):
        oracle.check(o[key], want[key], key)
    oracle.check(o["y"], oracle.linear(o["h"], wd, None, x)["y"], "y")
    want = oracle.linear_backward(dy, o["h"], wd)
    oracle.check(o["dh"], want["dx"], "dh")
    oracle.check(o["dwd"], want["dw"], "dwd")
    want = oracle.gated_backward(o["dh"], x, wg, wu, o["gate"], o["up"])
    for key, name in (("dx", "dx"), ("dwg", "dw_gate"), ("dwu", "dw_up")):
        oracle.check(o[key], want[name], key)


def test_block_gradient_against_differences():
    """<gradient, v> of the whole block against differences of its definition in 64 bits, along random directions.

    Each gradient is off from the true one elementwise by at most what its operators allow on their inputs plus the effect of
    the rounded h, gate, up and dh; that effect is below 3 u of the same sums of absolute products, so the tolerance is
    4 times the operators' own (the last one's error model already has the first u)."""
    dtype = torch.float16
    x, wg, wu, wd, dy = _block_inputs(40, 136, 72, dtype, seed=3)
    o = _block(x, wg, wu, wd, dy)
    base = {"dx": x.double(), "dwg": wg.double(), "dwu": wu.double(), "dwd": wd.double()}

    def loss(p):
        a, _ = oracle.act("silu", p["dx"] @ p["dwg"].T)
        return ((a * (p["dx"] @ p["dwu"].T)) @ p["dwd"].T * dy.double()).sum()

    tol = oracle.gated_backward(o["dh"], x, wg, wu, o["gate"], o["up"])
    tol = {"dx": tol["dx"][1], "dwg": tol["dw_gate"][1], "dwu": tol["dw_up"][1],
           "dwd": oracle.linear_backward(dy, o["h"], wd)["dw"][1]}
    g = gen(9)
    for key in base:
        for _ in range(3):
            v = torch.randn(base[key].shape, device="cuda", generator=g, dtype=torch.float64)
            eps = 1e-5
            d = (loss({**base, key: base[key] + eps * v}) - loss({**base, key: base[key] - eps * v})) / (2 * eps)
            got = (o[key].double() * v).sum()
            assert abs(float(got - d)) <= 4 * float((tol[key] * v.abs()).sum()), key


@pytest.mark.parametrize("m", [1, 48, 300])
def test_capture_and_replay(cuda_rt, m):
    """A block captured once, replayed on new inputs, with a second graph and eager calls beside it."""
    n, k, dtype = 520, 264, torch.bfloat16
    ins = [_block_inputs(m, n, k, dtype, seed=s) for s in (1, 2, 3)]
    want = [_block(*i) for i in ins]
    live = [t.clone() for t in ins[0]]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block(*live, sync=False)
        graphs.append((graph, out))
    assert cuda_rt.in_flight() == 0
    for i in (1, 2):
        for t, src in zip(live, ins[i]):
            t.copy_(src)
        for graph, out in graphs:
            graph.replay()
            eager = _block(*live, sync=False)   # beside the replay, on the same inputs
            torch.cuda.synchronize()
            for key in out:
                assert torch.equal(out[key], want[i][key]), key
                assert torch.equal(eager[key], want[i][key]), key
    with pytest.raises(ValueError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            eas.ops.linear(live[0], live[1], torch.empty(m, n, device="cuda", dtype=dtype))
    cuda_rt.synchronize()


def test_streams(cuda_rt):
    """Calls in two streams at once, each with buffers that are dropped before the work is done."""
    m, n, k, dtype = 300, 520, 264, torch.float16
    ins = [_block_inputs(m, n, k, dtype, seed=s) for s in range(4)]
    want = [_block(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for rep in range(3):
        for i, args in enumerate(ins):
            s = streams[i % 2]
            with torch.cuda.stream(s):
                mine = [t.clone() for t in args]
                outs.append((i, _block(*mine, sync=False)))
                del mine
    torch.cuda.synchronize()
    for i, o in outs:
        for key in o:
            assert torch.equal(o[key], want[i][key]), (i, key)
    cuda_rt.synchronize()
    assert cuda_rt.in_flight() == 0


def test_buffers_of_another_stream(cuda_rt):
    """Buffers allocated on the default stream, used in another one and dropped while it is busy: their memory is not
    handed out again before the call is done."""
    m, n, k, dtype = 256, 512, 512, torch.bfloat16
    x, w = normal(gen(0), m, k, dtype), normal(gen(1), n, k, dtype, k ** -0.5)
    want = torch.empty(m, n, device="cuda", dtype=dtype)
    eas.ops.linear(x, w, want, act="silu")
    side = torch.cuda.Stream()
    for _ in range(5):
        y = torch.empty_like(want)
        mine = x.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            eas.ops.linear(mine, w, y, act="silu", _sync=False)
        del mine
        junk = [torch.full_like(x, float("nan")) for _ in range(4)]   # would take the dropped block
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        del junk
    cuda_rt.synchronize()


def test_memory_does_not_pile_up(cuda_rt):
    """Calls that run ahead of the GPU hold neither their scratch nor their callers' dropped buffers."""
    m, n, k, dtype = 2048, 2048, 256, torch.float16
    g = gen(0)
    x, w, dy, pre = (normal(g, *s, dtype) for s in ((m, k), (n, k), (m, n), (m, n)))
    dx = torch.empty_like(x)

    def step():
        eas.ops.linear_backward(dy.clone(), x, w, dx=dx, act="gelu", pre=pre, _sync=False)

    step()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for _ in range(100):
        step()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 4 * dy.numel() * 2
    cuda_rt.synchronize()


def test_repeated_calls_keep_their_checks(cuda_rt):
    """A call of shapes seen before is still checked for what its addresses and flags can make wrong."""
    m, n, k, dtype = 40, 64, 64, torch.float16
    g = gen(0)
    whole = torch.empty(4 * m * n + 8, device="cuda", dtype=dtype)
    x, w = normal(g, m, k, dtype), normal(g, n, k, dtype)
    want = torch.empty(m, n, device="cuda", dtype=dtype)
    eas.ops.linear(x, w, want)
    for _ in range(2):
        y = whole[:m * n].view(m, n)
        eas.ops.linear(x, w, y)
        assert torch.equal(y, want)
        odd = whole[1:1 + m * n].view(m, n)             # the same shape on another alignment
        eas.ops.linear(x, w, odd)
        assert torch.equal(odd, want)
        xo = whole[2 * m * n + 3:2 * m * n + 3 + m * k].view(m, k)
        xo.copy_(x)
        eas.ops.linear(xo, w, y)
        assert torch.equal(y, want)
        with pytest.raises(ValueError, match="overlaps"):
            eas.ops.linear(x, w, x)
        with pytest.raises(ValueError, match="overlaps"):
            eas.ops.linear(y, w, odd)
        res = want.clone()
        eas.ops.linear(x, w, res, residual=res)
        assert not torch.equal(res, want)
        with pytest.raises(ValueError, match="overlaps"):
            eas.ops.linear(x, w, whole[8:8 + m * n].view(m, n), residual=whole[:m * n].view(m, n))
        with pytest.raises(TypeError, match="_sync"):
            eas.ops.linear(x, w, y, _sync=None)
        with pytest.raises(ValueError, match="activation"):
            eas.ops.linear(x, w, y, act="tanh")
        with pytest.raises(TypeError, match="dtype"):
            eas.ops.linear(x, w, y.bfloat16())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2 = torch.empty_like(want)
            eas.ops.linear(x, w, y2, _sync=False)
        side.synchronize()
        assert torch.equal(y2, want)
    left, right = whole[:2 * m * n].view(m, 2 * n)[:, :n], whole[:2 * m * n].view(m, 2 * n)[:, n:]
    left.copy_(x)
    for _ in range(2):
        eas.ops.linear(left, w, right)                   # side by side in one matrix
        assert torch.equal(right, want) and torch.equal(left, x)
    cuda_rt.synchronize()


def test_eas_tensors(cuda_rt):
    """eas.Tensor buffers (f16) give what torch tensors give, mixed with them too."""
    m, n, k = 33, 136, 72
    x, wg, wu, wd, dy = _block_inputs(m, n, k, torch.float16)
    o = _block(x, wg, wu, wd, dy)
    t = lambda v: eas.tensor(v.cpu().numpy(), device="cuda")  # noqa: E731
    e = lambda *s: eas.empty(s, device="cuda", dtype="float16")  # noqa: E731
    h, gate, up, y = e(m, n), e(m, n), e(m, n), e(m, k)
    X, WG, WU, WD, DY = t(x), t(wg), t(wu), t(wd), t(dy)
    eas.ops.gated(X, WG, WU, h, gate=gate, up=up)
    eas.ops.linear(h, WD, y, residual=X)
    dh, dwd = e(m, n), e(k, n)
    eas.ops.linear_backward(DY, h, WD, dx=dh, dw=dwd)
    dx, dwg, dwu = e(m, k), e(n, k), e(n, k)
    eas.ops.gated_backward(dh, X, WG, WU, gate, up, dx=dx, dw_gate=dwg, dw_up=dwu)
    for key, v in (("h", h), ("y", y), ("dh", dh), ("dwd", dwd), ("dx", dx), ("dwg", dwg), ("dwu", dwu)):
        assert torch.equal(torch.from_numpy(v.numpy()).cuda(), o[key]), key
    mixed = torch.empty_like(o["y"])
    eas.ops.linear(h, wd, mixed, residual=x)
    assert torch.equal(mixed, o["y"])


def test_rows_past_32_bit_offsets():
    """Rows whose element offsets pass 2^32 (a very wide pitch)."""
    k, n, dtype = 64, 72, torch.float16
    pitch = (1 << 26) + 64
    rows = 70   # 70 * pitch elements > 2^32
    try:
        whole = torch.zeros(rows * pitch, device="cuda", dtype=dtype)
    except torch.OutOfMemoryError:
        pytest.skip("needs 9.4 GB")
    x = torch.as_strided(whole, (rows, k), (pitch, 1))
    y = torch.as_strided(whole, (rows, n), (pitch, 1), 128)
    pre = torch.as_strided(whole, (rows, n), (pitch, 1), 256)
    g = gen(0)
    x.copy_(normal(g, rows, k, dtype))
    w = normal(g, n, k, dtype, 0.1)
    eas.ops.linear(x, w, y, act="silu", pre=pre)
    want = oracle.linear(x, w, None, None, "silu")
    oracle.check(y, want["y"])
    oracle.check(pre, want["pre"])
    dx = torch.as_strided(whole, (rows, k), (pitch, 1), 512)
    eas.ops.linear_backward(y, x, w, dx=dx, act="silu", pre=pre)
    oracle.check(dx, oracle.linear_backward(y, x, w, pre, "silu")["dx"])
    y1 = torch.as_strided(whole, (5, n), (pitch * 16, 1), 1024)
    x1 = torch.as_strided(whole, (5, k), (pitch * 16, 1))
    eas.ops.linear(x1, w, y1)
    oracle.check(y1, oracle.linear(x1, w)["y"])
