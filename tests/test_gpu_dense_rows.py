"""GPU: eas.ops on up to 8 rows in every way that the kernel for them has, whatever addresses the rows start at.

Sparse small integers, whose every intermediate and result is exact, with NaN in all memory around the operands."""

import pytest
import torch

import eas
from dense_rows_shapes import SHAPES

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _ready(cuda_rt):
    yield
    cuda_rt.synchronize()
    torch.cuda.synchronize()


def sparse(g, rows, cols, dtype, per_row):
    v = torch.randint(0, 2, (rows, cols), device="cuda", generator=g) * 2.0 - 1
    return (v * (torch.rand(rows, cols, device="cuda", generator=g) < min(1.0, per_row / cols))).to(dtype)


def placed(t, front, pitch):
    """``t`` in rows of ``pitch`` values from ``front`` on, with NaN all around."""
    rows, cols = t.shape
    mem = torch.full((front + rows * pitch + 8,), float("nan"), device="cuda", dtype=t.dtype)
    view = mem.as_strided((rows, cols), (pitch, 1), front)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_exact(shape, odd, dtype):
    m, n, k = shape
    g = torch.Generator(device="cuda").manual_seed(m + n * 3 + k * 7)
    x, w, wu = sparse(g, m, k, dtype, 40), sparse(g, n, k, dtype, 40), sparse(g, n, k, dtype, 40)
    bias, res = sparse(g, 1, n, dtype, n)[0], sparse(g, m, n, dtype, n)
    z, u = x.double() @ w.double().T, x.double() @ wu.double().T
    assert z.abs().max() <= 100 and (z * u).abs().max() <= 250
    if odd:
        x, w, wu = (placed(t, f, k + p) for t, f, p in ((x, 1, 3), (w, 5, 2 - k % 2), (wu, 2, 4 + k % 2)))
    else:
        x, w, wu = (placed(t, 8, -(-k // 8) * 8) for t in (x, w, wu))
    out = torch.full((4, m, n + 3), 7.0, device="cuda", dtype=dtype)
    y, pre, h, gate = (o[:, :n] for o in out)
    eas.ops.linear(x, w, y, bias=bias, residual=res, act="relu", pre=pre)
    assert torch.equal(pre.double(), z + bias.double())
    assert torch.equal(y.double(), (z + bias.double()).clamp(min=0) + res.double())
    up = torch.empty_like(h)
    eas.ops.gated(x, w, wu, h, act="relu", gate=gate, up=up)
    assert torch.equal(gate.double(), z) and torch.equal(up.double(), u)
    assert torch.equal(h.double(), z.clamp(min=0) * u)
    assert (out[:, :, n:] == 7).all()
