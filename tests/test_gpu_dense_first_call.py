"""GPU: the first call of a process, inside a graph capture, without any warm-up before it."""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import ctypes
import torch
import eas
from easy_as_b200.runtime import cuda_ext

m, n, k = {shape}
gen = torch.Generator(device="cuda").manual_seed(1)
ints = lambda *s: torch.randint(-1, 2, s, device="cuda", generator=gen).half()
x, w, wu, dy, z = ints(m, k), ints(n, k), ints(n, k), ints(m, n), ints(m, n)
y, dx = torch.full((m, n), 7.0, device="cuda").half(), torch.full((m, k), 7.0, device="cuda").half()
dw, dwu, db = torch.zeros_like(w), torch.zeros_like(w), torch.zeros(n, device="cuda").half()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    if {backward}:
        eas.ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, act="relu", pre=z, _sync=False)
    else:
        eas.ops.linear(x, w, y, _sync=False)
assert (y == 7).all() and (dx == 7).all()     # captured, not run
graph.replay()
torch.cuda.synchronize()
if {backward}:
    dz = dy.double() * (z.double() > 0)
    assert torch.equal(dx.double(), dz @ w.double()) and torch.equal(dw.double(), dz.T @ x.double())
    assert torch.equal(db.double(), dz.sum(0))
else:
    assert torch.equal(y.double(), x.double() @ w.double().T)
lib = cuda_ext.load()
code = ctypes.c_int(-1)
assert lib.eas_gemm_status(0, ctypes.byref(code)) == 0 and code.value == 0
# the word that an expired wait is reported in was there
cuda_ext.check(lib.eas_wait_selftest(1000000, None), "selftest")
torch.cuda.synchronize()
assert lib.eas_gemm_status(0, ctypes.byref(code)) == 0 and code.value == cuda_ext.EAS_ERR_TIMEOUT
print("done")
"""


@pytest.mark.parametrize("shape", [(3, 40, 72), (40, 136, 200), (600, 520, 520)])
@pytest.mark.parametrize("backward", [False, True])
def test_first_call_is_captured(cuda_rt, shape, backward):
    program = PROGRAM.format(shape=shape, backward=backward)
    r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stdout + r.stderr
