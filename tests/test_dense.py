"""CPU: what eas.ops refuses, and the C entry points' checks of their arguments (no GPU)."""

import ctypes

import numpy as np
import pytest

import eas
from easy_as_b200.runtime import cuda_ext
from easy_as_b200.tensor import Tensor


def dev(rows, cols, *, at=0x10000000, device=0, dtype=np.float16):
    """An eas.Tensor on a device address that nothing reads: every check comes before the launch."""
    shape = (cols,) if rows is None else (rows, cols)
    return Tensor._from_cuda_ptr(at, shape, dtype, device, owner=None)


_next = [0x20000000]


def new(rows, cols, **kw):
    _next[0] += 1 << 24
    return dev(rows, cols, at=_next[0], **kw)


def linear_args():
    return {"x": new(4, 16), "w": new(8, 16), "y": new(4, 8)}


def test_names():
    assert eas.ops.ACTIVATIONS == ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
    import eas.ops as direct

    assert direct is eas.ops


@pytest.mark.parametrize("change,error,match", [
    ({"x": np.zeros((4, 16), np.float16)}, TypeError, "'x'"),
    ({"x": "nothing"}, TypeError, "'x'"),
    ({"x": eas.tensor(np.zeros((4, 16), np.float16))}, TypeError, "CUDA device"),
    ({"w": new(8, 16, dtype=np.float32)}, TypeError, "float16"),
    ({"x": new(4, 15)}, ValueError, "'x' has shape"),
    ({"y": new(4, 9)}, ValueError, "'y' has shape"),
    ({"y": new(5, 8)}, ValueError, "'y' has shape"),
    ({"w": new(None, 16)}, ValueError, "matrix"),
    ({"w": new(0, 16), "y": new(4, 0)}, ValueError, "at least one"),
    ({"x": new(4, 0), "w": new(8, 0)}, ValueError, "at least one"),
    ({"bias": new(None, 7)}, ValueError, "'bias'"),
    ({"bias": new(1, 8)}, ValueError, "'bias'"),
    ({"residual": new(1, 8)}, ValueError, "'residual'"),
    ({"pre": new(4, 16)}, ValueError, "'pre'"),
    ({"y": new(4, 8, device=1)}, ValueError, "different devices"),
    ({"act": "swish"}, ValueError, "unknown activation"),
    ({"_sync": 1}, TypeError, "_sync"),
])
def test_linear_refusals(change, error, match):
    args = {**linear_args(), **change}
    x, w, y = args.pop("x"), args.pop("w"), args.pop("y")
    with pytest.raises(error, match=match):
        eas.ops.linear(x, w, y, **args)


def test_torch_refusals():
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError, match="CUDA device"):
        eas.ops.linear(torch.zeros(4, 16, dtype=torch.float16), new(8, 16), new(4, 8))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        eas.ops.linear(torch.zeros(4, 16), new(8, 16), new(4, 8))


@pytest.mark.parametrize("y", [
    dev(4, 8, at=0x10000000),                  # x itself
    dev(4, 8, at=0x10000000 + 4 * 16 * 2 - 2),  # x's last element
    dev(4, 8, at=0x30000000),                  # the weight
    dev(4, 8, at=0x40000000 + 2),              # the residual, one element off
    dev(4, 8, at=0x50000000),                  # the bias
    dev(4, 8, at=0x60000000 + 4 * 8),          # pre
])
def test_overlaps_are_refused(y):
    with pytest.raises(ValueError, match="overlaps"):
        eas.ops.linear(dev(4, 16), dev(8, 16, at=0x30000000), y, residual=dev(4, 8, at=0x40000000),
                       bias=dev(None, 8, at=0x50000000), pre=dev(4, 8, at=0x60000000))


def test_side_by_side_columns_do_not_overlap():
    from easy_as_b200.ops import _Rows, _share

    def cols(first, count, rows=4, ld=32):
        return _Rows(0x1000 + 2 * first, rows, count, ld, (rows,), None)

    assert not _share(cols(0, 8), cols(8, 8)) and not _share(cols(8, 8), cols(0, 8))
    assert not _share(cols(24, 8), cols(32, 8))           # the next row's first columns, one row further
    assert _share(cols(0, 9), cols(8, 8)) and _share(cols(8, 8), cols(0, 9))
    assert _share(cols(30, 8), cols(0, 8))                # wraps into the next row
    assert _share(cols(0, 8), cols(8, 8, ld=40))          # other pitches: not told apart
    assert not _share(cols(0, 8, rows=0), cols(0, 8))


def test_gated_refusals():
    x, wg, wu, h = new(4, 16), new(8, 16), new(8, 16), new(4, 8)
    with pytest.raises(ValueError, match="both of gate and up"):
        eas.ops.gated(x, wg, wu, h, gate=new(4, 8))
    with pytest.raises(ValueError, match="'w_up'"):
        eas.ops.gated(x, wg, new(9, 16), h)
    with pytest.raises(ValueError, match="'h'"):
        eas.ops.gated(x, wg, wu, new(4, 16))
    g = new(4, 8)
    with pytest.raises(ValueError, match="overlaps"):
        eas.ops.gated(x, wg, wu, h, gate=g, up=g)
    with pytest.raises(ValueError, match="unknown activation"):
        eas.ops.gated(x, wg, wu, h, act=None)


def test_backward_refusals():
    dy, x, w = new(4, 8), new(4, 16), new(8, 16)
    with pytest.raises(ValueError, match="needs pre"):
        eas.ops.linear_backward(dy, x, w, dx=new(4, 16), act="gelu")
    with pytest.raises(ValueError, match="'dx'"):
        eas.ops.linear_backward(dy, x, w, dx=new(4, 8))
    with pytest.raises(ValueError, match="'dw'"):
        eas.ops.linear_backward(dy, x, w, dw=new(16, 8))
    with pytest.raises(ValueError, match="'dbias'"):
        eas.ops.linear_backward(dy, x, w, dbias=new(None, 16))
    with pytest.raises(ValueError, match="overlaps"):
        eas.ops.linear_backward(dy, x, w, dx=x)
    with pytest.raises(ValueError, match="overlaps"):
        eas.ops.gated_backward(dy, x, w, new(8, 16), dy, dy, dw_gate=w)
    with pytest.raises(ValueError, match="'gate'"):
        eas.ops.gated_backward(dy, x, w, new(8, 16), x, dy, dx=new(4, 16))
    eas.ops.linear_backward(dy, x, w)   # nothing asked for: nothing to do


_vp, _u64 = ctypes.c_void_p, ctypes.c_uint64
_TAIL = [("scratch_bytes", _u64), ("M", ctypes.c_uint32), ("N", ctypes.c_uint32), ("K", ctypes.c_uint32),
         ("dev", ctypes.c_int), ("dtype", ctypes.c_int), ("act", ctypes.c_int)]


def _struct(pointers, pitches):
    class Args(ctypes.Structure):
        _fields_ = [(n, _vp) for n in pointers.split() + ["scratch"]] + [(n, _u64) for n in pitches.split()] + _TAIL

    return Args


#: the argument structs as include/eas_cuda.h declares them
ARGS = {
    "eas_linear": _struct("x w bias residual y pre", "ldx ldw ldr ldy ldp"),
    "eas_gated": _struct("x w_gate w_up h gate up", "ldx ldwg ldwu ldh ldg ldu"),
    "eas_linear_backward": _struct("dy pre x w dx dw db", "lddy ldp ldx ldw lddx lddw"),
    "eas_gated_backward": _struct("dh gate up x w_gate w_up dx dw_gate dw_up",
                                  "lddh ldg ldu ldx ldwg ldwu lddx lddwg lddwu"),
}


def _call(name, **change):
    a = ARGS[name](M=4, N=8, K=16, act=0 if name in ("eas_linear", "eas_gated") else 1)
    for i, (field, kind) in enumerate(a._fields_):
        if field in ("bias", "residual", "scratch") or (name, field) in (("eas_linear", "pre"), ("eas_gated", "gate"),
                                                                        ("eas_gated", "up")):
            continue
        if kind is _vp:
            setattr(a, field, 4096 * (i + 1))
        elif field.startswith("ld"):
            setattr(a, field, 16)
    for field, v in change.items():
        assert any(field == f for f, _k in a._fields_)
        setattr(a, field, v)
    return getattr(cuda_ext.load(), name)(ctypes.byref(a), None)


def test_argument_structs_match_the_header():
    """Field order of each struct in the header, and the sizes that eas.ops packs."""
    import re
    from pathlib import Path

    from easy_as_b200 import ops

    text = (Path(__file__).resolve().parent.parent / "include" / "eas_cuda.h").read_text()
    for name, cls in ARGS.items():
        body = next(b for b, n in re.findall(r"typedef struct \{(.*?)\} (\w+);", text, re.S) if n == name + "_args")
        fields = []
        for decl in body.split(";"):
            names = re.sub(r"const void|void|uint64_t|uint32_t|int32_t", "", decl).replace("*", "")
            fields += [f.strip() for f in names.split(",") if f.strip()]
        assert fields == [f for f, _k in cls._fields_], name
        entry = next(e for e in (ops._E_LINEAR, ops._E_GATED, ops._E_LINEAR_BACKWARD, ops._E_GATED_BACKWARD)
                     if e.name == name)
        assert entry.pointers.size + entry.rest.size == ctypes.sizeof(cls), name
    for name in ARGS:
        assert getattr(cuda_ext.load(), name)(None, None) == cuda_ext.EAS_ERR_VALUE


@pytest.mark.parametrize("name", ["eas_linear", "eas_gated", "eas_linear_backward", "eas_gated_backward"])
@pytest.mark.parametrize("change,match", [
    ({"dtype": 2}, "dtype"), ({"dtype": -1}, "dtype"), ({"act": 6}, "activation"), ({"act": -1}, "activation"),
    ({"N": 0}, "positive"), ({"K": 0}, "positive"), ({"M": 0xffffffff}, "exceeds"), ({"K": 0x80000000}, "exceeds"),
    ({"x": None}, "null"), ({"x": 4097}, "odd"), ({"ldx": 15}, "pitch"),
])
def test_c_entries_check_their_arguments(name, change, match):
    assert _call(name, **change) == cuda_ext.EAS_ERR_VALUE
    assert match in cuda_ext.last_error() and name in cuda_ext.last_error()


@pytest.mark.parametrize("name", ["eas_linear_backward", "eas_gated_backward"])
def test_c_entries_want_their_scratch(name):
    lib = cuda_ext.load()
    need = ctypes.c_uint64()
    op = 2 if name == "eas_linear_backward" else 3
    assert lib.eas_dense_scratch(op, 4, 8, 16, 1, 7 if op == 2 else 3, 0, ctypes.byref(need)) == 0
    assert need.value > 0 and need.value % 256 == 0
    for scratch, nbytes in ((None, need.value), (65536, need.value - 1), (65536 + 16, need.value)):
        assert _call(name, scratch=scratch, scratch_bytes=nbytes) == cuda_ext.EAS_ERR_VALUE
        assert "scratch" in cuda_ext.last_error()


def test_extension_is_built_and_leaves_doubtful_calls_alone():
    torch = pytest.importorskip("torch")
    from easy_as_b200 import build, ops

    assert build.OPS_STAMP.read_text().strip() == build.ops_hash()
    ext = ops._load_ext()
    assert ext
    t = torch.zeros(4, 4, dtype=torch.float16)
    for bufs in ((t, t, t), (new(4, 4),), (None, 3), [t], (None,) * 17):
        assert ext.quick(0, 0, bufs, True) is None            # no CUDA tensors, other objects, no plan
    assert ext.quick(0, -1, (None,), True) is None             # an unknown activation
    assert ext.quick(0, 0, (None,), 1) is None                 # a flag that is not bool
    assert ext.leave(0, 0, (t,), 1, b"", 0, 0, ()) is False     # nothing kept for them either
    with pytest.raises(TypeError):
        ext.quick(0, 0, (t,))
    with pytest.raises(TypeError):
        ext.quick("x", 0, (t,), True)


def test_gpu_tests_reach_every_kernel():
    """The sizes of the exact GPU tests run every kernel that any call can reach (each is instantiated for some)."""
    import random

    import dense_shapes as ds

    covered = set().union(*(ds.kernels(s) for s in ds.SHAPES + ds.BIG + ds.VARIANTS))
    rng = random.Random(0)
    for _ in range(6000):
        shape = tuple(int(2 ** rng.uniform(0, 13.5)) for _ in range(3))
        missing = ds.kernels(shape) - covered
        assert not missing, (shape, missing)
    assert {k[1] for k in covered} == {0, 1, 2}


def test_plan_checks_its_arguments():
    import dense_shapes as ds

    assert ds.plan(ds.LINEAR, 1, 4096, 4096)[0] == 0
    assert ds.plan(ds.LINEAR, 8192, 8192, 8192)[0] == 2
    for bad in ((4, 1, 1, 1, 0), (2, 1, 1, 1, 0), (2, 1, 1, 1, 4), (0, 0, 1, 1, 0), (0, 1, 0, 1, 0)):
        with pytest.raises(ValueError):
            ds.plan(*bad)


def test_scratch_query_checks_its_arguments():
    lib = cuda_ext.load()
    need = ctypes.c_uint64(5)
    assert lib.eas_dense_scratch(4, 1, 1, 1, 0, 0, 0, ctypes.byref(need)) == cuda_ext.EAS_ERR_VALUE
    assert lib.eas_dense_scratch(0, 1, 0, 1, 0, 0, 0, ctypes.byref(need)) == cuda_ext.EAS_ERR_VALUE
    assert lib.eas_dense_scratch(0, 1, 1, 1, 0, 0, 0, None) == cuda_ext.EAS_ERR_VALUE
    assert lib.eas_dense_scratch(2, 0, 1, 1, 0, 7, 15, ctypes.byref(need)) == 0 and need.value == 0


def test_kernels_read_by_plain_loads():
    """The grid before may write what a dense kernel reads while that one is being set up: its loads stay behind
    the wait, and are no read-only ones."""
    from pathlib import Path

    import easy_as_b200

    sources = sorted((Path(easy_as_b200.__file__).parent / "csrc").glob("dense*.cu*"))
    assert len(sources) >= 3
    for path in sources:
        text = path.read_text()
        assert "__ldg(" not in text and "ld.global.nc" not in text and "__restrict__" not in text, path.name
        for body in text.split("__global__ void")[1:]:
            assert "grid_order();" in body, path.name
