"""Dense layers of a model as operators: ``eas.ops``.

=====================  ==========================================================================
``linear``             ``z = x W^T + bias``, ``y = act(z) + residual``
``linear_backward``    ``dz = dy act'(z)``, ``dx = dz W``, ``dW = dz^T x``, ``dbias = sum of dz's rows``
``gated``              ``g = x Wg^T``, ``u = x Wu^T``, ``h = act(g) u``
``gated_backward``     ``dg = dh u act'(g)``, ``du = dh act(g)``, ``dx = dg Wg + du Wu``,
                       ``dWg = dg^T x``, ``dWu = du^T x``
=====================  ==========================================================================

The calls have the manner of kernel launches: device buffers in, results written into buffers
that the caller passes, ``_sync=True`` to wait (``False`` inside a CUDA-graph capture).  Buffers
are torch CUDA tensors (f16 or bf16, launched on torch's current stream of their device) or
``eas.Tensor`` on ``cuda`` (f16); all of one call have one dtype and one device.  Matrices may
have any row pitch.  ``x`` and the results have any number of leading dimensions, which count
together as the rows (tokens); weights are ``[outputs, inputs]``.  A result must have unit stride
along its last dimension and rows that do not overlap; an input that does not is copied first.

Sums are kept in f32 and every result is rounded once.  The backward passes also round ``dz``,
``dg`` and ``du``, which are operands of matrix products, to the operands' dtype, which adds half a
step of that dtype to the error of ``dx`` and the weights' gradients; ``dbias`` is summed from the
unrounded values.  In f16 they are rounded times a power of two, which the results are divided by, where
the largest of them would be infinite or many of them would have less than f16's full precision.
All results are the same bits on every run.

The calls are plain launches: torch's autograd does not see them (nor that a buffer was written),
and gradients come from the backward calls.

``act`` is one of ``none``, ``relu``, ``gelu`` (with erf), ``gelu_tanh``, ``silu``, ``sigmoid``.
"""

from __future__ import annotations

import ctypes
import struct
import sys
from typing import Any

from .runtime import cuda_ext, get_runtime
from .tensor import Tensor

__all__ = ["ACTIVATIONS", "gated", "gated_backward", "linear", "linear_backward"]

ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
_ACT = {name: i for i, name in enumerate(ACTIVATIONS)}

# eas_dense_scratch's numbers (include/eas_cuda.h)
_LINEAR, _GATED, _LINEAR_BACKWARD, _GATED_BACKWARD = range(4)
_DX, _DW, _DB = 1, 2, 4


class _Entry:
    """A C entry point: its argument struct is pointers (inputs, outputs, scratch), row pitches, scratch
    bytes, M, N, K, device, dtype, activation."""

    def __init__(self, op: int, name: str, buffers: int, pitches: int):
        self.op, self.name = op, name
        self.pointers = struct.Struct(f"={buffers + 1}Q")
        self.rest = struct.Struct(f"={pitches + 1}Q3I3i")


_E_LINEAR = _Entry(_LINEAR, "eas_linear", 6, 5)
_E_GATED = _Entry(_GATED, "eas_gated", 6, 6)
_E_LINEAR_BACKWARD = _Entry(_LINEAR_BACKWARD, "eas_linear_backward", 7, 6)
_E_GATED_BACKWARD = _Entry(_GATED_BACKWARD, "eas_gated_backward", 9, 9)


# The extension that repeats a checked call (csrc/ops_torch.cpp), loaded with the first torch tensor:
# None before, False where it is not built for this torch (every call then takes the full path).
_ext: Any = None
_ext_lib: Any = None


def _load_ext() -> Any:
    global _ext, _ext_lib
    import importlib.machinery
    import importlib.util

    from . import build

    _ext = False
    try:
        if build.OPS_STAMP.read_text().strip() == build.ops_hash():
            loader = importlib.machinery.ExtensionFileLoader("eas_ops", str(build.OPS))
            mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("eas_ops", loader))
            loader.exec_module(mod)
            lib = cuda_ext.load()
            mod.init(sys.modules["torch"].nn.Parameter, _address(lib.eas_stream_is_capturing))
            _ext, _ext_lib = mod, lib
    except (OSError, ImportError):
        pass
    return _ext


def _address(fn: Any) -> int:
    return int(ctypes.cast(fn, ctypes.c_void_p).value or 0)


def _quick(entry: _Entry, act: str, bufs: tuple[Any, ...], sync: bool) -> bool:
    """Make the call from the plan of an earlier one, if there is one for these buffers."""
    if not _ext or _ext_lib is not cuda_ext._lib:
        return False
    r = _ext.quick(entry.op, _ACT.get(act, -1), bufs, sync)
    if r is None:
        return False
    rc, device, stream, capturing = r
    if rc:
        cuda_ext.check(rc, entry.name)
    get_runtime().finish_native(device, stream, None, sync, capturing)
    return True


class _Rows:
    """A buffer as rows: pointer, rows, columns, row pitch in elements, leading shape."""

    __slots__ = ("ptr", "rows", "cols", "ld", "lead", "keep")

    def __init__(self, ptr: int, rows: int, cols: int, ld: int, lead: tuple[int, ...], keep: Any):
        self.ptr, self.rows, self.cols, self.ld, self.lead, self.keep = ptr, rows, cols, ld, lead, keep

    def span(self) -> int:
        """Bytes from the first element to the last."""
        return 2 * ((self.rows - 1) * self.ld + self.cols) if self.rows and self.cols else 0


class _Call:
    """The buffers of one call: checked one by one, then launched together."""

    __slots__ = ("what", "dtype", "device", "torch", "ins", "outs", "copied", "in_place")

    def __init__(self, what: str):
        self.what = what
        self.dtype: int | None = None
        self.device: int | None = None
        self.torch: Any = None   # the torch module once a torch tensor was seen
        self.ins: list[_Rows] = []
        self.outs: list[tuple[str, _Rows]] = []
        self.copied = False      # some input was copied into plain rows first
        self.in_place: tuple[_Rows, _Rows] | None = None   # an output that may be that input

    def _common(self, name: str, dtype: int, device: int) -> None:
        if self.dtype is None:
            self.dtype, self.device = dtype, device
            return
        if dtype != self.dtype:
            raise TypeError(f"{self.what}: {name!r} must have the dtype of the other buffers "
                            f"({('float16', 'bfloat16')[self.dtype]})")
        if device != self.device:
            raise ValueError(f"buffers on different devices: {self.device} and {device}")

    def _rows(self, name: str, v: Any, written: bool) -> _Rows:
        if type(v) is Tensor:
            if v.dtype.itemsize != 2:
                raise TypeError(f"{self.what}: {name!r} must be float16, got {v.dtype}")
            if v.device != "cuda":
                raise TypeError(f"{self.what}: {name!r} must be on a CUDA device")
            self._common(name, 0, v._cuda_device())
            shape = v.shape
            if not shape:
                raise ValueError(f"{self.what}: {name!r} needs at least one dimension")
            cols = shape[-1]
            lead = tuple(shape[:-1])
            rows = 1
            for d in lead:
                rows *= d
            return _Rows(v._cuda_ptr(), rows, cols, cols if rows > 1 else (cols + 7) // 8 * 8, lead, v)
        torch = sys.modules.get("torch")
        if torch is None or not isinstance(v, torch.Tensor):
            raise TypeError(f"{self.what}: expected a torch CUDA tensor or an eas.Tensor on cuda for {name!r}, "
                            f"got {type(v)!r}")
        dt = v.dtype
        if dt is torch.float16:
            code = 0
        elif dt is torch.bfloat16:
            code = 1
        else:
            raise TypeError(f"{self.what}: {name!r} must be float16 or bfloat16, got {dt}")
        if not v.is_cuda:
            raise TypeError(f"{self.what}: {name!r} must be on a CUDA device, got {v.device}")
        self.torch = torch
        self._common(name, code, v.get_device())
        if v.is_neg():   # a view whose memory holds the negatives
            if written:
                raise ValueError(f"{self.what}: {name!r} is written and must not be a negative view")
            v = v.detach().resolve_neg()
            self.copied = True
        shape = tuple(v.shape)
        n = len(shape)
        if n == 2:
            rows, cols = shape
            ld, unit = v.stride()
        elif n == 1:
            rows, cols = 1, shape[0]
            ld, unit = cols, v.stride(0)
        elif n == 0:
            raise ValueError(f"{self.what}: {name!r} needs at least one dimension")
        else:
            try:
                flat = v.detach().view(-1, shape[-1]) if v.numel() else v.detach().reshape(0, shape[-1])
            except RuntimeError:
                if written:
                    raise ValueError(f"{self.what}: the leading dimensions of {name!r} are written as one and "
                                     "must be contiguous among themselves") from None
                flat = v.detach().reshape(-1, shape[-1])
                self.copied = True
            rows, cols = flat.shape
            ld, unit = flat.stride()
            v = flat
        if rows <= 1:
            ld = (cols + 7) // 8 * 8   # no second row: any pitch, and this one suits the kernels
        if (unit != 1 and cols > 1) or ld < cols:
            if written:
                raise ValueError(f"{self.what}: {name!r} is written and needs unit stride along its last dimension "
                                 "and rows that do not overlap")
            v = v.detach().contiguous()
            ld = cols
            self.copied = True
        return _Rows(v.data_ptr(), rows, cols, ld, shape[:-1], v)

    def read(self, name: str, v: Any) -> _Rows:
        r = self._rows(name, v, False)
        self.ins.append(r)
        return r

    def write(self, name: str, v: Any) -> _Rows:
        r = self._rows(name, v, True)
        self.outs.append((name, r))
        return r

    def weight(self, name: str, r: _Rows) -> None:
        if len(r.lead) != 1:
            raise ValueError(f"{self.what}: {name!r} must be a matrix")

    def shape(self, name: str, r: _Rows, lead: tuple[int, ...], cols: int) -> None:
        if r.cols != cols or r.lead != lead:
            raise ValueError(f"{self.what}: {name!r} has shape {(*r.lead, r.cols)}, expected {(*lead, cols)}")

    def sizes(self, rows: int, n: int, k: int) -> None:
        if n == 0 or k == 0:
            raise ValueError(f"{self.what}: a layer needs at least one input and one output (got {k} and {n})")
        if max(rows, n, k) > 0x7fffff00:
            raise ValueError(f"{self.what}: a dimension exceeds 2^31 - 256")

    def no_overlap(self) -> None:
        """No output shares an element with an input or another output (but for ``in_place``)."""
        in_place = self.in_place
        for i, (name, o) in enumerate(self.outs):
            lo, hi = o.ptr, o.ptr + 2 * ((o.rows - 1) * o.ld + o.cols)
            for r in self.ins:
                if r.ptr < hi and lo < r.ptr + 2 * ((r.rows - 1) * r.ld + r.cols) and _share(o, r):
                    if in_place is None or o is not in_place[0] or r is not in_place[1] or not _same(o, r):
                        raise ValueError(f"{self.what}: {name!r} overlaps an input")
            for _n, r in self.outs[:i]:
                if r.ptr < hi and lo < r.ptr + 2 * ((r.rows - 1) * r.ld + r.cols) and _share(o, r):
                    raise ValueError(f"{self.what}: {name!r} overlaps another output")

    def launch(self, entry: _Entry, bufs: tuple[_Rows | None, ...], pitched: tuple[_Rows | None, ...],
               sizes: tuple[int, int, int], act: int, outputs: int, off: int, sync: bool, given: tuple[Any, ...]) -> None:
        rt = get_runtime()
        device = self.device
        torch = self.torch
        with rt.on_device(device):
            stream = int(torch._C._cuda_getCurrentRawStream(device)) if torch is not None else 0
            capturing = rt.check_capture(stream, sync)
            lib = rt.lib()
            need = ctypes.c_uint64()
            cuda_ext.check(lib.eas_dense_scratch(entry.op, *sizes, act, outputs, off, ctypes.byref(need)), self.what)
            nbytes, owner = need.value, None
            rest = entry.rest.pack(*(r.ld if r else 0 for r in pitched), nbytes, *sizes, device, self.dtype, act)
            pointers = [r.ptr if r else 0 for r in bufs]
            call = getattr(lib, entry.name)
            keep = None
            if not (sync or capturing):
                # buffers must outlive an asynchronous launch: torch's allocator learns which stream uses
                # them (its scratch is that stream's already), the others are kept until it is done
                held = [r.keep for r in bufs if r is not None]
                keep = [b for b in held if type(b) is Tensor]
                if torch is not None:
                    on = torch.cuda.current_stream(device)
                    for b in held:
                        if type(b) is not Tensor:
                            b.record_stream(on)
            if not nbytes:
                rc = call(entry.pointers.pack(*pointers, 0) + rest, stream)
            elif torch is not None:   # on the launch stream: the current one of this device
                owner = torch.empty(nbytes, dtype=torch.uint8, device=f"cuda:{device}")
                rc = call(entry.pointers.pack(*pointers, owner.data_ptr()) + rest, stream)
            else:
                with rt.scratch_turn:
                    ptr, owner = rt.scratch(device, stream, self.what, nbytes)
                    rc = call(entry.pointers.pack(*pointers, ptr) + rest, stream)
            cuda_ext.check(rc, self.what)
            if keep is not None and torch is None and owner is not None:
                keep.append(owner)
            rt.finish_native(device, stream, keep, sync, capturing)
        if torch is not None and not self.copied and _ext is not False and (_ext or _load_ext()):
            self._leave_plan(entry, bufs, given, act, rest, nbytes)

    def _leave_plan(self, entry: _Entry, bufs: tuple[_Rows | None, ...], given: tuple[Any, ...], act: int, rest: bytes,
                    nbytes: int) -> None:
        """Let the extension repeat this call (``given``: the buffers as they came)."""
        outs = [o for _n, o in self.outs]
        apart = []
        for i, o in enumerate(bufs):
            if o is None or all(o is not v for v in outs):
                continue
            for j, r in enumerate(bufs):
                if r is None or r is o or (j > i and any(r is v for v in outs)):
                    continue
                one = self.in_place is not None and o is self.in_place[0] and r is self.in_place[1]
                apart.append((i, o.span(), j, r.span(), one and (o.ld == r.ld or o.rows <= 1)))
        _ext.leave(entry.op, act, given, _address(getattr(_ext_lib, entry.name)), rest, self.device, nbytes, tuple(apart))


def _share(a: _Rows, b: _Rows) -> bool:
    """Whether two row sets whose address ranges meet have an element in common (False only when both
    lie in one pitch, side by side; a single row lies in any)."""
    if not a.rows or not b.rows or not a.cols or not b.cols:
        return False
    if (a.rows > 1 or b.rows > 1) and (b.ptr - a.ptr) % 2 == 0:
        ld = a.ld if a.rows > 1 else b.ld
        if b.rows == 1 or b.ld == ld:
            d = ((b.ptr - a.ptr) // 2) % ld
            return not (d >= a.cols and d + b.cols <= ld)
    return True


def _same(a: _Rows, b: _Rows) -> bool:
    return a.ptr == b.ptr and (a.ld == b.ld or a.rows <= 1)


def _activation(what: str, act: str) -> int:
    code = _ACT.get(act)
    if code is None:
        raise ValueError(f"{what}: unknown activation {act!r} (expected one of {', '.join(ACTIVATIONS)})")
    return code


def _flag(sync: Any) -> bool:
    if not isinstance(sync, bool):
        raise TypeError(f"_sync must be bool, got {type(sync)!r}")
    return sync


def _off(r: _Rows, bit: int) -> int:
    return bit if (r.ptr | (r.ld << 1)) & 15 else 0


def linear(x: Any, w: Any, y: Any, *, bias: Any = None, residual: Any = None, act: str = "none", pre: Any = None,
           _sync: bool = True) -> None:
    """``y = act(x W^T + bias) + residual``, with ``x [..., K]``, ``w [N, K]``, ``bias [N]``,
    ``residual`` and ``y [..., N]``.

    ``pre [..., N]``, if given, receives ``x W^T + bias``, which :func:`linear_backward` needs when
    there is an activation.  ``y`` may be ``residual`` itself.
    """
    given = (x, w, bias, residual, y, pre)
    if _quick(_E_LINEAR, act, given, _sync):
        return
    what = "linear"
    code, sync = _activation(what, act), _flag(_sync)
    c = _Call(what)
    X, W, Y = c.read("x", x), c.read("w", w), c.write("y", y)
    n, k = W.rows, W.cols
    c.weight("w", W)
    c.shape("x", X, X.lead, k)
    c.shape("y", Y, X.lead, n)
    B = R = P = None
    if bias is not None:
        B = c.read("bias", bias)
        c.shape("bias", B, (), n)
    if residual is not None:
        R = c.read("residual", residual)
        c.shape("residual", R, X.lead, n)
    if pre is not None:
        P = c.write("pre", pre)
        c.shape("pre", P, X.lead, n)
    c.sizes(X.rows, n, k)
    if X.rows == 0:
        return
    if R is not None:
        c.in_place = (Y, R)
    c.no_overlap()
    c.launch(_E_LINEAR, (X, W, B, R, Y, P), (X, W, R, Y, P), (X.rows, n, k), code, 0, _off(X, 1) | _off(W, 2), sync, given)


def gated(x: Any, w_gate: Any, w_up: Any, h: Any, *, act: str = "silu", gate: Any = None, up: Any = None,
          _sync: bool = True) -> None:
    """``h = act(x Wg^T) * (x Wu^T)``, with ``x [..., K]``, ``w_gate`` and ``w_up [N, K]``, ``h [..., N]``.

    ``gate`` and ``up [..., N]``, if given (both or neither), receive the two products, which
    :func:`gated_backward` needs.
    """
    given = (x, w_gate, w_up, h, gate, up)
    if _quick(_E_GATED, act, given, _sync):
        return
    what = "gated"
    code, sync = _activation(what, act), _flag(_sync)
    c = _Call(what)
    X, G, U, H = c.read("x", x), c.read("w_gate", w_gate), c.read("w_up", w_up), c.write("h", h)
    n, k = G.rows, G.cols
    c.weight("w_gate", G)
    c.shape("w_up", U, G.lead, k)
    c.shape("x", X, X.lead, k)
    c.shape("h", H, X.lead, n)
    SG = SU = None
    if (gate is None) != (up is None):
        raise ValueError("gated: pass both of gate and up, or neither")
    if gate is not None:
        SG, SU = c.write("gate", gate), c.write("up", up)
        c.shape("gate", SG, X.lead, n)
        c.shape("up", SU, X.lead, n)
    c.sizes(X.rows, n, k)
    if X.rows == 0:
        return
    c.no_overlap()
    c.launch(_E_GATED, (X, G, U, H, SG, SU), (X, G, U, H, SG, SU), (X.rows, n, k), code, 0,
             _off(X, 1) | _off(G, 2) | _off(U, 4), sync, given)


def linear_backward(dy: Any, x: Any, w: Any, *, dx: Any = None, dw: Any = None, dbias: Any = None, act: str = "none",
                    pre: Any = None, _sync: bool = True) -> None:
    """Gradients of :func:`linear`: with ``dz = dy * act'(pre)``, ``dx = dz W``, ``dw = dz^T x`` and
    ``dbias = sum of dz's rows``, each if its buffer is given.

    ``pre`` is what :func:`linear` stored there (not needed for ``act="none"``).  The gradient of
    the residual is ``dy`` itself.
    """
    given = (dy, pre, x, w, dx, dw, dbias)
    if _quick(_E_LINEAR_BACKWARD, act, given, _sync):
        return
    what = "linear_backward"
    code, sync = _activation(what, act), _flag(_sync)
    c = _Call(what)
    DY, X, W = c.read("dy", dy), c.read("x", x), c.read("w", w)
    n, k = W.rows, W.cols
    c.weight("w", W)
    c.shape("x", X, X.lead, k)
    c.shape("dy", DY, X.lead, n)
    P = DX = DW = DB = None
    if pre is not None:
        P = c.read("pre", pre)
        c.shape("pre", P, X.lead, n)
    elif code:
        raise ValueError(f"linear_backward: act={act!r} needs pre, as linear(..., pre=...) stored it")
    outputs = 0
    if dx is not None:
        DX = c.write("dx", dx)
        c.shape("dx", DX, X.lead, k)
        outputs |= _DX
    if dw is not None:
        DW = c.write("dw", dw)
        c.shape("dw", DW, W.lead, k)
        outputs |= _DW
    if dbias is not None:
        DB = c.write("dbias", dbias)
        c.shape("dbias", DB, (), n)
        outputs |= _DB
    c.sizes(X.rows, n, k)
    if not outputs:
        return
    c.no_overlap()
    c.launch(_E_LINEAR_BACKWARD, (DY, P, X, W, DX, DW, DB), (DY, P, X, W, DX, DW), (X.rows, n, k), code, outputs,
             _off(X, 1) | _off(W, 2) | _off(DY, 8), sync, given)


def gated_backward(dh: Any, x: Any, w_gate: Any, w_up: Any, gate: Any, up: Any, *, dx: Any = None,
                   dw_gate: Any = None, dw_up: Any = None, act: str = "silu", _sync: bool = True) -> None:
    """Gradients of :func:`gated`: with ``dg = dh * up * act'(gate)`` and ``du = dh * act(gate)``,
    ``dx = dg Wg + du Wu``, ``dw_gate = dg^T x`` and ``dw_up = du^T x``, each if its buffer is given.

    ``gate`` and ``up`` are what :func:`gated` stored there.
    """
    given = (dh, gate, up, x, w_gate, w_up, dx, dw_gate, dw_up)
    if _quick(_E_GATED_BACKWARD, act, given, _sync):
        return
    what = "gated_backward"
    code, sync = _activation(what, act), _flag(_sync)
    c = _Call(what)
    DH, X, G, U = c.read("dh", dh), c.read("x", x), c.read("w_gate", w_gate), c.read("w_up", w_up)
    SG, SU = c.read("gate", gate), c.read("up", up)
    n, k = G.rows, G.cols
    c.weight("w_gate", G)
    c.shape("w_up", U, G.lead, k)
    c.shape("x", X, X.lead, k)
    for name, r in (("dh", DH), ("gate", SG), ("up", SU)):
        c.shape(name, r, X.lead, n)
    DX = DG = DU = None
    outputs = 0
    if dx is not None:
        DX = c.write("dx", dx)
        c.shape("dx", DX, X.lead, k)
        outputs |= _DX
    if dw_gate is not None:
        DG = c.write("dw_gate", dw_gate)
        c.shape("dw_gate", DG, G.lead, k)
        outputs |= _DW
    if dw_up is not None:
        DU = c.write("dw_up", dw_up)
        c.shape("dw_up", DU, G.lead, k)
        outputs |= _DW
    c.sizes(X.rows, n, k)
    if not outputs:
        return
    c.no_overlap()
    c.launch(_E_GATED_BACKWARD, (DH, SG, SU, X, G, U, DX, DG, DU), (DH, SG, SU, X, G, U, DX, DG, DU), (X.rows, n, k), code,
             outputs, _off(X, 1) | _off(G, 2) | _off(U, 4) | _off(DH, 8), sync, given)
