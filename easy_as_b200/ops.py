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
``dg`` and ``du``, which are operands of matrix products, to the operands' dtype; ``dbias`` is
summed from the unrounded values.  All results are the same bits on every run.

``act`` is one of ``none``, ``relu``, ``gelu`` (with erf), ``gelu_tanh``, ``silu``, ``sigmoid``.
"""

from __future__ import annotations

import ctypes
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


class _Rows:
    """A buffer as rows: pointer, rows, columns, row pitch in elements, leading shape."""

    __slots__ = ("ptr", "rows", "cols", "ld", "lead", "keep")

    def __init__(self, ptr: int, rows: int, cols: int, ld: int, lead: tuple[int, ...], keep: Any):
        self.ptr, self.rows, self.cols, self.ld, self.lead, self.keep = ptr, rows, cols, ld, lead, keep


class _Call:
    """The buffers of one call: checked one by one, then launched together."""

    __slots__ = ("what", "dtype", "device", "torch", "ins", "outs")

    def __init__(self, what: str):
        self.what = what
        self.dtype: int | None = None
        self.device: int | None = None
        self.torch: Any = None   # the torch module once a torch tensor was seen
        self.ins: list[_Rows] = []
        self.outs: list[tuple[str, _Rows]] = []

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
            return _Rows(v._cuda_ptr(), rows, cols, cols, lead, v)
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
            rows, cols = flat.shape
            ld, unit = flat.stride()
            v = flat
        if rows <= 1:
            ld = cols
        if (unit != 1 and cols > 1) or ld < cols:
            if written:
                raise ValueError(f"{self.what}: {name!r} is written and needs unit stride along its last dimension "
                                 "and rows that do not overlap")
            v = v.detach().contiguous()
            ld = cols
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

    def no_overlap(self, in_place: tuple[_Rows, _Rows] | None = None) -> None:
        """No output shares an element with an input or another output (``in_place``: a pair that may be one)."""
        for i, (name, o) in enumerate(self.outs):
            lo, hi = o.ptr, o.ptr + 2 * ((o.rows - 1) * o.ld + o.cols)
            for r in self.ins:
                if r.ptr < hi and lo < r.ptr + 2 * ((r.rows - 1) * r.ld + r.cols) and _share(o, r):
                    if in_place is None or o is not in_place[0] or r is not in_place[1] or not _same(o, r):
                        raise ValueError(f"{self.what}: {name!r} overlaps an input")
            for _n, r in self.outs[:i]:
                if r.ptr < hi and lo < r.ptr + 2 * ((r.rows - 1) * r.ld + r.cols) and _share(o, r):
                    raise ValueError(f"{self.what}: {name!r} overlaps another output")

    def launch(self, entry: Any, head: tuple[Any, ...], tail: tuple[Any, ...], scratch: tuple[int, ...] | None,
               sync: bool) -> None:
        rt = get_runtime()
        device = self.device
        torch = self.torch
        with rt.on_device(device):
            stream = int(torch._C._cuda_getCurrentRawStream(device)) if torch is not None else 0
            capturing = rt.check_capture(stream, sync)
            lib = rt.lib()
            ptr, nbytes, owner = None, 0, None
            if scratch is not None:
                need = ctypes.c_uint64()
                cuda_ext.check(lib.eas_dense_scratch(*scratch, ctypes.byref(need)), self.what)
                nbytes = need.value
                if nbytes:
                    if torch is not None:   # on the launch stream: the current one of this device
                        owner = torch.empty(nbytes, dtype=torch.uint8, device=f"cuda:{device}")
                        ptr = owner.data_ptr()
                    else:
                        ptr, owner = rt.scratch(device, stream, self.what, nbytes)
            cuda_ext.check(getattr(lib, entry)(device, *head, *tail, ptr, nbytes, stream), self.what)
            keep = None
            if not (sync or capturing):
                # buffers must outlive the launch: torch's allocator learns which stream uses them (its
                # scratch is that stream's already), the others are kept until it is done
                bufs = [r.keep for r in self.ins] + [r.keep for _n, r in self.outs]
                if torch is not None:
                    on = torch.cuda.current_stream(device)
                    for b in bufs:
                        if type(b) is not Tensor:
                            b.record_stream(on)
                keep = [b for b in bufs if type(b) is Tensor]
                if torch is None and owner is not None:
                    keep.append(owner)
            rt.finish_native(device, stream, keep, sync, capturing)


def _share(a: _Rows, b: _Rows) -> bool:
    """Whether two row sets whose address ranges meet have an element in common (False only when both
    lie in one pitch, side by side)."""
    if not a.rows or not b.rows or not a.cols or not b.cols:
        return False
    if a.rows > 1 and b.rows > 1 and a.ld == b.ld and (b.ptr - a.ptr) % 2 == 0:
        d = ((b.ptr - a.ptr) // 2) % a.ld
        return not (d >= a.cols and d + b.cols <= a.ld)
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
    c.no_overlap((Y, R) if R is not None else None)
    off = _off(X, 1) | _off(W, 2)
    c.launch("eas_linear",
             (X.ptr, W.ptr, B.ptr if B else None, R.ptr if R else None, Y.ptr, P.ptr if P else None, X.rows, n, k),
             (X.ld, W.ld, R.ld if R else 0, Y.ld, P.ld if P else 0, c.dtype, code),
             (_LINEAR, X.rows, n, k, code, 0, off) if off else None, sync)


def gated(x: Any, w_gate: Any, w_up: Any, h: Any, *, act: str = "silu", gate: Any = None, up: Any = None,
          _sync: bool = True) -> None:
    """``h = act(x Wg^T) * (x Wu^T)``, with ``x [..., K]``, ``w_gate`` and ``w_up [N, K]``, ``h [..., N]``.

    ``gate`` and ``up [..., N]``, if given (both or neither), receive the two products, which
    :func:`gated_backward` needs.
    """
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
    off = _off(X, 1) | _off(G, 2) | _off(U, 4)
    c.launch("eas_gated",
             (X.ptr, G.ptr, U.ptr, H.ptr, SG.ptr if SG else None, SU.ptr if SU else None, X.rows, n, k),
             (X.ld, G.ld, U.ld, H.ld, SG.ld if SG else 0, SU.ld if SU else 0, c.dtype, code),
             (_GATED, X.rows, n, k, code, 0, off) if off else None, sync)


def linear_backward(dy: Any, x: Any, w: Any, *, dx: Any = None, dw: Any = None, dbias: Any = None, act: str = "none",
                    pre: Any = None, _sync: bool = True) -> None:
    """Gradients of :func:`linear`: with ``dz = dy * act'(pre)``, ``dx = dz W``, ``dw = dz^T x`` and
    ``dbias = sum of dz's rows``, each if its buffer is given.

    ``pre`` is what :func:`linear` stored there (not needed for ``act="none"``).  The gradient of
    the residual is ``dy`` itself.
    """
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
    off = _off(X, 1) | _off(W, 2) | _off(DY, 8)
    c.launch("eas_linear_backward",
             (DY.ptr, P.ptr if P else None, X.ptr, W.ptr, DX.ptr if DX else None, DW.ptr if DW else None,
              DB.ptr if DB else None, X.rows, n, k),
             (DY.ld, P.ld if P else 0, X.ld, W.ld, DX.ld if DX else 0, DW.ld if DW else 0, c.dtype, code),
             (_LINEAR_BACKWARD, X.rows, n, k, code, outputs, off), sync)


def gated_backward(dh: Any, x: Any, w_gate: Any, w_up: Any, gate: Any, up: Any, *, dx: Any = None,
                   dw_gate: Any = None, dw_up: Any = None, act: str = "silu", _sync: bool = True) -> None:
    """Gradients of :func:`gated`: with ``dg = dh * up * act'(gate)`` and ``du = dh * act(gate)``,
    ``dx = dg Wg + du Wu``, ``dw_gate = dg^T x`` and ``dw_up = du^T x``, each if its buffer is given.

    ``gate`` and ``up`` are what :func:`gated` stored there.
    """
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
    off = _off(X, 1) | _off(G, 2) | _off(U, 4) | _off(DH, 8)
    c.launch("eas_gated_backward",
             (DH.ptr, SG.ptr, SU.ptr, X.ptr, G.ptr, U.ptr, DX.ptr if DX else None, DG.ptr if DG else None,
              DU.ptr if DU else None, X.rows, n, k),
             (DH.ld, SG.ld, SU.ld, X.ld, G.ld, U.ld, DX.ld if DX else 0, DG.ld if DG else 0, DU.ld if DU else 0,
              c.dtype, code),
             (_GATED_BACKWARD, X.rows, n, k, code, outputs, off), sync)
