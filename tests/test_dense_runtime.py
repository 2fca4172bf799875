"""CPU: what eas.ops hands to a stand-in for the native library, which keeps a current device as CUDA does."""

import ctypes
import sys

import numpy as np
import pytest

import eas
from easy_as_b200 import ops
from easy_as_b200.runtime import cuda_ext
from easy_as_b200.tensor import Tensor


class Library:
    """The entries that an operator's call needs.  A dense entry makes the operands' device current and restores the
    one before; stream 0 is the current device's."""

    def __init__(self, scratch=0):
        self.current, self.calls, self.need = 0, [], scratch
        self.events, self.buffers, self.status = {}, {}, {}

    def eas_get_device(self, out):
        out._obj.value = self.current
        return 0

    def eas_set_device(self, dev):
        self.current = dev
        return 0

    def eas_dense_scratch(self, op, m, n, k, act, outputs, off, out):
        out._obj.value = self.need
        return 0

    def _entry(self, args, stream):
        *_pitches, _nbytes, m, n, k, dev, _dtype, _act = ops._E_LINEAR.rest.unpack(args[ops._E_LINEAR.pointers.size:])
        self.calls.append(("launch", dev, stream))
        return 0

    eas_linear = _entry

    def eas_alloc_buffer(self, dev, nbytes, out):
        self.current = dev
        buf = ctypes.create_string_buffer(int(nbytes))
        self.buffers[ctypes.addressof(buf)] = (dev, buf)
        out._obj.value = ctypes.addressof(buf)
        return 0

    def eas_free_buffer(self, ptr):
        self.calls.append(("free", self.buffers.pop(int(ptr))[0]))
        return 0

    def eas_stream_synchronize(self, stream):
        self.calls.append(("wait", self.current, stream))
        return 0

    def eas_gemm_status(self, dev, out):
        self.calls.append(("status", dev))
        out._obj.value = self.status.pop(dev, 0)
        return 0

    def eas_event_create(self, out):
        out._obj.value = len(self.events) + 1
        self.events[out._obj.value] = self.current
        return 0

    def eas_event_record(self, ev, stream):
        if self.events[ev] != self.current and not stream:
            return cuda_ext.EAS_ERR_VALUE   # an event of another device
        self.calls.append(("record", self.current, stream))
        return 0

    def eas_event_synchronize(self, ev):
        self.calls.append(("event wait", self.events[ev]))
        return 0

    def eas_stream_wait_event(self, stream, ev):
        self.calls.append(("stream waits", self.current, stream, self.events[ev]))
        return 0

    def eas_stream_is_capturing(self, stream, out):
        out._obj.value = 0
        return 0

    def eas_last_error(self):
        return b"stand-in"


@pytest.fixture
def rt(monkeypatch):
    from easy_as_b200.runtime.cuda import CudaRuntime

    lib = Library()
    monkeypatch.setattr(cuda_ext, "_lib", lib)
    monkeypatch.setitem(sys.modules, "torch", None)   # a program without torch
    runtime = CudaRuntime()
    monkeypatch.setattr(ops, "get_runtime", lambda: runtime)
    runtime.fake = lib
    yield runtime
    runtime._pending.clear()
    runtime._bucket_keep, runtime._bucket_n = [], 0


def call(device, at=0x10000000, sync=True):
    t = [Tensor._from_cuda_ptr(at + (i << 20) + (device << 24), s, np.float16, device, owner=None)
         for i, s in enumerate([(4, 16), (8, 16), (4, 8)])]
    eas.ops.linear(*t, _sync=sync)
    return t


def test_a_waiting_call_waits_on_its_own_device(rt):
    """Whatever device is current: the wait is for the call's stream 0, and the device before is current again."""
    for device, current in ((0, 1), (1, 0), (1, 1), (3, 0)):
        rt.fake.current = current
        rt.fake.calls.clear()
        call(device)
        assert rt.fake.calls == [("launch", device, 0), ("wait", device, 0), ("status", device)]
        assert rt.fake.current == current


def test_an_asynchronous_call_is_covered_by_an_event_of_its_device(rt):
    """Also where the group of launches is closed by a launch on another device, or by a wait."""
    call(0, sync=False)
    rt.fake.current = 1
    call(1, sync=False)          # closes device 0's group while device 1 is current
    rt.fake.current = 2
    rt.synchronize()
    assert [c for c in rt.fake.calls if c[0] == "record"] == [("record", 0, 0), ("record", 1, 0)]
    assert [c for c in rt.fake.calls if c[0] == "event wait"] == [("event wait", 0), ("event wait", 1)]
    assert rt.fake.current == 2


def test_scratch_grows_behind_a_wait_on_its_device(rt):
    rt.fake.need = 1000
    call(1, sync=False)
    rt.fake.current = 0
    rt.fake.need = 5000
    rt.fake.calls.clear()
    call(1, sync=False)
    assert rt.fake.calls[:3] == [("wait", 1, 0), ("free", 1), ("launch", 1, 0)]
    rt.synchronize()


def test_a_dlpack_consumer_waits_on_the_tensors_device(rt, monkeypatch):
    """Its default stream (1) is the one of the device that it is given a tensor of."""
    monkeypatch.setattr(sys.modules["easy_as_b200.tensor"], "_runtime", lambda: rt)
    y = call(1, sync=False)[2]
    y.__dlpack__(stream=1)
    assert rt.fake.calls[-1] == ("stream waits", 1, 0, 1) and rt.fake.current == 0
