"""CPU: what eas.ops hands to a stand-in for the native library, which keeps a current device as CUDA does."""

import ctypes
import sys
import threading
import time

import numpy as np
import pytest

import eas
from easy_as_b200 import ops
from easy_as_b200.runtime import cuda_ext
from easy_as_b200.tensor import Tensor


class Library:
    """The entries that an operator's call needs.  A dense entry makes the operands' device current and restores the
    one before; stream 0 is the current device's.  Each thread has a current device of its own."""

    def __init__(self, scratch=0):
        self.calls, self.need = [], scratch
        self.order = []   # launches and events by pointer and event
        self.events, self.buffers, self.status = {}, {}, {}
        self.threads = threading.local()
        self.nap = 0.0   # how long each entry lets other threads run

    @property
    def current(self):
        return getattr(self.threads, "device", 0)

    @current.setter
    def current(self, device):
        self.threads.device = device

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
        time.sleep(self.nap)
        self.calls.append(("launch", dev, stream))
        self.order.append(("launch", dev, ops._E_LINEAR.pointers.unpack_from(args)[0]))
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
        time.sleep(self.nap)
        out._obj.value = len(self.events) + 1
        self.events[out._obj.value] = self.current
        return 0

    def eas_event_record(self, ev, stream):
        if self.events[ev] != self.current and not stream:
            return cuda_ext.EAS_ERR_VALUE   # an event of another device
        self.calls.append(("record", self.current, stream))
        self.order.append(("record", self.current, ev))
        time.sleep(self.nap)
        return 0

    def eas_event_synchronize(self, ev):
        time.sleep(self.nap)
        self.calls.append(("event wait", self.events[ev]))
        self.order.append(("done", self.events[ev], ev))
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


def call(device, at=0x10000000, sync=True, owner=None):
    t = [Tensor._from_cuda_ptr(at + (i << 20) + (device << 24), s, np.float16, device, owner=owner)
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


def in_threads(count, work):
    errors = []

    def run(i):
        try:
            work(i)
        except BaseException as e:  # noqa: BLE001 (shown below)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and not any(t.is_alive() for t in threads), errors


class Owner:
    """Memory of one call's buffers: tells when it is let go."""

    def __init__(self, log, ptr):
        self.log, self.ptr = log, ptr

    def __del__(self):
        self.log.append(("released", None, self.ptr))


def test_threads_with_launches_under_way(rt, monkeypatch):
    """Four threads on four devices: buffers are let go only when an event of their device, recorded behind their
    launch, has come; the counts agree at the end, and no event is in use twice."""
    monkeypatch.setenv("EAS_MAX_IN_FLIGHT", "8")
    rt.fake.nap = 1e-4
    lib, before = rt.fake, sys.getswitchinterval()

    def work(device):
        for i in range(60):
            at = (0x100 + i) << 32
            call(device, at, sync=False, owner=Owner(lib.order, at + (device << 24)))

    sys.setswitchinterval(1e-5)
    try:
        in_threads(4, work)
    finally:
        sys.setswitchinterval(before)
    rt.synchronize()
    assert rt.in_flight() == 0 and rt._pending_n == 0 and not rt._pending
    pooled = [ev for pool in rt._event_pool.values() for ev in pool]
    assert sorted(pooled) == sorted(lib.events)
    assert all(lib.events[ev] == device for device, pool in rt._event_pool.items() for ev in pool)
    launched, covered, recorded = {}, set(), {}
    for what, device, v in lib.order:
        if what == "launch":
            launched[v] = device
        elif what == "record":
            recorded[v] = {p for p, d in launched.items() if d == device}
        elif what == "done":
            covered |= recorded[v]
        else:
            assert v in covered
            covered.discard(v)
            del launched[v]
    assert sum(c[0] == "released" for c in lib.order) == 240 and not launched


def test_a_group_is_listed_until_its_event_has_come(rt):
    """A consumer's stream that another thread makes wait meanwhile waits for it too."""
    call(0, sync=False)
    seen = []
    wait = rt.fake.eas_event_synchronize

    def event_synchronize(ev):
        other = threading.Thread(target=rt.stream_wait_pending, args=(77,))
        other.start()
        other.join(60)
        seen.append([c for c in rt.fake.calls if c[0] == "stream waits"])
        return wait(ev)

    rt.fake.eas_event_synchronize = event_synchronize
    rt.synchronize()
    assert seen == [[("stream waits", 0, 77, 0)]] and rt.in_flight() == 0


def test_threads_take_turns_with_a_streams_scratch(rt):
    """The launches of one call are queued together: another thread's call on the stream, which has the same scratch,
    queues its own before or behind them, and its growth does not free what is about to be used."""
    log, need = [], threading.local()
    entry = rt.fake._entry

    def launches(args, stream):
        scratch = ops._E_LINEAR.pointers.unpack_from(args)[-1]
        log.append((threading.get_ident(), scratch))
        time.sleep(1e-4)
        assert scratch in rt.fake.buffers       # not freed meanwhile
        log.append((threading.get_ident(), scratch))
        return entry(args, stream)

    def scratch_bytes(op, m, n, k, act, outputs, off, out):
        out._obj.value = need.bytes
        time.sleep(1e-5)
        return 0

    def work(i):
        for j in range(40):
            need.bytes = 1000 * (j // 4 + 1 + i)
            call(0)

    rt.fake.eas_linear, rt.fake.eas_dense_scratch = launches, scratch_bytes
    in_threads(4, work)
    assert len(log) == 320 and log[::2] == log[1::2]
