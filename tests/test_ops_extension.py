"""CPU: the torch extension of eas.ops, built against a stand-in for torch's headers: tensors are Python objects, and the
allocator and the stream do what a test asks of them."""

import ctypes
import importlib.machinery
import importlib.util
import shutil
import subprocess
import sys
import sysconfig
import types

import pytest

HEADERS = {
    "ATen/core/Tensor.h": r"""
#pragma once
#include <Python.h>
#include <cstdint>
#include <stdexcept>
#include <vector>
inline PyObject* standin(const char* name) {  // a new reference
  PyObject* m = PyImport_ImportModule("eas_ops_standin");
  PyObject* v = m ? PyObject_GetAttrString(m, name) : nullptr;
  Py_XDECREF(m);
  if (!v) throw std::runtime_error(name);
  return v;
}
inline long standin_number(const char* name) {
  PyObject* v = standin(name);
  const long n = PyLong_AsLong(v);
  Py_DECREF(v);
  return n;
}
namespace at {
enum Layout { kStrided };
struct DataPtr {
  void* p = nullptr;
  void* get() const { return p; }
};
struct Storage {
  DataPtr d;
  const DataPtr& data_ptr() const { return d; }
};
struct Tensor {
  bool there = false;
  int64_t ptr = 0, type = 5, device = 0, neg = 0;
  std::vector<int64_t> shape, pitch;
  bool defined() const { return there; }
  bool is_cuda() const { return true; }
  bool is_neg() const { return neg; }
  bool has_storage() const { return true; }
  Layout layout() const { return kStrided; }
  int64_t dim() const { return (int64_t)shape.size(); }
  int64_t scalar_type() const { return type; }
  int64_t get_device() const { return device; }
  const std::vector<int64_t>& sizes() const { return shape; }
  const std::vector<int64_t>& strides() const { return pitch; }
  void* mutable_data_ptr() const { return reinterpret_cast<void*>(ptr); }
  Storage storage() const { return {{reinterpret_cast<void*>(ptr)}}; }
};
}  // namespace at
""",
    "c10/cuda/CUDAStream.h": r"""
#pragma once
#include <ATen/core/Tensor.h>
namespace c10 {
using DeviceIndex = signed char;
namespace cuda {
struct CUDAStream {
  void* s;
  void* stream() const { return s; }
};
inline CUDAStream getCurrentCUDAStream(DeviceIndex) { return {reinterpret_cast<void*>(standin_number("stream"))}; }
}  // namespace cuda
}  // namespace c10
""",
    "c10/cuda/CUDAFunctions.h": r"""
#pragma once
#include <ATen/core/Tensor.h>
namespace c10::cuda { inline int current_device() { return (int)standin_number("device"); } }
""",
    "c10/cuda/CUDACachingAllocator.h": r"""
#pragma once
#include <c10/cuda/CUDAStream.h>
namespace c10::cuda::CUDACachingAllocator {
struct Allocator {
  at::DataPtr allocate(size_t) {
    if (standin_number("full")) throw std::runtime_error("no memory");
    return {reinterpret_cast<void*>(4096)};
  }
};
inline Allocator* get() {
  static Allocator a;
  return &a;
}
inline void recordStream(const at::DataPtr& p, CUDAStream) {
  PyObject* list = standin("recorded");
  PyObject* v = PyLong_FromLongLong(reinterpret_cast<long long>(p.get()));
  PyList_Append(list, v);
  Py_DECREF(v);
  Py_DECREF(list);
  if (standin_number("foreign") == reinterpret_cast<long>(p.get())) throw std::runtime_error("not this allocator's");
}
}  // namespace c10::cuda::CUDACachingAllocator
""",
    "torch/csrc/autograd/python_variable.h": r"""
#pragma once
#include <ATen/core/Tensor.h>
inline PyObject* standin_class() {
  static PyObject* cls = standin("Tensor");
  return cls;
}
#define THPVariableClass standin_class()
inline std::vector<int64_t> standin_list(PyObject* o, const char* name) {
  PyObject* v = PyObject_GetAttrString(o, name);
  std::vector<int64_t> r;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(v); ++i) r.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(v, i)));
  Py_DECREF(v);
  return r;
}
inline const at::Tensor& THPVariable_Unpack(PyObject* o) {
  static at::Tensor t;
  t.there = true;
  t.ptr = standin_list(o, "ptr")[0];
  t.neg = standin_list(o, "neg")[0];
  t.shape = standin_list(o, "shape");
  t.pitch = standin_list(o, "strides");
  return t;
}
""",
}


class FakeTensor:
    def __init__(self, ptr, shape, neg=False):
        self.ptr, self.shape, self.neg = (ptr,), shape, (int(neg),)
        self.strides = tuple(shape[1:]) + (1,)


@pytest.fixture(scope="module")
def extension(tmp_path_factory):
    from easy_as_b200 import build

    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    root = tmp_path_factory.mktemp("standin")
    for name, text in HEADERS.items():
        path = root / name
        path.parent.mkdir(parents=True, exist_ok=True)
        path.write_text(text)
    so = root / "eas_ops.so"
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-w", f"-I{root}",
                    f"-I{sysconfig.get_paths()['include']}", str(build.OPS_SOURCE), "-o", str(so)], check=True)
    module = types.ModuleType("eas_ops_standin")
    module.Tensor = FakeTensor
    sys.modules["eas_ops_standin"] = module
    loader = importlib.machinery.ExtensionFileLoader("eas_ops", str(so))
    ext = importlib.util.module_from_spec(importlib.util.spec_from_loader("eas_ops", loader))
    loader.exec_module(ext)
    yield ext, module
    del sys.modules["eas_ops_standin"]


_ENTRY = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
_CAPTURING = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int))


class Planned:
    """The extension with a plan for three matrices whose C entry counts its launches."""

    def __init__(self, extension, apart=(), scratch=256):
        self.ext, self.world = extension
        self.launches, self.status = [], 0
        self.world.stream, self.world.device, self.world.full, self.world.foreign = 64, 0, 0, -1
        self.world.recorded, self.capturing = [], 0

        def entry(args, stream):
            self.launches.append((list(ctypes.cast(args, ctypes.POINTER(ctypes.c_uint64))[:5]), stream,
                                  len(self.world.recorded)))
            return self.status

        def capturing(stream, out):
            out[0] = self.capturing
            return 0

        self.keep = _ENTRY(entry), _CAPTURING(capturing)
        address = [ctypes.cast(f, ctypes.c_void_p).value for f in self.keep]
        self.bufs = tuple(FakeTensor(p, (4, 8)) for p in (1 << 20, 2 << 20, 3 << 20))
        self.ext.init(type("Parameter", (), {}), address[1])
        assert self.ext.leave(0, 1, self.bufs, address[0], b"\x07" + bytes(7), 0, scratch, apart) is True

    def quick(self, sync=False, bufs=None):
        return self.ext.quick(0, 1, self.bufs if bufs is None else bufs, sync)


def test_a_planned_call_is_repeated(extension):
    p = Planned(extension)
    assert p.quick() == (0, 0, 64, 0) and p.quick(sync=True) == (0, 0, 64, 0)
    assert p.launches[0][0] == [1 << 20, 2 << 20, 3 << 20, 4096, 7] and p.launches[0][1] == 64
    assert len(p.launches) == 2 and p.world.recorded == [1 << 20, 2 << 20, 3 << 20]   # not for the waiting one
    p.capturing = 1
    assert p.quick() == (0, 0, 64, 1) and len(p.world.recorded) == 3
    p.status = 4
    assert p.quick() == (4, 0, 64, 1)


def test_nothing_is_launched_that_the_full_path_launches_again(extension):
    """Whatever goes wrong on the quick way goes wrong before the launch: "no plan" means that nothing ran."""
    p = Planned(extension, apart=((2, 64, 0, 64, 0),))
    for foreign in (1 << 20, 3 << 20):
        p.world.foreign = foreign               # an allocator that refuses a pointer
        assert p.quick() is None and not p.launches
    p.world.foreign, p.world.full = -1, 1       # no memory for the scratch
    assert p.quick() is None and not p.launches
    p.world.full, p.world.device = 0, 1         # another device is current
    assert p.quick() is None and not p.launches
    p.world.device, p.capturing = 0, 1          # a waiting call inside a capture
    assert p.quick(sync=True) is None and not p.launches
    p.capturing = 0
    a, b, c = p.bufs
    for bufs in ((a, b, FakeTensor((1 << 20) + 48, (4, 8))),    # the result overlaps the first
                 (a, b, FakeTensor((3 << 20) + 2, (4, 8))),     # no 16-byte boundary
                 (FakeTensor(1 << 20, (4, 8), neg=True), b, c),  # memory of the negatives
                 (a, b, FakeTensor(3 << 20, (4, 9))), (a, b, None), (a, b)):
        assert p.quick(bufs=bufs) is None and not p.launches
    p.world.recorded = []
    assert p.quick() == (0, 0, 64, 0) and len(p.launches) == 1
    assert p.launches[0][2] == 3                # the streams were told before
