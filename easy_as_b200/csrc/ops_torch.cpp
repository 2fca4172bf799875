// ops_torch.cpp — the quick way of eas.ops for torch tensors: a CPython extension (module eas_ops).
//
// A call of eas.ops is checked in full in Python the first time that its operator and activation come
// with these shapes, strides, dtypes and devices.  It then leaves a plan here: the C entry point's
// argument struct but for its pointers, the scratch it needs, and which buffers may not overlap.
// Later calls find the plan and only check what addresses can make wrong; anything doubtful is
// left to the Python path, which raises or handles it.  Nothing is kept of a call's buffers.
#define PY_SSIZE_T_CLEAN
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

constexpr int kMostBuffers = 16;

struct Apart {
  int a, b;
  uint64_t na, nb;  // bytes from the first element to the last
  bool may_be_one;  // b may be the same buffer as a
};

struct Plan {
  int (*call)(const void*, void*);
  std::string rest;
  int device;
  uint64_t scratch;
  std::vector<Apart> apart;
};

using Key = std::vector<int64_t>;

struct KeyHash {
  size_t operator()(const Key& k) const {
    uint64_t h = 0x9e3779b97f4a7c15ull;
    for (int64_t v : k) h = (h ^ (uint64_t)v) * 0xff51afd7ed558ccdull, h ^= h >> 32;
    return (size_t)h;
  }
};

std::unordered_map<Key, Plan, KeyHash> g_plans;
PyTypeObject* g_parameter = nullptr;
int (*g_capturing)(void*, int*) = nullptr;

// The key of a call, and its tensors (undefined for None); false when there can be no plan for it.
bool make_key(long op, long act, PyObject* bufs, Key& key, at::Tensor* tensors) {
  if (act < 0 || !PyTuple_Check(bufs) || PyTuple_GET_SIZE(bufs) > kMostBuffers) return false;
  key.reserve(80);
  key.push_back(op * 256 + act);
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(bufs); ++i) {
    PyObject* o = PyTuple_GET_ITEM(bufs, i);
    if (o == Py_None) {
      key.push_back(-1);
      continue;
    }
    if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass) && Py_TYPE(o) != g_parameter) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_neg()) return false;
    key.push_back(((int64_t)t.dim() << 32) | ((int64_t)t.scalar_type() << 16) | (int64_t)t.get_device());
    for (int64_t v : t.sizes()) key.push_back(v);
    for (int64_t v : t.strides()) key.push_back(v);
    tensors[i] = t;
  }
  return true;
}

// quick(op, act, bufs, sync) -> None (no plan: the full path), or (status, device, stream, capturing)
PyObject* quick(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4) {
    PyErr_SetString(PyExc_TypeError, "quick(op, act, bufs, sync)");
    return nullptr;
  }
  const long op = PyLong_AsLong(args[0]), act = PyLong_AsLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (!PyBool_Check(args[3])) Py_RETURN_NONE;
  const bool sync = args[3] == Py_True;
  try {
    Key key;
    at::Tensor tensors[kMostBuffers];
    if (!make_key(op, act, args[2], key, tensors)) Py_RETURN_NONE;
    const auto it = g_plans.find(key);
    if (it == g_plans.end()) Py_RETURN_NONE;
    const Plan& p = it->second;
    const int n = (int)PyTuple_GET_SIZE(args[2]);
    uint64_t block[kMostBuffers + 1 + 64];
    uint64_t any = 0;
    for (int i = 0; i < n; ++i) {
      block[i] = tensors[i].defined() ? reinterpret_cast<uint64_t>(tensors[i].mutable_data_ptr()) : 0;
      any |= block[i];
    }
    if (any & 15) Py_RETURN_NONE;
    for (const Apart& v : p.apart) {
      const uint64_t a = block[v.a], b = block[v.b];
      if (a < b + v.nb && b < a + v.na && !(v.may_be_one && a == b)) Py_RETURN_NONE;
    }
    if (c10::cuda::current_device() != p.device || p.rest.size() > 64 * 8) Py_RETURN_NONE;
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.device);
    int capturing = 0;
    if (stream.stream()) g_capturing(stream.stream(), &capturing);
    if (capturing && sync) Py_RETURN_NONE;
    at::DataPtr scratch;  // on the launch stream: goes back to it at the end of this scope
    block[n] = 0;
    if (p.scratch) {
      scratch = c10::cuda::CUDACachingAllocator::get()->allocate(p.scratch);
      block[n] = reinterpret_cast<uint64_t>(scratch.get());
    }
    std::memcpy(block + n + 1, p.rest.data(), p.rest.size());
    // Last before the launch: behind it nothing may throw, for the full path would launch again.
    if (!sync && !capturing)  // the buffers outlive the launch wherever they were allocated
      for (int i = 0; i < n; ++i)
        if (tensors[i].defined())
          c10::cuda::CUDACachingAllocator::recordStream(tensors[i].storage().data_ptr(), stream);
    int rc;
    auto* call = p.call;
    const int device = p.device;
    Py_BEGIN_ALLOW_THREADS;
    rc = call(block, stream.stream());
    Py_END_ALLOW_THREADS;
    return Py_BuildValue("iiKi", rc, device, (unsigned long long)reinterpret_cast<uintptr_t>(stream.stream()), capturing);
  } catch (const std::exception&) {
    Py_RETURN_NONE;  // a tensor without memory of its own, no memory for the scratch, ...: the full path tells
  }
}

// leave(op, act, bufs, address, rest, device, scratch, apart): the plan of a call that passed all checks
PyObject* leave(PyObject*, PyObject* args) {
  long op, act;
  PyObject *bufs, *apart;
  unsigned long long address, scratch;
  const char* rest;
  Py_ssize_t rest_size;
  int device;
  if (!PyArg_ParseTuple(args, "llOKy#iKO", &op, &act, &bufs, &address, &rest, &rest_size, &device, &scratch, &apart))
    return nullptr;
  try {
    Key key;
    at::Tensor tensors[kMostBuffers];
    if (!make_key(op, act, bufs, key, tensors)) Py_RETURN_FALSE;
    Plan p;
    p.call = reinterpret_cast<int (*)(const void*, void*)>((uintptr_t)address);
    p.rest.assign(rest, (size_t)rest_size);
    p.device = device;
    p.scratch = scratch;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(apart); ++i) {
      Apart v;
      int one;
      unsigned long long na, nb;
      if (!PyArg_ParseTuple(PyTuple_GET_ITEM(apart, i), "iKiKp", &v.a, &na, &v.b, &nb, &one)) return nullptr;
      v.na = na, v.nb = nb, v.may_be_one = one != 0;
      p.apart.push_back(v);
    }
    if (g_plans.size() >= 4096) g_plans.clear();
    g_plans[std::move(key)] = std::move(p);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_TRUE;
}

// init(parameter_class, address of eas_stream_is_capturing)
PyObject* init(PyObject*, PyObject* args) {
  PyObject* cls;
  unsigned long long capturing;
  if (!PyArg_ParseTuple(args, "O!K", &PyType_Type, &cls, &capturing)) return nullptr;
  Py_INCREF(cls);
  g_parameter = reinterpret_cast<PyTypeObject*>(cls);
  g_capturing = reinterpret_cast<int (*)(void*, int*)>((uintptr_t)capturing);
  g_plans.clear();
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"quick", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(quick)), METH_FASTCALL, nullptr},
    {"leave", leave, METH_VARARGS, nullptr},
    {"init", init, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "eas_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_eas_ops() { return PyModule_Create(&g_module); }
