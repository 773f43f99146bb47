// The call layer of lich_b200/microscaled.py: a callable that checks its tensors against an operator's shapes and dtypes
// and calls the C entry on their device's current stream.
//
// Small operators take a few microseconds on the GPU, and the same checks made attribute by attribute in Python take two
// (7.5 us a call against 4.5 on one host; the launch itself is 2.5).  Whatever is not the plain case goes to the wrapped
// Python operator, which knows every refusal and the rest: keyword arguments, another number of arguments, a tensor that
// does not fit, a device that is not the current one.
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <new>
#include <vector>

#include "../../include/ipc_b200.h"

namespace {

enum Kind { STORE, RESTORE, WEIGHT, BACKWARD, QUANTIZE, RESTORE4, FORWARD, KINDS };
constexpr int kTensors[KINDS] = {3, 3, 4, 5, 3, 3, 5};
constexpr int kInts[KINDS] = {3, 4, 7, 6, 5, 3, 4};
constexpr int kMost = 5;

struct Spec {
  std::vector<int64_t> shape;
  c10::ScalarType dtype;
};

struct Call {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  PyObject* op;  // the Python operator
  int kind;
  void* fn;      // its C entry
  int v[8];      // the entry's integer arguments
  float alpha;
  Spec* spec;
  // the workspace of the last stream it ran on (WEIGHT, BACKWARD), and what owns that memory
  int ws_device;
  cudaStream_t ws_stream;
  void* ws;
  size_t ws_bytes;
  PyObject* ws_owner;
};

bool fits(const at::Tensor& t, const Spec& s, int device) {
  if (!t.is_cuda() || t.scalar_type() != s.dtype || t.get_device() != device || !t.is_contiguous()) return false;
  const auto sizes = t.sizes();
  return sizes.size() == s.shape.size() && std::equal(sizes.begin(), sizes.end(), s.shape.begin());
}

PyObject* call(PyObject* self, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  Call* c = reinterpret_cast<Call*>(self);
  const int n = kTensors[c->kind];
  void* p[kMost] = {};
  int device = -1;
  cudaStream_t s = nullptr;
  bool plain = PyVectorcall_NARGS(nargsf) == n && (kwnames == nullptr || PyTuple_GET_SIZE(kwnames) == 0);
  // Nothing may leave a C function by a C++ exception, and torch throws at tensors without storage of their own (torch.vmap,
  // torch.func), at layouts that are not dense and at errors of the device: the Python operator, which meets the same, raises.
  try {
    for (int i = 0; plain && i < n; ++i) {
      if (!THPVariable_CheckExact(args[i])) {
        plain = false;
        break;
      }
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      if (i == 0) device = t.is_cuda() ? (int)t.get_device() : -1;
      plain = device >= 0 && fits(t, c->spec[i], device);
      if (plain) p[i] = t.data_ptr();
    }
    plain = plain && device == (int)c10::cuda::current_device();
    if (plain) s = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  } catch (...) {
    plain = false;
  }
  if (!plain) return PyObject_Vectorcall(c->op, args, nargsf, kwnames);
  // The workspace this call launches with.  All threads share the object, and one on another stream may replace what it
  // remembers as soon as this thread gives up the interpreter lock: nothing of *c that changes is read after that.
  void* ws = c->ws;
  size_t ws_bytes = c->ws_bytes;
  if ((c->kind == WEIGHT || c->kind == BACKWARD) && (c->ws_device != device || c->ws_stream != s)) {
    PyObject* r = PyObject_CallMethod(c->op, "_workspace", "iK", device, (unsigned long long)(uintptr_t)s);
    if (r == nullptr) return nullptr;
    unsigned long long bytes = 0;
    PyObject *at = nullptr, *owner = nullptr;
    const int ok = PyArg_ParseTuple(r, "OK|O", &at, &bytes, &owner);
    if (ok) {
      c->ws = ws = at == Py_None ? nullptr : reinterpret_cast<void*>((uintptr_t)PyLong_AsUnsignedLongLong(at));
      c->ws_bytes = ws_bytes = (size_t)bytes;
      c->ws_device = device;
      c->ws_stream = s;
      Py_XINCREF(owner);
      Py_XSETREF(c->ws_owner, owner);
    }
    Py_DECREF(r);
    if (!ok || PyErr_Occurred()) return nullptr;
  }
  const int* v = c->v;
  auto i8 = [&](int i) { return static_cast<signed char*>(p[i]); };
  auto u8 = [&](int i) { return static_cast<unsigned char*>(p[i]); };
  int rc = IPC_OK;
  PyThreadState* save = PyEval_SaveThread();  // a full launch queue blocks
  switch (c->kind) {
    case STORE:
      rc = reinterpret_cast<decltype(&ipc_mx8_store)>(c->fn)(p[0], i8(1), u8(2), v[0], v[1], v[2], s);
      break;
    case RESTORE:
      rc = reinterpret_cast<decltype(&ipc_mx8_restore)>(c->fn)(i8(0), u8(1), p[2], v[0], v[1], v[2], v[3], s);
      break;
    case WEIGHT:
      rc = reinterpret_cast<decltype(&ipc_mx8_weight)>(c->fn)(v[0], p[0], p[1], i8(2), u8(3), v[1], v[2], v[3], c->alpha, 0,
                                                              v[4], v[5], v[6], ws, ws_bytes, s);
      break;
    case BACKWARD:
      rc = reinterpret_cast<decltype(&ipc_mx8_backward)>(c->fn)(p[4], p[0], p[1], i8(2), u8(3), v[0], v[1], v[2], v[3],
                                                                v[4], v[5], ws, ws_bytes, s);
      break;
    case QUANTIZE:
      rc = reinterpret_cast<decltype(&ipc_mxfp4_quantize)>(c->fn)(p[0], u8(1), u8(2), v[0], v[1], v[2], v[3], v[4], s);
      break;
    case RESTORE4:
      rc = reinterpret_cast<decltype(&ipc_mxfp4_restore)>(c->fn)(u8(0), u8(1), p[2], v[0], v[1], v[2], s);
      break;
    default:
      rc = reinterpret_cast<decltype(&ipc_mxfp4_forward)>(c->fn)(u8(0), u8(1), u8(2), u8(3), p[4], v[0], v[1], v[2], v[3], s);
  }
  PyEval_RestoreThread(save);
  if (rc != IPC_OK) return PyObject_CallMethod(c->op, "_failed", "i", rc);
  Py_RETURN_NONE;
}

// Call(op, kind, entry address, [(shape, dtype), ...], (integers, ...), alpha)
PyObject* make(PyTypeObject* type, PyObject* args, PyObject*) {
  PyObject *op, *specs, *ints;
  int kind;
  unsigned long long fn;
  double alpha;
  if (!PyArg_ParseTuple(args, "OiKO!O!d", &op, &kind, &fn, &PyList_Type, &specs, &PyTuple_Type, &ints, &alpha)) return nullptr;
  if (kind < 0 || kind >= KINDS || PyList_GET_SIZE(specs) != kTensors[kind] || PyTuple_GET_SIZE(ints) != kInts[kind]) {
    PyErr_SetString(PyExc_ValueError, "a call's kind, tensors and integers do not belong together");
    return nullptr;
  }
  Call* c = reinterpret_cast<Call*>(type->tp_alloc(type, 0));
  if (c == nullptr) return nullptr;
  c->vectorcall = call;
  c->kind = kind;
  c->fn = reinterpret_cast<void*>((uintptr_t)fn);
  c->alpha = (float)alpha;
  c->ws_device = -1;
  c->spec = new (std::nothrow) Spec[kMost];
  if (c->spec == nullptr) {
    Py_DECREF(c);
    return PyErr_NoMemory();
  }
  for (int i = 0; i < kInts[kind]; ++i) c->v[i] = (int)PyLong_AsLong(PyTuple_GET_ITEM(ints, i));
  for (int i = 0; i < kTensors[kind] && !PyErr_Occurred(); ++i) {
    PyObject *shape, *dtype;
    if (!PyArg_ParseTuple(PyList_GET_ITEM(specs, i), "O!O", &PyTuple_Type, &shape, &dtype)) break;
    if (!THPDtype_Check(dtype)) {
      PyErr_SetString(PyExc_TypeError, "a torch.dtype is needed");
      break;
    }
    c->spec[i].dtype = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
    try {
      for (Py_ssize_t d = 0; d < PyTuple_GET_SIZE(shape); ++d)
        c->spec[i].shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, d)));
    } catch (const std::bad_alloc&) {
      PyErr_NoMemory();
    }
  }
  if (PyErr_Occurred()) {
    Py_DECREF(c);
    return nullptr;
  }
  Py_INCREF(op);
  c->op = op;
  return reinterpret_cast<PyObject*>(c);
}

void drop(PyObject* self) {
  Call* c = reinterpret_cast<Call*>(self);
  delete[] c->spec;
  Py_XDECREF(c->ws_owner);
  Py_XDECREF(c->op);
  Py_TYPE(self)->tp_free(self);
}

PyObject* attribute(PyObject* self, PyObject* name) {  // everything but the call is the operator's
  Call* c = reinterpret_cast<Call*>(self);
  PyObject* r = c->op ? PyObject_GetAttr(c->op, name) : nullptr;
  if (r != nullptr || (PyErr_Occurred() && !PyErr_ExceptionMatches(PyExc_AttributeError))) return r;
  PyErr_Clear();
  return PyObject_GenericGetAttr(self, name);
}

PyTypeObject call_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mx_call", "Checked calls of the microscaled operators.", -1, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mx_call(void) {
  call_type.tp_name = "lich_b200._mx_call.Call";
  call_type.tp_basicsize = sizeof(Call);
  call_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  call_type.tp_vectorcall_offset = offsetof(Call, vectorcall);
  call_type.tp_call = PyVectorcall_Call;
  call_type.tp_new = make;
  call_type.tp_dealloc = drop;
  call_type.tp_getattro = attribute;
  if (PyType_Ready(&call_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (m == nullptr) return nullptr;
  Py_INCREF(&call_type);
  if (PyModule_AddObject(m, "Call", reinterpret_cast<PyObject*>(&call_type)) < 0) {
    Py_DECREF(&call_type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
