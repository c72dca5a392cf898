// rows.cpp — the optimizer's host path: lists of torch tensors to the C ABI's
// rows (dr_grad_tensor, dr_adamw_tensor), checked on the way.
//
// A step over many tensors asks each for its address, sizes, strides, type and
// device.  From Python that is 0.8 us a tensor, more than the GPU's work on
// small ones; here it is 0.1 us.  Tensors are read through the DLPack exchange
// functions that torch.Tensor publishes, so nothing of torch is linked.  Every
// function answers only for lists that are simple (dense, contiguous, of known
// types, on one CUDA device) and otherwise returns None or -1, upon which the
// Python side looks at the tensors one by one and raises or copies.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cstdint>
#include <new>

#include "diffrast.h"

namespace {

// DLPack's structs and exchange table, as its specification lays them out.
struct DLDevice {
  int32_t device_type, device_id;
};
struct DLDataType {
  uint8_t code, bits;
  uint16_t lanes;
};
struct DLTensor {
  void* data;
  DLDevice device;
  int32_t ndim;
  DLDataType dtype;
  int64_t* shape;
  int64_t* strides;
  uint64_t byte_offset;
};
struct DLPackExchangeAPI {
  uint32_t major, minor;
  void* prev_api;
  void* managed_tensor_allocator;
  void* managed_tensor_from_py_object_no_sync;
  void* managed_tensor_to_py_object_no_sync;
  int (*dltensor_from_py_object_no_sync)(void* py_object, DLTensor* out);
  int (*current_work_stream)(int32_t device_type, int32_t device_id, void** out);
};
constexpr int32_t kCuda = 2;
constexpr uint8_t kFloat = 2, kBfloat = 4;

const DLPackExchangeAPI* api = nullptr;
PyTypeObject* tensor_type = nullptr;
PyObject* grad_name = nullptr;

// What a row needs of a tensor; false where it is not a simple one.
struct Seen {
  DLTensor t;
  int64_t n;
  int32_t type, bytes;
};

bool look(PyObject* o, Seen& s) {
  if (!PyObject_TypeCheck(o, tensor_type)) return false;
  if (api->dltensor_from_py_object_no_sync(o, &s.t) != 0) {
    PyErr_Clear();
    return false;
  }
  const DLTensor& t = s.t;
  if (t.device.device_type != kCuda || t.dtype.lanes != 1) return false;
  if (t.dtype.code == kFloat && t.dtype.bits == 32) s.type = DR_F32;
  else if (t.dtype.code == kBfloat && t.dtype.bits == 16) s.type = DR_BF16;
  else if (t.dtype.code == kFloat && t.dtype.bits == 16) s.type = DR_F16;
  else return false;
  s.bytes = t.dtype.bits / 8;
  s.n = 1;
  for (int d = 0; d < t.ndim; ++d) s.n *= t.shape[d];
  if (t.strides && s.n > 1) {
    int64_t expect = 1;
    for (int d = t.ndim - 1; d >= 0; --d) {
      if (t.shape[d] != 1 && t.strides[d] != expect) return false;
      expect *= t.shape[d];
    }
  }
  return true;
}

char* address(const Seen& s) { return static_cast<char*>(s.t.data) + s.t.byte_offset; }

// The list's or tuple's items; nullptr for anything else.
PyObject** items(PyObject* o, Py_ssize_t& n) {
  if (!PyList_Check(o) && !PyTuple_Check(o)) return nullptr;
  n = PySequence_Fast_GET_SIZE(o);
  return PySequence_Fast_ITEMS(o);
}

// grads(tensors, apart) -> (device index, dr_grad_tensor rows as bytes), or
// None.  apart: also None where two tensors share memory.
PyObject* grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  Py_ssize_t n = 0;
  PyObject** it = nargs == 2 ? items(args[0], n) : nullptr;
  if (!it || n == 0) Py_RETURN_NONE;
  PyObject* bytes = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(dr_grad_tensor));
  if (!bytes) return nullptr;
  auto* rows = reinterpret_cast<dr_grad_tensor*>(PyBytes_AS_STRING(bytes));
  int32_t device = -1;
  bool fine = true;
  for (Py_ssize_t i = 0; fine && i < n; ++i) {
    Seen s;
    fine = look(it[i], s) && (i == 0 || s.t.device.device_id == device);
    if (!fine) break;
    device = s.t.device.device_id;
    rows[i] = {address(s), s.n, s.type, 0};
  }
  if (fine && n > 1 && PyObject_IsTrue(args[1]) == 1) {
    struct Span {
      uintptr_t begin, end;
    };
    Span* spans = new (std::nothrow) Span[n];
    fine = spans != nullptr;
    Py_ssize_t k = 0;
    for (Py_ssize_t i = 0; fine && i < n; ++i)
      if (rows[i].n) {
        const uintptr_t b = (uintptr_t)rows[i].data;
        spans[k++] = {b, b + (uintptr_t)rows[i].n * (rows[i].type == DR_F32 ? 4 : 2)};
      }
    if (fine) std::sort(spans, spans + k, [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (Py_ssize_t i = 1; i < k; ++i) fine = fine && spans[i - 1].end <= spans[i].begin;
    delete[] spans;
  }
  PyObject* found = fine ? Py_BuildValue("(iO)", (int)device, bytes) : Py_NewRef(Py_None);
  Py_DECREF(bytes);
  return found;
}

// step(params, grads or None, table, device) -> 0, or -1: looks each parameter
// (its address is its row's, see below) and gradient over and fills the rows'
// grad and grad_type.  grads None: the parameters' .grad.
PyObject* step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  Py_ssize_t n = 0, ng = 0;
  PyObject** ps = nargs == 4 ? items(args[0], n) : nullptr;
  PyObject** gs = nargs == 4 && args[1] != Py_None ? items(args[1], ng) : nullptr;
  if (!ps || (args[1] != Py_None && (!gs || ng != n))) return PyLong_FromLong(-1);
  Py_buffer table;
  if (PyObject_GetBuffer(args[2], &table, PyBUF_WRITABLE) != 0) return nullptr;
  const long device = PyLong_AsLong(args[3]);
  bool fine = table.len >= n * (Py_ssize_t)sizeof(dr_adamw_tensor);
  auto* rows = static_cast<dr_adamw_tensor*>(table.buf);
  for (Py_ssize_t i = 0; fine && i < n; ++i) {
    Seen p, g;
    // The caller's memory is held since the optimizer was made, so nothing
    // else can have come to its address.
    fine = look(ps[i], p) && address(p) == rows[i].param && p.n == rows[i].n && p.type == rows[i].param_type &&
           p.t.device.device_id == device;
    if (!fine) break;
    PyObject* grad = gs ? gs[i] : PyObject_GetAttr(ps[i], grad_name);
    if (!grad) {
      PyErr_Clear();
      fine = false;
      break;
    }
    fine = look(grad, g) && g.t.device.device_id == device && g.t.ndim == p.t.ndim &&
           std::equal(g.t.shape, g.t.shape + g.t.ndim, p.t.shape) &&
           (g.type == p.type || g.type == DR_F32 || p.type == DR_F32);
    if (fine) {
      rows[i].grad = address(g);
      rows[i].grad_type = g.type;
    }
    if (!gs) Py_DECREF(grad);  // the parameter holds it
  }
  PyBuffer_Release(&table);
  return PyLong_FromLong(fine ? 0 : -1);
}

PyMethodDef methods[] = {
    {"grads", (PyCFunction)(void (*)(void))grads, METH_FASTCALL, "tensors, apart -> (device, rows) or None"},
    {"step", (PyCFunction)(void (*)(void))step, METH_FASTCALL, "params, grads or None, table, device -> 0 or -1"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", "Tensors to the C ABI's rows.", -1, methods,
                      nullptr,               nullptr, nullptr,                         nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rows() {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* type = torch ? PyObject_GetAttrString(torch, "Tensor") : nullptr;
  Py_XDECREF(torch);
  PyObject* capsule = type ? PyObject_GetAttrString(type, "__dlpack_c_exchange_api__") : nullptr;
  if (!capsule) return nullptr;
  api = static_cast<const DLPackExchangeAPI*>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
  Py_DECREF(capsule);
  if (!api) return nullptr;
  if (api->major != 1 || !api->dltensor_from_py_object_no_sync) {
    PyErr_SetString(PyExc_ImportError, "torch's DLPack exchange table is of another version");
    return nullptr;
  }
  tensor_type = reinterpret_cast<PyTypeObject*>(type);
  grad_name = PyUnicode_InternFromString("grad");
  return grad_name ? PyModule_Create(&module) : nullptr;
}
