// rows.cpp — the optimizer's host path: lists of torch tensors to the C ABI's
// rows (dr_grad_tensor, dr_adamw_tensor), checked on the way.
//
// A step over many tensors asks each for its address, sizes, strides, type and
// device.  From Python that is 0.8 us a tensor, more than the GPU's work on
// small ones; here it is 0.1 us.  Tensors are read through the DLPack exchange
// functions that torch.Tensor publishes, so nothing of torch is linked.  The look
// at the lists answers only for lists that are simple (dense, contiguous, of known
// types, on one CUDA device) and otherwise returns None or False, upon which the
// Python side looks at the tensors one by one and raises or copies.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <mutex>
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
PyObject *grad_name, *is_neg_name;

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

// Whether the memory holds the values negated (the imaginary part of a lazily
// conjugated tensor, which autograd hands out too).  Such a view steps over the
// real parts, so that it is contiguous, and gets here, with one element alone.
bool negated(PyObject* o, const Seen& s) {
  if (s.n != 1) return false;
  PyObject* is = PyObject_CallMethodNoArgs(o, is_neg_name);
  if (!is) PyErr_Clear();
  const bool plain = is == Py_False;
  Py_XDECREF(is);
  return !plain;
}

char* address(const Seen& s) { return static_cast<char*>(s.t.data) + s.t.byte_offset; }

// The list's or tuple's items; nullptr for anything else.
PyObject** items(PyObject* o, Py_ssize_t& n) {
  if (!PyList_Check(o) && !PyTuple_Check(o)) return nullptr;
  n = PySequence_Fast_GET_SIZE(o);
  return PySequence_Fast_ITEMS(o);
}

// One of torch.Tensor's attributes, read by the getter that its descriptor
// names: 3.6 us for 120 gradients, 4.8 with a look-up by name each.
struct Attribute {
  PyObject* name;
  PyGetSetDef* def;  // nullptr: not such a descriptor
  bool find(PyObject* type, const char* text) {
    name = PyUnicode_InternFromString(text);
    PyObject* d = name ? PyObject_GetAttr(type, name) : nullptr;
    def = d && Py_TYPE(d) == &PyGetSetDescr_Type ? reinterpret_cast<PyGetSetDescrObject*>(d)->d_getset : nullptr;
    return d != nullptr;  // kept, as the type is
  }
  PyObject* of(PyObject* o) const { return def ? def->get(o, def->closure) : PyObject_GetAttr(o, name); }
};
Attribute requires_grad, is_leaf;

// Whether o is a leaf that autograd differentiates for: a parameter, no gradient.
bool is_parameter(PyObject* o) {
  PyObject* needs = requires_grad.of(o);
  PyObject* leaf = needs == Py_False ? Py_NewRef(Py_False) : is_leaf.of(o);
  PyErr_Clear();
  const bool gradient = needs && leaf == Py_False;
  Py_XDECREF(needs);
  Py_XDECREF(leaf);
  return !gradient;
}

// grads(tensors, written) -> (device index, dr_grad_tensor rows as bytes, whether the norm needs work), or None.
// None in the list is passed over.  written: also None where two tensors share memory, or one is a parameter.
PyObject* grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  Py_ssize_t items_n = 0, n = 0;
  PyObject** it = nargs == 2 ? items(args[0], items_n) : nullptr;
  for (Py_ssize_t i = 0; it && i < items_n; ++i) n += it[i] != Py_None;
  if (n == 0) Py_RETURN_NONE;
  const bool written = PyObject_IsTrue(args[1]) == 1;
  PyObject* bytes = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(dr_grad_tensor));
  if (!bytes) return nullptr;
  auto* rows = reinterpret_cast<dr_grad_tensor*>(PyBytes_AS_STRING(bytes));
  int32_t device = -1;
  int64_t rounded = 0;
  bool fine = true;
  for (Py_ssize_t i = 0, row = 0; fine && i < items_n && row < n; ++i) {
    if (it[i] == Py_None) continue;
    Seen s;
    fine = look(it[i], s) && (row == 0 || s.t.device.device_id == device) && !(written && is_parameter(it[i]));
    if (!fine) break;
    device = s.t.device.device_id;
    rows[row++] = {address(s), s.n, s.type, 0};
    rounded += (s.n + 2047) / 2048 * 2048;
  }
  if (fine && n > 1 && written) {
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
  const bool small = n <= DR_GRAD_NORM_SMALL_COUNT && rounded <= DR_GRAD_NORM_SMALL_ELEMENTS;
  PyObject* found = fine ? Py_BuildValue("(iOO)", (int)device, bytes, small ? Py_False : Py_True) : Py_NewRef(Py_None);
  Py_DECREF(bytes);
  return found;
}

// The C ABI's functions, from the binding that has loaded the library: called
// from here they cost 2 us less than through ctypes.
decltype(&dr_ctx_set_stream) set_stream = nullptr;
decltype(&dr_last_error) last_error = nullptr;
decltype(&dr_grad_norm) grad_norm = nullptr;
decltype(&dr_clip_grad_norm) clip_grad_norm = nullptr;
decltype(&dr_adamw_step) adamw_step = nullptr;

// bind(dr_ctx_set_stream, dr_last_error, dr_grad_norm, dr_clip_grad_norm, dr_adamw_step): their addresses.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d, e;
  if (!PyArg_ParseTuple(args, "KKKKK", &a, &b, &c, &d, &e)) return nullptr;
  set_stream = reinterpret_cast<decltype(set_stream)>(a);
  last_error = reinterpret_cast<decltype(last_error)>(b);
  grad_norm = reinterpret_cast<decltype(grad_norm)>(c);
  clip_grad_norm = reinterpret_cast<decltype(clip_grad_norm)>(d);
  adamw_step = reinterpret_cast<decltype(adamw_step)>(e);
  Py_RETURN_NONE;
}

template <typename T>
T* pointer(PyObject* o) {
  return o == Py_None ? nullptr : static_cast<T*>(PyLong_AsVoidPtr(o));
}

// Torch's current stream of the device; false with an exception set.
bool current_stream(long device, void** stream) {
  if (api->current_work_stream(kCuda, (int32_t)device, stream) == 0) return true;
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "no current stream");
  return false;
}

// stream(device) -> torch's current stream of the device, as a number.
PyObject* stream(PyObject*, PyObject* device) {
  void* now = nullptr;
  const long index = PyLong_AsLong(device);
  if (PyErr_Occurred() || !current_stream(index, &now)) return nullptr;
  return PyLong_FromVoidPtr(now);
}

// A context serves one call at a time, and keeps the stream and the last error
// of it.  These contexts are used from here alone, and a call of any thread has
// its turn from setting the stream to copying the error; it waits for it and
// launches without the GIL.
std::mutex turn;

// None, or (status, message).
template <typename Call>
PyObject* launch(dr_ctx* ctx, void* stream, Call call) {
  dr_status st;
  char text[512] = "";
  Py_BEGIN_ALLOW_THREADS
  {
    std::lock_guard<std::mutex> mine(turn);
    set_stream(ctx, stream);
    st = call();
    if (st != DR_OK) snprintf(text, sizeof text, "%s", last_error(ctx));
  }
  Py_END_ALLOW_THREADS
  if (st == DR_OK) Py_RETURN_NONE;
  return Py_BuildValue("(is)", (int)st, text);
}

// norm(ctx, device, rows, max_norm, norm, work) -> None or (status, message): dr_grad_norm, or with max_norm > 0
// dr_clip_grad_norm, of the rows (bytes) that grads() or the Python side made.
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6 || !PyBytes_Check(args[2]) || !set_stream) {
    PyErr_SetString(PyExc_TypeError, "norm(ctx, device, rows, max_norm, norm, work)");
    return nullptr;
  }
  auto* ctx = pointer<dr_ctx>(args[0]);
  const long device = PyLong_AsLong(args[1]);
  const auto* rows = reinterpret_cast<const dr_grad_tensor*>(PyBytes_AS_STRING(args[2]));
  const int count = (int)(PyBytes_GET_SIZE(args[2]) / (Py_ssize_t)sizeof(dr_grad_tensor));
  const double max_norm = PyFloat_AsDouble(args[3]);
  auto* out = pointer<float>(args[4]);
  auto* work = pointer<void>(args[5]);
  void* stream = nullptr;
  if (PyErr_Occurred() || !current_stream(device, &stream)) return nullptr;
  return launch(ctx, stream, [&] {
    return max_norm > 0.0 ? clip_grad_norm(ctx, rows, count, max_norm, out, work)
                          : grad_norm(ctx, rows, count, out, work);
  });
}

// step(params, grads, table, device, ctx, lr, lr_device, beta1, beta2, eps, bits, max_norm, norm, work, ticket)
// -> None or (status, message), or False.  Looks each parameter (its address is its row's, see below) and gradient
// over, fills the rows' grad and grad_type and calls dr_adamw_step.  grads None: the parameters' .grad.  params None:
// the rows (bytes) are filled, and False does not come back.
PyObject* step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 15 || !set_stream) {
    PyErr_SetString(PyExc_TypeError, "step: 15 arguments");
    return nullptr;
  }
  auto* ctx = pointer<dr_ctx>(args[4]);
  const long device = PyLong_AsLong(args[3]);
  const double lr = PyFloat_AsDouble(args[5]), beta1 = PyFloat_AsDouble(args[7]), beta2 = PyFloat_AsDouble(args[8]);
  const double eps = PyFloat_AsDouble(args[9]), max_norm = PyFloat_AsDouble(args[11]);
  const int bits = (int)PyLong_AsLong(args[10]);
  auto* lr_device = pointer<const float>(args[6]);
  auto* out = pointer<float>(args[12]);
  auto* work = pointer<void>(args[13]);
  auto* ticket = pointer<uint32_t>(args[14]);
  if (PyErr_Occurred()) return nullptr;
  Py_buffer table;
  Py_ssize_t n = 0, ng = 0;
  const bool ready = args[0] == Py_None;
  PyObject** ps = ready ? nullptr : items(args[0], n);
  PyObject** gs = args[1] != Py_None ? items(args[1], ng) : nullptr;
  if (!ready && (!ps || (args[1] != Py_None && (!gs || ng != n)))) Py_RETURN_FALSE;
  if (PyObject_GetBuffer(args[2], &table, ready ? PyBUF_SIMPLE : PyBUF_WRITABLE) != 0) return nullptr;
  if (ready) n = table.len / (Py_ssize_t)sizeof(dr_adamw_tensor);
  bool fine = table.len >= n * (Py_ssize_t)sizeof(dr_adamw_tensor);
  auto* rows = static_cast<dr_adamw_tensor*>(table.buf);
  for (Py_ssize_t i = 0; fine && !ready && i < n; ++i) {
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
           (g.type == p.type || g.type == DR_F32 || p.type == DR_F32) && !negated(grad, g);
    if (fine) {
      rows[i].grad = address(g);
      rows[i].grad_type = g.type;
    }
    if (!gs) Py_DECREF(grad);  // the parameter holds it
  }
  PyObject* result = nullptr;
  void* stream = nullptr;
  if (!fine)
    result = Py_NewRef(Py_False);
  else if (current_stream(device, &stream))
    result = launch(ctx, stream, [&] {
      return adamw_step(ctx, rows, (int)n, lr, lr_device, beta1, beta2, eps, bits, max_norm, out, work, ticket);
    });
  PyBuffer_Release(&table);
  return result;
}

PyMethodDef methods[] = {
    {"grads", (PyCFunction)(void (*)(void))grads, METH_FASTCALL, "tensors, written -> (device, rows, needs work) or None"},
    {"bind", bind, METH_VARARGS, "addresses of dr_ctx_set_stream, dr_last_error, dr_grad_norm, dr_clip_grad_norm, dr_adamw_step"},
    {"stream", stream, METH_O, "device -> its current stream"},
    {"norm", (PyCFunction)(void (*)(void))norm, METH_FASTCALL, "ctx, device, rows, max_norm, norm, work -> None or (status, message)"},
    {"step", (PyCFunction)(void (*)(void))step, METH_FASTCALL, "params, grads, table, ... -> None, (status, message) or False"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", "Tensors to the C ABI's rows.", -1, methods,
                      nullptr,               nullptr, nullptr,                         nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rows() {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* type = torch ? PyObject_GetAttrString(torch, "Tensor") : nullptr;
  Py_XDECREF(torch);
  if (!type) return nullptr;
  PyObject* capsule = PyObject_GetAttrString(type, "__dlpack_c_exchange_api__");
  api = capsule ? static_cast<const DLPackExchangeAPI*>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api")) : nullptr;
  Py_XDECREF(capsule);
  if (!api || api->major != 1 || !api->dltensor_from_py_object_no_sync || !api->current_work_stream) {
    PyErr_SetString(PyExc_ImportError, "torch has no DLPack exchange table of version 1");
    return nullptr;
  }
  tensor_type = reinterpret_cast<PyTypeObject*>(type);
  grad_name = PyUnicode_InternFromString("grad");
  is_neg_name = PyUnicode_InternFromString("is_neg");
  const bool named = grad_name && is_neg_name && requires_grad.find(type, "requires_grad") && is_leaf.find(type, "is_leaf");
  return named ? PyModule_Create(&module) : nullptr;
}
