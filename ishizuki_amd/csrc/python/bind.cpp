// The attention calls from Python without ctypes: a decode step's calls cost the host more than the GPU. A call, with
// others before and after it, through ctypes and checks in Python and through this: norms and rotation of one token 11.7
// and 5.6 us, attention of one token over 777 15.4 and 10.1, a step of 16 tokens written and read back 26.4 and 10.8.
//
// Each function takes the arguments of its namesake in attention.py by position. It serves calls whose arguments fit as
// they are; for any other, and when the library does not answer with ISHZ_OK, it returns NotImplemented, and attention.py
// makes the call with its own checks, copies and errors.
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "../../../include/ishizuki_hip.h"

namespace {
struct Unfit {};  // an argument that attention.py looks at
void fits(bool ok) {
  if (!ok) throw Unfit{};
}
const at::Tensor &tensor(PyObject *o, int device) {
  fits(THPVariable_CheckExact(o));
  const at::Tensor &t = THPVariable_Unpack(o);
  fits(t.is_cuda() && t.get_device() == device);
  return t;
}
int dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return ISHZ_DT_F32;
    case at::kHalf: return ISHZ_DT_F16;
    case at::kBFloat16: return ISHZ_DT_BF16;
    default: throw Unfit{};
  }
}
int count(int64_t n) {
  fits(n >= 0 && n <= INT_MAX);
  return (int)n;
}
int whole(PyObject *o) {
  fits(PyLong_CheckExact(o));
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Unfit{};
  }
  fits(v >= INT_MIN && v <= INT_MAX);
  return (int)v;
}
double number(PyObject *o) {
  fits(PyFloat_CheckExact(o) || PyLong_CheckExact(o));
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Unfit{};
  }
  return v;
}
int truth(PyObject *o) {
  fits(PyBool_Check(o));
  return o == Py_True;
}

// [rows, heads, dim] whose rows and heads start on 16 bytes. The stride of a single row or head counts for nothing.
struct Heads {
  void *p = nullptr;
  int64_t row = 0, head = 0;
  int rows = 0, heads = 0, dim = 0, dtype = 0;
  at::ScalarType type = at::kFloat;
  Heads() = default;
  Heads(PyObject *o, int device) {
    const at::Tensor &t = tensor(o, device);
    fits(t.dim() == 3);
    type = t.scalar_type();
    dtype = dtype_of(type);
    p = t.data_ptr();
    rows = count(t.size(0)), heads = count(t.size(1)), dim = count(t.size(2));
    row = rows > 1 ? t.stride(0) : (int64_t)heads * dim, head = heads > 1 ? t.stride(1) : dim;
    const int64_t step = dtype == ISHZ_DT_F32 ? 4 : 8;
    fits(t.stride(2) == 1 && row % step == 0 && head % step == 0 && ((uintptr_t)p & 15) == 0);
  }
};
struct Turn {
  const int32_t *positions = nullptr;
  const uint64_t *turns = nullptr;
  int rot = 0;
  Turn(PyObject *at_, PyObject *table, int rows, int device) {
    if (table == Py_None) {
      fits(at_ == Py_None || THPVariable_Check(at_));
      return;
    }
    const at::Tensor &p = tensor(at_, device), &t = tensor(table, device);
    fits(t.scalar_type() == at::kLong && t.dim() == 1 && t.is_contiguous());
    fits(p.scalar_type() == at::kInt && p.dim() == 1 && p.size(0) == rows && p.is_contiguous());
    positions = p.data_ptr<int32_t>(), turns = (const uint64_t *)t.data_ptr<int64_t>(), rot = count(2 * t.size(0));
  }
};
const float *weight(PyObject *o, int dim, int device) {
  if (o == Py_None) return nullptr;
  const at::Tensor &w = tensor(o, device);
  fits(w.scalar_type() == at::kFloat && w.dim() == 1 && w.size(0) == dim && w.is_contiguous());
  return w.data_ptr<float>();
}
struct Cache {
  void *k, *v;
  float *ks, *vs;
  int format, blocks, heads, dim;
  Cache(PyObject *o, int device) {
    fits(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4);
    const at::Tensor &a = tensor(PyTuple_GET_ITEM(o, 0), device), &b = tensor(PyTuple_GET_ITEM(o, 1), device);
    const at::Tensor &c = tensor(PyTuple_GET_ITEM(o, 2), device), &d = tensor(PyTuple_GET_ITEM(o, 3), device);
    fits(a.scalar_type() == at::kChar || a.scalar_type() == at::kFloat8_e4m3fn);
    format = a.scalar_type() == at::kChar ? ISHZ_KV_INT8 : ISHZ_KV_E4M3;
    fits(a.dim() == 4 && b.dim() == 4 && c.dim() == 2 && d.dim() == 2);
    blocks = count(a.size(0)), heads = count(a.size(1)), dim = count(a.size(3));
    fits(a.size(2) == ISHZ_KV_BLOCK && b.scalar_type() == a.scalar_type() && b.size(0) == blocks && b.size(1) == heads &&
         b.size(2) == dim && b.size(3) == ISHZ_KV_BLOCK);
    for (const at::Tensor *s : {&c, &d}) fits(s->scalar_type() == at::kFloat && s->size(0) == blocks && s->size(1) == heads);
    fits(a.is_contiguous() && b.is_contiguous() && c.is_contiguous() && d.is_contiguous());
    k = a.data_ptr(), v = b.data_ptr(), ks = c.data_ptr<float>(), vs = d.data_ptr<float>();
  }
};
struct Batch {
  const int32_t *table, *lengths, *starts;
  int width, sequences, max_rows, max_length;
  Batch(PyObject *o, int device) {
    fits(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 5);
    const at::Tensor &a = tensor(PyTuple_GET_ITEM(o, 0), device), &b = tensor(PyTuple_GET_ITEM(o, 1), device);
    const at::Tensor &c = tensor(PyTuple_GET_ITEM(o, 2), device);
    fits(a.scalar_type() == at::kInt && b.scalar_type() == at::kInt && c.scalar_type() == at::kInt);
    fits(a.dim() == 2 && b.dim() == 1 && c.dim() == 1 && a.is_contiguous() && b.is_contiguous() && c.is_contiguous());
    sequences = count(b.size(0)), width = count(a.size(1));
    fits(a.size(0) == sequences && c.size(0) == (int64_t)sequences + 1);
    table = a.data_ptr<int32_t>(), lengths = b.data_ptr<int32_t>(), starts = c.data_ptr<int32_t>();
    max_rows = whole(PyTuple_GET_ITEM(o, 3)), max_length = whole(PyTuple_GET_ITEM(o, 4));
  }
};
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int device) {
  return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, device));
}
void *stream(int device) { return (void *)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

PyObject *norm_rope(int device, PyObject *const *a) {
  const Heads q(a[0], device), k(a[1], device);
  fits(k.rows == q.rows && k.dim == q.dim && k.type == q.type);
  const Turn t(a[2], a[3], q.rows, device);
  const float *const qw = weight(a[4], q.dim, device), *const kw = weight(a[5], q.dim, device);
  const double eps = number(a[6]), factor = number(a[8]);
  const int interleaved = truth(a[7]);
  const at::Tensor qo = empty({q.rows, q.heads, q.dim}, q.type, device), ko = empty({k.rows, k.heads, k.dim}, k.type, device);
  fits(ishz_norm_rope(q.p, q.row, q.head, q.heads, k.p, k.row, k.head, k.heads, q.dtype, q.rows, q.dim, t.positions, t.turns,
                      t.rot, interleaved, (float)factor, qw, kw, (float)eps, qo.data_ptr(), ko.data_ptr(), stream(device)) == ISHZ_OK);
  PyObject *const x = THPVariable_Wrap(qo), *const y = THPVariable_Wrap(ko);
  PyObject *const pair = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return pair;
}

PyObject *append(int device, PyObject *const *a) {
  const Heads k(a[0], device), v(a[1], device);
  const Cache c(a[2], device);
  const Batch b(a[3], device);
  fits(k.heads == c.heads && k.dim == c.dim && v.rows == k.rows && v.heads == k.heads && v.dim == k.dim && v.type == k.type);
  const Heads q = a[4] == Py_None ? Heads() : Heads(a[4], device);
  if (q.p || a[4] != Py_None) fits(q.rows == k.rows && q.dim == k.dim && q.type == k.type);
  const Turn t(a[5], a[6], k.rows, device);
  const float *const qw = weight(a[7], k.dim, device), *const kw = weight(a[8], k.dim, device);
  const double eps = number(a[9]), factor = number(a[11]);
  const int interleaved = truth(a[10]);
  at::Tensor out;
  if (a[4] != Py_None) out = empty({q.rows, q.heads, q.dim}, q.type, device);
  fits(ishz_kv_append(k.p, k.row, k.head, v.p, v.row, v.head, k.dtype, k.rows, c.k, c.v, c.ks, c.vs, c.format, c.blocks, c.heads,
                      c.dim, b.table, b.width, b.lengths, b.starts, b.sequences, b.max_rows, q.p, q.row, q.head, q.heads,
                      t.positions, t.turns, t.rot, interleaved, (float)factor, qw, kw, (float)eps,
                      out.defined() ? out.data_ptr() : nullptr, stream(device)) == ISHZ_OK);
  if (out.defined()) return THPVariable_Wrap(out);
  Py_RETURN_TRUE;
}

PyObject *read(int device, PyObject *const *a) {
  const Cache c(a[0], device);
  const Batch b(a[1], device);
  const int tail = a[2] == Py_None ? b.max_length : whole(a[2]);
  fits(tail >= 0 && THPDtype_Check(a[3]));
  const at::ScalarType type = reinterpret_cast<THPDtype *>(a[3])->scalar_type;
  const int dtype = dtype_of(type);
  const at::Tensor k = empty({b.sequences, tail, c.heads, c.dim}, type, device), v = empty({b.sequences, tail, c.heads, c.dim}, type, device);
  fits(ishz_kv_read(c.k, c.v, c.ks, c.vs, c.format, c.blocks, c.heads, c.dim, b.table, b.width, b.lengths, b.sequences, tail, dtype,
                    k.data_ptr(), v.data_ptr(), stream(device)) == ISHZ_OK);
  PyObject *const x = THPVariable_Wrap(k), *const y = THPVariable_Wrap(v);
  PyObject *const pair = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return pair;
}

PyObject *attend(int device, PyObject *const *a) {
  const Heads q(a[0], device);
  const Cache c(a[1], device);
  const Batch b(a[2], device);
  fits(q.dim == c.dim);
  const double scale = a[3] == Py_None ? 1.0 / std::sqrt((double)c.dim) : number(a[3]);
  const int causal = truth(a[4]), window = whole(a[5]);
  const at::Tensor out = empty({q.rows, q.heads, q.dim}, q.type, device);
  const size_t bytes = ishz_kv_attend_workspace_size(q.rows, q.heads, c.heads, c.dim, b.sequences, b.max_rows, b.max_length);
  at::Tensor ws;
  if (bytes) ws = empty({(int64_t)bytes}, at::kByte, device);
  fits(ishz_kv_attend(q.p, q.row, q.head, q.heads, q.dtype, q.rows, c.k, c.v, c.ks, c.vs, c.format, c.blocks, c.heads, c.dim, b.table,
                      b.width, b.lengths, b.starts, b.sequences, b.max_rows, b.max_length, (float)scale, causal, window,
                      out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes, stream(device)) == ISHZ_OK);
  return THPVariable_Wrap(out);
}

// No exception leaves: what goes wrong here (an allocation, too) goes wrong again, with its message, in attention.py.
template <PyObject *(*F)(int, PyObject *const *), Py_ssize_t N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    if (n == N) return F((int)c10::hip::current_device(), args);
  } catch (...) {
  }
  Py_RETURN_NOTIMPLEMENTED;
}
#define ISHZ_ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ISHZ_ENTRY(norm_rope, 9), ISHZ_ENTRY(append, 12), ISHZ_ENTRY(read, 4), ISHZ_ENTRY(attend, 6), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "The attention calls whose arguments fit as they are.", -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
