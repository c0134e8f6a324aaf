// torch_calls.cpp -- the row operators' calls from Python without ctypes: a
// CPython module that takes torch tensors, makes the outputs and calls the C
// entry points of libffn_b200.so (include/ffn_b200.h).
//
// A small call's kernels take a few microseconds, less than ctypes, torch's
// Python constructors and the checks in Python together (14 us for one row's
// norm).  A function here handles the plain case -- CUDA tensors of the current
// device in the shapes and types that the entry point takes as they are -- and
// returns None for anything else, which the callers in ffn_b200.py then check,
// copy or refuse.  An entry point's error comes back as its (negative) code.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ffn_b200.h"

namespace {

struct Fallback {};

const at::Tensor *tensor(PyObject *o) {  // nullptr for None
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) throw Fallback();
  return &THPVariable_Unpack(o);
}
const at::Tensor &need(PyObject *o) {
  const at::Tensor *t = tensor(o);
  if (!t) throw Fallback();
  return *t;
}
int dt_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FFN_B200_DT_F32;
    case at::kBFloat16: return FFN_B200_DT_BF16;
    case at::kHalf: return FFN_B200_DT_F16;
    default: throw Fallback();
  }
}
int device_here(const at::Tensor &t) {  // a CUDA tensor's, where it is the current one
  if (!t.is_cuda()) throw Fallback();
  const int d = t.get_device();
  if (d != c10::cuda::current_device()) throw Fallback();
  return d;
}
// Row stride of a 2-d tensor with these sizes (-1: any), contiguous inside a row.
size_t ld_of(const at::Tensor &t, int dev, at::ScalarType dt, int64_t rows, int64_t cols) {
  if (t.dim() != 2 || !t.is_cuda() || t.get_device() != dev || t.scalar_type() != dt) throw Fallback();
  const int64_t r = t.size(0), c = t.size(1), ld = t.stride(0);
  if ((rows >= 0 && r != rows) || (cols >= 0 && c != cols)) throw Fallback();
  if ((c > 1 && t.stride(1) != 1) || (r > 1 && ld < c)) throw Fallback();
  return (size_t)(r > 1 ? ld : std::max(ld, c));
}
template <typename T>
const T *vec_of(const at::Tensor &t, int dev, at::ScalarType dt, int64_t n) {
  if (!t.is_cuda() || t.get_device() != dev || t.scalar_type() != dt || t.numel() != n || !t.is_contiguous()) throw Fallback();
  return static_cast<const T *>(t.const_data_ptr());
}
const float *f32s(const at::Tensor *t, int dev, int64_t n) { return t ? vec_of<float>(*t, dev, at::kFloat, n) : nullptr; }
at::Tensor rows_new(int64_t r, int64_t c, at::ScalarType dt, int dev) {
  return at::empty({r, c}, at::TensorOptions().dtype(dt).device(at::kCUDA, dev));
}
void *stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
PyObject *code(int rc) { return PyLong_FromLong(rc); }
double number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Fallback();
  }
  return v;
}
long whole(PyObject *o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Fallback();
  }
  return v;
}

// (pre_w, post_w, alpha, beta, eps, y, residual, gate) -> (h, xn)
PyObject *block_norm(PyObject *const *a) {
  const at::Tensor *pre = tensor(a[0]), *post = tensor(a[1]), *res = tensor(a[6]), *gate = tensor(a[7]);
  const at::Tensor &y = need(a[5]);
  const int dev = device_here(y);
  ffn_b200_block_norm_desc d{};
  d.dtype = dt_of(y.scalar_type());
  const at::ScalarType st = y.scalar_type();
  const size_t ld_y = ld_of(y, dev, st, -1, -1);
  const int64_t rows = y.size(0), cols = y.size(1);
  const size_t ld_r = res ? ld_of(*res, dev, st, rows, cols) : 0;
  d.rows = rows, d.cols = cols;
  d.alpha = (float)number(a[2]), d.beta = (float)number(a[3]), d.eps = (float)number(a[4]);
  if (gate) {
    if (gate->dim() == 1 && gate->size(0) == cols) d.gate_kind = FFN_B200_GATE_CHANNEL;
    else if (gate->dim() == 2 && gate->size(0) == rows && gate->size(1) == 1) d.gate_kind = FFN_B200_GATE_TOKEN;
    else throw Fallback();
    d.gate = f32s(gate, dev, gate->numel());
  }
  d.post_w = f32s(post, dev, cols);
  d.pre_w = f32s(pre, dev, cols);
  at::Tensor h = rows_new(rows, cols, st, dev), xn;
  if (pre) xn = rows_new(rows, cols, st, dev);
  const int rc = ffn_b200_block_norm(&d, y.const_data_ptr(), ld_y, res ? res->const_data_ptr() : nullptr, ld_r, h.data_ptr(),
                                     cols, pre ? xn.data_ptr() : nullptr, cols, nullptr, 0, nullptr, stream_of(dev));
  if (rc) return code(rc);
  PyObject *out = PyTuple_New(2);
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(h));
  PyObject *second = pre ? THPVariable_Wrap(xn) : Py_None;
  if (!pre) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(out, 1, second);
  return out;
}

// (w, ld, scale, bias, groups, rows, cols, x, offsets) -> out, in x's type
PyObject *int8_linear(PyObject *const *a) {
  const at::Tensor &w = need(a[0]), &scale = need(a[2]), &x = need(a[7]);
  const at::Tensor *bias = tensor(a[3]), *off = tensor(a[8]);
  const long ld = whole(a[1]), groups = whole(a[4]), n = whole(a[5]), k = whole(a[6]);
  const int dev = device_here(x);
  if (w.get_device() != dev || w.scalar_type() != at::kChar) throw Fallback();
  const at::ScalarType st = x.scalar_type();
  const int dt = dt_of(st);
  const size_t ld_x = ld_of(x, dev, st, -1, k);
  const int64_t rows = x.size(0);
  const int32_t *po = off ? vec_of<int32_t>(*off, dev, at::kInt, groups + 1) : nullptr;
  const float *ps = f32s(&scale, dev, groups * n), *pb = f32s(bias, dev, groups * n);
  at::Tensor out = rows_new(rows, n, st, dev), ws;
  const size_t nb = ffn_b200_int8_linear_ws_bytes(rows, k, groups, po);
  if (nb) ws = at::empty({(int64_t)nb}, at::TensorOptions().dtype(at::kChar).device(at::kCUDA, dev));
  const int rc = ffn_b200_int8_linear(rows, n, k, groups, po, dt, x.const_data_ptr(), ld_x,
                                      static_cast<const int8_t *>(w.const_data_ptr()), ld, ps, pb, dt, out.data_ptr(), n,
                                      nb ? ws.data_ptr() : nullptr, nb, stream_of(dev));
  return rc ? code(rc) : THPVariable_Wrap(out);
}

// (idx, expert_begin, expert_end) -> (offsets, pos, src)
PyObject *moe_sort(PyObject *const *a) {
  const at::Tensor &idx = need(a[0]);
  const long e0 = whole(a[1]), e1 = whole(a[2]);
  const int dev = device_here(idx);
  if (idx.dim() != 2 || idx.scalar_type() != at::kInt || !idx.is_contiguous() || idx.size(1) == 0 || e1 <= e0 ||
      e1 - e0 > 4096 || e0 < 0 || e1 > 0x7fffffffL)
    throw Fallback();
  const int64_t n = idx.size(0), k = idx.size(1);
  const auto opt = at::TensorOptions().dtype(at::kInt).device(at::kCUDA, dev);
  at::Tensor off = at::empty({e1 - e0 + 1}, opt), pos = at::empty({n, k}, opt), src = at::empty({n * k}, opt);
  const int rc = ffn_b200_moe_sort(n, k, static_cast<const int32_t *>(idx.const_data_ptr()), (int32_t)e0, (int32_t)e1,
                                   static_cast<int32_t *>(off.data_ptr()), static_cast<int32_t *>(pos.data_ptr()),
                                   static_cast<int32_t *>(src.data_ptr()), stream_of(dev));
  if (rc) return code(rc);
  PyObject *out = PyTuple_New(3);
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(off));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(pos));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(src));
  return out;
}

void pairs_of(const at::Tensor &pos, int dev, int64_t &n, int64_t &k, const int32_t *&p) {
  if (pos.dim() != 2 || pos.size(1) == 0) throw Fallback();
  n = pos.size(0), k = pos.size(1);
  p = vec_of<int32_t>(pos, dev, at::kInt, n * k);
}

// (x, pos, out) -> out
PyObject *moe_permute(PyObject *const *a) {
  const at::Tensor &x = need(a[0]);
  const at::Tensor *given = tensor(a[2]);
  const int dev = device_here(x);
  int64_t n, k;
  const int32_t *p;
  pairs_of(need(a[1]), dev, n, k, p);
  const at::ScalarType st = x.scalar_type();
  const size_t es = x.element_size(), ld_x = ld_of(x, dev, st, n, -1);
  const int64_t cols = x.size(1);
  if (!given && st == at::kChar) throw Fallback();  // int8 codes keep their padded rows
  at::Tensor made;
  if (!given) made = rows_new(n * k, cols, st, dev);
  const at::Tensor &out = given ? *given : made;
  const size_t ld_o = ld_of(out, dev, st, -1, cols);
  const int rc = ffn_b200_moe_permute(n, k, cols * es, x.const_data_ptr(), ld_x * es, p, out.size(0), out.data_ptr(), ld_o * es,
                                      nullptr, nullptr, stream_of(dev));
  if (rc) return code(rc);
  if (!given) return THPVariable_Wrap(made);
  Py_INCREF(a[2]);
  return a[2];
}

// (y, pos, weight, residual) -> out
PyObject *moe_combine(PyObject *const *a) {
  const at::Tensor &y = need(a[0]);
  const at::Tensor *w = tensor(a[2]), *res = tensor(a[3]);
  const int dev = device_here(y);
  int64_t n, k;
  const int32_t *p;
  pairs_of(need(a[1]), dev, n, k, p);
  const at::ScalarType st = y.scalar_type();
  const int dt = dt_of(st);
  const size_t ld_y = ld_of(y, dev, st, -1, -1);
  const int64_t cols = y.size(1);
  const size_t ld_r = res ? ld_of(*res, dev, st, n, cols) : 0;
  const float *pw = f32s(w, dev, n * k);
  at::Tensor out = rows_new(n, cols, st, dev);
  const int rc = ffn_b200_moe_combine(n, k, cols, dt, y.const_data_ptr(), ld_y, y.size(0), p, pw,
                                      res ? res->const_data_ptr() : nullptr, ld_r, out.data_ptr(), cols, stream_of(dev));
  return rc ? code(rc) : THPVariable_Wrap(out);
}

// One call: the arguments' count checked, the plain case or None, and C++
// exceptions (torch's allocator out of memory, say) as Python ones.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *call(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return F(a);
  } catch (const Fallback &) {
    Py_RETURN_NONE;
  } catch (const c10::Error &) {
    Py_RETURN_NONE;  // the Python path meets the same error and reports it
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
#define FFN_METHOD(name, n) {#name, (PyCFunction)(void (*)(void))call<name, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FFN_METHOD(block_norm, 8), FFN_METHOD(int8_linear, 9), FFN_METHOD(moe_sort, 3),
                         FFN_METHOD(moe_permute, 3), FFN_METHOD(moe_combine, 4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ffn_b200_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ffn_b200_torch() { return PyModule_Create(&module); }
