// The common form of the 4-bit and group norm entry points of amos_amd/ops.py in one native call each: contiguous
// tensors on the current device and its current stream.  Small operators take a few microseconds on the GPU, and
// their argument checks, allocations and foreign call took more than that in the interpreter (group norm with its
// statistics, 1 x 7 x 7 x 512: 11.1 us a call there, 6.6 here).  Every function returns None for a call it does not take,
// a wrong one among them: the caller then goes the long way, which checks, allocates and raises.
#include <ATen/ATen.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "amos_mi355x.h"

namespace {

// given by setup()
PyObject *mx_class, *get_device, *get_stream, *s_codes, *s_scales, *s_shape;
decltype(&amos_mxfp4_quantize) c_quantize;
decltype(&amos_mxfp4_dequantize) c_dequantize;
decltype(&amos_mxfp4_gemm) c_gemm;
decltype(&amos_mxfp4_gemm_workspace_bytes) c_gemm_bytes;
decltype(&amos_group_norm) c_norm;
decltype(&amos_group_norm_backward) c_norm_backward;
decltype(&amos_group_norm_workspace_bytes) c_norm_bytes;

struct NotTaken {};   // thrown inside a call: leave it to the long way

int float_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return AMOS_F32;
    case at::kHalf: return AMOS_F16;
    case at::kBFloat16: return AMOS_BF16;
    default: throw NotTaken();
  }
}
at::ScalarType dtype_of(PyObject* o) {
  if (!THPDtype_Check(o)) throw NotTaken();
  return ((THPDtype*)o)->scalar_type;
}
struct Where {
  int device = -1;
  void* stream = nullptr;
};
// a dense tensor on the device of the first one, which has to be the current device
const at::Tensor& tensor(PyObject* o, Where& w) {
  if (!THPVariable_CheckExact(o) && !THPVariable_Check(o)) throw NotTaken();
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || !t.is_contiguous()) throw NotTaken();
  if (w.device < 0) w.device = t.get_device();
  if (t.get_device() != w.device) throw NotTaken();
  return t;
}
void* pointer(const at::Tensor& t) { return t.data_ptr(); }
// the current stream, as a handle, once the tensors are known
bool current(Where& w) {
  PyObject* d = PyObject_CallNoArgs(get_device);
  if (!d) return false;
  const long now = PyLong_AsLong(d);
  if (now != w.device) {
    Py_DECREF(d);
    if (PyErr_Occurred()) return false;
    throw NotTaken();
  }
  PyObject* s = PyObject_CallOneArg(get_stream, d);
  Py_DECREF(d);
  if (!s) return false;
  w.stream = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return !PyErr_Occurred();
}
at::Tensor empty(at::IntArrayRef shape, at::ScalarType t, const Where& w) {
  return at::empty(shape, at::TensorOptions().dtype(t).device(at::Device(at::kCUDA, (at::DeviceIndex)w.device)));
}
struct Scratch {
  at::Tensor memory;
  void* at = nullptr;
  Scratch(size_t need, const Where& w) {
    if (!need) return;
    memory = empty({(int64_t)need + 255}, at::kByte, w);
    at = (void*)(((uintptr_t)memory.data_ptr() + 255) & ~(uintptr_t)255);
  }
};
template <class F>
int call(F body) {   // (without the interpreter's lock: a launch may wait for room in its queue)
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = body();
  Py_END_ALLOW_THREADS
  return rc;
}
int64_t integer(PyObject* o) {
  if (!PyLong_CheckExact(o)) throw NotTaken();
  int overflow = 0;
  const int64_t v = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (overflow) throw NotTaken();
  return v;
}

// ---- Mxfp4 ----------------------------------------------------------------------------------------
struct Mx {
  at::Tensor codes, scales;
  int64_t rows = 0, cols = 0;
};
bool is_mx(PyObject* o) { return (PyObject*)Py_TYPE(o) == mx_class; }
Mx unpack(PyObject* o, Where& w) {
  Mx q;
  PyObject *c = PyObject_GetAttr(o, s_codes), *s = c ? PyObject_GetAttr(o, s_scales) : nullptr, *shape = s ? PyObject_GetAttr(o, s_shape) : nullptr;
  bool ok = shape && THPVariable_Check(c) && THPVariable_Check(s) && PyTuple_CheckExact(shape) && PyTuple_GET_SIZE(shape) == 2;
  if (ok) {
    q.codes = THPVariable_Unpack(c);
    q.scales = THPVariable_Unpack(s);
    q.rows = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0));
    q.cols = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 1));
  }
  Py_XDECREF(c);
  Py_XDECREF(s);
  Py_XDECREF(shape);
  PyErr_Clear();
  const int64_t pitch = (q.cols + 127) / 128 * 64;
  if (!ok || q.rows < 1 || q.cols < 1) throw NotTaken();
  const auto is = [&](const at::Tensor& t, int64_t wide) {
    return t.is_cuda() && t.scalar_type() == at::kByte && t.dim() == 2 && t.size(0) == q.rows && t.size(1) == wide && t.is_contiguous();
  };
  if (!is(q.codes, pitch) || !is(q.scales, pitch / 16)) throw NotTaken();
  if (w.device < 0) w.device = q.codes.get_device();
  if (q.codes.get_device() != w.device || q.scales.get_device() != w.device) throw NotTaken();
  return q;
}
PyObject* wrap_mx(const Mx& q) {
  PyTypeObject* const type = (PyTypeObject*)mx_class;
  PyObject* const o = type->tp_alloc(type, 0);
  if (!o) return nullptr;
  PyObject *c = THPVariable_Wrap(q.codes), *s = THPVariable_Wrap(q.scales), *shape = Py_BuildValue("(LL)", (long long)q.rows, (long long)q.cols);
  const bool ok = c && s && shape && PyObject_SetAttr(o, s_codes, c) == 0 && PyObject_SetAttr(o, s_scales, s) == 0 && PyObject_SetAttr(o, s_shape, shape) == 0;
  Py_XDECREF(c);
  Py_XDECREF(s);
  Py_XDECREF(shape);
  if (!ok) {
    Py_DECREF(o);
    return nullptr;
  }
  return o;
}

// rows(codes, scales, cols): how many rows a matrix of these tensors has
PyObject* rows_of(PyObject* const* a) {
  Where w;
  const at::Tensor &codes = tensor(a[0], w), &scales = tensor(a[1], w);
  const int64_t cols = integer(a[2]), pitch = cols < 1 ? 0 : (cols + 127) / 128 * 64;
  if (!pitch || codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte || codes.dim() != 2 || scales.dim() != 2 || codes.size(0) < 1 ||
      codes.size(1) != pitch || scales.size(0) != codes.size(0) || scales.size(1) != pitch / 16)
    throw NotTaken();
  return PyLong_FromLongLong(codes.size(0));
}

// quantize(x, axis, out)
PyObject* quantize(PyObject* const* a) {
  Where w;
  const at::Tensor& x = tensor(a[0], w);
  const int64_t axis = integer(a[1]);
  if (x.dim() != 2 || x.numel() == 0 || axis < -2 || axis > 1) throw NotTaken();
  const amos_mxfp4_desc_t d = {x.size(0), x.size(1), float_code(x.scalar_type()), (int32_t)(axis & 1)};
  const int64_t rows = axis & 1 ? d.rows : d.cols, cols = axis & 1 ? d.cols : d.rows, pitch = (cols + 127) / 128 * 64;
  Mx q;
  const bool given = a[2] != Py_None;
  if (given) {
    if (!is_mx(a[2])) throw NotTaken();
    q = unpack(a[2], w);
    if (q.rows != rows || q.cols != cols) throw NotTaken();
  }
  if (!current(w)) return nullptr;
  if (!given) {
    q.rows = rows;
    q.cols = cols;
    q.codes = empty({rows, pitch}, at::kByte, w);
    q.scales = empty({rows, pitch / 16}, at::kByte, w);
  }
  if (call([&] { return c_quantize(&d, pointer(x), pointer(q.codes), pointer(q.scales), w.stream); })) throw NotTaken();
  if (!given) return wrap_mx(q);
  Py_INCREF(a[2]);
  return a[2];
}

// dequantize(q, dtype, out)
PyObject* dequantize(PyObject* const* a) {
  Where w;
  if (!is_mx(a[0])) throw NotTaken();
  const Mx q = unpack(a[0], w);
  const at::ScalarType t = dtype_of(a[1]);
  const amos_mxfp4_desc_t d = {q.rows, q.cols, float_code(t), 1};
  at::Tensor out;
  if (a[2] != Py_None) {
    out = tensor(a[2], w);
    if (out.scalar_type() != t || out.dim() != 2 || out.size(0) != q.rows || out.size(1) != q.cols) throw NotTaken();
  }
  if (!current(w)) return nullptr;
  if (!out.defined()) out = empty({q.rows, q.cols}, t, w);
  if (call([&] { return c_dequantize(&d, pointer(q.codes), pointer(q.scales), pointer(out), w.stream); })) throw NotTaken();
  if (a[2] == Py_None) return THPVariable_Wrap(out);
  Py_INCREF(a[2]);
  return a[2];
}

// gemm(a, b, out, out_dtype, add, bias)
PyObject* gemm(PyObject* const* a) {
  Where w;
  if (!is_mx(a[1])) throw NotTaken();
  const Mx b = unpack(a[1], w);
  Mx q;
  at::Tensor x;
  amos_mxfp4_gemm_desc_t d = {0, b.rows, b.cols, AMOS_MXFP4, 0};
  if (is_mx(a[0])) {
    q = unpack(a[0], w);
    d.M = q.rows;
    if (q.cols != d.K) throw NotTaken();
  } else {
    x = tensor(a[0], w);
    if (x.dim() != 2 || x.size(0) < 1 || x.size(1) != d.K) throw NotTaken();
    d.M = x.size(0);
    d.a_dtype = float_code(x.scalar_type());
  }
  const auto is_c = [&](const at::Tensor& t) { return t.dim() == 2 && t.size(0) == d.M && t.size(1) == d.N; };
  at::Tensor out, add, bias;
  at::ScalarType t;
  if (a[2] != Py_None) {
    out = tensor(a[2], w);
    if (!is_c(out)) throw NotTaken();
    t = out.scalar_type();
  } else {
    t = dtype_of(a[3]);
  }
  d.out_dtype = float_code(t);
  amos_mxfp4_epilogue_t e = {nullptr, nullptr, 0, 0};
  if (a[4] != Py_None) {
    add = tensor(a[4], w);
    if (!is_c(add)) throw NotTaken();
    e.add = pointer(add);
    e.add_dtype = float_code(add.scalar_type());
  }
  if (a[5] != Py_None) {
    bias = tensor(a[5], w);
    if (bias.dim() != 1 || bias.size(0) != d.N) throw NotTaken();
    e.bias = pointer(bias);
    e.bias_dtype = float_code(bias.scalar_type());
  }
  if (!current(w)) return nullptr;
  if (!out.defined()) out = empty({d.M, d.N}, t, w);
  const size_t need = c_gemm_bytes(&d);
  const Scratch scratch(need, w);
  const bool dense = x.defined();
  if (call([&] {
        return c_gemm(&d, e.add || e.bias ? &e : nullptr, dense ? pointer(x) : pointer(q.codes), dense ? nullptr : pointer(q.scales), pointer(b.codes),
                      pointer(b.scales), pointer(out), scratch.at, need, w.stream);
      }))
    throw NotTaken();
  if (a[2] == Py_None) return THPVariable_Wrap(out);
  Py_INCREF(a[2]);
  return a[2];
}

// ---- group norm -----------------------------------------------------------------------------------
// descriptor from x, dy or y's type, groups, coefficients, activation and layout
amos_group_norm_desc_t norm_desc(const at::Tensor& x, at::ScalarType y, PyObject* groups, const at::Tensor& weight, const at::Tensor& bias, double eps,
                                 PyObject* activation, PyObject* layout) {
  amos_group_norm_desc_t d = {};
  if (!PyUnicode_CheckExact(layout)) throw NotTaken();
  const auto is = [](PyObject* o, const char* name) { return PyUnicode_CompareWithASCIIString(o, name) == 0; };
  const bool deep = x.dim() == 5;
  if (is(layout, deep ? "ndhwc" : "nhwc")) d.layout = AMOS_LAYOUT_NHWC;
  else if (is(layout, deep ? "dhwnc" : "hwnc")) d.layout = AMOS_LAYOUT_HWNC;
  else throw NotTaken();
  if ((!deep && x.dim() != 4) || x.numel() == 0) throw NotTaken();
  const int first = d.layout == AMOS_LAYOUT_NHWC ? 1 : 0;   // of the spatial dimensions
  d.N = x.size(first ? 0 : x.dim() - 2);
  d.C = x.size(x.dim() - 1);
  d.D = deep ? x.size(first) : 1;
  d.H = x.size(first + deep);
  d.W = x.size(first + deep + 1);
  const int64_t g = integer(groups);
  if (g < 1 || g > d.C || d.C % g || g > INT32_MAX) throw NotTaken();
  d.groups = (int32_t)g;
  if (activation == Py_None) d.activation = AMOS_ACT_NONE;
  else if (!PyUnicode_CheckExact(activation)) throw NotTaken();
  else if (is(activation, "silu")) d.activation = AMOS_ACT_SILU;
  else if (is(activation, "relu")) d.activation = AMOS_ACT_RELU;
  else if (is(activation, "none")) d.activation = AMOS_ACT_NONE;
  else throw NotTaken();
  d.x_dtype = float_code(x.scalar_type());
  d.y_dtype = float_code(y);
  for (const at::Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    if (t->dim() != 1 || t->size(0) != d.C) throw NotTaken();
    d.affine_dtype = float_code(t->scalar_type());
  }
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) throw NotTaken();
  d.eps = (float)eps;
  return d;
}
void* maybe(const at::Tensor& t) { return t.defined() ? pointer(t) : nullptr; }
at::Tensor optional(PyObject* o, Where& w) { return o == Py_None ? at::Tensor() : tensor(o, w); }
PyObject* wrap_or_none(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
PyObject* triple(PyObject* a, PyObject* b, PyObject* c) {   // takes the references over
  PyObject* const r = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  Py_XDECREF(c);
  return r;
}

// group_norm(x, groups, weight, bias, eps, activation, layout, out_dtype, out, stats)
PyObject* group_norm(PyObject* const* a) {
  Where w;
  const at::Tensor& x = tensor(a[0], w);
  const at::Tensor weight = optional(a[2], w), bias = optional(a[3], w);
  if (!PyFloat_CheckExact(a[4]) || !PyBool_Check(a[9])) throw NotTaken();
  at::Tensor out = optional(a[8], w), mean, rstd;
  if (out.defined() && (out.sizes() != x.sizes() || (a[7] != Py_None && dtype_of(a[7]) != out.scalar_type()))) throw NotTaken();
  const at::ScalarType t = out.defined() ? out.scalar_type() : a[7] == Py_None ? x.scalar_type() : dtype_of(a[7]);
  const amos_group_norm_desc_t d = norm_desc(x, t, a[1], weight, bias, PyFloat_AS_DOUBLE(a[4]), a[5], a[6]);
  if (!current(w)) return nullptr;
  const bool given = out.defined(), stats = a[9] == Py_True;
  if (!given) out = empty(x.sizes(), t, w);
  if (stats) {
    mean = empty({d.N, d.groups}, at::kFloat, w);
    rstd = empty({d.N, d.groups}, at::kFloat, w);
  }
  const size_t need = c_norm_bytes(&d, 0);
  const Scratch scratch(need, w);
  if (call([&] {
        return c_norm(&d, pointer(x), maybe(weight), maybe(bias), pointer(out), (float*)maybe(mean), (float*)maybe(rstd), scratch.at, need, w.stream);
      }))
    throw NotTaken();
  PyObject* y = given ? a[8] : THPVariable_Wrap(out);
  if (given) Py_INCREF(y);
  return stats ? triple(y, THPVariable_Wrap(mean), THPVariable_Wrap(rstd)) : y;
}

// group_norm_backward(dy, x, mean, rstd, groups, weight, bias, activation, layout)
PyObject* group_norm_backward(PyObject* const* a) {
  Where w;
  const at::Tensor &dy = tensor(a[0], w), &x = tensor(a[1], w), &mean = tensor(a[2], w), &rstd = tensor(a[3], w);
  const at::Tensor weight = optional(a[5], w), bias = optional(a[6], w);
  if (dy.sizes() != x.sizes()) throw NotTaken();
  const amos_group_norm_desc_t d = norm_desc(x, dy.scalar_type(), a[4], weight, bias, 0.0, a[7], a[8]);
  for (const at::Tensor* t : {&mean, &rstd})
    if (t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != d.N || t->size(1) != d.groups) throw NotTaken();
  if (!current(w)) return nullptr;
  const at::Tensor dx = empty(x.sizes(), x.scalar_type(), w);
  at::Tensor dweight, dbias;
  if (weight.defined()) dweight = empty({d.C}, at::kFloat, w);
  if (bias.defined()) dbias = empty({d.C}, at::kFloat, w);
  const size_t need = c_norm_bytes(&d, 1);
  const Scratch scratch(need, w);
  if (call([&] {
        return c_norm_backward(&d, pointer(dy), pointer(x), maybe(weight), maybe(bias), (const float*)pointer(mean), (const float*)pointer(rstd), pointer(dx),
                               (float*)maybe(dweight), (float*)maybe(dbias), scratch.at, need, w.stream);
      }))
    throw NotTaken();
  return triple(THPVariable_Wrap(dx), wrap_or_none(dweight), wrap_or_none(dbias));
}

template <PyObject* (*BODY)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N || !mx_class) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments, or setup() has not run");
    return nullptr;
  }
  try {
    return BODY(args);
  } catch (const NotTaken&) {
    Py_RETURN_NONE;
  }
  END_HANDLE_TH_ERRORS
}

// setup(Mxfp4, current device function, current stream function, addresses of the seven C entry points)
PyObject* setup(PyObject*, PyObject* args) {
  PyObject *type, *device, *stream;
  unsigned long long at[7];
  if (!PyArg_ParseTuple(args, "OOOKKKKKKK", &type, &device, &stream, at, at + 1, at + 2, at + 3, at + 4, at + 5, at + 6)) return nullptr;
  if (!PyType_Check(type)) {
    PyErr_SetString(PyExc_TypeError, "the first argument is the Mxfp4 class");
    return nullptr;
  }
  c_quantize = (decltype(c_quantize))at[0];
  c_dequantize = (decltype(c_dequantize))at[1];
  c_gemm = (decltype(c_gemm))at[2];
  c_gemm_bytes = (decltype(c_gemm_bytes))at[3];
  c_norm = (decltype(c_norm))at[4];
  c_norm_backward = (decltype(c_norm_backward))at[5];
  c_norm_bytes = (decltype(c_norm_bytes))at[6];
  s_codes = PyUnicode_InternFromString("codes");
  s_scales = PyUnicode_InternFromString("scales");
  s_shape = PyUnicode_InternFromString("shape");
  if (!s_codes || !s_scales || !s_shape) return nullptr;
  Py_INCREF(device);
  Py_INCREF(stream);
  Py_INCREF(type);
  get_device = device;
  get_stream = stream;
  mx_class = type;
  Py_RETURN_NONE;
}

template <PyObject* (*BODY)(PyObject* const*), int N>
PyMethodDef method(const char* name, const char* doc) {
  return {name, (PyCFunction)(void (*)())(&entry<BODY, N>), METH_FASTCALL, doc};
}
PyMethodDef methods[] = {
    {"setup", setup, METH_VARARGS, "setup(Mxfp4, current device, current stream, seven addresses)"},
    method<rows_of, 3>("rows", "rows(codes, scales, cols)"),
    method<quantize, 3>("quantize", "quantize(x, axis, out)"),
    method<dequantize, 3>("dequantize", "dequantize(q, dtype, out)"),
    method<gemm, 6>("gemm", "gemm(a, b, out, out_dtype, add, bias)"),
    method<group_norm, 10>("group_norm", "group_norm(x, groups, weight, bias, eps, activation, layout, out_dtype, out, stats)"),
    method<group_norm_backward, 9>("group_norm_backward", "group_norm_backward(dy, x, mean, rstd, groups, weight, bias, activation, layout)"),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
