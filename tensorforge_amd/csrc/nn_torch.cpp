// The residual block's operators on torch tensors: what tforge_nn.py calls.
// Checks the tensors, allocates the results and the workspace from torch's
// allocator (which orders both with the current stream, under graph capture
// too) and calls the C ABI on torch's current stream.
//
// A call of a small operator is bound by the host, so this layer is native and
// its arguments are positional: norm of one row of 2048 into 8 bits 18.0 us a call
// with the same steps in Python (ctypes), 5.4 us here.
//
// Where an input wants a gradient, rms_norm and linear return None, and tforge_nn.py
// goes through autograd; the calls without a gradient refuse.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "tforge_hip.h"

namespace {

using at::ScalarType;
using at::Tensor;

int type_of(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return TF_T_F32;
    case ScalarType::BFloat16: return TF_T_BF16;
    case ScalarType::Half: return TF_T_F16;
    case ScalarType::Float8_e4m3fn: return TF_T_F8;
    default: return -1;
  }
}

bool half_type(ScalarType t) { return t == ScalarType::BFloat16 || t == ScalarType::Half; }

const Tensor &tensor(PyObject *o, const char *name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " is not a tensor");
  return THPVariable_Unpack(o);
}

const Tensor *optional(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }

// In reverse mode, or in forward mode (a tangent, which no_grad does not hide).
bool wants_grad(std::initializer_list<const Tensor *> all) {
  const bool reverse = at::GradMode::is_enabled();
  for (const Tensor *t : all)
    if (t && ((reverse && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

void no_gradient(const char *call, std::initializer_list<const Tensor *> all) {
  TORCH_CHECK_VALUE(!wants_grad(all), call, " has no gradient, and a tensor wants one: call it under torch.no_grad(), or on detached tensors");
}

void same_type(const Tensor &t, const char *name, ScalarType a, ScalarType b) {
  TORCH_CHECK_TYPE(t.scalar_type() == a || t.scalar_type() == b, name, " is ", t.scalar_type(), ", not ", a,
                   a == b ? "" : " or ", a == b ? "" : c10::toString(b));
}

// A tensor as rows: its leading dimensions taken together.
struct Rows {
  void *p;
  int64_t m, n, ld;
};

Rows rows(const Tensor &t, const char *name) {
  const int64_t dims = t.dim();
  TORCH_CHECK_VALUE(dims > 0, name, " has no dimension");
  const int64_t n = t.size(dims - 1);
  int64_t m = 1, ld = n;
  bool first = true;
  TORCH_CHECK_VALUE(n <= 1 || t.stride(dims - 1) == 1, name, ": the elements of a row are not next to each other (strides ",
                    t.strides(), ")");
  for (int64_t i = dims - 2; i >= 0; --i) {
    const int64_t s = t.size(i);
    if (s == 1) continue;
    if (first) ld = t.stride(i), first = false;
    else
      TORCH_CHECK_VALUE(t.numel() == 0 || t.stride(i) == ld * m, name, ": its leading dimensions are not one run of rows (strides ",
                        t.strides(), ")");
    m *= s;
  }
  TORCH_CHECK_VALUE(m <= 1 || ld >= n || n == 0, name, ": rows overlap (strides ", t.strides(), ")");
  return {t.data_ptr(), m, n, m > 1 ? ld : n};
}

Rows rows_of(const Tensor &t, const char *name, int64_t m, int64_t n, ScalarType type) {
  same_type(t, name, type, type);
  const Rows r = rows(t, name);
  TORCH_CHECK_VALUE(r.m == m && r.n == n, name, " is ", r.m, " x ", r.n, ", not ", m, " x ", n);
  return r;
}

void *vector(const Tensor &t, const char *name, int64_t n, ScalarType a, ScalarType b) {
  same_type(t, name, a, b);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1), name, " is not a contiguous vector of ", n);
  return t.data_ptr();
}

// A k x n matrix in either memory order.
struct Weights {
  void *p;
  int64_t n, ld;
  int order;
};

Weights weights(const Tensor &w, int64_t k, ScalarType type) {
  same_type(w, "w", type, type);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == k, "w is ", w.sizes(), ", not ", k, " x n");
  const int64_t n = w.size(1), s0 = w.stride(0), s1 = w.stride(1);
  if ((s0 == 1 || k <= 1) && (s1 >= k || n <= 1)) return {w.data_ptr(), n, n > 1 ? s1 : k, 1};
  TORCH_CHECK_VALUE((s1 == 1 || n <= 1) && (s0 >= n || k <= 1),
                    "w: neither its rows nor its columns are contiguous (strides ", w.strides(), ")");
  return {w.data_ptr(), n, k > 1 ? s0 : n, 0};
}

// Every tensor of a call is on the one GPU.
void on_gpu(const Tensor &x, std::initializer_list<const Tensor *> others) {
  TORCH_CHECK_VALUE(x.is_cuda(), "the tensors are on ", x.device(), ", not on a GPU");
  for (const Tensor *t : others)
    TORCH_CHECK_VALUE(!t || t->device() == x.device(), "a tensor is on ", t->device(), ", the others on ", x.device());
}

// The device the call runs on, made current for its duration, and its stream.
struct On {
  c10::OptionalDeviceGuard guard;
  void *stream;
  explicit On(const Tensor &x) {
    if (x.device().index() != c10::hip::current_device()) guard.reset_device(x.device());
    stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  }
};

// Allocated past torch's dispatcher, which would take as long again.
Tensor fresh(const Tensor &like, at::IntArrayRef size, ScalarType type) {
  return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}

// What the library refuses is a ValueError, what HIP reports a RuntimeError.
void check(int rc) {
  TORCH_CHECK_VALUE(rc != TF_E_ARG, tf_last_error());
  TORCH_CHECK(rc >= 0, tf_last_error());
}

PyObject *wrap(const Tensor *t) {
  if (!t) Py_RETURN_NONE;
  return THPVariable_Wrap(*t);
}

PyObject *tuple(std::initializer_list<const Tensor *> all) {
  PyObject *r = PyTuple_New(static_cast<Py_ssize_t>(all.size()));
  Py_ssize_t i = 0;
  for (const Tensor *t : all) PyTuple_SET_ITEM(r, i++, wrap(t));
  return r;
}

void count(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "takes ", want, " arguments, got ", got); }

int integer(PyObject *o, const char *name) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(v == static_cast<int>(v), name, " = ", v, " is out of range");
  return static_cast<int>(v);
}

double number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

c10::SmallVector<int64_t, 6> with_last(const Tensor &t, int64_t n) {
  c10::SmallVector<int64_t, 6> s(t.sizes().begin(), t.sizes().end());
  s.back() = n;
  return s;
}

void float_type(const Tensor &x, const char *name) {
  TORCH_CHECK_TYPE(x.scalar_type() == ScalarType::Float || half_type(x.scalar_type()), name, " is ", x.scalar_type(),
                   ", not Float, BFloat16 or Half");
}

// (x, weight, residual, eps, quantize) -> (y, h) or (q, scale, h)
PyObject *rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor &x = tensor(a[0], "x"), &weight = tensor(a[1], "weight");
  const Tensor *residual = optional(a[2], "residual");
  const bool quantize = a[4] == Py_True;
  float_type(x, "x");
  const ScalarType t = x.scalar_type();
  if (wants_grad({&x, &weight, residual})) Py_RETURN_NONE;
  const Rows xr = rows(x, "x");
  tf_rms_norm_args_t g{};
  g.x = xr.p, g.x_ld = xr.ld, g.rows = xr.m, g.d = xr.n, g.eps = static_cast<float>(number(a[3]));
  g.weight = vector(weight, "weight", xr.n, t, ScalarType::Float);
  g.type = type_of(t), g.weight_type = type_of(weight.scalar_type()), g.y_type = quantize ? TF_T_F8 : g.type;
  if (residual) {
    const Rows r = rows_of(*residual, "residual", xr.m, xr.n, t);
    g.residual = r.p, g.residual_ld = r.ld;
  }
  on_gpu(x, {&weight, residual});
  const On on(x);
  Tensor y = fresh(x, x.sizes(), quantize ? ScalarType::Float8_e4m3fn : t), h, scale;
  g.y = y.data_ptr(), g.y_ld = g.h_ld = xr.n;
  if (residual) h = fresh(x, x.sizes(), t), g.h = h.data_ptr();
  if (quantize) scale = fresh(x, x.sizes().slice(0, x.dim() - 1), ScalarType::Float), g.scale = scale.data_ptr<float>();
  check(tf_rms_norm(&g, on.stream));
  const Tensor *hp = residual ? &h : nullptr;
  return quantize ? tuple({&y, &scale, hp}) : tuple({&y, hp});
  END_HANDLE_TH_ERRORS
}

// (x) -> (q, scale)
PyObject *quantize_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 1);
  const Tensor &x = tensor(a[0], "x");
  float_type(x, "x");
  no_gradient("quantize_rows", {&x});
  const Rows r = rows(x, "x");
  on_gpu(x, {});
  const On on(x);
  const Tensor q = fresh(x, x.sizes(), ScalarType::Float8_e4m3fn);
  const Tensor scale = fresh(x, x.sizes().slice(0, x.dim() - 1), ScalarType::Float);
  check(tf_quantize_rows(r.p, r.ld, r.m, r.n, type_of(x.scalar_type()), q.data_ptr(), r.n, scale.data_ptr<float>(), on.stream));
  return tuple({&q, &scale});
  END_HANDLE_TH_ERRORS
}

// (dy, h, weight, eps, dh) -> (dx, dweight)
PyObject *rms_norm_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor &dy = tensor(a[0], "dy"), &h = tensor(a[1], "h"), &weight = tensor(a[2], "weight");
  const Tensor *dh = optional(a[4], "dh");
  float_type(h, "h");
  no_gradient("rms_norm_grad", {&dy, &h, &weight, dh});
  const ScalarType t = h.scalar_type();
  const Rows hr = rows(h, "h"), gr = rows_of(dy, "dy", hr.m, hr.n, t);
  tf_rms_norm_grad_args_t g{};
  g.h = hr.p, g.h_ld = hr.ld, g.rows = hr.m, g.d = hr.n, g.dy = gr.p, g.dy_ld = gr.ld, g.eps = static_cast<float>(number(a[3]));
  g.weight = vector(weight, "weight", hr.n, t, ScalarType::Float);
  g.type = type_of(t), g.weight_type = type_of(weight.scalar_type());
  if (dh) {
    const Rows r = rows_of(*dh, "dh", hr.m, hr.n, t);
    g.dh = r.p, g.dh_ld = r.ld;
  }
  on_gpu(h, {&dy, &weight, dh});
  const On on(h);
  const Tensor dx = fresh(h, h.sizes(), t), dw = fresh(h, {hr.n}, weight.scalar_type());
  g.dx = dx.data_ptr(), g.dx_ld = hr.n, g.dweight = dw.data_ptr();
  check(tf_rms_norm_grad_workspace(g.rows, g.d, &g.workspace_bytes));
  Tensor space;
  if (g.workspace_bytes) space = fresh(h, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte), g.workspace = space.data_ptr();
  check(tf_rms_norm_grad(&g, on.stream));
  return tuple({&dx, &dw});
  END_HANDLE_TH_ERRORS
}

// (x, w, bias, act, residual, keep, x_scale, w_scale, out_dtype, tile, splits) -> out or (out, z)
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w");
  const Tensor *bias = optional(a[2], "bias"), *residual = optional(a[4], "residual");
  const Tensor *xs = optional(a[6], "x_scale"), *ws = optional(a[7], "w_scale");
  const bool keep = a[5] == Py_True;
  const ScalarType t = x.scalar_type();
  const bool f8 = t == ScalarType::Float8_e4m3fn;
  TORCH_CHECK_TYPE(half_type(t) || f8, "x is ", t, ", not BFloat16, Half or Float8_e4m3fn");
  ScalarType to = f8 ? ScalarType::BFloat16 : t;
  if (a[8] != Py_None) {
    TORCH_CHECK_TYPE(THPDtype_Check(a[8]), "out_dtype is not a dtype");
    to = reinterpret_cast<THPDtype *>(a[8])->scalar_type;
    TORCH_CHECK_TYPE(half_type(to) && (f8 || to == t), "out_dtype is ", to,
                     f8 ? ", not BFloat16 or Half" : ": 16-bit products keep x's type");
  }
  TORCH_CHECK_VALUE(f8 || (!xs && !ws), "scales belong to 8-bit products");
  if (f8) no_gradient("an 8-bit product", {&x, &w, bias, residual, xs, ws});
  else if (wants_grad({&x, &w, bias, residual})) Py_RETURN_NONE;
  const Rows xr = rows(x, "x");
  const Weights wr = weights(w, xr.n, t);
  tf_linear_args_t g{};
  g.x = xr.p, g.x_ld = xr.ld, g.m = xr.m, g.k = xr.n, g.w = wr.p, g.w_ld = wr.ld, g.n = wr.n, g.w_order = wr.order;
  g.type = type_of(t), g.out_type = type_of(to), g.act = integer(a[3], "activation");
  g.tile = integer(a[9], "tile"), g.splits = integer(a[10], "splits");
  if (bias) g.bias = vector(*bias, "bias", wr.n, to, ScalarType::Float), g.bias_type = type_of(bias->scalar_type());
  if (residual) {
    const Rows r = rows_of(*residual, "residual", xr.m, wr.n, to);
    g.residual = r.p, g.residual_ld = r.ld;
  }
  if (f8) {
    TORCH_CHECK_VALUE(wr.order == 1, "8-bit weights have to lie column by column: pass weight.t() of an n x k weight");
    TORCH_CHECK_VALUE(xs && ws, "an 8-bit product needs x_scale and w_scale");
    same_type(*xs, "x_scale", ScalarType::Float, ScalarType::Float);
    TORCH_CHECK_VALUE(xs->numel() == xr.m && xs->is_contiguous(), "x_scale is not a contiguous vector of ", xr.m);
    g.x_scale = xs->data_ptr<float>();
    g.w_scale = static_cast<const float *>(vector(*ws, "w_scale", wr.n, ScalarType::Float, ScalarType::Float));
  }
  on_gpu(x, {&w, bias, residual, xs, ws});
  const On on(x);
  const auto size = with_last(x, wr.n);
  Tensor out = fresh(x, size, to), z, space;
  g.out = out.data_ptr(), g.out_ld = g.z_ld = wr.n;
  if (keep) z = fresh(x, size, to), g.z = z.data_ptr();
  check(tf_linear_workspace(&g, &g.workspace_bytes));
  if (g.workspace_bytes) {
    space = fresh(x, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte);
    g.workspace = space.data_ptr();
  }
  check(tf_linear(&g, on.stream));
  return keep ? tuple({&out, &z}) : wrap(&out);
  END_HANDLE_TH_ERRORS
}

// (dy, x, w, z, act, bias_dtype, want_dx, want_dw, tile, splits, terms) -> (dx, dw, dbias)
PyObject *linear_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor &dy = tensor(a[0], "dy"), &x = tensor(a[1], "x"), &w = tensor(a[2], "w");
  const Tensor *z = optional(a[3], "z");
  const ScalarType t = x.scalar_type();
  TORCH_CHECK_TYPE(half_type(t), "x is ", t, ", not BFloat16 or Half");
  no_gradient("linear_grad", {&dy, &x, &w, z});
  const bool want_dx = a[6] == Py_True, want_dw = a[7] == Py_True;
  const Rows xr = rows(x, "x");
  const Weights wr = weights(w, xr.n, t);
  const Rows gr = rows_of(dy, "dy", xr.m, wr.n, t);
  tf_linear_grad_args_t g{};
  g.dy = gr.p, g.dy_ld = gr.ld, g.x = xr.p, g.x_ld = xr.ld, g.w = wr.p, g.w_ld = wr.ld, g.w_order = wr.order;
  g.m = xr.m, g.n = wr.n, g.k = xr.n, g.type = type_of(t), g.act = integer(a[4], "activation");
  g.tile = integer(a[8], "tile"), g.splits = integer(a[9], "splits"), g.terms = integer(a[10], "terms");
  if (g.act) {
    TORCH_CHECK_VALUE(z, "an activation's gradient needs z: call linear with keep=True");
    const Rows r = rows_of(*z, "z", xr.m, wr.n, t);
    g.z = r.p, g.z_ld = r.ld;
  }
  ScalarType bt = t;
  const bool want_db = a[5] != Py_None;
  if (want_db) {
    TORCH_CHECK_TYPE(THPDtype_Check(a[5]), "bias_dtype is not a dtype");
    bt = reinterpret_cast<THPDtype *>(a[5])->scalar_type;
    TORCH_CHECK_TYPE(bt == t || bt == ScalarType::Float, "bias_dtype is ", bt, ", not ", t, " or Float");
  }
  on_gpu(x, {&dy, &w, z});
  const On on(x);
  Tensor dx, dw, db;
  if (want_dx) dx = fresh(x, x.sizes(), t), g.dx = dx.data_ptr(), g.dx_ld = xr.n;
  if (want_dw) {
    dw = wr.order ? fresh(x, {wr.n, xr.n}, t).t() : fresh(x, {xr.n, wr.n}, t);
    g.dw = dw.data_ptr(), g.dw_ld = wr.order ? xr.n : wr.n;
  }
  if (want_db) db = fresh(x, {wr.n}, bt), g.dbias = db.data_ptr(), g.bias_type = type_of(bt);
  check(tf_linear_grad_workspace(&g, &g.workspace_bytes));
  Tensor space;
  if (g.workspace_bytes) space = fresh(x, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte), g.workspace = space.data_ptr();
  check(tf_linear_grad(&g, on.stream));
  return tuple({want_dx ? &dx : nullptr, want_dw ? &dw : nullptr, want_db ? &db : nullptr});
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"rms_norm", reinterpret_cast<PyCFunction>(rms_norm), METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(quantize_rows), METH_FASTCALL, nullptr},
    {"rms_norm_grad", reinterpret_cast<PyCFunction>(rms_norm_grad), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(linear), METH_FASTCALL, nullptr},
    {"linear_grad", reinterpret_cast<PyCFunction>(linear_grad), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nn_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nn_torch() { return PyModule_Create(&module); }
