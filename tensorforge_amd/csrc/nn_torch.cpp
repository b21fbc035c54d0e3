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
// goes through autograd; linear_xent's is here; the calls without a gradient refuse.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
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
    case ScalarType::Char: return TF_T_I8;
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

ScalarType eight_bits(PyObject *o) {
  TORCH_CHECK_TYPE(THPDtype_Check(o), "the 8-bit type is not a dtype");
  const ScalarType to = reinterpret_cast<THPDtype *>(o)->scalar_type;
  TORCH_CHECK_TYPE(to == ScalarType::Float8_e4m3fn || to == ScalarType::Char, "8-bit rows are Float8_e4m3fn or Char, not ", to);
  return to;
}
// quantize: false, true (e4m3) or the 8-bit type.
bool wants_eight_bits(PyObject *o, ScalarType &to) {
  if (o == Py_False) return false;
  if (THPDtype_Check(o)) return to = eight_bits(o), true;
  const int truth = o == Py_True ? 1 : PyObject_IsTrue(o);
  if (truth < 0) throw python_error();
  if (truth) to = ScalarType::Float8_e4m3fn;
  return truth != 0;
}

// (x, weight, residual, eps, quantize) -> (y, h) or (q, scale, h)
PyObject *rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor &x = tensor(a[0], "x"), &weight = tensor(a[1], "weight");
  const Tensor *residual = optional(a[2], "residual");
  float_type(x, "x");
  const ScalarType t = x.scalar_type();
  ScalarType to = t;
  const bool quantize = wants_eight_bits(a[4], to);
  if (wants_grad({&x, &weight, residual})) Py_RETURN_NONE;
  const Rows xr = rows(x, "x");
  tf_rms_norm_args_t g{};
  g.x = xr.p, g.x_ld = xr.ld, g.rows = xr.m, g.d = xr.n, g.eps = static_cast<float>(number(a[3]));
  g.weight = vector(weight, "weight", xr.n, t, ScalarType::Float);
  g.type = type_of(t), g.weight_type = type_of(weight.scalar_type()), g.y_type = type_of(to);
  if (residual) {
    const Rows r = rows_of(*residual, "residual", xr.m, xr.n, t);
    g.residual = r.p, g.residual_ld = r.ld;
  }
  on_gpu(x, {&weight, residual});
  const On on(x);
  Tensor y = fresh(x, x.sizes(), to), h, scale;
  g.y = y.data_ptr(), g.y_ld = g.h_ld = xr.n;
  if (residual) h = fresh(x, x.sizes(), t), g.h = h.data_ptr();
  if (quantize) scale = fresh(x, x.sizes().slice(0, x.dim() - 1), ScalarType::Float), g.scale = scale.data_ptr<float>();
  check(tf_rms_norm(&g, on.stream));
  const Tensor *hp = residual ? &h : nullptr;
  return quantize ? tuple({&y, &scale, hp}) : tuple({&y, hp});
  END_HANDLE_TH_ERRORS
}

// (x, dtype) -> (q, scale)
PyObject *quantize_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 2);
  const Tensor &x = tensor(a[0], "x");
  float_type(x, "x");
  const ScalarType to = eight_bits(a[1]);
  no_gradient("quantize_rows", {&x});
  const Rows r = rows(x, "x");
  on_gpu(x, {});
  const On on(x);
  const Tensor q = fresh(x, x.sizes(), to);
  const Tensor scale = fresh(x, x.sizes().slice(0, x.dim() - 1), ScalarType::Float);
  check(tf_quantize_rows_to(r.p, r.ld, r.m, r.n, type_of(x.scalar_type()), q.data_ptr(), r.n, type_of(to), scale.data_ptr<float>(),
                            on.stream));
  return tuple({&q, &scale});
  END_HANDLE_TH_ERRORS
}

// What rows x d values take in 8 bits, as one contiguous tensor of bytes.
int64_t kept_bytes(int64_t m, int64_t n) {
  long long bytes;
  check(tf_keep8_bytes(m, n, &bytes));
  return bytes;
}
void *kept_rows(const Tensor &t, const char *name, int64_t m, int64_t n) {
  same_type(t, name, ScalarType::Byte, ScalarType::Byte);
  const int64_t bytes = kept_bytes(m, n);
  TORCH_CHECK_VALUE(t.is_contiguous() && t.numel() == bytes, name, ", ", m, " x ", n, " kept in 8 bits, is not ", bytes, " contiguous bytes");
  return t.data_ptr();
}

// (x, positive, masked) -> bytes
PyObject *keep8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 3);
  const Tensor &x = tensor(a[0], "x");
  float_type(x, "x");
  no_gradient("keep8", {&x});
  const Rows r = rows(x, "x");
  on_gpu(x, {});
  const On on(x);
  const Tensor kept = fresh(x, {kept_bytes(r.m, r.n)}, ScalarType::Byte);
  const auto keep = a[2] == Py_True ? tf_keep8_masked : tf_keep8;
  check(keep(r.p, r.ld, r.m, r.n, type_of(x.scalar_type()), a[1] == Py_True, kept.data_ptr(), on.stream));
  return wrap(&kept);
  END_HANDLE_TH_ERRORS
}

// (bytes, shape, dtype) -> x
PyObject *restore8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 3);
  const Tensor &kept = tensor(a[0], "kept");
  TORCH_CHECK_TYPE(PyTuple_Check(a[1]) && THPDtype_Check(a[2]), "shape is not a tuple, or dtype not a dtype");
  c10::SmallVector<int64_t, 6> size;
  int64_t m = 1;
  const Py_ssize_t dims = PyTuple_GET_SIZE(a[1]);
  TORCH_CHECK_VALUE(dims > 0, "the shape has no dimension");
  for (Py_ssize_t i = 0; i < dims; ++i) {
    const int64_t s = PyLong_AsLongLong(PyTuple_GET_ITEM(a[1], i));
    if (s == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(s >= 0 && s <= (1LL << 30) && (i + 1 == dims || s * m <= (1LL << 30)), "the shape's sizes are out of range");
    size.push_back(s);
    if (i + 1 < dims) m *= s;
  }
  const ScalarType t = reinterpret_cast<THPDtype *>(a[2])->scalar_type;
  TORCH_CHECK_TYPE(t == ScalarType::Float || half_type(t), "what is kept is Float, BFloat16 or Half, not ", t);
  const void *p = kept_rows(kept, "kept", m, size.back());
  on_gpu(kept, {});
  const On on(kept);
  const Tensor x = fresh(kept, size, t);
  check(tf_restore8(p, m, size.back(), type_of(t), x.data_ptr(), size.back(), on.stream));
  return wrap(&x);
  END_HANDLE_TH_ERRORS
}

// (dy, h, weight, eps, dh) -> (dx, dweight); kept: h is what keep8 gave.
template <bool kept>
PyObject *rms_norm_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor &dy = tensor(a[0], "dy"), &h = tensor(a[1], "h"), &weight = tensor(a[2], "weight");
  const Tensor *dh = optional(a[4], "dh");
  if (kept) float_type(dy, "dy");
  else float_type(h, "h");
  no_gradient("rms_norm_grad", {&dy, &h, &weight, dh});
  const ScalarType t = kept ? dy.scalar_type() : h.scalar_type();
  Rows hr = rows(kept ? dy : h, "h");
  const Rows gr = rows_of(dy, "dy", hr.m, hr.n, t);
  if (kept) hr.p = kept_rows(h, "h", hr.m, hr.n);
  tf_rms_norm_grad_args_t g{};
  g.h = hr.p, g.h_ld = hr.ld, g.rows = hr.m, g.d = hr.n, g.dy = gr.p, g.dy_ld = gr.ld, g.eps = static_cast<float>(number(a[3]));
  g.weight = vector(weight, "weight", hr.n, t, ScalarType::Float);
  g.type = type_of(t), g.weight_type = type_of(weight.scalar_type()), g.kept = kept ? TF_KEPT_H : 0;
  if (dh) {
    const Rows r = rows_of(*dh, "dh", hr.m, hr.n, t);
    g.dh = r.p, g.dh_ld = r.ld;
  }
  on_gpu(h, {&dy, &weight, dh});
  const On on(h);
  const Tensor dx = fresh(h, kept ? dy.sizes() : h.sizes(), t), dw = fresh(h, {hr.n}, weight.scalar_type());
  g.dx = dx.data_ptr(), g.dx_ld = hr.n, g.dweight = dw.data_ptr();
  check(tf_rms_norm_grad_workspace(g.rows, g.d, &g.workspace_bytes));
  Tensor space;
  if (g.workspace_bytes) space = fresh(h, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte), g.workspace = space.data_ptr();
  check(tf_rms_norm_grad(&g, on.stream));
  return tuple({&dx, &dw});
  END_HANDLE_TH_ERRORS
}

// (x, w, bias, act, residual, keep, x_scale, w_scale, out_dtype, tile, splits) -> out or (out, z);
// kept: (out, z's bytes in 8 bits).
template <bool kept>
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w");
  const Tensor *bias = optional(a[2], "bias"), *residual = optional(a[4], "residual");
  const Tensor *xs = optional(a[6], "x_scale"), *ws = optional(a[7], "w_scale");
  const bool keep = kept || a[5] == Py_True;
  const ScalarType t = x.scalar_type();
  const bool eight = t == ScalarType::Float8_e4m3fn || t == ScalarType::Char;
  TORCH_CHECK_TYPE(half_type(t) || (eight && !kept), "x is ", t, ", not BFloat16, Half, Float8_e4m3fn or Char");
  ScalarType to = eight ? ScalarType::BFloat16 : t;
  if (a[8] != Py_None) {
    TORCH_CHECK_TYPE(THPDtype_Check(a[8]), "out_dtype is not a dtype");
    to = reinterpret_cast<THPDtype *>(a[8])->scalar_type;
    TORCH_CHECK_TYPE(half_type(to) && (eight || to == t), "out_dtype is ", to,
                     eight ? ", not BFloat16 or Half" : ": 16-bit products keep x's type");
  }
  TORCH_CHECK_VALUE(eight || (!xs && !ws), "scales belong to 8-bit products");
  if (eight) no_gradient("an 8-bit product", {&x, &w, bias, residual, xs, ws});
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
  if (eight) {
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
  if (kept) z = fresh(x, {kept_bytes(xr.m, wr.n)}, ScalarType::Byte), g.z = z.data_ptr(), g.kept = TF_KEPT_Z;
  else if (keep) z = fresh(x, size, to), g.z = z.data_ptr();
  check(tf_linear_workspace(&g, &g.workspace_bytes));
  if (g.workspace_bytes) {
    space = fresh(x, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte);
    g.workspace = space.data_ptr();
  }
  check(tf_linear(&g, on.stream));
  return keep ? tuple({&out, &z}) : wrap(&out);
  END_HANDLE_TH_ERRORS
}

// (dy, x, w, z, act, bias_dtype, want_dx, want_dw, tile, splits, terms) -> (dx, dw, dbias);
// some_kept: x and z may be what keep8 gave, bytes.
template <bool some_kept>
PyObject *linear_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor &dy = tensor(a[0], "dy"), &x = tensor(a[1], "x"), &w = tensor(a[2], "w");
  const Tensor *z = optional(a[3], "z");
  const bool kept = some_kept && x.scalar_type() == ScalarType::Byte;
  const ScalarType t = kept ? dy.scalar_type() : x.scalar_type();
  TORCH_CHECK_TYPE(half_type(t), kept ? "dy is " : "x is ", t, ", not BFloat16 or Half");
  no_gradient("linear_grad", {&dy, &x, &w, z});
  const bool want_dx = a[6] == Py_True, want_dw = a[7] == Py_True;
  TORCH_CHECK_VALUE(!kept || w.dim() == 2, "w is ", w.sizes(), ", not k x n");
  Rows xr = kept ? Rows{nullptr, rows(dy, "dy").m, w.size(0), w.size(0)} : rows(x, "x");
  if (kept) xr.p = kept_rows(x, "x", xr.m, xr.n);
  const Weights wr = weights(w, xr.n, t);
  const Rows gr = rows_of(dy, "dy", xr.m, wr.n, t);
  tf_linear_grad_args_t g{};
  g.dy = gr.p, g.dy_ld = gr.ld, g.x = xr.p, g.x_ld = xr.ld, g.w = wr.p, g.w_ld = wr.ld, g.w_order = wr.order;
  g.m = xr.m, g.n = wr.n, g.k = xr.n, g.type = type_of(t), g.act = integer(a[4], "activation");
  g.tile = integer(a[8], "tile"), g.splits = integer(a[9], "splits"), g.terms = integer(a[10], "terms");
  if (g.act) {
    TORCH_CHECK_VALUE(z, "an activation's gradient needs z: call linear with keep=True");
    if (some_kept && z->scalar_type() == ScalarType::Byte) {
      g.z = kept_rows(*z, "z", xr.m, wr.n), g.kept = TF_KEPT_Z;
    } else {
      const Rows r = rows_of(*z, "z", xr.m, wr.n, t);
      g.z = r.p, g.z_ld = r.ld;
    }
  }
  if (kept) g.kept |= TF_KEPT_X;
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
  if (want_dx) dx = fresh(x, kept ? at::IntArrayRef(with_last(dy, xr.n)) : x.sizes(), t), g.dx = dx.data_ptr(), g.dx_ld = xr.n;
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

// The targets of x's rows.
const long long *targets(const Tensor &t, const Tensor &x) {
  static_assert(sizeof(long long) == sizeof(int64_t), "targets are 64-bit");
  same_type(t, "target", ScalarType::Long, ScalarType::Long);
  TORCH_CHECK_VALUE(t.sizes() == x.sizes().slice(0, x.dim() - 1) && t.is_contiguous(), "target is not a contiguous tensor of ",
                    x.sizes().slice(0, x.dim() - 1));
  return reinterpret_cast<const long long *>(t.data_ptr<int64_t>());
}

long long integer64(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// The loss of checked operands, and what its gradient takes.
struct Xent {
  Tensor loss, lse, count;
};
void xent_operands(const Tensor &x, const Tensor &w, const Tensor &target, Rows &xr, Weights &wr) {
  const ScalarType t = x.scalar_type();
  TORCH_CHECK_TYPE(half_type(t), "x is ", t, ", not BFloat16 or Half");
  xr = rows(x, "x");
  wr = weights(w, xr.n, t);
  targets(target, x);
}

// reduction: 0 none, 1 sum, 2 mean
Xent xent(const Tensor &x, const Tensor &w, const Tensor &target, int64_t ignore, int64_t reduction) {
  Rows xr;
  Weights wr;
  xent_operands(x, w, target, xr, wr);
  tf_linear_xent_args_t g{};
  g.target = targets(target, x);
  g.x = xr.p, g.x_ld = xr.ld, g.m = xr.m, g.k = xr.n, g.w = wr.p, g.w_ld = wr.ld, g.n = wr.n, g.w_order = wr.order;
  g.type = type_of(x.scalar_type()), g.ignore = ignore;
  on_gpu(x, {&w, &target});
  const On on(x);
  const at::IntArrayRef shape = x.sizes().slice(0, x.dim() - 1);
  Xent r{fresh(x, shape, ScalarType::Float), fresh(x, shape, ScalarType::Double), {}};
  g.loss = r.loss.data_ptr<float>(), g.lse = r.lse.data_ptr<double>();
  Tensor one, space;
  if (reduction) one = fresh(x, {}, ScalarType::Float), (reduction == 1 ? g.sum : g.mean) = one.data_ptr<float>();
  if (reduction == 2) r.count = fresh(x, {}, ScalarType::Float), g.count = r.count.data_ptr<float>();
  check(tf_linear_xent_workspace(&g, &g.workspace_bytes));
  if (g.workspace_bytes) space = fresh(x, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte), g.workspace = space.data_ptr();
  check(tf_linear_xent(&g, on.stream));
  if (reduction) r.loss = one;
  return r;
}

std::pair<Tensor, Tensor> xent_grad(const Tensor &dloss, const Tensor &x, const Tensor &w, const Tensor &target, const Tensor &lse,
                                    const Tensor *number, int64_t ignore, bool want_dx, bool want_dw) {
  Rows xr;
  Weights wr;
  xent_operands(x, w, target, xr, wr);
  const ScalarType t = x.scalar_type();
  tf_linear_xent_grad_args_t g{};
  g.target = targets(target, x);
  const at::IntArrayRef shape = x.sizes().slice(0, x.dim() - 1);
  same_type(lse, "lse", ScalarType::Double, ScalarType::Double);
  TORCH_CHECK_VALUE(lse.sizes() == shape && lse.is_contiguous(), "lse is not a contiguous tensor of ", shape);
  same_type(dloss, "dloss", ScalarType::Float, ScalarType::Float);
  g.dloss_rows = dloss.dim() != 0;
  TORCH_CHECK_VALUE(dloss.dim() == 0 || (dloss.sizes() == shape && dloss.is_contiguous()), "dloss is not one number or a contiguous tensor of ", shape);
  if (number) {
    same_type(*number, "count", ScalarType::Float, ScalarType::Float);
    TORCH_CHECK_VALUE(number->numel() == 1, "count is not one number");
    g.count = number->data_ptr<float>();
  }
  g.lse = lse.data_ptr<double>(), g.dloss = dloss.data_ptr<float>();
  g.x = xr.p, g.x_ld = xr.ld, g.m = xr.m, g.k = xr.n, g.w = wr.p, g.w_ld = wr.ld, g.n = wr.n, g.w_order = wr.order;
  g.type = type_of(t), g.ignore = ignore;
  on_gpu(x, {&w, &target, &lse, &dloss, number});
  const On on(x);
  Tensor dx, dw, space;
  if (want_dx) dx = fresh(x, x.sizes(), t), g.dx = dx.data_ptr(), g.dx_ld = xr.n;
  if (want_dw) {
    dw = wr.order ? fresh(x, {wr.n, xr.n}, t).t() : fresh(x, {xr.n, wr.n}, t);
    g.dw = dw.data_ptr(), g.dw_ld = wr.order ? xr.n : wr.n;
  }
  check(tf_linear_xent_grad_workspace(&g, &g.workspace_bytes));
  if (g.workspace_bytes) space = fresh(x, {static_cast<int64_t>(g.workspace_bytes)}, ScalarType::Byte), g.workspace = space.data_ptr();
  check(tf_linear_xent_grad(&g, on.stream));
  return {dx, dw};
}

// The loss under autograd, natively: a step of a small classifier is bound by the host (61 x 1001 x
// 333 102 us through a Python function, whose backward waits for the interpreter's lock).
struct XentFunction : torch::autograd::Function<XentFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &target,
                                                int64_t ignore, int64_t reduction) {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Xent r = xent(x, w, target, ignore, reduction);
    ctx->save_for_backward({x, w, target, r.lse, r.count});
    ctx->saved_data["ignore"] = ignore;
    if (r.count.defined()) ctx->mark_non_differentiable({r.lse, r.count});
    else ctx->mark_non_differentiable({r.lse});
    ctx->set_materialize_grads(false);
    if (!r.count.defined()) return {r.loss, r.lse};
    return {r.loss, r.lse, r.count};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list all(5);
    if (!grads[0].defined()) return all;
    const auto saved = ctx->get_saved_variables();
    const bool again = at::GradMode::is_enabled();
    {
      const at::NoGradGuard none;
      std::tie(all[0], all[1]) = xent_grad(grads[0].contiguous(), saved[0], saved[1], saved[2], saved[3], saved[4].defined() ? &saved[4] : nullptr,
                                           ctx->saved_data["ignore"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    }
    if (again) {  // what a second derivative reaches raises
      const auto refuse = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice: the gradient calls have no gradient (once_differentiable)", 1);
      for (Tensor &t : all)
        if (t.defined()) t = (*refuse)({t.detach().set_requires_grad(true)})[0];
    }
    return all;
  }
};

// (x, w, target, ignore, reduction) -> (loss, lse, count)
PyObject *linear_xent(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w"), &target = tensor(a[2], "target");
  const int64_t ignore = integer64(a[3]), reduction = integer(a[4], "reduction");
  if (wants_grad({&x, &w})) {
    Rows xr;
    Weights wr;
    xent_operands(x, w, target, xr, wr);
    const auto r = XentFunction::apply(x, w, target, ignore, reduction);
    return tuple({&r[0], &r[1], r.size() > 2 ? &r[2] : nullptr});
  }
  const Xent r = xent(x, w, target, ignore, reduction);
  return tuple({&r.loss, &r.lse, r.count.defined() ? &r.count : nullptr});
  END_HANDLE_TH_ERRORS
}

// (dloss, x, w, target, lse, count, ignore, want_dx, want_dw) -> (dx, dw)
PyObject *linear_xent_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9);
  const Tensor &dloss = tensor(a[0], "dloss"), &x = tensor(a[1], "x"), &w = tensor(a[2], "w"), &target = tensor(a[3], "target");
  const Tensor &lse = tensor(a[4], "lse"), *number = optional(a[5], "count");
  no_gradient("linear_cross_entropy_grad", {&dloss, &x, &w, &lse, number});
  const auto [dx, dw] = xent_grad(dloss, x, w, target, lse, number, integer64(a[6]), a[7] == Py_True, a[8] == Py_True);
  return tuple({dx.defined() ? &dx : nullptr, dw.defined() ? &dw : nullptr});
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"rms_norm", reinterpret_cast<PyCFunction>(rms_norm), METH_FASTCALL, nullptr},
    {"linear_xent", reinterpret_cast<PyCFunction>(linear_xent), METH_FASTCALL, nullptr},
    {"linear_xent_grad", reinterpret_cast<PyCFunction>(linear_xent_grad), METH_FASTCALL, nullptr},
    {"keep8", reinterpret_cast<PyCFunction>(keep8), METH_FASTCALL, nullptr},
    {"restore8", reinterpret_cast<PyCFunction>(restore8), METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(quantize_rows), METH_FASTCALL, nullptr},
    {"rms_norm_grad", reinterpret_cast<PyCFunction>(rms_norm_grad<false>), METH_FASTCALL, nullptr},
    {"rms_norm_grad8", reinterpret_cast<PyCFunction>(rms_norm_grad<true>), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(linear<false>), METH_FASTCALL, nullptr},
    {"linear_keep8", reinterpret_cast<PyCFunction>(linear<true>), METH_FASTCALL, nullptr},
    {"linear_grad", reinterpret_cast<PyCFunction>(linear_grad<false>), METH_FASTCALL, nullptr},
    {"linear_grad8", reinterpret_cast<PyCFunction>(linear_grad<true>), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nn_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nn_torch() { return PyModule_Create(&module); }
