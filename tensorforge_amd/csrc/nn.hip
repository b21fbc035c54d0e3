// C ABI of the residual block's operators (declared at the end of
// include/tforge_hip.h) but the loss over a vocabulary: checks of arguments and the
// order of launches.
#include "nn_plan.hpp"

using namespace tfnn;

namespace {

// ---- norm ---------------------------------------------------------------------

// The scales of rows without elements: quantised as they are, whose largest magnitude is
// then the least that counts.
hipError_t scales_of_nothing(float *scale, long long rows, int y_type, hipStream_t stream) {
  NormParams p;
  p.scale = scale, p.rows = rows;
  return launch_rms_norm(p, TF_T_F32, y_type, stream);
}

int rms_norm(const tf_rms_norm_args_t *a, hipStream_t stream) {
  const char *call = "tf_rms_norm";
  if (!a) return fail(TF_E_ARG, "tf_rms_norm: null arguments");
  Checks c{call, {}};
  c.one_of("type", a->type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.one_of("weight_type", a->weight_type, {a->type, TF_T_F32});
  c.one_of("y_type", a->y_type, {a->type, TF_T_F8, TF_T_I8});
  c.size("rows", a->rows);
  c.size("d", a->d);
  c.need(a->eps >= 0, "eps is negative or not a number");
  c.matrix("x", a->x, a->x_ld, a->rows, a->d, a->type, true);
  c.matrix("residual", a->residual, a->residual_ld, a->rows, a->d, a->type, false);
  c.matrix("h", a->h, a->h_ld, a->rows, a->d, a->type, a->residual != nullptr);
  c.need(a->residual || !a->h, "h without a residual: it would be x");
  c.vector("weight", a->weight, a->d, a->weight_type, true);
  c.matrix("y", a->y, a->y_ld, a->rows, a->d, a->y_type, true);
  c.vector("scale", a->scale, a->rows, TF_T_F32, eight_bits(a->y_type));
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->rows == 0) return TF_OK;
  if (a->d == 0) return eight_bits(a->y_type) ? hip(scales_of_nothing(a->scale, a->rows, a->y_type, stream), call) : TF_OK;
  NormParams p;
  p.x = a->x, p.residual = a->residual, p.weight = a->weight, p.y = a->y, p.h = a->h, p.scale = a->scale;
  p.x_ld = a->x_ld, p.residual_ld = a->residual_ld, p.y_ld = a->y_ld, p.h_ld = a->h_ld, p.rows = a->rows;
  p.d = static_cast<int>(a->d), p.weight_type = a->weight_type, p.eps = a->eps;
  return hip(launch_rms_norm(p, a->type, a->y_type, stream), call);
}

int quantize_rows(const char *call, const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                  int y_type, float *scale, hipStream_t stream) {
  Checks c{call, {}};
  c.one_of("type", type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.one_of("y_type", y_type, {TF_T_F8, TF_T_I8});
  c.size("rows", rows);
  c.size("d", d);
  c.matrix("x", x, x_ld, rows, d, type, true);
  c.matrix("y", y, y_ld, rows, d, y_type, true);
  c.vector("scale", scale, rows, TF_T_F32, true);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (rows == 0) return TF_OK;
  if (d == 0) return hip(scales_of_nothing(scale, rows, y_type, stream), call);
  NormParams p;
  p.x = x, p.y = y, p.scale = scale, p.x_ld = x_ld, p.y_ld = y_ld, p.rows = rows, p.d = static_cast<int>(d);
  return hip(launch_rms_norm(p, type, y_type, stream), call);
}

int rms_norm_grad(const tf_rms_norm_grad_args_t *a, hipStream_t stream) {
  const char *call = "tf_rms_norm_grad";
  if (!a) return fail(TF_E_ARG, "tf_rms_norm_grad: null arguments");
  Checks c{call, {}};
  c.one_of("type", a->type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.one_of("weight_type", a->weight_type, {a->type, TF_T_F32});
  c.size("rows", a->rows);
  c.size("d", a->d);
  c.need(a->eps >= 0, "eps is negative or not a number");
  c.one_of("kept", a->kept, {0, TF_KEPT_H});
  c.matrix("dy", a->dy, a->dy_ld, a->rows, a->d, a->type, true);
  if (a->kept) c.kept("h", a->h, a->rows, a->d, true);
  else c.matrix("h", a->h, a->h_ld, a->rows, a->d, a->type, true);
  c.matrix("dh", a->dh, a->dh_ld, a->rows, a->d, a->type, false);
  c.vector("weight", a->weight, a->d, a->weight_type, true);
  c.matrix("dx", a->dx, a->dx_ld, a->rows, a->d, a->type, true);
  c.vector("dweight", a->dweight, a->d, a->weight_type, true);
  if (c.fine()) c.workspace(a->workspace, a->workspace_bytes, norm_grad_shares(a->rows, a->d) * a->d * 4);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->d == 0) return TF_OK;
  NormGradParams p;
  p.kept = a->kept != 0;
  p.dy = a->dy, p.h = a->h, p.dh = a->dh, p.weight = a->weight, p.dx = a->dx, p.dw = a->dweight;
  p.shares = static_cast<float *>(a->workspace);
  p.dy_ld = a->dy_ld, p.h_ld = a->h_ld, p.dh_ld = a->dh_ld, p.dx_ld = a->dx_ld, p.rows = a->rows;
  p.d = static_cast<int>(a->d), p.weight_type = a->weight_type, p.eps = a->eps;
  return hip(launch_rms_norm_grad(p, a->type, stream), call);
}

// ---- kept in 8 bits ---------------------------------------------------------------

int keep8(const char *call, const void *x, long long x_ld, long long rows, long long d, int type, int positive, bool masked, void *kept,
          hipStream_t stream) {
  Checks c{call, {}};
  c.one_of("type", type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.one_of("positive", positive, {0, 1});
  c.size("rows", rows);
  c.size("d", d);
  c.matrix("x", x, x_ld, rows, d, type, true);
  c.kept("kept", kept, rows, d, true);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (rows == 0 || d == 0) return TF_OK;
  return hip(launch_keep(x, x_ld, rows, static_cast<int>(d), type, positive != 0, masked, kept, stream), call);
}

// ---- products -------------------------------------------------------------------

void check_linear_sizes(Checks &c, const tf_linear_args_t *a) {
  c.one_of("type", a->type, {TF_T_BF16, TF_T_F16, TF_T_F8, TF_T_I8});
  if (eight_bits(a->type)) c.one_of("out_type", a->out_type, {TF_T_BF16, TF_T_F16});
  else c.one_of("out_type", a->out_type, {a->type});
  c.size("m", a->m);
  c.size("n", a->n);
  c.size("k", a->k);
  c.one_of("kept", a->kept, {0, TF_KEPT_Z});
  c.need(!a->kept || !eight_bits(a->type), "8-bit products do not keep z in 8 bits");
  c.need(a->type != TF_T_I8 || a->k <= kMostI8, "k = ", a->k, ": sums of more than ", kMostI8, " products of 8-bit integers pass 32 bits");
  check_choice(c, a->tile, a->splits);
}

Product product_of(const tf_linear_args_t *a) {
  Product q{a->type, a->out_type, {}, {}, {}};
  q.a = {a->x, a->x_ld, a->m, a->k, false, false};
  q.b = a->w_order ? Operand{a->w, a->w_ld, a->n, a->k, false, false} : Operand{a->w, a->w_ld, a->k, a->n, true, false};
  GemmParams &p = q.p;
  p.bias = a->bias, p.residual = a->residual, p.sa = a->x_scale, p.sb = a->w_scale, p.out = a->out, p.z = a->z;
  p.ldr = a->residual_ld, p.ldo = a->out_ld, p.ldz = a->z_ld;
  p.m = static_cast<int>(a->m), p.n = static_cast<int>(a->n), p.k = static_cast<int>(a->k);
  p.act = a->act, p.bias_f32 = a->bias_type == TF_T_F32;
  return q;
}

// z kept in 8 bits: the bytes of the z in 16 that a product writes first where it cannot write the
// codes itself (split, few rows, loads through registers).
long long z_bytes(const tf_linear_args_t *a, const Choice &c) { return a->kept && !fused_z(c) ? round16(2 * a->m * a->n) : 0; }

int linear_workspace(const tf_linear_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_workspace: null arguments");
  Checks c{"tf_linear_workspace", {}};
  check_linear_sizes(c, a);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->m && a->n) {
    const Choice plan = choose(product_of(a), a->tile, a->splits);
    *bytes = plan.bytes() + z_bytes(a, plan);
  } else {
    *bytes = 0;
  }
  return TF_OK;
}

int linear(const tf_linear_args_t *a, hipStream_t stream) {
  const char *call = "tf_linear";
  if (!a) return fail(TF_E_ARG, "tf_linear: null arguments");
  Checks c{call, {}};
  check_linear_sizes(c, a);
  const bool eight = eight_bits(a->type);
  c.one_of("w_order", a->w_order, {0, 1});
  c.need(!eight || a->w_order == 1, "8-bit weights lie as n rows of k (w_order 1)");
  c.one_of("act", a->act, {TF_ACT_NONE, TF_ACT_RELU, TF_ACT_GELU, TF_ACT_SILU});
  if (a->bias) c.one_of("bias_type", a->bias_type, {a->out_type, TF_T_F32});
  c.matrix("x", a->x, a->x_ld, a->n ? a->m : 0, a->k, a->type, true);
  if (a->w_order) c.matrix("w", a->w, a->w_ld, a->m ? a->n : 0, a->k, a->type, true);
  else c.matrix("w", a->w, a->w_ld, a->m ? a->k : 0, a->n, a->type, true);
  c.vector("bias", a->bias, a->n, a->bias_type, false);
  c.matrix("residual", a->residual, a->residual_ld, a->m, a->n, a->out_type, false);
  c.matrix("out", a->out, a->out_ld, a->m, a->n, a->out_type, true);
  if (a->kept) c.kept("z", a->z, a->m, a->n, true);
  else c.matrix("z", a->z, a->z_ld, a->m, a->n, a->out_type, false);
  c.vector("x_scale", a->x_scale, a->m, TF_T_F32, eight);
  c.vector("w_scale", a->w_scale, a->n, TF_T_F32, eight);
  c.need(eight || (!a->x_scale && !a->w_scale), "scales belong to 8-bit products");
  if (a->workspace_bytes) c.workspace(a->workspace, a->workspace_bytes, 1);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->m == 0 || a->n == 0) return TF_OK;
  Product q = product_of(a);
  if (!a->kept) return hip(run_product(q, a->tile, a->splits, a->workspace, a->workspace_bytes, stream), call);
  const Choice plan = choose(q, a->tile, a->splits);
  const long long z16 = z_bytes(a, plan);
  c.workspace(a->workspace, a->workspace_bytes, plan.bytes() + z16);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  char *ws = static_cast<char *>(a->workspace);
  q.p.z = z16 ? ws + plan.bytes() : nullptr, q.p.ldz = a->n;
  hipError_t e = run_product(q, a->tile, a->splits, ws, plan.bytes(), stream, z16 ? nullptr : a->z);
  if (e == hipSuccess && z16)
    e = launch_keep(ws + plan.bytes(), a->n, a->m, static_cast<int>(a->n), a->type, a->act == TF_ACT_RELU, true, a->z, stream);
  return hip(e, call);
}

// How a gradient runs: the workspace's parts and the products.
struct GradPlan {
  bool own_dz = false;   // dz lies in the workspace: an activation's, or an aligned copy of dy
  int terms = 1;         // of dz
  int rows = 0;          // of a workgroup of dz
  long dz_ld = 0, count = 1;                  // shares of the bias gradient
  long long dz = 0, shares = 0, x = 0, product = 0;  // bytes; x: restored from 8 bits
  bool pair = false;                          // both products in one launch, in these ranges of k,
  int dx_splits = 1, dw_splits = 1;           // and of `product`, the bytes of
  long long copies = 0, dx_parts = 0;         // aligned copies of w and x, and dx's parts
  Product dx, dw;
  long long bytes() const { return dz + shares + x + product; }
};

// Both products on 64 x 64 tiles in one launch (1148 x 848 x 209 bfloat16 silu 16.7 us, 35.8 in
// launches apart; 4096 x 8192 x 2048 244 us against 238 apart): the aligned copies of x and w come with
// dz, one more launch joins the ranges of k of both.  Predicted as predicted() does,
// two workgroups on a CU; us.  The time of what it finds, and the ranges in `g`.
double plan_pair(GradPlan &g) {
  const GemmParams &dx = g.dx.p, &dw = g.dw.p;
  const double t1 = static_cast<double>(ceil_div(dx.m, 64)) * ceil_div(dx.n, 64);
  const double t2 = static_cast<double>(ceil_div(dw.m, 64)) * ceil_div(dw.n, 64);
  double best = 1e30;
  if (t1 + t2 > 2048) return best;
  const double slabs1 = ceil_div(dx.k, 64), slabs2 = ceil_div(dw.k, 64), all = t1 * slabs1 + t2 * slabs2;
  for (int s1 = 1; s1 == 1 || s1 * 2 <= slabs1; s1 *= 2) {
    for (int s2 = 1; s2 == 1 || s2 * 2 <= slabs2; s2 *= 2) {
      const double w = (t1 * s1 + t2 * s2) / 256;
      if (s1 > 16 || s2 > 16 || (w > 4 && s1 * s2 > 1)) break;
      const double longest = std::max(std::ceil(slabs1 / s1), std::ceil(slabs2 / s2));
      double us = 4.3 + 2 * std::max(0.0, std::ceil(w / 2) - 1) + g.terms * std::max(longest * (w <= 1 ? 0.29 : 0.38), all * 0.19 / 256);
      const double parts = (s1 > 1 ? s1 * static_cast<double>(dx.m) * dx.n : 0) + (s2 > 1 ? s2 * static_cast<double>(dw.m) * dw.n : 0);
      if (parts > 0) us += 3.3 + 8 * parts / 7e6;
      if (us < best) best = us, g.dx_splits = s1, g.dw_splits = s2;
    }
  }
  return best;
}

// Unless the caller says otherwise, up to this many multiply-adds a product of the rounded dz is
// not taken alone: what the rounding left goes in as a second term, into the same float sums.  A
// small gradient then errs by its own rounding only; larger ones, where a second
// product would cost as much again, by sqrt(2) of it.  bfloat16 gelu, two terms here and
// one just above: 512 x 512 x 520 14.0 us, x 544 11.0; 2048 x 256 x 264 17.1, x 280 15.0.
constexpr double kTwoTerms = 1.4e8;

GradPlan plan_grad(const tf_linear_grad_args_t *a) {
  GradPlan g{};
  const int m = static_cast<int>(a->m), n = static_cast<int>(a->n), k = static_cast<int>(a->k);
  if (n == 0) return g;
  const double work = static_cast<double>(m) * n * k;
  const bool smooth = a->act == TF_ACT_GELU || a->act == TF_ACT_SILU;
  g.dz_ld = n <= 64 ? ceil_div(n, 8) * 8 : ceil_div(n, 64) * 64;
  const Operand dy{a->dy, a->dy_ld, m, n, false, false};
  const auto lay = [&](bool own, int rows) {
    g.own_dz = own;
    g.dz = own ? round16(2 * a->m * g.dz_ld) * g.terms : 0;
    g.rows = rows;
    g.count = ceil_div(m, rows);
    g.shares = a->dbias && g.count > 1 ? round16(4 * g.count * a->n) : 0;
  };
  g.terms = !smooth ? 1 : a->terms ? a->terms : work <= kTwoTerms ? 2 : 1;
  const bool odd = !direct_loads(dy, 2);
  // A workgroup of dz takes all of up to 256 rows where that spares the bias gradient a
  // second launch; else 64, or 32 where that leaves CUs without work.
  lay(m && (a->act != TF_ACT_NONE || (odd && m > 64 && work > 1e6)),
      a->dbias && m <= SLOPE_WHOLE ? SLOPE_WHOLE : ceil_div(m, 64) * ceil_div(n, 256) < 512 ? SLOPE_FEW : SLOPE_MANY);
  if (k == 0) return g;
  const bool nk = a->w_order == 1;
  const auto dz = [&](bool mn) {
    return g.own_dz ? Operand{nullptr, g.dz_ld, m, n, mn, true} : Operand{a->dy, a->dy_ld, m, n, mn, false};
  };
  g.dx = {a->type, a->type, dz(false), nk ? Operand{a->w, a->w_ld, n, k, true, false} : Operand{a->w, a->w_ld, k, n, false, false}, {}};
  g.dx.p.m = m, g.dx.p.n = k, g.dx.p.k = n, g.dx.p.out = a->dx, g.dx.p.ldo = a->dx_ld;
  Operand x{a->x, a->x_ld, m, k, true, false};
  if (a->kept & TF_KEPT_X && a->dw) x.ld = packed_ld(x, 2), x.ours = true, g.x = packed_bytes(x, 2);
  g.dw = {a->type, a->type, nk ? dz(true) : x, nk ? x : dz(true), {}};
  g.dw.p.m = nk ? n : k, g.dw.p.n = nk ? k : n, g.dw.p.k = m, g.dw.p.out = a->dw, g.dw.p.ldo = a->dw_ld;
  if (g.terms == 2) {
    g.dx.p.terms = g.dw.p.terms = 2;
    g.dx.p.a_term = (nk ? g.dw.p.a_term : g.dw.p.b_term) = -(g.dz / 2);  // what the rounding left lies behind
  }
  // One launch for both where it takes less; below 8 us two cannot.
  double pair = 1e30;
  long long copies = 0;
  if (!a->tile && !a->splits && a->dx && a->dw && m) {
    copies = (direct_loads(g.dx.b, 2) ? 0 : packed_bytes(g.dx.b, 2)) + (direct_loads(x, 2) ? 0 : packed_bytes(x, 2));
    const bool more = !g.own_dz && !a->dbias && (odd || copies || g.x);  // a launch for the copies alone
    pair = plan_pair(g) + (more ? 4 : 0) + copies * 0.21e-6;
  }
  if (pair > 8) {
    double apart = g.shares ? 5 : 1;  // the sum's launch, or a gap between two
    if (a->dx && m) {
      const Choice c = choose(g.dx, a->tile, a->splits);
      g.product = c.bytes(), apart += c.us;
    }
    if (a->dw) {
      const Choice c = choose(g.dw, a->tile, a->splits);
      g.product = std::max(g.product, c.bytes()), apart += c.us;
    }
    if (pair > apart) return g;
  }
  g.pair = true;
  lay(a->act != TF_ACT_NONE || odd, SLOPE_FEW);
  g.dx.a = dz(false);
  (nk ? g.dw.a : g.dw.b) = dz(true);
  g.copies = copies;
  g.dx_parts = part_bytes(m, k, {TILE_64, g.dx_splits, 0});
  g.product = copies + g.dx_parts + part_bytes(g.dw.p.m, g.dw.p.n, {TILE_64, g.dw_splits, 0});
  return g;
}

void check_grad_sizes(Checks &c, const tf_linear_grad_args_t *a) {
  c.one_of("type", a->type, {TF_T_BF16, TF_T_F16});
  c.one_of("act", a->act, {TF_ACT_NONE, TF_ACT_RELU, TF_ACT_GELU, TF_ACT_SILU});
  c.one_of("w_order", a->w_order, {0, 1});
  c.size("m", a->m);
  c.size("n", a->n);
  c.size("k", a->k);
  check_choice(c, a->tile, a->splits);
  c.one_of("terms", a->terms, {0, 1, 2});
  c.one_of("kept", a->kept, {0, TF_KEPT_X, TF_KEPT_Z, TF_KEPT_X | TF_KEPT_Z});
}

int linear_grad_workspace(const tf_linear_grad_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_grad_workspace: null arguments");
  Checks c{"tf_linear_grad_workspace", {}};
  check_grad_sizes(c, a);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  *bytes = plan_grad(a).bytes();
  return TF_OK;
}

int linear_grad(const tf_linear_grad_args_t *a, hipStream_t stream) {
  const char *call = "tf_linear_grad";
  if (!a) return fail(TF_E_ARG, "tf_linear_grad: null arguments");
  Checks c{call, {}};
  check_grad_sizes(c, a);
  const long long wr = a->w_order ? a->n : a->k, wc = a->w_order ? a->k : a->n;
  if (a->dbias) c.one_of("bias_type", a->bias_type, {a->type, TF_T_F32});
  c.matrix("dy", a->dy, a->dy_ld, a->m, a->n, a->type, true);
  if (a->kept & TF_KEPT_Z) c.kept("z", a->z, a->m, a->n, a->act != TF_ACT_NONE);
  else c.matrix("z", a->z, a->z_ld, a->m, a->n, a->type, a->act != TF_ACT_NONE);
  if (a->kept & TF_KEPT_X) c.kept("x", a->x, a->m, a->k, a->dw != nullptr);
  else c.matrix("x", a->x, a->x_ld, a->m, a->k, a->type, a->dw != nullptr);
  c.matrix("w", a->w, a->w_ld, wr, wc, a->type, a->dx != nullptr);
  c.matrix("dx", a->dx, a->dx_ld, a->m, a->k, a->type, false);
  c.matrix("dw", a->dw, a->dw_ld, wr, wc, a->type, false);
  c.vector("dbias", a->dbias, a->n, a->bias_type, false);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  GradPlan g = plan_grad(a);
  c.workspace(a->workspace, a->workspace_bytes, g.bytes());
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);

  char *ws = static_cast<char *>(a->workspace);
  float *shares = reinterpret_cast<float *>(ws + g.dz);
  char *const restored = ws + g.dz + g.shares;
  void *rest = restored + g.x;
  const int m = static_cast<int>(a->m), n = static_cast<int>(a->n), k = static_cast<int>(a->k);
  char *const parts = static_cast<char *>(rest) + g.copies;
  hipError_t e = hipSuccess;
  PackParams pack;
  if (g.copies) {
    Operand &w = g.dx.b, &x = a->w_order ? g.dw.b : g.dw.a;
    char *to = static_cast<char *>(rest);
    if (!direct_loads(w, 2)) to += copy_of(w, 2, to, pack);
    if (!direct_loads(x, 2)) copy_of(x, 2, to, pack);
  }
  if (g.x) {  // beside dz: x in 16 bits
    Operand &x = a->w_order ? g.dw.b : g.dw.a;
    const int i = pack.pieces[0] ? 1 : 0;
    pack.from[i] = a->x, pack.rows[i] = m, pack.columns[i] = k, pack.kept[i] = true;
    pack.to[i] = restored, pack.to_ld[i] = x.ld, pack.pieces[i] = x.lines * x.ld / 8;
    x.p = restored;
  }
  if (m && n && (g.own_dz || a->dbias)) {
    SlopeParams s{};
    s.rows = g.rows;
    s.kept = (a->kept & TF_KEPT_Z) != 0;
    s.dy = a->dy, s.z = a->z, s.dy_ld = a->dy_ld, s.z_ld = a->z_ld, s.m = m, s.n = n, s.act = a->act;
    if (g.own_dz) s.dz = ws, s.dz_ld = g.dz_ld, s.lo = g.terms == 2 ? g.dz / 4 : 0;
    if (a->dbias && g.shares) s.shares = shares;
    if (a->dbias && !g.shares) s.sums = a->dbias, s.sums_type = a->bias_type;
    e = launch_act_slope(s, pack, a->type, stream);
  } else if (pack.pieces[0]) {
    e = launch_pack(pack, a->type, stream);
  }
  if (e == hipSuccess && a->dbias && n && ((g.shares && !g.pair) || !m))
    e = launch_share_sum(shares, m ? g.count : 0, n, a->dbias, a->bias_type, stream);
  if (e != hipSuccess || !k) return hip(e, call);
  if (g.own_dz) g.dx.a.p = (a->w_order ? g.dw.a.p : g.dw.b.p) = g.terms == 2 ? ws + g.dz / 2 : ws;
  if (g.pair) {
    place(g.dx, {TILE_64, g.dx_splits, 0}, parts);
    place(g.dw, {TILE_64, g.dw_splits, 0}, parts + g.dx_parts);
    ShareParams sum;
    if (g.shares) sum = {shares, a->dbias, static_cast<int>(g.count), n, a->bias_type};
    e = a->type == TF_T_BF16 ? launch_gemm_pair_bf16(g.dx.p, g.dx.b.mn, g.dw.p, sum, stream)
                             : launch_gemm_pair_f16(g.dx.p, g.dx.b.mn, g.dw.p, sum, stream);
    if (e == hipSuccess && g.dx_splits * g.dw_splits > 1) e = launch_gemm_join_pair(g.dx.p, g.dw.p, a->type, stream);
    return hip(e, call);
  }
  if (a->dx && m) {
    if (n) {
      e = run_product(g.dx, a->tile, a->splits, rest, g.product, stream);
    } else {  // a sum of nothing
      Product q{a->type, a->type, {}, {}, {}};
      q.p.m = m, q.p.n = k, q.p.out = a->dx, q.p.ldo = a->dx_ld;
      e = run_product(q, 0, 1, nullptr, 0, stream);
    }
  }
  if (e == hipSuccess && a->dw && n) e = run_product(g.dw, a->tile, a->splits, rest, g.product, stream);
  return hip(e, call);
}

}  // namespace

extern "C" {

int tf_rms_norm(const tf_rms_norm_args_t *args, void *stream) {
  return guarded([&] { return rms_norm(args, static_cast<hipStream_t>(stream)); });
}

int tf_quantize_rows(const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                     float *scale, void *stream) {
  return guarded([&] {
    return quantize_rows("tf_quantize_rows", x, x_ld, rows, d, type, y, y_ld, TF_T_F8, scale, static_cast<hipStream_t>(stream));
  });
}

int tf_quantize_rows_to(const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                        int y_type, float *scale, void *stream) {
  return guarded([&] {
    return quantize_rows("tf_quantize_rows_to", x, x_ld, rows, d, type, y, y_ld, y_type, scale, static_cast<hipStream_t>(stream));
  });
}

int tf_rms_norm_grad_workspace(long long rows, long long d, long long *bytes) {
  return guarded([&] {
    Checks c{"tf_rms_norm_grad_workspace", {}};
    c.size("rows", rows);
    c.size("d", d);
    c.need(bytes != nullptr, "null arguments");
    if (!c.fine()) return fail(TF_E_ARG, c.wrong);
    *bytes = norm_grad_shares(rows, d) * d * 4;
    return TF_OK;
  });
}

int tf_rms_norm_grad(const tf_rms_norm_grad_args_t *args, void *stream) {
  return guarded([&] { return rms_norm_grad(args, static_cast<hipStream_t>(stream)); });
}

int tf_keep8_bytes(long long rows, long long d, long long *bytes) {
  return guarded([&] {
    Checks c{"tf_keep8_bytes", {}};
    c.size("rows", rows);
    c.size("d", d);
    c.need(bytes != nullptr, "null arguments");
    if (!c.fine()) return fail(TF_E_ARG, c.wrong);
    *bytes = rows * ceil_div(d, 32) * 33;
    return TF_OK;
  });
}

int tf_keep8(const void *x, long long x_ld, long long rows, long long d, int type, int positive, void *kept, void *stream) {
  return guarded([&] { return keep8("tf_keep8", x, x_ld, rows, d, type, positive, false, kept, static_cast<hipStream_t>(stream)); });
}

int tf_keep8_masked(const void *x, long long x_ld, long long rows, long long d, int type, int positive, void *kept, void *stream) {
  return guarded([&] { return keep8("tf_keep8_masked", x, x_ld, rows, d, type, positive, true, kept, static_cast<hipStream_t>(stream)); });
}

int tf_restore8(const void *kept, long long rows, long long d, int type, void *x, long long x_ld, void *stream) {
  return guarded([&] {
    Checks c{"tf_restore8", {}};
    c.one_of("type", type, {TF_T_F32, TF_T_BF16, TF_T_F16});
    c.size("rows", rows);
    c.size("d", d);
    c.kept("kept", kept, rows, d, true);
    c.matrix("x", x, x_ld, rows, d, type, true);
    if (!c.fine()) return fail(TF_E_ARG, c.wrong);
    if (rows == 0 || d == 0) return TF_OK;
    return hip(launch_restore(kept, rows, static_cast<int>(d), type, x, x_ld, static_cast<hipStream_t>(stream)), "tf_restore8");
  });
}

int tf_linear_workspace(const tf_linear_args_t *args, long long *bytes) {
  return guarded([&] { return linear_workspace(args, bytes); });
}

int tf_linear(const tf_linear_args_t *args, void *stream) {
  return guarded([&] { return linear(args, static_cast<hipStream_t>(stream)); });
}

int tf_linear_grad_workspace(const tf_linear_grad_args_t *args, long long *bytes) {
  return guarded([&] { return linear_grad_workspace(args, bytes); });
}

int tf_linear_grad(const tf_linear_grad_args_t *args, void *stream) {
  return guarded([&] { return linear_grad(args, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
