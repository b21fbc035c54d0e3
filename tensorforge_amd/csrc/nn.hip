// C ABI of the residual block's operators (declared at the end of
// include/tforge_hip.h): checks of arguments, the choice of tile and of ranges
// of k, and the order of launches.
#include <algorithm>
#include <cstdint>
#include <string>

#include "errors.h"
#include "nn_kernels.h"
#include "tforge_hip.h"

using tfk::fail;
using tfk::guarded;
using namespace tfnn;

namespace {

constexpr long long kMostSize = 1LL << 30;

int size_of(int type) { return type == TF_T_F32 ? 4 : type == TF_T_F8 ? 1 : 2; }

// The first thing wrong with a call's arguments.  Messages are built only where
// one is wanted: the checks of a good call cost some tens of nanoseconds.
struct Checks {
  const char *call;
  std::string wrong;

  bool fine() const { return wrong.empty(); }
  template <typename... Parts>
  void need(bool ok, const Parts &...parts) {
    if (ok || !wrong.empty()) return;
    wrong = std::string(call) + ": ";
    (void)std::initializer_list<int>{(add(parts), 0)...};
  }
  void add(const char *s) { wrong += s; }
  void add(long long v) { wrong += std::to_string(v); }
  void size(const char *name, long long v) {
    need(v >= 0 && v <= kMostSize, name, " = ", v, " is not between 0 and 2^30");
  }
  void one_of(const char *name, int v, std::initializer_list<int> allowed) {
    need(std::find(allowed.begin(), allowed.end(), v) != allowed.end(), name, " = ", static_cast<long long>(v),
         " is not one this call takes");
  }
  // A matrix of rows x cols elements; `wanted`: it may not be missing.
  void matrix(const char *name, const void *p, long long ld, long long rows, long long cols, int type, bool wanted) {
    if (!fine() || rows <= 0 || cols <= 0) return;
    need(p || !wanted, name, " is a null pointer");
    if (!p) return;
    need(reinterpret_cast<uintptr_t>(p) % size_of(type) == 0, name, " is not aligned to its elements");
    need(ld >= cols, name, ": ", ld, " elements between rows of ", cols);
    need(ld <= (1LL << 40), name, ": ", ld, " elements between rows are too many");
  }
  void vector(const char *name, const void *p, long long n, int type, bool wanted) {
    matrix(name, p, n, 1, n, type, wanted);
  }
  void workspace(const void *p, long long given, long long needed) {
    need(given >= needed, "the workspace has ", given, " bytes, ", needed, " are needed");
    need(needed == 0 || (p && reinterpret_cast<uintptr_t>(p) % 16 == 0), "the workspace is null or not 16-byte aligned");
  }
};

int hip(hipError_t e, const char *call) {
  return e == hipSuccess ? TF_OK : fail(TF_E_HIP, std::string(call) + " failed: " + hipGetErrorString(e));
}

// ---- norm ---------------------------------------------------------------------

int rms_norm(const tf_rms_norm_args_t *a, hipStream_t stream) {
  const char *call = "tf_rms_norm";
  if (!a) return fail(TF_E_ARG, "tf_rms_norm: null arguments");
  Checks c{call, {}};
  c.one_of("type", a->type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.one_of("weight_type", a->weight_type, {a->type, TF_T_F32});
  c.one_of("y_type", a->y_type, {a->type, TF_T_F8});
  c.size("rows", a->rows);
  c.size("d", a->d);
  c.need(a->eps >= 0, "eps is negative or not a number");
  c.matrix("x", a->x, a->x_ld, a->rows, a->d, a->type, true);
  c.matrix("residual", a->residual, a->residual_ld, a->rows, a->d, a->type, false);
  c.matrix("h", a->h, a->h_ld, a->rows, a->d, a->type, a->residual != nullptr);
  c.need(a->residual || !a->h, "h without a residual: it would be x");
  c.vector("weight", a->weight, a->d, a->weight_type, true);
  c.matrix("y", a->y, a->y_ld, a->rows, a->d, a->y_type, true);
  c.vector("scale", a->scale, a->rows, TF_T_F32, a->y_type == TF_T_F8);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->rows == 0 || a->d == 0) return TF_OK;
  NormParams p;
  p.x = a->x, p.residual = a->residual, p.weight = a->weight, p.y = a->y, p.h = a->h, p.scale = a->scale;
  p.x_ld = a->x_ld, p.residual_ld = a->residual_ld, p.y_ld = a->y_ld, p.h_ld = a->h_ld, p.rows = a->rows;
  p.d = static_cast<int>(a->d), p.weight_type = a->weight_type, p.eps = a->eps;
  return hip(launch_rms_norm(p, a->type, a->y_type == TF_T_F8, stream), call);
}

int quantize_rows(const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                  float *scale, hipStream_t stream) {
  const char *call = "tf_quantize_rows";
  Checks c{call, {}};
  c.one_of("type", type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.size("rows", rows);
  c.size("d", d);
  c.matrix("x", x, x_ld, rows, d, type, true);
  c.matrix("y", y, y_ld, rows, d, TF_T_F8, true);
  c.vector("scale", scale, rows, TF_T_F32, d > 0);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (rows == 0 || d == 0) return TF_OK;
  NormParams p;
  p.x = x, p.y = y, p.scale = scale, p.x_ld = x_ld, p.y_ld = y_ld, p.rows = rows, p.d = static_cast<int>(d);
  return hip(launch_rms_norm(p, type, true, stream), call);
}

long long round16(long long bytes) { return (bytes + 15) & ~15LL; }

int rms_norm_grad(const tf_rms_norm_grad_args_t *a, hipStream_t stream) {
  const char *call = "tf_rms_norm_grad";
  if (!a) return fail(TF_E_ARG, "tf_rms_norm_grad: null arguments");
  Checks c{call, {}};
  c.one_of("type", a->type, {TF_T_F32, TF_T_BF16, TF_T_F16});
  c.one_of("weight_type", a->weight_type, {a->type, TF_T_F32});
  c.size("rows", a->rows);
  c.size("d", a->d);
  c.need(a->eps >= 0, "eps is negative or not a number");
  c.matrix("dy", a->dy, a->dy_ld, a->rows, a->d, a->type, true);
  c.matrix("h", a->h, a->h_ld, a->rows, a->d, a->type, true);
  c.matrix("dh", a->dh, a->dh_ld, a->rows, a->d, a->type, false);
  c.vector("weight", a->weight, a->d, a->weight_type, true);
  c.matrix("dx", a->dx, a->dx_ld, a->rows, a->d, a->type, true);
  c.vector("dweight", a->dweight, a->d, a->weight_type, true);
  if (c.fine()) c.workspace(a->workspace, a->workspace_bytes, norm_grad_shares(a->rows, a->d) * a->d * 4);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->d == 0) return TF_OK;
  NormGradParams p;
  p.dy = a->dy, p.h = a->h, p.dh = a->dh, p.weight = a->weight, p.dx = a->dx, p.dw = a->dweight;
  p.shares = static_cast<float *>(a->workspace);
  p.dy_ld = a->dy_ld, p.h_ld = a->h_ld, p.dh_ld = a->dh_ld, p.dx_ld = a->dx_ld, p.rows = a->rows;
  p.d = static_cast<int>(a->d), p.weight_type = a->weight_type, p.eps = a->eps;
  return hip(launch_rms_norm_grad(p, a->type, stream), call);
}

// ---- products -------------------------------------------------------------------

// A product's operands as the kernels see them.
struct Product {
  int type, out_type;
  bool amn, bmn;
  GemmParams p;
};

// Whether the loads may go straight into LDS: 16-byte aligned rows of whole
// pieces, and every offset inside a tile's slab below 2^31 bytes.
bool direct_loads(const void *base, long ld, bool mn, int own, int k, int size) {
  const int piece = 16 / size;
  const long span = mn ? 64 * ld * size + 1024 : 256 * ld * size + 256;
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld % piece == 0 && (mn ? own : k) % piece == 0 && span < (1L << 31);
}

struct Plan {
  int tile, splits;
};

long ceil_div(long a, long b) { return (a + b - 1) / b; }

// The C tile and the ranges of k for a product of these sizes.
//
// Up to 64 rows a workgroup's time is what it reads, at about 35 bytes a
// nanosecond (what a CU's misses to L2 and beyond sustain): for the few-row
// kernel its columns' and all rows' whole k, for the 64 x 64 tile its range of
// k, and 3.3 us for the join where k is split.  The smaller estimate runs.
// Measured, bfloat16, us (few-row / tile), w 4096 x 4096 as n rows of k: 7.7 / 10.8
// for 1 row, 9.8 / 11.1 for 16, 13.7 / 11.6 for 32; as k rows of n: 11.4 / 11.6, 13.4 /
// 12.2, 16.1 / 12.5; 8192 deep and 2048 wide: 11.3 / 12.0 for 1 row, 16.6 / 12.2 for 16.
Plan plan_product(long m, long n, long k, int type, bool amn, bool bmn, bool dma, int tile, int splits) {
  const int size = size_of(type);
  const long slabs = ceil_div(k, 128 / size);
  const bool rows = m <= 64 && !amn && (!bmn || n >= 32);
  const auto split = [&](int t) {
    const long tiles = ceil_div(m, tile_size(t)) * ceil_div(n, tile_size(t));
    const long s = splits ? splits : std::min<long>({256 / std::max<long>(1, tiles), slabs / 4, 16});
    return static_cast<int>(std::max<long>(1, std::min(s, slabs)));
  };
  if (rows && !tile) {
    const long cols = bmn ? 32 : 16, s = split(TILE_64);
    const long few = ceil_div(ceil_div(n, cols), 256) * (cols + m) * k * size / 36;
    const long many = ceil_div(ceil_div(n, 64) * s, 256) * (64 + m) * (k / s) * size / 33 * (dma ? 1 : 2) + (s > 1 ? 3300 : 0);
    tile = few <= many ? TILE_ROWS : TILE_64;
  }
  if (tile == TILE_ROWS && rows) return {TILE_ROWS, 1};
  if (!tile || tile == TILE_ROWS) tile = m <= 64 || n <= 64 || ceil_div(m, 128) * ceil_div(n, 128) < 128 ? TILE_64
                    : dma && ceil_div(m, 256) * ceil_div(n, 256) >= 192            ? TILE_256
                                                                                   : TILE_128;
  if (!dma && tile == TILE_256) tile = TILE_128;
  return {tile, split(tile)};
}

long long part_bytes(long m, long n, const Plan &plan) {
  return plan.splits > 1 ? round16(4LL * plan.splits * m * ((n + 3) & ~3L)) : 0;
}

// The workspace that serves this product whatever the alignment of its operands.
long long product_bytes(long m, long n, long k, int type, bool amn, bool bmn, int tile, int splits) {
  return std::max(part_bytes(m, n, plan_product(m, n, k, type, amn, bmn, true, tile, splits)),
                  part_bytes(m, n, plan_product(m, n, k, type, amn, bmn, false, tile, splits)));
}

hipError_t run_product(Product &q, int tile, int splits, void *workspace, long long bytes, hipStream_t stream) {
  GemmParams &p = q.p;
  const int size = size_of(q.type);
  const bool dma = direct_loads(p.a, p.lda, q.amn, p.m, p.k, size) && direct_loads(p.b, p.ldb, q.bmn, p.n, p.k, size);
  Plan plan = plan_product(p.m, p.n, p.k, q.type, q.amn, q.bmn, dma, tile, splits);
  if (part_bytes(p.m, p.n, plan) > bytes) plan = plan_product(p.m, p.n, p.k, q.type, q.amn, q.bmn, dma, tile, 1);
  p.tiles_m = static_cast<int>(ceil_div(p.m, tile_size(plan.tile)));
  p.tiles_n = static_cast<int>(ceil_div(p.n, tile_size(plan.tile)));
  p.splits = plan.splits;
  p.parts = static_cast<float *>(workspace);
  const hipError_t e = q.type == TF_T_BF16  ? launch_gemm_bf16(p, q.amn, q.bmn, plan.tile, dma, stream)
                       : q.type == TF_T_F16 ? launch_gemm_f16(p, q.amn, q.bmn, plan.tile, dma, stream)
                                            : launch_gemm_f8(p, q.out_type, plan.tile, dma, stream);
  return e == hipSuccess && plan.splits > 1 ? launch_gemm_join(p, q.out_type, stream) : e;
}

void check_choice(Checks &c, int tile, int splits) {
  c.one_of("tile", tile, {0, TILE_256, TILE_128, TILE_64, TILE_ROWS});
  c.need(splits >= 0 && splits <= 64, "splits = ", static_cast<long long>(splits), " is not between 0 and 64");
}

void check_linear_sizes(Checks &c, const tf_linear_args_t *a) {
  c.one_of("type", a->type, {TF_T_BF16, TF_T_F16, TF_T_F8});
  if (a->type == TF_T_F8) c.one_of("out_type", a->out_type, {TF_T_BF16, TF_T_F16});
  else c.one_of("out_type", a->out_type, {a->type});
  c.size("m", a->m);
  c.size("n", a->n);
  c.size("k", a->k);
  check_choice(c, a->tile, a->splits);
}

int linear_workspace(const tf_linear_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_workspace: null arguments");
  Checks c{"tf_linear_workspace", {}};
  check_linear_sizes(c, a);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  *bytes = a->m && a->n ? product_bytes(a->m, a->n, a->k, a->type, false, a->w_order == 0, a->tile, a->splits) : 0;
  return TF_OK;
}

int linear(const tf_linear_args_t *a, hipStream_t stream) {
  const char *call = "tf_linear";
  if (!a) return fail(TF_E_ARG, "tf_linear: null arguments");
  Checks c{call, {}};
  check_linear_sizes(c, a);
  const bool f8 = a->type == TF_T_F8;
  c.one_of("w_order", a->w_order, {0, 1});
  c.need(!f8 || a->w_order == 1, "8-bit weights lie as n rows of k (w_order 1)");
  c.one_of("act", a->act, {TF_ACT_NONE, TF_ACT_RELU, TF_ACT_GELU, TF_ACT_SILU});
  if (a->bias) c.one_of("bias_type", a->bias_type, {a->out_type, TF_T_F32});
  c.matrix("x", a->x, a->x_ld, a->n ? a->m : 0, a->k, a->type, true);
  if (a->w_order) c.matrix("w", a->w, a->w_ld, a->m ? a->n : 0, a->k, a->type, true);
  else c.matrix("w", a->w, a->w_ld, a->m ? a->k : 0, a->n, a->type, true);
  c.vector("bias", a->bias, a->n, a->bias_type, false);
  c.matrix("residual", a->residual, a->residual_ld, a->m, a->n, a->out_type, false);
  c.matrix("out", a->out, a->out_ld, a->m, a->n, a->out_type, true);
  c.matrix("z", a->z, a->z_ld, a->m, a->n, a->out_type, false);
  c.vector("x_scale", a->x_scale, a->m, TF_T_F32, f8);
  c.vector("w_scale", a->w_scale, a->n, TF_T_F32, f8);
  c.need(f8 || (!a->x_scale && !a->w_scale), "scales belong to 8-bit products");
  if (a->workspace_bytes) c.workspace(a->workspace, a->workspace_bytes, 1);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->m == 0 || a->n == 0) return TF_OK;
  Product q{a->type, a->out_type, false, a->w_order == 0, {}};
  GemmParams &p = q.p;
  p.a = a->x, p.b = a->w, p.bias = a->bias, p.residual = a->residual, p.sa = a->x_scale, p.sb = a->w_scale;
  p.out = a->out, p.z = a->z, p.lda = a->x_ld, p.ldb = a->w_ld, p.ldr = a->residual_ld, p.ldo = a->out_ld, p.ldz = a->z_ld;
  p.m = static_cast<int>(a->m), p.n = static_cast<int>(a->n), p.k = static_cast<int>(a->k);
  p.act = a->act, p.bias_f32 = a->bias_type == TF_T_F32;
  return hip(run_product(q, a->tile, a->splits, a->workspace, a->workspace_bytes, stream), call);
}

// The gradient's workspace: dz, its column sums' shares, then one product's parts.
struct GradSpace {
  long long dz = 0, shares = 0, parts = 0, dz_ld = 0;
  long long bytes() const { return dz + shares + parts; }
};

GradSpace grad_space(const tf_linear_grad_args_t *a) {
  GradSpace s;
  if (a->m == 0 || a->n == 0) return s;
  s.dz_ld = (a->n + 7) & ~7LL;
  if (a->act != TF_ACT_NONE) s.dz = round16(2 * a->m * s.dz_ld);
  s.shares = round16(4 * column_shares(a->m) * a->n);
  if (a->k) {
    s.parts = product_bytes(a->m, a->k, a->n, a->type, false, a->w_order == 1, a->tile, a->splits);
    s.parts = std::max(s.parts, a->w_order ? product_bytes(a->n, a->k, a->m, a->type, true, true, a->tile, a->splits)
                                           : product_bytes(a->k, a->n, a->m, a->type, true, true, a->tile, a->splits));
  }
  return s;
}

void check_grad_sizes(Checks &c, const tf_linear_grad_args_t *a) {
  c.one_of("type", a->type, {TF_T_BF16, TF_T_F16});
  c.one_of("act", a->act, {TF_ACT_NONE, TF_ACT_RELU, TF_ACT_GELU, TF_ACT_SILU});
  c.one_of("w_order", a->w_order, {0, 1});
  c.size("m", a->m);
  c.size("n", a->n);
  c.size("k", a->k);
  check_choice(c, a->tile, a->splits);
}

int linear_grad_workspace(const tf_linear_grad_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_grad_workspace: null arguments");
  Checks c{"tf_linear_grad_workspace", {}};
  check_grad_sizes(c, a);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  *bytes = grad_space(a).bytes();
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
  c.matrix("z", a->z, a->z_ld, a->m, a->n, a->type, a->act != TF_ACT_NONE);
  c.matrix("x", a->x, a->x_ld, a->m, a->k, a->type, a->dw != nullptr);
  c.matrix("w", a->w, a->w_ld, wr, wc, a->type, a->dx != nullptr);
  c.matrix("dx", a->dx, a->dx_ld, a->m, a->k, a->type, false);
  c.matrix("dw", a->dw, a->dw_ld, wr, wc, a->type, false);
  c.vector("dbias", a->dbias, a->n, a->bias_type, false);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  const GradSpace space = grad_space(a);
  c.workspace(a->workspace, a->workspace_bytes, space.bytes());
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);

  char *ws = static_cast<char *>(a->workspace);
  const int m = static_cast<int>(a->m), n = static_cast<int>(a->n), k = static_cast<int>(a->k);
  const void *dz = a->dy;
  long dz_ld = a->dy_ld;
  hipError_t e = hipSuccess;
  if (m && n && (a->act != TF_ACT_NONE || a->dbias)) {
    SlopeParams s{a->dy, a->z, nullptr, a->dbias ? reinterpret_cast<float *>(ws + space.dz) : nullptr, a->dy_ld, a->z_ld,
                  space.dz_ld, m, n, a->act};
    if (a->act != TF_ACT_NONE) {
      dz = s.dz = ws;
      dz_ld = space.dz_ld;
    }
    e = launch_act_slope(s, a->type, stream);
  }
  if (e == hipSuccess && a->dbias && n)
    e = launch_share_sum(reinterpret_cast<float *>(ws + space.dz), m ? column_shares(m) : 0, n, a->dbias, a->bias_type, stream);
  void *parts = ws + space.dz + space.shares;
  if (e == hipSuccess && a->dx && m && k) {
    Product q{a->type, a->type, false, a->w_order == 1, {}};
    GemmParams &p = q.p;
    p.a = dz, p.lda = dz_ld, p.b = a->w, p.ldb = a->w_ld, p.out = a->dx, p.ldo = a->dx_ld;
    p.m = m, p.n = k, p.k = n;
    e = run_product(q, a->tile, a->splits, parts, space.parts, stream);
  }
  if (e == hipSuccess && a->dw && n && k) {
    Product q{a->type, a->type, true, true, {}};
    GemmParams &p = q.p;
    const bool nk = a->w_order == 1;
    p.a = nk ? dz : a->x, p.lda = nk ? dz_ld : a->x_ld, p.b = nk ? a->x : dz, p.ldb = nk ? a->x_ld : dz_ld;
    p.out = a->dw, p.ldo = a->dw_ld;
    p.m = nk ? n : k, p.n = nk ? k : n, p.k = m;
    e = run_product(q, a->tile, a->splits, parts, space.parts, stream);
  }
  return hip(e, call);
}

}  // namespace

extern "C" {

int tf_rms_norm(const tf_rms_norm_args_t *args, void *stream) {
  return guarded([&] { return rms_norm(args, static_cast<hipStream_t>(stream)); });
}

int tf_quantize_rows(const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                     float *scale, void *stream) {
  return guarded([&] { return quantize_rows(x, x_ld, rows, d, type, y, y_ld, scale, static_cast<hipStream_t>(stream)); });
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
