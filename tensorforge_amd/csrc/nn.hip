// C ABI of the residual block's operators (declared at the end of
// include/tforge_hip.h): checks of arguments, the choice of tile and of ranges
// of k, and the order of launches.
#include <algorithm>
#include <cmath>
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
constexpr long long kMostI8 = (1LL << 31) / (128 * 128) - 1;  // products of two codes in a 32-bit sum

bool eight_bits(int type) { return type == TF_T_F8 || type == TF_T_I8; }
int size_of(int type) { return type == TF_T_F32 ? 4 : eight_bits(type) ? 1 : 2; }

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
  // Rows kept in 8 bits.
  void kept(const char *name, const void *p, long long rows, long long d, bool wanted) {
    if (!fine() || rows <= 0 || d <= 0) return;
    need(p || !wanted, name, " is a null pointer");
    need(reinterpret_cast<uintptr_t>(p) % 16 == 0, name, ", kept in 8 bits, is not 16-byte aligned");
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

// ---- products -------------------------------------------------------------------

// One operand as the kernels see it: `lines` lines of `length` contiguous
// elements; mn: lines of its own dimension, not of k.  ours: in the workspace,
// aligned, whole pieces a line, zeros in the pad.
struct Operand {
  const void *p = nullptr;
  long ld = 0, lines = 0, length = 0;
  bool mn = false, ours = false;
};

struct Product {
  int type, out_type;
  Operand a, b;
  GemmParams p;  // sizes, output and epilogue
};

long ceil_div(long a, long b) { return (a + b - 1) / b; }
long long round16(long long bytes) { return (bytes + 15) & ~15LL; }

// Whether an operand's loads may go straight into LDS: 16-byte aligned lines of
// whole pieces, and every offset inside a tile's slab below 2^31 bytes.
bool direct_loads(const Operand &o, int size) {
  const int piece = 16 / size;
  const long span = o.mn ? 64 * o.ld * size + 1024 : 256 * o.ld * size + 256;
  if (span >= (1L << 31)) return false;
  return o.ours || (reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.ld % piece == 0 && o.length % piece == 0);
}

// Whether loads of these lines may start off four bytes.
bool off_four(const Operand &o, int size) {
  return reinterpret_cast<uintptr_t>(o.p) % 4 || o.ld * size % 4 || (o.mn && o.length * size % 4);
}

// The same operand copied to aligned lines: whole cache lines, so that no 128 bytes
// of a tile's line lie in two.
long packed_ld(const Operand &o, int size) { return ceil_div(o.length, 128 / size) * (128 / size); }
long long packed_bytes(const Operand &o, int size) { return round16(o.lines * packed_ld(o, size) * size); }

struct Plan {
  int tile, splits;
  double us;  // predicted
};

// What a product takes on one tile (us), fitted to 7444 measurements on MI355X: 500 products
// with sizes drawn from 64 to 8192, bfloat16 and 8 bits, each tile, k in 1 to 16 ranges; it
// errs by 6 to 9% (root mean square), and its choices take 1.8% longer than the best of
// them (of 250 others: 3.5%).  `most` workgroups fit on a CU; one takes `end` and `slab` for each of its slabs (64
// elements of k in 16 bits, 128 in 8) with the CU to itself, `end_most` and `slab_most` (8
// bits: times f8) when it is full.  A last round of workgroups that leaves CUs empty takes
// at least `rest` of a full one.  A split adds its join, start and per 1e6 results and
// range; results that are written cost their bytes, per 1e6.  Both sides (us, bfloat16):
// 512 x 4096 x 4096 64/128/256-tile 28.4 / 44.3 / 80.6, 2048 x 4096 x 4096 101 / 62.8 / 84,
// 4096^3 190 / 122 / 105; split 1/2/4 ways 256 x 4096 x 4096 64-tile 23.6 / 21.0 / 24.4,
// 2048 x 2048 x 8192 128-tile 88.6 / 72.7 / -, 96 x 2048 x 8192 64-tile 41.6 / 25.5 / 17.5
// (8: 15.6); 4096 x 4096 x 64 64/64 x 128/128/256-tile 15.2 / 16.6 / 14.1 / 12.4.
struct TileCost {
  int most;
  double start, end, end_most, slab, slab_most, f8, rest, join, join_part, written;
};
constexpr TileCost kCost256{1, 7.0, 3.5, 1.3, 1.03, 1.21, 1.12, 1.0, 1.1, 1.34, 1.02};
constexpr TileCost kCost128{2, 5.5, 0.0, 0.57, 0.58, 0.78, 1.23, 0.78, 1.8, 1.56, 0.82};
constexpr TileCost kCost64x128{2, 2.5, 1.9, 2.9, 0.38, 0.58, 1.1, 0.49, 2.4, 1.36, 0.28};
constexpr TileCost kCost64{3, 3.6, 0.04, 0.58, 0.27, 0.56, 1.09, 0.6, 2.5, 1.74, 0.21};
// Loads through registers (64 x 64), fitted to 200 products of odd sizes: within 6%.
constexpr TileCost kCostAny{3, 3.9, 0.55, 3.0, 0.28, 0.92, 1.09, 0.2, 2.5, 1.74, 1.37};

// Few slabs of LDS let five 64 x 64 tiles on a CU, from 768 on: 3.5, and a workgroup 0.46
// and 0.22 a slab.  read: the operands' bytes at 8 TB/s.
double predicted(double m, double n, double slabs, double read, bool dma, bool f8, int tile, int splits) {
  const TileCost &c = !dma ? kCostAny : tile == TILE_256 ? kCost256 : tile == TILE_128 ? kCost128 : tile == TILE_64 ? kCost64 : kCost64x128;
  const double each = std::ceil(slabs / splits), results = m * n / 1e6, most = c.most;
  const double w = std::ceil(m / tile_rows(tile)) * std::ceil(n / tile_columns(tile)) * splits / 256;  // workgroups a CU
  const double slab_most = f8 ? c.slab_most * c.f8 : c.slab_most;
  double us;
  if (dma && tile == TILE_64 && w > 3) {
    us = 3.5 + w * (0.46 + each * (f8 ? 0.22 * c.f8 : 0.22));
  } else {
    const double full = each * slab_most + c.end_most, rounds = std::floor(w / most), rest = w - rounds * most;
    us = c.start + rounds * full;
    if (rest > 0 && rounds > 0) us += full * (c.rest + (1 - c.rest) * rest / most);
    if (rest > 0 && rounds == 0) {  // spread over the CUs: how full one is
      const double of = most > 1 ? (std::ceil(rest) - 1) / (most - 1) : 0;
      const double slab = c.slab + (slab_most - c.slab) * (most > 1 ? of : rest);  // one alone: the power limit
      us += each * slab + c.end + (c.end_most - c.end) * of;
    }
  }
  us = std::max(us, 4.5 + read);
  return splits > 1 ? us + c.join + c.join_part * splits * results : std::max(us, 4.5 + results * c.written);
}

// The C tile and the ranges of k for a product of these sizes: the least
// predicted time.  Up to 64 rows the few-row kernel stands beside the tiles; a workgroup
// reads its columns' k at about 110 bytes a nanosecond and all rows' (from the caches) at
// 45, fitted to 200 products of 1 to 64 rows.  Measured, bfloat16, us
// (few-row / 64-tile), w 4096 x 4096 as n rows of k: 7.7 / 10.8 for 1 row, 9.8 / 11.1
// for 16, 13.7 / 11.6 for 32; as k rows of n: 11.4 / 11.6, 13.4 / 12.2, 16.1 / 12.5 (w partly
// in the caches; from memory alone 1 row takes 17.8 so, 7.7 on n rows of k).
// A left operand of two terms counts as twice the rows here, as twice the slabs on the tiles.
// Lines off four bytes take it longer (150 more): 5 x 4224 x 1022 5.3, x 1023 10.6 (8.1 on the
// 64-tile); 4 x 5911 x 5281 40.8 and 21.8.
Plan plan_product(const Product &q, bool dma, int tile, int splits) {
  const long m = q.p.m, n = q.p.n, k = q.p.k;
  const int type = q.type, terms = q.p.terms;
  const bool amn = q.a.mn, bmn = q.b.mn;
  const int size = size_of(type);
  const long slabs = ceil_div(k, 128 / size);
  // A launch takes fewer than 2^32 threads.  (Through registers its grid may have two sides.)
  const auto tiles_of = [&](int t) { return ceil_div(m, tile_rows(t)) * ceil_div(n, tile_columns(t)); };
  const auto fits = [&](int t, long blocks) { return blocks * tile_threads(t) < (1L << 32); };
  const bool rows = m * terms <= 64 && !amn && (!bmn || n >= 32) && fits(TILE_ROWS, ceil_div(n, bmn ? 32 : 16));
  if (tile == TILE_ROWS && rows) return {TILE_ROWS, 1, 0};
  if (tile == TILE_ROWS || (!dma && tile != TILE_64) || (terms > 1 && tile == TILE_256)) tile = 0;
  splits = static_cast<int>(std::max<long>(0, std::min<long>(splits, std::max<long>(1, slabs))));
  if (m * ceil_div(n, 4) >= (1L << 31)) splits = 1;  // the join counts quads in 32 bits; so many need no split
  if (tile && dma && !fits(tile, tiles_of(tile) * std::max(1, splits))) tile = 0;
  Plan best{TILE_64, 1, 1e30};
  const double read = (static_cast<double>(m) + n) * k * terms * size / 8e6;
  if (rows && !tile) {
    const long cols = bmn ? 32 : 16;
    const double bytes = static_cast<double>(k) * size / 1e3;
    const double of_b = cols / 110.0 * (!off_four(q.b, size) ? 1 : bmn ? 1.9 : 7.5);
    const double of_a = m * terms / 45.0 * (off_four(q.a, size) ? 3.3 : 1);
    best = {TILE_ROWS, 1, 3.4 + std::max(read, ceil_div(ceil_div(n, cols), 256) * (of_b + of_a) * bytes)};
  }
  for (int t : {TILE_64, TILE_64x128, TILE_128, TILE_256}) {
    if (tile ? t != tile : (t != TILE_64 && !dma) || (t == TILE_256 && terms > 1)) continue;
    // Tiles mostly empty, and splits into more than four workgroups a CU, never win.
    if (!tile && t != TILE_64 && (2 * m <= tile_rows(t) || 2 * n <= tile_columns(t)) && fits(TILE_64, tiles_of(TILE_64))) continue;
    const long tiles = tiles_of(t);
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (s > 1 && (splits || s * 2 > slabs || tiles * s > 1024)) break;
      const int ranges = splits ? splits : s;
      if (dma && !fits(t, tiles * ranges)) continue;
      const double us = predicted(m, n, slabs * terms, read, dma, size == 1, t, ranges);
      if (us < best.us) best = {t, ranges, us};
    }
  }
  return best;
}

long long part_bytes(long m, long n, const Plan &plan) {
  return plan.splits > 1 ? round16(4LL * plan.splits * m * ((n + 3) & ~3L)) : 0;
}

// How a product runs.  Operands that cannot be loaded straight into LDS are
// copied to aligned lines first (pack) where the faster kernels gain more than the
// copy takes, about 3.7 us and 0.21 for its 1e6 bytes; results in rows off 16 bytes then
// take 0.28 more for each 1e6 (fitted to the same products; the choices take 1.8% longer than
// the best).  Long matrices of lines far shorter than a cache line, whose copies would take many
// times their memory (2^30 rows of one element 128 GB for 2), stay as they are.  4095 x 4097 x 1023 bfloat16 110 us through registers, 62 with both copied; 777 x
// 1111 x 333 6.2 and 10.4.
constexpr long long kCopies = 256 << 20;  // bytes any copies may have

struct Choice {
  Plan plan;
  bool dma = false, pack_a = false, pack_b = false;
  double us = 0;  // predicted, copies and all
  long long parts = 0, copies = 0;
  long long bytes() const { return parts + copies; }
};

Choice choose(const Product &q, int tile, int splits, bool packing = true) {
  const GemmParams &p = q.p;
  const int size = size_of(q.type);
  Choice c;
  const bool da = direct_loads(q.a, size), db = direct_loads(q.b, size);
  c.dma = da && db;
  c.plan = plan_product(q, c.dma, tile, splits);
  c.us = c.plan.us;
  if (!c.dma && packing && p.k > 0 && c.plan.tile != TILE_ROWS) {
    const long long copies = (da ? 0 : packed_bytes(q.a, size)) + (db ? 0 : packed_bytes(q.b, size));
    const long long own = ((da ? 0 : q.a.lines * q.a.length) + (db ? 0 : q.b.lines * q.b.length)) * size;
    const auto fits = [&](const Operand &o) { return 256 * packed_ld(o, size) * size + 1024 < (1L << 31); };
    const Plan fast = plan_product(q, true, tile, splits);
    const double us = fast.us + 3.7 + copies * 0.21e-6 + (p.n % 8 ? 0.28e-6 * p.m * p.n : 0);
    if (fits(q.a) && fits(q.b) && copies <= std::max(4 * own, kCopies) && ((tile && tile != TILE_64 && tile != TILE_ROWS) || us < c.us)) {
      c.plan = fast;
      c.us = us;
      c.dma = true;
      c.pack_a = !da;
      c.pack_b = !db;
      c.copies = copies;
    }
  }
  c.parts = part_bytes(p.m, p.n, c.plan);
  return c;
}

// Fills in the kernels' view of a product that runs on this plan.
void place(Product &q, const Plan &plan, void *parts) {
  GemmParams &p = q.p;
  p.a = q.a.p, p.lda = q.a.ld, p.b = q.b.p, p.ldb = q.b.ld;
  p.tiles_m = static_cast<int>(ceil_div(p.m, tile_rows(plan.tile)));
  p.tiles_n = static_cast<int>(ceil_div(p.n, tile_columns(plan.tile)));
  p.splits = plan.splits;
  p.parts = static_cast<float *>(parts);
}

// The operand becomes its aligned copy at `to`, one more of `pack`; the copy's bytes.
long long copy_of(Operand &o, int size, char *to, PackParams &pack) {
  const int i = pack.pieces[0] ? 1 : 0;
  const long ld = packed_ld(o, size);
  const long long bytes = packed_bytes(o, size);
  pack.from[i] = o.p, pack.from_ld[i] = o.ld, pack.rows[i] = o.lines, pack.columns[i] = static_cast<int>(o.length);
  pack.to[i] = to, pack.to_ld[i] = ld, pack.pieces[i] = o.lines * ld * size / 16;
  o.p = to, o.ld = ld, o.ours = true;
  return bytes;
}

hipError_t run_product(Product &q, int tile, int splits, void *workspace, long long bytes, hipStream_t stream) {
  const int size = size_of(q.type);
  Choice c = choose(q, tile, splits);
  if (c.bytes() > bytes) c = choose(q, tile, 1, false);
  hipError_t e = hipSuccess;
  if (c.pack_a || c.pack_b) {
    char *to = static_cast<char *>(workspace) + c.parts;
    PackParams pack;
    if (c.pack_a) to += copy_of(q.a, size, to, pack);
    if (c.pack_b) copy_of(q.b, size, to, pack);
    e = launch_pack(pack, q.type, stream);
    if (e != hipSuccess) return e;
  }
  place(q, c.plan, workspace);
  e = q.type == TF_T_BF16  ? launch_gemm_bf16(q.p, q.a.mn, q.b.mn, c.plan.tile, c.dma, stream)
      : q.type == TF_T_F16 ? launch_gemm_f16(q.p, q.a.mn, q.b.mn, c.plan.tile, c.dma, stream)
      : q.type == TF_T_F8  ? launch_gemm_f8(q.p, q.out_type, c.plan.tile, c.dma, stream)
                           : launch_gemm_i8(q.p, q.out_type, c.plan.tile, c.dma, stream);
  return e == hipSuccess && c.plan.splits > 1 ? launch_gemm_join(q.p, q.type, q.out_type, stream) : e;
}

void check_choice(Checks &c, int tile, int splits) {
  c.one_of("tile", tile, {0, TILE_256, TILE_128, TILE_64, TILE_ROWS, TILE_64x128});
  c.need(splits >= 0 && splits <= 64, "splits = ", static_cast<long long>(splits), " is not between 0 and 64");
}

void check_linear_sizes(Checks &c, const tf_linear_args_t *a) {
  c.one_of("type", a->type, {TF_T_BF16, TF_T_F16, TF_T_F8, TF_T_I8});
  if (eight_bits(a->type)) c.one_of("out_type", a->out_type, {TF_T_BF16, TF_T_F16});
  else c.one_of("out_type", a->out_type, {a->type});
  c.size("m", a->m);
  c.size("n", a->n);
  c.size("k", a->k);
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

int linear_workspace(const tf_linear_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_workspace: null arguments");
  Checks c{"tf_linear_workspace", {}};
  check_linear_sizes(c, a);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  *bytes = a->m && a->n ? choose(product_of(a), a->tile, a->splits).bytes() : 0;
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
  c.matrix("z", a->z, a->z_ld, a->m, a->n, a->out_type, false);
  c.vector("x_scale", a->x_scale, a->m, TF_T_F32, eight);
  c.vector("w_scale", a->w_scale, a->n, TF_T_F32, eight);
  c.need(eight || (!a->x_scale && !a->w_scale), "scales belong to 8-bit products");
  if (a->workspace_bytes) c.workspace(a->workspace, a->workspace_bytes, 1);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (a->m == 0 || a->n == 0) return TF_OK;
  Product q = product_of(a);
  return hip(run_product(q, a->tile, a->splits, a->workspace, a->workspace_bytes, stream), call);
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
  return guarded([&] {
    Checks c{"tf_keep8", {}};
    c.one_of("type", type, {TF_T_F32, TF_T_BF16, TF_T_F16});
    c.one_of("positive", positive, {0, 1});
    c.size("rows", rows);
    c.size("d", d);
    c.matrix("x", x, x_ld, rows, d, type, true);
    c.kept("kept", kept, rows, d, true);
    if (!c.fine()) return fail(TF_E_ARG, c.wrong);
    if (rows == 0 || d == 0) return TF_OK;
    return hip(launch_keep(x, x_ld, rows, static_cast<int>(d), type, positive != 0, kept, static_cast<hipStream_t>(stream)), "tf_keep8");
  });
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
