// What the C ABI's calls share: checks of arguments, the operands of a product as the
// kernels see them, and the choice of tile and of ranges of k.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "errors.h"
#include "nn_kernels.h"
#include "tforge_hip.h"

namespace tfnn {

using tfk::fail;
using tfk::guarded;

constexpr long long kMostSize = 1LL << 30;
constexpr long long kMostI8 = (1LL << 31) / (128 * 128) - 1;  // products of two codes in a 32-bit sum

inline bool eight_bits(int type) { return type == TF_T_F8 || type == TF_T_I8; }
inline int size_of(int type) { return type == TF_T_F32 ? 4 : eight_bits(type) ? 1 : 2; }

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

inline int hip(hipError_t e, const char *call) {
  return e == hipSuccess ? TF_OK : fail(TF_E_HIP, std::string(call) + " failed: " + hipGetErrorString(e));
}


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
  bool square = false;  // on the square tiles alone
  bool logits = false;  // the loss's: statistics or dz leave a tile
};

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }
inline long long round16(long long bytes) { return (bytes + 15) & ~15LL; }

// Whether an operand's loads may go straight into LDS: 16-byte aligned lines of
// whole pieces, and every offset inside a tile's slab below 2^31 bytes.
inline bool direct_loads(const Operand &o, int size) {
  const int piece = 16 / size;
  const long span = o.mn ? 64 * o.ld * size + 1024 : 256 * o.ld * size + 256;
  if (span >= (1L << 31)) return false;
  return o.ours || (reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.ld % piece == 0 && o.length % piece == 0);
}

// Whether loads of these lines may start off four bytes.
inline bool off_four(const Operand &o, int size) {
  return reinterpret_cast<uintptr_t>(o.p) % 4 || o.ld * size % 4 || (o.mn && o.length * size % 4);
}

// The same operand copied to aligned lines: whole cache lines, so that no 128 bytes
// of a tile's line lie in two.
inline long packed_ld(const Operand &o, int size) { return ceil_div(o.length, 128 / size) * (128 / size); }
inline long long packed_bytes(const Operand &o, int size) { return round16(o.lines * packed_ld(o, size) * size); }

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
// logits: without a time for written results, which the large tiles' ends do not need there (8192 rows, 32768 classes and
// k of 512, bfloat16, 128/256-tile: the loss 303 / 271, its gradient 1132 / 1035).
inline double predicted(double m, double n, double slabs, double read, bool dma, bool f8, int tile, int splits, bool logits) {
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
  return splits > 1 ? us + c.join + c.join_part * splits * results : std::max(us, logits ? 0.0 : 4.5 + results * c.written);
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
inline Plan plan_product(const Product &q, bool dma, int tile, int splits) {
  const long m = q.p.m, n = q.p.n, k = q.p.k;
  const int type = q.type, terms = q.p.terms;
  const bool amn = q.a.mn, bmn = q.b.mn;
  const int size = size_of(type);
  const long slabs = ceil_div(k, 128 / size);
  // A launch takes fewer than 2^32 threads.  (Through registers its grid may have two sides.)
  const auto tiles_of = [&](int t) { return ceil_div(m, tile_rows(t)) * ceil_div(n, tile_columns(t)); };
  const auto fits = [&](int t, long blocks) { return blocks * tile_threads(t) < (1L << 32); };
  const bool rows = !q.square && m * terms <= 64 && !amn && (!bmn || n >= 32) && fits(TILE_ROWS, ceil_div(n, bmn ? 32 : 16));
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
    if (q.square && t == TILE_64x128) continue;
    // Tiles mostly empty, and splits into more than four workgroups a CU, never win.
    if (!tile && t != TILE_64 && (2 * m <= tile_rows(t) || 2 * n <= tile_columns(t)) && fits(TILE_64, tiles_of(TILE_64))) continue;
    const long tiles = tiles_of(t);
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (s > 1 && (splits || s * 2 > slabs || tiles * s > 1024)) break;
      const int ranges = splits ? splits : s;
      if (dma && !fits(t, tiles * ranges)) continue;
      const double us = predicted(m, n, slabs * terms, read, dma, size == 1, t, ranges, q.logits);
      if (us < best.us) best = {t, ranges, us};
    }
  }
  return best;
}

inline long long part_bytes(long m, long n, const Plan &plan) {
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

inline Choice choose(const Product &q, int tile, int splits, bool packing = true) {
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
inline void place(Product &q, const Plan &plan, void *parts) {
  GemmParams &p = q.p;
  p.a = q.a.p, p.lda = q.a.ld, p.b = q.b.p, p.ldb = q.b.ld;
  p.tiles_m = static_cast<int>(ceil_div(p.m, tile_rows(plan.tile)));
  p.tiles_n = static_cast<int>(ceil_div(p.n, tile_columns(plan.tile)));
  p.splits = plan.splits;
  p.parts = static_cast<float *>(parts);
}

// The operand becomes its aligned copy at `to`, one more of `pack`; the copy's bytes.
inline long long copy_of(Operand &o, int size, char *to, PackParams &pack) {
  const int i = pack.pieces[0] ? 1 : 0;
  const long ld = packed_ld(o, size);
  const long long bytes = packed_bytes(o, size);
  pack.from[i] = o.p, pack.from_ld[i] = o.ld, pack.rows[i] = o.lines, pack.columns[i] = static_cast<int>(o.length);
  pack.to[i] = to, pack.to_ld[i] = ld, pack.pieces[i] = o.lines * ld * size / 16;
  o.p = to, o.ld = ld, o.ours = true;
  return bytes;
}

// Whether the product's own kernel can write z in 8 bits: unsplit, loads straight into LDS, more than a few rows.
inline bool fused_z(const Choice &c) { return c.dma && c.plan.splits == 1 && c.plan.tile != TILE_ROWS; }

inline hipError_t run_product(Product &q, int tile, int splits, void *workspace, long long bytes, hipStream_t stream, void *z8 = nullptr) {
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
  if (z8) {
    KeptGemmParams p;
    static_cast<GemmParams &>(p) = q.p;
    p.groups = ceil_div(p.n, 32);
    p.codes = static_cast<unsigned char *>(z8), p.exponents = p.codes + p.m * p.groups * 32;
    return launch_gemm_kept(p, q.type, q.b.mn, c.plan.tile, stream);
  }
  e = q.type == TF_T_BF16  ? launch_gemm_bf16(q.p, q.a.mn, q.b.mn, c.plan.tile, c.dma, stream)
      : q.type == TF_T_F16 ? launch_gemm_f16(q.p, q.a.mn, q.b.mn, c.plan.tile, c.dma, stream)
      : q.type == TF_T_F8  ? launch_gemm_f8(q.p, q.out_type, c.plan.tile, c.dma, stream)
                           : launch_gemm_i8(q.p, q.out_type, c.plan.tile, c.dma, stream);
  return e == hipSuccess && c.plan.splits > 1 ? launch_gemm_join(q.p, q.type, q.out_type, stream) : e;
}

inline void check_choice(Checks &c, int tile, int splits) {
  c.one_of("tile", tile, {0, TILE_256, TILE_128, TILE_64, TILE_ROWS, TILE_64x128});
  c.need(splits >= 0 && splits <= 64, "splits = ", static_cast<long long>(splits), " is not between 0 and 64");
}

}  // namespace tfnn
