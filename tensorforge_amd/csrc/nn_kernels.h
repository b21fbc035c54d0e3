// Parameters and launchers of the residual block's operators (norm, products,
// gradients): what the C ABI (nn.hip) hands to the kernels' translation units.
#pragma once

#include <hip/hip_runtime.h>

namespace tfnn {

// The values of TF_T_* in tforge_hip.h.
enum Type { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2, TYPE_F8 = 3, TYPE_I8 = 4 };

// *_ld: elements between two rows.
struct NormParams {
  const void *x = nullptr, *residual = nullptr;
  const void *weight = nullptr;  // null: rows are quantised as they are
  void *y = nullptr, *h = nullptr;
  float *scale = nullptr;  // 8-bit output only
  long x_ld = 0, residual_ld = 0, y_ld = 0, h_ld = 0, rows = 0;
  int d = 0, weight_type = 0;
  float eps = 0;
};

struct NormGradParams {
  const void *dy, *h, *dh, *weight;  // h in `type`, or kept in 8 bits
  bool kept;
  void *dx, *dw;
  float *shares;  // norm_grad_shares(rows, d) x d
  long dy_ld, h_ld, dh_ld, dx_ld, rows;
  int d, weight_type;
  float eps;
};

struct GemmParams {
  const void *a = nullptr, *b = nullptr;
  const void *bias = nullptr, *residual = nullptr;
  const float *sa = nullptr, *sb = nullptr;  // 8 bits: scales of A's rows and B's columns
  void *out = nullptr, *z = nullptr;
  float *parts = nullptr;  // splits > 1: splits x m x (n up to a multiple of 4); of 8-bit integers, integers
  long lda = 0, ldb = 0, ldr = 0, ldo = 0, ldz = 0;
  int m = 0, n = 0, k = 0;
  int tiles_m = 0, tiles_n = 0, splits = 1;
  int act = 0, bias_f32 = 0;
  int terms = 1;                // 2: another term of A at a + a_term, or of B at b + b_term (bytes);
                                // the first is what the other's rounding left
  long a_term = 0, b_term = 0;  // (all tiles but 256; few rows: of A, up to 32 rows)
};

// C tiles of the product kernels; but for 64 x 64 they load straight into LDS only.
// TILE_ROWS: all of up to 64 rows, the waves of a workgroup split k (the left
// operand along k only).
enum Tile { TILE_256 = 1, TILE_128 = 2, TILE_64 = 3, TILE_ROWS = 4, TILE_64x128 = 5 };
constexpr int tile_rows(int tile) { return tile == TILE_256 ? 256 : tile == TILE_128 ? 128 : 64; }
constexpr int tile_threads(int tile) { return tile == TILE_256 ? 512 : tile == TILE_ROWS ? 1024 : 256; }  // at most
constexpr int tile_columns(int tile) { return tile == TILE_64x128 ? 128 : tile_rows(tile); }

// amn, bmn: the operand's own dimension (m, n) is contiguous, not k.
hipError_t launch_gemm_bf16(const GemmParams &p, bool amn, bool bmn, int tile, bool dma, hipStream_t stream);
hipError_t launch_gemm_f16(const GemmParams &p, bool amn, bool bmn, int tile, bool dma, hipStream_t stream);
hipError_t launch_gemm_f8(const GemmParams &p, int out_type, int tile, bool dma, hipStream_t stream);
hipError_t launch_gemm_i8(const GemmParams &p, int out_type, int tile, bool dma, hipStream_t stream);
// A sum of `count` shares of d floats, rounded to `type`; d = 0: none.
struct ShareParams {
  const float *shares = nullptr;
  void *out = nullptr;
  int count = 0, d = 0, type = 0;
};
// Both products of a small layer's gradient in one launch, 64 x 64 tiles, loads
// straight into LDS: dx with amn false, dw with amn and bmn true; and a sum.
hipError_t launch_gemm_pair_bf16(const GemmParams &dx, bool bmn, const GemmParams &dw, const ShareParams &sum, hipStream_t stream);
hipError_t launch_gemm_pair_f16(const GemmParams &dx, bool bmn, const GemmParams &dw, const ShareParams &sum, hipStream_t stream);

// A product that keeps z in 8 bits: rows of `groups` groups.
struct KeptGemmParams : GemmParams {
  unsigned char *codes = nullptr, *exponents = nullptr;
  long groups = 0;
};
// All tiles but the few rows', unsplit, loads straight into LDS; z is null.
hipError_t launch_gemm_kept(const KeptGemmParams &p, int type, bool bmn, int tile, hipStream_t stream);

// The products of the loss over a vocabulary and of its gradient.  The loss of row m is
// lse[m] - logit(m, target[m]); a row whose target is `ignore` does not count, one whose
// target is outside of the vocabulary is NaN.
struct XentParams : GemmParams {
  const long long *target = nullptr;
  long long ignore = 0;
  int vocabulary = 0, column0 = 0;  // all columns, and this piece's first
  // XENT_STATS: of each row and a tile's columns t, the largest logit times log2(e) as it was rounded, and the sum of
  // exp2(logit * log2(e) - t): tiles_n x m pairs.  And the target's logit, as it is.
  float *stats = nullptr, *target_logit = nullptr;
  // XENT_SLOPE: out = (exp(logit - lse) - [column is the target]) * unit, zeros up to a multiple of 8 columns.  One dloss
  // for all rows: the unit is `power`, and dloss / count / power comes with XENT_SUM.  A row's own: dloss / count, in
  // float16 times scale[0].
  const double *lse = nullptr;
  const float *dloss = nullptr, *count = nullptr, *scale = nullptr;
  float power = 1.0f;
  int dloss_rows = 0;
  long lo = 0;  // not 0: what dz's rounding left, rounded, that many elements behind
  // XENT_SUM: out = (product + sum) * dloss / count / power (scale[1] or 1 with a dloss a row), or the new sum; m x (n up to a
  // multiple of 4) floats.
  float *sum = nullptr;
  int add = 0, last = 0;
  // The rows are twice as many: of both terms of dz, the value's and then what its rounding left, whose products
  // go to `parts` for the join to add.
  int halves = 0;
};
enum XentProduct { XENT_STATS, XENT_SLOPE, XENT_SUM };
// Tiles 256, 128 and 64.  XENT_STATS and XENT_SLOPE: amn false.
hipError_t launch_xent_bf16(const XentParams &p, XentProduct what, bool amn, bool bmn, int tile, bool dma, hipStream_t stream);
hipError_t launch_xent_f16(const XentParams &p, XentProduct what, bool amn, bool bmn, int tile, bool dma, hipStream_t stream);

// Up to two matrices copied to rows of whole 16-byte pieces, zeros in the pad.
struct PackParams {
  const void *from[2] = {};
  void *to[2] = {};
  long from_ld[2] = {}, to_ld[2] = {}, rows[2] = {};  // elements
  int columns[2] = {};
  long pieces[2] = {};  // rows x to_ld in pieces; 0: none
  bool kept[2] = {};    // what is kept in 8 bits, restored in the copies' type
};
hipError_t launch_pack(const PackParams &p, int type, hipStream_t stream);

// out = epilogue(sum of the splits' parts), which are those of a product of `type`.
hipError_t launch_gemm_join(const GemmParams &p, int type, int out_type, hipStream_t stream);
// The same of a pair's products, those that are split.
hipError_t launch_gemm_join_pair(const GemmParams &dx, const GemmParams &dw, int out_type, hipStream_t stream);

struct SlopeParams {
  const void *dy, *z;  // z in `type`, or kept in 8 bits
  bool kept;
  void *dz;       // m x dz_ld, columns from n on zero; null: sums alone
  long lo;        // not 0: what dz's rounding left, rounded, that many elements behind
  float *shares;  // ceil(m / rows) x n; null with one share, or without sums
  void *sums;     // with one share, the sums themselves, of sums_type; else null
  long dy_ld, z_ld, dz_ld;
  int m, n, act, sums_type;
  int rows;  // a workgroup's: one of SlopeRows
};
enum SlopeRows { SLOPE_FEW = 32, SLOPE_MANY = 64, SLOPE_WHOLE = 256 };
// dz = dy * act'(z) (act none: dy), and dz's column sums; beside them the copies of `pack`.
hipError_t launch_act_slope(const SlopeParams &p, const PackParams &pack, int type, hipStream_t stream);
// out[0..d) = sum of `count` shares, in order, rounded to `type`.
hipError_t launch_share_sum(const float *shares, long count, int d, void *out, int type, hipStream_t stream);

// Rows into 8 bits in groups (nn_common.hpp) and back.  positive: values above zero keep a code above zero; masked:
// minus infinity is kept.
hipError_t launch_keep(const void *x, long ld, long rows, int d, int type, bool positive, bool masked, void *kept, hipStream_t stream);
hipError_t launch_restore(const void *kept, long rows, int d, int type, void *x, long ld, hipStream_t stream);

long norm_grad_shares(long rows, long d);
hipError_t launch_rms_norm(const NormParams &p, int type, int y_type, hipStream_t stream);
hipError_t launch_rms_norm_grad(const NormGradParams &p, int type, hipStream_t stream);

}  // namespace tfnn
