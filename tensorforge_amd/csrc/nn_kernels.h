// Parameters and launchers of the residual block's operators (norm, products,
// gradients): what the C ABI (nn.hip) hands to the kernels' translation units.
#pragma once

#include <hip/hip_runtime.h>

namespace tfnn {

// The values of TF_T_* in tforge_hip.h.
enum Type { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2, TYPE_F8 = 3 };

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
  const void *dy, *h, *dh, *weight;
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
  float *parts = nullptr;  // splits > 1: splits x m x (n up to a multiple of 4)
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

// Up to two matrices copied to rows of whole 16-byte pieces, zeros in the pad.
struct PackParams {
  const void *from[2] = {};
  void *to[2] = {};
  long from_ld[2] = {}, to_ld[2] = {}, rows[2] = {};  // elements
  int columns[2] = {};
  long pieces[2] = {};  // rows x to_ld in pieces; 0: none
};
hipError_t launch_pack(const PackParams &p, int size, hipStream_t stream);

// out = epilogue(sum of the splits' parts).
hipError_t launch_gemm_join(const GemmParams &p, int out_type, hipStream_t stream);
// The same of a pair's products, those that are split.
hipError_t launch_gemm_join_pair(const GemmParams &dx, const GemmParams &dw, int out_type, hipStream_t stream);

struct SlopeParams {
  const void *dy, *z;
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

long norm_grad_shares(long rows, long d);
hipError_t launch_rms_norm(const NormParams &p, int type, bool to_f8, hipStream_t stream);
hipError_t launch_rms_norm_grad(const NormGradParams &p, int type, hipStream_t stream);

}  // namespace tfnn
