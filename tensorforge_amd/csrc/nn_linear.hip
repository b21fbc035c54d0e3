// What the products need beside the matrix kernels: the join of a product split
// along k, aligned copies of operands, and the activation's slope with the bias
// gradient's sums.
#include "nn_gemm.hpp"

#include <algorithm>
#include <type_traits>

namespace tfnn {
namespace {

// Four columns a thread: the parts' sum in order, then the tile kernels' epilogue.
// Bound by latency: 64 x 4096 of four parts 3.0-3.8 us.  (Joined by the last of a tile's
// workgroups instead, behind a fence, the whole product took 22.9 us against 13.1: the caches'
// write-back costs more than the launch.)
template <typename S, typename O, int ACT>
__device__ __forceinline__ void join_four(const GemmParams &p, unsigned block) {
  typedef typename Vec<S, 4>::type S4;  // the parts' type: float, or int
  // (plan_product splits no product of 2^31 quads or more.  A 64-bit division takes 0.3 us here.)
  const unsigned quads = (p.n + 3u) / 4, id = block * 256 + threadIdx.x;
  const int m = static_cast<int>(id / quads), n = static_cast<int>(id % quads) * 4;
  const long ld = 4L * quads;
  if (m >= p.m) return;
  const S *part = reinterpret_cast<const S *>(p.parts) + m * ld + n;
  S4 sum = *reinterpret_cast<const S4 *>(part);
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) sum += *reinterpret_cast<const S4 *>(part + s * (p.m * ld));
  float v[4], bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(sum[i]);
  if (p.sa) {
    typedef typename std::conditional<std::is_same<S, int>::value, i8, f8>::type T;
    float sb[4];
    load_some(p.sb + n, p.n - n, sb);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = scaled<T>(sum[i], p.sa[m], sb[i]);
  }
  load_bias<O>(p, n, bias);
  finish<O, ACT>(p, m, n, v, bias);
}
template <typename S, typename O, int ACT>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmParams p) {
  join_four<S, O, ACT>(p, blockIdx.x);
}
template <typename O>
__global__ __launch_bounds__(256) void gemm_join_pair_kernel(GemmParams dx, GemmParams dw, unsigned first) {
  const unsigned block = blockIdx.x;
  if (block < first) join_four<float, O, ACT_NONE>(dx, block);
  else join_four<float, O, ACT_NONE>(dw, block - first);
}

unsigned join_blocks(const GemmParams &p) { return static_cast<unsigned>((p.m * ((p.n + 3L) / 4) + 255) / 256); }

template <typename S, typename O>
void join(const GemmParams &p, hipStream_t stream) {
  const dim3 grid(join_blocks(p));
  if (p.act == ACT_RELU) gemm_join_kernel<S, O, ACT_RELU><<<grid, 256, 0, stream>>>(p);
  else if (p.act == ACT_GELU) gemm_join_kernel<S, O, ACT_GELU><<<grid, 256, 0, stream>>>(p);
  else if (p.act == ACT_SILU) gemm_join_kernel<S, O, ACT_SILU><<<grid, 256, 0, stream>>>(p);
  else gemm_join_kernel<S, O, ACT_NONE><<<grid, 256, 0, stream>>>(p);
}

// Copies to aligned lines, 16 bytes a thread.  Bound by memory: 7168 x 2107 and 8063 x 2107
// bfloat16 23 us (64 MB read and written, 5.6 TB/s).
// KEPT: some of it may be kept in 8 bits.
template <typename T, bool KEPT = false>
__device__ __forceinline__ void pack_piece(const PackParams &p, long block) {
  constexpr int N = kPiece<T>;
  long id = block * 256 + threadIdx.x;
  const int q = id >= p.pieces[0];
  if (q) id -= p.pieces[0];
  if (id >= p.pieces[q]) return;
  const long per = p.to_ld[q] / N, row = id / per;
  const int c = static_cast<int>(id % per) * N;
  if constexpr (KEPT) {
    if (p.kept[q]) {
      float u[8];
      load_kept8<T>(kept_at(p.from[q], p.rows[q], p.columns[q]), row, c, u);
      typename Vec<T, 8>::type w;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = kept_as<T>(u[i]);
      *reinterpret_cast<typename Vec<T, 8>::type *>(static_cast<T *>(p.to[q]) + row * p.to_ld[q] + c) = w;
      return;
    }
  }
  const i32x4 v = load_piece_any(static_cast<const T *>(p.from[q]) + row * p.from_ld[q], c, p.columns[q]);
  *reinterpret_cast<i32x4 *>(static_cast<T *>(p.to[q]) + row * p.to_ld[q] + c) = v;
}
template <typename T, bool KEPT>
__global__ __launch_bounds__(256) void pack_kernel(PackParams p) {
  pack_piece<T, KEPT>(p, block_of());
}
long pack_blocks(const PackParams &p) { return (p.pieces[0] + p.pieces[1] + 255) / 256; }

// Without a branch, also where columns end inside a piece: 4096 x 8191 bfloat16 gelu 49 us
// against 80 with one (4096 x 8192 44 either way).
template <typename T>
__device__ __forceinline__ void load_slope8(const T *row, int c, int n, float (&v)[8]) {
  const auto u = __builtin_bit_cast(typename Vec<T, 8>::type, load_piece_any(row, c, n));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(u[i]);
}

template <typename T>
constexpr float largest = __is_same(T, f16) ? 65504.0f : 0x1.fep127f;  // finite

// 8 columns a thread; CT threads side by side, the others down the workgroup's rows.
// The workgroups from `blocks` on make copies.  Bound by memory with arithmetic close
// behind (gelu's slope is some 50 instructions an element): 4096 x 8192 bfloat16 gelu 44 us
// with the sums (201 MB, 4.6 TB/s).  Workgroups of 32 rows where 64 leave CUs idle: 4736 x
// 141 float16 19.6 us with 64, 8.8 with 32; of all up to 256 rows where that saves the sum's launch.
// KEPT: z may be kept in 8 bits, and a copy restored from 8 bits: 4096 x 8192 gelu with 4096 x 2048 of x restored
// 42 to 49 us.
template <typename T, int ACT, int CT, bool KEPT>
__global__ __launch_bounds__(256) void act_slope_kernel(SlopeParams p, PackParams pack, int blocks) {
  const long block = block_of();
  if (block >= blocks) {
    pack_piece<T, KEPT>(pack, block - blocks);
    return;
  }
  const Kept kept = kept_at(p.z, p.m, p.n);
  constexpr int LANES = 256 / CT, COLS = CT * 8;
  const int column_blocks = (p.n + COLS - 1) / COLS, bc = static_cast<int>(block) % column_blocks, br = static_cast<int>(block) / column_blocks;
  const int c = bc * COLS + threadIdx.x % CT * 8, lane = threadIdx.x / CT, left = p.n - c, rows = p.rows;
  const long row0 = static_cast<long>(br) * rows;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
  if (left > 0) {
    const int end = static_cast<int>(min(static_cast<long>(rows), p.m - row0));
#pragma unroll 4
    for (int r = lane; r < end; r += LANES) {
      const long row = row0 + r;
      float g[8], z[8];
      load_slope8(static_cast<const T *>(p.dy) + row * p.dy_ld, c, p.n, g);
      if constexpr (ACT != ACT_NONE) {
        if (KEPT && p.kept) load_kept8<T>(kept, row, c, z);
        else load_slope8(static_cast<const T *>(p.z) + row * p.z_ld, c, p.n, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= act_slope<ACT>(z[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += g[i];
      if (p.dz) {
        typename Vec<T, 8>::type hi, lo;
        T *to = static_cast<T *>(p.dz) + row * p.dz_ld + c;
        if (p.lo) {
          // Two terms.  An infinity has no second one (it would be a NaN); a finite value past
          // the type's largest is that and the rest, which the products' float sums hold.
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool finite = __builtin_fabsf(g[i]) < __builtin_inff();
            hi[i] = static_cast<T>(i < left ? (finite ? __builtin_fminf(__builtin_fmaxf(g[i], -largest<T>), largest<T>) : g[i]) : 0.0f);
            lo[i] = static_cast<T>(i < left && finite ? g[i] - static_cast<float>(hi[i]) : 0.0f);
          }
          *reinterpret_cast<typename Vec<T, 8>::type *>(to + p.lo) = lo;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) hi[i] = i < left ? static_cast<T>(g[i]) : static_cast<T>(0.0f);
        }
        *reinterpret_cast<typename Vec<T, 8>::type *>(to) = hi;
      }
    }
  }
  if (!p.shares && !p.sums) return;
  __shared__ float part[LANES][8][CT + 1];
#pragma unroll
  for (int i = 0; i < 8; ++i) part[lane][i][threadIdx.x % CT] = sum[i];
  __syncthreads();
  const int e = threadIdx.x % COLS, at = bc * COLS + e;
  if (threadIdx.x >= COLS) return;
  float v = 0.0f;
#pragma unroll
  for (int q = 0; q < LANES; ++q) v += part[q][e % 8][e / 8];
  if (at >= p.n) return;
  if (p.sums) store_as(p.sums, p.sums_type, at, v);
  else p.shares[static_cast<long>(br) * p.n + at] = v;
}

template <typename T, int ACT, bool KEPT>
void slope(const SlopeParams &p, const PackParams &pack, hipStream_t stream) {
  const int columns = p.rows == SLOPE_WHOLE ? 32 : p.rows == SLOPE_FEW ? 128 : 256;
  const int blocks = (p.m + p.rows - 1) / p.rows * ((p.n + columns - 1) / columns);
  const dim3 grid = grid_of(blocks + pack_blocks(pack), 256);
  if (p.rows == SLOPE_WHOLE) act_slope_kernel<T, ACT, 4, KEPT><<<grid, 256, 0, stream>>>(p, pack, blocks);
  else if (p.rows == SLOPE_FEW) act_slope_kernel<T, ACT, 16, KEPT><<<grid, 256, 0, stream>>>(p, pack, blocks);
  else act_slope_kernel<T, ACT, 32, KEPT><<<grid, 256, 0, stream>>>(p, pack, blocks);
}

template <typename T, bool KEPT>
void slope(const SlopeParams &p, const PackParams &pack, hipStream_t stream) {
  if (p.act == ACT_RELU) slope<T, ACT_RELU, KEPT>(p, pack, stream);
  else if (p.act == ACT_GELU) slope<T, ACT_GELU, KEPT>(p, pack, stream);
  else if (p.act == ACT_SILU) slope<T, ACT_SILU, KEPT>(p, pack, stream);
  else slope<T, ACT_NONE, KEPT>(p, pack, stream);
}
bool some_kept(const PackParams &p) { return p.kept[0] || p.kept[1]; }
template <typename T>
void slope(const SlopeParams &p, const PackParams &pack, hipStream_t stream) {
  p.kept || some_kept(pack) ? slope<T, true>(p, pack, stream) : slope<T, false>(p, pack, stream);
}

}  // namespace

hipError_t launch_pack(const PackParams &p, int type, hipStream_t stream) {
  const dim3 grid = grid_of(pack_blocks(p), 256);
  if (some_kept(p)) type == TYPE_BF16 ? pack_kernel<bf16, true><<<grid, 256, 0, stream>>>(p) : pack_kernel<f16, true><<<grid, 256, 0, stream>>>(p);
  else if (type == TYPE_F8 || type == TYPE_I8) pack_kernel<f8, false><<<grid, 256, 0, stream>>>(p);
  else pack_kernel<bf16, false><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

hipError_t launch_gemm_join(const GemmParams &p, int type, int out_type, hipStream_t stream) {
  if (type == TYPE_I8) out_type == TYPE_BF16 ? join<int, bf16>(p, stream) : join<int, f16>(p, stream);
  else out_type == TYPE_BF16 ? join<float, bf16>(p, stream) : join<float, f16>(p, stream);
  return hipGetLastError();
}

hipError_t launch_gemm_join_pair(const GemmParams &dx, const GemmParams &dw, int out_type, hipStream_t stream) {
  const unsigned first = dx.splits > 1 ? join_blocks(dx) : 0;
  const dim3 grid(first + (dw.splits > 1 ? join_blocks(dw) : 0));
  if (out_type == TYPE_BF16) gemm_join_pair_kernel<bf16><<<grid, 256, 0, stream>>>(dx, dw, first);
  else gemm_join_pair_kernel<f16><<<grid, 256, 0, stream>>>(dx, dw, first);
  return hipGetLastError();
}

hipError_t launch_act_slope(const SlopeParams &p, const PackParams &pack, int type, hipStream_t stream) {
  type == TYPE_BF16 ? slope<bf16>(p, pack, stream) : slope<f16>(p, pack, stream);
  return hipGetLastError();
}

}  // namespace tfnn
