// What the products need beside the matrix kernels: the join of a product split
// along k, and the activation's slope with the bias gradient's sums.
#include "nn_gemm.hpp"

#include <algorithm>

namespace tfnn {
namespace {

// Four columns a thread: the parts' sum in order, then the tile kernels' epilogue.
template <typename O, int ACT>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmParams p) {
  const long ld = (p.n + 3) & ~3, id = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  const int m = static_cast<int>(id / (ld / 4)), n = static_cast<int>(id % (ld / 4)) * 4;
  if (m >= p.m) return;
  const float *part = p.parts + m * ld + n;
  f32x4 sum = *reinterpret_cast<const f32x4 *>(part);
  for (int s = 1; s < p.splits; ++s) sum += *reinterpret_cast<const f32x4 *>(part + s * (p.m * ld));
  float v[4] = {sum.x, sum.y, sum.z, sum.w}, bias[4];
  if (p.sa) {
    float sb[4];
    load_some(p.sb + n, p.n - n, sb);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] * p.sa[m] * sb[i];
  }
  load_bias<O>(p, n, bias);
  finish<O, ACT>(p, m, n, v, bias);
}

template <typename O>
void join(const GemmParams &p, hipStream_t stream) {
  const long threads = static_cast<long>(p.m) * ((p.n + 3) / 4);
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
  if (p.act == ACT_RELU) gemm_join_kernel<O, ACT_RELU><<<grid, 256, 0, stream>>>(p);
  else if (p.act == ACT_GELU) gemm_join_kernel<O, ACT_GELU><<<grid, 256, 0, stream>>>(p);
  else if (p.act == ACT_SILU) gemm_join_kernel<O, ACT_SILU><<<grid, 256, 0, stream>>>(p);
  else gemm_join_kernel<O, ACT_NONE><<<grid, 256, 0, stream>>>(p);
}

constexpr int kSlopeRows = 64;

// 256 columns x 64 rows a workgroup: 32 threads of 8 columns by 8 rows.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_slope_kernel(SlopeParams p) {
  const int column_blocks = (p.n + 255) / 256, bc = blockIdx.x % column_blocks, br = blockIdx.x / column_blocks;
  const int c = (bc * 32 + threadIdx.x % 32) * 8, lane = threadIdx.x / 32;
  const long row0 = static_cast<long>(br) * kSlopeRows;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
  const int left = p.n - c;
  if (left > 0) {
    for (int r = lane; r < kSlopeRows && row0 + r < p.m; r += 8) {
      const long row = row0 + r;
      float g[8], z[8];
      load_some(static_cast<const T *>(p.dy) + row * p.dy_ld + c, left, g);
      if constexpr (ACT != ACT_NONE) {
        load_some(static_cast<const T *>(p.z) + row * p.z_ld + c, left, z);
        typename Vec<T, 8>::type out;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = g[i] * act_slope<ACT>(z[i]);
          sum[i] += v;
          out[i] = i < left ? static_cast<T>(v) : static_cast<T>(0.0f);
        }
        *reinterpret_cast<typename Vec<T, 8>::type *>(static_cast<T *>(p.dz) + row * p.dz_ld + c) = out;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += g[i];
      }
    }
  }
  if (!p.shares) return;
  __shared__ float part[8][8][33];
#pragma unroll
  for (int i = 0; i < 8; ++i) part[lane][i][threadIdx.x % 32] = sum[i];
  __syncthreads();
  const int i = threadIdx.x % 8, col = threadIdx.x / 8, at = (bc * 32 + col) * 8 + i;
  float v = 0.0f;
#pragma unroll
  for (int q = 0; q < 8; ++q) v += part[q][i][col];
  if (at < p.n) p.shares[static_cast<long>(br) * p.n + at] = v;
}

template <typename T>
void slope(const SlopeParams &p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(column_shares(p.m) * ((p.n + 255) / 256)));
  if (p.act == ACT_RELU) act_slope_kernel<T, ACT_RELU><<<grid, 256, 0, stream>>>(p);
  else if (p.act == ACT_GELU) act_slope_kernel<T, ACT_GELU><<<grid, 256, 0, stream>>>(p);
  else if (p.act == ACT_SILU) act_slope_kernel<T, ACT_SILU><<<grid, 256, 0, stream>>>(p);
  else act_slope_kernel<T, ACT_NONE><<<grid, 256, 0, stream>>>(p);
}

}  // namespace

long column_shares(long m) { return (m + kSlopeRows - 1) / kSlopeRows; }

hipError_t launch_gemm_join(const GemmParams &p, int out_type, hipStream_t stream) {
  out_type == TYPE_BF16 ? join<bf16>(p, stream) : join<f16>(p, stream);
  return hipGetLastError();
}

hipError_t launch_act_slope(const SlopeParams &p, int type, hipStream_t stream) {
  type == TYPE_BF16 ? slope<bf16>(p, stream) : slope<f16>(p, stream);
  return hipGetLastError();
}

}  // namespace tfnn
