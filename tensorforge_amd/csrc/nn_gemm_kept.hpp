// The products whose pre-activation is kept in 8 bits (nn_common.hpp's groups) as they write it: the
// direct tiles, unsplit.  Bound as the products themselves, with two bytes an element less to write
// than in 16 bits, and no pass over it afterwards.
#pragma once

#include "nn_gemm.hpp"
#include "nn_wide.hpp"

namespace tfnn {

// out = act(z) + residual, and the codes of z rounded to T (as keep8 of a kept z, masked, would give them).  A
// group's columns are four lanes' of the patch: tiles start at multiples of 32.
struct KeptResults {
  typedef KeptGemmParams Params;
  template <typename T, int BM, int BN, int WM, int WN, int ROWS, int MI, int NI>
  static __device__ __forceinline__ void finish(const KeptGemmParams &p, f32x4 (&acc)[MI][NI], int, lds_char *, lds_char *patch, int m0, int n0,
                                                int wm, int wn, int, int) {
    const int mw = m0 + wm * (BM / WM), n = n0 + wn * (BN / WN) + threadIdx.x % (NI * 2) * 8, left = p.n - n;
    const long length = p.groups * kGroup;
    float bias[8];
    load_bias<T>(p, n, bias);
    with_act(p.act, [&](auto act) {
      by_rows<ROWS>(acc, patch, [&](int row, int, float (&v)[8]) {
        const int m = mw + row;
        if (m >= p.m) return;  // the four lanes of a group together
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] += bias[i];
          z[i] = i < left ? static_cast<float>(static_cast<T>(v[i])) : 0.0f;
        }
        uint32_t exponent;
        const u32x2 codes = group_codes<true>(z, act() == ACT_RELU, exponent);
        if (n < length) {
          *reinterpret_cast<u32x2 *>(p.codes + m * length + n) = codes;
          if (n % kGroup == 0) p.exponents[m * p.groups + n / kGroup] = static_cast<uint8_t>(exponent);
        }
        if (left <= 0) return;
        float res[8];
        if (p.residual) load_some(static_cast<const T *>(p.residual) + m * p.ldr + n, left, res);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_value<act()>(v[i]);
        if (p.residual) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += res[i];
        }
        store_some<BM == 256>(static_cast<T *>(p.out) + m * p.ldo + n, left, v);
      });
    });
  }
};

template <typename T, bool BMN, int BM, int BN, int ST>
__global__ __launch_bounds__(256) void gemm_kept_kernel(KeptGemmParams p) {
  __shared__ __align__(1024) char smem[tile_lds<BM, BN, ST>()];
  gemm_tile<T, T, false, BMN, BM, BN, 2, 2, ST, true, 1, KeptResults>(p, blockIdx.x, gridDim.x, (lds_char *)smem);
}
template <typename T, bool BMN>
__global__ __launch_bounds__(512, 2) void gemm_kept_wide_kernel(KeptGemmParams p) {
  __shared__ __align__(1024) char smem[kWideLds];
  gemm_wide<T, T, false, BMN, KeptResults>(p, (lds_char *)smem);
}

template <typename T, bool BMN>
hipError_t launch_kept_as(const KeptGemmParams &p, int tile, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.tiles_m) * p.tiles_n);
  if (tile == TILE_256) gemm_kept_wide_kernel<T, BMN><<<grid, 512, 0, stream>>>(p);
  else if (tile == TILE_128) gemm_kept_kernel<T, BMN, 128, 128, 2><<<grid, 256, 0, stream>>>(p);
  else if (tile == TILE_64x128) gemm_kept_kernel<T, BMN, 64, 128, 3><<<grid, 256, 0, stream>>>(p);
  else if (grid.x <= 768) gemm_kept_kernel<T, BMN, 64, 64, 3><<<grid, 256, 0, stream>>>(p);  // as launch_tile
  else gemm_kept_kernel<T, BMN, 64, 64, 2><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace tfnn
