// The products of the loss over a vocabulary: nn_gemm.hpp's and nn_wide.hpp's tiles with
// epilogues of their own.  The logits stay in the accumulators; what leaves a tile is two floats a
// row (the loss), or the logits' gradient in 16 bits (for one piece of the vocabulary).
#pragma once

#include "nn_gemm.hpp"
#include "nn_wide.hpp"

namespace tfnn {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// A lane holds of each 16 x 16 block the row lane % 16 and four columns from lane / 16 * 4.

// Logarithms of sums are kept as pairs: t, and the sum of exp2(value * log2(e) - t).  t is the
// largest value times log2(e), rounded: whatever it was rounded to, the pair stands for the sum.
// -inf: no value yet.
__device__ __forceinline__ float from_of(float t) { return t == -__builtin_inff() ? 0.0f : t; }
__device__ __forceinline__ f32x2 joined(f32x2 a, f32x2 b) {
  const float t = __builtin_fmaxf(a.x, b.x), from = from_of(t);
  return f32x2{t, a.y * fast_exp2(a.x - from) + b.y * fast_exp2(b.x - from)};
}

// Each row's pair over the tile's columns: a lane's own columns, the four lanes of a row, the
// waves side by side in LDS.  Bound by the product, whose tile ends with this: 8192 x 65536 x 2048 bfloat16
// 1.60 to 1.75 ms (1.26 to 1.38 PFLOP/s, the library's product 1.57), a round of 256 tiles 50 us of which some
// 4 are these exponentials; 16 x 32000 x 4096 44.7 us, w's bytes at 5.9 TB/s.
struct Stats {
  typedef XentParams Params;
  template <typename T, int BM, int BN, int WM, int WN, int ROWS, int MI, int NI>
  static __device__ __forceinline__ void finish(const XentParams &p, f32x4 (&acc)[MI][NI], int, lds_char *lds, lds_char *, int m0, int n0,
                                                int wm, int wn, int tm, int tn) {
    const int lane = threadIdx.x % 64, l = lane % 16, g = lane / 16, nw = n0 + wn * (BN / WN), nt = tn * BN;
    auto *slots = reinterpret_cast<__attribute__((address_space(3))) f32x2 *>(lds);
    const bool whole = nw >= nt && nw + NI * 16 <= p.n;
    // The targets, all under way at once.
    long long target[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) target[i] = p.target[min(m0 + wm * (BM / WM) + i * 16 + l, p.m - 1)];
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int in_tile = wm * (BM / WM) + i * 16 + l, m = m0 + in_tile;
      // The target's logit, by the one lane that holds it.
      if (target[i] >= max(nw, nt) && target[i] < min(nw + NI * 16, p.n) && static_cast<int>(target[i] - nw) / 4 % 4 == g && m < p.m &&
          m >= tm * BM) {
        const int t = static_cast<int>(target[i] - nw);
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t / 16 == j && t % 4 == e) v = acc[i][j][e];
        p.target_logit[m] = v;
      }
      if (!whole) {  // columns of another tile, or of none
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = nw + j * 16 + g * 4 + e;
            if (n < nt || n >= p.n) acc[i][j][e] = -__builtin_inff();
          }
      }
      float top = acc[i][0][0], sum = 0.0f;
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __builtin_fmaxf(top, acc[i][j][e]);
      top = __builtin_fmaxf(top, __shfl_xor(top, 16));
      top = __builtin_fmaxf(top, __shfl_xor(top, 32)) * kLog2e;
      const float from = from_of(top);  // a NaN is in the sum
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += fast_exp2(__builtin_fmaf(acc[i][j][e], kLog2e, -from));
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (g == 0) slots[wn * BM + in_tile] = f32x2{top, sum};
    }
    wait_lds();
    barrier();
    for (int r = threadIdx.x; r < BM; r += 64 * WM * WN) {
      const int m = m0 + r;
      if (m >= p.m || m < tm * BM) continue;
      f32x2 s = slots[r];
#pragma unroll
      for (int w = 1; w < WN; ++w) s = joined(s, slots[w * BM + r]);
      reinterpret_cast<f32x2 *>(p.stats)[static_cast<long>(tn) * p.m + m] = s;
    }
  }
};

// What a finished sum of the gradient's products is multiplied by.
__device__ __forceinline__ float sum_unit(const XentParams &p) {
  if (p.dloss_rows) return p.scale ? p.scale[1] : 1.0f;
  return *p.dloss / (p.count && *p.count > 0.0f ? *p.count : 1.0f) / p.power;
}
// Zeros stay (rows that do not count, where dloss is no number).
__device__ __forceinline__ float in_unit(float v, float unit) { return v == 0.0f ? 0.0f : v * unit; }

// The logits' gradient, in T: without dloss where that is one for all.  The target's -(1 - p), most of it,
// then lies where T's spacing is least against it, and is exact while p is small.  8192 x 65536 x 2048 bfloat16:
// dx and dw 0.0025 off 64 bits with dloss in it, 0.0017 without (their own rounding).
struct Slope {
  typedef XentParams Params;
  template <typename T, int BM, int BN, int WM, int WN, int ROWS, int MI, int NI>
  static __device__ __forceinline__ void finish(const XentParams &p, f32x4 (&acc)[MI][NI], int, lds_char *, lds_char *patch, int m0, int n0,
                                                int wm, int wn, int tm, int tn) {
    const int lane = threadIdx.x % 64, l = lane % 16, g = lane / 16, mw = m0 + wm * (BM / WM), nw = n0 + wn * (BN / WN);
    const float unit = p.dloss_rows ? (p.scale ? p.scale[0] : 1.0f) / (p.count ? *p.count : 1.0f) : p.power;
    const bool whole = nw + NI * 16 <= p.n;
    // What the rows need, all under way at once.  Rows past the last are not written.
    long long target[MI];
    float lse[MI], rest[MI], d[MI];  // lse * log2(e) in two floats: large logits keep what their differences are worth
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = min(mw + i * 16 + l, p.m - 1);
      target[i] = p.target[m];
      const double scaled = p.lse[m] * kLog2e;
      lse[i] = static_cast<float>(scaled);
      rest[i] = __builtin_fabsf(lse[i]) < __builtin_inff() ? static_cast<float>(scaled - lse[i]) : 0.0f;
      d[i] = p.dloss_rows ? p.dloss[m] * unit : unit;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const bool dead = target[i] == p.ignore, valid = target[i] >= 0 && target[i] < p.vocabulary;
      if (!valid) d[i] = __builtin_nanf("");
      const long long from = valid ? target[i] - p.column0 - nw : -1;
      const int t = static_cast<int>(from);
      const bool here = from >= 0 && from < NI * 16 && t / 4 % 4 == g;
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fast_exp2(__builtin_fmaf(acc[i][j][e], kLog2e, -lse[i]) - rest[i]) * d[i];
      if (here) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t / 16 == j && t % 4 == e) acc[i][j][e] -= d[i];
      }
      if (dead) {
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      if (!whole) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (nw + j * 16 + g * 4 + e >= p.n) acc[i][j][e] = 0.0f;
      }
    }
    const int end = (p.n + 7) & ~7;  // the next product reads whole pieces
    T *out = static_cast<T *>(p.out);
    by_rows<ROWS>(acc, patch, [&](int row, int column, const float (&v)[8]) {
      const int m = mw + row, n = nw + column;
      if (m >= p.m || m < tm * BM || n >= p.n || n + 7 < tn * BN) return;
      T *to = out + m * p.ldo;
      store_some(to + n, end - n, v);
      for (int c = n + 8; n + 8 >= p.n && c < end; ++c) to[c] = static_cast<T>(0.0f);  // a tile moved back ends with n
      if (p.lo) {
        float left[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          left[i] = v[i] - static_cast<float>(static_cast<T>(v[i]));
          if (!(__builtin_fabsf(left[i]) < __builtin_inff())) left[i] = 0.0f;
        }
        to += p.lo;
        store_some(to + n, end - n, left);
        for (int c = n + 8; n + 8 >= p.n && c < end; ++c) to[c] = static_cast<T>(0.0f);
      }
    });
  }
};

// A product added to what earlier pieces left.  Of 8192 rows and classes and k of 2048, bfloat16: dx 212 us (134 MB
// of sums read and written in one round's end), dw 205.
struct Sum {
  typedef XentParams Params;
  template <typename T, int BM, int BN, int WM, int WN, int ROWS, int MI, int NI>
  static __device__ __forceinline__ void finish(const XentParams &p, f32x4 (&acc)[MI][NI], int split, lds_char *, lds_char *patch, int m0,
                                                int n0, int wm, int wn, int tm, int tn) {
    const int mw = m0 + wm * (BM / WM), nw = n0 + wn * (BN / WN), nt = tn * BN;
    const long ld = (p.n + 3) & ~3;
    float *part = p.parts + split * (p.m * ld);
    const float unit = sum_unit(p);
    by_rows<ROWS>(acc, patch, [&](int row, int column, float (&v)[8]) {
      const int m = mw + row, n = nw + column, left = p.n - n;
      if (m >= p.m || m < tm * BM || left <= 0 || n + 7 < nt) return;
      if (p.splits > 1 || p.halves) {
        store_some(part + m * ld + n, left, v);
        return;
      }
      if (p.add) {
        float u[8];
        load_some(p.sum + m * ld + n, left, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += u[i];
      }
      if (p.last) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = in_unit(v[i], unit);
        store_some(static_cast<T *>(p.out) + m * p.ldo + n, left, v);
      } else if (n >= nt) {
        store_some(p.sum + m * ld + n, left, v);
      } else {  // a tile moved back: the columns before its own are another's sum
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left && n + i >= nt) p.sum[m * ld + n + i] = v[i];
      }
    });
  }
};

template <typename T, typename E, bool AMN, bool BMN, int BM, int ST, bool DMA>
__global__ __launch_bounds__(256, DMA ? 1 : 3) void xent_tile_kernel(XentParams p) {
  __shared__ __align__(1024) char smem[tile_lds<BM, BM, ST>()];
  const int block = static_cast<int>(block_of()), blocks = p.tiles_m * p.tiles_n * p.splits;
  if (block < blocks) gemm_tile<T, T, AMN, BMN, BM, BM, 2, 2, ST, DMA, 1, E>(p, block, blocks, (lds_char *)smem);
}
template <typename T, typename E, bool AMN, bool BMN>
__global__ __launch_bounds__(512, 2) void xent_wide_kernel(XentParams p) {
  __shared__ __align__(1024) char smem[kWideLds];
  gemm_wide<T, T, AMN, BMN, E>(p, (lds_char *)smem);
}

template <typename T, typename E, bool AMN, bool BMN>
hipError_t launch_xent_as(const XentParams &p, int tile, bool dma, hipStream_t stream) {
  const long blocks = static_cast<long>(p.tiles_m) * p.tiles_n * p.splits;
  const dim3 grid = grid_of(blocks, 256);
  if (!dma) xent_tile_kernel<T, E, AMN, BMN, 64, 2, false><<<grid, 256, 0, stream>>>(p);
  else if (tile == TILE_256) xent_wide_kernel<T, E, AMN, BMN><<<dim3(static_cast<unsigned>(blocks)), 512, 0, stream>>>(p);
  else if (tile == TILE_128) xent_tile_kernel<T, E, AMN, BMN, 128, 2, true><<<grid, 256, 0, stream>>>(p);
  else xent_tile_kernel<T, E, AMN, BMN, 64, 3, true><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_xent(const XentParams &p, XentProduct what, bool amn, bool bmn, int tile, bool dma, hipStream_t stream) {
  if (what == XENT_STATS) return bmn ? launch_xent_as<T, Stats, false, true>(p, tile, dma, stream) : launch_xent_as<T, Stats, false, false>(p, tile, dma, stream);
  if (what == XENT_SLOPE) return bmn ? launch_xent_as<T, Slope, false, true>(p, tile, dma, stream) : launch_xent_as<T, Slope, false, false>(p, tile, dma, stream);
  if (amn) return launch_xent_as<T, Sum, true, true>(p, tile, dma, stream);
  return bmn ? launch_xent_as<T, Sum, false, true>(p, tile, dma, stream) : launch_xent_as<T, Sum, false, false>(p, tile, dma, stream);
}

}  // namespace tfnn
