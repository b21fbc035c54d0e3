// Activations into 8 bits (nn_common.hpp's groups of 32) and back.
//
// Bound by memory: a thread takes 8 elements, four threads a group, whose largest
// magnitude they find by two exchanges; kUnroll pieces a thread under way together.
// 8192 x 8192 bfloat16 38 us there (5.3 TB/s) and 30 back (6.7), 70 for both in turn.
#include "nn_common.hpp"

#include <algorithm>

namespace tfnn {
namespace {

constexpr int kUnroll = 4;

// Piece `id` of 8 elements: its row and its first element there.  FLAT: the rows follow each
// other without gaps, whole groups each, and are one.
template <bool FLAT>
struct Place {
  long row;
  int c;
  __device__ __forceinline__ Place(long id, long pieces) {
    if constexpr (FLAT) row = 0, c = 0;
    else if (id >> 32) row = id / pieces, c = static_cast<int>(id - row * pieces) * 8;
    else {
      const uint32_t r = static_cast<uint32_t>(id) / static_cast<uint32_t>(pieces);
      row = r, c = static_cast<int>(static_cast<uint32_t>(id) - r * static_cast<uint32_t>(pieces)) * 8;
    }
  }
};

template <typename T, bool FLAT, bool MASKED>
__global__ __launch_bounds__(256) void keep_kernel(const T *x, long ld, int d, long all, long pieces, bool positive, uint8_t *codes,
                                                   uint8_t *exponents) {
  constexpr int N = 16 / sizeof(T);
  const long first = block_of() * (256 * kUnroll) + threadIdx.x;
  float v[kUnroll][8];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long id = min(first + u * 256, all - 1);  // all is a multiple of four: the quads repeat whole
    const Place<FLAT> at(id, pieces);
#pragma unroll
    for (int q = 0; q < 8 / N; ++q) {
      i32x4 raw;
      if constexpr (FLAT) raw = *reinterpret_cast<const loose16 *>(x + id * 8 + q * N);
      else raw = load_piece_any(x + at.row * ld, at.c + q * N, d);
      const auto e = __builtin_bit_cast(typename Vec<T, N>::type, raw);
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][q * N + i] = static_cast<float>(e[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long id = first + u * 256;
    uint32_t e;
    const u32x2 c = group_codes<MASKED>(v[u], positive, e);
    if (id >= all) continue;
    *reinterpret_cast<u32x2 *>(codes + id * 8) = c;
    if (threadIdx.x % 4 == 0) exponents[id / 4] = static_cast<uint8_t>(e);
  }
}

template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void restore_kernel(T *x, long ld, int d, long all, long pieces, const uint8_t *codes,
                                                      const uint8_t *exponents) {
  const long first = block_of() * (256 * kUnroll) + threadIdx.x;
  u32x2 c[kUnroll];
  uint32_t e[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long id = min(first + u * 256, all - 1);
    c[u] = *reinterpret_cast<const u32x2 *>(codes + id * 8);
    e[u] = exponents[id / 4];
  }
  float v[kUnroll][8];
  bool masked = false;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) masked |= restore_codes<T>(c[u], e[u], v[u]);
  if (masked) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) restore_masked(c[u], v[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long id = first + u * 256;
    if (id >= all) continue;
    const Place<FLAT> at(id, pieces);
    T *to = FLAT ? x + id * 8 : x + at.row * ld + at.c;
    typename Vec<T, 8>::loose w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = kept_as<T>(v[u][i]);
    const int left = FLAT ? 8 : d - at.c;
    if (left >= 8) {
      *reinterpret_cast<typename Vec<T, 8>::loose *>(to) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) to[i] = w[i];
    }
  }
}

struct Sizes {
  long pieces, all;  // of a row, of all
  bool flat;
  dim3 grid;
};
Sizes sizes_of(long ld, long rows, long d) {
  const long pieces = (d + kGroup - 1) / kGroup * 4, all = rows * pieces;
  return {pieces, all, d % kGroup == 0 && (ld == d || rows == 1), grid_of((all + 256 * kUnroll - 1) / (256 * kUnroll), 256)};
}

template <typename T, bool MASKED>
void keep(const void *x, long ld, long rows, int d, bool positive, const Kept &to, hipStream_t stream) {
  const Sizes s = sizes_of(ld, rows, d);
  const T *from = static_cast<const T *>(x);
  uint8_t *codes = const_cast<uint8_t *>(to.codes), *exponents = const_cast<uint8_t *>(to.exponents);
  if (s.flat) keep_kernel<T, true, MASKED><<<s.grid, 256, 0, stream>>>(from, ld, d, s.all, s.pieces, positive, codes, exponents);
  else keep_kernel<T, false, MASKED><<<s.grid, 256, 0, stream>>>(from, ld, d, s.all, s.pieces, positive, codes, exponents);
}

template <typename T>
void keep(const void *x, long ld, long rows, int d, bool positive, bool masked, const Kept &to, hipStream_t stream) {
  masked ? keep<T, true>(x, ld, rows, d, positive, to, stream) : keep<T, false>(x, ld, rows, d, positive, to, stream);
}

template <typename T>
void restore(const Kept &from, long rows, int d, void *x, long ld, hipStream_t stream) {
  const Sizes s = sizes_of(ld, rows, d);
  T *to = static_cast<T *>(x);
  if (s.flat) restore_kernel<T, true><<<s.grid, 256, 0, stream>>>(to, ld, d, s.all, s.pieces, from.codes, from.exponents);
  else restore_kernel<T, false><<<s.grid, 256, 0, stream>>>(to, ld, d, s.all, s.pieces, from.codes, from.exponents);
}

}  // namespace

hipError_t launch_keep(const void *x, long ld, long rows, int d, int type, bool positive, bool masked, void *kept, hipStream_t stream) {
  const Kept to = kept_at(kept, rows, d);
  if (type == TYPE_F32) keep<float>(x, ld, rows, d, positive, masked, to, stream);
  else if (type == TYPE_BF16) keep<bf16>(x, ld, rows, d, positive, masked, to, stream);
  else keep<f16>(x, ld, rows, d, positive, masked, to, stream);
  return hipGetLastError();
}

hipError_t launch_restore(const void *kept, long rows, int d, int type, void *x, long ld, hipStream_t stream) {
  const Kept from = kept_at(kept, rows, d);
  if (type == TYPE_F32) restore<float>(from, rows, d, x, ld, stream);
  else if (type == TYPE_BF16) restore<bf16>(from, rows, d, x, ld, stream);
  else restore<f16>(from, rows, d, x, ld, stream);
  return hipGetLastError();
}

}  // namespace tfnn
