// What the residual block's operators share: element types, rounding,
// activations and wave reductions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "nn_kernels.h"

namespace tfnn {

typedef __bf16 bf16;
typedef _Float16 f16;
struct f8 {  // OCP e4m3: largest value 448, no infinities
  uint8_t bits;
};
struct i8 {  // an 8-bit integer
  int8_t bits;
};

template <typename T, int N>
struct Vec {
  typedef T type __attribute__((ext_vector_type(N)));
  // The same at the element's own alignment.  One 128-bit access all the same:
  // global memory takes any byte address.
  typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// f(0), f(1), ... f(N-1), each with its number as a constant.
template <int I>
struct Int {
  __host__ __device__ constexpr operator int() const { return I; }
  __host__ __device__ constexpr int operator()() const { return I; }
};
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unroll(F &&f) {
  if constexpr (I < N) {
    f(Int<I>{});
    unroll<N, I + 1>(f);
  }
}

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// exp2 and 1/x in one instruction each (about 1 ulp).
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

constexpr float kLog2e = 1.44269504088896340736f;

// The normal distribution's upper tail q = P(Z > |x|), and e = exp(-x^2/2), which its density
// takes too.  q/e falls smoothly from 1/2 to 1/(|x| sqrt(2 pi)): as a polynomial of degree 7 in
// t = 1/(1 + 0.26 |x|), fitted for the least largest relative error over 0 <= |x| <= 14 (3.3e-7;
// 7e-7 with float's roundings, and exp's own).  Small tails are as exact as large ones: gelu
// of far negative values is nothing but the tail, and its values range over all of bfloat16's exponents.
__device__ __forceinline__ float normal_tail(float x, float &density_exp) {
  const float a = __builtin_fabsf(x);
  const float t = fast_rcp(__builtin_fmaf(0.26f, a, 1.0f));
  density_exp = fast_exp2(-0.5f * kLog2e * a * a);
  float p = __builtin_fmaf(-0.07714982330799103f, t, 0.24596595764160156f);
  p = __builtin_fmaf(p, t, -0.1348378211259842f);
  p = __builtin_fmaf(p, t, 0.19164182245731354f);
  p = __builtin_fmaf(p, t, 0.06050647050142288f);
  p = __builtin_fmaf(p, t, 0.1108865812420845f);
  p = __builtin_fmaf(p, t, 0.10295169055461884f);
  p = __builtin_fmaf(p, t, 3.4941571357194334e-05f);
  return p * density_exp;
}

// 1/(1 + exp(-x)).
__device__ __forceinline__ float sigmoid(float x) { return fast_rcp(1.0f + fast_exp2(-kLog2e * x)); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == ACT_RELU) return (z > 0.0f || z != z) ? z : 0.0f;  // NaN stays, -0 becomes +0
  if constexpr (ACT == ACT_GELU) {
    // z*Phi(z) = max(z, 0) - |z|*tail, which is exact where the tail is 0 (the
    // bound keeps infinity * 0 out) and stays NaN through the tail.
    float e;
    const float q = normal_tail(z, e);
    return __builtin_fmaf(-__builtin_fminf(__builtin_fabsf(z), 1e30f), q, __builtin_fmaxf(z, 0.0f));
  }
  if constexpr (ACT == ACT_SILU) return z == -__builtin_inff() ? -0.0f : z * sigmoid(z);
  return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
  if constexpr (ACT == ACT_GELU) {
    float e;
    const float q = normal_tail(z, e);
    const float v = __builtin_fmaf(z * 0.39894228040143267794f, e, z > 0.0f ? 1.0f - q : q);
    return __builtin_fabsf(z) == __builtin_inff() ? (z > 0.0f ? 1.0f : 0.0f) : v;
  }
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    const float v = __builtin_fmaf(z * s, 1.0f - s, s);
    return __builtin_fabsf(z) == __builtin_inff() ? (z > 0.0f ? 1.0f : 0.0f) : v;
  }
  return 1.0f;
}

typedef int loose16 __attribute__((ext_vector_type(4), aligned(1)));

// 16 bytes from element c >= 0 of a row of `length` elements (the same for all
// lanes), zeros past its end; nothing outside the row is touched, at any
// alignment.  WHOLE: length is a multiple of a piece, so a piece is inside or
// outside.  Otherwise length is at least a piece, and the row's last 16 bytes
// serve the pieces that reach past its end, shifted down.  Either way one load
// and no branch: the loads of many pieces can be under way together.
template <bool WHOLE, typename T>
__device__ __forceinline__ i32x4 load_piece(const T *row, int c, int length) {
  constexpr int N = 16 / sizeof(T), BITS = 8 * sizeof(T);
  const int at = min(c, length - N), past = c - at;
  const i32x4 v = *reinterpret_cast<const loose16 *>(row + at);
  if constexpr (WHOLE) {
    return past ? i32x4{0, 0, 0, 0} : v;
  } else {
    const auto u = __builtin_bit_cast(unsigned __int128, v) >> (min(past, N - 1) * BITS);
    return past >= N ? i32x4{0, 0, 0, 0} : __builtin_bit_cast(i32x4, u);
  }
}

// The same for any length, element by element where the row is shorter than a piece.
template <typename T>
__device__ __forceinline__ i32x4 load_piece_any(const T *row, int c, int length) {
  constexpr int N = 16 / sizeof(T);
  if (length >= N) return load_piece<false>(row, c, length);
  union {
    i32x4 v;
    T e[N];
  } u;
  u.v = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < N - 1; ++e)
    if (c + e < length) u.e[e] = row[c + e];
  return u.v;
}

// Rounds `v` to `type` at element `i` of `out`.
__device__ __forceinline__ void store_as(void *out, int type, long i, float v) {
  if (type == TYPE_F32) static_cast<float *>(out)[i] = v;
  else if (type == TYPE_BF16) static_cast<bf16 *>(out)[i] = static_cast<bf16>(v);
  else static_cast<f16 *>(out)[i] = static_cast<f16>(v);
}

// A launch takes fewer than 2^32 threads along a side: workgroups beyond 2^31 of them go
// along y.  The last row of workgroups may have some too many.
inline dim3 grid_of(long blocks, int threads) {
  const long most = (1L << 31) / threads;
  return blocks <= most ? dim3(static_cast<unsigned>(blocks)) : dim3(static_cast<unsigned>(most), static_cast<unsigned>((blocks + most - 1) / most));
}
__device__ __forceinline__ long block_of() { return blockIdx.x + static_cast<long>(blockIdx.y) * gridDim.x; }

// Sum / maximum over groups of 64 lanes; every lane gets the result.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// A NaN anywhere stays: fmaxf alone would drop it.
__device__ __forceinline__ float max_keep_nan(float a, float b) { return (a > b || a != a) ? a : b; }
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max_keep_nan(v, __shfl_xor(v, o));
  return v;
}

// The shares' sum, in order: 16 columns a workgroup of 256, 4 threads of four columns by
// 64 rows of shares.  Bound by latency: 16 loads in flight a thread; 768 x 4096 5 us.
__device__ __forceinline__ void share_sum(const float *shares, int count, int d, void *out, int type, int block, float (*part)[17]) {
  const int c = block * 16 + threadIdx.x % 4 * 4, lane = threadIdx.x / 4;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c + 4 <= d) {
    const float *p = shares + c;
    for (int q = lane; q < count; q += 1024) {
      f32x4 v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (q + i * 64 < count) v[i] = *reinterpret_cast<const Vec<float, 4>::loose *>(p + static_cast<long>(q + i * 64) * d);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (q + i * 64 < count) s += v[i];
    }
  } else {
    for (int q = lane; q < count; q += 64)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < d) s[i] += shares[static_cast<long>(q) * d + c + i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[lane][threadIdx.x % 4 * 4 + i] = s[i];
  __syncthreads();
  if (threadIdx.x < 64) {
    // 4 threads a column, 16 rows each, joined in lane order.
    const int col = threadIdx.x / 4, at = block * 16 + col;
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < 16; ++q) v += part[threadIdx.x % 4 * 16 + q][col];
    v += __shfl_xor(v, 1);
    v += __shfl_xor(v, 2);
    if (threadIdx.x % 4 == 0 && at < d) store_as(out, type, at, v);
  }
}

// The 8-bit code's scale: the row's largest magnitude over the largest code (448, or
// 127 as an integer), taken as at least 2^-100 so that a row of zeros keeps a finite factor.
template <typename O>
constexpr float kCodeMax = __is_same(O, i8) ? 127.0f : 448.0f;
constexpr float kCodeTiny = 0x1p-100f;
__device__ __forceinline__ float code_top(float top) { return top < kCodeTiny ? kCodeTiny : top; }

// Four integers of up to 8 bits, nearest to v (ties to even), in one word.  Beside 1.5 * 2^23 a
// float's spacing is 1, so the addition rounds and leaves the integer in the lowest byte.  (A NaN
// leaves some code.)
__device__ __forceinline__ uint32_t round_to_bytes(float a, float b, float c, float d) {
  constexpr float kOne = 12582912.0f;
  const auto bits = [](float v) {
#pragma clang fp contract(off)  // v is rounded before: fused with v's last product, ties would fall otherwise than the formula's
    return __builtin_bit_cast(uint32_t, v + kOne);
  };
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits(d), bits(c), 0x0c0c0400u), __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u),
                               0x05040100u);
}

// ---- what is kept in 8 bits -----------------------------------------------------
//
// Rows in groups of 32 neighbours: a group's values are integers of -127..127 times its unit,
// the least power of two (2^-126 at least) whose integers stay within 127.  rows x groups x 32
// codes, zeros behind a row's end, then rows x groups exponents: the unit is 2^(exponent - 127),
// a float of that exponent field.  A group with an infinity or a NaN has the exponent 255 (an
// infinite unit) and codes 0, which make NaN.  `masked`: minus infinity is the code -128 instead and counts
// for no unit, so that a hidden unit masked by its bias has a slope of 0 and leaves its neighbours
// alone.  A unit of two's power restores exactly: the values need no more than bfloat16's bits.
constexpr int kGroup = 32;

struct Kept {
  const uint8_t *codes = nullptr, *exponents = nullptr;
  long groups = 0;  // of a row
};
__host__ __device__ inline Kept kept_at(const void *p, long rows, long d) {
  const long groups = (d + kGroup - 1) / kGroup;
  const uint8_t *codes = static_cast<const uint8_t *>(p);
  return {codes, codes + rows * groups * kGroup, groups};
}

// The exponent for a group's largest magnitude (as bits, which order as magnitudes do, NaN above
// all).  2^6 * 1.m of the unit below rounds past 127 from 1.m = 127.5/64 on: a carry from there.
__device__ __forceinline__ uint32_t group_exponent(uint32_t top) {
  const int e = static_cast<int>((top + 0x10000u) >> 23) - 6;
  return top >= 0x7f800000u ? 255u : static_cast<uint32_t>(max(e, 1));
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The values of 8 codes but for minus infinity's; whether there is one, which restore_masked then puts in.  A largest
// value that was rounded up past T's numbers (64 units of 2^122) is T's largest (float16's, whose groups may be a wider type's: float32's, and then kept_as); a group that stands for NaN has
// no bound.
template <typename T>
__device__ __forceinline__ bool restore_codes(u32x2 codes, uint32_t exponent, float (&v)[8]) {
  const float unit = __builtin_bit_cast(float, exponent << 23);
  const float most = exponent == 255 ? __builtin_nanf("") : __is_same(T, bf16) ? 0x1.fep127f : 0x1.fffffep127f;
  const u32x2 u = codes ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float code = static_cast<float>((i < 4 ? u.x : u.y) >> (8 * (i & 3)) & 255u);
    v[i] = __builtin_amdgcn_fmed3f((code - 128.0f) * unit, -most, most);
  }
  const u32x2 zero = (u - 0x01010101u) & ~u;  // the lowest byte that is 0 leaves its highest bit
  return (zero.x | zero.y) & 0x80808080u;
}
__device__ __forceinline__ void restore_masked(u32x2 codes, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)) & 255u) == 0x80u) v[i] = -__builtin_inff();
}

// The largest of four neighbouring lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 0xf, 0xf, true)));  // lanes 1 0 3 2
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4e, 0xf, 0xf, true)));  // lanes 2 3 0 1
}

// The codes of a lane's 8 values; four neighbouring lanes hold a group, whose exponent each gets.
template <bool MASKED>
__device__ __forceinline__ u32x2 group_codes(const float (&v)[8], bool positive, uint32_t &exponent) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  const bool infinite = MASKED && top == 0x7f800000u;  // seldom: the rest costs a branch a lane
  if (infinite) {
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, v[i] == -__builtin_inff() ? 0u : __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  }
  exponent = group_exponent(quad_max(top));
  const float inverse = __builtin_bit_cast(float, (254u - min(exponent, 253u)) << 23);
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t[i] = v[i] * inverse;
    if (positive && v[i] > 0.0f) t[i] = __builtin_fmaxf(t[i], 1.0f);
  }
  if (infinite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __builtin_fmaxf(t[i], -128.0f);  // minus infinity's code; others are -127.5 at least
  }
  return exponent == 255 ? u32x2{0, 0} : u32x2{round_to_bytes(t[0], t[1], t[2], t[3]), round_to_bytes(t[4], t[5], t[6], t[7])};
}

// 8 values from c (a multiple of 8) of a row; zeros past its last group.
struct KeptCodes {
  u32x2 codes;
  uint32_t exponent;
};
__device__ __forceinline__ KeptCodes load_codes8(const Kept &k, long row, int c) {
  const long length = k.groups * kGroup, at = min(static_cast<long>(c), length - 8);
  const KeptCodes v = {*reinterpret_cast<const u32x2 *>(k.codes + row * length + at), k.exponents[row * k.groups + at / kGroup]};
  return c > at ? KeptCodes{{0, 0}, 1} : v;
}
template <typename T>
__device__ __forceinline__ void restore8(const KeptCodes &k, float (&v)[8]) {
  if (restore_codes<T>(k.codes, k.exponent, v)) restore_masked(k.codes, v);
}
template <typename T>
__device__ __forceinline__ void load_kept8(const Kept &k, long row, int c, float (&v)[8]) {
  restore8<T>(load_codes8(k, row, c), v);
}

// A kept value in T: a finite one past float16's largest is that.
template <typename T>
__device__ __forceinline__ T kept_as(float v) {
  if constexpr (__is_same(T, f16)) {
    const float near = __builtin_fminf(__builtin_fmaxf(v, -65504.0f), 65504.0f);
    return static_cast<T>(__builtin_fabsf(v) < __builtin_inff() ? near : v);
  } else {
    return static_cast<T>(v);
  }
}

}  // namespace tfnn
