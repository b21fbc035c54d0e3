// Matrix products in 16 and 8 bits with a fused epilogue, on the matrix cores.
//
//   C[m][n] = sum over k of A(m, k) * B(k, n)
//
// Each operand lies in memory with k contiguous (rows of k) or with its own
// dimension contiguous (columns of k: a k x n matrix row by row, or the
// transposed left operand of a weight gradient).  Tiles go through LDS in slabs
// of 128 bytes of k a row (64 elements of 16 bits, 128 of 8): the bytes, the
// LDS layout and the reads are the same for all types.
#pragma once

#include "nn_common.hpp"
#include "nn_kernels.h"

namespace tfnn {

typedef __attribute__((address_space(3))) char lds_char;

template <typename T>
constexpr int kSlab = 128 / sizeof(T);  // elements of k in a slab
template <typename T>
constexpr int kPiece = 16 / sizeof(T);  // elements in a 16-byte piece

// LDS layout of one operand's slab, ROWS x 128 bytes.
//
// k contiguous: row after row; the 16-byte piece c of row r is at place
// c ^ (r & 7), so that the 8 rows a quarter-wave reads at one c lie in
// different banks.
//
// Own dimension contiguous: blocks of 64 rows (of the own dimension), in each
// 64 k-lines of 128 bytes; the piece c of line k is at place c ^ turn(k), so that
// the eight lines that two transposing reads of 16 lanes touch at once (k and k + 8)
// lie in different banks.
//
// Either way 1 KiB = 8 lines are one wave's 16-byte load, straight into LDS.

__device__ __forceinline__ int line_turn(int k) { return 2 * ((k & 3) ^ (k >> 3 & 1)); }

// A read piece: 8 (16-bit) or 16 (8-bit) elements along k of one row.
__device__ __forceinline__ i32x4 lds_read16(const lds_char *p) {
  return *reinterpret_cast<const __attribute__((address_space(3))) i32x4 *>(p);
}

// ds_read_b64_tr_b16: of 16 lanes, lane 4r + q names line r, columns 4q..4q+3 of a
// 4 x 16 block; lane j receives column j's four lines.
__device__ __forceinline__ i16x4 lds_read_tr(const lds_char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(p));
}

// Fragment reader of one operand: read<OFF>(kk) gives, for the 16 rows from row
// OFF (a multiple of 16) of the wave's range, this lane's row and its 16 bytes of
// k: pieces g (kk = 0) or 4 + g (kk = 1), g = lane / 16.
template <bool MN>
struct FragReader {
  uint32_t at[MN ? 4 : 2];
  __device__ __forceinline__ void init(int row0) {
    const int lane = threadIdx.x % 64, g = lane / 16, l = lane % 16;
    if constexpr (!MN) {
      at[0] = (row0 + l) * 128 + ((g ^ (l & 7)) << 4);
      at[1] = at[0] ^ 64;
    } else {
      const int r = l / 4, q = l % 4;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int row = row0 + b * 16;  // row0: a multiple of 16
        at[b] = row / 64 * 8192 + (8 * g + r) * 128 + (((row % 64 / 8 + q / 2) ^ line_turn(8 * g + r)) << 4) + (q & 1) * 8;
      }
    }
  }
  template <int OFF, int KK>
  __device__ __forceinline__ i32x4 read(const lds_char *slab) const {
    if constexpr (!MN) {
      return lds_read16(slab + at[KK] + OFF * 128);
    } else {
      // Rows advance by whole 64-row blocks beyond the first four 16-row steps.
      const lds_char *p = slab + at[OFF % 64 / 16] + OFF / 64 * 8192 + KK * 32 * 128;
      union {
        i16x4 h[2];
        i32x4 v;
      } u;
      u.h[0] = lds_read_tr(p);
      u.h[1] = lds_read_tr(p + 4 * 128);
      return u.v;
    }
  }
};

// Buffer resource of `bytes` bytes from `base`; loads past it give zeros.
__device__ __forceinline__ i32x4 buffer_resource(const void *base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return i32x4{__builtin_amdgcn_readfirstlane(static_cast<int>(a)),
               __builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32) & 0xffff), static_cast<int>(bytes), 0x00020000};
}

// 16 bytes a lane from resource + offset to LDS at `lds` + 16 * lane, without
// registers in between.  The caller waits on vmcnt.  (The wait state between the
// write of m0 and its use is the s_nop.)
__device__ __forceinline__ void load_to_lds(i32x4 resource, uint32_t offset, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(offset), "s"(resource)
      : "memory", "m0");
}

constexpr uint32_t kNowhere = 0x80000000u;  // past every resource: reads zeros
constexpr uint32_t kResourceBytes = 0x7fffffffu;

// Loads one operand's slabs.  DMA: straight into LDS; needs 16-byte aligned rows
// and whole pieces (k, or the own dimension, a multiple of the piece), and rows'
// offsets within a tile below 2^31 bytes.  Otherwise through registers, with any
// alignment and any tail.
template <typename T, bool MN, int ROWS, int NW, bool DMA>
struct SlabLoader {
  static constexpr int PER_WAVE = ROWS / 8 / NW;  // 1 KiB loads a wave
  const char *matrix, *base;      // element (0, 0); the tile's first of slab 0
  long step, ld;                  // bytes between slabs, between lines
  int row_first, row_end, k_first, k_end;  // the tile's start and the matrix's end
  uint32_t offset[DMA ? PER_WAVE : 1];     // of this lane's pieces from base
  long far[DMA ? 1 : PER_WAVE];            // the same without the limit

  // Place of this lane's piece of load i: (line, piece) of the layout above.
  static __device__ __forceinline__ void place(int i, int &row, int &k) {
    const int lane = threadIdx.x % 64, t = (threadIdx.x / 64) * PER_WAVE + i;
    if constexpr (!MN) {
      row = t * 8 + lane / 8;
      k = ((lane % 8) ^ (lane / 8)) * kPiece<T>;
    } else {
      k = t % 8 * 8 + lane / 8;
      row = t / 8 * 64 + ((lane % 8) ^ line_turn(k)) * kPiece<T>;
    }
  }

  // own0: the tile's first row; k0: its first k (a whole slab's).
  __device__ __forceinline__ void init(const void *matrix_, long ld_, int own, int own0, int k0, int k1) {
    constexpr long E = sizeof(T);
    matrix = static_cast<const char *>(matrix_);
    ld = ld_ * E;
    row_first = own0;
    row_end = own;
    k_first = k0;
    k_end = k1;
    base = matrix + (MN ? k0 * ld + own0 * E : own0 * ld + k0 * E);
    step = MN ? kSlab<T> * ld : 128;
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) {
        int row, k;
        place(i, row, k);
        offset[i] = row < own - own0 ? static_cast<uint32_t>(MN ? k * ld + row * E : row * ld + k * E) : kNowhere;
      }
    } else {
      // Rows past a matrix shorter than the tile repeat its last (their results are not
      // written); pieces past it start earlier and are shifted.
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) {
        int row, k;
        place(i, row, k);
        const int at = min(row, own - own0 - (MN ? kPiece<T> : 1));
        far[i] = MN ? k * ld + at * E : at * ld + k * E;
      }
    }
  }

  // DMA: starts the loads of slab s into `lds`.
  __device__ __forceinline__ void issue(int s, uint32_t lds) {
    const i32x4 res = buffer_resource(base + s * step, kResourceBytes);
    const int left = k_end - k_first - s * kSlab<T>;
    const uint32_t wave = lds + (threadIdx.x / 64) * (PER_WAVE * 1024);
    if (left >= kSlab<T>) {
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i)
        load_to_lds(res, offset[i], __builtin_amdgcn_readfirstlane(wave + i * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) {
        int row, k;
        place(i, row, k);
        load_to_lds(res, k < left ? offset[i] : kNowhere, __builtin_amdgcn_readfirstlane(wave + i * 1024));
      }
    }
  }

  // Registers: whether the matrix is too small for the unguarded loads.
  __device__ __forceinline__ bool tiny() const { return k_end < kSlab<T> || (MN && row_end < kPiece<T>); }
  // Where slab s is read from, in k from the first: the last starts so that it lies inside.
  __device__ __forceinline__ int slab_at(int s) const { return min(s * kSlab<T>, k_end - kSlab<T> - k_first); }
  // Reads slab s: no branch, so that the compiler counts exactly the loads it has to wait for.
  __device__ __forceinline__ void fetch(int s, i32x4 (&held)[PER_WAVE]) const {
    const char *from = base + slab_at(s) * (MN ? ld : static_cast<long>(sizeof(T)));
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i) held[i] = *reinterpret_cast<const loose16 *>(from + far[i]);
  }
  // Reads any slab: what lies outside becomes zeros.
  __device__ __forceinline__ void fetch_guarded(int s, i32x4 (&held)[PER_WAVE]) const {
    const int length = MN ? row_end : k_end, lines = MN ? k_end : row_end;
    const auto read = [&](auto whole) {
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) {
        int row, k;
        place(i, row, k);
        row += row_first;
        k += k_first + s * kSlab<T>;
        const int line = MN ? k : row, at = MN ? row : k;
        const T *p = reinterpret_cast<const T *>(matrix + min(line, lines - 1) * ld);
        if constexpr (whole()) held[i] = load_piece<false>(p, at, length);
        else held[i] = load_piece_any(p, at, length);
        if (line >= lines) held[i] = i32x4{0, 0, 0, 0};
      }
    };
    if (length >= kPiece<T>) read(Int<1>{});
    else read(Int<0>{});
  }
  // Puts what fetch read of slab s into LDS, without the k that the slab before had.
  __device__ __forceinline__ void put(int s, lds_char *lds, i32x4 (&held)[PER_WAVE]) const {
    constexpr int P = kPiece<T>, BITS = 8 * sizeof(T);
    const int had = s * kSlab<T> - slab_at(s);
    if (had > 0) {
#pragma unroll
      for (int i = 0; i < PER_WAVE; ++i) {
        int row, k;
        place(i, row, k);
        if constexpr (MN) {
          if (k < had) held[i] = i32x4{0, 0, 0, 0};
        } else {
          const int drop = had - k, bits = max(0, min(drop, P - 1)) * BITS;
          const auto u = __builtin_bit_cast(unsigned __int128, held[i]) >> bits << bits;
          held[i] = drop >= P ? i32x4{0, 0, 0, 0} : __builtin_bit_cast(i32x4, u);
        }
      }
    }
    if constexpr (MN) {
      if (row_first + ROWS > row_end) {
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) {
          int row, k;
          place(i, row, k);
          const int past = max(0, row - (row_end - row_first - P));
          const auto u = __builtin_bit_cast(unsigned __int128, held[i]) >> (min(past, P - 1) * BITS);
          held[i] = past >= P ? i32x4{0, 0, 0, 0} : __builtin_bit_cast(i32x4, u);
        }
      }
    }
    put_as_is(lds, held);
  }
  static __device__ __forceinline__ void put_as_is(lds_char *lds, const i32x4 (&held)[PER_WAVE]) {
    lds_char *wave = lds + (threadIdx.x / 64) * (PER_WAVE * 1024) + (threadIdx.x % 64) * 16;
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i)
      *reinterpret_cast<__attribute__((address_space(3))) i32x4 *>(wave + i * 1024) = held[i];
  }
};

// One 16 x 16 block's product over a slab.  The right operand goes first: the
// block comes out with a lane's four values in one row of C, next to each other.
__device__ __forceinline__ f32x4 block_mma(bf16, i32x4 a0, i32x4 a1, i32x4 b0, i32x4 b1, f32x4 c) {
  typedef bf16 v8 __attribute__((ext_vector_type(8)));
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, b0), __builtin_bit_cast(v8, a0), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, b1), __builtin_bit_cast(v8, a1), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 block_mma(f16, i32x4 a0, i32x4 a1, i32x4 b0, i32x4 b1, f32x4 c) {
  typedef f16 v8 __attribute__((ext_vector_type(8)));
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, b0), __builtin_bit_cast(v8, a0), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, b1), __builtin_bit_cast(v8, a1), c, 0, 0, 0);
}
// 8 bits: one instruction takes both pieces; the order of k inside it is the
// same on both sides, so any order will do.  (Scales 0, 0: the unscaled form.)  It adds
// float sums of eight products, each of which it cuts off 13 bits below the largest of the
// eight (measured with products of powers of two; the 16 x 16 x 32 form does the same).
// The sums are off by 1.5e-5 in the root mean square.  As bfloat16 the codes would be multiplied
// exactly, at half the rate; the result's rounding to 16 bits hides the difference.
__device__ __forceinline__ f32x4 block_mma(f8, i32x4 a0, i32x4 a1, i32x4 b0, i32x4 b1, f32x4 c) {
  const i32x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
  const i32x8 b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, 0, 0, 0);
}

// 8-bit integers: sums of 32-bit integers, exact while k is at most 131071 (128 * 128 * k < 2^31).
// A loop of nothing but these reaches 3.9 POP/s at the power limit (e4m3's instruction 4.5, 32 x 32 x 32
// blocks of integers 3.3), and the products stand so too: 8192^3 487 us, e4m3 404.
__device__ __forceinline__ i32x4 block_mma(i8, i32x4 a0, i32x4 a1, i32x4 b0, i32x4 b1, i32x4 c) {
  c = __builtin_amdgcn_mfma_i32_16x16x64_i8(b0, a0, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(b1, a1, c, 0, 0, 0);
}

// A 16 x 16 block's four sums a lane, and one of them.
template <typename T>
struct SumsOf {
  typedef f32x4 four;
  typedef float one;
};
template <>
struct SumsOf<i8> {
  typedef i32x4 four;
  typedef int one;
};
template <typename T>
using sums4 = typename SumsOf<T>::four;

// An 8-bit product's sum times its scales.  Of integers in three roundings everywhere: left to the
// compiler, some kernels would fuse the last with the bias's addition and others not, and the
// results' bits would depend on the tile.
template <typename T>
__device__ __forceinline__ float scaled(typename SumsOf<T>::one sum, float sa, float sb) {
  if constexpr (__is_same(T, i8)) {
#pragma clang fp contract(off)
    return static_cast<float>(sum) * sa * sb;
  } else {
    return sum * sa * sb;
  }
}

// What is not finite becomes finite, by one instruction (a NaN the least number).
__device__ __forceinline__ f32x4 made_finite(f32x4 v) {
  constexpr float kMost = 0x1.fffffep127f;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i], -kMost, kMost);
  return v;
}

// ---- epilogue ---------------------------------------------------------------

// N consecutive values from p[0..left), zeros past them.
template <int N, typename T>
__device__ __forceinline__ void load_some(const T *p, int left, float (&v)[N]) {
  if (left >= N) {
    const typename Vec<T, N>::loose u = *reinterpret_cast<const typename Vec<T, N>::loose *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? static_cast<float>(p[i]) : 0.0f;
  }
}
// STREAM: past the caches, for results that would push the operands out of them.
template <bool STREAM = false, int N, typename T, typename V>
__device__ __forceinline__ void store_some(T *p, int left, const V (&v)[N]) {
  if (left >= N) {
    typename Vec<T, N>::loose u;
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = static_cast<T>(v[i]);
    if constexpr (STREAM) __builtin_nontemporal_store(u, reinterpret_cast<typename Vec<T, N>::loose *>(p));
    else *reinterpret_cast<typename Vec<T, N>::loose *>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = static_cast<T>(v[i]);
  }
}

template <typename O, int N>
__device__ __forceinline__ void load_bias(const GemmParams &p, int n, float (&v)[N]) {
  if (!p.bias) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
  } else if (p.bias_f32) {
    load_some(static_cast<const float *>(p.bias) + n, p.n - n, v);
  } else {
    load_some(static_cast<const O *>(p.bias) + n, p.n - n, v);
  }
}

// z = v + bias (kept if asked for); out = act(z) + residual, rounded once.
template <typename O, int ACT, bool STREAM = false, int N>
__device__ __forceinline__ void finish(const GemmParams &p, int m, int n, float (&v)[N], const float (&bias)[N]) {
  const int left = p.n - n;
  float res[N];
  if (p.residual) load_some(static_cast<const O *>(p.residual) + m * p.ldr + n, left, res);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += bias[i];
  if (p.z) store_some<STREAM>(static_cast<O *>(p.z) + m * p.ldz + n, left, v);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = act_value<ACT>(v[i]);
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += res[i];
  }
  store_some<STREAM>(static_cast<O *>(p.out) + m * p.ldo + n, left, v);
}

// f(constant) for the product's activation.
template <typename F>
__device__ __forceinline__ void with_act(int act, F &&f) {
  switch (act) {
    case ACT_RELU: f(Int<ACT_RELU>{}); break;
    case ACT_GELU: f(Int<ACT_GELU>{}); break;
    case ACT_SILU: f(Int<ACT_SILU>{}); break;
    default: f(Int<ACT_NONE>{}); break;
  }
}

// A wave's accumulators reach memory through LDS of its own: ROWS x COLS floats,
// the four of quad c in row r at place c ^ (r mod COLS/4).  The blocks come a
// few columns of many rows at a time; from LDS a row's lanes write whole cache
// lines (and read the residual's).  Straight from the blocks, in 16-byte parts of
// rows, the whole product took a twelfth longer at 8192^3 (883 us, 815 this way).
template <int COLS>
__device__ __forceinline__ uint32_t patch_at(int row, int quad) {
  return row * (COLS * 4) + ((quad ^ (row & (COLS / 4 - 1))) << 4);
}

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The blocks reach memory by rows through the wave's patch of LDS (nn_gemm.hpp), ROWS at a
// time: put(row, column, eight values), both from the wave's first.
template <int ROWS, int MI, int NI, typename F>
__device__ __forceinline__ void by_rows(const f32x4 (&acc)[MI][NI], lds_char *patch, F &&put) {
  constexpr int COLS = NI * 16, LANES = COLS / 8;
  const int lane = threadIdx.x % 64, c = lane % LANES;
#pragma unroll
  for (int h = 0; h < MI * 16 / ROWS; ++h) {
#pragma unroll
    for (int i = 0; i < ROWS / 16; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<__attribute__((address_space(3))) f32x4 *>(patch + patch_at<COLS>(i * 16 + lane % 16, j * 4 + lane / 16)) =
            acc[h * (ROWS / 16) + i][j];
    wait_lds();
#pragma unroll 4
    for (int row = lane / LANES; row < ROWS; row += 64 / LANES) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 u = __builtin_bit_cast(f32x4, lds_read16(patch + patch_at<COLS>(row, c * 2 + q)));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[q * 4 + i] = u[i];
      }
      put(h * ROWS + row, c * 8, v);
    }
  }
}

// (m0, n0): the patch's place in C.  (mt, nt): the workgroup's own first row and
// column; where its tile was moved back into the matrix, what lies before them is
// another's (eight columns across nt are written by both, with the same values).
template <typename T, typename O, int ROWS, int COLS, bool STREAM = false>
__device__ __forceinline__ void write_patch(const GemmParams &p, int split, const lds_char *patch, int m0, int n0, int mt,
                                            int nt) {
  constexpr int LANES = COLS / 8, STEP = 64 / LANES;
  const int lane = threadIdx.x % 64, n = n0 + lane % LANES * 8, left = p.n - n;
  if (left <= 0 || n + 7 < nt) return;
  typedef typename SumsOf<T>::one Sum;
  const auto take = [&](int row, auto (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto u = __builtin_bit_cast(sums4<T>, lds_read16(patch + patch_at<COLS>(row, lane % LANES * 2 + h)));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[h * 4 + i] = u[i];
    }
  };
  if (p.splits > 1) {  // one range of k of several: sums joined by gemm_join_kernel
    const long ld = (p.n + 3) & ~3;
    Sum *part = reinterpret_cast<Sum *>(p.parts) + split * (p.m * ld);
    for (int row = lane / LANES; row < ROWS; row += STEP) {
      const int m = m0 + row;
      if (m >= p.m || m < mt) continue;
      Sum v[8];
      take(row, v);
      store_some(part + m * ld + n, left, v);
    }
    return;
  }
  float bias[8], sb[8];
  load_bias<O>(p, n, bias);
  if constexpr (sizeof(T) == 1) load_some(p.sb + n, left, sb);
  with_act(p.act, [&](auto act) {
#pragma unroll 4
    for (int row = lane / LANES; row < ROWS; row += STEP) {
      const int m = m0 + row;
      if (m >= p.m || m < mt) continue;
      float v[8];
      if constexpr (sizeof(T) == 1) {
        Sum sums[8];
        take(row, sums);
        const float sa = p.sa[m];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = scaled<T>(sums[i], sa, sb[i]);
      } else {
        take(row, v);
      }
      finish<O, act(), STREAM>(p, m, n, v, bias);
    }
  });
}

// ---- tile order ---------------------------------------------------------------

// Workgroups are dealt to the 8 XCDs in turn; each XCD gets one run of
// consecutive tiles, walked in bands of 8 tile rows, so that its L2 holds the
// rows and columns it shares.
__device__ __forceinline__ void tile_of(const GemmParams &p, int id, int total, int &tm, int &tn, int &split) {
  const int xcd = id & 7, per = total >> 3, more = total & 7;
  int t = xcd * per + min(xcd, more) + (id >> 3);
  const int tiles = p.tiles_m * p.tiles_n;
  split = t / tiles;
  t -= split * tiles;
  const int band = 8 * p.tiles_n, first = t / band * 8, rows = min(8, p.tiles_m - first);
  t %= band;
  tm = first + t % rows;
  tn = t / rows;
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A workgroup's barrier for LDS: what was written before it is read behind it.
// (Loads and stores of memory are not waited for.)
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---- the tile kernel ----------------------------------------------------------

// BM x BN of C a workgroup, WM x WN waves, ST slabs of LDS.  One barrier a slab:
// behind it slab s has arrived for all waves and slab s-1 is used up, so slab
// s+ST-1 may take its place while s is multiplied.
//
// 128 x 128 where 256 x 256 leaves CUs idle, 64 x 128 and 64 x 64 below that; bound by
// each CU's turn of LDS reads and matrix instructions, two or more workgroups on a CU
// filling each other's waits.  bfloat16, 128/64 x 128/64 tile: 2048 x 4096 x 4096 60.0 / 75.9 /
// 88.4 us (1145 TFLOP/s), 1024 x 4096 x 4096 46.5 / 39.2 / 45.6 (876), 512 x 4096 x 4096 32.2 /
// 30.3 / 26.1 (658).
//
// Of `blocks` workgroups this is number `block`.  An operand of two terms (what a value's
// rounding left, and the value) is multiplied term after term into the same sums.  What the
// rounding left comes first: it is finite, so a sum of it that is not finite has met an
// infinity or a NaN of the other operand, and is made finite.  The value meets the same one
// and gives these elements their infinity or NaN; both would give infinity - infinity or
// infinity * 0.  (TERMS is a constant: with the choice in the kernel one term took up to 4%
// longer, 256 x 83 x 800 8.0 to 8.3 us.)
template <int BM, int BN, int ST>
constexpr int tile_lds() {
  return ST * (BM + BN) * 128;
}
//
// E: what becomes of the sums; Results writes them with bias, activation and residual.
struct Results {
  typedef GemmParams Params;
};
template <typename T, typename O, bool AMN, bool BMN, int BM, int BN, int WM, int WN, int ST, bool DMA, int TERMS, typename E = Results>
__device__ __forceinline__ void gemm_tile(const typename E::Params &p, int block, int blocks, lds_char *lds) {
  constexpr int NW = WM * WN, MI = BM / WM / 16, NI = BN / WN / 16, STAGE = (BM + BN) * 128;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  int tm, tn, split;
  tile_of(p, block, blocks, tm, tn, split);
  const int slabs = (p.k + kSlab<T> - 1) / kSlab<T>;
  const int s0 = static_cast<int>(static_cast<long>(slabs) * split / p.splits);
  const int count = static_cast<int>(static_cast<long>(slabs) * (split + 1) / p.splits) - s0;
  const int k0 = s0 * kSlab<T>;
  SlabLoader<T, AMN, BM, NW, DMA> la;
  SlabLoader<T, BMN, BN, NW, DMA> lb;
  // Loads through registers: a tile that would reach past the matrix's end starts earlier.
  const int m0 = DMA ? tm * BM : max(0, min(tm * BM, p.m - BM)), n0 = DMA ? tn * BN : max(0, min(tn * BN, p.n - BN));
  constexpr int LOADS = decltype(la)::PER_WAVE + decltype(lb)::PER_WAVE;

  const int wave = threadIdx.x / 64, wm = wave / WN, wn = wave % WN;
  FragReader<AMN> fa;
  FragReader<BMN> fb;
  fa.init(wm * (BM / WM));
  fb.init(wn * (BN / WN));
  sums4<T> acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = sums4<T>{0, 0, 0, 0};

  const auto multiply = [&](const lds_char *slab) {
    i32x4 a[2][MI], b[2][NI];
    unroll<MI>([&](auto i) {
      a[0][i] = fa.template read<16 * i, 0>(slab);
      a[1][i] = fa.template read<16 * i, 1>(slab);
    });
    unroll<NI>([&](auto j) {
      b[0][j] = fb.template read<16 * j, 0>(slab + BM * 128);
      b[1][j] = fb.template read<16 * j, 1>(slab + BM * 128);
    });
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = block_mma(T{}, a[0][i], a[1][i], b[0][j], b[1][j], acc[i][j]);
  };

  for (int term = 0; term < TERMS; ++term) {
    la.init(static_cast<const char *>(p.a) + term * p.a_term, p.lda, p.m, m0, k0, p.k);
    lb.init(static_cast<const char *>(p.b) + term * p.b_term, p.ldb, p.n, n0, k0, p.k);
    if (term) barrier();  // the last term's slabs are used up
    if constexpr (DMA) {
#pragma unroll
      for (int s = 0; s < ST - 1; ++s)
        if (s < count) {
          la.issue(s, lds0 + s * STAGE);
          lb.issue(s, lds0 + s * STAGE + BM * 128);
        }
      int at = 0;
      for (int s = 0; s < count; ++s) {
        if (ST > 2 && s + ST - 2 < count) wait_loads<(ST - 2) * LOADS>();
        else wait_loads<0>();
        barrier();
        const int into = at == 0 ? ST - 1 : at - 1;
        if (s + ST - 1 < count) {
          la.issue(s + ST - 1, lds0 + into * STAGE);
          lb.issue(s + ST - 1, lds0 + into * STAGE + BM * 128);
        }
        multiply(lds + at * STAGE);
        wait_lds();
        at = at == ST - 1 ? 0 : at + 1;
      }
    } else {
      // DEEP slabs are under way in registers while one is multiplied; past the last they
      // repeat it.  With branches around the loads the compiler waits for all of them:
      // 1536 x 256 x 2558 bfloat16 30.7 us, two slabs deep; 14.2 this way.
      // (Four of lines not along k do not leave registers for three workgroups a CU: 100 odd
      // products took 3.7% longer.)
      constexpr int DEEP = AMN || BMN ? 3 : 4;
      i32x4 ha[DEEP][decltype(la)::PER_WAVE], hb[DEEP][decltype(lb)::PER_WAVE];
      if (count > 0 && !la.tiny() && !lb.tiny()) {
#pragma unroll
        for (int q = 0; q < DEEP; ++q) {
          la.fetch(q, ha[q]);
          lb.fetch(q, hb[q]);
        }
        la.put(0, lds, ha[0]);
        lb.put(0, lds + BM * 128, hb[0]);
        constexpr int TURN = DEEP % 2 ? 2 * DEEP : DEEP;  // steps until slab and LDS place come together again
        const auto step = [&](auto h, int s) {
          wait_lds();
          barrier();
          la.fetch(s + h() + DEEP, ha[h() % DEEP]);
          lb.fetch(s + h() + DEEP, hb[h() % DEEP]);
          multiply(lds + h() % 2 * STAGE);
          la.put(s + h() + 1, lds + (1 - h() % 2) * STAGE, ha[(h() + 1) % DEEP]);
          lb.put(s + h() + 1, lds + (1 - h() % 2) * STAGE + BM * 128, hb[(h() + 1) % DEEP]);
        };
        int s = 0;
        for (; s + TURN <= count; s += TURN) unroll<TURN>([&](auto h) { step(h, s); });
        unroll<TURN - 1>([&](auto h) {
          if (s + h() < count) step(h, s);
        });
      } else {
        for (int s = 0; s < count; ++s) {
          la.fetch_guarded(s, ha[0]);
          lb.fetch_guarded(s, hb[0]);
          wait_lds();
          barrier();
          la.put_as_is(lds, ha[0]);
          lb.put_as_is(lds + BM * 128, hb[0]);
          wait_lds();
          barrier();
          multiply(lds);
        }
      }
    }
    wait_lds();
    if constexpr (TERMS > 1) {
      if (term + 1 < TERMS) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = made_finite(acc[i][j]);
      }
    }
  }
  barrier();  // the slabs' LDS is the patches' now
  constexpr int COLS = BN / WN, ROWS = BM / WM / ((BM / WM) * COLS > 4096 ? 2 : 1);  // 16 KiB a wave at most
  static_assert(NW * ROWS * COLS * 4 <= (DMA ? ST : 2) * STAGE, "the patches fit into the slabs' LDS");
  lds_char *patch = lds + wave * (ROWS * COLS * 4);
  if constexpr (__is_same(E, Results)) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int h = 0; h < BM / WM / ROWS; ++h) {
#pragma unroll
      for (int i = 0; i < ROWS / 16; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
          *reinterpret_cast<__attribute__((address_space(3))) sums4<T> *>(
              patch + patch_at<COLS>(i * 16 + lane % 16, j * 4 + lane / 16)) = acc[h * (ROWS / 16) + i][j];
      wait_lds();
      write_patch<T, O, ROWS, COLS>(p, split, patch, m0 + wm * (BM / WM) + h * ROWS, n0 + wn * COLS, tm * BM, tn * BN);
    }
  } else {
    E::template finish<T, BM, BN, WM, WN, ROWS>(p, acc, split, lds, patch, m0, n0, wm, wn, tm, tn);
  }
}

template <typename T, typename O, bool AMN, bool BMN, int BM, int BN, int WM, int WN, int ST, bool DMA, int TERMS>
__global__ __launch_bounds__(64 * WM *WN, DMA ? 1 : 3) void gemm_tile_kernel(GemmParams p) {
  __shared__ __align__(1024) char smem[tile_lds<BM, BN, ST>()];
  if constexpr (DMA) {
    gemm_tile<T, O, AMN, BMN, BM, BN, WM, WN, ST, DMA, TERMS>(p, blockIdx.x, gridDim.x, (lds_char *)smem);
  } else {  // the one tile of odd operands: also where its grid has a second side
    const int block = static_cast<int>(block_of()), blocks = p.tiles_m * p.tiles_n * p.splits;
    if (block < blocks) gemm_tile<T, O, AMN, BMN, BM, BN, WM, WN, ST, DMA, TERMS>(p, block, blocks, (lds_char *)smem);
  }
}

// A small layer's two gradient products in one launch: dx (its left operand along
// k) by the first `first` workgroups, dw (both along their own dimensions) by the
// next `second`, the bias gradient's sum by the others.  Bound by latency: 256 x 256 x 128
// float16 5.1 us (one launch each: 5 + 5), 768 x 256 x 344 in ranges of k 7.0 (6.2 + 11.1).
template <typename T, bool BMN, int TERMS>
__global__ __launch_bounds__(256) void gemm_pair_kernel(GemmParams dx, GemmParams dw, ShareParams sum, int first, int second) {
  constexpr int ST = 3;  // three workgroups on a CU; with four slabs, two: 100 drawn gradients took 2% longer
  __shared__ __align__(1024) char smem[tile_lds<64, 64, ST>()];
  const int block = blockIdx.x;
  if (block < first)
    gemm_tile<T, T, false, BMN, 64, 64, 2, 2, ST, true, TERMS>(dx, block, first, (lds_char *)smem);
  else if (block < first + second)
    gemm_tile<T, T, true, true, 64, 64, 2, 2, ST, true, TERMS>(dw, block - first, second, (lds_char *)smem);
  else
    share_sum(sum.shares, sum.count, sum.d, sum.out, sum.type, block - first - second, reinterpret_cast<float (*)[17]>(smem));
}

// ---- few rows -----------------------------------------------------------------

// Waves of a few-row workgroup: 16, or 8 where their registers would not fit.
constexpr int rows_waves(bool bmn, int mi) { return bmn && mi > 1 ? 8 : 16; }

// Up to 16*MI rows of C: bound by the right operand's one read, so the waves of
// a workgroup stream it side by side, each its own slabs of k, and meet in LDS
// at the end.  No barrier on the way.  16 columns a workgroup where the right
// operand lies along k: its pieces are fragments as they come.  32 columns where
// it lies along n: a wave turns its slab over in LDS of its own, 64-byte lines
// with piece c of line k at c ^ (k & 2).  The left operand's pieces come from the
// caches.  Any alignment.  The last workgroup's columns are moved back into the
// matrix (n >= 32 where the right operand lies along n) and a last part of a slab
// is read apart, so the loads on the way are unguarded.  A left operand of two
// terms takes twice the blocks of rows, joined with the waves' sums.  Bound by a CU's
// misses while it streams its columns: 1 x 4096 x 4096 bfloat16 (n rows of k) 7.8 us
// (33.5 MB, 4.3 TB/s with the launch), 16 x 2048 x 8192 in 8 bits 9.8 us.
template <typename T, typename O, bool BMN, int MI>
__global__ __launch_bounds__(64 * rows_waves(BMN, MI)) void gemm_rows_kernel(GemmParams p) {
  constexpr int NB = BMN ? 2 : 1, NW = rows_waves(BMN, MI), WP = BMN ? 4 : 2;  // pieces a lane of one slab of B
  constexpr int P = kPiece<T>;
  constexpr int TURN = BMN ? NW * 4096 : 0, JOIN = NW * MI * NB * 1024;
  __shared__ __align__(1024) char smem[TURN > JOIN ? TURN : JOIN];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, g = lane / 16, l = lane % 16;
  // Neighbouring columns on one XCD: they share the lines of B that lie along n.
  const int per = gridDim.x >> 3, more = gridDim.x & 7, xcd = blockIdx.x & 7;
  const int nt = (xcd * per + min(xcd, more) + static_cast<int>(blockIdx.x >> 3)) * 16 * NB;
  const int n0 = BMN ? min(nt, p.n - 16 * NB) : nt;
  const int slabs = p.k / kSlab<T>;  // whole ones
  const T *a[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {  // rows past the last repeat it; their results are not written
    const int term = MI > 1 && p.terms == 2 && i >= MI / 2, row = (i - (term ? MI / 2 : 0)) * 16 + l;
    a[i] = reinterpret_cast<const T *>(static_cast<const char *>(p.a) + term * p.a_term) + min(row, p.m - 1) * p.lda;
  }
  const T *b = static_cast<const T *>(p.b);
  if constexpr (BMN) b += (lane / 4) * p.ldb + n0 + lane % 4 * 8;
  else b += min(n0 + l, p.n - 1) * p.ldb;

  struct Held {
    i32x4 a[MI][2], b[WP];
  };
  const auto fetch = [&](Held &h, int s) {
    const int k0 = s * kSlab<T>;
#pragma unroll
    for (int i = 0; i < WP; ++i)
      h.b[i] = *reinterpret_cast<const loose16 *>(BMN ? b + (k0 + i * 16) * p.ldb : b + k0 + (i * 4 + g) * P);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) h.a[i][q] = *reinterpret_cast<const loose16 *>(a[i] + k0 + (q * 4 + g) * P);
  };
  sums4<T> acc[MI][NB];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = sums4<T>{0, 0, 0, 0};
  lds_char *turn = (lds_char *)smem + wave * 4096;
  const auto multiply = [&](Held &h) {
    i32x4 bf[NB][2];
    if constexpr (BMN) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = i * 16 + lane / 4;
        *reinterpret_cast<__attribute__((address_space(3))) i32x4 *>(turn + k * 64 + (((lane % 4) ^ (k & 2)) << 4)) = h.b[i];
      }
      const int r = l / 4, q = l % 4;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const lds_char *at = turn + (kk * 32 + 8 * g + r) * 64 + (((2 * j + q / 2) ^ (r & 2)) << 4) + (q & 1) * 8;
          union {
            i16x4 h[2];
            i32x4 v;
          } u;
          u.h[0] = lds_read_tr(at);
          u.h[1] = lds_read_tr(at + 4 * 64);
          bf[j][kk] = u.v;
        }
    } else {
      bf[0][0] = h.b[0];
      bf[0][1] = h.b[1];
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = block_mma(T{}, h.a[i][0], h.a[i][1], bf[j][0], bf[j][1], acc[i][j]);
  };
  // DEEP slabs are in flight while one is multiplied.
  constexpr int DEEP = MI == 1 && !BMN ? 4 : 2;
  Held held[DEEP];
  int s = wave;
#pragma unroll
  for (int q = 0; q < DEEP; ++q)
    if (s + q * NW < slabs) fetch(held[q], s + q * NW);
  for (; s < slabs; s += DEEP * NW) {
#pragma unroll
    for (int q = 0; q < DEEP; ++q) {
      if (s + q * NW < slabs) {
        multiply(held[q]);
        if (s + (q + DEEP) * NW < slabs) fetch(held[q], s + (q + DEEP) * NW);
      }
    }
  }
  if (p.k % kSlab<T> && wave == slabs % NW) {  // what is left of k
    const int k0 = slabs * kSlab<T>;
    Held &h = held[0];
    const auto rest = [&](auto whole) {  // whole: k is at least a piece
      const auto piece = [&](const T *row, int at) {
        if constexpr (whole()) return load_piece<false>(row, at, p.k);
        else return load_piece_any(row, at, p.k);
      };
#pragma unroll
      for (int i = 0; i < WP; ++i) {
        if constexpr (BMN) {
          const int k = k0 + i * 16 + lane / 4;
          const i32x4 v = *reinterpret_cast<const loose16 *>(b + (min(k, p.k - 1) - lane / 4) * p.ldb);
          h.b[i] = k < p.k ? v : i32x4{0, 0, 0, 0};
        } else {
          h.b[i] = piece(b, k0 + (i * 4 + g) * P);
        }
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q) h.a[i][q] = piece(a[i], k0 + (q * 4 + g) * P);
    };
    if (p.k >= P) rest(Int<1>{});
    else rest(Int<0>{});
    multiply(h);
  }
  // The waves' sums, added in wave order.
  __syncthreads();
  sums4<T> *join = reinterpret_cast<sums4<T> *>(smem);
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) join[(wave * MI * NB + i * NB + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  const int block = wave;
  const int blocks = MI > 1 && p.terms == 2 ? MI / 2 * NB : MI * NB;
  if (block >= blocks) return;
  sums4<T> v = join[block * 64 + lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) v += join[(w * MI * NB + block) * 64 + lane];
  if constexpr (sizeof(T) == 2) {
    if (blocks < MI * NB) {  // the other term, as in gemm_tile
      v = made_finite(v);
#pragma unroll
      for (int w = 0; w < NW; ++w) v += join[(w * MI * NB + blocks + block) * 64 + lane];
    }
  }
  const int m = block / NB * 16 + l, n = n0 + block % NB * 16 + g * 4;
  if (m >= p.m || n >= p.n || n + 3 < nt) return;
  float out[4], bias[4];
  load_bias<O>(p, n, bias);
  if constexpr (sizeof(T) == 1) {
    float sb[4];
    load_some(p.sb + n, p.n - n, sb);
    const float sa = p.sa[m];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = scaled<T>(v[i], sa, sb[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = v[i];
  }
  with_act(p.act, [&](auto act) { finish<O, act()>(p, m, n, out, bias); });
}

}  // namespace tfnn
