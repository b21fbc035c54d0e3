// Root-mean-square norm with the residual's addition, in the input's type or in
// 8 bits (e4m3 or integers) with a scale a row, the row quantisation alone, and the norm's gradient.
//
//   h = x + residual           r = 1/sqrt(mean(h^2) + eps)
//   y = (h*r)*w                scale = max|y| / top, code = nearest(y * (top * (1/max|y|))), top 448 or 127
//   g = dy*w, xhat = h*r       dx = r*(g - xhat*mean(g*xhat)) + dh,  dw = sum over rows of dy*xhat
//
// All of it is bound by memory.  A row stays in its threads' registers between
// its read and its write, so every tensor is read once and written once; both
// sums a row needs (of squares, and the largest |h*w|, as max|y| = r*max|h*w|)
// come from one pass and one reduction.
#include "nn_common.hpp"
#include "nn_kernels.h"

#include <algorithm>

namespace tfnn {
namespace {

// Row lengths: WHOLE, a multiple of 8; TAIL, at least 8; ANY, shorter ones too.
enum Length { WHOLE, TAIL, ANY };

// 8 elements from c of a row of `length`; zeros past its end.
template <Length L, typename T>
__device__ __forceinline__ void load8(const T *row, int c, int length, float (&v)[8]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int q = 0; q < 8 / N; ++q) {
    i32x4 raw;
    if constexpr (L == ANY) raw = load_piece_any(row, c + q * N, length);
    else raw = load_piece<L == WHOLE>(row, c + q * N, length);
    const auto u = __builtin_bit_cast(typename Vec<T, N>::type, raw);
#pragma unroll
    for (int i = 0; i < N; ++i) v[q * N + i] = static_cast<float>(u[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, int left, const float (&v)[8]) {
  if (left >= 8) {
    typename Vec<T, 8>::loose u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = static_cast<T>(v[i]);
    *reinterpret_cast<typename Vec<T, 8>::loose *>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = static_cast<T>(v[i]);
  }
}

__device__ __forceinline__ void store8(f8 *p, int left, const float (&v)[8]) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  if (left >= 8) {
    typedef int loose2 __attribute__((ext_vector_type(2), aligned(1)));
    *reinterpret_cast<loose2 *>(p) = loose2{lo, hi};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i].bits = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ void store8(i8 *p, int left, const float (&v)[8]) {
  const uint32_t lo = round_to_bytes(v[0], v[1], v[2], v[3]), hi = round_to_bytes(v[4], v[5], v[6], v[7]);
  if (left >= 8) {
    typedef uint32_t loose2 __attribute__((ext_vector_type(2), aligned(1)));
    *reinterpret_cast<loose2 *>(p) = loose2{lo, hi};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i].bits = static_cast<int8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

template <Length L>
__device__ __forceinline__ void load_weight8(const NormParams &p, int c, float (&w)[8]) {
  if (!p.weight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.0f;
  } else if (p.weight_type == TYPE_F32) {
    load8<L>(static_cast<const float *>(p.weight), c, p.d, w);
  } else if (p.weight_type == TYPE_BF16) {
    load8<L>(static_cast<const bf16 *>(p.weight), c, p.d, w);
  } else {
    load8<L>(static_cast<const f16 *>(p.weight), c, p.d, w);
  }
}

// Sum of `sum`, and sum or maximum (MAX) of `more`, over the NT threads of a
// row.  With NT = 256 the four waves meet in LDS (ROWS rows a workgroup, each in a
// place of its own); `turn` alternates between two places, so one barrier a row is
// enough.  Every thread of the workgroup calls it equally often.
template <int NT, bool MAX, int ROWS = 1>
__device__ __forceinline__ void row_reduce(float &sum, float &more, int turn) {
  sum = wave_sum(sum);
  more = MAX ? wave_max(more) : wave_sum(more);
  if constexpr (NT > 64) {
    __shared__ float part[2][2][ROWS * NT / 64];
    const int wave = threadIdx.x / 64, first = threadIdx.x / NT * (NT / 64);
    if (threadIdx.x % 64 == 0) {
      part[turn][0][wave] = sum;
      part[turn][1][wave] = more;
    }
    __syncthreads();
    sum = part[turn][0][first];
    more = part[turn][1][first];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) {
      sum += part[turn][0][first + i];
      more = MAX ? max_keep_nan(more, part[turn][1][first + i]) : more + part[turn][1][first + i];
    }
  }
}

// CH pieces of 8 elements a thread, NT threads a row, 256/NT rows a workgroup.
// The weights stay in registers over a workgroup's rows; so do the comparisons of a row's end with
// a thread's 64 places, those of the wide forms partly in lanes of vector registers (10 to 166
// scalar registers spilled so here and in the gradient, none to memory).  Compared anew each row,
// with no such spill, bfloat16 took 0 to 5% less and float32 up to 8% more (8192 x 8191 156 to
// 169 us).  Bound by memory: 16384 x 8192
// bfloat16 with a residual into 8 bits 173 us (940 MB, 5.4 TB/s; a large copy does 5.1),
// 8192 x 8192 quantised alone 34 us (6.0); one row of 2048 2.6 us, a launch's latency.
template <typename T, typename O, int NT, int CH, Length L>
__global__ __launch_bounds__(256) void rms_norm_kernel(NormParams p) {
  constexpr int RPB = 256 / NT;
  const int t = threadIdx.x % NT, sub = threadIdx.x / NT;
  float w[CH][8];
#pragma unroll
  for (int j = 0; j < CH; ++j) load_weight8<L>(p, (j * NT + t) * 8, w[j]);
  int turn = 0;
  for (long row = static_cast<long>(blockIdx.x) * RPB + sub; row < p.rows; row += static_cast<long>(gridDim.x) * RPB) {
    const T *x = static_cast<const T *>(p.x) + row * p.x_ld;
    float h[CH][8];
#pragma unroll
    for (int j = 0; j < CH; ++j) load8<L>(x, (j * NT + t) * 8, p.d, h[j]);
    if (p.residual) {
      const T *res = static_cast<const T *>(p.residual) + row * p.residual_ld;
      T *ho = static_cast<T *>(p.h) + row * p.h_ld;
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        float v[8];
        load8<L>(res, (j * NT + t) * 8, p.d, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] += v[i];
      }
#pragma unroll
      for (int j = 0; j < CH; ++j) store8(ho + (j * NT + t) * 8, p.d - (j * NT + t) * 8, h[j]);
    }
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = __builtin_fmaf(h[j][i], h[j][i], sum);
        if constexpr (sizeof(O) == 1) top = max_keep_nan(top, __builtin_fabsf(h[j][i] * w[j][i]));
      }
    row_reduce<NT, true>(sum, top, turn);
    turn ^= 1;
    const float r = p.weight ? rsqrtf(sum / static_cast<float>(p.d) + p.eps) : 1.0f;
    float f = 1.0f;
    if constexpr (sizeof(O) == 1) {
      const float most = code_top(top * r);
      f = kCodeMax<O> * (1.0f / most);
      if (t == 0) p.scale[row] = most / kCodeMax<O>;
    }
    O *y = static_cast<O *>(p.y) + row * p.y_ld;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = h[j][i] * r * w[j][i];
        if constexpr (sizeof(O) == 1) v[i] *= f;
      }
      store8(y + (j * NT + t) * 8, p.d - (j * NT + t) * 8, v);
    }
  }
}

// Rows longer than a workgroup's registers hold: a second read of the row (from
// the caches) in place of keeping it.  4096 x 32768 bfloat16 with a residual 308 us (3.5 TB/s).
template <typename T, typename O>
__global__ __launch_bounds__(256) void rms_norm_long_kernel(NormParams p) {
  constexpr int NT = 256;
  const long row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_ld;
  const T *res = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_ld : nullptr;
  float sum = 0.0f, top = 0.0f;
  for (int c = threadIdx.x * 8; c < p.d; c += NT * 8) {
    float v[8], u[8], w[8];
    load8<TAIL>(x, c, p.d, v);
    if (res) {
      load8<TAIL>(res, c, p.d, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += u[i];
    }
    load_weight8<TAIL>(p, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum = __builtin_fmaf(v[i], v[i], sum);
      if constexpr (sizeof(O) == 1) top = max_keep_nan(top, __builtin_fabsf(v[i] * w[i]));
    }
  }
  row_reduce<NT, true>(sum, top, 0);
  const float r = p.weight ? rsqrtf(sum / static_cast<float>(p.d) + p.eps) : 1.0f;
  float f = 1.0f;
  if constexpr (sizeof(O) == 1) {
    const float most = code_top(top * r);
    f = kCodeMax<O> * (1.0f / most);
    if (threadIdx.x == 0) p.scale[row] = most / kCodeMax<O>;
  }
  for (int c = threadIdx.x * 8; c < p.d; c += NT * 8) {
    float v[8], u[8], w[8];
    load8<TAIL>(x, c, p.d, v);
    if (res) {
      load8<TAIL>(res, c, p.d, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += u[i];
      store8(static_cast<T *>(p.h) + row * p.h_ld + c, p.d - c, v);
    }
    load_weight8<TAIL>(p, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = v[i] * r * w[i];
      if constexpr (sizeof(O) == 1) v[i] *= f;
    }
    store8(static_cast<O *>(p.y) + row * p.y_ld + c, p.d - c, v);
  }
}

// Rows a gradient workgroup takes at a time.  More rows leave fewer shares to add
// up, but go in step: 777 x 1111 in float32 18.3 us a call with one, 13.7 with two
// (shares' sum 9 to 5); 8192 x 4096 in bfloat16, where the rows' time counts, 60 us
// with one of 256 threads, 71 with two.
constexpr int grad_rows(int nt, int ch) { return nt == 64 ? 4 : ch == 1 ? 2 : 1; }

// A workgroup alone: its share is the sum.
__device__ __forceinline__ void store_weight8(const NormGradParams &p, int c, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < p.d) store_as(p.dw, p.weight_type, c + i, v[i]);
}

// 8 elements of the norm's input, in T or kept in 8 bits (8192 x 4096 bfloat16 with dh 40 us against 51 in 16 bits).
template <bool KEPT, Length L, typename T>
__device__ __forceinline__ void load_h8(const NormGradParams &p, const Kept &kept, long row, int c, float (&v)[8]) {
  if constexpr (KEPT) load_kept8<T>(kept, row, c, v);
  else load8<L>(static_cast<const T *>(p.h) + row * p.h_ld, c, p.d, v);
}

// The gradient's dx, and this workgroup's rows' share of dw, kept in registers over
// its rows.  The shares are added by share_sum_kernel, in a fixed order.  Bound by
// memory: 8192 x 4096 bfloat16 with dh 57 us, 51 and 5 for the sum (268 MB, 5.2 TB/s
// in the first); 777 x 1111 float32 13 us: a workgroup's load, reduction
// and stores one after the other 7, the sum's launch 4, the gap between them.
template <typename T, int NT, int CH, Length L, bool KEPT>
__global__ __launch_bounds__(NT *grad_rows(NT, CH)) void rms_norm_grad_kernel(NormGradParams p) {
  constexpr int RPB = grad_rows(NT, CH), THREADS = NT * RPB;
  const Kept kept = kept_at(p.h, p.rows, p.d);
  const int t = threadIdx.x % NT, sub = threadIdx.x / NT;
  const NormParams wp{.weight = p.weight, .d = p.d, .weight_type = p.weight_type};
  float w[CH][8], dw[CH][8];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    load_weight8<L>(wp, (j * NT + t) * 8, w[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.0f;
  }
  int turn = 0;
  // All of a workgroup's threads go through equally many rows (the barrier); one
  // past the end repeats the last and leaves nothing.
  const long step = static_cast<long>(gridDim.x) * RPB;
  for (long row0 = static_cast<long>(blockIdx.x) * RPB; row0 < p.rows; row0 += step) {
    const bool past = row0 + sub >= p.rows;
    const long row = past ? p.rows - 1 : row0 + sub;
    float h[CH][8], g[CH][8];
    KeptCodes codes[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if constexpr (KEPT) codes[j] = load_codes8(kept, row, (j * NT + t) * 8);
      else load8<L>(static_cast<const T *>(p.h) + row * p.h_ld, (j * NT + t) * 8, p.d, h[j]);
    }
#pragma unroll
    for (int j = 0; j < CH; ++j)
      load8<L>(static_cast<const T *>(p.dy) + row * p.dy_ld, (j * NT + t) * 8, p.d, g[j]);
    if constexpr (KEPT) {
#pragma unroll
      for (int j = 0; j < CH; ++j) restore8<T>(codes[j], h[j]);
    }
    float sum = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = __builtin_fmaf(h[j][i], h[j][i], sum);
        dot = __builtin_fmaf(g[j][i] * w[j][i], h[j][i], dot);
      }
    row_reduce<NT, false, RPB>(sum, dot, turn);
    turn ^= 1;
    if (past) continue;
    const float r = rsqrtf(sum / static_cast<float>(p.d) + p.eps);
    const float c = dot * r * r / static_cast<float>(p.d);  // xhat*mean(g*xhat) = h*c
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int at = (j * NT + t) * 8;
      float v[8], u[8];
      if (p.dh) load8<L>(static_cast<const T *>(p.dh) + row * p.dh_ld, at, p.d, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = r * __builtin_fmaf(-c, h[j][i], g[j][i] * w[j][i]);
        if (p.dh) v[i] += u[i];
        dw[j][i] = __builtin_fmaf(g[j][i] * r, h[j][i], dw[j][i]);
      }
      store8(static_cast<T *>(p.dx) + row * p.dx_ld + at, p.d - at, v);
    }
  }
  float *share = p.shares + static_cast<long>(blockIdx.x) * p.d;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = (j * NT + t) * 8;
      if (p.shares) store8(share + c, p.d - c, dw[j]);
      else store_weight8(p, c, dw[j]);
    }
  } else {
    // The rows' sums meet in LDS: one share a workgroup.
    __shared__ float part[RPB][NT * CH * 8];
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) part[sub][(j * 8 + i) * NT + t] = dw[j][i];
    __syncthreads();
    for (int e = threadIdx.x; e < NT * CH * 8; e += THREADS) {
      const int at = ((e / NT / 8) * NT + e % NT) * 8 + e / NT % 8;
      float s = part[0][e];
#pragma unroll
      for (int q = 1; q < RPB; ++q) s += part[q][e];
      if (at >= p.d) continue;
      if (p.shares) share[at] = s;
      else store_as(p.dw, p.weight_type, at, s);
    }
  }
}

// Rows longer than a workgroup's registers hold.  Workgroups own fixed rows; a
// share of dw is added up in place, in memory, by the threads that own its columns: more
// bytes than the rows themselves.  4096 x 32768 bfloat16 653 us (1.2 TB/s of the rows' bytes).
template <typename T, bool KEPT>
__global__ __launch_bounds__(256) void rms_norm_grad_long_kernel(NormGradParams p) {
  constexpr int NT = 256;
  const Kept kept = kept_at(p.h, p.rows, p.d);
  const NormParams wp{.weight = p.weight, .d = p.d, .weight_type = p.weight_type};
  float *share = p.shares + static_cast<long>(blockIdx.x) * p.d;
  int turn = 0;
  bool first = true;
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T *gp = static_cast<const T *>(p.dy) + row * p.dy_ld;
    float sum = 0.0f, dot = 0.0f;
    for (int c = threadIdx.x * 8; c < p.d; c += NT * 8) {
      float h[8], g[8], w[8];
      load_h8<KEPT, TAIL, T>(p, kept, row, c, h);
      load8<TAIL>(gp, c, p.d, g);
      load_weight8<TAIL>(wp, c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = __builtin_fmaf(h[i], h[i], sum);
        dot = __builtin_fmaf(g[i] * w[i], h[i], dot);
      }
    }
    row_reduce<NT, false>(sum, dot, turn);
    turn ^= 1;
    const float r = rsqrtf(sum / static_cast<float>(p.d) + p.eps);
    const float k = dot * r * r / static_cast<float>(p.d);
    for (int c = threadIdx.x * 8; c < p.d; c += NT * 8) {
      float h[8], g[8], w[8], u[8], s[8];
      load_h8<KEPT, TAIL, T>(p, kept, row, c, h);
      load8<TAIL>(gp, c, p.d, g);
      load_weight8<TAIL>(wp, c, w);
      if (p.dh) load8<TAIL>(static_cast<const T *>(p.dh) + row * p.dh_ld, c, p.d, u);
      if (!first) load8<TAIL>(share, c, p.d, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] = __builtin_fmaf(g[i] * r, h[i], first ? 0.0f : s[i]);
        const float v = r * __builtin_fmaf(-k, h[i], g[i] * w[i]);
        g[i] = p.dh ? v + u[i] : v;
      }
      store8(static_cast<T *>(p.dx) + row * p.dx_ld + c, p.d - c, g);
      store8(share + c, p.d - c, s);
    }
    first = false;
  }
}

__global__ __launch_bounds__(256) void share_sum_kernel(const float *shares, int count, int d, void *out, int type) {
  __shared__ float part[64][17];
  share_sum(shares, count, d, out, type, static_cast<int>(block_of()), part);
}

// Workgroups beyond this many would each take few rows for the weights they load.
constexpr long kNormGroups = 2048;

// The register kernels hold up to 64 elements a thread.
constexpr int kLongest = 16384;

unsigned wave_groups(long rows) { return static_cast<unsigned>(std::min<long>((rows + 3) / 4, kNormGroups)); }

int pieces(long d) { return static_cast<int>((d + 7) / 8); }

template <typename T, typename O, Length L>
void norm_launch_as(const NormParams &p, hipStream_t stream) {
  const int n = pieces(p.d);
  const dim3 waves(wave_groups(p.rows));
  const dim3 groups(static_cast<unsigned>(std::min<long>(p.rows, kNormGroups)));
  if (n <= 64) rms_norm_kernel<T, O, 64, 1, L><<<waves, 256, 0, stream>>>(p);
  else if (n <= 128) rms_norm_kernel<T, O, 64, 2, L><<<waves, 256, 0, stream>>>(p);
  else if (n <= 256) rms_norm_kernel<T, O, 256, 1, L><<<groups, 256, 0, stream>>>(p);
  else if (n <= 512) rms_norm_kernel<T, O, 256, 2, L><<<groups, 256, 0, stream>>>(p);
  else if (n <= 1024) rms_norm_kernel<T, O, 256, 4, L><<<groups, 256, 0, stream>>>(p);
  else rms_norm_kernel<T, O, 256, 8, L><<<groups, 256, 0, stream>>>(p);
}

// A launch takes fewer than 2^32 threads.  Long rows come one a workgroup: 2^24 of them
// would be 512 GB.  Rows under 8 elements take a wave each, of the same bounded number: one
// a workgroup took 979 us for 1048576 x 4 bfloat16, this way 187 (and its gradient 791, 7535 so).
template <typename T, typename O>
void norm_launch(const NormParams &p, hipStream_t stream) {
  if (p.d > kLongest) rms_norm_long_kernel<T, O><<<dim3(static_cast<unsigned>(p.rows)), 256, 0, stream>>>(p);
  else if (p.d < 8) rms_norm_kernel<T, O, 64, 1, ANY><<<dim3(wave_groups(p.rows)), 256, 0, stream>>>(p);
  else if (p.d % 8 == 0) norm_launch_as<T, O, WHOLE>(p, stream);
  else norm_launch_as<T, O, TAIL>(p, stream);
}

template <typename T, Length L, bool KEPT>
void norm_grad_launch_as(const NormGradParams &p, dim3 grid, hipStream_t stream) {
  const int n = pieces(p.d);
  if (n <= 64) rms_norm_grad_kernel<T, 64, 1, L, KEPT><<<grid, 64 * grad_rows(64, 1), 0, stream>>>(p);
  else if (n <= 128) rms_norm_grad_kernel<T, 64, 2, L, KEPT><<<grid, 64 * grad_rows(64, 2), 0, stream>>>(p);
  else if (n <= 256) rms_norm_grad_kernel<T, 256, 1, L, KEPT><<<grid, 256 * grad_rows(256, 1), 0, stream>>>(p);
  else if (n <= 512) rms_norm_grad_kernel<T, 256, 2, L, KEPT><<<grid, 256 * grad_rows(256, 2), 0, stream>>>(p);
  else if (n <= 1024) rms_norm_grad_kernel<T, 256, 4, L, KEPT><<<grid, 256 * grad_rows(256, 4), 0, stream>>>(p);
  else rms_norm_grad_kernel<T, 256, 8, L, KEPT><<<grid, 256 * grad_rows(256, 8), 0, stream>>>(p);
}

template <typename T, bool KEPT>
hipError_t norm_grad_launch(NormGradParams p, hipStream_t stream) {
  const long shares = norm_grad_shares(p.rows, p.d);
  if (shares == 1 && p.d <= kLongest) p.shares = nullptr;
  const dim3 grid(static_cast<unsigned>(shares));
  if (shares) {
    if (p.d > kLongest) rms_norm_grad_long_kernel<T, KEPT><<<grid, 256, 0, stream>>>(p);
    else if (p.d < 8) rms_norm_grad_kernel<T, 64, 1, ANY, KEPT><<<grid, 64 * grad_rows(64, 1), 0, stream>>>(p);
    else if (p.d % 8 == 0) norm_grad_launch_as<T, WHOLE, KEPT>(p, grid, stream);
    else norm_grad_launch_as<T, TAIL, KEPT>(p, grid, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.shares) return e;
  }
  return launch_share_sum(p.shares, shares, p.d, p.dw, p.weight_type, stream);
}

}  // namespace

// Workgroups, each with a share of the weight's gradient: as many as are on the GPU
// at once, and a quarter less where that is 1024, for fewer shares to add.  us a call,
// bfloat16, with 512 / 768 / 1024: 8192 x 4096 65.5 / 57.8 / 60.8; 8192 x 8192 83.9 / - /
// 91.8 (256: 100); 4096 x 16384 107 / - / 130 (256: 98).  Few rows go to one workgroup,
// up to `steps` after each other, whose share is the sum: no second launch (16 x 287 8.7 us a call
// with it, 6.0 without; 2 x 4032 8.8 and 6.1).
long norm_grad_shares(long rows, long d) {
  const int n = pieces(d);
  const long at_a_time = n > 256 ? 1 : n <= 128 ? 4 : 2;  // grad_rows of the kernel that runs
  const long steps = n <= 256 ? 5 : n <= 512 ? 4 : n <= 1024 ? 2 : 1;
  if (d <= kLongest && rows <= steps * at_a_time) return rows > 0;
  const long most = n <= 256 ? 512 : n <= 512 ? 768 : n <= 1024 ? 512 : 256;
  return std::min<long>((rows + at_a_time - 1) / at_a_time, most);
}

hipError_t launch_share_sum(const float *shares, long count, int d, void *out, int type, hipStream_t stream) {
  share_sum_kernel<<<grid_of((d + 15L) / 16, 256), 256, 0, stream>>>(shares, static_cast<int>(count), d, out, type);
  return hipGetLastError();
}

template <typename T>
hipError_t norm_launch_to(const NormParams &p, int y_type, hipStream_t stream) {
  if (y_type == TYPE_F8) norm_launch<T, f8>(p, stream);
  else if (y_type == TYPE_I8) norm_launch<T, i8>(p, stream);
  else norm_launch<T, T>(p, stream);
  return hipGetLastError();
}

hipError_t launch_rms_norm(const NormParams &p, int type, int y_type, hipStream_t stream) {
  if (type == TYPE_F32) return norm_launch_to<float>(p, y_type, stream);
  return type == TYPE_BF16 ? norm_launch_to<bf16>(p, y_type, stream) : norm_launch_to<f16>(p, y_type, stream);
}

template <bool KEPT>
hipError_t norm_grad_launch_of(const NormGradParams &p, int type, hipStream_t stream) {
  if (type == TYPE_F32) return norm_grad_launch<float, KEPT>(p, stream);
  return type == TYPE_BF16 ? norm_grad_launch<bf16, KEPT>(p, stream) : norm_grad_launch<f16, KEPT>(p, stream);
}

hipError_t launch_rms_norm_grad(const NormGradParams &p, int type, hipStream_t stream) {
  return p.kept ? norm_grad_launch_of<true>(p, type, stream) : norm_grad_launch_of<false>(p, type, stream);
}

}  // namespace tfnn
