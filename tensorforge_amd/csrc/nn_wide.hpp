// The 256 x 256 tile of the large products.
//
// Eight waves, two to a SIMD, each 128 x 64 of C (eight by four 16 x 16 blocks).  A slab
// (128 bytes of k a row) takes a wave two phases: its columns and its first 64
// rows, then its other 64 rows; in each it reads its fragments from LDS and then
// multiplies (32 matrix instructions, 512 cycles).  The waves are two groups,
// half a phase apart, one on each SIMD's either side: while one multiplies, the
// other reads.  Barriers keep the turns.
//
// Loads go straight into LDS, a few between the matrix instructions, each part of
// a slab into the place of the same part two slabs before as soon as both groups
// have read that: they have four turns (about 2000 cycles) to arrive.
//
// One workgroup fills a CU's registers and 128 of its 160 KiB of LDS.  Bound by the
// matrix cores at the clock that the power limit leaves: 8192^3 bfloat16 750 us (1466
// TFLOP/s; a loop of nothing but these instructions runs at 2070), 8 bits 2940
// TFLOP/s, 4096^3 101 us (1361); with fewer tiles than CUs the smaller tiles win.
// 16 x 16 blocks draw less power than 32 x 32 ones (loop alone 2070 against 1850).
#pragma once

#include "nn_gemm.hpp"

namespace tfnn {

// Loads one operand's slabs of 256 rows by 1 KiB pieces (nn_gemm.hpp's layout).
// PARTS 2: rows 0-63 and 128-191, then the others.  Each wave loads PER pieces of
// a part.
template <typename T, bool MN, int PARTS>
struct WideLoader {
  static constexpr int PER = 4 / PARTS;
  const char *base;
  long step;
  int k_size;
  uint32_t offset[PARTS][PER];

  static __device__ __forceinline__ int piece(int wave, int part, int i) {
    const int u = wave * PER + i;
    return PARTS == 2 ? (u / 8 * 2 + part) * 8 + u % 8 : u;
  }
  static __device__ __forceinline__ void place(int part, int i, int &row, int &k) {
    const int lane = threadIdx.x % 64, t = piece(threadIdx.x / 64, part, i);
    if constexpr (!MN) {
      row = t * 8 + lane / 8;
      k = ((lane % 8) ^ (lane / 8)) * kPiece<T>;
    } else {
      k = t % 8 * 8 + lane / 8;
      row = t / 8 * 64 + ((lane % 8) ^ line_turn(k)) * kPiece<T>;
    }
  }
  __device__ __forceinline__ void init(const void *matrix, long ld, int own, int own0, int k0, int k1) {
    constexpr long E = sizeof(T);
    ld *= E;
    base = static_cast<const char *>(matrix) + (MN ? k0 * ld + own0 * E : own0 * ld + k0 * E);
    step = MN ? kSlab<T> * ld : 128;
    k_size = k1 - k0;
#pragma unroll
    for (int q = 0; q < PARTS; ++q)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        int row, k;
        place(q, i, row, k);
        offset[q][i] = row < own - own0 ? static_cast<uint32_t>(MN ? k * ld + row * E : row * ld + k * E) : kNowhere;
      }
  }
  // Before a part's loads of slab s, in order of s.  The last slab may be partial:
  // what lies past k becomes zeros.
  __device__ __forceinline__ void enter(int s, int part) {
    const int left = k_size - s * kSlab<T>;
    if (left > 0 && left < kSlab<T>) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        int row, k;
        place(part, i, row, k);
        if (k >= left) offset[part][i] = kNowhere;
      }
    }
  }
  // Slab s's resource: empty past the last one, where loads give zeros and touch
  // no memory (so that every slab has the same loads to wait for).
  __device__ __forceinline__ i32x4 resource(int s) const {
    return buffer_resource(base + s * step, s * kSlab<T> < k_size ? kResourceBytes : 0);
  }
  __device__ __forceinline__ void issue(i32x4 res, int wave, int part, int i, uint32_t lds) const {
    load_to_lds(res, offset[part][i], lds + piece(wave, part, i) * 1024);
  }
};

constexpr int kWideLds = 2 * 2 * 256 * 128;
template <typename T, typename O, bool AMN, bool BMN, typename E = Results>
__device__ __forceinline__ void gemm_wide(const typename E::Params &p, lds_char *lds) {
  constexpr int STAGE = 2 * 256 * 128, HALF = 256 * 128;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wm = wave / 4, wn = wave % 4;
  int tm, tn, split;
  tile_of(p, blockIdx.x, gridDim.x, tm, tn, split);
  const int slabs = (p.k + kSlab<T> - 1) / kSlab<T>;
  const int s0 = static_cast<int>(static_cast<long>(slabs) * split / p.splits);
  const int count = static_cast<int>(static_cast<long>(slabs) * (split + 1) / p.splits) - s0;
  const int k0 = s0 * kSlab<T>, k1 = min(p.k, k0 + count * kSlab<T>);
  WideLoader<T, AMN, 2> la;
  WideLoader<T, BMN, 1> lb;
  la.init(p.a, p.lda, p.m, tm * 256, k0, k1);
  lb.init(p.b, p.ldb, p.n, tn * 256, k0, k1);
  FragReader<AMN> fa;
  FragReader<BMN> fb;
  fa.init(wm * 128);
  fb.init(wn * 64);
  sums4<T> acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = sums4<T>{0, 0, 0, 0};

  // Slabs 0 and 1, but for slab 1's second half of A, which the first phase loads.
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const i32x4 ra = la.resource(s), rb = lb.resource(s);
    lb.enter(s, 0);
    la.enter(s, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) lb.issue(rb, wave, 0, i, lds0 + s * STAGE + HALF);
#pragma unroll
    for (int i = 0; i < 2; ++i) la.issue(ra, wave, 0, i, lds0 + s * STAGE);
    if (s == 0) {
      la.enter(0, 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) la.issue(ra, wave, 1, i, lds0);
    }
  }
  wait_loads<6>();
  barrier();
  if (wm == 1) barrier();  // the second group: half a phase behind

  i32x4 a[4][2], b[4][2];
  for (int s = 0; s < count; ++s) {
    lds_char *slab = lds + (s & 1) * STAGE;
    unroll<2>([&](auto h) {
      // Fragments.
      if constexpr (h == 0) unroll<4>([&](auto j) {
        b[j][0] = fb.template read<16 * j, 0>(slab + HALF);
        b[j][1] = fb.template read<16 * j, 1>(slab + HALF);
      });
      unroll<4>([&](auto i) {
        a[i][0] = fa.template read<64 * h + 16 * i, 0>(slab);
        a[i][1] = fa.template read<64 * h + 16 * i, 1>(slab);
      });
      // What the first group reads in its next turn has arrived: the loads that
      // this wave issued four (the first group) or three turns ago.
      if (wm == 1) {
        if constexpr (h == 0) wait_loads<6>();
        else wait_loads<2>();
      }
      // Phase 0 loads the second half of A of slab s + 1, phase 1 the columns and
      // the first half of A of slab s + 2: places that both groups have read.
      const int to = h == 0 ? s + 1 : s + 2;
      const uint32_t place = lds0 + (to & 1) * STAGE;
      const i32x4 ra = la.resource(to), rb = lb.resource(to);
      la.enter(to, h == 0);
      if constexpr (h == 1) lb.enter(to, 0);
      wait_lds();
      __builtin_amdgcn_sched_barrier(0);
      barrier();
      __builtin_amdgcn_s_setprio(1);
      unroll<16>([&](auto ij) {
        constexpr int i = ij / 4, j = ij % 4;
        acc[4 * h + i][j] = block_mma(T{}, a[i][0], a[i][1], b[j][0], b[j][1], acc[4 * h + i][j]);
        if constexpr (h == 0) {
          if constexpr (ij % 4 == 1 && ij / 4 < 2) la.issue(ra, wave, 1, ij / 4, place);
        } else {
          if constexpr (ij % 2 == 1 && ij / 2 < 4) lb.issue(rb, wave, 0, ij / 2, place + HALF);
          if constexpr (ij % 2 == 1 && ij / 2 >= 4 && ij / 2 < 6) la.issue(ra, wave, 0, ij / 2 - 4, place);
        }
      });
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      if (wm == 0) wait_loads<8>();
      barrier();
    });
  }
  if (wm == 0) barrier();
  wait_loads<0>();  // the empty ones past the end
  barrier();
  // Through LDS (nn_gemm.hpp), 64 rows at a time.  Results of this size stream past
  // the caches: 8192^3 in bfloat16 1389 TFLOP/s without that, 1423 with it.
  lds_char *patch = lds + wave * (64 * 64 * 4);
  if constexpr (__is_same(E, Results)) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<__attribute__((address_space(3))) sums4<T> *>(patch + patch_at<64>(i * 16 + lane % 16, j * 4 + lane / 16)) =
              acc[4 * h + i][j];
      wait_lds();
      write_patch<T, O, 64, 64, true>(p, split, patch, tm * 256 + wm * 128 + h * 64, tn * 256 + wn * 64, 0, 0);
    }
  } else {
    E::template finish<T, 256, 256, 2, 4, 64>(p, acc, split, lds, patch, tm * 256, tn * 256, wm, wn, tm, tn);
  }
}

template <typename T, typename O, bool AMN, bool BMN>
__global__ __launch_bounds__(512, 2) void gemm_wide_kernel(GemmParams p) {
  __shared__ __align__(1024) char smem[kWideLds];
  gemm_wide<T, O, AMN, BMN>(p, (lds_char *)smem);
}

}  // namespace tfnn
