// The loss over a vocabulary and its gradient: what they need beside the products
// (nn_xent_gemm.hpp), and their calls of the C ABI.
//
//   z = x @ w    lse[m] = log(sum over n of exp(z[m][n]))    loss[m] = lse[m] - z[m][target[m]]
//   dz[m][n] = (exp(z[m][n] - lse[m]) - [n = target[m]]) * dloss[m]    dx = dz @ w^T    dw = x^T @ dz
//
// The loss is one product whose logits never leave the accumulators.  The gradient takes the
// vocabulary piece by piece: the logits again, their gradient in 16 bits, and the two products with
// it; dx is added up over the pieces in float32.
#include "nn_plan.hpp"
#include "nn_xent_gemm.hpp"

using namespace tfnn;

namespace {

struct RowsParams {
  const float *stats, *target_logit;
  const long long *target;
  long long ignore;
  double *lse;
  float *loss, *sum, *mean, *count;
  int m, n, parts;
};

// The sum of a workgroup's 1024 values in a fixed order.
template <typename S>
__device__ __forceinline__ S group_sum(S v, S *part) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
  __syncthreads();
  S s = 0;
  for (int i = 0; i < 16; ++i) s += part[i];
  return s;
}

__device__ __forceinline__ void write_totals(const RowsParams &p, double sum, double count) {
  if (threadIdx.x) return;
  if (p.sum) *p.sum = static_cast<float>(sum);
  if (p.count) *p.count = static_cast<float>(count);
  if (p.mean) *p.mean = count > 0.0 ? static_cast<float>(sum / count) : 0.0f;
}

// R rows a workgroup, 1024/R threads a row that share the parts, kBatch of them under way at a
// time.  One workgroup of all rows adds up the losses too.  Bound by latency: 16 rows of 500 parts
// 4.2 us.
template <int R>
__global__ __launch_bounds__(1024) void xent_rows_kernel(RowsParams p) {
  constexpr int LANES = 1024 / R, kBatch = 8;
  __shared__ f32x2 part[LANES][R];
  __shared__ float sums[16];
  const int r = threadIdx.x % R, lane = threadIdx.x / R;
  const long m = block_of() * R + r;
  const f32x2 none = {-__builtin_inff(), 0.0f};
  f32x2 s = none;
  if (m < p.m) {
    const f32x2 *from = reinterpret_cast<const f32x2 *>(p.stats) + m;
    for (int q = lane; q < p.parts; q += LANES * kBatch) {
      f32x2 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int at = q + i * LANES;
        v[i] = from[static_cast<long>(min(at, p.parts - 1)) * p.m];
        if (at >= p.parts) v[i] = none;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) s = joined(s, v[i]);
    }
  }
  part[lane][r] = s;
  __syncthreads();
#pragma unroll
  for (int left = LANES / 4; left >= 1; left /= 4) {  // 4 to 1, in lane order
    if (lane < left) {
#pragma unroll
      for (int i = 1; i < 4; ++i) s = joined(s, part[lane + i * left][r]);
      part[lane][r] = s;
    }
    __syncthreads();
  }
  float loss = 0.0f, counts = 0.0f;
  if (lane == 0 && m < p.m) {
    constexpr float kLn2 = 0.693147180559945309f;
    const float log_sum = log2f(s.y);
    const long long target = p.target[m];
    if (target != p.ignore) {
      counts = 1.0f;
      // Not lse - logit: large logits would leave their roundings where their difference is small.  A row without a
      // logit that counts has none.
      loss = target >= 0 && target < p.n && s.x != -__builtin_inff() ? (__builtin_fmaf(-p.target_logit[m], kLog2e, s.x) + log_sum) * kLn2 : __builtin_nanf("");
    }
    p.lse[m] = (static_cast<double>(s.x) + log_sum) / kLog2e;
    p.loss[m] = loss;
  }
  if (gridDim.x * gridDim.y == 1 && (p.sum || p.mean || p.count)) {
    loss = group_sum(loss, sums);
    counts = group_sum(counts, sums);
    write_totals(p, loss, counts);
  }
}
// 16 rows a workgroup (with 64: 64 x 32000 12.3 us against 9.6 with the product, 1024 x 32000 33.8 and 33.0), but 64 where
// that makes one workgroup of all and spares the totals' launch.
bool one_group(long m, bool totals) { return m <= 16 || (m <= 64 && totals); }

// Sums of up to 2^30 rows: in 64 bits.
__global__ __launch_bounds__(1024) void xent_totals_kernel(RowsParams p) {
  __shared__ double sums[16];
  double loss = 0.0, counts = 0.0;
  for (long m = threadIdx.x; m < p.m; m += 1024) {
    loss += p.loss[m];
    counts += p.target[m] != p.ignore;
  }
  loss = group_sum(loss, sums);
  counts = group_sum(counts, sums);
  write_totals(p, loss, counts);
}

// float16's gradient of the logits is taken in a unit that lets the largest reach 2^15: small probabilities
// would be lost below the type's smallest numbers.  With a dloss a row: the unit's inverse and the unit.
__global__ __launch_bounds__(1024) void xent_scale_kernel(XentParams p, float *scale) {
  __shared__ float part[16];
  float top = 0.0f;
  for (long m = threadIdx.x; m < p.m; m += 1024) {
    const float d = __builtin_fabsf(p.dloss[m]);
    if (p.target[m] != p.ignore && d < __builtin_inff()) top = __builtin_fmaxf(top, d);
  }
  top = wave_max(top);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; ++i) top = __builtin_fmaxf(top, part[i]);
  if (p.count) top /= *p.count;
  const int e = static_cast<int>(__builtin_bit_cast(uint32_t, top) >> 23 & 255) - 127;  // top below 2^(e + 1)
  const int up = top > 0.0f && top < __builtin_inff() ? max(-100, min(14 - e, 100)) : 0;
  scale[0] = __builtin_bit_cast(float, static_cast<uint32_t>(127 + up) << 23);
  scale[1] = __builtin_bit_cast(float, static_cast<uint32_t>(127 - up) << 23);
}

// Sum's epilogue for a product in ranges of k, or of both terms of dz; four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void xent_join_kernel(XentParams p) {
  const int rows = p.halves ? p.m / 2 : p.m;
  const long quads = (p.n + 3L) / 4, id = block_of() * 256 + threadIdx.x, ld = quads * 4, m = id / quads, n = id % quads * 4;
  if (m >= rows) return;
  const auto added = [&](long row) {
    const float *part = p.parts + row * ld + n;
    f32x4 v = *reinterpret_cast<const f32x4 *>(part);
#pragma unroll 4
    for (int s = 1; s < p.splits; ++s) v += *reinterpret_cast<const f32x4 *>(part + s * (p.m * ld));
    return v;
  };
  f32x4 v = added(m);
  if (p.halves) v += made_finite(added(rows + m));  // as in gemm_tile
  f32x4 *sum = reinterpret_cast<f32x4 *>(p.sum + m * ld + n);
  if (p.add) v += *sum;
  if (!p.last) {
    *sum = v;
    return;
  }
  const float unit = sum_unit(p);
  T *out = static_cast<T *>(p.out) + m * p.ldo + n;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.n) out[i] = static_cast<T>(in_unit(v[i], unit));
}

// The weights' gradient of up to 64 rows of x: out[r][c] = sum over m of R[m][r] * C[m][c], one of
// both (dz) in two terms.  Bound by writing it.  A workgroup keeps COLUMNS columns of C as fragments in
// LDS and its waves go down the rows, 16 at a time, R's fragments gathered as they lie (both
// operands are small and come from the caches).  2 x 59648 x 3436 bfloat16 114 us (410 MB written, 3.6
// TB/s) where 64 x 64 tiles took 421, 16 x 32000 x 4096 67 (121 on 128 x 128 tiles).
struct OuterParams {
  const void *r, *c;
  long r_ld, c_ld, lo;  // lo: the second term's elements behind dz's
  int k, rows, columns; // k: x's rows
};
template <typename T, bool TWO_R, int KS, int COLUMNS>
__global__ __launch_bounds__(256) void xent_outer_kernel(OuterParams q, XentParams p) {
  constexpr int BLOCKS = COLUMNS / 16, TC = TWO_R ? 1 : 2, TR = TWO_R ? 2 : 1;
  __shared__ __align__(1024) char smem[BLOCKS * KS * TC * 1024 + 4 * 4096];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, l = lane % 16, g = lane / 16;
  lds_char *frags = (lds_char *)smem, *patch = frags + BLOCKS * KS * TC * 1024 + wave * 4096;
  // Eight rows of x from 32 * ks + 8 * g on, of one column of its operand.
  const auto gather = [&](const T *from, long ld, int ks) {
    typename Vec<T, 8>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = ks * 32 + g * 8 + i;
      const T e = from[min(m, q.k - 1) * ld];
      v[i] = m < q.k ? e : static_cast<T>(0.0f);
    }
    return __builtin_bit_cast(i32x4, v);
  };
  const auto multiply = [&](const i32x4 (&a)[KS], const lds_char *at, f32x4 c) {
    const i32x4 none = {0, 0, 0, 0};
    return block_mma(T{}, a[0], KS > 1 ? a[KS - 1] : none, lds_read16(at), KS > 1 ? lds_read16(at + (KS - 1) * 1024) : none, c);
  };
  const int c0 = blockIdx.x * COLUMNS;
  for (int f = wave; f < BLOCKS * TC * KS; f += 4) {
    const int ks = f % KS, term = f / KS % TC, block = f / KS / TC;
    const T *from = static_cast<const T *>(q.c) + term * q.lo + min(c0 + block * 16 + l, q.columns - 1);
    *reinterpret_cast<__attribute__((address_space(3))) i32x4 *>(frags + f * 1024 + lane * 16) = gather(from, q.c_ld, ks);
  }
  __syncthreads();
  const float unit = sum_unit(p);
  const lds_char *mine = frags + lane * 16;
  for (int r0 = (blockIdx.y * 4 + wave) * 16; r0 < q.rows; r0 += gridDim.y * 64) {
    i32x4 a[TR][KS];
#pragma unroll
    for (int t = 0; t < TR; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) a[t][ks] = gather(static_cast<const T *>(q.r) + t * q.lo + min(r0 + l, q.rows - 1), q.r_ld, ks);
    for (int b = 0; b < BLOCKS; b += 4) {
      if (c0 + b * 16 >= q.columns) break;
      f32x4 acc[1][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const lds_char *at = mine + (b + j) * (TC * KS * 1024);
        // What the rounding left first, as in gemm_tile.
        acc[0][j] = made_finite(multiply(a[TR - 1], at + (TC - 1) * KS * 1024, f32x4{0.0f, 0.0f, 0.0f, 0.0f}));
        acc[0][j] = multiply(a[0], at, acc[0][j]);
      }
      by_rows<16>(acc, patch, [&](int row, int column, float (&v)[8]) {
        const int r = r0 + row, c = c0 + b * 16 + column, left = q.columns - c;
        if (r >= q.rows || left <= 0) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = in_unit(v[i], unit);
        store_some(static_cast<T *>(p.out) + r * p.ldo + c, left, v);
      });
    }
  }
}

template <typename T, bool TWO_R, int COLUMNS>
void launch_outer_as(const OuterParams &q, const XentParams &p, hipStream_t stream) {
  // As many workgroups down the rows as make four for each CU.  Of 64 columns they are there at once; of 256 their LDS (16 KB
  // and 16 KB for each 32 rows of x and term of C) lets 2 to 5 be, and the others follow.
  const long across = (q.columns + COLUMNS - 1L) / COLUMNS, down = std::max(1L, std::min((1024 + across - 1) / across, (q.rows + 63L) / 64));
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(down));
  if (q.k <= 32) xent_outer_kernel<T, TWO_R, 1, COLUMNS><<<grid, 256, 0, stream>>>(q, p);
  else xent_outer_kernel<T, TWO_R, 2, COLUMNS><<<grid, 256, 0, stream>>>(q, p);
}
// 256 columns a workgroup, or 64 where that leaves CUs without one: 61 x 1001 x 333 float16 12.0 us with 256.
template <typename T, bool TWO_R>
void launch_outer(const OuterParams &q, const XentParams &p, hipStream_t stream) {
  const bool few = ((q.columns + 255L) / 256) * ((q.rows + 63L) / 64) < 256;
  few ? launch_outer_as<T, TWO_R, 64>(q, p, stream) : launch_outer_as<T, TWO_R, 256>(q, p, stream);
}

hipError_t launch_product(const XentParams &p, int type, XentProduct what, bool amn, bool bmn, const Choice &c, hipStream_t stream) {
  return type == TF_T_BF16 ? launch_xent_bf16(p, what, amn, bmn, c.plan.tile, c.dma, stream)
                           : launch_xent_f16(p, what, amn, bmn, c.plan.tile, c.dma, stream);
}

// Puts a product's operands and plan into the kernels' parameters.
void place_xent(XentParams &p, Product &q, const Choice &c, void *parts) {
  place(q, c.plan, parts);
  static_cast<GemmParams &>(p) = q.p;
}

Product logits_of(const void *x, long x_ld, const void *w, long w_ld, int w_order, int type, long m, long n, long k) {
  Product q{type, type, {}, {}, {}, true, true};
  q.a = {x, x_ld, m, k, false, false};
  q.b = w_order ? Operand{w, w_ld, n, k, false, false} : Operand{w, w_ld, k, n, true, false};
  q.p.m = static_cast<int>(m), q.p.n = static_cast<int>(n), q.p.k = static_cast<int>(k);
  return q;
}

// ---- the loss -----------------------------------------------------------------

void check_sizes(Checks &c, int type, int w_order, long long m, long long n, long long k) {
  c.one_of("type", type, {TF_T_BF16, TF_T_F16});
  c.one_of("w_order", w_order, {0, 1});
  c.size("m", m);
  c.size("n", n);
  c.size("k", k);
  c.need(n != 0, "n = 0: no class");
  if (c.fine()) c.need(ceil_div(m, 64) * ceil_div(n, 64) < (1LL << 31), m, " rows of ", n, " classes are too many");
}

struct LossPlan {
  Product q;
  Choice c;
  long long stats = 0, target_logit = 0;  // bytes
  long long bytes() const { return stats + target_logit + c.copies; }
};

LossPlan plan_loss(const tf_linear_xent_args_t *a) {
  LossPlan l{};
  l.q = logits_of(a->x, a->x_ld, a->w, a->w_ld, a->w_order, a->type, a->m, a->n, a->k);
  if (!a->m) return l;
  l.c = choose(l.q, 0, 1);
  l.stats = round16(8 * ceil_div(a->n, tile_columns(l.c.plan.tile)) * a->m);
  l.target_logit = round16(4 * a->m);
  return l;
}

int loss_workspace(const tf_linear_xent_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_xent_workspace: null arguments");
  Checks c{"tf_linear_xent_workspace", {}};
  check_sizes(c, a->type, a->w_order, a->m, a->n, a->k);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  *bytes = plan_loss(a).bytes();
  return TF_OK;
}

int loss(const tf_linear_xent_args_t *a, hipStream_t stream) {
  const char *call = "tf_linear_xent";
  if (!a) return fail(TF_E_ARG, "tf_linear_xent: null arguments");
  Checks c{call, {}};
  check_sizes(c, a->type, a->w_order, a->m, a->n, a->k);
  c.matrix("x", a->x, a->x_ld, a->m, a->k, a->type, true);
  c.matrix("w", a->w, a->w_ld, a->m ? (a->w_order ? a->n : a->k) : 0, a->w_order ? a->k : a->n, a->type, true);
  if (a->m) c.need(a->target && reinterpret_cast<uintptr_t>(a->target) % 8 == 0, "target is null or not aligned");
  if (a->m) c.need(a->lse && reinterpret_cast<uintptr_t>(a->lse) % 8 == 0, "lse is null or not aligned");
  c.vector("loss", a->loss, a->m, TF_T_F32, true);
  c.vector("sum", a->sum, 1, TF_T_F32, false);
  c.vector("mean", a->mean, 1, TF_T_F32, false);
  c.vector("count", a->count, 1, TF_T_F32, false);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  LossPlan l = plan_loss(a);
  c.workspace(a->workspace, a->workspace_bytes, l.bytes());
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  const bool totals = a->sum || a->mean || a->count;
  char *ws = static_cast<char *>(a->workspace);
  RowsParams r{reinterpret_cast<float *>(ws), reinterpret_cast<float *>(ws + l.stats), a->target, a->ignore, a->lse, a->loss, a->sum, a->mean,
               a->count, static_cast<int>(a->m), static_cast<int>(a->n), 0};
  hipError_t e = hipSuccess;
  if (a->m) {
    PackParams pack;
    char *to = ws + l.stats + l.target_logit;
    if (l.c.pack_a) to += copy_of(l.q.a, 2, to, pack);
    if (l.c.pack_b) copy_of(l.q.b, 2, to, pack);
    if (pack.pieces[0]) e = launch_pack(pack, a->type, stream);
    XentParams p;
    place_xent(p, l.q, l.c, nullptr);
    p.target = a->target, p.vocabulary = static_cast<int>(a->n);
    p.stats = reinterpret_cast<float *>(ws), p.target_logit = reinterpret_cast<float *>(ws + l.stats);
    if (e == hipSuccess) e = launch_product(p, a->type, XENT_STATS, false, l.q.b.mn, l.c, stream);
    r.parts = p.tiles_n;
    if (e == hipSuccess) {
      if (a->m <= 16 || !one_group(a->m, totals)) xent_rows_kernel<16><<<grid_of((a->m + 15) / 16, 1024), 1024, 0, stream>>>(r);
      else xent_rows_kernel<64><<<grid_of((a->m + 63) / 64, 1024), 1024, 0, stream>>>(r);
      e = hipGetLastError();
    }
  }
  if (e == hipSuccess && totals && (a->m == 0 || !one_group(a->m, totals))) {
    xent_totals_kernel<<<1, 1024, 0, stream>>>(r);
    e = hipGetLastError();
  }
  return hip(e, call);
}

// ---- its gradient ---------------------------------------------------------------

// The vocabulary goes in pieces of equal width, multiples of 256, whose gradient of the logits takes up
// to kPieceBytes, but at least kLeastColumns wide: dx's sums are read and written once a piece.  us, bfloat16:
// 8192 x 65536 x 2048 in pieces of 64 / 128 / 512 MB 5711 / 5321 / 5374, 65536 x 65536 x 1024 in
// pieces of 4096 / 8192 / 16384 columns 23990 / 22980 / 22840.
constexpr long long kPieceBytes = 128 << 20;
constexpr long kLeastColumns = 8192;

// Up to so many rows the products take what dz's rounding left as a second term, into the same sums:
// they are bound by reading w and writing dw, and a class that few rows have would see dz's rounding
// in its dw (2 x 59648 x 3436 bfloat16: dw 0.0003 off 64 bits in one term, its own rounding 0.00018).
// dx takes the terms as so many rows more, which share one read of w, and dw has a kernel of its own.
constexpr long kTwoTermRows = 64;

struct GradPlan {
  int terms = 1;
  long width = 0, pieces = 0, dz_ld = 0;
  Operand x, w;                      // as they lie, or their aligned copies
  bool copy_x = false, copy_w = false;
  long long scale = 0, dz = 0, sum = 0, copies = 0, parts = 0;  // bytes
  long long bytes() const { return scale + dz + sum + copies + parts; }
};

struct Piece {
  Product z, dx, dw;
  Choice cz, cdx, cdw;
};

// The products of `n` columns; their operands' addresses are those of the first piece.
Piece piece_of(const GradPlan &g, const tf_linear_xent_grad_args_t *a, long n) {
  Piece s;
  const bool nk = a->w_order == 1;
  const int m = static_cast<int>(a->m), k = static_cast<int>(a->k);
  const auto w_as = [&](bool mn) {
    Operand o = g.w;
    (nk ? o.lines : o.length) = n;
    o.mn = mn;
    return o;
  };
  const auto x_as = [&](bool mn) {
    Operand o = g.x;
    o.mn = mn;
    return o;
  };
  const int rows = m * g.terms;  // of dz
  const auto dz_as = [&](bool mn) { return Operand{nullptr, g.dz_ld, mn ? m : rows, n, mn, true}; };
  s.z = {a->type, a->type, x_as(false), w_as(!nk), {}, true, true};
  s.z.p.m = m, s.z.p.n = static_cast<int>(n), s.z.p.k = k;
  s.dx = {a->type, a->type, dz_as(false), w_as(nk), {}, true};
  s.dx.p.m = rows, s.dx.p.n = k, s.dx.p.k = static_cast<int>(n);
  s.dw = {a->type, a->type, nk ? dz_as(true) : x_as(true), nk ? x_as(true) : dz_as(true), {}, true};
  s.dw.p.m = static_cast<int>(nk ? n : k), s.dw.p.n = static_cast<int>(nk ? k : n), s.dw.p.k = m;
  if (m) s.cz = choose(s.z, 0, 1, false), s.cdx = choose(s.dx, 0, 0, false);
  if (m && g.terms == 2) {
    s.cdx.parts = round16(4LL * s.cdx.plan.splits * rows * ((k + 3) & ~3L));
  } else {
    s.cdw = choose(s.dw, 0, 0, false);
  }
  return s;
}

GradPlan plan_grad(const tf_linear_xent_grad_args_t *a) {
  GradPlan g;
  const long m = a->m, n = a->n, k = a->k;
  if (!k) return g;
  const long most = std::max(kLeastColumns, static_cast<long>(kPieceBytes / (2 * std::max(1L, m))));
  g.pieces = ceil_div(n, most);
  g.width = std::min(n, ceil_div(ceil_div(n, g.pieces), 256) * 256);
  g.pieces = ceil_div(n, g.width);
  g.dz_ld = g.width <= 64 ? ceil_div(g.width, 8) * 8 : ceil_div(g.width, 64) * 64;
  const Product z = logits_of(a->x, a->x_ld, a->w, a->w_ld, a->w_order, a->type, m, n, k);
  g.x = z.a, g.w = z.b;
  if (m) {  // one copy serves all three products
    const Choice c = choose(z, 0, 1);
    g.copy_x = c.pack_a, g.copy_w = c.pack_b, g.copies = c.copies;
    if (g.copy_x) g.x.ld = packed_ld(g.x, 2), g.x.ours = true;
    if (g.copy_w) g.w.ld = packed_ld(g.w, 2), g.w.ours = true;
  }
  g.scale = a->type == TF_T_F16 && a->dloss_rows && m ? 16 : 0;
  g.terms = m && m <= kTwoTermRows ? 2 : 1;
  g.dz = round16(2 * m * g.dz_ld) * g.terms;
  g.sum = a->dx && g.pieces > 1 ? round16(4 * m * ((k + 3) & ~3L)) : 0;
  for (const long width : {g.width, n - (g.pieces - 1) * g.width}) {
    const Piece s = piece_of(g, a, width);
    g.parts = std::max({g.parts, a->dx ? s.cdx.parts : 0, a->dw ? s.cdw.parts : 0});
  }
  return g;
}

void check_grad_sizes(Checks &c, const tf_linear_xent_grad_args_t *a) {
  check_sizes(c, a->type, a->w_order, a->m, a->n, a->k);
}

int grad_workspace(const tf_linear_xent_grad_args_t *a, long long *bytes) {
  if (!a || !bytes) return fail(TF_E_ARG, "tf_linear_xent_grad_workspace: null arguments");
  Checks c{"tf_linear_xent_grad_workspace", {}};
  check_grad_sizes(c, a);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  *bytes = plan_grad(a).bytes();
  return TF_OK;
}

// One of the two products that add up, with its join.
hipError_t run_sum(XentParams p, Product &q, const Choice &c, int type, void *parts, hipStream_t stream) {
  place_xent(p, q, c, parts);
  hipError_t e = launch_product(p, type, XENT_SUM, q.a.mn, q.b.mn, c, stream);
  if (e != hipSuccess || (p.splits == 1 && !p.halves)) return e;
  const dim3 grid = grid_of(((p.halves ? p.m / 2 : p.m) * ((p.n + 3L) / 4) + 255) / 256, 256);
  type == TF_T_BF16 ? xent_join_kernel<bf16><<<grid, 256, 0, stream>>>(p) : xent_join_kernel<f16><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

int grad(const tf_linear_xent_grad_args_t *a, hipStream_t stream) {
  const char *call = "tf_linear_xent_grad";
  if (!a) return fail(TF_E_ARG, "tf_linear_xent_grad: null arguments");
  Checks c{call, {}};
  check_grad_sizes(c, a);
  const bool nk = a->w_order == 1;
  c.one_of("dloss_rows", a->dloss_rows, {0, 1});
  c.matrix("x", a->x, a->x_ld, a->m, a->k, a->type, true);
  c.matrix("w", a->w, a->w_ld, a->m ? (nk ? a->n : a->k) : 0, nk ? a->k : a->n, a->type, true);
  if (a->m) c.need(a->target && reinterpret_cast<uintptr_t>(a->target) % 8 == 0, "target is null or not aligned");
  if (a->m) c.need(a->lse && reinterpret_cast<uintptr_t>(a->lse) % 8 == 0, "lse is null or not aligned");
  c.vector("dloss", a->dloss, a->m ? (a->dloss_rows ? a->m : 1) : 0, TF_T_F32, true);
  c.vector("count", a->count, 1, TF_T_F32, false);
  c.matrix("dx", a->dx, a->dx_ld, a->m, a->k, a->type, false);
  c.matrix("dw", a->dw, a->dw_ld, nk ? a->n : a->k, nk ? a->k : a->n, a->type, false);
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  GradPlan g = plan_grad(a);
  c.workspace(a->workspace, a->workspace_bytes, g.bytes());
  if (!c.fine()) return fail(TF_E_ARG, c.wrong);
  if (!a->k || (!a->dx && !a->dw) || (!a->m && !a->dw)) return TF_OK;
  char *ws = static_cast<char *>(a->workspace);
  float *scale = g.scale ? reinterpret_cast<float *>(ws) : nullptr;
  char *const dz = ws + g.scale, *const sum = dz + g.dz, *const copies = sum + g.sum, *const parts = copies + g.copies;
  hipError_t e = hipSuccess;
  PackParams pack;
  if (g.copy_x || g.copy_w) {
    const Product z = logits_of(a->x, a->x_ld, a->w, a->w_ld, a->w_order, a->type, a->m, a->n, a->k);
    char *to = copies;
    if (g.copy_x) g.x = z.a, to += copy_of(g.x, 2, to, pack);
    if (g.copy_w) g.w = z.b, copy_of(g.w, 2, to, pack);
    e = launch_pack(pack, a->type, stream);
  }
  XentParams base;
  base.target = a->target, base.ignore = a->ignore, base.vocabulary = static_cast<int>(a->n);
  base.lse = a->lse, base.dloss = a->dloss, base.count = a->count, base.scale = scale;
  base.dloss_rows = a->m ? a->dloss_rows : 1;  // without rows dloss is not read
  base.power = a->type == TF_T_F16 ? 32768.0f : 1.0f;
  base.m = static_cast<int>(a->m);
  if (e == hipSuccess && scale) {
    xent_scale_kernel<<<1, 1024, 0, stream>>>(base, scale);
    e = hipGetLastError();
  }
  for (long i = 0; i < g.pieces && e == hipSuccess; ++i) {
    const long column0 = i * g.width, n = std::min<long>(g.width, a->n - column0);
    Piece s = piece_of(g, a, n);
    const auto from_column = [&](const void *w, long ld) { return static_cast<const char *>(w) + 2 * column0 * (nk ? ld : 1); };
    s.z.b.p = s.dx.b.p = from_column(g.w.p, g.w.ld);
    s.dx.a.p = (nk ? s.dw.a.p : s.dw.b.p) = dz;
    if (a->m) {
      XentParams p = base;
      place_xent(p, s.z, s.cz, nullptr);
      p.lo = g.terms == 2 ? a->m * g.dz_ld : 0;
      p.out = dz, p.ldo = g.dz_ld, p.column0 = static_cast<int>(column0);
      e = launch_product(p, a->type, XENT_SLOPE, false, s.z.b.mn, s.cz, stream);
    }
    if (e == hipSuccess && a->dx && a->m) {
      XentParams p = base;
      p.halves = g.terms == 2;
      p.sum = reinterpret_cast<float *>(sum), p.add = i > 0, p.last = i + 1 == g.pieces;
      s.dx.p.out = a->dx, s.dx.p.ldo = a->dx_ld;
      e = run_sum(p, s.dx, s.cdx, a->type, parts, stream);
    }
    if (e == hipSuccess && a->dw) {
      XentParams p = base;
      p.last = 1;
      s.dw.p.out = const_cast<char *>(from_column(a->dw, a->dw_ld)), s.dw.p.ldo = a->dw_ld;
      if (g.terms == 2) {
        const OuterParams q{s.dw.a.p, s.dw.b.p, s.dw.a.ld, s.dw.b.ld, a->m * g.dz_ld, static_cast<int>(a->m), s.dw.p.m, s.dw.p.n};
        p.out = s.dw.p.out, p.ldo = a->dw_ld;
        if (a->type == TF_T_BF16) nk ? launch_outer<bf16, true>(q, p, stream) : launch_outer<bf16, false>(q, p, stream);
        else nk ? launch_outer<f16, true>(q, p, stream) : launch_outer<f16, false>(q, p, stream);
        e = hipGetLastError();
      } else {
        e = run_sum(p, s.dw, s.cdw, a->type, parts, stream);
      }
    }
  }
  return hip(e, call);
}

}  // namespace

extern "C" {

int tf_linear_xent_workspace(const tf_linear_xent_args_t *args, long long *bytes) {
  return guarded([&] { return loss_workspace(args, bytes); });
}

int tf_linear_xent(const tf_linear_xent_args_t *args, void *stream) {
  return guarded([&] { return loss(args, static_cast<hipStream_t>(stream)); });
}

int tf_linear_xent_grad_workspace(const tf_linear_xent_grad_args_t *args, long long *bytes) {
  return guarded([&] { return grad_workspace(args, bytes); });
}

int tf_linear_xent_grad(const tf_linear_xent_grad_args_t *args, void *stream) {
  return guarded([&] { return grad(args, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
