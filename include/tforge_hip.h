/*
 * libtforge_hip -- C ABI of the MI355X (gfx950) backend for TensorForge's GPU
 * hot path: the fused fp32 relu(A @ B + bias) kernel, plain matmul, and the
 * bias_add / relu / add epilogues that --tforge-gpu-pipeline emits.
 *
 * The reference crosses three boundaries on this path (paths in the
 * TensorForge tree); this library replaces all three in one process:
 *   1. compile:  tensorforge-opt --tforge-gpu-pipeline="<opts>" + the NVVM/ptxas
 *                chain (python/tforge_gpu.py:66-91)          -> tf_compile
 *   2. kernel ABI: one noalias device pointer per entry argument, then the
 *                result out-param (runners/gpu/tforge-gpu-bench.cu:20-24;
 *                lib/Transforms/Gpu.cpp:494-512, 563-570)   -> tf_launch
 *   3. runner:   tforge-gpu-bench --mode kernel|cublas [--info-only]
 *                (runners/gpu/tforge-gpu-bench.cu:92-140, 175-383)
 *                                                           -> tf_run, tf_bench,
 *                                                              tf_kernel_info
 *
 * Conventions: plain pointers and sizes only.  Every int-returning function
 * returns 0 on success or a negative TF_E* code, and tf_last_error() then
 * holds the message (the reference printed it and exited 1:
 * runners/gpu/tforge-gpu-bench.cu:52-70; the Python wrapper raises
 * RuntimeError with it, python/tforge_cpu.py:216-222).  Handles are not shared
 * between threads.  All tensors of compiled programs are row-major float32.
 *
 * Beside compiled programs the library has the operators of the residual MLP
 * block in 16 and 8 bits, for training and serving (no counterpart in the
 * reference): tf_rms_norm, tf_quantize_rows, tf_linear and the gradients
 * tf_rms_norm_grad and tf_linear_grad, what keeps activations in 8 bits for these
 * (tf_keep8), and the loss over a vocabulary (tf_linear_xent), at the end of this file.
 */
#ifndef TFORGE_HIP_H
#define TFORGE_HIP_H

#ifdef __cplusplus
extern "C" {
#endif

#define TF_OK 0
#define TF_E_PARSE -1    /* program text does not parse or verify            */
#define TF_E_OPTIONS -2  /* malformed pipeline option string                 */
#define TF_E_PLAN -3     /* program/option combination the pipeline rejects */
#define TF_E_ARG -4      /* bad argument to an API call                       */
#define TF_E_HIP -5      /* HIP runtime error                                 */
#define TF_E_BLAS -6     /* vendor BLAS baseline unavailable or failed        */

#define TF_FAMILY_DIRECT 0      /* tile-k=0: one FMA chain per output          */
#define TF_FAMILY_STAGED 1      /* tile-k>0: LDS-staged FP32 MFMA              */
#define TF_FAMILY_ELEMENTWISE 2 /* programs without a matmul                   */
#define TF_FAMILY_WAVEK 4       /* tile-k>0 with wave-split-k: the waves of a
                                   workgroup split K, partial tiles summed in
                                   LDS (one launch, no workspace)              */

#define TF_MODE_KERNEL 0 /* the compiled program                            */
#define TF_MODE_BLAS 1   /* rocBLAS sgemm + a separate epilogue kernel: the
                            counterpart of the reference's --mode cublas
                            (runners/gpu/tforge-gpu-bench.cu:303-318)       */

typedef struct tf_kernel tf_kernel_t; /* opaque: one compiled tforge program */

/* Device facts; replaces the runner's cuDeviceGetName/driver queries
 * (runners/gpu/tforge-gpu-bench.cu:180-186, 367-368). */
typedef struct {
  char name[256];
  char arch[64];
  int compute_units;
  int max_clock_mhz;
  int lds_bytes_per_cu;
  int max_threads_per_cu;
  long long l2_bytes;
  long long global_mem_bytes;
  int driver_version;
  int runtime_version;
} tf_device_info_t;

/* Static launch description of one kernel of a compiled program; replaces
 * the tforge.launch attribute / launch.json (lib/Transforms/Gpu.cpp:572-577,
 * python/tforge_gpu.py:42-51, 88-90). */
typedef struct {
  char kernel[96];   /* instantiation name                                   */
  char args[160];    /* buffer order, reference "argN" spelling              */
  char ops[96];      /* fused ops of this launch, e.g. matmul+bias_add+relu  */
  int family;        /* TF_FAMILY_*                                          */
  int grid[3];
  int block[3];
  long long m, n, k; /* problem of this launch (k = 0 for element ops)       */
  int lds_bytes;     /* static LDS of the instantiation                      */
} tf_launch_info_t;

/* Resources and occupancy of one kernel; replaces --info-only
 * (runners/gpu/tforge-gpu-bench.cu:278-291).  Needs a GPU. */
typedef struct {
  int regs;          /* VGPRs per lane as reported by hipFuncGetAttributes   */
  int local_bytes;   /* private (scratch) bytes per lane                     */
  int static_smem;   /* static LDS bytes per workgroup                       */
  int blocks_per_cu; /* hipOccupancyMaxActiveBlocksPerMultiprocessor         */
  double theo_occupancy; /* resident waves / max waves per CU                */
  int threads;
} tf_kernel_resources_t;

/* One buffer of the program's kernel ABI (argN order: entry arguments, then
 * the result). */
typedef struct {
  char name[64];
  int role;          /* 0 input, 1 output                                     */
  long long rows, cols; /* 2-D view: leading dims flattened into rows         */
} tf_buffer_info_t;

/* Timing of tf_bench; replaces the runner's JSON line
 * (runners/gpu/tforge-gpu-bench.cu:363-381). */
typedef struct {
  double median_ms, min_ms, mean_ms, std_ms;
  double clock_median_mhz, clock_min_mhz, clock_max_mhz;
  double power_median_w;
  int warmup, reps, l2_flush;
  long long padded[3]; /* problem the kernel ran at (Mp, Np, Kp)             */
} tf_bench_result_t;

const char *tf_last_error(void);

/* Device 0 facts (the reference runner also uses device 0 and reports its
 * name and driver in the JSON line, runners/gpu/tforge-gpu-bench.cu:367-381). */
int tf_device_info(tf_device_info_t *out);

/* Parse + verify `program` (tforge text, diagnostics name `source_name`),
 * parse `options` (--tforge-gpu-pipeline option string, may be empty), plan the
 * launches and select the gfx950 instantiations.  No GPU work: runs on a host
 * without a GPU.  Replaces python/tforge_gpu.py:66-91 (compile_kernel's
 * tool chain).  Options are the reference's (include/TensorForge/Pipelines.h:45-72)
 * plus four backend options: split-k=S (S workgroups per output tile along K,
 * then an ordered reduction launch), mask-edges (staged kernels accept shapes
 * that are not tile multiples), wave-split-k (each wave of a workgroup
 * reduces its own K range of the workgroup's tile, the partial tiles are
 * added in LDS in wave order: one launch for shapes with few output tiles)
 * and xcd-swizzle (default on).
 * Staged configurations (tile-k > 0) give each 64-lane wave an
 * (8*TM) x (8*TN) output tile of MFMA blocks.  Where that wave tile cannot
 * tile the block -- fewer than 64 threads, or a wave tile taller or wider
 * than the block tile, as in 30 of the reference's 105 Stage 9
 * configurations (python/costmodel.py:49-60) -- the same block tile and
 * tile-k run on a stand-in wave layout: one wave over the whole block when
 * there are fewer than 64 threads (thread tile BM/8 x BN/8), otherwise the
 * same threads and accumulators per lane with the long side of the thread
 * tile shortened to fit.  tf_kernel_launch_info then reports the block
 * actually launched and the instantiation's name. */
int tf_compile(const char *source_name, const char *program, const char *options, tf_kernel_t **out);
void tf_kernel_free(tf_kernel_t *k);

/* The compiled program's launches (one, or two for the residual block) and
 * buffers: what the reference reads back from launch.json and the runner's
 * --grid/--block/--args flags (python/tforge_gpu.py:42-51, 88-90;
 * runners/gpu/tforge-gpu-bench.cu:20-24, 92-140). */
int tf_kernel_num_launches(const tf_kernel_t *k);
int tf_kernel_launch_info(const tf_kernel_t *k, int launch, tf_launch_info_t *out);
/* tf_kernel_launch_info describes the options' own kernel; this one the kernel that
 * runs where every buffer is 16-byte aligned, chosen by the problem's size with the
 * same results bit for bit: a direct GEMM's chains on the matrix cores, element ops
 * as one stream of vectors, a staged kernel's form for crowded grids, or the options'
 * own.  On other buffers direct GEMMs and element ops run the options' own kernel and
 * staged ones are refused.  No counterpart in the reference, which launches the kernel
 * it generated. */
int tf_kernel_run_info(const tf_kernel_t *k, int launch, tf_launch_info_t *out);
int tf_kernel_num_buffers(const tf_kernel_t *k); /* entry arguments + 1 result */
int tf_kernel_buffer_info(const tf_kernel_t *k, int index, tf_buffer_info_t *out);
/* Shape (rows x cols) of buffer `index` as tf_run / tf_bench copy it from and
 * to host memory: the compiled shape, or, with `logical_mnk`, the logical
 * shape of the buffer's role in the single matmul chain (A m x k, B k x n,
 * bias 1 x n, residual and result m x n; an unused argument keeps its compiled
 * shape).  Fails with TF_E_ARG where tf_run would refuse the logical sizes (a
 * multi-launch program, sizes above the compiled ones, or one buffer in two
 * roles whose logical shapes differ).  The counterpart of the reference
 * runner's per-buffer --in-dir file sizes (runners/gpu/tforge-gpu-bench.cu:214-232). */
int tf_kernel_host_shape(const tf_kernel_t *k, const long long *logical_mnk, int index, long long *rows,
                         long long *cols);
/* Resources and occupancy of one launch's kernel (tf_kernel_run_info's): the
 * runner's --info-only (runners/gpu/tforge-gpu-bench.cu:278-291). */
int tf_kernel_info(const tf_kernel_t *k, int launch, tf_kernel_resources_t *out);

/* Kernel ABI: enqueue every launch of the program on `stream` (a hipStream_t,
 * NULL for the default stream) with caller-owned device buffers in argN order,
 * shaped as compiled: tf_kernel_num_buffers(k) pointers, the inputs then the
 * result, each to the float32 elements tf_kernel_buffer_info reports.  A NULL
 * pointer for a non-empty buffer is refused (TF_E_ARG) before any launch.
 * Intermediates of multi-launch programs and the split-K
 * partial-sum workspace are allocated once per handle on first use; calls on
 * one handle that overlap on different streams share them.  No
 * synchronisation.  Replaces cuLaunchKernel with the marshalled argN list
 * (runners/gpu/tforge-gpu-bench.cu:259-299). */
int tf_launch(tf_kernel_t *k, void *const *device_buffers, void *stream);

/* tf_launch without any device allocation, for callers that cannot allocate
 * (code under HIP graph capture, serving loops, harnesses that forbid
 * hipMalloc).  No counterpart in the reference.  Same arguments and kernels as
 * tf_launch; the split-K workspace and the intermediates of multi-launch
 * programs come from one fixed 32 MiB device array per GPU (held from the
 * library's first use on that GPU until the process ends) instead of the
 * handle's buffers.  A program that needs more scratch than that is refused
 * with TF_E_ARG before anything is enqueued.  Nothing in the array needs
 * clearing between calls (every slice and intermediate is written whole
 * before it is read), but every call on one GPU shares it: calls that overlap
 * on that GPU -- from any handle or stream -- race, so serialise them.
 * `stream` must belong to the current device (TF_E_ARG otherwise).  The
 * array's device address is looked up on the first call on each device; that
 * first call may itself be under stream capture. */
int tf_launch_noalloc(tf_kernel_t *k, void *const *device_buffers, void *stream);

/* Correctness run, as the runner's "--warmup 0 --reps 1 --in-dir --out":
 * uploads host inputs, NaN-prefills the output, runs once, downloads the
 * result.  `logical_mnk` (may be NULL) gives the unpadded M, N, K of a
 * single-matmul program compiled at a padded shape: inputs and output are then
 * at the logical shape and the library pads and unpads with device copies,
 * as the reference runner does (runners/gpu/tforge-gpu-bench.cu:214-232,
 * 292-302, 323-331).  host_inputs holds one row-major float32 array per
 * input, each of the size tf_kernel_host_shape reports for the same
 * `logical_mnk` (M x K, K x N and N elements for A, B and bias at a logical
 * shape; the compiled shapes otherwise), and host_out has room for the result;
 * the library copies exactly those sizes.  mode is TF_MODE_KERNEL or TF_MODE_BLAS. */
int tf_run(tf_kernel_t *k, int mode, const long long *logical_mnk, const float *const *host_inputs,
           float *host_out);

/* Timing run: inputs from `host_inputs` (or, if NULL, uniform[-1,1] from
 * `seed`), `warmup` untimed runs, then `reps` runs each bracketed by a HIP
 * event pair on the library's stream (pad copies included when padded, an
 * optional 512 MiB L2/MALL flush before each rep outside the events), the
 * shader clock (tf_clock_probe) and, where amdsmi loads, the power sampled
 * after each rep.  Replaces
 * runners/gpu/tforge-gpu-bench.cu:337-381. */
int tf_bench(tf_kernel_t *k, int mode, const long long *logical_mnk, const float *const *host_inputs,
             unsigned seed, int warmup, int reps, int flush, tf_bench_result_t *out);

/* Shader clock (MHz) measured on the device: a probe kernel after the work
 * already queued on `stream` (a hipStream_t, NULL for the default stream)
 * counts shader-clock cycles against the 100 MHz wall clock in one workgroup
 * per XCD; mean, min and max over the XCDs (min/max may be NULL).
 * Synchronises the stream.  Each call writes its own result slot (64 slots
 * per GPU, taken round robin), so calls from several threads or streams may
 * overlap.  tf_bench takes one such sample after every rep;
 * the reference samples the SM clock through NVML instead
 * (runners/gpu/tforge-gpu-bench.cu:333-361). */
int tf_clock_probe(void *stream, double *mean_mhz, double *min_mhz, double *max_mhz);

/* Per-rep event times (ms) of the last tf_bench on this handle, up to `cap`
 * values; returns the count.  No counterpart in the reference (its runner
 * prints only median/min/std); for callers that want the distribution. */
int tf_bench_samples(const tf_kernel_t *k, double *out_ms, int cap);

/* Registry introspection: number of ahead-of-time instantiations and the
 * staged configuration of entry i (family, bm, bn, tm, tn, bk, promote,
 * vectorize) -- what the autotuner may select.  No counterpart in the
 * reference, which generates each kernel on demand. */
int tf_registry_size(void);
int tf_registry_entry(int i, int *family, int *cfg7, char *name, int name_cap);

/* ---- operators of the residual MLP block --------------------------------------
 *
 * Plain calls on device pointers: no handle, no allocation, no synchronisation;
 * everything is enqueued on `stream` (a hipStream_t, NULL for the default
 * stream) as kernel launches alone, so a call may be captured in a HIP graph.
 * Matrices have their rows contiguous; *_ld is the distance between two rows in
 * elements (>= the row's length).  Any row length, distance and alignment of the
 * elements is accepted; 16-byte aligned rows run fastest.  Sizes are at most
 * 2^30.  Outputs and the workspace overlap nothing but where said.  A size of
 * zero is a call without work, except that gradients summed over no rows and
 * products over no k are written as sums of nothing, and the scales of rows
 * without elements as those of zeros.
 * Arithmetic is float32 from the inputs on and every output is rounded once,
 * but for two values that the products take in fewer bits: the gradients' dz
 * (tf_linear_grad) and, inside the matrix instructions of 8-bit products, the
 * products of eight neighbouring k (tf_linear).
 * Sums are taken in a fixed order: equal calls give equal bits.
 * Arguments that cannot hold give TF_E_ARG before anything is enqueued. */

#define TF_T_F32 0
#define TF_T_BF16 1
#define TF_T_F16 2
#define TF_T_F8 3 /* OCP e4m3: 8 bits, largest value 448 */
#define TF_T_I8 4 /* 8-bit integers (two's complement)    */

#define TF_ACT_NONE 0
#define TF_ACT_RELU 1 /* NaN stays, as in compiled programs */
#define TF_ACT_GELU 2 /* z * P(normal <= z) */
#define TF_ACT_SILU 3 /* z / (1 + exp(-z)) */

/* h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight, row by row, the norm
 * taken of the sum before h is rounded.  With y_type TF_T_F8 y is in 8 bits with
 * one scale a row: top = max(max|y|, 2^-100), scale = top/448, code = the value
 * nearest to y * (448 * (1/top)) (ties to even); with TF_T_I8 the same with 127 in
 * 448's place, in integers of -127..127.  In 8 bits a row that holds an
 * infinity or a NaN stands for NaN throughout (codes times scale); in `type` its
 * infinities give NaN and its finite values 0, a NaN gives NaN throughout. */
typedef struct {
  const void *x, *residual; /* rows x d of `type`; residual may be NULL          */
  const void *weight;       /* d of weight_type                                  */
  void *y;                  /* rows x d of y_type                                */
  void *h;                  /* rows x d of `type`; NULL without a residual; may be
                               x or residual itself                               */
  float *scale;             /* rows; 8-bit y only                                 */
  long long x_ld, residual_ld, y_ld, h_ld;
  long long rows, d;
  int type;        /* TF_T_F32, TF_T_BF16, TF_T_F16                               */
  int weight_type; /* `type` or TF_T_F32                                          */
  int y_type;      /* `type`, TF_T_F8 or TF_T_I8                                  */
  float eps;       /* >= 0                                                        */
} tf_rms_norm_args_t;
int tf_rms_norm(const tf_rms_norm_args_t *args, void *stream);

/* x (rows x d of `type`) in 8 bits with one scale a row, as tf_rms_norm's. */
int tf_quantize_rows(const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                     float *scale, void *stream);

/* The same into y_type: TF_T_F8 or TF_T_I8. */
int tf_quantize_rows_to(const void *x, long long x_ld, long long rows, long long d, int type, void *y, long long y_ld,
                        int y_type, float *scale, void *stream);

/* Activations kept in 8 bits for a backward pass: rows x d values in groups of 32
 * neighbours of a row, each value an integer of -127..127 times its group's unit, the
 * least power of two (2^-126 at least) whose integers stay within 127 (nearest, ties
 * to even).  In memory, 16-byte aligned, tf_keep8_bytes(rows, d) in all: rows x
 * ceil(d/32) x 32 integers, zeros behind a row's end, then rows x ceil(d/32)
 * bytes e, the unit being 2^(e-127).  A group that holds an infinity or a NaN has e =
 * 255 and zeros, and stands for NaN throughout.
 * positive: values above zero keep an integer of at least 1, so that relu's
 * gradient from a pre-activation kept so is that of the pre-activation itself, where the
 * group is finite.
 * tf_keep8_masked: minus infinity is the integer -128 instead and counts for no unit.  It comes back
 * as itself, with a slope of 0 under every activation, and its neighbours as without it.
 * tf_restore8 gives the values in `type`: exact in TF_T_F32 and TF_T_BF16, in
 * TF_T_F16 rounded; finite ones past the type's largest number (to which a group's largest
 * value may have been rounded up) are that. */
int tf_keep8_bytes(long long rows, long long d, long long *bytes);
int tf_keep8(const void *x, long long x_ld, long long rows, long long d, int type, int positive, void *kept, void *stream);
int tf_keep8_masked(const void *x, long long x_ld, long long rows, long long d, int type, int positive, void *kept, void *stream);
int tf_restore8(const void *kept, long long rows, long long d, int type, void *x, long long x_ld, void *stream);

/* Which operands of a gradient are kept in 8 bits (their *_ld does not count). */
#define TF_KEPT_H 1 /* tf_rms_norm_grad's h        */
#define TF_KEPT_X 1 /* tf_linear_grad's x          */
#define TF_KEPT_Z 2 /* tf_linear_grad's z, tf_linear's */

/* tf_rms_norm's gradient.  r = 1/sqrt(mean(h^2) + eps), xhat = h*r:
 *   dx = r*(dy*weight - xhat*mean(dy*weight*xhat)) + dh     (also the residual's)
 *   dweight = sum over rows of dy*xhat */
typedef struct {
  const void *dy, *h; /* rows x d of `type`; h: the norm's input (x + residual)     */
  const void *dh;     /* rows x d: the gradient that reaches h past the norm, or NULL */
  const void *weight; /* d of weight_type                                           */
  void *dx;           /* rows x d of `type`; may be dy or dh itself                 */
  void *dweight;      /* d of weight_type                                           */
  long long dy_ld, h_ld, dh_ld, dx_ld;
  long long rows, d;
  int type, weight_type; /* as tf_rms_norm's                                        */
  float eps;
  int kept;        /* 0, or TF_KEPT_H                                               */
  void *workspace; /* 16-byte aligned, tf_rms_norm_grad_workspace(rows, d) bytes    */
  long long workspace_bytes;
} tf_rms_norm_grad_args_t;
int tf_rms_norm_grad_workspace(long long rows, long long d, long long *bytes);
int tf_rms_norm_grad(const tf_rms_norm_grad_args_t *args, void *stream);

/* z = x @ w + bias;  out = act(z) + residual.  x is m x k, w is k x n in either
 * memory order.  With type TF_T_F8 or TF_T_I8 x has a scale a row and w a scale a
 * column, z = (x @ w) * x_scale[m] * w_scale[n] + bias, and w_order is 1.
 *
 * Sums over k are float32; of TF_T_I8 they are 32-bit integers, exact, any codes
 * of -128..127 allowed and k at most 131071, and are rounded to float32 before the
 * scales: the same bits whatever the tile and the splits.
 * In e4m3 the matrix instruction adds the products of
 * eight neighbouring k (0..7, 8..15, ...) first, aligned to the largest of the eight
 * and cut off 13 bits below it.  A sum of products of random signs is off by 1.5e-5
 * of itself by this, a 250th of bfloat16's rounding; where the sum cancels, by
 * 2^-10 of the largest product for each eight k at most. */
typedef struct {
  const void *x, *w;
  const void *bias;     /* n of bias_type, or NULL                                  */
  const void *residual; /* m x n of out_type, or NULL                               */
  const float *x_scale, *w_scale; /* 8 bits only: m, n                              */
  void *out;            /* m x n of out_type                                        */
  void *z;              /* m x n of out_type: the pre-activation kept, or NULL      */
  void *workspace;      /* 16-byte aligned; with fewer bytes than tf_linear_workspace
                           asks for (none: 0) the call runs unsplit along k, without
                           aligned copies                                           */
  long long workspace_bytes;
  long long x_ld, w_ld, residual_ld, out_ld, z_ld;
  long long m, n, k;
  int w_order;   /* 0: w lies as k rows of n, 1: as n rows of k                      */
  int type;      /* TF_T_BF16, TF_T_F16, TF_T_F8, TF_T_I8                            */
  int out_type;  /* `type`; TF_T_BF16 or TF_T_F16 for 8 bits                         */
  int bias_type; /* out_type or TF_T_F32                                             */
  int act;       /* TF_ACT_*                                                         */
  int tile;      /* C tile: 0 by the sizes, 1: 256x256, 2: 128x128, 3: 64x64, 4: all of
                    up to 64 rows, k split over a workgroup's waves, 5: 64x128; one that
                    cannot run these operands gives way to the choice by sizes       */
  int splits;    /* ranges of k: 0 by the sizes, or 1..64                            */
  int kept;      /* 0, or TF_KEPT_Z: z is written in 8 bits, as tf_keep8_masked of the z
                    in out_type would (relu's with `positive`); not of 8-bit products,
                    and the workspace has to be whole                                */
} tf_linear_args_t;
/* Bytes of workspace for these arguments: sizes, types, distances and the
 * alignment of x and w count, the memory is not touched. */
int tf_linear_workspace(const tf_linear_args_t *args, long long *bytes);
int tf_linear(const tf_linear_args_t *args, void *stream);

/* tf_linear's gradient in 16 bits: dz = dy * act'(z), dx = dz @ w^T, dw = x^T @ dz
 * in w's memory order, dbias = sum over rows of dz.  The residual's gradient is dy.
 *
 * dbias sums dz in float32.  The products take it in `type`: exactly with
 * TF_ACT_NONE and TF_ACT_RELU; with the smooth activations rounded, in one term, or
 * in two (the value and what its rounding left, 16 bits more), as `terms` says.  In
 * one term the products err by sqrt(2) of their own rounding; two take them twice
 * as long.  By the sizes: two up to 1.4e8 multiply-adds (m * n * k), one above.  A
 * dz past float16's largest value is an infinity in one term, itself in two. */
typedef struct {
  const void *dy, *x, *w; /* m x n, m x k, k x n in either order                    */
  const void *z;          /* m x n: the kept pre-activation; NULL with TF_ACT_NONE  */
  void *dx, *dw;          /* each may be NULL: not wanted                           */
  void *dbias;            /* n of bias_type, or NULL                                */
  void *workspace;        /* 16-byte aligned, tf_linear_grad_workspace's bytes       */
  long long workspace_bytes;
  long long dy_ld, x_ld, w_ld, z_ld, dx_ld, dw_ld;
  long long m, n, k;
  int w_order;   /* of w and dw, as tf_linear's                                     */
  int type;      /* TF_T_BF16, TF_T_F16                                             */
  int bias_type; /* `type` or TF_T_F32                                              */
  int act;
  int tile, splits; /* both products', as tf_linear's                                */
  int terms;     /* of dz in the products: 0 by the sizes, 1 or 2                   */
  int kept;      /* 0, or TF_KEPT_X, TF_KEPT_Z or both: x goes into its product
                    rounded to `type`, z into the slope as it is                     */
} tf_linear_grad_args_t;
/* As tf_linear_workspace; which of dx, dw and dbias are wanted counts too. */
int tf_linear_grad_workspace(const tf_linear_grad_args_t *args, long long *bytes);
int tf_linear_grad(const tf_linear_grad_args_t *args, void *stream);

/* The cross entropy of logits z = x @ w that are never in memory as a whole:
 *   lse[m] = log(sum over n of exp(z[m][n])),  loss[m] = lse[m] - z[m][target[m]]
 * w as tf_linear's.  A row whose target is `ignore` does not count: its loss is 0.  A
 * target outside of 0..n-1 otherwise gives NaN.  Sums over k, logits, exponentials and
 * their sums are float32.  A logit of minus infinity adds nothing.  A row with a logit of plus infinity or
 * NaN is NaN, one whose logits are all minus infinity has that lse and a loss of NaN.  Exponents are taken in
 * base 2, so that logits past 2.358e38 (2^128 / log2(e)) stand for these infinities. */
typedef struct {
  const void *x, *w;       /* m x k, k x n in either order                          */
  const long long *target; /* m                                                     */
  float *loss;             /* m                                                     */
  double *lse;             /* m; in 64 bits for the gradient: where a row is sure of its
                              class, it takes a small difference of large numbers    */
  float *sum, *mean, *count; /* one float each, or NULL: of the losses of the rows that
                              count, and their number; a mean of no rows is 0       */
  void *workspace;         /* 16-byte aligned, tf_linear_xent_workspace's bytes     */
  long long workspace_bytes;
  long long x_ld, w_ld;
  long long m, n, k;       /* n >= 1                                                */
  long long ignore;
  int w_order, type;       /* type: TF_T_BF16, TF_T_F16                             */
} tf_linear_xent_args_t;
/* Bytes of workspace for these arguments, as tf_linear_workspace: 8 for each row and
 * tile of columns, and aligned copies of odd operands. */
int tf_linear_xent_workspace(const tf_linear_xent_args_t *args, long long *bytes);
int tf_linear_xent(const tf_linear_xent_args_t *args, void *stream);

/* Its gradient, from the dloss of every row (or one for all) and the kept lse:
 *   dz[m][n] = (exp(z[m][n] - lse[m]) - [n == target[m]]) * dloss[m] / count
 *   dx = dz @ w^T,  dw = x^T @ dz in w's memory order
 * The logits are computed again, for a piece of the vocabulary at a time, and the
 * products take dz in `type`: rounded once, up to 64 rows in two terms (the value and
 * what its rounding left, 16 bits more).  One dloss for all rows is multiplied into
 * their sums instead, and float16 has a unit that lets the largest dz reach 2^15.
 * Sums are float32, over the pieces too.  A row that does not count
 * has a dz of zeros whatever its x holds (dw is the product all the same: an x that is
 * not finite gives NaN there). */
typedef struct {
  const void *x, *w;
  const long long *target;
  const double *lse;       /* m                                                     */
  const float *dloss;      /* m with dloss_rows, else one                           */
  const float *count;      /* one float, or NULL for 1: the mean's gradient takes
                              tf_linear_xent's count                                */
  void *dx, *dw;           /* each may be NULL: not wanted                          */
  void *workspace;         /* 16-byte aligned, tf_linear_xent_grad_workspace's bytes */
  long long workspace_bytes;
  long long x_ld, w_ld, dx_ld, dw_ld;
  long long m, n, k;
  long long ignore;
  int w_order, type;
  int dloss_rows;          /* 0 or 1                                                */
  int reserved;            /* 0                                                     */
} tf_linear_xent_grad_args_t;
/* A piece's dz of up to 128 MB (or 8192 columns), float32 sums of dx where there is
 * more than one piece, parts of split products, aligned copies. */
int tf_linear_xent_grad_workspace(const tf_linear_xent_grad_args_t *args, long long *bytes);
int tf_linear_xent_grad(const tf_linear_xent_grad_args_t *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TFORGE_HIP_H */
