/*
 * vcsr_spmm.h - C ABI of the MI355X (gfx950) VCSR SpMM library.
 *
 * Sparse A (CSR, FP32) x dense B (row-major, FP32) = dense C (row-major).
 * The path: Matrix Market / synthetic load -> COO -> CSR -> VCSR build
 * (column segments of width `segw`, rows of each segment sorted by nnz
 * descending, packed depth-major into bundles of `bundle` lanes) -> HIP kernel.
 *
 * Every entry point returns 0 on success or a nonzero VCSR_E* status; the
 * message of the last failure on the calling thread is vcsr_last_error().
 * No C++ exception crosses this boundary.  Streams and events are passed as
 * `void*` (a hipStream_t / hipEvent_t of the library's own HIP runtime; NULL
 * is the null stream), so the header needs no HIP or framework include.
 *
 * Each declaration names the reference interface it replaces
 * (MuuSeoTia/VCSR-SPMM, path:line).
 */
#ifndef VCSR_SPMM_H
#define VCSR_SPMM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ status */
enum {
    VCSR_OK = 0,
    VCSR_EINVAL = 1,  /* bad argument (shape, pointer, parameter)            */
    VCSR_EIO = 2,     /* file open / parse failure                           */
    VCSR_ENOMEM = 3,  /* host or device allocation failed                    */
    VCSR_EDEVICE = 4, /* HIP runtime error, or no GPU                        */
    VCSR_ERANGE = 5,  /* index out of range, or a size overflows int32       */
    VCSR_ESTATE = 6   /* object not in the required state (e.g. not uploaded) */
};

/* Thread-local text of the last failing call on this thread ("" if none). */
const char* vcsr_last_error(void);
/* Library version string. */
const char* vcsr_version(void);

/* ------------------------------------------------------- COO (host, owned) */
/* Replaces `struct COO` / `read_matrix_market_coo` (include/mmio.hpp:15-46). */
typedef struct vcsr_coo vcsr_coo;
typedef struct {
    int32_t M, N;
    int64_t nnz;
    const int32_t* rows; /* 0-based */
    const int32_t* cols; /* 0-based */
    const float* vals;
} vcsr_coo_view;

/* Read a coordinate Matrix Market file with the reference's semantics
 * (include/mmio.hpp:22-46): every line starting with '%' and every empty line
 * before the size line is skipped (so `symmetric`/`pattern` qualifiers are
 * ignored), indices are 1-based unless the first entry has a 0 row or column,
 * values are read as double and narrowed to float.  expand_symmetric != 0 is
 * an opt-in extension (not in the reference): when the banner says
 * `symmetric`, every off-diagonal (r,c,v) also yields (c,r,v). */
int vcsr_mtx_read(const char* path, int32_t expand_symmetric, vcsr_coo** out);
/* Wrap caller arrays (copied) as a COO object. */
int vcsr_coo_create(int32_t M, int32_t N, int64_t nnz, const int32_t* rows,
                    const int32_t* cols, const float* vals, vcsr_coo** out);
int vcsr_coo_view_get(const vcsr_coo* coo, vcsr_coo_view* out);
void vcsr_coo_free(vcsr_coo* coo);

/* Synthetic A of BASELINE config `cfg` (1..5) for `seed`, as COO in
 * generation order (rows ascending, columns in draw order).  Deterministic
 * for (cfg, seed).  Not in the reference (it reads SuiteSparse files). */
int vcsr_gen_coo(int32_t cfg, uint64_t seed, vcsr_coo** out);
/* Synthetic dense operand: rows x cols floats, row-major, into `out`
 * (caller-owned host buffer).  dist 0 = U[-1,1) on a 2^-23 grid,
 * dist 1 = N(0,1).  Element i depends only on (seed, i). */
int vcsr_gen_dense(uint64_t seed, int32_t dist, int64_t rows, int32_t cols,
                   float* out);

/* ------------------------------------------------------- CSR (host, owned) */
/* Replaces `struct CSR` / `coo_to_csr` (include/csr.hpp:8-37). */
typedef struct vcsr_csr vcsr_csr;
typedef struct {
    int32_t M, N, nnz;
    const int32_t* row_ptr; /* M+1 */
    const int32_t* col;     /* nnz */
    const float* val;       /* nnz */
} vcsr_csr_view;

/* COO -> CSR with the reference's result: rows bucketed in input order, then
 * each row's entries ordered by column with the same std::sort call as
 * include/csr.hpp:28-35 (duplicates kept, not merged).  Row indices outside
 * [0,M) fail with VCSR_ERANGE (as csr.hpp:19); column indices outside [0,N)
 * also fail (the reference leaves them unchecked). */
int vcsr_coo_to_csr(const vcsr_coo* coo, vcsr_csr** out);
/* Wrap caller CSR arrays (copied, validated) as a CSR object. */
int vcsr_csr_create(int32_t M, int32_t N, const int32_t* row_ptr,
                    const int32_t* col, const float* val, vcsr_csr** out);
int vcsr_csr_view_get(const vcsr_csr* csr, vcsr_csr_view* out);
void vcsr_csr_free(vcsr_csr* csr);

/* ------------------------------------------------------------ VCSR format */
enum {
    VCSR_LAYOUT_H = 0,  /* csr_to_vcsr_spmm, include/vcsr.hpp:25-109          */
    VCSR_LAYOUT_S = 1,  /* csr_to_vcsr_seg / _opt, src/vcsr_seg.cu:24-113    */
    VCSR_LAYOUT_TC = 2  /* csr_to_vcsr_tc (segw=16, bundle=16), src/vcsr_tc.cu:26-106 */
};

typedef struct vcsr_fmt vcsr_fmt;
typedef struct {
    int32_t M, N, segw, bundle, layout;
    int32_t num_groups;   /* G */
    int32_t num_segments; /* S = ceil(N/segw) */
    int64_t num_slots;    /* P = sum_g depth_g * bundle */
    const int32_t* group_ptr;      /* G+1: first slot of group g            */
    const int32_t* group_depth;    /* G                                      */
    const int32_t* group_seg_base; /* G: first column of the group's segment */
    const int32_t* group_rows;     /* G*bundle: row per lane, -1 = padding   */
    const int32_t* lcol;           /* P: column within segment, -1 = padding */
    const float* val;              /* P: value (0 where lcol == -1)          */
    /* S+1: first group of each segment.  The reference keeps it for layout S
     * only (src/vcsr_seg.cu:21,53,109); here it is derived for every layout. */
    const int32_t* segment_group_start;
} vcsr_arrays;

/* Build the VCSR format of a CSR matrix.  Arrays are bit-identical to the
 * reference builder of `layout` on the same CSR (same group order, same row
 * permutation including the order of rows with equal counts, same padding).
 * Layout TC forces segw=16 and bundle=16 like src/vcsr_tc.cu:27-28.
 * nthreads <= 0 uses every hardware thread; segments are built in parallel
 * and concatenated in segment order, which does not change the result. */
int vcsr_build(const vcsr_csr* csr, int32_t segw, int32_t bundle,
               int32_t layout, int32_t nthreads, vcsr_fmt** out);
int vcsr_fmt_arrays(const vcsr_fmt* fmt, vcsr_arrays* out);
/* Write a built format (its host arrays and the row-tile view settings of
 * vcsr_fmt_set_tile_rows / _windows) to a file, and read one back as a new
 * handle that is bit-identical to the saved one and not uploaded, so a
 * matrix's format is built once (the reference rebuilds it every run,
 * src/main.cpp:128-149).  A file that cannot be read is VCSR_EIO; one whose
 * contents break the format's invariants (array sizes, group pointers,
 * rows, columns, segment table) is VCSR_EINVAL.  No reference counterpart. */
int vcsr_fmt_save(const vcsr_fmt* fmt, const char* path);
int vcsr_fmt_load(const char* path, vcsr_fmt** out);
/* Copy the format to the current device (once; later calls are no-ops).
 * Replaces the per-call cudaMallocAsync/cudaMemcpyAsync of
 * src/kernels.cu:139-151 and the one-time static upload of
 * src/vcsr_seg.cu:196-211.  The handle owns the device copy: no globals. */
int vcsr_fmt_upload(vcsr_fmt* fmt, void* stream);
/* Tile height of the row-tile view vcsr_fmt_upload derives for the
 * tile-stationary kernel (VCSR_KERNEL_TILE): rows = 1, 2, 3, 4, 8 or 16
 * forces it, 0 (the default) picks it from the matrix.  16-row tiles run on
 * the FP32 matrix cores (dense sub-blocks, layout TC matrices).  Only before
 * the upload (VCSR_ESTATE after).  No reference counterpart. */
int vcsr_fmt_set_tile_rows(vcsr_fmt* fmt, int32_t rows);
/* fixed != 0: cut the rows into fixed windows of the tile height (which must
 * then be set) instead of tiles of rows that share columns.  With 16
 * rows this is FastSpMM's condensed-tile layout (16-row windows whose
 * distinct columns form 16-column blocks; build_cst_from_csr,
 * src/fastspmm.cu:129-233), computed on FP32 MFMA instead of FP16 WMMA
 * (run_fastspmm_gpu, src/fastspmm.cu:257-303).  Only before the upload
 * (VCSR_ESTATE after); an upload without a tile height is VCSR_EINVAL. */
int vcsr_fmt_set_tile_windows(vcsr_fmt* fmt, int32_t fixed);
/* The uploaded view's tile height, tile count and entry count (B-row slice
 * loads per column tile of one SpMM; nnz for tile height 1).  No reference
 * counterpart. */
int vcsr_fmt_tile_info(const vcsr_fmt* fmt, int32_t* rows, int64_t* tiles, int64_t* entries);
/* Free host and device memory (replaces destroy_vcsr_*_device,
 * src/vcsr_seg.cu:233-243). */
void vcsr_fmt_free(vcsr_fmt* fmt);

/* ----------------------------------------------------------------- SpMM */
/* All GPU entry points take device pointers; B is N x O and C is M x O,
 * row-major with leading dimension O, FP32, int32 indices.
 * If `ms` is non-NULL the call is synchronous like the reference wrappers:
 * it records events around the kernel on `stream`, waits, and stores the
 * kernel-only time in *ms.  If `ms` is NULL the kernel is only enqueued. */

/* C = A*B, one thread per row, C zeroed and accumulated in global memory
 * (the algorithm of csr_spmm_kernel, src/kernels.cu:15-33).  Overwrites C.
 * Replaces run_csr_spmm_gpu (src/kernels.cu:107-118). */
int spmm_csr_naive(int32_t M, const int32_t* d_rowptr, const int32_t* d_col,
                   const float* d_val, const float* dB, int32_t O, float* dC,
                   void* stream, float* ms);

/* C = A*B on plain CSR with rows spread over the lanes of a wavefront: each
 * row's (column, value) pairs are read once and shared by its lanes, C is
 * written once (overwritten; no reset needed).  The ASpT-style competitor:
 * replaces run_aspt_spmm_gpu (src/aspt.cu:144-196), which needs O % 64 == 0;
 * this takes any O and one more argument, N (the rows of B), which bounds
 * B's addressing: a column outside [0, N) contributes nothing. */
int spmm_csr_wave(int32_t M, int32_t N, const int32_t* rowptr, const int32_t* col,
                  const float* val, const float* dB, int32_t O, float* dC, void* stream,
                  float* ms);

/* C += A*B over an uploaded VCSR format (any layout) with the fastest kernel
 * (VCSR_KERNEL_AUTO).  C is accumulated into: zero it first, as
 * main.cpp:126-143 does.  tileK is the C/B column tile of the segment-major
 * kernels (spmm_vcsr_ex); the row- and tile-stationary kernels size their
 * column tiles from O.
 * Replaces run_vcsr_spmm_gpu (src/kernels.cu:120-167),
 * run_vcsr_seg_spmm_gpu (src/vcsr_seg.cu:191-231) and
 * run_vcsr_opt_spmm_gpu (src/vcsr_opt.cu:243-285). */
int spmm_vcsr(const vcsr_fmt* fmt, const float* dB, int32_t O, int32_t tileK,
              float* dC, void* stream, float* ms);

/* Kernel selection of spmm_vcsr_ex (all consume the same uploaded format). */
enum {
    VCSR_KERNEL_AUTO = 0,    /* the fastest kernel for the format (currently TILE) */
    VCSR_KERNEL_SEGMENT = 1, /* segment-major streaming on the vector ALUs, B tile
                                in LDS, C flushed with FP32 atomics per group   */
    VCSR_KERNEL_MFMA = 2,    /* segment-major, group collapsed to a dense tile on
                                FP32 MFMA, C flushed with FP32 atomics          */
    VCSR_KERNEL_ROW = 3,     /* row-stationary: one wavefront per C row walks the
                                row's (group, lane) slots; C written once, no
                                atomics                                         */
    VCSR_KERNEL_TILE = 4     /* tile-stationary: runs of 1, 2, 3, 4 or 8
                                consecutive rows sharing columns are walked
                                together on the vector ALUs, and 16-row tiles
                                (dense sub-blocks) on FP32 MFMA; each B row
                                slice loaded once per tile; C written once    */
};

/* spmm_vcsr with an explicit kernel and C semantics: accumulate = 1 gives
 * C += A*B (the reference's semantics), accumulate = 0 gives C = A*B without
 * a separate reset (the ROW and TILE kernels write every row once; the
 * segment-major kernels clear C on the stream first).  tileK applies to the
 * segment-major kernels.  Calls on one format must not overlap in time: the
 * ROW and TILE kernels keep a scratch buffer in the format for the partial
 * sums of very long rows / tiles.  vcsr_fmt_upload sizes it for every O
 * (a format with split rows or tiles is launched in column slices of at
 * most 256 columns), so with `ms` NULL a call only enqueues kernels — no
 * allocation, memset or synchronisation — and can be captured into a HIP
 * graph.  Only if the upload found too little device memory for that
 * buffer does the first call that needs it wait for the stream and
 * allocate it.
 * No reference counterpart (the reference selects kernels by --algo in
 * src/main.cpp:119-163 and always accumulates). */
int spmm_vcsr_ex(const vcsr_fmt* fmt, const float* dB, int32_t O, int32_t tileK,
                 float* dC, void* stream, float* ms, int32_t kernel,
                 int32_t accumulate);

/* The default kernel (VCSR_KERNEL_TILE, as spmm_vcsr_ex runs it) without any
 * device allocation in the call, for callers that cannot allocate: code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc.  No counterpart in the reference.  accumulate as in
 * spmm_vcsr_ex (0: C = A*B, 1: C += A*B).  Enqueued on `stream`, not waited
 * for, no timing.  The partial rows of split tiles live in a fixed device
 * array of 16 MiB (4 Mi floats) that each GPU holds until the process ends;
 * a format and O that need more fail with VCSR_ERANGE before any launch
 * (spmm_vcsr_ex has no such limit).  Every call on one GPU uses that GPU's
 * array, so calls that overlap in time on one GPU race; its contents are
 * written before they are read, so a call never sees an earlier one's.
 * The format must be uploaded to the current device; the upload looks up
 * the array's device address, so even the first call may be made under
 * graph capture. */
int spmm_vcsr_noalloc(const vcsr_fmt* fmt, const float* dB, int32_t O, float* dC,
                      void* stream, int32_t accumulate);

/* C += A*B on FP32 MFMA: every group is collapsed to a dense bundle x segw
 * tile and multiplied by the segment's B tile on the matrix cores (FP32 in,
 * FP32 accumulate).  Meant for dense sub-blocks (layout TC); valid for any
 * layout.  Replaces run_vcsr_tc_spmm_gpu (src/vcsr_tc.cu:197-232), which
 * used FP16 WMMA. */
int spmm_vcsr_mfma(const vcsr_fmt* fmt, const float* dB, int32_t O,
                   float* dC, void* stream, float* ms);

/* Work of the FP32-MFMA kernel for one SpMM of width O with column tile
 * tileK (0 as spmm_vcsr_mfma uses): the MFMA instructions it issues (every
 * group as a dense tile, padding included) and the FLOPs of each.  For
 * reporting MFMA utilisation: useful fraction = 2*nnz*O / (ops*flops_per_op),
 * achieved rate = ops*flops_per_op / time against the FP32 MFMA peak.
 * Host only (no upload needed).  No reference counterpart. */
int vcsr_mfma_work(const vcsr_fmt* fmt, int32_t O, int32_t tileK, int64_t* ops,
                   int32_t* flops_per_op);
/* The same for the tile-stationary kernel on an uploaded format whose view
 * has 16-row tiles (v_mfma_f32_16x16x4f32 per four entries, column tile and
 * column part, padding entries included); ops = 0 for other tile heights.
 * No reference counterpart. */
int vcsr_tile_mfma_work(const vcsr_fmt* fmt, int32_t O, int64_t* ops, int32_t* flops_per_op);

/* What one SpMM of width O with `kernel` (VCSR_KERNEL_AUTO resolved) launches
 * on an uploaded format, for reports that name the timed work.  For the
 * tile-stationary kernel: the row-tile view (tile height, tiles, entries =
 * B-row slice loads per column tile), whether its tiles run on the FP32
 * matrix cores, floats per lane, column slices (one launch each) and their
 * width, reduce-kernel launches and split rows, and the partial-row floats
 * of scratch; other kernels report only `kernel`.  The same for any
 * alignment of B and C.  No reference counterpart. */
typedef struct {
    int32_t kernel;
    int32_t tile_rows;
    int64_t tiles;
    int64_t entries;
    int32_t matrix_cores;
    int32_t vec;
    int32_t column_slices;
    int32_t slice_cols;
    int32_t reduce_launches;
    int32_t split_rows;
    int64_t scratch_floats;
} vcsr_launch_info;
int vcsr_launch_info_get(const vcsr_fmt* fmt, int32_t O, int32_t kernel, vcsr_launch_info* out);

/* ------------------------------------------------------ vendor baseline */
/* rocSPARSE SpMM (CSR int32 x row-major dense, FP32, default algorithm,
 * C = A*B) on caller-owned device arrays: the counterpart of
 * run_cusparse_spmm (src/kernels.cu:169-235), for comparison only.
 * vcsr_vendor_plan_create sets up the handle, descriptors and work buffer
 * (the reference does this inside every call, outside its timed region) and
 * binds the plan to these arrays; vcsr_vendor_spmm computes on `stream` and,
 * if ms is non-NULL, waits and stores the time of the SpMM call alone.
 * spmm_csr_vendor is the one-shot form with the reference's behaviour
 * (returns after the computation).  Failures of the library are
 * VCSR_EDEVICE with its status in vcsr_last_error(). */
typedef struct vcsr_vendor_plan vcsr_vendor_plan;
int vcsr_vendor_plan_create(int32_t M, int32_t N, int32_t nnz, const int32_t* rowptr,
                            const int32_t* col, const float* val, const float* dB,
                            int32_t O, float* dC, void* stream, vcsr_vendor_plan** out);
int vcsr_vendor_spmm(vcsr_vendor_plan* plan, void* stream, float* ms);
void vcsr_vendor_plan_free(vcsr_vendor_plan* plan);
int spmm_csr_vendor(int32_t M, int32_t N, int32_t nnz, const int32_t* rowptr,
                    const int32_t* col, const float* val, const float* dB, int32_t O,
                    float* dC, void* stream, float* ms);

/* CPU CSR SpMM, C = A*B in FP32, for each row: p ascending, k inner, one
 * fused multiply-add per term (the loop order of src/kernels.cu:25-32).
 * nthreads <= 0 uses every hardware thread (rows are independent, so the
 * result does not depend on it).  The reference has no CPU SpMM; its README
 * promises an L2-difference check (README.md:38-39) that needs one. */
int spmm_csr_cpu(int32_t M, const int32_t* rowptr, const int32_t* col,
                 const float* val, const float* B, int32_t O, float* C,
                 int32_t nthreads);

/* -------------------------------------------------- dense operators */
/* What stands next to the sparse product in a layer: the RMS norm of its
 * output and the layer's input, a dense (linear) layer, their gradients, and
 * the optimizer's step.  No counterpart in the reference, which has the sparse
 * product alone.
 *
 * Matrices are row-major on the device with any row stride `ld*` in elements
 * (>= the row length; 0 = rows back to back) and any alignment of their
 * element type; 16-byte aligned rows are the fastest.  A call enqueues kernels
 * on `stream` and nothing else (no allocation, copy or synchronisation), so it
 * can be captured into a HIP graph; with a non-NULL `ms` it waits and stores
 * the kernels' time, as the SpMM calls do.  Calls that overlap in time need
 * workspaces of their own.  Bad arguments are VCSR_EINVAL, sizes or strides
 * past what a kernel addresses VCSR_ERANGE, before any launch.  Results do not
 * vary from call to call: no atomics. */
enum {
    VCSR_F32 = 0,
    VCSR_BF16 = 1,
    VCSR_FP8 = 2 /* OCP e4m3 (largest value 448, no infinities) */
};
enum {
    VCSR_ACT_NONE = 0,
    VCSR_ACT_RELU = 1,
    VCSR_ACT_GELU = 2, /* 0.5 z (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) */
    VCSR_ACT_SILU = 3  /* z / (1 + exp(-z))                               */
};

/* t = x + residual;  y = t / sqrt(mean(t^2) + eps) * weight, row by row, in
 * FP32.  For y of VCSR_FP8, y_scale[m] = max(max_c |y|, 1e-30) / 448 and the
 * codes are y / y_scale[m] rounded to e4m3.  A row with a NaN or an infinity
 * gives NaN for all of y or for what it multiplies, and no other row does.  The
 * sum of a row's squares is FP32's too: past 3.4e38 (all |t| from 1.8e19 on) its
 * rstd and finite y are zero. */
typedef struct {
    int64_t M;           /* rows; 0 is no work                               */
    int32_t C;           /* columns, >= 1                                    */
    int32_t x_type;      /* x, residual, sum: VCSR_F32 or VCSR_BF16          */
    int32_t y_type;      /* VCSR_F32, VCSR_BF16 or VCSR_FP8                  */
    float eps;           /* >= 0                                             */
    const void* x;       int64_t ldx;
    const void* residual; int64_t ldr;  /* NULL: t = x                       */
    const float* weight; /* C                                                */
    void* sum;           int64_t ldsum; /* NULL, or t rounded to x_type; may
                                           be x or residual itself           */
    void* y;             int64_t ldy;   /* may be x or residual itself, if of
                                           one type                          */
    float* y_scale;      /* M, for VCSR_FP8 (NULL otherwise)                 */
    float* rstd;         /* NULL, or M: 1 / sqrt(mean(t^2) + eps)            */
} vcsr_rmsnorm_args;
int vcsr_rmsnorm(const vcsr_rmsnorm_args* args, void* stream, float* ms);

/* Gradients of vcsr_rmsnorm: with s the saved sum (or x), h = s * rstd and
 * g = dy * weight:  dx = dsum + rstd * (g - h * mean(g * h)),
 * dweight = sum over rows of dy * h.  dx is the gradient of x and of the
 * residual alike. */
typedef struct {
    int64_t M;
    int32_t C;
    int32_t x_type;      /* s, dsum, dx: VCSR_F32 or VCSR_BF16               */
    int32_t y_type;      /* dy: VCSR_F32 or VCSR_BF16                        */
    const void* dy;      int64_t lddy;
    const void* s;       int64_t lds;
    const float* weight; /* C                                                */
    const float* rstd;   /* M                                                */
    const void* dsum;    int64_t lddsum; /* NULL, or what flows into `sum`   */
    void* dx;            int64_t lddx;   /* may be dsum, s or dy itself      */
    float* dweight;      /* C (zeros for M = 0), or NULL                     */
    void* workspace;     size_t workspace_bytes;
} vcsr_rmsnorm_grad_args;
/* Bytes of workspace for the sizes and types of `args` (its pointers are not
 * read, except which of them are NULL). */
int vcsr_rmsnorm_grad_workspace(const vcsr_rmsnorm_grad_args* args, size_t* bytes);
int vcsr_rmsnorm_grad(const vcsr_rmsnorm_grad_args* args, void* stream, float* ms);

/* z = x W^T + bias;  y = act(z) + residual.  W has one row per output column.
 * Products are summed in FP32 (FP32 operands on the FP32 matrix cores); VCSR_FP8
 * operands carry a scale per row: z[m][n] = x_scale[m] * w_scale[n] * (x W^T)
 * + bias[n].  y and z are rounded once, and are other matrices than x and w. */
typedef struct {
    int64_t M;           /* rows of x and y; 0 is no work                    */
    int32_t N, K;        /* outputs and inputs of a row, >= 1                */
    int32_t x_type;      /* x and w: VCSR_F32, VCSR_BF16 or VCSR_FP8         */
    int32_t y_type;      /* y, z, residual: VCSR_F32 or VCSR_BF16            */
    int32_t act;         /* VCSR_ACT_*                                       */
    const void* x;       int64_t ldx;
    const void* w;       int64_t ldw;   /* N x K                             */
    const float* x_scale; /* M, for VCSR_FP8 (NULL otherwise)                */
    const float* w_scale; /* N, for VCSR_FP8 (NULL otherwise)                */
    const float* bias;   /* N or NULL                                        */
    const void* residual; int64_t ldr;  /* NULL, or M x N; may be y itself   */
    void* z;             int64_t ldz;   /* NULL, or z for the gradient       */
    void* y;             int64_t ldy;
    void* workspace;     size_t workspace_bytes;
} vcsr_linear_args;
/* Bytes of workspace for the sizes and types of `args` (its pointers are not
 * read, except which of them are NULL). */
int vcsr_linear_workspace(const vcsr_linear_args* args, size_t* bytes);
int vcsr_linear(const vcsr_linear_args* args, void* stream, float* ms);

/* Gradients of vcsr_linear on VCSR_F32 or VCSR_BF16 operands: dz = dy *
 * act'(z), dx = dz W, dw = dz^T x, dbias = sum over rows of dz (the residual's
 * gradient is dy).  For VCSR_BF16 operands dz is rounded to bf16 before the two
 * products (the matrix cores' operand type), an FP32 dy too; dbias sums the
 * unrounded dz.
 * dx and dw are other matrices than those their products read: w for dx, x for dw,
 * for both dy where it is dz as it lies (no activation, x_type = y_type), and
 * each other's operands where both are asked for. */
typedef struct {
    int64_t M;
    int32_t N, K;
    int32_t x_type;      /* x, w, dx, dw: VCSR_F32 or VCSR_BF16              */
    int32_t y_type;      /* dy, z: VCSR_F32 or VCSR_BF16                     */
    int32_t act;
    const void* dy;      int64_t lddy;
    const void* z;       int64_t ldz;   /* may be NULL for VCSR_ACT_NONE     */
    const void* x;       int64_t ldx;   /* needed for dw                     */
    const void* w;       int64_t ldw;   /* needed for dx                     */
    void* dx;            int64_t lddx;  /* M x K, or NULL                    */
    void* dw;            int64_t lddw;  /* N x K (zeros for M = 0), or NULL  */
    float* dbias;        /* N (zeros for M = 0), or NULL                     */
    void* workspace;     size_t workspace_bytes;
} vcsr_linear_grad_args;
/* As vcsr_linear_workspace. */
int vcsr_linear_grad_workspace(const vcsr_linear_grad_args* args, size_t* bytes);
int vcsr_linear_grad(const vcsr_linear_grad_args* args, void* stream, float* ms);

/* AdamW over all tensors of a model in one launch.  With g = grad_scale *
 * grad:  m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,
 * param = param (1 - lr weight_decay)
 *         - lr / (1 - beta1^step) * m / (sqrt(v / (1 - beta2^step)) + eps).
 * States are FP32, or VCSR_FP8 with one FP32 scale per block of 256
 * consecutive values of a tensor (the last block may be shorter): m holds
 * m / m_scale, v holds sqrt(v) / v_scale, each scale is max(largest magnitude
 * of the block, 1e-30) / 448, and a nonzero sqrt(v) is stored as the smallest
 * code (2^-9) where it would round to zero, so that no step divides by a lost
 * v.  All zero bytes are a valid fresh state of either type. */
typedef struct {
    int64_t n;           /* values; 0 is allowed                             */
    int32_t grad_type;   /* VCSR_F32 or VCSR_BF16                            */
    int32_t state_type;  /* VCSR_F32 or VCSR_FP8                             */
    float* param;
    const void* grad;
    void *m, *v;
    float *m_scale, *v_scale; /* ceil(n / 256) each, for VCSR_FP8            */
    void* copy;          /* NULL, or n values: param rounded to bf16         */
    double weight_decay;
} vcsr_adamw_tensor;
/* Held in 64 bits until the step's FP32 constants (1 - beta1, lr / (1 -
 * beta1^step), ...) are formed from them, each rounded once. */
typedef struct {
    double lr, beta1, beta2, eps, grad_scale;
    int64_t step;        /* 1 for the first */
} vcsr_adamw_hyper;
typedef struct vcsr_adamw vcsr_adamw;
/* Binds the tensors' addresses (they stay the caller's) to a plan on the
 * current device; tensors must not overlap.  A step only enqueues its kernel.
 * All tensors together have fewer than 2^24 chunks of up to 2048 values. */
int vcsr_adamw_create(const vcsr_adamw_tensor* tensors, int32_t count, void* stream,
                      vcsr_adamw** out);
int vcsr_adamw_step(const vcsr_adamw* plan, const vcsr_adamw_hyper* hyper, void* stream,
                    float* ms);
void vcsr_adamw_free(vcsr_adamw* plan);

/* --------------------------------------------------- device plumbing */
/* Minimal HIP helpers so hosts (ctypes, the CLI) need no other GPU runtime. */
int vcsr_device_count(int32_t* n);
/* The calling thread's device. */
int vcsr_device_current(int32_t* device);
int vcsr_device_name(char* buf, int32_t len);
int vcsr_dev_malloc(void** ptr, size_t bytes);
int vcsr_dev_free(void* ptr);
int vcsr_memcpy_h2d(void* dst, const void* src, size_t bytes, void* stream);
int vcsr_memcpy_d2h(void* dst, const void* src, size_t bytes, void* stream);
/* Device-to-device copy, enqueued on `stream` (not waited for). */
int vcsr_memcpy_d2d(void* dst, const void* src, size_t bytes, void* stream);
int vcsr_memset_d(void* dst, int32_t value, size_t bytes, void* stream);
int vcsr_stream_create(void** stream);
int vcsr_stream_destroy(void* stream);
int vcsr_stream_sync(void* stream);
int vcsr_device_sync(void);
int vcsr_event_create(void** event);
int vcsr_event_destroy(void* event);
int vcsr_event_record(void* event, void* stream);
int vcsr_event_elapsed(void* start, void* stop, float* ms);

#ifdef __cplusplus
}
#endif
#endif /* VCSR_SPMM_H */
