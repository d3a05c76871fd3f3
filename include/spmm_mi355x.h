/*
 * spmm_mi355x.h — C ABI of the MI355X (gfx950) SpMM library `libspmm_mi355x.so`.
 *
 * This is the drop-in boundary for the SpMM hot path of Ascend-SpMM.  Every
 * entry point below replaces one call site of the reference's CANN/aclnn
 * layer or one of its host-side preprocessing routines; the citation next to
 * each declaration names the reference code it stands in for (paths are
 * relative to the Ascend-SpMM repository root).
 *
 * Conventions
 *  - Plain pointers and sizes only; no C++ or torch types cross this boundary.
 *  - All device pointers are HIP device memory owned by the caller.  The
 *    library never allocates device memory for its outputs; scratch space is
 *    the caller-provided workspace, sized by the matching *_workspace call.
 *  - Launches are asynchronous on the given stream unless the comment says
 *    the call synchronises (the *_plan calls read a few sizes back).
 *  - Index arrays of one call share one index type (int32 or int64); value
 *    arrays and the dense operand share one value type (fp16 or fp32).
 *  - Kernels never read outside the extents passed in: row pointers are
 *    clamped to the index arrays and out-of-range column ids contribute zero.
 *  - On failure a call returns a non-zero spmm_status and records a message
 *    retrievable (per thread) with spmm_last_error().
 *  - Reentrant: calls on different streams may run concurrently.
 */
#ifndef SPMM_MI355X_H_
#define SPMM_MI355X_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes.  Each maps to one Python exception type in the extension,
 * matching what the reference raises for the same condition:
 * INVALID_ARGUMENT -> ValueError   (std::invalid_argument in the reference)
 * OUT_OF_RANGE     -> IndexError   (std::out_of_range)
 * OVERFLOW         -> OverflowError(std::overflow_error)
 * CONTRACT         -> RuntimeError (TORCH_CHECK failures)
 * DEVICE           -> RuntimeError (a HIP runtime error) */
typedef enum spmm_status {
  SPMM_OK = 0,
  SPMM_ERR_INVALID_ARGUMENT = 1,
  SPMM_ERR_OUT_OF_RANGE = 2,
  SPMM_ERR_OVERFLOW = 3,
  SPMM_ERR_CONTRACT = 4,
  SPMM_ERR_DEVICE = 5
} spmm_status;

typedef enum spmm_index_type { SPMM_INDEX_I32 = 0, SPMM_INDEX_I64 = 1 } spmm_index_type;
/* BF16: the dense operators and those around experts only. */
typedef enum spmm_value_type {
  SPMM_VALUE_F16 = 0,
  SPMM_VALUE_F32 = 1,
  SPMM_VALUE_F64 = 2,
  SPMM_VALUE_BF16 = 3
} spmm_value_type;

/* Opaque HIP stream (hipStream_t); NULL is the default stream. */
typedef void* spmm_stream;

/* Message of the last failed call on this thread ("" if none). */
const char* spmm_last_error(void);

/* Library version string, e.g. "spmm_mi355x 0.1 gfx950". */
const char* spmm_version(void);

/* ------------------------------------------------------------------------
 * spmm_csr — C[M,N] = A[M,K] (CSR) x dense[K,N]
 *
 * Replaces EXEC_NPU_CMD(aclnnSpmmCsr, ...) in spmm_csr_impl_npu
 * (extension/custom_op.cpp:67-88) and the tiling + kernel behind it
 * (kernels/op_host/spmm_csr.cpp:8-35, kernels/op_kernel/spmm_csr.cpp:226-569).
 * The reference's per-core `start` array is a tiling aid; the MI355X kernel
 * partitions on the device, so `start` is not an argument here.
 *
 * Every output row is written (rows without nonzeros become zero), so `out`
 * need not be cleared.  Each row is accumulated in fp32 in nonzero order and
 * rounded once to the value type (round-to-nearest-even).  Rows longer than
 * the library's fixed split length are cut at split points that depend only
 * on the row pointer, and their fp32 pieces are added in order, so results are
 * deterministic and identical for every feature width N.
 * ---------------------------------------------------------------------- */
typedef struct spmm_csr_desc {
  int64_t rows;        /* M: rowptr holds rows + 1 entries                 */
  int64_t nnz;         /* extent of col[] and value[]                      */
  int64_t dense_rows;  /* K: rows of dense                                 */
  int64_t width;       /* N: columns of dense and out (row-major, contiguous) */
  int32_t index_type;  /* spmm_index_type                                  */
  int32_t value_type;  /* spmm_value_type (F16 or F32)                     */
} spmm_csr_desc;

spmm_status spmm_csr_workspace(const spmm_csr_desc* desc, size_t* bytes);

spmm_status spmm_csr_run(const spmm_csr_desc* desc,
                         const void* rowptr, const void* col, const void* value,
                         const void* dense, void* out,
                         void* workspace, size_t workspace_bytes,
                         spmm_stream stream);

/* Allocation-free spmm_csr: same arguments (minus the workspace), same
 * kernels and bit-identical results as spmm_csr_run.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Its scratch is a fixed device array inside the library, of
 * spmm_csr_noalloc_max_scratch() bytes (64 MiB) per GPU, held from the
 * library's load until the process ends; the call allocates nothing.  A call
 * whose scratch (spmm_csr_workspace's figure) exceeds it fails with
 * SPMM_ERR_CONTRACT before touching the device.  Every call on one GPU shares
 * that GPU's array, so calls that overlap on one GPU (different streams, or
 * host threads, without ordering between them) race and must not be made.
 * The first call on each device looks up the array's device address
 * (hipGetSymbolAddress) and keeps it; make that first call outside stream
 * capture (one eager call before capturing), so that no capture sees the
 * lookup.  Later calls only launch kernels and may be captured. */
size_t spmm_csr_noalloc_max_scratch(void);

spmm_status spmm_csr_run_noalloc(const spmm_csr_desc* desc,
                                 const void* rowptr, const void* col, const void* value,
                                 const void* dense, void* out, spmm_stream stream);

/* Gather-rate probe.  No counterpart in the reference: a measurement for
 * callers judging spmm_csr_run against what the GPU can gather.  It runs the
 * dense-row gathers of spmm_csr_run over the same nonzeros (column ids and
 * values staged per tile, one 16-byte piece of every nonzero's dense row per
 * lane, fp32 FMAs) without the row bookkeeping, partial sums or output rows,
 * and writes one float per thread to `sink` (spmm_gather_probe_sink(desc)
 * floats, 16-byte aligned).  int32 column ids; dense operand up to 4 GB;
 * rowptr is not read. */
size_t spmm_gather_probe_sink(const spmm_csr_desc* desc);

spmm_status spmm_gather_probe(const spmm_csr_desc* desc, const void* col, const void* value,
                              const void* dense, float* sink, spmm_stream stream);

/* Thread-per-row scalar CSR SpMM, same arguments and result contract as
 * spmm_csr_run (same sums in the same order within a row; no workspace).
 * No counterpart in the reference: it is the baseline that the block path's
 * speed-up is stated against (one thread per output row, nonzeros in order,
 * 16-byte pieces of the dense row), for callers comparing kernels. */
spmm_status spmm_csr_rowscalar_run(const spmm_csr_desc* desc,
                                   const void* rowptr, const void* col, const void* value,
                                   const void* dense, void* out, spmm_stream stream);

/* ------------------------------------------------------------------------
 * spmm_mixed — the spmm_ascend_cube operator:
 *   out[16*s + r, :]  = sum_{b in [Crowptr[s], Crowptr[s+1])} Cvalue[16*b + r] * dense[Ccol[b], :]
 *   out[i, :]        += sum_{p in [Vrowptr[i], Vrowptr[i+1])} Vvalue[p] * dense[Vcol[p], :]
 * with out rows = max(16 * block_windows, vector_rows).
 *
 * Replaces EXEC_NPU_CMD(aclnnSpmmAscendCube, ...) in spmm_ascend_cube_impl_npu
 * (extension/custom_op.cpp:115-152), its tiling
 * (kernels/op_host/spmm_ascend_cube.cpp:8-51) and the mixed AIC/AIV kernel
 * (kernels/op_kernel/spmm_ascend_cube.cpp:16-311, 543-907).  The per-core
 * Cstart/Vstart arrays of the reference are not needed.
 *
 * The block part (16x1 BCSR windows) runs on fp16/fp32 MFMA.  The vector
 * part runs the CSR gather path of spmm_csr first; for rows of block windows
 * that have blocks it leaves the fp32 vector sum in the workspace, and the
 * block kernel adds it after the block sum and rounds once.  With
 * block_windows == 0 the result is bit-identical to spmm_csr on the same CSR.
 * Every output row is written.  dense, out and Cvalue must be 16-byte
 * aligned (SPMM_ERR_CONTRACT otherwise).
 * ---------------------------------------------------------------------- */
typedef struct spmm_mixed_desc {
  int64_t block_windows;  /* Crowptr.numel - 1                              */
  int64_t block_count;    /* Ccol_ids.numel                                 */
  int64_t block_values;   /* Cvalue.numel (>= 16 * blocks referenced)       */
  int64_t vector_rows;    /* Vrowptr.numel - 1                              */
  int64_t vector_nnz;     /* min(Vcol_ids.numel, Vvalue.numel)              */
  int64_t dense_rows;     /* K                                              */
  int64_t width;          /* N                                              */
  int32_t index_type;
  int32_t value_type;
} spmm_mixed_desc;

spmm_status spmm_mixed_workspace(const spmm_mixed_desc* desc, size_t* bytes);

spmm_status spmm_mixed_run(const spmm_mixed_desc* desc,
                           const void* Crowptr, const void* Ccol, const void* Cvalue,
                           const void* Vrowptr, const void* Vcol, const void* Vvalue,
                           const void* dense, void* out,
                           void* workspace, size_t workspace_bytes,
                           spmm_stream stream);

/* Number of output rows spmm_mixed_run writes: max(16*block_windows, vector_rows). */
int64_t spmm_mixed_out_rows(const spmm_mixed_desc* desc);

/* ------------------------------------------------------------------------
 * spmm_cube_op — the legacy spmm_cube operator.  Window w (16 output rows)
 * owns nonzeros [rowptr[w], rowptr[w+1]); each carries col = (c << 4) | r,
 * c the dense row and r the row inside the window.  Maximal runs of
 * consecutive nonzeros with equal c form one 16x1 block whose row r is the
 * value of the run's last nonzero with row r:
 *   out[16*w + r, :] = sum over window w's runs of block[r] * dense[c, :]
 * with out rows = 16 * windows, every row written.  Replaces
 * EXEC_NPU_CMD(aclnnSpmmCube, ...) in spmm_cube_impl_npu
 * (extension/custom_op.cpp:91-113) and its kernel
 * (kernels/op_kernel/spmm_cube.cpp:53-146).  Decoded on the device into the
 * block layout of spmm_mixed_run and run on its MFMA block kernel.  c outside
 * [0, dense_rows) contributes zero.  Width contract: 0 < N <= 1024 (fp16) or
 * 512 (fp32), N % 16 == 0; dense and out 16-byte aligned; nnz < 2^31 - 1.
 * The workspace holds the decoded blocks (16 values per nonzero at most).
 * ---------------------------------------------------------------------- */
typedef struct spmm_cube_op_desc {
  int64_t windows;     /* rowptr.numel - 1                                */
  int64_t nnz;         /* col.numel (== value.numel)                      */
  int64_t dense_rows;  /* K                                               */
  int64_t width;       /* N                                               */
  int32_t index_type;
  int32_t value_type;
} spmm_cube_op_desc;

spmm_status spmm_cube_op_workspace(const spmm_cube_op_desc* desc, size_t* bytes);

spmm_status spmm_cube_op_run(const spmm_cube_op_desc* desc,
                             const void* rowptr, const void* col, const void* value,
                             const void* dense, void* out,
                             void* workspace, size_t workspace_bytes,
                             spmm_stream stream);

/* ------------------------------------------------------------------------
 * Row permutation of a node tensor (P and P^T of the graph layout).
 *
 * spmm_pack_rows:    packed[inv[i], :] = src[i, :] for i < rows; every other
 *                    packed row is zero (if inv repeats a packed row, the
 *                    largest i wins).  Replaces pack_node_tensor's
 *                    new_zeros + index_copy_ (spmm_npu.py:23-47).  Needs a
 *                    workspace of spmm_pack_workspace(packed_rows) bytes.
 * spmm_restore_rows: dst[i, :] = packed[inv[i], :].  Replaces
 *                    restore_node_tensor's index_select (spmm_npu.py:50-62).
 * `row_bytes` is the byte size of one row (any element type).  `inv` is int64.
 * Entries of inv outside [0, packed_rows) are skipped by pack and give a zero
 * row in restore (the Python layer rejects them before the call, as the
 * reference does).
 * ---------------------------------------------------------------------- */
size_t spmm_pack_workspace(int64_t packed_rows);

spmm_status spmm_pack_rows(const void* src, int64_t rows, int64_t row_bytes,
                           const int64_t* inv, void* packed, int64_t packed_rows,
                           void* workspace, size_t workspace_bytes,
                           spmm_stream stream);

spmm_status spmm_restore_rows(const void* packed, int64_t packed_rows, int64_t row_bytes,
                              const int64_t* inv, int64_t rows, void* dst,
                              spmm_stream stream);

/* ------------------------------------------------------------------------
 * Preprocessing on the GPU (layout conversion and work partitioning).
 *
 * The reference runs these on the host with ATen accessors; here they are
 * device pipelines whose outputs are bit-identical to the reference's
 * (integer arrays, and values copied bit for bit).  Index outputs use the
 * input's index type; permutations are int64.
 *
 * Each conversion is two calls on the same workspace:
 *   *_workspace(...)  bytes of workspace (depends only on the sizes)
 *   *_plan(...)       runs the pipeline into the workspace and returns the
 *                     output sizes (synchronises the stream)
 *   *_fill(...)       writes the outputs into caller buffers of those sizes
 * Input requirements (checked on the device, reported by *_plan):
 *   row pointer monotone within [0, nnz]  -> SPMM_ERR_INVALID_ARGUMENT
 *   column ids in [0, cols)               -> SPMM_ERR_CONTRACT
 *   (bcsr / cube) ascending columns per row, as the reference's docs
 *   require (extension/custom_op.cpp:1430,1440) -> SPMM_ERR_INVALID_ARGUMENT
 * ---------------------------------------------------------------------- */
typedef struct spmm_csr_matrix {
  int64_t rows;        /* rowptr holds rows + 1 entries                    */
  int64_t cols;
  int64_t nnz;         /* extent of col[] and value[]                      */
  int32_t index_type;  /* spmm_index_type                                  */
  int32_t value_type;  /* spmm_value_type: F16, F32 or F64 (copied only)   */
  const void* rowptr;  /* device pointers                                  */
  const void* col;
  const void* value;
} spmm_csr_matrix;

/* A plan's few host-side numbers.  *_plan stores them at the head of the
 * workspace for its *_fill, which reads them back (a synchronisation each);
 * *_plan_record returns them to the caller instead, and *_fill_record takes
 * them, so a conversion synchronises once.  A record goes with the workspace
 * and the matrix of its plan.  Opaque. */
typedef struct spmm_plan_record {
  int64_t words[16];
} spmm_plan_record;

/* csr_to_bcsr: BCSR(16x1).  Replaces ToBCSR / csr_to_bcsr
 * (extension/custom_op.cpp:594-746).  Outputs: crow_window_ptr[nwin+1],
 * unique_col_ids[blocks], value[16*blocks], nwin = ceil(rows/window_size),
 * 1 <= window_size <= 16. */
size_t spmm_bcsr_workspace(const spmm_csr_matrix* m, int64_t window_size);
spmm_status spmm_bcsr_plan(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                           size_t workspace_bytes, spmm_stream stream, int64_t* blocks);
spmm_status spmm_bcsr_fill(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                           size_t workspace_bytes, void* crow_window_ptr, void* unique_col_ids,
                           void* value, spmm_stream stream);
spmm_status spmm_bcsr_plan_record(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                                  size_t workspace_bytes, spmm_stream stream, int64_t* blocks,
                                  spmm_plan_record* record);
spmm_status spmm_bcsr_fill_record(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                                  size_t workspace_bytes, const spmm_plan_record* record,
                                  void* crow_window_ptr, void* unique_col_ids, void* value,
                                  spmm_stream stream);

/* csr_to_ascend_cube: 16x16 cube tiles.  Replaces your_logic_kernel /
 * csr_to_ascend_cube (extension/custom_op.cpp:429-592).  Outputs:
 * crow_window_ptr[nwin+1] (tile offsets), unique_col_ids[16*tiles] (zero
 * padded per window), value[256*tiles]. */
size_t spmm_cube_workspace(const spmm_csr_matrix* m, int64_t window_size);
spmm_status spmm_cube_plan(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                           size_t workspace_bytes, spmm_stream stream, int64_t* tiles);
spmm_status spmm_cube_fill(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                           size_t workspace_bytes, void* crow_window_ptr, void* unique_col_ids,
                           void* value, spmm_stream stream);
spmm_status spmm_cube_plan_record(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                                  size_t workspace_bytes, spmm_stream stream, int64_t* tiles,
                                  spmm_plan_record* record);
spmm_status spmm_cube_fill_record(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                                  size_t workspace_bytes, const spmm_plan_record* record,
                                  void* crow_window_ptr, void* unique_col_ids, void* value,
                                  spmm_stream stream);

/* block_level_split: density-threshold BCSR(window_size x 1) + CSR split.
 * Replaces hybrid_split_impl / block_level_split
 * (extension/custom_op.cpp:1139-1348, 1390-1412).  Outputs:
 * crow_window_ptr[nwin+1], unique_col_ids[kept_blocks],
 * value[window_size*kept_blocks], vrow_window_ptr[window_size*nwin+1],
 * vcol_indices[vector_nnz], vvalue[vector_nnz]. */
size_t spmm_hybrid_workspace(const spmm_csr_matrix* m, int64_t window_size);
spmm_status spmm_hybrid_plan(const spmm_csr_matrix* m, double a, int64_t window_size,
                             void* workspace, size_t workspace_bytes, spmm_stream stream,
                             int64_t* kept_blocks, int64_t* vector_nnz);
spmm_status spmm_hybrid_fill(const spmm_csr_matrix* m, double a, int64_t window_size,
                             void* workspace, size_t workspace_bytes, void* crow_window_ptr,
                             void* unique_col_ids, void* value, void* vrow_window_ptr,
                             void* vcol_indices, void* vvalue, spmm_stream stream);
spmm_status spmm_hybrid_plan_record(const spmm_csr_matrix* m, double a, int64_t window_size,
                                    void* workspace, size_t workspace_bytes, spmm_stream stream,
                                    int64_t* kept_blocks, int64_t* vector_nnz,
                                    spmm_plan_record* record);
spmm_status spmm_hybrid_fill_record(const spmm_csr_matrix* m, int64_t window_size, void* workspace,
                                    size_t workspace_bytes, const spmm_plan_record* record,
                                    void* crow_window_ptr, void* unique_col_ids, void* value,
                                    void* vrow_window_ptr, void* vcol_indices, void* vvalue,
                                    spmm_stream stream);

/* preprocess: the 295/505 cost-model AIC/AIV task mapping with the marginal
 * window split, row permutation and (graph_layout on a square matrix) the
 * renumbered columns and the fixed-layout transpose P*A^T*P^T.  Replaces
 * taskmapping / preprocess (extension/custom_op.cpp:749-1137, with
 * boundary_bucket_sort.h and packed_column_reindex.h).  window_size must be
 * 16 (SPMM_ERR_CONTRACT otherwise, as the reference's TORCH_CHECK). */
typedef struct spmm_taskmap_info {
  int64_t aic_windows;            /* crow_window_ptr: aic_windows + 1       */
  int64_t aic_blocks;             /* unique_col_ids; value: 16*aic_blocks   */
  int64_t packed_rows;            /* vrow_window_ptr: packed_rows + 1; permutation */
  int64_t vector_nnz;             /* vcol_indices, vvalue                   */
  int64_t packed_layout_supported;
  int64_t marginal_window;        /* -1 if none                             */
  int64_t marginal_aic_blocks;
  int64_t marginal_total_blocks;
  int64_t shared_windows;
  double estimated_aic_cost;
  double estimated_aiv_cost;
  double estimated_max_cost;
  /* transpose_* (graph layout only; all 0 otherwise)                     */
  int64_t t_windows;              /* transpose_crow_window_ptr: t_windows+1 */
  int64_t t_blocks;               /* transpose_unique_col_ids; value 16*t_blocks */
  int64_t t_rows;                 /* transpose_vrow_window_ptr: t_rows + 1  */
  int64_t t_vector_nnz;
} spmm_taskmap_info;

typedef struct spmm_taskmap_out {
  void* crow_window_ptr;
  void* unique_col_ids;
  void* value;
  void* vrow_window_ptr;
  void* vcol_indices;
  void* vvalue;
  void* renumbered_unique_col_ids;  /* graph layout: aic_blocks entries   */
  void* renumbered_vcol_indices;    /* graph layout: vector_nnz entries   */
  void* transpose_crow_window_ptr;
  void* transpose_unique_col_ids;
  void* transpose_value;
  void* transpose_vrow_window_ptr;
  void* transpose_vcol_indices;
  void* transpose_vvalue;
  int64_t* permutation;             /* packed_rows entries (-1 = padding)  */
  int64_t* inv_permutation;         /* rows entries                        */
} spmm_taskmap_out;

size_t spmm_taskmap_workspace(const spmm_csr_matrix* m, int64_t window_size, int graph_layout);
spmm_status spmm_taskmap_plan(const spmm_csr_matrix* m, int64_t window_size, int graph_layout,
                              void* workspace, size_t workspace_bytes, spmm_stream stream,
                              spmm_taskmap_info* info);
spmm_status spmm_taskmap_fill(const spmm_csr_matrix* m, int64_t window_size, int graph_layout,
                              void* workspace, size_t workspace_bytes,
                              const spmm_taskmap_out* out, spmm_stream stream);
spmm_status spmm_taskmap_plan_record(const spmm_csr_matrix* m, int64_t window_size,
                                     int graph_layout, void* workspace, size_t workspace_bytes,
                                     spmm_stream stream, spmm_taskmap_info* info,
                                     spmm_plan_record* record);
spmm_status spmm_taskmap_fill_record(const spmm_csr_matrix* m, int64_t window_size,
                                     int graph_layout, void* workspace, size_t workspace_bytes,
                                     const spmm_plan_record* record, const spmm_taskmap_out* out,
                                     spmm_stream stream);

/* Stores info's numbers in one launch, each to a device buffer of one element:
 * ints = packed_rows, packed_layout_supported, marginal_window,
 * marginal_aic_blocks, marginal_total_blocks, shared_windows; doubles =
 * estimated aic, aiv and max cost. */
spmm_status spmm_taskmap_scalars(const spmm_taskmap_info* info, int64_t* const* ints,
                                 double* const* doubles, spmm_stream stream);

/* ------------------------------------------------------------------------
 * Dense operators of a graph layer with typed nodes, for training on the
 * graphs that the operators above multiply with.  No counterpart in the
 * reference.  Values are F16, BF16 or F32; every sum is held in fp32 or more
 * and each output is rounded once.  Row strides are in elements, the last
 * dimension is contiguous, and no alignment beyond the element's is required.
 * ---------------------------------------------------------------------- */

/* layer_norm: y = (x - mean) * rstd * weight + bias over each row of x, with
 * rstd = 1 / sqrt(var + eps) and the biased variance.  weight and bias hold
 * `width` values of param_type (value_type or F32); NULL stands for 1 and 0.
 * mean and rstd (fp32, one per row) are written where not NULL; the gradient
 * takes them. */
typedef struct spmm_norm_desc {
  int64_t rows;
  int64_t width;
  int64_t x_stride;     /* elements between rows of x                      */
  int64_t grad_stride;  /* elements between rows of grad (gradient only)   */
  double eps;
  int32_t value_type;   /* x, y, grad, dx                                  */
  int32_t param_type;   /* weight, bias, dweight, dbias                    */
} spmm_norm_desc;

spmm_status spmm_layer_norm_run(const spmm_norm_desc* desc, const void* x, const void* weight,
                                const void* bias, void* y, float* mean, float* rstd,
                                spmm_stream stream);

/* Gradient of layer_norm with respect to x, weight and bias, from the
 * incoming gradient `grad` and the forward call's mean and rstd; each of dx,
 * dweight and dbias may be NULL.  The sums over rows are added in an order
 * that depends on the sizes alone, so results repeat exactly. */
spmm_status spmm_layer_norm_grad_workspace(const spmm_norm_desc* desc, size_t* bytes);
spmm_status spmm_layer_norm_grad_run(const spmm_norm_desc* desc, const void* x, const void* weight,
                                     const float* mean, const float* rstd, const void* grad,
                                     void* dx, void* dweight, void* dbias, void* workspace,
                                     size_t workspace_bytes, spmm_stream stream);

/* grouped_matmul: out[r] = x[r] * weight[g] for the rows r of group g, that
 * is offsets[g] <= r < offsets[g + 1].  offsets (device memory, `groups` + 1
 * ascending entries of index_type) may leave groups empty; rows before
 * offsets[0] and from offsets[groups] on become zero.  weight[g] is
 * inner x width, at weight + g * weight_stride; transposed: stored as
 * width x inner, each group's matrix contiguous either way.  inner, width and
 * the row strides are below 2^22, rows below 2^31, groups at most 2^24.  A single
 * row's strides are not used.  The forward call's workspace is 0 bytes. */
typedef struct spmm_grouped_desc {
  int64_t rows;           /* of x, out and grad                            */
  int64_t groups;
  int64_t inner;          /* columns of x                                  */
  int64_t width;          /* columns of out                                */
  int64_t x_stride;       /* elements between rows of x                    */
  int64_t grad_stride;    /* elements between rows of grad (gradients only) */
  int64_t weight_stride;  /* elements between the groups' matrices         */
  int32_t weight_transposed;
  int32_t index_type;
  int32_t value_type;
} spmm_grouped_desc;

spmm_status spmm_grouped_workspace(const spmm_grouped_desc* desc, size_t* bytes);
spmm_status spmm_grouped_run(const spmm_grouped_desc* desc, const void* x, const void* weight,
                             const void* offsets, void* out, void* workspace,
                             size_t workspace_bytes, spmm_stream stream);

/* Its gradients: dx[r] = grad[r] * weight[g]^T (zero outside the groups), and
 * dweight[g] = x_g^T * grad_g (zero for an empty group), contiguous and in
 * weight's storage order.  dx or dweight may be NULL. */
spmm_status spmm_grouped_grad_workspace(const spmm_grouped_desc* desc, size_t* bytes);
spmm_status spmm_grouped_grad_run(const spmm_grouped_desc* desc, const void* x, const void* weight,
                                  const void* offsets, const void* grad, void* dx, void* dweight,
                                  void* workspace, size_t workspace_bytes, spmm_stream stream);

/* orthogonalize: `steps` Newton-Schulz steps on each of `batch` matrices of
 * rows x width (contiguous, extents below 2^22).  X = update / (|update|_F + eps), then each step
 * replaces X by a X + (b A + c A A) X with A = X X^T (for more rows than
 * columns the same polynomial from the right).  coefficients: 3 * steps host
 * values (a, b, c of each step).  out may be update itself.  X is held in fp32;
 * the products' factors have 22 bits or more, a BF16 update's 11 where
 * min(rows, width) >= 128, unless `precise` is set. */
typedef struct spmm_orthogonalize_desc {
  int64_t batch;
  int64_t rows;
  int64_t width;
  int64_t steps;
  const double* coefficients;
  double eps;
  int32_t value_type;
  int32_t precise;  /* not 0: factors of 22 bits for BF16 too                */
} spmm_orthogonalize_desc;

spmm_status spmm_orthogonalize_workspace(const spmm_orthogonalize_desc* desc, size_t* bytes);
spmm_status spmm_orthogonalize_run(const spmm_orthogonalize_desc* desc, const void* update,
                                   void* out, void* workspace, size_t workspace_bytes,
                                   spmm_stream stream);

/* ------------------------------------------------------------------------
 * Operators around a layer of experts: rows of a table by ids, the experts of
 * each row from a router's logits, rows brought to their experts (whose ranges
 * spmm_grouped_run takes) and back, and log probabilities of labels.  Types,
 * sums and strides as above.  Launches only: all of them may be captured.
 * ---------------------------------------------------------------------- */

/* embedding: out[i] = scale * weight[ids[i]], a row of zeros for an id outside
 * [0, table_rows).  ids and table rows below 2^30, the width below 2^22. */
typedef struct spmm_embedding_desc {
  int64_t count;          /* ids, and rows of out and grad                 */
  int64_t table_rows;
  int64_t width;
  int64_t weight_stride;  /* elements between rows of weight               */
  int64_t grad_stride;    /* elements between rows of grad (gradient only) */
  double scale;           /* finite in fp32                                */
  int32_t index_type;
  int32_t value_type;
} spmm_embedding_desc;

spmm_status spmm_embedding_run(const spmm_embedding_desc* desc, const void* weight, const void* ids,
                               void* out, spmm_stream stream);

/* Its gradient: dweight[v] = scale * the sum of grad[i] over ids[i] = v in the
 * order of i, every row of the contiguous table_rows x width written. */
spmm_status spmm_embedding_grad_workspace(const spmm_embedding_desc* desc, size_t* bytes);
spmm_status spmm_embedding_grad_run(const spmm_embedding_desc* desc, const void* ids, const void* grad,
                                    void* dweight, void* workspace, size_t workspace_bytes,
                                    spmm_stream stream);

typedef enum spmm_score { SPMM_SCORE_SOFTMAX = 0, SPMM_SCORE_SIGMOID = 1 } spmm_score;

/* route: the top_k experts of each row by score + bias, best first, ties to the
 * lowest index, and their weights: scale * score, divided by the sum of the
 * chosen scores where `renormalize` is set.  bias (fp32, one an expert, NULL
 * for none) has no part in the weights.  With groups > 1 the experts are that
 * many equal consecutive groups, and only those of the top_groups groups with
 * the greatest sums of their two best values are chosen from.  An expert whose
 * logit or bias is -inf is never chosen; where fewer than top_k are left, the
 * rest of `chosen` is -1 and their weights 0.  NaN counts as greatest.
 * Values are compared in 64 bits (the logits themselves without bias and
 * groups).  stats (fp32, 2 a row, or NULL) is what the gradient of a softmax
 * that is not renormalised takes. */
typedef struct spmm_route_desc {
  int64_t rows;
  int64_t experts;        /* 1 to 1024                                     */
  int64_t logits_stride;  /* elements between rows of logits               */
  int64_t top_k;          /* 1 to 64                                       */
  int64_t groups;         /* 1 to 64, divides the experts                  */
  int64_t top_groups;
  double scale;           /* positive, a normal fp32 number                */
  int32_t score;          /* spmm_score                                    */
  int32_t renormalize;
  int32_t value_type;     /* logits and dlogits                            */
} spmm_route_desc;

spmm_status spmm_route_run(const spmm_route_desc* desc, const void* logits, const float* bias,
                           float* weights, int32_t* chosen, float* stats, spmm_stream stream);

/* Gradient with respect to the logits (contiguous), from that of the weights. */
spmm_status spmm_route_grad_run(const spmm_route_desc* desc, const void* logits, const int32_t* chosen,
                                const float* weights, const float* stats, const float* grad,
                                void* dlogits, spmm_stream stream);

/* Plan of rows for experts: the `choices` expert ids sorted by expert, equal
 * ones in their order, those outside [0, experts) behind all.  place[i] is the
 * packed row of choice i, offsets[e] to offsets[e + 1] are expert e's packed
 * rows.  choices below 2^31, experts 1 to 2048. */
spmm_status spmm_expert_plan_workspace(int64_t choices, int64_t experts, size_t* bytes);
spmm_status spmm_expert_plan_run(int32_t index_type, const void* ids, int64_t choices, int64_t experts,
                                 int32_t* offsets, int32_t* place, void* workspace,
                                 size_t workspace_bytes, spmm_stream stream);

/* With the plan of `rows` x top_k choices: packed[place[r][j]] = x[r], zero for
 * a choice of no expert, and its gradient dx[r] = sum over j of
 * grad[place[r][j]].  Packed tensors have rows * top_k rows. */
typedef struct spmm_experts_desc {
  int64_t rows;
  int64_t top_k;          /* choices a row, 1 to 64                        */
  int64_t experts;        /* of the plan                                   */
  int64_t width;
  int64_t stride;         /* elements between rows of the first tensor     */
  int64_t grad_stride;    /* of grad (spmm_expert_restore_grad_run only)   */
  int32_t value_type;
} spmm_experts_desc;

spmm_status spmm_expert_pack_run(const spmm_experts_desc* desc, const void* x, const int32_t* place,
                                 const int32_t* offsets, void* packed, spmm_stream stream);
spmm_status spmm_expert_pack_grad_run(const spmm_experts_desc* desc, const void* grad,
                                      const int32_t* place, const int32_t* offsets, void* dx,
                                      spmm_stream stream);

/* out[r] = sum over j of weights[r][j] * y[place[r][j]] (fp32 weights; nothing
 * for a choice of no expert), and its gradients: dy (rows of no expert zero)
 * and dweights, either may be NULL. */
spmm_status spmm_expert_restore_run(const spmm_experts_desc* desc, const void* y, const float* weights,
                                    const int32_t* place, const int32_t* offsets, void* out,
                                    spmm_stream stream);
spmm_status spmm_expert_restore_grad_run(const spmm_experts_desc* desc, const void* y,
                                         const float* weights, const int32_t* place,
                                         const int32_t* offsets, const void* grad, void* dy,
                                         float* dweights, spmm_stream stream);

/* log_probs: of each row's softmax, the log probability of class targets[r]
 * (0 for a target outside the classes), the entropy, and the `top` likeliest
 * classes with their log probabilities, best first, ties to the lowest index;
 * a logit of -inf or NaN is none of them (id -1, -inf).  A row whose logits are
 * all -inf has the log probability -inf, no entropy and no gradient.  stats
 * (fp32, 2 a row, or NULL) is for the gradient. */
typedef struct spmm_log_probs_desc {
  int64_t rows;
  int64_t classes;        /* below 2^31                                    */
  int64_t logits_stride;  /* elements between rows of logits               */
  int64_t top;            /* 0 to 64, at most the classes                  */
  int32_t index_type;     /* targets                                       */
  int32_t value_type;     /* logits and dlogits                            */
} spmm_log_probs_desc;

spmm_status spmm_log_probs_workspace(const spmm_log_probs_desc* desc, size_t* bytes);
spmm_status spmm_log_probs_run(const spmm_log_probs_desc* desc, const void* logits, const void* targets,
                               float* logp, float* entropy, float* top_values, int32_t* top_ids,
                               float* stats, void* workspace, size_t workspace_bytes,
                               spmm_stream stream);

/* Gradient with respect to the logits (contiguous) from those of logp and the
 * entropy, either of which may be NULL. */
spmm_status spmm_log_probs_grad_run(const spmm_log_probs_desc* desc, const void* logits,
                                    const void* targets, const float* stats, const float* entropy,
                                    const float* grad_logp, const float* grad_entropy, void* dlogits,
                                    spmm_stream stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* SPMM_MI355X_H_ */
