/*
 * C ABI of the MI355X (gfx950) piecewise-linear-embedding kernels.
 *
 * Plain pointers and sizes only; every device pointer refers to memory on the
 * device that is current on the calling thread, and every launch is enqueued
 * on `stream` (a hipStream_t; NULL = the null stream).  No entry point
 * allocates device memory or synchronises the host: scratch space is passed in
 * by the caller (see ple_backward_workspace_bytes).
 *
 * Return value: PLE_OK (0), a negative PLE_E_* argument error, or a positive
 * hipError_t from the launch.  ple_error_string() names every code.
 *
 * Reference interfaces replaced (paths relative to the reference checkout):
 *   ple_forward_launch   <- ple_forward_cuda   csrc/forward_cuda.cu:687-860
 *                           (registered at csrc/ops.cpp:35-44, :62-75)
 *   ple_backward_launch  <- ple_backward_cuda  csrc/backward_cuda.cu:1528-1725
 *                           (registered at csrc/ops.cpp:46-58, :62-75)
 *   ple_encode_launch / ple_encode_backward_launch
 *                        <- upstream rtdl_num_embeddings.PiecewiseLinearEncoding
 *                           (external dependency of the reference, pinned at
 *                           requirements.txt:1; no operator counterpart)
 *   ple_forward_epilogue_launch / ple_backward_epilogue_launch
 *                        <- the module tail run as PyTorch ops after the
 *                           forward operator, src/rtdl_num_embeddings_cuda/
 *                           module.py:230-248 (no operator counterpart)
 * The reference exposes these only through the torch dispatcher; this ABI is
 * the layer under this build's own dispatcher registration, and is what a
 * ctypes / cgo / JNI binding would call.
 */
#ifndef PLE_HIP_H_
#define PLE_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
enum {
    PLE_DTYPE_F32 = 0,
    PLE_DTYPE_F16 = 1,
    PLE_DTYPE_BF16 = 2,
};

/* error codes (negative: rejected before any launch) */
enum {
    PLE_OK = 0,
    PLE_E_NULL_POINTER = -1,
    PLE_E_BAD_SHAPE = -2,
    PLE_E_BAD_DTYPE = -3,
    PLE_E_BAD_INDEX_WIDTH = -4,
    PLE_E_TOO_LARGE = -5,
    PLE_E_WORKSPACE = -6,
    PLE_E_UNSUPPORTED = -7,
    PLE_E_MISALIGNED = -8,
    PLE_E_SCRATCH_LIMIT = -9,
};

/* Bytes of bin index per (sample, feature) for a given max_n_bins:
 * 1 up to 256 bins, 2 up to 32768, else 4 (reference _meta.py:14-19). */
int ple_bin_index_bytes(int64_t max_n_bins);

/*
 * Forward: for every (n, f)
 *   k      = searchsorted(bin_edges[f, :n_bins[f]+1], x[n, f], right) - 1,
 *            clamped to [0, n_bins[f]-1]                 -> bin_indices[n, f]
 *   frac   = (x[n, f] - bin_edges[f, k]) * inv_bin_widths[f, k]
 *   r      = fma(q(frac), q(weight[f, phys(k), :]), sum_{j<k} q(weight[f, j, :]))
 *   out    = round_quant(r) (+ bias[f, :])               -> output[n, f, :]
 * with q / round_quant = round trip through quant_dtype and
 * phys(k) = (k == n_bins[f]-1) ? max_n_bins-1 : k.
 *
 *   x               float32 [N, F]
 *   bin_edges       float32 [F, B+1]  (+inf padded past n_bins[f])
 *   inv_bin_widths  float32 [F, B]    (0 padded)
 *   n_bins          int32   [F]       (1 <= n_bins[f] <= B)
 *   weight          float32 [F, B, D]
 *   bias            float32 [F, D] or NULL (added after quantisation)
 *   output          output_dtype [N, F, D]
 *   bin_indices     [N, F] of ple_bin_index_bytes(B) bytes each (uint8 /
 *                   int16 / int32)
 *   quant_dtype     PLE_DTYPE_* used for q() and round_quant()
 *   output_dtype    PLE_DTYPE_* of the stored output
 * Supported pairings: output_dtype == quant_dtype with bias NULL (the
 * reference operator), or output_dtype == PLE_DTYPE_F32 with a bias (the
 * module's "x_ple + bias" fused into the store); others -> PLE_E_UNSUPPORTED.
 * N may be 0 (no launch).  F, B, D >= 1, any D (as the reference operator,
 * csrc/forward_cuda.cu:764-766: only the reference module asserts D <= 64);
 * B <= 2^24 and F * B * D < 2^30 (else PLE_E_TOO_LARGE).  Every such shape
 * runs: per-feature tables that fit LDS take the table kernel, larger ones
 * (many bins times a wide row) a kernel that keeps prefix checkpoints in LDS
 * and reads the weights from global memory -- bit-identical results; rows of
 * more than 64 lanes' columns are split into column chunks.
 */
int ple_forward_launch(const float *x, const float *bin_edges, const float *inv_bin_widths,
                       const int32_t *n_bins, const float *weight, const float *bias,
                       void *output, void *bin_indices, int64_t N, int64_t F, int64_t B,
                       int64_t D, int quant_dtype, int output_dtype, void *stream);

/* Scratch bytes ple_backward_launch needs for these sizes (0 is possible). */
size_t ple_backward_workspace_bytes(int64_t N, int64_t F, int64_t B, int64_t D);

/*
 * Backward of ple_forward_launch.
 *   grad_x[n, f]  = iw_k * <g, q(W[f, phys(k)])>
 *                   + [k > 0 and x == e_k] * iw_{k-1} * <g, q(W[f, k-1])>
 *   grad_weight[f, phys(k)] = sum_{bin=k} q(frac) g + sum_{bin>k} g
 *                   (slots no bin maps to are written as 0)
 *   grad_bias[f]  = sum_n grad_output[n, f]   (unrounded grad_output)
 * where g = grad_output rounded through quant_dtype (identity for F32).
 * Supported pairings: quant_dtype == grad_dtype (the reference operator,
 * whose gradient arrives in the forward's output dtype), or grad_dtype ==
 * PLE_DTYPE_F32 with any quant_dtype; others -> PLE_E_UNSUPPORTED.
 * Each of grad_x / grad_weight / grad_bias may be NULL (not computed).
 * Reductions are deterministic: a fixed summation order, no atomics on
 * floating-point data.
 *
 *   grad_output     grad_dtype [N, F, D]
 *   bin_indices     as produced by ple_forward_launch
 *   workspace       >= ple_backward_workspace_bytes(N, F, B, D) bytes,
 *                   256-byte aligned, contents need not be initialised
 * Shapes as for ple_forward_launch; all of them run (tables beyond the
 * sorted path's LDS take deterministic fallback kernels).
 */
int ple_backward_launch(const void *grad_output, const float *x, const float *bin_edges,
                        const float *inv_bin_widths, const int32_t *n_bins,
                        const float *weight, const void *bin_indices, float *grad_x,
                        float *grad_weight, float *grad_bias, int64_t N, int64_t F,
                        int64_t B, int64_t D, int grad_dtype, int quant_dtype,
                        void *workspace, size_t workspace_bytes, void *stream);

/*
 * ple_backward_launch without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No counterpart in the reference.  The
 * workspace is a static device array of PLE_NOALLOC_SCRATCH_BYTES that each
 * GPU the library runs on holds until the process ends; sizes whose
 * ple_backward_workspace_bytes exceed it return PLE_E_SCRATCH_LIMIT before
 * any launch.  Nothing is allocated or freed.  Every call on one GPU shares
 * that GPU's array: calls that overlap on one GPU (other streams, other host
 * threads) race.  Arguments and results as ple_backward_launch.
 */
#define PLE_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)
int ple_backward_launch_noalloc(const void *grad_output, const float *x, const float *bin_edges,
                                const float *inv_bin_widths, const int32_t *n_bins, const float *weight,
                                const void *bin_indices, float *grad_x, float *grad_weight, float *grad_bias,
                                int64_t N, int64_t F, int64_t B, int64_t D, int grad_dtype, int quant_dtype,
                                void *stream);

/*
 * The backward's launch plan for a shape, for benchmarks and memory
 * accounting; no counterpart in the reference (its launcher picks private,
 * sorted or atomic dW paths internally, csrc/backward_cuda.cu:1141-1463, and
 * reports nothing).  grad_output: the gradient that will be passed (its
 * alignment picks the lane width; NULL = 16-byte aligned); relu / linear0:
 * the module epilogue of ple_backward_epilogue_launch (0 for
 * ple_backward_launch).  Fills *info; returns PLE_OK or PLE_E_*.
 *   sorted             1: the fused sort + reduce + dx kernel; 0: the
 *                      fallback dx and histogram kernels
 *   chunks             sample chunks with dW / db partials in the workspace
 *                      (sorted path with 1 chunk: the gradient kernel writes
 *                      grad_weight / grad_bias itself, no finalize kernel)
 *   features_per_group features per gradient-kernel workgroup (sorted and
 *                      matrix-core paths)
 *   columns_per_lane   gradient elements a lane holds per row (sorted path)
 *   lanes_per_row      lanes that share a row (sorted path)
 *   threads            gradient-kernel workgroup size
 *   lds_bytes          gradient-kernel LDS per workgroup
 *   workspace_bytes    workspace a launch that writes grad_weight / grad_bias
 *                      needs (0 for grad_x alone)
 *   bins_per_window    bins whose tables and histogram cells a workgroup holds
 *                      in LDS (sorted path; B when all of them fit)
 *   windows            workgroups per feature group, one per window of bins
 *                      (sorted path; 1 when all bins fit)
 *   matrix_cores       1: the histograms as one-hot products on the matrix
 *                      cores (16-bit gradients in their own dtype, rows of 8,
 *                      16, 24 or 32 columns, at most 96 bins, at most 8
 *                      chunks); sorted is 0 then
 */
typedef struct ple_backward_plan_info {
    int sorted;
    int chunks;
    int features_per_group;
    int columns_per_lane;
    int lanes_per_row;
    int threads;
    size_t lds_bytes;
    size_t workspace_bytes;
    int bins_per_window;
    int windows;
    int matrix_cores;
} ple_backward_plan_info_t;
int ple_backward_plan_query(const void *grad_output, int64_t N, int64_t F, int64_t B, int64_t D,
                            int grad_dtype, int quant_dtype, int relu, int linear0,
                            ple_backward_plan_info_t *info);

/*
 * Module epilogue fused into the kernels.  No counterpart in the reference's
 * operator API: the reference module runs this tail as separate PyTorch ops
 * after its forward operator (src/rtdl_num_embeddings_cuda/module.py:230-248).
 *   version A:  v = x_ple + bias;             out = relu ? relu(v) : v
 *   version B:  out = (lin_bias + lin_weight * x) + (relu ? relu(x_ple) : x_ple)
 * where x_ple is ple_forward_launch's output (rounded through quant_dtype) and
 * the arithmetic after it is fp32 (the output is float32).  relu follows
 * torch.relu: NaN passes, v <= 0 gives 0.  With relu, relu_mask holds one bit
 * per element, bit (j % 32) of word [n, f, j / 32] set where the ReLU passed
 * its input; the forward writes it (when non-NULL) and the backward reads it.
 */
typedef struct ple_epilogue {
    const float *bias;          /* [F, D] or NULL (version A) */
    const float *lin_weight;    /* [F, D] or NULL: linear0 weight (version B) */
    const float *lin_bias;      /* [F, D] linear0 bias, required with lin_weight */
    int relu;                   /* 0 or 1 */
    uint32_t *relu_mask;        /* [N, F, ceil(D / 32)] uint32, see above */
} ple_epilogue_t;

/* Forward with an epilogue: exactly one of bias / lin_weight non-NULL;
 * output float32 [N, F, D]; other arguments as ple_forward_launch. */
int ple_forward_epilogue_launch(const float *x, const float *bin_edges, const float *inv_bin_widths,
                                const int32_t *n_bins, const float *weight,
                                const ple_epilogue_t *epilogue, float *output, void *bin_indices,
                                int64_t N, int64_t F, int64_t B, int64_t D, int quant_dtype,
                                void *stream);

/*
 * Backward of ple_forward_epilogue_launch (grad_output float32 [N, F, D]).
 * With g_ple = relu ? grad_output * pass : grad_output, rounded through
 * quant_dtype for grad_x / grad_weight as in ple_backward_launch, and
 * grad_x += <grad_output[n, f], lin_weight[f]> for version B;
 *   grad_bias[f]       = sum_n g_ple (unrounded)         (version A)
 *   grad_lin_weight[f] = sum_n grad_output[n, f] * x[n, f] (version B)
 *   grad_lin_bias[f]   = sum_n grad_output[n, f]           (version B)
 * The backward reads lin_weight (non-NULL: version B, else version A), relu
 * and relu_mask; bias and lin_bias are not read.  Any gradient pointer may be
 * NULL; grad_bias must be NULL for version B and the linear0 gradients NULL
 * for version A.  The workspace is sized by ple_backward_workspace_bytes.
 */
int ple_backward_epilogue_launch(const float *grad_output, const float *x, const float *bin_edges,
                                 const float *inv_bin_widths, const int32_t *n_bins,
                                 const float *weight, const void *bin_indices,
                                 const ple_epilogue_t *epilogue, float *grad_x, float *grad_weight,
                                 float *grad_bias, float *grad_lin_weight, float *grad_lin_bias,
                                 int64_t N, int64_t F, int64_t B, int64_t D, int quant_dtype,
                                 void *workspace, size_t workspace_bytes, void *stream);

/*
 * Dense piecewise-linear encoding: the output of the upstream
 * PiecewiseLinearEncoding module (rtdl_num_embeddings==0.0.12), which the
 * reference's module builds on; no counterpart in the reference's operators.
 * For feature f (n_bins[f] = n bins, b and frac as in ple_forward_launch) the
 * n components at columns offsets[f] .. offsets[f] + n - 1 of row n are
 *   1 (k < b), frac (k == b), 0 (k > b);   NaN x: all NaN.
 *   offsets         int32 [F], offsets[f] = sum_{j<f} n_bins[j]
 *   output          float32 [N, total_bins], total_bins = sum_f n_bins[f]
 * At most 2409 features (PLE_E_UNSUPPORTED beyond; the backward has no such
 * limit).
 */
int ple_encode_launch(const float *x, const float *bin_edges, const float *inv_bin_widths,
                      const int32_t *n_bins, const int32_t *offsets, float *output, int64_t N,
                      int64_t F, int64_t B, int64_t total_bins, void *stream);

/* Backward of ple_encode_launch: grad_x[n, f] = g[n, offsets[f] + b] * iw_b
 * (+ g[n, offsets[f] + b - 1] * iw_{b-1} when b > 0 and x == e_b). */
int ple_encode_backward_launch(const float *grad_output, const float *x, const float *bin_edges,
                               const float *inv_bin_widths, const int32_t *n_bins,
                               const int32_t *offsets, float *grad_x, int64_t N, int64_t F,
                               int64_t B, int64_t total_bins, void *stream);

/*
 * The launch plan of ple_encode_launch (backward 0) or
 * ple_encode_backward_launch (backward 1) for a shape, without launching.
 * `output` may be NULL (then taken as 16-byte aligned).  Returns the error the
 * launch would return for the sizes, else fills `info`; all zeros: no feature
 * groups, but whole rows (forward) or one thread per (sample, feature) pair
 * (backward).
 *   features_per_group  adjacent features whose columns a workgroup writes
 *   features_searched   features whose bins it searches: with 16-byte stores up
 *                       to three more, whose columns share its last vector
 *   groups, chunks      feature groups, sample chunks
 *   rows_per_block      samples searched together
 *   pairs_per_block     (sample, feature) pairs that the threads of a workgroup
 *                       search together, at most: rows_per_block *
 *                       features_searched never exceeds it
 *   lds_tables          1: the group's edges and inverse widths are kept in LDS
 */
typedef struct ple_encode_plan_info {
    int features_per_group;
    int features_searched;
    int groups;
    int chunks;
    int rows_per_block;
    int pairs_per_block;
    int lds_tables;
    size_t lds_bytes;
} ple_encode_plan_info_t;
int ple_encode_plan_query(const void *output, int64_t N, int64_t F, int64_t B, int64_t total_bins,
                          int backward, ple_encode_plan_info_t *info);

/*
 * Embedding lookup with scaling (tokens, or categorical columns next to the
 * numerical ones); no counterpart in the reference.
 *   output[i, :] = scale * weight[row(i), :], rounded once to output_dtype
 *   row(i) = tokens[i], or offsets[f] + tokens[i] with f = i % F for
 *            categorical tokens [N, F] (T = N * F) of F tables in one
 * A negative token is a missing value: its output is 0.  A token beyond its
 * table (its column's size, or V rows) gives NaN.  Neither reads the table.
 *   tokens     int32 or int64 (token_bytes 4 or 8) [T]
 *   offsets    int64 [F + 1], the columns' first rows and V, not decreasing;
 *              or NULL (F is not used then; pass 1)
 *   weight     weight_dtype [V, D]
 *   output     output_dtype [T, D]
 * T may be 0.  T, V < 2^31 - 1, D <= 2^20 (else PLE_E_TOO_LARGE).
 */
int ple_lookup_launch(const void *tokens, int token_bytes, const int64_t *offsets, const void *weight, void *output,
                      int64_t T, int64_t F, int64_t V, int64_t D, float scale, int weight_dtype, int output_dtype,
                      void *stream);

/* Scratch bytes ple_lookup_backward_launch needs for these sizes. */
size_t ple_lookup_backward_workspace_bytes(int64_t T, int64_t V, int64_t D);

/*
 * Backward of ple_lookup_launch: every row of grad_weight is written,
 *   grad_weight[r, :] = scale * sum_{i: row(i) = r} grad_output[i, :]
 * summed in 32 bits in a fixed order (the tokens are sorted; no atomics on
 * floating-point data) and rounded once to weight_dtype; 0 for rows without
 * tokens.  Missing tokens, tokens beyond their table and tokens equal to
 * padding_idx (>= 0; a negative one: none) have no gradient.
 *   workspace  >= ple_lookup_backward_workspace_bytes(T, V, D) bytes, 256-byte
 *              aligned, contents need not be initialised
 */
int ple_lookup_backward_launch(const void *grad_output, const void *tokens, int token_bytes, const int64_t *offsets,
                               void *grad_weight, int64_t T, int64_t F, int64_t V, int64_t D, int64_t padding_idx,
                               float scale, int grad_dtype, int weight_dtype, void *workspace, size_t workspace_bytes,
                               void *stream);

/*
 * The launch plan of ple_lookup_backward_launch for a shape, without launching.
 * `grad_output` and `grad_weight` may be NULL (then taken as aligned).  Returns
 * the error the launch would return for the sizes (PLE_E_TOO_LARGE too where the
 * sums' grid would pass 2^32 threads, a gradient larger than a device's memory),
 * else fills `info`.
 *   one_workgroup    1: one workgroup sorts, in LDS; 0: several, pass by pass
 *   passes           passes of the sort, each of digit_bits bits of the row
 *   sort_workgroups  workgroups that sort
 *   sum_workgroups   workgroups that add up runs of equal rows
 *   clear_rows       rows without tokens a clearing workgroup looks at
 *   most_threads     threads of the largest launch, below 2^32
 *   workspace_bytes  as ple_lookup_backward_workspace_bytes
 */
typedef struct ple_lookup_plan_info {
    int one_workgroup;
    int passes;
    int digit_bits;
    int sort_workgroups;
    int64_t sum_workgroups;
    int64_t clear_rows;
    int64_t most_threads;
    size_t workspace_bytes;
} ple_lookup_plan_info_t;
int ple_lookup_backward_plan_query(const void *grad_output, const void *grad_weight, int64_t T, int64_t V, int64_t D,
                                   int grad_dtype, int weight_dtype, ple_lookup_plan_info_t *info);

/*
 * Norms after and before a block, fused with the block's gate and the residual
 * scale; no counterpart in the reference.  For every row of the residual
 * stream r and the block's output (the branch) y, both [N, D]:
 *   p = post_norm(y) * post_weight + post_bias
 *   s = residual_scale * r + h(gate) * p, stored in stream_dtype
 *   n = pre_norm(s) * pre_weight + pre_bias, stored in branch_dtype
 * A norm is none, rms (x / sqrt(mean(x^2) + eps)) or layer ((x - mean) /
 * sqrt(var + eps)); the norm before the next block reads s as it is stored.
 * h is the identity, sigmoid or tanh.  The gate has gate_rows rows, 1, N or a
 * divisor of N: row n uses gate row n / (N / gate_rows).  Weights, biases and
 * the gate may each be NULL (1, 0 and 1).  Sums, means and factors are 32-bit.
 *   stream_dtype  of r and s: branch_dtype, or PLE_DTYPE_F32
 *   branch_dtype  of y and n
 *   param_dtype   of weights, biases and gate
 * D <= PLE_NORM_MAX_WIDTH (else PLE_E_TOO_LARGE).
 */
enum {
    PLE_NORM_NONE = 0,
    PLE_NORM_RMS = 1,
    PLE_NORM_LAYER = 2,
};
enum {
    PLE_GATE_IDENTITY = 0,
    PLE_GATE_SIGMOID = 1,
    PLE_GATE_TANH = 2,
};
#define PLE_NORM_MAX_WIDTH 8192
typedef struct ple_norm {
    const void *post_weight, *post_bias;  /* [D] or NULL */
    const void *gate;                     /* [gate_rows, D] or NULL */
    const void *pre_weight, *pre_bias;    /* [D] or NULL */
    int64_t gate_rows;
    int post_norm, pre_norm;              /* PLE_NORM_* */
    int gate_activation;                  /* PLE_GATE_* */
    int stream_dtype, branch_dtype, param_dtype;
    float residual_scale, eps;
} ple_norm_t;

/*
 * Forward.  branch NULL: only the norm before a block, n = pre_norm(r) (no
 * post norm, no gate, residual_scale 1; stream_out NULL).  pre_norm none:
 * normed NULL.
 *   stats   float32 [N, 4], 16-byte aligned: mean and factor of y, of s
 */
int ple_residual_norm_launch(const void *residual, const void *branch, const ple_norm_t *norm, void *stream_out,
                             void *normed, float *stats, int64_t N, int64_t D, void *stream);

/* Gradients that ple_residual_norm_backward_launch writes; NULL: not wanted. */
typedef struct ple_norm_grads {
    void *residual;                       /* stream_dtype [N, D] */
    void *branch;                         /* branch_dtype [N, D] */
    void *post_weight, *post_bias;        /* param_dtype [D] */
    void *gate;                           /* param_dtype [gate_rows, D] */
    void *pre_weight, *pre_bias;          /* param_dtype [D] */
} ple_norm_grads_t;

/* Scratch bytes the backward needs (on the current device). */
size_t ple_residual_norm_backward_workspace_bytes(const ple_norm_t *norm, int64_t N, int64_t D);

/*
 * Backward of ple_residual_norm_launch.  grad_stream (stream_dtype) and
 * grad_normed (branch_dtype) may be NULL (zero); stream_in is the forward's
 * stream_out (its residual, where there was no branch).  Sums over rows are
 * 32-bit in a fixed order, without atomics.
 *   workspace  >= ple_residual_norm_backward_workspace_bytes() bytes, 256-byte
 *              aligned, contents need not be initialised
 */
int ple_residual_norm_backward_launch(const void *grad_stream, const void *grad_normed, const void *stream_in,
                                      const void *branch, const float *stats, const ple_norm_t *norm,
                                      const ple_norm_grads_t *grads, int64_t N, int64_t D, void *workspace,
                                      size_t workspace_bytes, void *stream);

/*
 * Distillation from a teacher's top logits, with optional hard labels; no
 * counterpart in the reference.  For every row, with q = softmax(z / T) of the
 * student's logits z [V] and p_k = exp(t_k / T - l) of the teacher's K logits:
 *   loss = alpha T^2 (sum_k p_k (log p_k - log q_{c_k}) + rest)
 *          + (1 - alpha) (log sum exp z - z[label])
 * teacher_lse NULL: l is the log-sum over the row's own K logits (p sums to 1)
 * and rest 0.  Else l = teacher_lse[n], the log-sum of exp(t / T) over the
 * teacher's whole vocabulary, and rest = rho (log rho - log Q) with rho = 1 -
 * sum p and Q the student's mass outside the K classes.
 * Negative classes and labels are absent (a row without classes has only its
 * label's term, and the other way round).  A class or label >= V makes the
 * row's loss and gradient NaN.  A row whose logits are all -inf has loss and
 * gradient 0.  A class may occur twice.  labels NULL: the first term alone.
 *   logits           dtype [N, V]
 *   teacher_logits   teacher_dtype [N, K]
 *   teacher_classes  int32 or int64 (class_bytes 4 or 8) [N, K]
 *   teacher_lse      float32 [N] or NULL
 *   labels           int64 [N] or NULL
 *   loss             float32 [N]
 *   stats            float32 [N, PLE_DISTILL_STATS], 16-byte aligned, for the
 *                    backward
 *   workspace        >= ple_distill_workspace_bytes(N, V) bytes (0 is
 *                    possible), 256-byte aligned, need not be initialised
 * 1e-6 < T < 1e6, 0 <= alpha <= 1 (else PLE_E_UNSUPPORTED); V <= 2^30, K <=
 * 2^20, N <= 2^24, N * V <= 2^40 (else PLE_E_TOO_LARGE).
 */
#define PLE_DISTILL_STATS 8
size_t ple_distill_workspace_bytes(int64_t N, int64_t V);
int ple_distill_launch(const void *logits, const void *teacher_logits, const void *teacher_classes, int class_bytes,
                       const float *teacher_lse, const int64_t *labels, float *loss, float *stats, int64_t N, int64_t V,
                       int64_t K, float temperature, float alpha, int dtype, int teacher_dtype, void *workspace,
                       size_t workspace_bytes, void *stream);

/* Backward of ple_distill_launch: grad_logits (dtype [N, V]) = grad_loss[n] *
 * d loss[n] / d logits[n], from the forward's stats; the teacher has no
 * gradient. */
int ple_distill_backward_launch(const float *grad_loss, const void *logits, const void *teacher_logits,
                                const void *teacher_classes, int class_bytes, const int64_t *labels, const float *stats,
                                void *grad_logits, int64_t N, int64_t V, int64_t K, float temperature, float alpha,
                                int dtype, int teacher_dtype, void *stream);

/*
 * Group norm with an activation, channels last; no counterpart in the
 * reference.  A sample x [S, C] has G groups of C / G adjacent channels; a
 * group's values over all S rows are standardised together:
 *   y = act((x - mean) / sqrt(var + eps) * weight[c] + bias[c])
 *   x, y         dtype [N, S, C]
 *   weight, bias param_dtype [C], or NULL: 1, 0
 *   stats        float32 [N, G, 2], 8-byte aligned: mean and 1 / sqrt(var + eps)
 *   workspace    >= ple_group_norm_workspace_bytes() bytes (0 is possible),
 *                256-byte aligned, need not be initialised
 * Results share no memory with anything that is read.
 * Statistics and sums are 32-bit in a fixed order (workgroups that share a sample
 * and wait in vain for each other, milliseconds, compute what is missing
 * themselves, to the same bits).  C <= 2^20, S < 2^31, N < 2^31,
 * N * S * C < 2^44 (else PLE_E_TOO_LARGE); G divides C (else PLE_E_BAD_SHAPE).
 */
enum {
    PLE_ACT_NONE = 0,
    PLE_ACT_RELU = 1,
    PLE_ACT_SILU = 2,
    PLE_ACT_GELU = 3,    /* z times the standard normal distribution at z */
};
size_t ple_group_norm_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int dtype);
int ple_group_norm_launch(const void *x, const void *weight, const void *bias, void *y, float *stats, int64_t N,
                          int64_t S, int64_t C, int64_t G, int activation, float eps, int dtype, int param_dtype,
                          void *workspace, size_t workspace_bytes, void *stream);

/* Backward of ple_group_norm_launch, from its x and stats.  grad_x (dtype),
 * grad_weight and grad_bias (param_dtype [C]) may be NULL: not wanted. */
size_t ple_group_norm_backward_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int dtype);
int ple_group_norm_backward_launch(const void *grad_y, const void *x, const float *stats, const void *weight,
                                   const void *bias, void *grad_x, void *grad_weight, void *grad_bias, int64_t N,
                                   int64_t S, int64_t C, int64_t G, int activation, int dtype, int param_dtype,
                                   void *workspace, size_t workspace_bytes, void *stream);

/*
 * The launch plan of ple_group_norm_launch (backward != 0: of its backward) for a
 * shape, without launching.  `x` may be NULL; its alignment stands for that of all
 * [N, S, C] tensors.  Returns the error the launch would return for the sizes,
 * else fills `info` (all 0 without rows).
 *   form             PLE_GROUP_*
 *   lane_channels    channels a lane takes of a row
 *   slabs            of a row's channels, a workgroup each
 *   members          PLE_GROUP_SHARED: workgroups that share a sample's slab
 *   params_end       one past the last channel whose weight and bias a lane reads
 *   workspace_bytes  as ple_group_norm[_backward]_workspace_bytes
 */
enum {
    PLE_GROUP_HELD = 0,    /* a workgroup holds a sample's slab */
    PLE_GROUP_SHARED = 1,  /* several do, and exchange what they know */
    PLE_GROUP_SPLIT = 2,   /* pieces of samples, read twice */
};
typedef struct ple_group_norm_plan_info {
    int form;
    int lane_channels;
    int slabs;
    int members;
    int64_t params_end;
    size_t workspace_bytes;
} ple_group_norm_plan_info_t;
int ple_group_norm_plan_query(const void *x, int64_t N, int64_t S, int64_t C, int64_t G, int dtype, int backward,
                              ple_group_norm_plan_info_t *info);

/*
 * Learned bias of attention scores by relative position; no counterpart in the
 * reference.  With p = starts[b] (or offset) the position of a sample's first
 * query:
 *   out[b, h, i, j] = weight[buckets[clamp(j - p - i, -far, far) + far], h]
 * A negative bucket has no bias (0, no gradient), one >= R gives NaN.  causal:
 * -inf where j > p + i.
 *   weight    weight_dtype [R, H]
 *   buckets   int32 [2 far + 1]
 *   starts    int64 [B], or NULL: offset for all (then B is 1)
 *   out       out_dtype [B, H, q, k]
 * 1 <= far <= 2^24; q, k <= 2^23; B, H, R < 2^31, B * H * q * k < 2^44, |offset| <= 2^60
 * (else PLE_E_TOO_LARGE); positions beyond 2^60 count as 2^60.
 */
int ple_relative_bias_launch(const void *weight, const int32_t *buckets, const int64_t *starts, void *out, int64_t B,
                             int64_t H, int64_t q, int64_t k, int64_t R, int64_t far, int64_t offset, int causal,
                             int weight_dtype, int out_dtype, void *stream);

/* Backward of ple_relative_bias_launch: grad_weight (weight_dtype [R, H]) from
 * grad_output (out_dtype [B, H, q, k]), whose masked entries do not count.  Sums
 * are 32-bit in a fixed order.  workspace: as above, >=
 * ple_relative_bias_backward_workspace_bytes() bytes. */
size_t ple_relative_bias_backward_workspace_bytes(int64_t B, int64_t H, int64_t q, int64_t k, int64_t R, int64_t far);
int ple_relative_bias_backward_launch(const void *grad_output, const int32_t *buckets, const int64_t *starts,
                                      void *grad_weight, int64_t B, int64_t H, int64_t q, int64_t k, int64_t R,
                                      int64_t far, int64_t offset, int causal, int out_dtype, int weight_dtype,
                                      void *workspace, size_t workspace_bytes, void *stream);

/*
 * The norm of many gradients together, and their scaling to a limit; no
 * counterpart in the reference.
 *   norm = (sum |g|^p)^(1/p) over all elements of all tensors, p 1 or 2, or
 *          max |g|; summed in 64 bits, in a fixed order, rounded to 32; NaN if
 *          an element is
 *   out = g * min(1, limit / (norm + 1e-6))
 * The list lies in host memory and is read before the call returns; its
 * addresses go into the kernels' arguments (and so into a captured graph).
 */
typedef struct ple_grad {
    const void *grad;        /* numel elements of dtype */
    void *out;               /* scaling: numel elements of out_dtype; grad itself
                              * (and its dtype), or memory that no tensor of the
                              * list shares */
    int64_t numel;           /* 0 to 2^40 */
    int dtype, out_dtype;    /* PLE_DTYPE_* (the norm does not look at out and out_dtype) */
} ple_grad_t;
enum { PLE_NORM_P1 = 1, PLE_NORM_P2 = 2, PLE_NORM_INF = 3 };

/* norm: float32, one element; workspace >= ple_grad_norm_workspace_bytes()
 * bytes, 256-byte aligned, need not be initialised. */
size_t ple_grad_norm_workspace_bytes(const ple_grad_t *grads, int64_t count);
int ple_grad_norm_launch(const ple_grad_t *grads, int64_t count, int kind, float *norm, void *workspace,
                         size_t workspace_bytes, void *stream);

/* out from the norm in device memory.  Gradients that stay in place are not
 * touched where nothing is clipped; limit >= 0 (an infinite one clips nothing). */
int ple_grad_scale_launch(const ple_grad_t *grads, int64_t count, const float *norm, float limit, void *stream);

/* Both: the norm of ple_grad_norm_launch, and out scaled with it. */
int ple_grad_clip_launch(const ple_grad_t *grads, int64_t count, int kind, float limit, float *norm, void *workspace,
                         size_t workspace_bytes, void *stream);

/*
 * Planner overrides, for tuning sweeps and for tests that run every kernel
 * form on the same inputs.  No counterpart in the reference (its launchers
 * have no knobs).  Each knob holds 0 -- the planner's own choice, the default
 * -- or a forced value, read by every later launch of the process:
 *   PLE_TUNE_FWD_FS         features per forward workgroup (power of two)
 *   PLE_TUNE_FWD_WG_PER_CU  forward workgroups per CU the chunking aims for
 *   PLE_TUNE_FWD_FB         forward workgroup size (256 or 512 threads)
 *   PLE_TUNE_FWD_VEC        outputs per lane (1, 2 or 4; 16-bit outputs 8)
 *   PLE_TUNE_FWD_WIDE       1: the wide-table forward kernel for any shape
 *   PLE_TUNE_BWD_SIMPLE     1: the fallback backward kernels for any shape
 *   PLE_TUNE_BWD_SIMPLE_GLOBAL 1: their histogram cells in global memory
 *   PLE_TUNE_BWD_VEC        1: one gradient element per lane; 4: at most four
 *                           (no 8-element lanes for 16-bit gradients)
 *   PLE_TUNE_BWD_FS         features per backward sub-tile (1, 2, 4, 8, 16;
 *                           the matrix-core backward's groups: 1, 2, 4)
 *   PLE_TUNE_BWD_RB         reducer threads per backward workgroup (256 or 512)
 *   PLE_TUNE_BWD_WG_PER_CU  backward workgroups per CU
 *   PLE_TUNE_BWD_MFMA       1: no matrix-core backward (the sorted path for
 *                           16-bit gradients too); 2: the matrix-core backward
 *                           for every shape it can take (also past 8 chunks)
 *   PLE_TUNE_BWD_STREAM     1: the matrix-core backward reads its gradient with
 *                           plain loads; 2: past the caches
 *   PLE_TUNE_GROUP_POLLS    n: workgroups that share a sample of a group norm
 *                           look n - 1 times for what another knows, before
 *                           they compute it themselves
 * A forced value the shape cannot take is ignored.  Returns the knob's
 * previous value, or PLE_E_BAD_SHAPE for an unknown knob.  Not synchronised
 * with launches running on other threads.
 */
enum {
    PLE_TUNE_FWD_FS = 0,
    PLE_TUNE_FWD_WG_PER_CU = 1,
    PLE_TUNE_FWD_FB = 2,
    PLE_TUNE_FWD_VEC = 3,
    PLE_TUNE_FWD_WIDE = 4,
    PLE_TUNE_BWD_SIMPLE = 5,
    PLE_TUNE_BWD_SIMPLE_GLOBAL = 6,
    PLE_TUNE_BWD_VEC = 7,
    PLE_TUNE_BWD_FS = 8,
    PLE_TUNE_BWD_RB = 9,
    PLE_TUNE_BWD_WG_PER_CU = 10,
    PLE_TUNE_BWD_MFMA = 11,
    PLE_TUNE_BWD_STREAM = 12,
    PLE_TUNE_GROUP_POLLS = 13,
    PLE_TUNE_COUNT = 14,
};
int ple_set_tuning(int knob, int value);

/*
 * Kernel timing, for benchmarks; no counterpart in the reference.  After
 * ple_timing_start(slots), each of the next `slots` launches of the forward
 * (resp. backward) entry points records a HIP event pair on its stream around
 * its main kernel: PLE_TIMER_FORWARD brackets the forward kernel,
 * PLE_TIMER_BACKWARD the backward's gradient kernel (the sorted-path kernel,
 * or the fallback path's dx and histogram kernels), not the finalize that
 * turns its partials into grad_weight / grad_bias.  ple_timing_read waits for
 * the recorded pairs and returns their summed duration in milliseconds and
 * their number.  ple_timing_stop ends recording; ple_timing_start(0) also
 * releases the events.  The events belong to the device current at
 * ple_timing_start.  Returns PLE_OK, PLE_E_* or a hipError_t.
 */
enum {
    PLE_TIMER_FORWARD = 0,
    PLE_TIMER_BACKWARD = 1,
    PLE_TIMER_COUNT = 2,
};
int ple_timing_start(int slots);
int ple_timing_stop(void);
int ple_timing_read(int which, double *ms_total, int *count);

/* Human-readable name of a return code (static storage). */
const char *ple_error_string(int code);

/* ABI version of this header: (major << 16) | minor. */
int ple_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* PLE_HIP_H_ */
