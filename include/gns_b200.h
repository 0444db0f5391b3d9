/*
 * gns_b200.h - C ABI of the B200 (sm_100a) Gram Newton-Schulz library.
 *
 * Plain pointers, element strides and sizes; no framework types. Every call is
 * asynchronous on the given CUDA stream, allocates no device memory (callers
 * pass a workspace where one is needed), performs no host synchronisation and
 * returns GNS_OK (0) or a negative error code. gns_last_error() returns the
 * message of the most recent failure on the calling host thread.
 *
 * Element type codes: GNS_F16 = 0, GNS_BF16 = 1, GNS_F32 = 2.
 * Matrices are batched [batch, rows, cols] with element strides
 * (batch_stride, row_stride, col_stride). Interface citations refer to files of
 * the reference project afrenkai/Gram-Newton-Schulz-Ampere.
 */
#ifndef GNS_B200_H_
#define GNS_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define GNS_API __attribute__((visibility("default")))
#else
#define GNS_API
#endif

typedef struct CUstream_st* gns_stream_t;

enum {
  GNS_F16 = 0,
  GNS_BF16 = 1,
  GNS_F32 = 2,
};

enum {
  GNS_OK = 0,
  GNS_ERR_ARGUMENT = -1,   /* invalid shape, dtype or scalar */
  GNS_ERR_LAYOUT = -2,     /* strides/alignment a TMA tile load cannot express */
  GNS_ERR_WORKSPACE = -3,  /* workspace missing or too small */
  GNS_ERR_CUDA = -4,       /* a CUDA runtime/driver call failed */
  GNS_ERR_DEVICE = -5,     /* device is not sm_100 */
  GNS_ERR_UNSUPPORTED = -6 /* size beyond a documented kernel limit */
};

/* Library version, e.g. 100 for 0.1.0. */
GNS_API int gns_version(void);

/* Message of the last failing call on this host thread ("" if none). */
GNS_API const char* gns_last_error(void);

/* Reads (and optionally clears) the device status word that kernels set when a
 * bounded wait gives up (0 = no failure). Synchronises the current device. */
GNS_API int gns_device_status(int* status, int clear);

/* Per-launch timing of the tcgen05 GEMM (no counterpart in the reference; used by
 * bench.py for the live roofline). gns_profile_enable(n) records a CUDA event pair
 * and the algorithmic flop count (2mnk, or mnk for symmetric products) for each of
 * the next n GEMM launches on any stream; gns_profile_collect synchronises those
 * events, writes up to `capacity` records, frees them and stops recording. */
GNS_API int gns_profile_enable(int capacity);
GNS_API int gns_profile_collect(int capacity, int* count, float* ms, double* flops, int* symmetric);

/* ------------------------------------------------------------------ GEMM
 * D = alpha * A @ B + beta * C, batched, fp32 accumulation on tcgen05.
 * A is [batch, m, k], B is [batch, k, n], C and D are [batch, m, n] with unit
 * column stride. A and B share one dtype (F16 or BF16); each may be stored with
 * either unit column stride (row-major) or unit row stride (a transposed view).
 * C (dtype c_dtype) is read only when beta != 0; it may alias D.
 * symmetric != 0 asserts the result is symmetric (m == n): only column >= row
 * is computed and mirrored, so D is exactly symmetric.
 * Replaces: TorchBackend.symmetric_matmul / symmetric_batch_matrix_matrix_product /
 * matmul / matmul_add (kernels/torch_ns.py:6-35, protocols.py:36-61) and the
 * CUTLASS exports cutlass_baddbmm / cutlass_symmetric_baddbmm
 * (kernels/cutlass_ns.cu:380-384, cutlass_ns.py:117-204). */
GNS_API int gns_gemm(int ab_dtype, int64_t batch, int64_t m, int64_t n, int64_t k,
             const void* a, int64_t a_bstride, int64_t a_rstride, int64_t a_cstride,
             const void* b, int64_t b_bstride, int64_t b_rstride, int64_t b_cstride,
             const void* c, int c_dtype, int64_t c_bstride, int64_t c_rstride,
             void* d, int d_dtype, int64_t d_bstride, int64_t d_rstride,
             float alpha, float beta, int symmetric, gns_stream_t stream);

/* ------------------------------------------------------- normalisation
 * out[b] = fp16(x[b] / (||x[b]||_F + eps)) with the norm taken in fp32.
 * x has unit column stride; out is [batch, rows, out_ld] fp16.
 * Replaces: the input normalisation of newton_schulz.py:81-84 / :141-144 / :304-307. */
GNS_API size_t gns_normalize_workspace_size(int64_t batch, int64_t rows, int64_t cols);
GNS_API int gns_frobenius_normalize(int x_dtype, int64_t batch, int64_t rows, int64_t cols,
                            const void* x, int64_t x_bstride, int64_t x_rstride,
                            void* out_f16, int64_t out_ld, float eps,
                            void* workspace, size_t workspace_bytes, gns_stream_t stream);

/* Same result as gns_frobenius_normalize, but it allocates nothing and takes no
 * workspace: for callers that cannot allocate device memory when they normalise
 * (their memory is owned by another pool or allocator, or an allocation could
 * block or fail in the middle of a step). Its scratch is a 64 KiB array inside
 * the library, held on every GPU that loads it until the process exits; it
 * serves at most 8192 matrices per call, and larger batches return
 * GNS_ERR_UNSUPPORTED with a message. Each call asks the runtime for the
 * array's device address on the current device (no allocation); the first call
 * on a device also loads the library's device code there, so make that first
 * call before any stream capture. Every call shares the one array and the
 * previous call's contents remain in it (the counters that must start at zero
 * are cleared by each call), so calls that can overlap on the GPU (different
 * streams, or concurrent host threads) race and must be serialised by the caller.
 * No counterpart in the reference. */
GNS_API int gns_frobenius_normalize_noalloc(int x_dtype, int64_t batch, int64_t rows, int64_t cols,
                                            const void* x, int64_t x_bstride, int64_t x_rstride,
                                            void* out_f16, int64_t out_ld, float eps, gns_stream_t stream);

/* Failure path of the normalisation's bounded wait (no counterpart in the
 * reference). Each normalisation CTA waits for the other row slices of its
 * matrix; a wait still unfinished after the limit (default 2 s) records status
 * 4 for gns_device_status and fills the CTA's slice of the output with NaN.
 * gns_set_wait_limit_ns sets that limit process-wide (1 ms to 10 s) and returns
 * the previous one. gns_selftest_normalize_timeout launches the normalisation
 * on a small contiguous fp32 batch (at most 64 matrices, 2^20 elements each;
 * out is [batch, rows, cols] fp16, workspace as for gns_frobenius_normalize)
 * waiting for one arrival more than it launches, so every wait runs out: the
 * call returns GNS_OK, the device status reads 4 afterwards and the output is
 * NaN. It exists so that tests can exercise the failure path without a fault. */
GNS_API int gns_set_wait_limit_ns(unsigned long long limit_ns, unsigned long long* previous);
GNS_API int gns_selftest_normalize_timeout(int64_t batch, int64_t rows, int64_t cols, const float* x,
                                           void* out_f16, void* workspace, size_t workspace_bytes,
                                           gns_stream_t stream);

/* ---------------------------------------------------- Newton-Schulz chains
 * Whole orthogonalisation of a batch in one call: normalise, iterate with the
 * given (a, b, c) coefficient triples (coeffs[3*i + 0..2]), cast to out_dtype.
 * x and out have unit column stride and may not alias. Internal products run
 * in fp16 with fp32 accumulation, like the reference's fp16 torch path.
 *
 * gns_gram_newton_schulz follows build_gram_newton_schulz_operation
 * (newton_schulz.py:124-223); reset_mask bit i restarts from X at iteration i
 * (gram_newton_schulz_reset_iterations, default (2,)). Square inputs are
 * dispatched to the standard chain by the caller, as NewtonSchulz.__call__
 * does (newton_schulz.py:308-318).
 * gns_standard_newton_schulz follows build_standard_newton_schulz_operation
 * (newton_schulz.py:66-121). */
GNS_API size_t gns_newton_schulz_workspace_size(int64_t batch, int64_t rows, int64_t cols);
GNS_API int gns_gram_newton_schulz(int x_dtype, int64_t batch, int64_t rows, int64_t cols,
                           const void* x, int64_t x_bstride, int64_t x_rstride,
                           void* out, int out_dtype, int64_t out_bstride, int64_t out_rstride,
                           const double* coeffs, int n_iters, uint32_t reset_mask, float eps,
                           void* workspace, size_t workspace_bytes, gns_stream_t stream);
GNS_API int gns_standard_newton_schulz(int x_dtype, int64_t batch, int64_t rows, int64_t cols,
                               const void* x, int64_t x_bstride, int64_t x_rstride,
                               void* out, int out_dtype, int64_t out_bstride, int64_t out_rstride,
                               const double* coeffs, int n_iters, float eps,
                               void* workspace, size_t workspace_bytes, gns_stream_t stream);

/* Tactic switch of gns_gram_newton_schulz (process-wide; returns the previous
 * setting). Enabled (the default): non-square matrices whose short side is at
 * most 128 and whose long side is at most 3072 run as ONE fused kernel per call after
 * the normalisation: a CTA per matrix keeps G, P, GP and Q in shared memory and
 * runs every product of the chain without a launch boundary; the same kernel
 * runs gns_standard_newton_schulz for square matrices of side at most 128 (X, G
 * and P in shared memory). Disabled: every product is its own GEMM launch. Both tactics compute the same products in the
 * same order and rounding. The reference's CUTLASS backend picks among its
 * kernels the same way, by size (select_cutlass_tactic, kernels/cutlass_ns.py:109-114). */
GNS_API int gns_set_small_chain(int enabled);

/* Caps the SMs one GEMM launch occupies (process-wide; 0, the default, means
 * all; returns the previous cap). The GEMM's grid is persistent and assigns
 * tiles statically, so a CTA that cannot start because another kernel (a
 * collective running beside it) holds its SM delays the whole launch; with a
 * cap the launch leaves those SMs free. No counterpart in the reference. */
GNS_API int gns_set_gemm_sm_limit(int sms);

/* ------------------------------------- pieces of a column-sharded Gram chain
 * For a matrix whose long dimension is split across ranks (a wide matrix sharded
 * by columns, or a tall one by rows), Gram Newton-Schulz only needs the m x m
 * Gram matrix summed over ranks. The distributed layer runs:
 *   s  = gns_frobenius_sumsq(shard);  all-reduce(s);  Xh = gns_frobenius_scale(shard, s)
 *   G  = gns_gemm(Xh, Xh^T, symmetric, fp32 out);  all-reduce(G)
 *   Q  = gns_gram_iterations(G, iterations [begin, end) up to the next restart)
 *   restart: Xh = Q Xh (gns_gemm);  G = all-reduce(Xh Xh^T);  next segment
 *   out = Q Xh (gns_gemm)
 * The arithmetic follows newton_schulz.py:139-217; the reference itself has no
 * such entry points (it assembles whole matrices on owner ranks with an
 * all-to-all, distributed_orthogonalization.py:278-349).
 * gns_frobenius_sumsq writes sum(x^2) per matrix in fp32 (fixed summation order;
 * workspace: gns_normalize_workspace_size bytes). gns_frobenius_scale writes
 * fp16(x / (sqrt(sumsq[b]) + eps)). gns_gram_iterations takes G (fp32 or fp16,
 * m x m, symmetric), rounds it to fp16 and runs the Gram iterations
 * [it_begin, it_end) of the given schedule as one restart-free segment (G is
 * advanced after every iteration but the last), writing Q in fp16. */
GNS_API int gns_frobenius_sumsq(int x_dtype, int64_t batch, int64_t rows, int64_t cols,
                                const void* x, int64_t x_bstride, int64_t x_rstride, float* sumsq_out,
                                void* workspace, size_t workspace_bytes, gns_stream_t stream);
GNS_API int gns_frobenius_scale(int x_dtype, int64_t batch, int64_t rows, int64_t cols,
                                const void* x, int64_t x_bstride, int64_t x_rstride, const float* sumsq,
                                float eps, void* out_f16, int64_t out_ld, gns_stream_t stream);
GNS_API size_t gns_gram_iterations_workspace_size(int64_t batch, int64_t m);
GNS_API int gns_gram_iterations(int64_t batch, int64_t m, const void* gram, int gram_f32,
                                int64_t g_bstride, int64_t g_rstride, const double* coeffs, int n_iters,
                                int it_begin, int it_end, void* q_out,
                                int64_t q_bstride, int64_t q_rstride, void* workspace,
                                size_t workspace_bytes, gns_stream_t stream);

/* ----------------------------------------------------------- Muon (K5)
 * Multi-tensor momentum for `count` tensors of numel[i] elements each:
 *   m <- g + mu * m            (torch.add(g, m, alpha=mu, out=m), muon.py:429-434)
 *   u <- g + mu * m   if nesterov (muon.py:435-436), else u is not written
 *   mu == 0: m <- g            (muon.py:425-427)
 * grads/moms/updates are arrays of device pointers held in HOST memory; every
 * grad has g_dtype, every momentum m_dtype, every update u_dtype (torch's type
 * promotion of g_dtype and m_dtype). The gradient is first rounded to m_dtype
 * (muon.py:424). With nesterov, updates[i] may be NULL: that tensor's momentum
 * is advanced and no update is written (a rank that does not orthogonalise the
 * matrix needs only the momentum). */
GNS_API int gns_muon_momentum(int count, const void* const* grads, void* const* moms, void* const* updates,
                      const int64_t* numel, int g_dtype, int m_dtype, int u_dtype, float mu,
                      int nesterov, gns_stream_t stream);

/* Multi-tensor parameter update (muon.py:471-476):
 *   p <- p * decay            (only when apply_decay != 0; decay = 1 - lr * wd)
 *   p <- p - lr_adj[i] * o    (o read with its own dtype)
 * Each step rounds to the parameter dtype, as the two torch in-place ops do. */
GNS_API int gns_muon_apply(int count, void* const* params, const void* const* updates, const int64_t* numel,
                   int p_dtype, int o_dtype, float decay, int apply_decay, const float* lr_adj,
                   gns_stream_t stream);

/* ---------------------------------------------------------- Dion3 (K6-K8)
 * Row selection for one [batch, rows, cols] matrix stack (contiguous):
 *   m <- m + g;  p <- p * parameter_decay (if != 1);  row L1 norms of m;
 *   top-`selected` rows per matrix by L1 norm, emitted as ascending int64 indices;
 *   selected <- bf16(m[idx]);  m[idx] <- m[idx] * decay.
 * selected == rows selects every row (identity indices). selected must be in [1, rows].
 * m, g and p share `dtype`. Replaces select_rows (kernels/dion3_cuda.cu:336-351) and its
 * torch twin select_dion3_rows (dion3_update.py:14-70); at::topk is replaced by a
 * radix select whose index order is ascending. */
GNS_API size_t gns_dion3_select_workspace_size(int64_t batch, int64_t rows);
GNS_API int gns_dion3_select_rows(int dtype, int64_t batch, int64_t rows, int64_t cols, void* momentum,
                          const void* gradient, void* parameter, int64_t selected, float decay,
                          float parameter_decay, void* selected_out_bf16, int64_t* indices_out,
                          void* workspace, size_t workspace_bytes, gns_stream_t stream);

/* gns_dion3_select_rows over a list of `count` separate same-shape tensors
 * (rows x cols each, contiguous, one dtype): momenta[i], gradients[i] and
 * parameters[i] (parameters may be NULL when parameter_decay == 1) are the i-th
 * matrices; the outputs are one contiguous stack, selected_out_bf16 as
 * [count, selected, cols] and indices_out as [count, selected]; workspace:
 * gns_dion3_select_workspace_size(count, rows) bytes. The same kernels run over
 * all matrices in a few launches, so a Dion3 bucket costs three launches
 * instead of three per matrix. Replaces the per-tensor loop of
 * select_dion3_rows_cuda_batch (kernels/dion3_cuda.py:111-149). */
GNS_API int gns_dion3_select_rows_multi(int dtype, int count, int64_t rows, int64_t cols, void* const* momenta,
                                        const void* const* gradients, void* const* parameters, int64_t selected,
                                        float decay, float parameter_decay, void* selected_out_bf16,
                                        int64_t* indices_out, void* workspace, size_t workspace_bytes,
                                        gns_stream_t stream);

/* NorMuon normalisation + scatter update (kernels/dion3_cuda.cu:353-503,
 * dion3_update.py:73-148) for one [batch, rows, cols] parameter stack:
 *   v[idx] <- beta2 * v[idx] + (1 - beta2) * mean(u^2)        (fp32 variance [batch, rows])
 *   n = u / (sqrt(v[idx]) + eps), rescaled by ||u||_F / max(||n||_F, eps) per matrix
 *   p[idx] <- p[idx] - lr_adj * n   (p *= 1 - lr * wd first when wd != 0)
 * u is [batch, selected, cols] with dtype u_dtype and row stride u_rstride. */
GNS_API size_t gns_dion3_normalize_workspace_size(int64_t batch, int64_t selected);
GNS_API int gns_dion3_normalize_apply(int p_dtype, int u_dtype, int64_t batch, int64_t rows, int64_t cols,
                              int64_t selected, void* parameter, const void* update,
                              int64_t u_bstride, int64_t u_rstride, float* variance,
                              const int64_t* indices, float beta2, float eps, float lr, float wd,
                              float lr_adj, void* workspace, size_t workspace_bytes,
                              gns_stream_t stream);

/* gns_dion3_normalize_apply over a list of `count` separate same-shape
 * parameters (parameters[i], rows x cols, contiguous) and their variances
 * (variances[i], rows fp32); the update is one [count, selected, cols] stack
 * with strides (u_bstride, u_rstride) and indices one [count, selected] stack;
 * workspace: gns_dion3_normalize_workspace_size(count, selected) bytes.
 * Replaces the per-tensor loop of normalize_apply_rows_cuda_batch
 * (kernels/dion3_cuda.py:220-253). */
GNS_API int gns_dion3_normalize_apply_multi(int p_dtype, int u_dtype, int count, int64_t rows, int64_t cols,
                                            int64_t selected, void* const* parameters, const void* update,
                                            int64_t u_bstride, int64_t u_rstride, float* const* variances,
                                            const int64_t* indices, float beta2, float eps, float lr, float wd,
                                            float lr_adj, void* workspace, size_t workspace_bytes,
                                            gns_stream_t stream);

/* ------------------------------------------------------ AdamW / Lion groups
 * Multi-tensor replacements of Muon's per-parameter AdamW and Lion groups
 * (muon.py:516-583), same roundings as the torch sequence there (every
 * intermediate rounded to its tensor's dtype; division by a host scalar as a
 * multiplication by its float reciprocal). Tensors of one call share
 * p_dtype (parameters), g_dtype (gradients) and s_dtype (state), are
 * contiguous, and are updated in place. AdamW takes per-tensor bias
 * corrections computed on the host in double: lr_bc1[i] = float(lr / (1 -
 * beta1^step_i)) and inv_bc2[i] = float(1 / sqrt(1 - beta2^step_i)) (reciprocal in double).
 * Every scalar is the float rounding of the host's double value, as torch
 * passes scalars: one_minus_beta = float(1 - beta) is computed from the double
 * beta, decay = float(1 - lr * weight_decay), applied when apply_decay is set. */
GNS_API int gns_adamw_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs,
                           void* const* exp_avg_sqs, const int64_t* numel, int p_dtype, int g_dtype, int s_dtype,
                           const float* lr_bc1, const float* inv_bc2, float beta1, float beta2,
                           float one_minus_beta1, float one_minus_beta2, float epsilon, float decay,
                           int apply_decay, gns_stream_t stream);
GNS_API int gns_lion_step(int count, void* const* params, const void* const* grads, void* const* buffers,
                          const int64_t* numel, int p_dtype, int g_dtype, int s_dtype, float lr, float beta1,
                          float beta2, float one_minus_beta1, float one_minus_beta2, float decay, int apply_decay,
                          gns_stream_t stream);

/* The two halves of gns_dion3_normalize_apply as separate calls, for callers of
 * the reference's normalize_rows / apply_rows (kernels/dion3_cuda.py:151-192,
 * kernels/dion3_cuda.cu:353-470):
 * gns_dion3_normalize_rows updates the variance of the selected rows and writes
 * normalized (fp32, [batch * selected][cols], contiguous) = u / (sqrt(v) + eps)
 * and squared_norms (fp32, [batch][2]) = (sum |u|^2, sum |normalized|^2) per
 * matrix; workspace: gns_dion3_normalize_workspace_size bytes.
 * gns_dion3_apply_rows decays the parameter by (1 - lr * wd) and adds
 * -lr_adj * normalized * sqrt(sum |u|^2) / max(sqrt(sum |n|^2), eps) to the
 * selected rows, with the same roundings as the fused call. */
GNS_API int gns_dion3_normalize_rows(int u_dtype, int64_t batch, int64_t rows, int64_t cols, int64_t selected,
                                     const void* update, int64_t u_bstride, int64_t u_rstride, float* variance,
                                     const int64_t* indices, float beta2, float eps, float* normalized,
                                     float* squared_norms, void* workspace, size_t workspace_bytes,
                                     gns_stream_t stream);
GNS_API int gns_dion3_apply_rows(int p_dtype, int64_t batch, int64_t rows, int64_t cols, int64_t selected,
                                 void* parameter, const float* normalized, const int64_t* indices,
                                 const float* squared_norms, float lr, float wd, float lr_adj, float eps,
                                 gns_stream_t stream);

/* --------------------------------------------------- AdamW states in 8 bits
 * One AdamW step over `count` contiguous tensors, in fp32 arithmetic with one
 * rounding of the parameter (gns_adamw_step instead rounds after every step, as
 * the torch sequence it replaces):
 *   g' = s g;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
 *   p  = p * decay - lr_bc1[i] * m / (sqrt(v) * inv_bc2[i] + epsilon)
 * with lr_bc1[i] = lr / (1 - b1^step), inv_bc2[i] = 1 / sqrt(1 - b2^step) and
 * decay = 1 - lr * weight_decay. s is read from device memory at grad_scale (a
 * clipping factor, or the inverse of a loss scale), NULL meaning 1.
 * state_bits 32: exp_avgs and exp_avg_sqs are fp32. state_bits 8: they are e4m3
 * bytes, and exp_avg_scales[i] / exp_avg_sq_scales[i] hold one fp32 scale for
 * each 256 consecutive elements of tensor i (the last block may be shorter):
 * the value of an element is its e4m3 value times its block's scale. Scales are
 * the block's largest magnitude / 448; values round to nearest, and a second
 * moment above zero never rounds to zero. A block whose largest magnitude is
 * at most 1e-30 is held as zeros (a second moment there at the smallest code).
 * A gradient that is not finite makes its block's states NaN.
 * Parameters share p_dtype, gradients g_dtype. Tensors with numel 0 are skipped.
 * No counterpart in the reference. */
GNS_API int gns_adamw_states_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs,
                                  void* const* exp_avg_sqs, float* const* exp_avg_scales,
                                  float* const* exp_avg_sq_scales, const int64_t* numel, int p_dtype, int g_dtype,
                                  int state_bits, const float* lr_bc1, const float* inv_bc2, float beta1,
                                  float one_minus_beta1, float beta2, float one_minus_beta2, float epsilon,
                                  float decay, const float* grad_scale, gns_stream_t stream);
/* The same with 8-bit states whose values round up or down with the probabilities that
 * make their mean right, instead of to nearest. To nearest, a value that decays by less
 * than half a code a step stays where it is: a second moment above its exact value comes
 * down only as its block's scale does. The random bits follow from steps[i] (the tensor's
 * step number), the tensor's place i and the element's place in it: equal calls give equal
 * bits (for tensors that start on 16 bytes and that do not, different ones). */
GNS_API int gns_adamw_states_step_unbiased(int count, void* const* params, const void* const* grads,
                                           void* const* exp_avgs, void* const* exp_avg_sqs,
                                           float* const* exp_avg_scales, float* const* exp_avg_sq_scales,
                                           const int64_t* numel, int p_dtype, int g_dtype, const uint32_t* steps,
                                           const float* lr_bc1, const float* inv_bc2, float beta1,
                                           float one_minus_beta1, float beta2, float one_minus_beta2, float epsilon,
                                           float decay, const float* grad_scale, gns_stream_t stream);

/* ------------------------------------------------ products grouped by expert
 * Rows are sorted by group: group e owns the rows [ends[e - 1], ends[e]) (from 0
 * for the first). `ends` is in device memory, 32- or 64-bit integers (ends_bits);
 * its values are clamped to [0, rows] and to ascending order. left and right
 * share ab_dtype (F16 or BF16); sums are fp32. At most 1024 groups.
 *
 * gns_grouped_gemm: out[r] = left[r] . right[e] for the rows r of group e; rows
 * past the last end come out zero. left is [rows][k] with unit column stride,
 * right [group][k][n] with a unit stride along k or along n, out [rows][n] with
 * unit column stride. Base addresses 16-byte aligned and the other strides
 * multiples of 16 bytes (a TMA rule; out may have any row stride that keeps its rows apart).
 *
 * gns_grouped_gemm_reduce: out[e] = left[rows of e]^T . right[rows of e], zero for
 * a group without rows. left is [rows][m], right [rows][n], both with unit column
 * stride and aligned as above; out is [group][m][n] with unit column stride.
 * No counterpart in the reference (its products are batched, of equal sizes). */
GNS_API int gns_grouped_gemm(int ab_dtype, int64_t rows, int64_t n, int64_t k, int64_t groups, const void* left,
                             int64_t left_rstride, const void* right, int64_t right_gstride, int64_t right_rstride,
                             int64_t right_cstride, const void* ends, int ends_bits, void* out, int out_dtype,
                             int64_t out_rstride, gns_stream_t stream);
/* How gns_grouped_gemm runs a product of these sizes on the current device: the rows of
 * a tile (64, 128: a CTA; 256, 512: a pair) and the CTAs that share a tile's contraction
 * (1, 2, 4 or 8). */
GNS_API int gns_grouped_gemm_plan(int64_t rows, int64_t n, int64_t k, int64_t groups, int* tile_rows, int* split);
/* Copies [batch][rows][cols] of a 16-bit type with unit column stride, wherever its
 * rows start, to rows that start on 16 bytes (dst and its strides in 16-byte
 * multiples, a row of dst holding cols rounded up to 8): operands that the TMA rule
 * excludes. With `ends` (one for each of the batch, else NULL), matrices of groups
 * without rows are not copied. */
GNS_API int gns_align_rows(int64_t batch, int64_t rows, int64_t cols, const void* src, int64_t src_bstride,
                           int64_t src_rstride, const void* ends, int ends_bits, void* dst, int64_t dst_bstride,
                           int64_t dst_rstride, gns_stream_t stream);
GNS_API int gns_grouped_gemm_reduce(int ab_dtype, int64_t rows, int64_t m, int64_t n, int64_t groups,
                                    const void* left, int64_t left_rstride, const void* right, int64_t right_rstride,
                                    const void* ends, int ends_bits, void* out, int out_dtype, int64_t out_gstride,
                                    int64_t out_rstride, gns_stream_t stream);

/* -------------------------------------------------------------- layer norm
 * y = (x - mean) * rstd * weight + bias over the last dimension of [rows][cols],
 * rstd = 1 / sqrt(var + eps) with the biased variance; mean and rstd (fp32, one
 * value per row) are written for the backward pass. x has unit column stride and
 * x_rstride elements between rows; y is contiguous, of x's type. weight and bias
 * share w_dtype; bias may be NULL.
 * Backward: dx (contiguous, x's type), and dweight / dbias (w_dtype), the sums
 * over all rows of grad * (x - mean) * rstd and of grad, in fp32 and in a fixed
 * order; dbias may be NULL. rows may be 0 (the sums are then zero).
 * Rows that do not start and end on 16 bytes are read in whole multiples of 16 bytes: up
 * to 15 bytes on either side of a row, in the same 16 as one of its elements, are read
 * and not used.
 * No counterpart in the reference. */
GNS_API int gns_layer_norm_forward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* x,
                                   int64_t x_rstride, const void* weight, const void* bias, float eps, void* y,
                                   float* mean, float* rstd, gns_stream_t stream);
GNS_API size_t gns_layer_norm_backward_workspace_size(int64_t rows, int64_t cols);
GNS_API int gns_layer_norm_backward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* grad,
                                    int64_t grad_rstride, const void* x, int64_t x_rstride, const void* weight,
                                    const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                                    void* workspace, size_t workspace_bytes, gns_stream_t stream);

/* -------------------------------------------------- products of 8-bit matrices
 * out = left . right with e4m3 operands and fp32 scales for blocks of 128 of the
 * contraction: left [m][k] (unit column stride) has a scale for each row and block
 * [m][ceil(k / 128)], right [k][n] (unit stride along k or along n) one for each 128 x 128
 * block [ceil(k / 128)][ceil(n / 128)]; both arrays of scales have strides of their own.
 * Operands start on 16 bytes and their other strides are multiples of 16 (a TMA rule); out
 * [m][n] is F16, BF16 or F32 with unit column stride. Sums are fp32, rounded once; a block's
 * sum is multiplied by the fp32 product of its two scales.
 * No counterpart in the reference. */
GNS_API int gns_gemm_8bit(int64_t m, int64_t n, int64_t k, const void* left, int64_t left_rstride,
                          const float* left_scales, int64_t left_scale_rstride, int64_t left_scale_cstride,
                          const void* right, int64_t right_rstride, int64_t right_cstride, const float* right_scales,
                          int64_t right_scale_rstride, int64_t right_scale_cstride, void* out, int out_dtype,
                          int64_t out_rstride, gns_stream_t stream);
/* How gns_gemm_8bit runs a product of these sizes on the current device: the rows of left in a
 * tile (16, 32, 128: a CTA; 256: a pair of CTAs) and the CTAs that share a tile's contraction
 * (1, 2, 4 or 8). */
GNS_API int gns_gemm_8bit_plan(int64_t m, int64_t n, int64_t k, int* tile_rows, int* parts);
/* Codes and scales of x [rows][cols] (unit column stride, any row stride of at least cols, or 0):
 * blocks of block_rows (1 or 128) x 128, top = max(largest magnitude, 448 * 2^-126), scale =
 * top / 448, code = e4m3(x * (448 / top)) to nearest even. Rows of codes start on 16 bytes
 * (codes_rstride a multiple of 16) and are written up to cols rounded up to 16, zeros behind
 * the last column. scales [ceil(rows / block_rows)][ceil(cols / 128)] has strides of its own. */
GNS_API int gns_quantize_8bit(int x_dtype, int block_rows, int64_t rows, int64_t cols, const void* x, int64_t x_rstride,
                              void* codes, int64_t codes_rstride, float* scales, int64_t scale_rstride,
                              int64_t scale_cstride, gns_stream_t stream);

/* ----------------------------------------------------- root-mean-square norm
 * total = x + residual, rounded to x's type (x itself where residual is NULL; total is then
 * not written), y = total * rstd * weight, rstd = 1 / sqrt(mean(total^2) + eps). x and residual
 * share x_dtype and have unit column stride; y and total are contiguous; rstd is fp32.
 * The 8-bit form writes codes and scales (blocks of 1 x 128, as gns_quantize_8bit) of the
 * unrounded y in its place.
 * Backward: dx = the gradient through the norm + grad_total (NULL: none), of x and of the
 * residual alike; dweight sums over the rows in fp32, in a fixed order. rows may be 0.
 * x, residual, total, grad and grad_total are read in whole multiples of 16 bytes, as the
 * layer norm's rows are.
 * No counterpart in the reference. */
GNS_API int gns_rms_norm_forward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* x, int64_t x_rstride,
                                 const void* residual, int64_t residual_rstride, const void* weight, float eps, void* y,
                                 void* total, float* rstd, gns_stream_t stream);
GNS_API int gns_rms_norm_forward_8bit(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* x,
                                      int64_t x_rstride, const void* residual, int64_t residual_rstride,
                                      const void* weight, float eps, void* codes, int64_t codes_rstride, float* scales,
                                      int64_t scale_rstride, int64_t scale_cstride, void* total, float* rstd,
                                      gns_stream_t stream);
GNS_API size_t gns_rms_norm_backward_workspace_size(int64_t rows, int64_t cols);
GNS_API int gns_rms_norm_backward(int x_dtype, int w_dtype, int64_t rows, int64_t cols, const void* grad,
                                  int64_t grad_rstride, const void* total, int64_t total_rstride, const void* weight,
                                  const float* rstd, const void* grad_total, int64_t grad_total_rstride, void* dx,
                                  void* dweight, void* workspace, size_t workspace_bytes, gns_stream_t stream);

/* ------------------------------------------------------- distillation loss
 * loss = T^2 sum_j p_j (log p_j - log q[i_j]) of each row: p is the softmax of the row's
 * teacher logits over T, q that of its logits over T and the whole vocabulary. Entries whose
 * index is outside [0, vocabulary) have no part; a row without entries (or with -inf teacher
 * logits only) has a loss and a gradient of zero. top <= 1024, T in [1e-4, 1e4].
 * With grad (fp32, one value a row) and dlogits: dlogits = grad T (q - p), of the logits' type.
 * stats (fp32, two values a row: the largest logit and the sum of exponentials) is written
 * with the loss where it is not NULL; with loss NULL the gradient is formed from it. It starts
 * on 8 bytes.
 * logits, indices, teacher and dlogits have unit column stride.
 * No counterpart in the reference. */
GNS_API int gns_distillation_loss(int z_dtype, int64_t rows, int64_t vocabulary, int64_t top, const void* logits,
                                  int64_t logits_rstride, const void* indices, int index_bits, int64_t indices_rstride,
                                  const void* teacher, int teacher_dtype, int64_t teacher_rstride, float temperature,
                                  const float* grad, float* loss, float* stats, void* dlogits, int64_t dlogits_rstride,
                                  gns_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GNS_B200_H_ */
