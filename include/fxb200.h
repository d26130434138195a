/*
 * fxb200.h - C ABI of libfxb200.so, the sm_100a (B200) kernels behind the
 * fxlm / fxgpu operator surface.
 *
 * The reference launches runtime-compiled HIP kernels through ctypes
 * (ml/fxgpu/hip_kernel.py:50-145: compile_kernel / compile_module / launch).
 * This library is built ahead of time and exposes one plain C function per
 * operation instead. Conventions:
 *   - every pointer is a device pointer owned by the caller; the library
 *     never allocates or frees device memory (workspaces are passed in, their
 *     sizes come from the *_workspace functions);
 *   - `stream` is a cudaStream_t (NULL = legacy default stream); no function
 *     synchronises the host except fxb_device_error;
 *   - functions return FXB_OK (0) or a negative FXB_E* code; the message of
 *     the last failure on the calling thread is returned by fxb_last_error().
 *     Nothing exits, aborts or traps.
 *   - dtype codes: FXB_DTYPE_F32 / F16 / BF16.
 */
#ifndef FXB200_H
#define FXB200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FXB_OK 0
#define FXB_EINVAL (-1)      /* bad shape / stride / alignment / pointer */
#define FXB_EUNSUPPORTED (-2) /* valid request this build does not implement */
#define FXB_ECUDA (-3)       /* CUDA runtime / driver error (see fxb_last_error) */

#define FXB_DTYPE_F32 0
#define FXB_DTYPE_F16 1
#define FXB_DTYPE_BF16 2

/* ------------------------------------------------------------------ misc */

/* Library version (major*10000 + minor*100 + patch). */
int fxb_version(void);

/* Message of the last failed call on this thread ("" if none).
 * Replaces the RuntimeError text of _chk, ml/fxgpu/hip_kernel.py:45-47. */
const char* fxb_last_error(void);

/* Reads (and with clear != 0 resets) the device error word that kernels set
 * when a bounded wait expires (bit 1 GEMM, 2 attention, 4 gather, 8 cross-
 * entropy, 32 verification), or when the page table or pool of a KV cache does not fit a call
 * (bit 16). Synchronises
 * the current device. No reference counterpart (the reference has no bounded
 * waits). */
int fxb_device_error(int32_t* code, int32_t clear);

/* Number of streaming multiprocessors of the current device (grid sizing). */
int fxb_num_sms(int32_t* out);

/* Number of kernels this library has launched in this process (all devices). */
uint64_t fxb_launch_count(void);

/* ABI self-check for bindings: sizeof(fxb_gemm_args) for which == 0,
 * sizeof(fxb_attn_args) for which == 1, sizeof(fxb_tree_attn_args) for
 * which == 2, sizeof(fxb_kv_args) for which == 3, 0 otherwise. */
size_t fxb_abi_struct_size(int32_t which);

/* ------------------------------------------------------------------ RMSNorm */

/* y = x * rsqrt(mean(x^2) + eps) * w, rstd saved (fp32, one per row).
 * x, y: (rows, D) contiguous; w: (D,). D % 8 == 0, D <= 8192.
 * Replaces rms_norm_fwd (ml/fxlm/kernels/norm.hip:33) as launched by
 * _RMSNorm.forward (ml/fxlm/norm.py:45-60). */
int fxb_rmsnorm_fwd(int32_t dtype, const void* x, const void* w, void* y, float* rstd,
                    int64_t rows, int32_t D, float eps, void* stream);

/* Bytes of fp32 workspace fxb_rmsnorm_bwd needs for the dw partial sums. */
size_t fxb_rmsnorm_bwd_workspace(int64_t rows, int32_t D);

/* dx = rstd*w*dy - x*rstd^3*sum(x*w*dy)/D (+ dres when dres != NULL: the
 * gradient reaching x through a residual connection, summed in the same pass);
 * dw = sum_rows x*rstd*dy.
 * dw (dtype dw_dtype, e.g. an fp32 flat-gradient slot) is written
 * (dw_accumulate == 0) or added to (dw_accumulate != 0). Any D the forward
 * takes (D % 8 == 0, D <= 8192): rows of up to 2048 16-bit (1024 fp32)
 * elements are handled a warp per row, longer rows a block per row.
 * Deterministic: per-block partials, then a fixed-order sum.
 * Replaces rms_norm_bwd_dx + rms_norm_bwd_dw + part.sum(0)
 * (ml/fxlm/kernels/norm.hip:64,102; ml/fxlm/norm.py:62-84). */
int fxb_rmsnorm_bwd(int32_t dtype, const void* x, const void* w, const float* rstd,
                    const void* dy, const void* dres, void* dx, void* dw, int32_t dw_dtype,
                    int32_t dw_accumulate, float* workspace, int64_t rows, int32_t D,
                    void* stream);

/* fxb_rmsnorm_bwd without a workspace argument: the call allocates nothing.
 * It has no counterpart in the reference; this entry exists for callers
 * that cannot allocate device memory on the call path, e.g. a host runtime
 * with a fixed memory budget that owns no allocator, or code that must not
 * call cudaMalloc / cudaFree (which synchronise the device).
 * Same math, arguments and results as fxb_rmsnorm_bwd (identical block count,
 * so identical dw). The dw partials live in a file-scope device array of
 * fxb_rmsnorm_bwd_static_max_bytes() bytes (4 MiB), one per device:
 *  - the first call on a device looks up that array's address
 *    (cudaGetSymbolAddress) and caches it (again after the device's context
 *    was replaced, e.g. by cudaDeviceReset); make that first call before any
 *    stream capture;
 *  - a call whose partials need more than the array holds
 *    (fxb_rmsnorm_bwd_workspace(rows, D) > the maximum) returns FXB_EINVAL;
 *  - nothing in the array has to start at zero (each block writes all of its
 *    partials before they are read);
 *  - every call on a device shares the array, so two calls that overlap in
 *    time (different streams or host threads) race on it: issue them in order
 *    on one stream. */
size_t fxb_rmsnorm_bwd_static_max_bytes(void);
int fxb_rmsnorm_bwd_static(int32_t dtype, const void* x, const void* w, const float* rstd,
                           const void* dy, const void* dres, void* dx, void* dw,
                           int32_t dw_dtype, int32_t dw_accumulate, int64_t rows, int32_t D,
                           void* stream);

/* ------------------------------------------------------------------ cross entropy */

/* Row-wise softmax cross entropy with the gradient written in the same pass.
 *   row_loss[r] = logsumexp(row) - row[target]   (0 for rows that are not valid)
 *   grad[r,:]   = (softmax(row) - onehot(target)) * (*mul)   (0 for ignored rows)
 * A row is valid when target != ignore_index and 0 <= target < V. The caller
 * sums row_loss (fixed order, deterministic) where the reference accumulated
 * one scalar with atomics.
 * grad may be NULL (loss only) or equal to logits (in place).
 * logits/grad: (rows, V) with row stride ld (elements); target int64 (rows,);
 * row_loss fp32 (rows,); mul is an fp32 device scalar (no host sync).
 * Replaces ce_fwd_grad (ml/fxlm/kernels/ce.hip:32) as launched by _ce_rows
 * (ml/fxlm/cross_entropy.py:47-59). */
int fxb_ce_fwd_grad(int32_t dtype, const void* logits, int64_t ld, const int64_t* target,
                    void* grad, float* row_loss, const float* mul, int64_t rows, int32_t V,
                    int64_t ignore_index, void* stream);

/* ------------------------------------------------------------------ FlatAdamW */

/* scratch[0] += sum(g^2); flags |= 1 if any g is non-finite. g: flat (n,).
 * Replaces adamw_sumsq (ml/fxlm/kernels/optim.hip:26) over the per-tensor
 * TensorList of FlatAdamW._chunks (ml/fxlm/optim.py:107-144). */
int fxb_adamw_sumsq(int32_t gdtype, const void* grad, int64_t n, float* scratch,
                    int32_t* flags, void* stream);

/* Same result as fxb_adamw_sumsq, summed in a fixed order: per-block partial
 * sums go to the workspace `ws` (fxb_adamw_sumsq_ws_bytes() bytes, 4-byte
 * aligned, zero-filled once before its first use; every call leaves its
 * ticket counter at zero) and the block that finishes last adds them in
 * block order. The
 * norm is then bitwise reproducible, so data-parallel ranks holding the same
 * reduced gradient take bitwise identical optimizer steps. One workspace per
 * stream (concurrent calls must not share it). No reference counterpart: the
 * reference accumulates with atomicAdd (ml/fxlm/kernels/optim.hip:71). */
size_t fxb_adamw_sumsq_ws_bytes(void);
int fxb_adamw_sumsq_det(int32_t gdtype, const void* grad, int64_t n, float* scratch,
                        int32_t* flags, void* ws, void* stream);

/* One thread: found_inf = flags || !isfinite(scratch[0]);
 * norm = sqrt(scratch[0]) / scale; scratch[1] = clip coefficient
 * min(1, max_norm/(norm+1e-6)) (0 when found_inf); step += !found_inf;
 * flags and scratch[0] reset for the next step.
 * Replaces adamw_final (ml/fxlm/kernels/optim.hip:77-93). */
int fxb_adamw_final(float* scratch, int32_t* flags, int32_t* step, float* found_inf,
                    float* norm_out, const float* scale, float max_norm, void* stream);

/* Flat decoupled-weight-decay AdamW over n elements (skipped when *found_inf):
 *   g = grad * scratch[1] / scale; w -= lr*wd*w (segments with seg_wd != 0);
 *   m = b1*m + (1-b1) g; v = b2*v + (1-b2) g^2;
 *   w -= lr * (m / (1-b1^step)) / (sqrt(v / (1-b2^step)) + eps);
 *   master = w; param = (pdtype) w; grad = 0 (the gradient is consumed, also
 *   when the step is skipped, so the buffer is ready for the next backward).
 * Segments: seg_end[i] (exclusive, device int64, ascending, multiples of 8) and
 * seg_wd[i] (device int32), nseg <= 1024.
 * lr_dev: when non-NULL the learning rate is read from this device fp32
 * scalar and `lr` is ignored, so a captured CUDA graph can follow a schedule
 * (the host updates the scalar between replays).
 * Replaces adamw_update (ml/fxlm/kernels/optim.hip:96-162). */
int fxb_adamw_update(int32_t gdtype, int32_t pdtype, const void* grad, float* master,
                     float* m, float* v, void* param, int64_t n, const int64_t* seg_end,
                     const int32_t* seg_wd, int32_t nseg, const float* scratch,
                     const float* found_inf, const float* scale, const int32_t* step,
                     float lr, const float* lr_dev, float beta1, float beta2, float eps,
                     float weight_decay, void* stream);

/* ------------------------------------------------------------------ GEMM */

/* Epilogues applied to acc = sum_k A[m,k] * B[n,k] (fp32 in tensor memory). */
#define FXB_EPI_STORE 0     /* C = alpha*acc */
#define FXB_EPI_RESIDUAL 1  /* C = alpha*acc + R  (R may alias C: accumulate) */
#define FXB_EPI_GELU 2      /* Z = acc ; C = gelu_tanh(acc) */
#define FXB_EPI_DGELU 3     /* C = acc * gelu_tanh'(R)   (R = pre-activation) */
#define FXB_EPI_BIAS 4      /* C = acc + bias[n] */
#define FXB_EPI_BIAS_GELU 5 /* Z = acc + bias[n] ; C = gelu_tanh(Z) */
#define FXB_EPI_BIAS_SILU 6 /* Z = acc + bias[n] ; C = silu(Z) */
#define FXB_EPI_ACCUM_F32 7 /* C(fp32) += alpha*acc (red.add; enables split-K) */
#define FXB_EPI_DSILU 8     /* C = acc * silu'(R)        (R = pre-activation) */
#define FXB_EPI_GELU_DERIV 9 /* C = gelu_tanh(p) ; Z = gelu_tanh'(p), p = acc rounded to C's type */
#define FXB_EPI_MUL 10      /* C = alpha*acc*R  (with Z of FXB_EPI_GELU_DERIV as R: the
                               GELU backward without recomputing the activation) */

typedef struct fxb_gemm_args {
  int32_t dtype;     /* A/B dtype: FXB_DTYPE_BF16 / FXB_DTYPE_F16 (tensor cores) or
                        FXB_DTYPE_F32 (fp32 parity mode: C, R, Z, bias fp32 too) */
  int32_t M, N, K;
  const void* A;     /* a_trans == 0: (M,K) row stride lda; 1: (K,M) row stride lda */
  int64_t lda;
  int32_t a_trans;
  const void* B;     /* b_trans == 0: (N,K) row stride ldb; 1: (K,N) row stride ldb */
  int64_t ldb;
  int32_t b_trans;
  void* C;           /* (M,N) row stride ldc, dtype c_dtype */
  int64_t ldc;
  int32_t c_dtype;
  int32_t epilogue;  /* FXB_EPI_* */
  float alpha;
  const void* R;     /* residual / pre-activation input, dtype c_dtype, row stride ldr */
  int64_t ldr;
  void* Z;           /* second output (pre-activation), dtype c_dtype, row stride ldz */
  int64_t ldz;
  const void* bias;  /* (N,), dtype c_dtype */
  /* Optional scratch (NULL: none) of workspace_bytes >= fxb_gemm_workspace_size()
   * bytes, 16-byte aligned, whose first 4096 bytes (arrival counters) are
   * zero-filled once before its first use (the kernels leave them at zero). With it, tiles that would leave most of the
   * last wave idle are split along K and their pieces reduced through it; it
   * must not be shared by calls that can run concurrently (one per stream). */
  void* workspace;
  int64_t workspace_bytes;
} fxb_gemm_args;

/* tcgen05 / TMEM GEMM with TMA-fed operands. Requires K % 8 == 0 for K-major
 * operands and M (resp. N) % 8 == 0 for transposed ones (16-byte TMA rows),
 * 16-byte aligned bases, N % 8 == 0 for C.
 * dtype FXB_DTYPE_F32 runs an fp32 SIMT kernel instead (every epilogue, exact
 * tanh / exp, no shape or alignment constraints beyond positive leading
 * dimensions): the 1e-5 fp32 parity mode, not a fast path.
 * Replaces the rocBLAS matmuls on the hot path: nn.Linear qkv/proj/fc/fc2
 * (ml/fxlm/model.py:48-51,61,69-71), the linear-CE chunk mm's
 * (ml/fxlm/cross_entropy.py:131-135,180) and the fxgpu dW mm
 * (ml/fxgpu/fused_linear.py:94). */
int fxb_gemm(const fxb_gemm_args* args, void* stream);

/* Bytes of fxb_gemm_args.workspace that enable the tail split on the current
 * device. No reference counterpart (the reference's rocBLAS calls own their
 * scratch). */
size_t fxb_gemm_workspace_size(void);

/* The tile configuration fxb_gemm would use for this problem on the current
 * device: *pair = 1 for the CTA-pair (cta_group::2, 256-row) kernel, 0 for the
 * single-CTA (128-row) kernel; *bn = tile width; *splits = split-K factor
 * (> 1 for FXB_EPI_ACCUM_F32), or for the other epilogues the number of K
 * pieces of each tail tile when a workspace is given (1: no tail split).
 * Diagnostic; no reference counterpart. */
int fxb_gemm_plan(int32_t M, int32_t N, int32_t K, int32_t epilogue, int32_t* pair,
                  int32_t* bn, int32_t* splits);

/* Loss-only linear cross entropy with the logits kept on chip:
 *   row_loss[r] = logsumexp_v(x_r . w_v) - x_r . w_{target[r]}
 * (0 for rows whose target is ignore_index or outside [0, V)). The tcgen05
 * GEMM of x (N, D) by w (V, D)^T reduces each accumulator tile in tensor
 * memory to per-row (max, sum of exp) pairs and the target column's value
 * (fp32, before any rounding), so no (N, V) logits are written; a second
 * kernel merges the pairs per row. x, w bf16 or f16, 16-byte aligned, D and
 * V multiples of 8; workspace of fxb_linear_ce_loss_workspace(N, V) bytes,
 * 16-byte aligned. The caller sums row_loss (fixed order) and divides by the
 * number of valid rows.
 * Replaces the loss-only chunk loop of _linear_ce_loss_only
 * (ml/fxlm/cross_entropy.py:170-183: mm to a logits chunk, then ce_fwd_grad
 * without gradient, ml/fxlm/kernels/ce.hip:32). */
size_t fxb_linear_ce_loss_workspace(int64_t N, int32_t V);
int fxb_linear_ce_loss(int32_t dtype, const void* x, int64_t ldx, const void* w, int64_t ldw,
                       const int64_t* target, float* row_loss, void* workspace, int64_t N,
                       int32_t D, int32_t V, int64_t ignore_index, void* stream);

/* ------------------------------------------------------------------ attention */

typedef struct fxb_attn_args {
  int32_t dtype;          /* FXB_DTYPE_BF16 or FXB_DTYPE_F16 */
  int32_t B, T, H, D;     /* D = head dim (64 or 128) */
  float scale;
  int32_t causal;
  /* (B,T,H,D) views with unit stride on D; strides in elements (b, t, h) */
  const void* q; int64_t q_sb, q_st, q_sh;
  const void* k; int64_t k_sb, k_st, k_sh;
  const void* v; int64_t v_sb, v_st, v_sh;
  void* o;       int64_t o_sb, o_st, o_sh;   /* forward output; backward input */
  float* lse;                                /* (B,H,T) natural-log LSE of scaled scores */
  const void* dout; int64_t do_sb, do_st, do_sh;
  void* dq;      int64_t dq_sb, dq_st, dq_sh;
  void* dk;      int64_t dk_sb, dk_st, dk_sh;
  void* dv;      int64_t dv_sb, dv_st, dv_sh;
  float* workspace;                          /* backward: fxb_attn_bwd_workspace bytes */
} fxb_attn_args;

/* Causal / non-causal flash-attention forward: o = softmax(q k^T * scale) v,
 * lse = logsumexp of the scaled scores (natural log). dtype bf16 / f16 run
 * the tcgen05 kernel (strides multiples of 8 elements, 16-byte aligned
 * bases); dtype f32 runs an fp32 SIMT kernel (the 1e-5 parity mode; any
 * positive strides). Head dim 64 or 128.
 * Replaces attn_fwd (ml/fxlm/kernels/attention.hip:104) as launched by _fwd
 * (ml/fxlm/attention.py:87-104). */
int fxb_attn_fwd(const fxb_attn_args* args, void* stream);

/* Workspace bytes for fxb_attn_bwd (delta = rowsum(dO*O), fp32 dQ staging). */
size_t fxb_attn_bwd_workspace(int32_t B, int32_t T, int32_t H, int32_t D);

/* Flash-attention backward: dq, dk, dv from q, k, v, o, lse, dout (head dim
 * 64 or 128; bf16 / f16 on tensor cores, f32 as the forward).
 * Replaces attn_bwd_prep + attn_bwd_dkv + attn_bwd_dq
 * (ml/fxlm/kernels/attention.hip:229,256,411) as launched by _bwd
 * (ml/fxlm/attention.py:107-134). */
int fxb_attn_bwd(const fxb_attn_args* args, void* stream);

/* ------------------------------------------------------------------ embedding / glue */

/* out[b,t,:] = tok[idx[b,t],:] + pos[t,:]. idx int64 (B*T). Rows of out are D
 * contiguous; dtype bf16, f16 or f32; D % 8 == 0, 16-byte aligned buffers. Replaces tok_emb(idx) + pos_emb[:T] (ml/fxlm/model.py:118). */
int fxb_embedding_fwd(int32_t dtype, const int64_t* idx, const void* tok, const void* pos,
                      void* out, int64_t B, int64_t T, int32_t D, int64_t V, void* stream);

/* dtok_ws[idx[b,t],:] += dout[b,t,:], dpos_ws[t,:] += dout[b,t,:] (fp32
 * workspaces, zeroed by the caller, 16-byte aligned; fp32 vector reductions).
 * Backward of ml/fxlm/model.py:118. */
int fxb_embedding_bwd(int32_t dtype, const int64_t* idx, const void* dout, float* dtok_ws,
                      float* dpos_ws, int64_t B, int64_t T, int32_t D, int64_t V,
                      void* stream);

/* dst[i] = (accumulate ? dst[i] : 0) + src[i] * (scale ? *scale : 1) for i < n.
 * dst dtype ddtype, src dtype sdtype, scale an fp32 device scalar or NULL.
 * Carries the linear-CE backward rescale (ml/fxlm/cross_entropy.py:140-149). */
int fxb_axpy(int32_t ddtype, void* dst, int32_t sdtype, const void* src, const float* scale,
             int32_t accumulate, int64_t n, void* stream);

/* ------------------------------------------------------------------ fxgpu window model */

/* Xg[b, :] = X[idx[b] : idx[b] + window, :] flattened window-major (K = window*F),
 * i.e. Xg[b, w*F + f] = X[idx[b] + w, f]. X (R, F) row-major (bf16, f16 or
 * f32), F % 8 == 0,
 * idx int32; windows that leave [0, R) are written as zeros.
 * Replaces the A-operand gather and the Xg write-out of gather_gemm
 * (ml/fxgpu/gather_gemm.hip:17-180, launched by ml/fxgpu/fused_linear.py:76-85);
 * the GEMM itself runs through fxb_gemm with FXB_EPI_BIAS*. */
int fxb_gather_windows(int32_t dtype, const void* X, int64_t R, int32_t F, const int32_t* idx,
                       int32_t B, int32_t window, void* Xg, void* stream);

/* out[c] (fp32) = (accumulate ? out[c] : 0) + sum_r g[r, c]; g (rows, cols) row-major
 * (may be NULL when rows == 0). Deterministic (fixed summation order, no atomics).
 * The bias gradient db = g.sum(0) of ml/fxgpu/fused_linear.py:95. */
int fxb_colsum(int32_t dtype, const void* g, int64_t rows, int32_t cols, float* out,
               int32_t accumulate, void* stream);

/* ------------------------------------------------------------------ generation over a paged KV cache
 *
 * Not in the reference, whose sampler re-runs the whole window for every
 * token (ml/fxlm/sample.py:63-73). The cache is a pool of P pages of `page`
 * token slots each (page a power of two, 16..256). Sequence (batch row) s
 * holds its tokens in order in the pages table[s, 0..n_pages[s]); ref[p]
 * counts the rows that hold page p, and a page is free when its count is 0.
 * A page held by more than one row is full and is only read. Lengths, tables
 * and counts live on the device and every call is capturable in a CUDA graph.
 * Wrong contents of these arrays (a page id outside the pool where a page is
 * needed, a pool without enough free pages, a path that does not ascend) do
 * not fault: the access is skipped and bit 16 of the device error word is set
 * (fxb_device_error). */

/* Attention of the nodes of a token tree over the cache, which also writes
 * the nodes' keys and values:
 *   o[b,t,h] = sum_j p_j v_j,  p = softmax_j(scale * q[b,t,h] . k_j)
 * over j in the cache slots [0, lens[b]) of row b and the nodes j < n_nodes[b]
 * with bit j of mask[b,t] set; h's key head is h / (Hq/Hkv). A row without
 * any j, and rows t >= n_nodes[b], are written as zeros. k[b,j], v[b,j] of the
 * nodes j < n_nodes[b] go to the cache slots lens[b] + j (which have to be
 * held). T == 1 is plain decoding of one token.
 * What lies in slots from lens[b] on, in nodes from n_nodes[b] on and in nodes
 * that the mask hides does not reach a row's output, whatever its value. */
typedef struct fxb_tree_attn_args {
  int32_t dtype;            /* FXB_DTYPE_* of every tensor */
  int32_t B, T, Hq, Hkv, D; /* T <= 64; Hq a multiple of Hkv; D = 64 or 128 */
  int32_t page, P, W;       /* slots per page, pages of the pool, entries of a table row */
  float scale;
  /* element strides, unit stride on D; strides multiples of 16 bytes (that of an axis of one entry may be
   * anything), 16-byte aligned bases */
  const void* q; int64_t q_sb, q_st, q_sh;             /* (B,T,Hq,D) */
  const void* k; int64_t k_sb, k_st, k_sh;             /* (B,T,Hkv,D) */
  const void* v; int64_t v_sb, v_st, v_sh;
  void* o;       int64_t o_sb, o_st, o_sh;             /* (B,T,Hq,D) */
  void* k_pages; int64_t kp_sp, kp_sh, kp_st;          /* (P,Hkv,page,D) */
  void* v_pages; int64_t vp_sp, vp_sh, vp_st;
  const int32_t* table; int64_t table_sb;              /* (B,W) */
  const int32_t* lens;                                 /* (B,) */
  const int32_t* n_nodes;                              /* (B,) in [0,T] */
  const int64_t* mask; int64_t mask_sb;                /* (B,T); mask_sb 0: one tree for all rows */
  void* workspace; int64_t workspace_bytes;            /* fxb_tree_attn_workspace bytes */
} fxb_tree_attn_args;

/* Workspace bytes of fxb_tree_attn on the current device (partial results of
 * sequences that several thread blocks share), 16-byte aligned. Its first
 * fxb_tree_attn_workspace_zeroed(...) bytes have to be zero before its first
 * use; every call leaves them zero. One workspace per stream. */
size_t fxb_tree_attn_workspace(int32_t dtype, int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D);
size_t fxb_tree_attn_workspace_zeroed(int32_t dtype, int32_t B, int32_t T, int32_t Hq, int32_t Hkv,
                                      int32_t D);
int fxb_tree_attn(const fxb_tree_attn_args* args, void* stream);

/* Verification of drafted tokens. Row b is a tree of n_nodes[b] <= T <= 64
 * nodes, parents[b,c] < c; node 0 is the last committed token, the others
 * carry drafted tokens. p[b,i,:] is the target's distribution after node i.
 * The walk starts at node 0 and tries the children c of the current node in
 * index order: c is accepted, and becomes the current node, when
 *   with q (q[b,i,:]: the distribution from which each child of node i was
 *   drawn independently):  u[b,c] * q(x_c) < w(x_c), else
 *       w = max(w - q, 0) / sum(max(w - q, 0)),    w = p at first;
 *   without q (drafts that were not drawn at random):
 *       u[b,c] * m < w(x_c), else m = max(m - w(x_c), 0), w(x_c) = 0,
 *       w = p and m = 1 at first.
 * When no child is accepted, the next token is drawn from w (from p where w is
 * empty) by inversion with u[b,0]: the first token at which the running sum
 * exceeds floor(u * total). So accepted tokens and the next one are
 * distributed as if drawn from the target.
 * Sums are taken over floor(w * 2^36) in 64-bit integers, so results do not
 * depend on the order of summation; values that are not above 0 (NaN among
 * them) count as 0, values above 1 as 1.
 * A parent that is no earlier node counts as none; n_nodes outside [0, T] counts
 * as the nearer end (bit 16 of the device error word).
 * path (B,T): the accepted nodes in order, node 0 first, then -1; n_path (B):
 * their number; next (B): the drawn token, -1 for n_nodes == 0 or an empty row. */
int fxb_verify_tree(const int64_t* tokens, const int32_t* parents, const int32_t* n_nodes,
                    const float* p, int64_t p_sb, int64_t p_st, const float* q, int64_t q_sb,
                    int64_t q_st, const float* u, int32_t* path, int32_t* n_path, int64_t* next,
                    int32_t B, int32_t T, int32_t V, void* stream);

/* The cache of all layers, as fxb_kv_commit and fxb_kv_fork see it. */
typedef struct fxb_kv_args {
  int32_t elem_size;        /* bytes of one element (2 or 4); D * elem_size a multiple of 16 */
  int32_t L, P, H, page, D;
  void* k; int64_t k_sl, k_sp, k_sh, k_st;             /* (L,P,H,page,D), strides as above */
  void* v; int64_t v_sl, v_sp, v_sh, v_st;
  int32_t S, W;
  int32_t* table; int64_t table_ss;                    /* (S,W) */
  int32_t* n_pages;                                    /* (S,) */
  int32_t* lens;                                       /* (S,) */
  int32_t* ref;                                        /* (P,) */
} fxb_kv_args;

/* Commits a path of each row and makes room: token i < n_path[s] moves from
 * slot lens[s] + path[s,i] to slot lens[s] + i in every layer (path ascends
 * strictly; path == NULL: nothing moves and n_path counts as 0), then
 * lens_out[s] = lens[s] + n_path[s], and where room[s] > 0 (room may be NULL)
 * the row is given pages for lens_out[s] + room[s] slots: the lowest-numbered
 * free ones, rows in order. If the pool lacks them no row is given any. A token
 * whose entry does not ascend, or whose slot the row does not hold, stays where
 * it is, the others move; n_path outside [0, T] counts as the nearer end (bit
 * 16 of the device error word in each case). lens_out must be an array of its
 * own, neither lens nor another argument. */
int fxb_kv_commit(const fxb_kv_args* args, const int32_t* path, int64_t path_ss, int32_t T,
                  const int32_t* n_path, const int32_t* room, int32_t* lens_out, void* stream);

/* Row s becomes a fork of row parents[s] as it was before the call (s itself:
 * it stays; -1: it is emptied). Full pages are shared. A last page that is
 * only partly filled passes to one heir (the row itself, else the first row
 * that forks from it); the others get a copy of its filled slots in a page of
 * their own, the lowest-numbered pages that were free before the call, rows in
 * order. Pages held beyond the length, and pages that no row holds any more,
 * become free. If the pool lacks pages, or a parent is outside [-1, S),
 * nothing changes (bit 16 of the device error word). workspace:
 * fxb_kv_fork_workspace bytes, 16-byte aligned. */
size_t fxb_kv_fork_workspace(int32_t S, int32_t W);
int fxb_kv_fork(const fxb_kv_args* args, const int32_t* parents, void* workspace, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FXB200_H */
