/* Entry points of libmambaqc_hip.so beside the drop-in boundary of mambaqc_hip.h: products
 * and fused steps that the Python layers choose by size, each computing what operators of
 * mambaqc_hip.h or torch compute otherwise, and the operators of a recurrent stack (the gated
 * scan, the gate with norms and residual, the AdamW step). Conventions, status codes and dtype
 * codes are that header's. */
#ifndef MAMBAQC_HIP_EXT_H
#define MAMBAQC_HIP_EXT_H

#include "mambaqc_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* fp32 GEMM on the 16-bit matrix cores (each operand split into two fp16 pieces under a
 * power-of-two scale per row, three products per pair of pieces, fp32 accumulation):
 *   Y[m * ldy + n] = sum_k X[m * x_row + k * x_col] * W[n * w_row + k * w_col]
 * for m < M, n < N, k < K. One of x_row and x_col and one of w_row and w_col is 1 (and none
 * is negative), so X and W may be matrices or their transposes: F.linear and both of its
 * gradients (mambaqc/layers/quaternion_linear.py:145-161). Y may not overlap an operand.
 * Accuracy: each element is held to 2^-23 of itself, or to 2^-40 of its row's largest where that
 * is more; outputs that this last may put off by more than 2^-28 K of themselves (2^-20 below
 * K 256), all outputs of rows where more than an eighth of the elements are so small, and of
 * rows with an inf, are computed in plain fp32.
 * workspace: mqc_gemm_f32_workspace_bytes(M, N, K) bytes, 256-byte aligned (MQC_E_SPACE
 * if smaller). */
int64_t mqc_gemm_f32_workspace_bytes(int64_t M, int64_t N, int64_t K);
int mqc_gemm_f32(const float* X, int64_t x_row, int64_t x_col, const float* W, int64_t w_row,
                 int64_t w_col, float* Y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                 void* workspace, int64_t workspace_bytes, void* stream);

/* Up to four small fp32 products in one launch, Y[m * N + n] = sum_k X[m * xm + k * xk] *
 * W[n * wn + k * wk] (+ bias[n]). products: count rows of eleven values, X, xm, xk, W, wn, wk,
 * bias (or 0), Y, M, N, K (pointers as integers; one of xm, xk and one of wn, wk is 1). */
int mqc_gemm_f32_small(const int64_t* products, int64_t count, void* stream);

/* mqc_qln_bwd with its parameter sums: dq, and dgamma [d] and dbeta [d, 4] in fp32. rows and d at
 * least 1, d at most 4096; workspace of mqc_qln_bwd_sums_workspace_bytes(rows, d). */
int64_t mqc_qln_bwd_sums_workspace_bytes(int64_t rows, int64_t d);
int mqc_qln_bwd_sums(const void* q, const void* dout, const float* gamma, const float* mean,
                     const float* rstd, void* dq, float* dgamma, float* dbeta, int64_t rows,
                     int64_t d, float eps, int dtype, void* workspace, int64_t workspace_bytes,
                     void* stream);

/* out_i[c] = sum over r < rows of in_i[r * n_i + c] for up to three fp32 arrays (n_i 0: none),
 * in a fixed order, in one launch. */
int mqc_sum_rows(const float* in1, float* out1, int64_t n1, const float* in2, float* out2,
                 int64_t n2, const float* in3, float* out3, int64_t n3, int64_t rows,
                 void* stream);

/* mqc_cumprod_scan_fwd and mqc_ssm_q_fwd (from a zero state, without h_last) with the sequence
 * in chunks of chunk_len steps walked side by side, for few lanes (batch x lanes, lanes =
 * d_model x d_state for the SSM). chunk_len < seq_len; workspace (16-byte aligned) of
 * mqc_q_chunked_workspace_bytes (ssm 1 for the SSM); batch x chunks at most 65535. */
int64_t mqc_q_chunked_workspace_bytes(int64_t batch, int64_t seq_len, int64_t lanes,
                                      int64_t chunk_len, int ssm);
int mqc_cumprod_scan_chunked(const void* q, void* out, int64_t batch, int64_t seq_len,
                             int64_t lanes, int64_t chunk_len, int dtype, void* workspace,
                             int64_t workspace_bytes, void* stream);
int mqc_ssm_q_fwd_chunked(const void* q, const void* B, const void* Sq, const void* C,
                          const void* D, int64_t d_stride_b, int64_t d_stride_t,
                          int64_t d_stride_d, void* y, int64_t batch, int64_t seq_len,
                          int64_t d_model, int64_t d_state, int64_t chunk_len, int dtype,
                          void* workspace, int64_t workspace_bytes, void* stream);

/* mqc_ssm_fused_bc_fwd for short sequences, seq_len from 1 to 128 (MQC_E_LIMIT above): same
 * operands, dtypes, shapes and refusals, in tiles of 64 or 128 tokens that hold whole
 * sequences of the batch, each group of 16 states in a workgroup of its own. d_state > 16
 * needs workspace (mqc_ssm_fused_bc_short_workspace_bytes, 16-byte aligned) for the groups'
 * partial sums of y. h_last may be h0. */
int64_t mqc_ssm_fused_bc_short_workspace_bytes(int64_t batch, int64_t seq_len, int64_t d_inner,
                                               int64_t d_state);
int mqc_ssm_fused_bc_short_fwd(const void* x, const void* B_weight, const void* C_weight,
                               const void* delta, const void* s, const float* lambda_alpha,
                               const float* lambda_imag, const float* D, const void* h0, void* y,
                               void* h_last, int64_t batch, int64_t seq_len, int64_t d_inner,
                               int64_t d_state, float eps, int dtype, void* workspace,
                               int64_t workspace_bytes, void* stream);

/* One recurrent decode step of the block in four launches (bf16 or fp16; M = batch, 1 to 16
 * rows, K and 4 d_inner multiples of 32, X within the skinny GEMM's 64 KiB of LDS, else
 * MQC_E_LIMIT). Each rounds to dtype where the separate launches store.
 *
 * mqc_step_in_proj_conv: X [M, K] times W [>= channels + z_cols, K] (+ bias); the first
 * `channels` columns are one step of mqc_causal_conv_silu_step (continued from and shifting
 * tail [M, conv_k - 1, channels]) into act [M, channels], the next z_cols go to z [M, z_cols].
 * channels a multiple of 8, conv_k at most 4.
 * mqc_gemm_skinny4_nt: mqc_gemm_skinny_nt for four weights sharing X.
 * mqc_step_ssm: delta = softplus(dt_raw), s = sigmoid(g_raw) x, then one step of
 * mqc_ssm_fused_fwd in place on h (fp32 [batch, d_inner, d_state, 4]); d_state <= 64.
 * mqc_step_norm_out_gate: mqc_qln_fwd of Y [M, d_inner, 4], times W [d_model, 4 d_inner]
 * (+ bias), out = x + sigmoid(z) * that (x, out [M, d_model]; z rows z_row_stride apart). */
int mqc_step_in_proj_conv(const void* X, int64_t M, int64_t K, const void* W, const void* bias,
                          int64_t channels, int64_t z_cols, const float* conv_w,
                          const float* conv_b, int64_t conv_k, void* tail, void* act, void* z,
                          int dtype, void* stream);
int mqc_gemm_skinny4_nt(const void* X, int64_t M, int64_t K, const void* W1, const void* bias1,
                        void* Y1, int64_t N1, const void* W2, const void* bias2, void* Y2,
                        int64_t N2, const void* W3, const void* bias3, void* Y3, int64_t N3,
                        const void* W4, const void* bias4, void* Y4, int64_t N4, int dtype,
                        void* stream);
int mqc_step_ssm(const void* dt_raw, const void* g_raw, const void* x, const void* B,
                 const void* C, const float* lambda_alpha, const float* lambda_imag,
                 const float* D, float* h, void* y, int64_t batch, int64_t d_inner,
                 int64_t d_state, float eps, int dtype, void* stream);
int mqc_step_norm_out_gate(const void* Y, int64_t M, int64_t d_inner, const float* gamma,
                           const float* beta, float eps, const void* W, const void* bias,
                           int64_t d_model, const void* x, const void* z, int64_t z_row_stride,
                           void* out, int dtype, void* stream);
/* 1 where mqc_step_norm_out_gate takes M rows of d_inner quaternions, else 0. */
int mqc_step_norm_out_gate_fits(int64_t M, int64_t d_inner);

/* The gated scan over [batch, seq_len, width]: D = softplus(dt), a = exp(-D exp(log_rate)),
 *   h_t = a_t h_{t-1} + (1 - a_t) sigmoid(g_t) x_t,  y_t = h_t
 * from h0 (fp32 [batch, width]; NULL: zeros). reset (bytes [batch, seq_len], or NULL): where it is
 * not 0, h_{t-1} is taken as 0. Tokens of dt, g and x are *_row elements apart (all batch x seq_len
 * of them), y is dense. h_last (fp32, or NULL) may be h0. carries (fp32 [batch,
 * ceil(seq_len / mqc_gated_scan_chunk()), width], or NULL): the states that the backward starts
 * from, each chunk's before its first token.
 * workspace (16-byte aligned) of mqc_gated_scan_workspace_bytes. MQC_E_LIMIT for width or seq_len
 * above 2^31, batch above 65535, and walks of 2^32 threads (64 for each 64 channels and 16 steps of a
 * sequence). Chunks wait for one another within the launch, each for at most about a second; one that
 * waited in vain gives NaN for what follows it.
 *
 * Backward: gradients of dt, g, x (dense), log_rate [width], and of h0 (or NULL) from dy and
 * dh_last (or NULL); every size at least 1.
 * The step: one token of each sequence, h (fp32 [batch, width]) updated in place. */
int mqc_gated_scan_chunk(void);
int64_t mqc_gated_scan_workspace_bytes(int64_t batch, int64_t seq_len, int64_t width);
int mqc_gated_scan_fwd(const void* dt, int64_t dt_row, const void* g, int64_t g_row, const void* x,
                       int64_t x_row, const float* log_rate, const float* h0, const void* reset,
                       void* y, float* h_last, float* carries, int64_t batch, int64_t seq_len,
                       int64_t width, int dtype, void* workspace, int64_t workspace_bytes,
                       void* stream);
int mqc_gated_scan_bwd(const void* dt, int64_t dt_row, const void* g, int64_t g_row, const void* x,
                       int64_t x_row, const float* log_rate, const void* reset,
                       const float* carries, const void* dy, const float* dh_last, void* ddt,
                       void* dg, void* dx, float* dlog_rate, float* dh0, int64_t batch,
                       int64_t seq_len, int64_t width, int dtype, void* workspace,
                       int64_t workspace_bytes, void* stream);
int mqc_gated_scan_step(const void* dt, int64_t dt_row, const void* g, int64_t g_row, const void* x,
                        int64_t x_row, const float* log_rate, float* h, void* y, int64_t batch,
                        int64_t width, int dtype, void* stream);

/* Between two blocks, for each of `rows` rows of d (1 to mqc_gate_norm_max_width()) elements:
 *   v = sigmoid(z) y,  r = v / sqrt(mean v^2 + eps) post,  out = x + scale r,
 *   n = out / sqrt(mean out^2 + eps) pre
 * x, y, out and n dense, rows of z z_row elements apart; z NULL: v = y; post NULL: r = v. post, scale
 * and pre are [d]. stats (fp32 [rows, 2], or NULL) takes the two inverse norms for the backward. out
 * may be x or y, n may be y. MQC_E_LIMIT for a forward of 2^32 threads: 2^28, 2^27 or 2^26 rows of d up
 * to 64, 128 or 1024, 2^26 / ceil(d / 1024) wider ones.
 * Backward, from dout and dn (dense; either may be NULL, zeros): dx, dy and dz dense, dpost (with
 * post), dscale and dpre [d] summed over the rows in a fixed order; rows at least 1, workspace of
 * mqc_gate_norm_workspace_bytes. */
int64_t mqc_gate_norm_max_width(void);
int64_t mqc_gate_norm_workspace_bytes(int64_t rows, int64_t d);
int mqc_gate_norm_fwd(const void* x, const void* y, const void* z, int64_t z_row, const float* post,
                      const float* scale, const float* pre, void* out, void* n, float* stats,
                      int64_t rows, int64_t d, float eps, int dtype, void* stream);
int mqc_gate_norm_bwd(const void* x, const void* y, const void* z, int64_t z_row, const float* post,
                      const float* scale, const float* pre, const float* stats, const void* dout,
                      const void* dn, void* dx, void* dy, void* dz, float* dpost, float* dscale,
                      float* dpre, int64_t rows, int64_t d, int dtype, void* workspace,
                      int64_t workspace_bytes, void* stream);

/* One AdamW step over `count` tensors, each element in fp32:
 *   g = grad * (*clip);  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   p = p decay - m / (sqrt(v) root_scale + eps) step_size
 * (decay = 1 - lr weight_decay, step_size = lr / (1 - beta1^t), root_scale = 1 / sqrt(1 - beta2^t);
 * clip, a device float, may be NULL). Elements of p and grad are of the row's dtype.
 * mqc_adamw_step: rows of six values: p, grad, m, v, element count, dtype (pointers as integers);
 * m and v fp32.
 * mqc_adamw8_step: rows of nine: p, grad, m, r, m_scale, r_scale, element count, dtype, seed; m and
 * r = sqrt(v) e4m3 bytes, with a power-of-two scale (fp32) for each 256 elements. Rounded up or down
 * by seed, place and `step`, such that m's and v's means are kept.
 * Pointers are aligned to their elements; the rows are read before the call returns.
 *
 * mqc_grad_norm: rows of three values: grad, element count, dtype. *norm = the 2-norm of all their
 * elements (summed in 64 bits, in a fixed order), *clip = min(1, max_norm / (norm + 1e-6)); workspace
 * (8-byte aligned) of mqc_grad_norm_workspace_bytes. */
int mqc_adamw_step(const int64_t* tensors, int64_t count, float decay, float step_size,
                   float root_scale, float beta1, float one_minus_beta1, float beta2,
                   float one_minus_beta2, float eps, const float* clip, void* stream);
int mqc_adamw8_step(const int64_t* tensors, int64_t count, float decay, float step_size,
                    float root_scale, float beta1, float one_minus_beta1, float beta2,
                    float one_minus_beta2, float eps, const float* clip, uint32_t step,
                    void* stream);
int64_t mqc_grad_norm_workspace_bytes(const int64_t* tensors, int64_t count);
int mqc_grad_norm(const int64_t* tensors, int64_t count, double max_norm, float* norm, float* clip,
                  void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MAMBAQC_HIP_EXT_H */
