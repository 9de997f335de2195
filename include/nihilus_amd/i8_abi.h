/*
 * i8_abi.h -- C ABI of products in 8-bit integers with one scale per row of either operand (per token and per output channel) on an MI355X (gfx950),
 * and of the softmax cross entropy over a vocabulary on such an output projection, with its gradient.
 *
 * The conventions of attention_abi.h hold here: plain C, device pointers unless a name starts with host_, `stream` a hipStream_t, 0 / negative nh_status / positive
 * hipError_t as the result, no exception; calls are asynchronous on their stream, allocate nothing and keep nothing.  What a call needs for itself is in its workspace, whose
 * contents mean nothing before and after.  Calls with workspaces and results of their own are independent, on any streams and in captured graphs.
 *
 * Beside the Q8_0 calls of q8_0_abi.h, whose operands have a scale for each 32 values: there every block's sum is scaled by itself, which holds a prompt's
 * products to a fifth of the matrix rate; here a sum over all of K is scaled once.  A projection in the reference is mul_mat (kernel_types::mul_mat, cpu/avx_2.hpp:1296-1444), the
 * rows of its output projection go on to sampling (infra/core_traits.hpp:1186-1193).
 *
 * A tiled matrix [rows][k], of activations and of weights alike:
 *   int8   strips of 16 rows, ceil(rows / 16) of them; in each ceil(k / 64) fragments of 1024 bytes, byte 256 c + 16 r + j of which is value 64 step + 16 c + j of the
 *          strip's row r.  Values past k are zero.
 *   fp32   a scale for each row, strips * 16 of them, behind the last fragment.
 *   Value q of row r stands for q * scale[r].  (Rows past the last one may hold anything.)
 * Quantizing a row of fp32 values v:  scale = fp32(max |v| / 127),  q = the whole number nearest to v / scale (the true quotient), ties to even, within +-127.  A row of
 * zeros has scale 0 and q = 0.  A row that has an infinity or NaN has scale NaN and q = 0: what is formed from it is NaN.
 *
 * What a call writes (results, workspace) has no byte in common with what it reads or with anything else that it writes, but for a result that is the residual itself (NH_ERR_ARGUMENT).
 * Limits (NH_ERR_TOO_LARGE): rows up to 2^22, K up to 131008 (a sum of K products stays below 2^31), a matrix up to 32 GiB, ceil(M / 256) ceil(N / 256) up to 2^22.  Pointers are 16-byte aligned, or where noted only as their type.
 */
#ifndef NIHILUS_AMD_I8_ABI_H
#define NIHILUS_AMD_I8_ABI_H

#include "attention_abi.h" /* NH_F32, NH_F16, NH_BF16 */

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of a tiled matrix; negative: an nh_status. */
int64_t nh_i8_tiled_bytes(int64_t rows, int64_t k);

/* x [rows][k] of `type` (NH_F32, NH_F16, NH_BF16), x_stride elements from one row to the next, aligned as its type (faster where rows begin at multiples of 16 bytes). */
int nh_i8_quantize(const void* x, int type, int64_t x_stride, void* x_tiled, int64_t rows, int64_t k, void* stream);
/* The same of fp32((x * r) * norm_weight), r = fp32(1 / sqrt(mean of the row's x^2 + eps)), the mean in 64 bits; norm_weight fp32 [k]. */
int nh_i8_rms_norm_quantize(const void* x, int type, int64_t x_stride, const float* norm_weight, float eps, void* x_tiled, int64_t rows, int64_t k, void* stream);
/* The same of silu(gate) * up, silu(g) = g / (1 + exp(-g)), in fp32 (within 3 units of 2^-23 of itself, or of 2^-149; 0 for finite gates below -132). */
int nh_i8_silu_mul_quantize(const void* gate, const void* up, int type, int64_t gate_stride, int64_t up_stride, void* x_tiled, int64_t rows, int64_t k, void* stream);
/* A plain int8 matrix [rows][k] with scales fp32 [rows] into the tiled layout, and back. */
int nh_i8_tile(const int8_t* q, const float* scales, void* tiled, int64_t rows, int64_t k, void* stream);
int nh_i8_untile(const void* tiled, int8_t* q, float* scales, int64_t rows, int64_t k, void* stream);

/* y [M][N] of `type` = x . w^T + residual (NULL: none; [M][N] of the same type, may be y itself): the whole-number sum over K brought to fp32, times x's scale, times w's, plus the residual, rounded
 * once. */
int nh_i8_gemm(const void* w_tiled, const void* x_tiled, const void* residual, void* y, int type, int64_t M, int64_t N, int64_t K, void* stream);
/* quantize (norm_weight not NULL: rms_norm_quantize) and gemm; x and y of the same type.  workspace: nh_i8_mul_mat_workspace_bytes(M, K) bytes; one row of up to
 * 16384 values is quantized inside the product's launch and needs none (0, and the pointer may be NULL). */
int64_t nh_i8_mul_mat_workspace_bytes(int64_t M, int64_t K);
int nh_i8_mul_mat(const void* w_tiled, const void* x, int type, int64_t x_stride, const float* norm_weight, float eps, const void* residual, void* y, int64_t M, int64_t N, int64_t K,
	void* workspace, int64_t workspace_bytes, void* stream);

/* Softmax cross entropy of rows x [M][K] on an output projection w [N][K]:  l[m][n] = the product above in fp32,
 *   lse[m] = log sum_n exp l[m][n],   losses[m] = lse[m] - l[m][targets[m]],  0 where targets[m] (int32) is outside [0, N): such a row is not scored.
 * A loss is formed from the largest logit, not from the rounded lse, so that a small one keeps its digits however large the logits are.  These are formed a tile at a time and not kept. */
int64_t nh_i8_token_losses_workspace_bytes(int64_t M, int64_t N, int64_t K); /* up to about 64 MiB, whatever M is, unless N is far past a million */
int nh_i8_token_losses(const void* w_tiled, const void* x_tiled, const int32_t* targets, float* losses, float* lse, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream);

/* The gradient of sum_m grad[m] losses[m] (grad fp32 [M]; NULL: ones) with respect to what the rows of x stand for:
 *   dx[m][k] = grad[m] sum_n (exp(l[m][n] - lse[m]) - [n = targets[m]]) w[n][k],  zero for rows that are not scored;  dx [M][K] of `type`, rounded once.
 * losses and lse as nh_i8_token_losses gave them: the target's own slope is formed as exp(-losses[m]) - 1, the others are as exact as lse is (2^-24 |lse| relative to themselves).
 * The slopes are formed again from x and w, for 8192 rows at a time and so much of the vocabulary that they stay below 128 MiB, and enter the second product, times w's scales, as sums of two fp16
 * numbers (22 bits) below a power of two of the row's own: what is 2^-37 of the row's largest slope and of w's largest scale is lost. */
int64_t nh_i8_token_losses_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int type);
int nh_i8_token_losses_grad(const void* w_tiled, const void* x_tiled, const int32_t* targets, const float* losses, const float* lse, const float* grad, void* dx, int type, int64_t M, int64_t N,
	int64_t K, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif
