/* libymk — C-ABI of the token operators: root-mean-square norm with the residual's addition (and an 8-bit output), rows sorted by
 * expert and back, and the product of rows with their expert's matrix; each with its gradient.
 *
 * Conventions as in ymk.h: row-major views with a row stride in elements (ld >= C), activations YMK_F32 / YMK_H16 (and YMK_E4M3 where a
 * function says so), scales / gates / statistics fp32, `stream` a hipStream_t, return 0 or a negative YMK_E_* code, no allocation, no
 * synchronisation, no atomics on floating-point data: the same inputs give the same bits.  Every function may be captured into a graph;
 * a workspace belongs to the call (and, captured, to the graph) until the call has run.
 * Operands must lie on the current device; pointers and strides need the element type's alignment only (rows of any alignment take
 * 16-byte accesses) unless a function says more.  Zero rows: only what does not lie in rows is written (a sort's offsets; dweight, dW and
 * db: zeros).
 *
 * Gradients are calls of their own.
 *
 * A "pair" p = t * top_k + k is token t's k-th choice; a "row" is a place among the pairs sorted by expert. */
#ifndef YMK_TOKENS_H_
#define YMK_TOKENS_H_
#include "ymk.h"
#ifdef __cplusplus
extern "C" {
#endif

#define YMK_E4M3 2              /* OCP 8-bit float, 4 exponent and 3 mantissa bits: largest finite value 448, no infinities */
#define YMK_NORM_MAX_C 16384    /* widest row of the norms */
#define YMK_TOKEN_MAX_E 256     /* most experts */
#define YMK_TOKEN_MAX_K 16      /* most experts a token */

/* h = x + residual, rounded to dtype (residual == NULL: h is x itself and is not written); rstd = 1 / sqrt(mean(h^2) + eps);
 * y = h * rstd * weight, rounded once.  weight fp32 [C].  Statistics are those of the ROUNDED h, so that a gradient taken from the stored
 * h is the gradient of this very function; they are sums of squares in 32 bits (|h| < 1e18).
 * rstd fp32 [rows] or NULL.  h and y may alias x or residual (same stride).  C <= YMK_NORM_MAX_C. */
int ymk_rms_norm(int32_t dtype, const void* x, int32_t ldx, const void* residual, int32_t ldr, void* h, int32_t ldh, void* y, int32_t ldy,
                 float* rstd, int64_t rows, int32_t C, const float* weight, float eps, void* stream);

/* The same norm with an 8-bit output: scale[row] = max|y| / 448 and q = y / scale in e4m3 (round to nearest even), taken from the
 * unrounded y.  A row whose largest magnitude is below 448 * 2^-126 (an all-zero row, eps > 0) has scale 1 and zero codes; a row with a NaN or
 * an infinity has scale NaN and NaN codes.  ldq in bytes. */
int ymk_rms_norm_quant(int32_t dtype, const void* x, int32_t ldx, const void* residual, int32_t ldr, void* h, int32_t ldh, void* q,
                       int32_t ldq, float* scale, int64_t rows, int32_t C, const float* weight, float eps, void* stream);

/* Gradient: n = h * rstd, g = dy * weight, dx = rstd * (g - n * mean(g * n)) + dres (dres: the gradient that reaches h by its other
 * use, or NULL) — the gradient of x and of residual alike; dweight[c] = sum over rows of dy * n, fp32 (NULL: not wanted, no workspace).
 * dx may alias dy, h or dres. */
size_t ymk_rms_norm_backward_workspace_bytes(int64_t rows, int32_t C);
int ymk_rms_norm_backward(int32_t dtype, const void* dy, int32_t lddy, const void* h, int32_t ldh, const float* rstd, const float* weight,
                          const void* dres, int32_t lddr, void* dx, int32_t lddx, float* dweight, int64_t rows, int32_t C,
                          void* workspace, size_t workspace_bytes, void* stream);

/* Stable sort of the pairs by expert.  idx: dense [tokens][top_k], int32 or int64 (idx_bytes 4 | 8); a value outside [0, E) is a pair
 * without an expert.  offsets int32 [E + 1]: rows [offsets[e], offsets[e + 1]) are expert e's, offsets[0] = 0; src int32 [tokens * top_k]:
 * the pair of each row, ascending within an expert, -1 behind the last row; row int32 [tokens * top_k]: the row of each pair or -1.
 * E <= YMK_TOKEN_MAX_E, top_k <= YMK_TOKEN_MAX_K, tokens * top_k < 2^30. */
size_t ymk_token_sort_workspace_bytes(int64_t tokens, int32_t top_k, int32_t E);
int ymk_token_sort(const void* idx, int32_t idx_bytes, int64_t tokens, int32_t top_k, int32_t E, int32_t* offsets, int32_t* src,
                   int32_t* row, void* workspace, size_t workspace_bytes, void* stream);

/* xs[row[t][k]] = x[t], byte for byte (any element type): row_bytes of a row (at most 2^24), strides in bytes; with scale fp32 [tokens] (may be NULL)
 * also xs_scale[row[t][k]] = scale[t].  Rows behind the last one are left as they were.  Here and below a row outside [0, tokens * top_k) is
 * no row. */
int ymk_token_dispatch(const void* x, int64_t ldx_bytes, int64_t row_bytes, const float* scale, void* xs, int64_t ldxs_bytes,
                       float* xs_scale, const int32_t* row, int64_t tokens, int32_t top_k, void* stream);

/* y[t] = sum over k of w[t][k] * ys[row[t][k]] in fp32, in the order of k, rounded once; pairs without a row add nothing (a token that
 * has none gets zeros).  w fp32 [tokens][top_k], NULL = ones: that is the gradient of ymk_token_dispatch.  C <= 2^31 - 16, here and below. */
int ymk_token_combine(int32_t dtype, const void* ys, int32_t ldys, const int32_t* row, const float* w, void* y, int32_t ldy, int64_t tokens,
                      int32_t top_k, int32_t C, void* stream);

/* Gradient of ymk_token_combine: dys[row[t][k]] = w[t][k] * dy[t] and dw[t][k] = <dy[t], ys[row[t][k]]> (fp32; 0 without a row).  Rows of
 * dys behind the last one are left as they were. */
int ymk_token_combine_backward(int32_t dtype, const void* dy, int32_t lddy, const void* ys, int32_t ldys, const int32_t* row, const float* w,
                               void* dys, int32_t lddys, float* dw, int64_t tokens, int32_t top_k, int32_t C, void* stream);

/* The experts' product: for the rows r of expert e, i.e. offsets[e] <= r < offsets[e + 1],
 *     y[r] = act(x[r] W[e]^T + bias[e]),   W dense [E][Cout][Cin] of x's type, bias fp32 [E][Cout] or NULL, act YMK_ACT_*.
 * dtype YMK_F32 | YMK_H16, out_dtype the same; or YMK_E4M3 (x and W in 8 bits, W[e][o] standing for W * w_scale[e][o], x[r] for
 * x * x_scale[r], both scales fp32 and required) with out_dtype YMK_F32 | YMK_H16.  Products are added in 32 bits and the sum (scaled,
 * with bias and activation) is rounded once.  One exception: 8-bit products with a 16-bit output and 32 rows an expert or more, where the matrix
 * instruction adds 16 products at a time at the largest one's exponent, 13 bits deep, and those sums in 32 bits (1.5e-5 rms of the sum, under a
 * tenth of the output's rounding).  rows < 2^26.  offsets: device int32 [E + 1], ascending, within [0, rows] (values outside are clamped:
 * no access leaves the tensors); rows outside every expert are left as they were.  Cin and Cout in multiples of 16 bytes of their
 * elements (4 fp32, 8 16-bit, 16 8-bit; Cout of 8 for YMK_E4M3), all pointers and row strides 16-byte aligned, strides below 2^23 bytes. */
int ymk_expert_linear(int32_t dtype, int32_t out_dtype, const void* x, int32_t ldx, const float* x_scale, const void* w, const float* w_scale,
                      const float* bias, const int32_t* offsets, void* y, int32_t ldy, int64_t rows, int32_t E, int32_t Cin, int32_t Cout,
                      int32_t act, void* stream);
/* Gradient by x of the product without activation: dx[r] = dy[r] W[e].  YMK_F32 | YMK_H16. */
int ymk_expert_linear_dx(int32_t dtype, const void* dy, int32_t lddy, const void* w, const int32_t* offsets, void* dx, int32_t lddx, int64_t rows,
                         int32_t E, int32_t Cin, int32_t Cout, void* stream);
/* Gradients by W and bias: dw[e] = sum over e's rows of dy[r]^T x[r], dense [E][Cout][Cin] of dw_dtype (dtype or YMK_F32); db fp32
 * [E][Cout] = sum of dy[r], or NULL.  An expert without rows gets zeros. */
int ymk_expert_linear_dw(int32_t dtype, int32_t dw_dtype, const void* dy, int32_t lddy, const void* x, int32_t ldx, const int32_t* offsets,
                         void* dw, float* db, int64_t rows, int32_t E, int32_t Cin, int32_t Cout, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* YMK_TOKENS_H_ */
