/*
 * Operators for encoders that are trained on this library's neighbour
 * probabilities (or on another network's logits) and then place points that no
 * fit has seen: matrices in 8-bit floating point with a scale for each block
 * of 128 values and their products, a teacher's top list, and distillation
 * from such a list with its gradient.  The reference has none of them: it maps
 * the points it is given and no others.
 *
 * Conventions as in tsne_stages.h: device pointers, 0 for success and
 * tsne_hip_last_error() otherwise, everything asynchronous on `stream`.  No
 * call allocates, synchronises or keeps anything; where one needs a workspace,
 * the caller gives it (at least as many bytes as the function next to it says,
 * aligned to 16) and may use it for something else on the same stream right
 * after.  Results do not depend on the order in which workgroups run.
 *
 * `type` is the type of a matrix's values: 0 = 32-bit float, 1 = 16-bit float
 * (half), 2 = bfloat16.  Matrices are row-major, `..._stride` values from one
 * row to the next (at least the row's length), and may begin at any multiple
 * of their type's size.
 */
#ifndef TSNECUDA_TSNE_OPERATORS_H_
#define TSNECUDA_TSNE_OPERATORS_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Block-scaled 8-bit matrices.  A matrix of `rows` x `cols` is held as
 *   data    rows x 128 * ceil(cols / 128) bytes, e4m3 (448 the largest, no infinities), zeros behind a row's end,
 *   scales  rows x 4 * ceil(cols / 512) bytes, one for each 128 columns of a row: 2^(byte - 127), 255 = NaN,
 * both contiguous and aligned to 16 bytes; a value is data * scale.  Powers of two, because the matrix cores
 * multiply by them at no cost and because a value's nearest neighbour among the 8-bit ones is then decided without
 * a rounded division before it.
 *
 * tsne_hip_quantize_blocks: the scale of a block is the least power of two (2^-127 at least) with which its
 * largest finite magnitude is at most 448, 1 for a block of zeros; values are rounded to the nearest, ties to even.
 * A NaN or an infinity becomes NaN and has no say in the scale.  square = 0: a block is 128 consecutive values of
 * a row; square = 1: 128 x 128 values, so that the matrix and its transpose have the same scales (weights).
 * data / scales receive the matrix, data_t / scales_t its transpose (with blocks along ITS rows, i.e. down the
 * columns of x); either pair may be NULL.  x is read once for both. */
int tsne_hip_quantize_blocks(const void *x, int type, int64_t rows, int64_t cols, int64_t row_stride, int square,
                             uint8_t *data, uint8_t *scales, uint8_t *data_t, uint8_t *scales_t, void *stream);

/* c (m x n) = a (m x k) times the transpose of b (n x k), both block-scaled; k is the number of columns before
 * padding (what is behind it has to be zeros, as tsne_hip_quantize_blocks leaves it).  k <= 2^24.  Sums are in 32 bits.  A result
 * in bfloat16 (type 2) is formed by the 8-bit matrix instructions, which add products in groups of eight and drop what
 * lies more than 2^-13 below a group's largest (for normally distributed factors 1.5e-5 of a result, a hundredth of
 * its rounding; at most 7 * 2^-13 of the sum of the groups' largest, which where those cancel is more than the result's
 * rounding); one in halves or floats, and with exact = 1 any, by the bf16 instructions, which hold every product exactly,
 * at half the rate. */
int tsne_hip_matmul_blocks(const uint8_t *a, const uint8_t *a_scales, const uint8_t *b, const uint8_t *b_scales,
                           int64_t m, int64_t n, int64_t k, void *c, int type, int64_t c_stride, int exact,
                           void *workspace, int64_t workspace_bytes, void *stream);
int64_t tsne_hip_matmul_blocks_workspace(int64_t m, int64_t n, int64_t k, int type, int exact);

/* c (m x n) = quantised x (m x k) times the transpose of w (n x k, block-scaled): tsne_hip_quantize_blocks
 * (square = 0) and tsne_hip_matmul_blocks (exact = 0; with exact = 1 call the two) in one call, with the same bits.  x and
 * c have the same type. */
int tsne_hip_linear_blocks(const void *x, int type, int64_t m, int64_t k, int64_t x_stride, const uint8_t *w,
                           const uint8_t *w_scales, int64_t n, void *c, int64_t c_stride, void *workspace,
                           int64_t workspace_bytes, void *stream);
int64_t tsne_hip_linear_blocks_workspace(int64_t m, int64_t n, int64_t k, int type);

/* For every row of logits its k largest (values, descending; equal ones by ascending column) and their columns,
 * and lse = ln sum exp(z / temperature) over the whole row, all in 32 bits.  A column that is -infinity is never
 * listed: where a row has fewer than k others, the rest of its list is (-infinity, -1).  NaN counts as the largest;
 * it and +infinity make the row's lse NaN.  A row of -infinity has lse = -infinity.  1 <= k <= min(cols, 1024), cols < 2^31, temperature from 2^-126 on. */
int tsne_hip_top_logits(const void *logits, int type, int64_t rows, int64_t cols, int64_t row_stride, int k,
                        float temperature, float *values, int *indices, float *lse, void *workspace,
                        int64_t workspace_bytes, void *stream);
int64_t tsne_hip_top_logits_workspace(int64_t rows, int64_t cols, int type, int k);

/* Distillation: the divergence of a row's softmax q = softmax(z / temperature) from a teacher's list.
 * Teacher: p_j = exp(values_j / temperature - l) at column indices_j, j < k, where l is lse[row], or, with
 * lse = NULL, such that the list's p sum to 1.  Entries whose index is outside [0, cols) do not exist; a column may
 * be listed more than once (its p add up).
 *   loss[row] = w (sum_j p_j (ln p_j - ln q_j) + p_r (ln p_r - ln q_r)),   w = weights[row] (1 with weights = NULL).
 * The last term only with rest = 1 (needs lse): what the list leaves out, p_r = max(0, 1 - sum p), against q_r, the sum
 * of q over the columns that are not listed, as one event; it is left out where every column outside the list is
 * -infinity.  A listed column with p_j = 0 adds nothing.  w = 0: loss and gradient are exactly 0 and the row's
 * logits are not looked at.
 * grad (type of the logits, may be NULL, may be the logits themselves, but may not overlap them otherwise) receives the
 * derivative of loss[row] by z.
 * A column that is -infinity has q = 0 and, unless it is listed, gradient 0: with p_j > 0 on it the loss is
 * +infinity and its gradient -w p_j / temperature.  NaN and +infinity in a row make its loss and gradient NaN.
 * 1 <= k <= 1024, cols <= 2^20, temperature from 2^-126 on.  With perplexity's probabilities as the teacher: values = ln pij,
 * lse = NULL, temperature = 1. */
int tsne_hip_distill(const void *logits, int type, int64_t rows, int64_t cols, int64_t row_stride, const int *indices,
                     const float *values, int k, const float *lse, const float *weights, float temperature, int rest,
                     float *loss, void *grad, int64_t grad_stride, void *workspace, int64_t workspace_bytes,
                     void *stream);
int64_t tsne_hip_distill_workspace(int64_t rows, int64_t cols, int type, int k);

#ifdef __cplusplus
}
#endif

#endif /* TSNECUDA_TSNE_OPERATORS_H_ */
