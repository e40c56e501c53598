/*
 * pcu_b200_learn.h -- learning operators beside the strict path: group norm with an activation,
 * distillation from a teacher's top logits, and the product of 8-bit operands with a scale for
 * each block of 128.  The reference has no counterpart of any of them (its tensor nodes are
 * Crates/core/dialect/tensor.rs:3925-4345).
 *
 * The contract of pcu_b200.h holds: device pointers owned by the caller, one status word per call,
 * asynchronous calls on `stream` on the current device, outputs written even when a fault is
 * recorded, host-side errors as the return value, and a guarded form of every call for stages of a
 * guarded chain.  What differs:
 *   - Results are not defined bit by bit: sums run in another order than the index order, products
 *     and sums are contracted, and exponentials are approximations.  The same call on the same
 *     inputs gives the same bits.
 *   - F16 and BF16 tensors are taken beside F32 and F64.  The arithmetic on F16, BF16 and F32 is in
 *     binary32 ("wide" below: F32 for these three, F64 for F64) and rounds once, to nearest even,
 *     where a result is stored.
 *   - There is no underflow policy: results underflow gradually.  Factors that are 0 below 2^-126: softmax
 *     terms, SiLU's 1 / (1 + exp(-z)) and the normal density in GELU's slope, so that SiLU and its slope
 *     are 0 from z = -87.3 on, where they are -1.1e-36.  (In F64 that quotient is 0 below 2^-1024.)
 *   - Faults: a result that is not finite is recorded as InvalidFloatingOperand when it is NaN and
 *     as ArithmeticOverflow when it is an infinity; the events are given with each call.
 *   - Buffers must not overlap except where a call says so, and are aligned to their elements
 *     (PCU_B200_ERROR_INVALID_ARGUMENT otherwise).
 */
#ifndef PCU_B200_LEARN_H
#define PCU_B200_LEARN_H

#include "pcu_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of the learning operators beside PCU_B200_F32 and PCU_B200_F64 */
#define PCU_B200_F16 2
#define PCU_B200_BF16 3

/* ------------------------------------------------------------------ group norm */

#define PCU_B200_ACTIVATION_NONE 0
#define PCU_B200_ACTIVATION_RELU 1 /* z for z > 0, else 0 */
#define PCU_B200_ACTIVATION_SILU 2 /* z / (1 + exp(-z)) */
#define PCU_B200_ACTIVATION_GELU 3 /* z Phi(z), Phi the normal distribution function */

/* Group norm with an activation, channels last.  input is batch x positions x channels, element
 * (n, s, c) at n * input_batch_stride + s * input_stride + c; channel c is in group c / (channels /
 * groups).  Over the positions x (channels / groups) elements of each (n, group):
 *   mean, variance = mean of (x - mean)^2, r = 1 / sqrt(variance + eps),
 *   out = activation((x - mean) * r * weight[c] + bias[c]).
 * weight and bias are wide, `channels` elements, or NULL (1 and 0).  eps is a finite binary32
 * pattern, not negative.  stats receives (mean, r) for each (n, group), wide, 2 * batch * groups.
 * ReLU's slope at z = 0 is 0.  channels must be a multiple of groups; batch and
 * positions may be 0.  out has its own strides and may be input itself (same strides).
 * The variance is not the mean of x^2 less the square of the mean: its squares are taken about the mean, or,
 * where rows are read once, about the mean of the rows before, a block of rows at a time.
 * Events: the element's index (n * positions + s) * channels + c in out.  A group that holds a NaN
 * or an infinity gives NaN throughout.
 * Device workspace: pcu_b200_group_norm_workspace_size bytes (may be 0). */
size_t pcu_b200_group_norm_workspace_size(int dtype, uint64_t batch, uint64_t positions, uint64_t channels,
                                          uint64_t groups);
int pcu_b200_group_norm(int dtype, int activation, const void *input, const void *weight, const void *bias, void *out,
                        void *stats, uint64_t batch, uint64_t positions, uint64_t channels, uint64_t groups,
                        uint64_t input_batch_stride, uint64_t input_stride, uint64_t out_batch_stride,
                        uint64_t out_stride, uint32_t eps_bits_f32, void *workspace, size_t workspace_bytes,
                        uint64_t *status, void *stream);

/* The gradients of pcu_b200_group_norm for the gradient `upstream` of its output: gradient (laid
 * out by its own strides; it may be input or upstream itself, with the same strides), and the wide
 * weight_gradient and bias_gradient (channels each; NULL when not wanted).  stats is what the
 * forward call wrote.  With batch or positions 0 the parameters' gradients are zeros.
 * Whether z is above 0, for ReLU, is decided in binary64 for the given stats, weight and bias; where it is
 * not, upstream does not count, whatever it is.
 * Events: the element's index in gradient, then batch * positions * channels + c for
 * weight_gradient[c], then channels more + c for bias_gradient[c]. */
size_t pcu_b200_group_norm_backward_workspace_size(int dtype, uint64_t batch, uint64_t positions, uint64_t channels,
                                                   uint64_t groups);
int pcu_b200_group_norm_backward(int dtype, int activation, const void *input, const void *upstream,
                                 const void *weight, const void *bias, const void *stats, void *gradient,
                                 void *weight_gradient, void *bias_gradient, uint64_t batch, uint64_t positions,
                                 uint64_t channels, uint64_t groups, uint64_t input_batch_stride,
                                 uint64_t input_stride, uint64_t upstream_batch_stride, uint64_t upstream_stride,
                                 uint64_t gradient_batch_stride, uint64_t gradient_stride, void *workspace,
                                 size_t workspace_bytes, uint64_t *status, void *stream);

/* ------------------------------------------------------------------ distillation */

/* Most teacher entries a row can have. */
#define PCU_B200_DISTILL_TOP_MAX 1024

/* The loss of a student's logits against a teacher's top logits.  Row i holds the student's logits
 * z (vocab elements at i * logits_stride) and top_count teacher entries: top_indices and the wide
 * top_logits, both rows x top_count.  T is the temperature, a positive normal binary32 pattern.
 *   q = softmax(z / T) over the vocabulary, p = softmax(top / T) over the row's present entries,
 *   loss[i] = w_i * T^2 * sum_j p_j (ln p_j - ln q[index_j]),  w_i = row_weights[i] (wide; NULL: 1).
 * row_stats[2i], [2i + 1] receive m = max z and sum of exp((z - m) / T).  loss and row_stats are wide.
 *   - A negative index, or a teacher logit of -infinity, is an absent entry.  The same index may
 *     appear several times; each entry counts.
 *   - A student logit of -infinity is a masked vocabulary entry: q = 0 there.
 *   - A row with weight 0, or without a present entry, has nothing to learn from, whatever its logits
 *     are: loss 0, statistics (0, 1), gradient 0, no fault.
 * Events: the row.  InvalidFloatingOperand: a NaN or +infinity among the logits, no finite logit, a
 * present teacher entry that is NaN, +infinity or names an index >= vocab, or a weight or upstream
 * that is not finite; the row's loss and gradient are then NaN.  ArithmeticOverflow: the loss is
 * infinite (the teacher expects a masked vocabulary entry) or a gradient exceeds its type. */
int pcu_b200_distill_loss(int dtype, const void *logits, uint64_t rows, uint64_t vocab, uint64_t logits_stride,
                          const int64_t *top_indices, const void *top_logits, uint64_t top_count,
                          const void *row_weights, uint32_t temperature_bits_f32, void *loss, void *row_stats,
                          uint64_t *status, void *stream);

/* The gradient with respect to the logits, from the row_stats of the forward call:
 *   gradient[i][v] = u_i * w_i * T * (q_v - sum of p_j over index_j = v)
 * u = upstream: a wide element per row, one element when upstream_uniform, 1 when NULL.  gradient has
 * rows of gradient_stride elements and may be logits itself (same stride). */
int pcu_b200_distill_loss_backward(int dtype, const void *logits, uint64_t rows, uint64_t vocab,
                                   uint64_t logits_stride, const int64_t *top_indices, const void *top_logits,
                                   uint64_t top_count, const void *row_weights, uint32_t temperature_bits_f32,
                                   const void *row_stats, const void *upstream, int upstream_uniform, void *gradient,
                                   uint64_t gradient_stride, uint64_t *status, void *stream);

/* Loss and gradient in one call, when upstream does not depend on the loss (a mean over the rows):
 * the logits come from memory once.  row_stats may be NULL. */
int pcu_b200_distill_loss_step(int dtype, const void *logits, uint64_t rows, uint64_t vocab, uint64_t logits_stride,
                               const int64_t *top_indices, const void *top_logits, uint64_t top_count,
                               const void *row_weights, uint32_t temperature_bits_f32, void *loss, void *row_stats,
                               const void *upstream, int upstream_uniform, void *gradient, uint64_t gradient_stride,
                               uint64_t *status, void *stream);

/* ------------------------------------------------------------------ 8-bit block product */

/* Codes with 4 exponent and 3 fraction bits (e4m3: largest 448, NaN 0x7f, no infinity) and one scale
 * for each block of block_rows (1 or 128) rows x 128 columns of `input` (F32, F16 or BF16; rows of
 * input_stride elements).  A block's scale is the smallest power of two, at least 2^-126, that
 * brings its largest finite magnitude to 448 or below, 1 for a block of zeros; codes round
 * input / scale, which is exact, to nearest even.  codes has rows of codes_stride bytes (a multiple of 16 lets
 * pcu_b200_block_matmul use the tensor cores; the bytes behind a row are left alone), scales is
 * binary32, ceil(rows / block_rows) x ceil(columns / 128).
 * Events: the element's index row * columns + column; InvalidFloatingOperand for an element that is
 * not finite, whose code is NaN. */
int pcu_b200_block_quantize(int dtype, const void *input, uint64_t rows, uint64_t columns, uint64_t input_stride,
                            int block_rows, void *codes, uint64_t codes_stride, float *scales, uint64_t *status,
                            void *stream);

/* out[r][c] = sum over blocks b of 128 of left_scales[r][b] * right_scales[c / 128][b] *
 *             (sum over k in block b of left[r][k] * right[c][k]),
 * left: rows x inner codes with scales of 1 x 128 blocks (activations); right: columns x inner codes
 * with scales of 128 x 128 blocks (a weight matrix, its output features as rows).  out is F32, F16 or
 * BF16 (out_dtype) with rows of out_stride elements.  The sums are in binary32.  inner may be 0.
 * Scales are powers of two from 2^-126 on, as pcu_b200_block_quantize writes them (the tensor cores
 * apply them as exponents); any other scale gives NaN in its cells.
 * Codes with 16-byte aligned bases and strides run on the tensor cores; others give the same
 * results to rounding, slowly.
 * Events: the cell row * columns + column. */
int pcu_b200_block_matmul(int out_dtype, const void *left, const float *left_scales, const void *right,
                          const float *right_scales, void *out, uint64_t rows, uint64_t inner, uint64_t columns,
                          uint64_t left_stride, uint64_t right_stride, uint64_t out_stride, uint64_t *status,
                          void *stream);

/* ------------------------------------------------------------------ guarded forms */

/* The calls above as stages of a guarded chain (see pcu_b200_chain_reset): `status` is replaced by
 * (chain_records, chain_stage).  Event extents for pcu_b200_chain_validate: batch*positions*channels
 * for group norm, that + 2*channels for its backward, rows for distillation, rows*columns for the
 * quantiser and the product. */
int pcu_b200_guarded_group_norm(int dtype, int activation, const void *input, const void *weight, const void *bias,
                                void *out, void *stats, uint64_t batch, uint64_t positions, uint64_t channels,
                                uint64_t groups, uint64_t input_batch_stride, uint64_t input_stride,
                                uint64_t out_batch_stride, uint64_t out_stride, uint32_t eps_bits_f32, void *workspace,
                                size_t workspace_bytes, uint64_t *chain_records, uint32_t chain_stage, void *stream);
int pcu_b200_guarded_group_norm_backward(int dtype, int activation, const void *input, const void *upstream,
                                         const void *weight, const void *bias, const void *stats, void *gradient,
                                         void *weight_gradient, void *bias_gradient, uint64_t batch,
                                         uint64_t positions, uint64_t channels, uint64_t groups,
                                         uint64_t input_batch_stride, uint64_t input_stride,
                                         uint64_t upstream_batch_stride, uint64_t upstream_stride,
                                         uint64_t gradient_batch_stride, uint64_t gradient_stride, void *workspace,
                                         size_t workspace_bytes, uint64_t *chain_records, uint32_t chain_stage,
                                         void *stream);
int pcu_b200_guarded_distill_loss(int dtype, const void *logits, uint64_t rows, uint64_t vocab, uint64_t logits_stride,
                                  const int64_t *top_indices, const void *top_logits, uint64_t top_count,
                                  const void *row_weights, uint32_t temperature_bits_f32, void *loss, void *row_stats,
                                  uint64_t *chain_records, uint32_t chain_stage, void *stream);
int pcu_b200_guarded_distill_loss_backward(int dtype, const void *logits, uint64_t rows, uint64_t vocab,
                                           uint64_t logits_stride, const int64_t *top_indices, const void *top_logits,
                                           uint64_t top_count, const void *row_weights, uint32_t temperature_bits_f32,
                                           const void *row_stats, const void *upstream, int upstream_uniform,
                                           void *gradient, uint64_t gradient_stride, uint64_t *chain_records,
                                           uint32_t chain_stage, void *stream);
int pcu_b200_guarded_distill_loss_step(int dtype, const void *logits, uint64_t rows, uint64_t vocab,
                                       uint64_t logits_stride, const int64_t *top_indices, const void *top_logits,
                                       uint64_t top_count, const void *row_weights, uint32_t temperature_bits_f32,
                                       void *loss, void *row_stats, const void *upstream, int upstream_uniform,
                                       void *gradient, uint64_t gradient_stride, uint64_t *chain_records,
                                       uint32_t chain_stage, void *stream);
int pcu_b200_guarded_block_quantize(int dtype, const void *input, uint64_t rows, uint64_t columns,
                                    uint64_t input_stride, int block_rows, void *codes, uint64_t codes_stride,
                                    float *scales, uint64_t *chain_records, uint32_t chain_stage, void *stream);
int pcu_b200_guarded_block_matmul(int out_dtype, const void *left, const float *left_scales, const void *right,
                                  const float *right_scales, void *out, uint64_t rows, uint64_t inner,
                                  uint64_t columns, uint64_t left_stride, uint64_t right_stride, uint64_t out_stride,
                                  uint64_t *chain_records, uint32_t chain_stage, void *stream);

#ifdef __cplusplus
}
#endif
#endif
