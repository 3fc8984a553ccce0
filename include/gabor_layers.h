/*
 * gabor_layers.h - C ABI of the surfel decoder's layers: layer norm, linear
 * layers and activations over rows of features, forward and backward, with
 * what the backward pass needs of an input kept in 8 bits.
 *
 * The conventions are gabor_hip.h's: device pointers, counts and a HIP
 * stream; nothing allocates; a status code, and gs_last_error() for its
 * message. Rows are row-major with unit feature stride; inputs and output
 * gradients take a row stride (in values), outputs are contiguous.
 *
 * 8-bit form of rows x features values: values [rows, 32 G] int8 and
 * exponents [rows, G] uint8, G = ceil(features / 32). Bytes q of group g
 * stand for q 2^(b - 127), b the group's exponent byte: the smallest with
 * which the group's largest magnitude rounds to at most 127, within 1..248
 * (float16: 103..136); q is rounded to nearest, ties to even, and held to
 * -127..127. A group with an infinity or a NaN has b = 255 and reads back as
 * NaN. Bytes past `features` are zero.
 */
#ifndef GABOR_LAYERS_H
#define GABOR_LAYERS_H

#include "gabor_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of rows. */
#define GS_FLOAT32 0
#define GS_BFLOAT16 1
#define GS_FLOAT16 2

/* Activations. */
#define GS_ACTIVATION_SINE 0 /* sin(omega z) */
#define GS_ACTIVATION_GELU 1 /* z Phi(z), Phi the normal distribution's */
#define GS_ACTIVATION_SILU 2 /* z / (1 + exp(-z)) */

/* The 8-bit form of x, and a contiguous tensor of what it stands for. */
int gs_checkpoint8_write(int32_t dtype, const void* x, int64_t row_stride, int64_t rows,
                         int64_t features, void* values, void* exponents, void* stream);
int gs_checkpoint8_read(int32_t dtype, const void* values, const void* exponents, int64_t rows,
                        int64_t features, void* out, void* stream);

/* y = f(x), keeping x in 8 bits where values and exponents are not null, and
 * grad_x = grad_y f'(kept x). omega is read by the sine alone. */
int gs_activation_forward(int32_t dtype, int32_t kind, float omega, const void* x,
                          int64_t row_stride, int64_t rows, int64_t features, void* y,
                          void* values, void* exponents, void* stream);
int gs_activation_backward(int32_t dtype, int32_t kind, float omega, const void* grad_y,
                           int64_t grad_stride, const void* values, const void* exponents,
                           int64_t rows, int64_t features, void* grad_x, void* stream);

/* Layer norm over up to 16384 features; weight and bias (either may be null)
 * have the rows' type or float32. statistics [rows, 2] float32 (null: not
 * kept) = (mean - centre, inverse deviation); with values and exponents the
 * rows less their centre, min / 2 + max / 2, are kept in 8 bits (float32's
 * exponents), otherwise the centre is 0. The backward reads x or what was
 * kept, the other null; grad_weight and grad_bias may each be null, and
 * without both no workspace is needed. With no rows they are set to zero. */
int gs_layer_norm_forward(int32_t dtype, int32_t weight_dtype, const void* x, int64_t row_stride,
                          const void* weight, const void* bias, float eps, int64_t rows,
                          int64_t features, void* y, void* statistics, void* values,
                          void* exponents, void* stream);
size_t gs_layer_norm_backward_workspace_size(int64_t rows, int64_t features);
int gs_layer_norm_backward(int32_t dtype, int32_t weight_dtype, const void* grad_y,
                           int64_t grad_stride, const void* x, int64_t row_stride,
                           const void* values, const void* exponents, const void* statistics,
                           const void* weight, int64_t rows, int64_t features, void* grad_x,
                           void* grad_weight, void* grad_bias, void* workspace,
                           size_t workspace_bytes, void* stream);

/* y = x weight^T + bias (bias may be null), weight [outputs, features], all
 * of one type, keeping x in 8 bits where values and exponents are not null. */
int gs_linear_forward(int32_t dtype, const void* x, int64_t row_stride, const void* weight,
                      const void* bias, int64_t rows, int64_t features, int64_t outputs, void* y,
                      void* values, void* exponents, void* stream);
/* grad_x = grad_y weight. */
int gs_linear_backward_input(int32_t dtype, const void* grad_y, int64_t grad_stride,
                             const void* weight, int64_t rows, int64_t features, int64_t outputs,
                             void* grad_x, void* stream);
/* grad_weight = grad_y^T (kept x), grad_bias = the sum of grad_y's rows
 * (either may be null, and without grad_weight the kept x, too). */
size_t gs_linear_backward_weight_workspace_size(int32_t dtype, int64_t rows, int64_t features,
                                                int64_t outputs);
int gs_linear_backward_weight(int32_t dtype, const void* grad_y, int64_t grad_stride,
                              const void* values, const void* exponents, int64_t rows,
                              int64_t features, int64_t outputs, void* grad_weight,
                              void* grad_bias, void* workspace, size_t workspace_bytes,
                              void* stream);

/* Dropout: y = x / (1 - p) where the mask keeps a value, else 0; the backward
 * pass is the same call on grad_y. The mask is a function of the value's row
 * and column and of the seed (seed_at where that is not null: one 64-bit
 * word on the device, read when the kernel runs): Philox4x32-10 with the key
 * (seed's low word, high word) and the counter (column / 8, row's low word,
 * high word, 0) gives four words, whose eight halves, low ones first, are
 * the bits of eight columns; a value is kept where its bits are at least
 * t = rint(65536 p), and multiplied by 65536 / (65536 - t). */
int gs_dropout(int32_t dtype, double p, int64_t seed, const void* seed_at, const void* x,
               int64_t row_stride, int64_t rows, int64_t features, void* y, void* stream);

/* Rows in groups. The row at position p of 0 .. rows - 1 is order[p] (p where
 * order is null), group g has the positions offsets[g] .. offsets[g + 1] - 1,
 * and the rows at other positions are in no group. order is a permutation of
 * the rows, offsets [groups + 1] does not fall; both are held to the rows
 * that exist. rows <= 2^31 - 4096.
 *
 * gs_row_groups makes both of each row's group (index, int32 or with `wide`
 * int64; outside 0 .. groups - 1: of none, behind the last group), each
 * group's rows in their order, for up to 4096 groups. */
size_t gs_row_groups_workspace_size(int64_t rows, int64_t groups);
int gs_row_groups(int32_t wide, const void* index, int64_t rows, int64_t groups, int32_t* order,
                  int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream);

/* A linear layer by group: y = x weight[g]^T + bias[g] for the rows of group g
 * (weight [groups, outputs, features], bias [groups, outputs] or null), all of
 * one type; rows of no group have y = 0 and grad_x = 0. groups <= 2^20. */
int gs_grouped_linear_forward(int32_t dtype, const void* x, int64_t row_stride,
                              const void* weight, const void* bias, const int32_t* order,
                              const int32_t* offsets, int64_t rows, int64_t groups,
                              int64_t features, int64_t outputs, void* y, void* stream);
/* grad_x = grad_y weight[g]. */
int gs_grouped_linear_backward_input(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                     const void* weight, const int32_t* order,
                                     const int32_t* offsets, int64_t rows, int64_t groups,
                                     int64_t features, int64_t outputs, void* grad_x,
                                     void* stream);
/* grad_weight[g] = the sum over group g's rows of grad_y^T x, grad_bias[g] the
 * sum of grad_y (either may be null, and without grad_weight x, too; zero for a
 * group without rows). */
size_t gs_grouped_linear_backward_weight_workspace_size(int32_t dtype, int64_t rows,
                                                        int64_t groups, int64_t features,
                                                        int64_t outputs);
int gs_grouped_linear_backward_weight(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                      const void* x, int64_t row_stride, const int32_t* order,
                                      const int32_t* offsets, int64_t rows, int64_t groups,
                                      int64_t features, int64_t outputs, void* grad_weight,
                                      void* grad_bias, void* workspace, size_t workspace_bytes,
                                      void* stream);

/* A linear layer with a low-rank adapter by group: y = x weight^T + bias +
 * scale (x down[g]^T) up[g]^T for the rows of group g (weight [outputs,
 * features], bias [outputs] or null, down [groups, rank, features], up
 * [groups, outputs, rank]), all of one type; rows of no group have the first
 * two terms. rank <= 64. inner (gs_adapted_linear_inner_size bytes, 16-byte
 * aligned) receives scale x down[g]^T of every row, which the backward pass of
 * `up` reads. */
size_t gs_adapted_linear_inner_size(int64_t rows, int64_t rank);
int gs_adapted_linear_forward(int32_t dtype, const void* x, int64_t row_stride,
                              const void* weight, const void* bias, const void* down,
                              const void* up, float scale, const int32_t* order,
                              const int32_t* offsets, int64_t rows, int64_t groups,
                              int64_t features, int64_t outputs, int64_t rank, void* inner,
                              size_t inner_bytes, void* y, void* stream);
/* inner_grad (as large as inner) receives scale grad_y up[g], and grad_x (may
 * be null) grad_y weight + inner_grad down[g]. */
int gs_adapted_linear_backward_input(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                     const void* weight, const void* down, const void* up,
                                     float scale, const int32_t* order, const int32_t* offsets,
                                     int64_t rows, int64_t groups, int64_t features,
                                     int64_t outputs, int64_t rank, void* inner_grad,
                                     size_t inner_bytes, void* grad_x, void* stream);
/* grad_down[g] = the sum over group g's rows of inner_grad^T x, grad_up[g] that
 * of grad_y^T inner (either may be null, and then what it alone reads). */
size_t gs_adapted_linear_backward_adapters_workspace_size(int64_t rows, int64_t groups,
                                                          int64_t features, int64_t outputs,
                                                          int64_t rank);
int gs_adapted_linear_backward_adapters(int32_t dtype, const void* grad_y, int64_t grad_stride,
                                        const void* x, int64_t row_stride, const void* inner,
                                        const void* inner_grad, const int32_t* order,
                                        const int32_t* offsets, int64_t rows, int64_t groups,
                                        int64_t features, int64_t outputs, int64_t rank,
                                        void* grad_down, void* grad_up, void* workspace,
                                        size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GABOR_LAYERS_H */
