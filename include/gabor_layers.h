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
 * (either may be null). */
size_t gs_linear_backward_weight_workspace_size(int32_t dtype, int64_t rows, int64_t features,
                                                int64_t outputs);
int gs_linear_backward_weight(int32_t dtype, const void* grad_y, int64_t grad_stride,
                              const void* values, const void* exponents, int64_t rows,
                              int64_t features, int64_t outputs, void* grad_weight,
                              void* grad_bias, void* workspace, size_t workspace_bytes,
                              void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GABOR_LAYERS_H */
