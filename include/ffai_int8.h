/*
 * ffai_int8.h -- C ABI of linear layers in 8-bit integers on MI355X (gfx950): one scale per row of
 * activations (token) and per row of weights (output channel).
 *
 * Beside the single-row projections of ffai_gemv.h (at most 16 rows, f16 weights, or the
 * vocabulary in blocks of int8 as crates/ffai-mercury/src/asr/vocab_int8.rs quantizes it), these
 * take any number of rows: a prompt's tokens, a batch of sequences, an encoder's frames. No
 * counterpart in the reference.
 *
 *   s[m] = max_k |x[m][k]| * (1 / 127) in f32, both factors f32 (1 where the row is all zero): what
 *          `amax / 127` gives where a division by a constant is that product, as on this device
 *   q[m][k] = round-half-even(x[m][k] / s[m]), of the f32 quotient, in [-127, 127]
 *   acc[m][n] = sum_k q[m][k] * w[n][k], exact in 32-bit integers (in_dim <= 131072)
 *   y[m][n] = (f32(acc) * s[m]) * w_scale[n] + bias[n] in f32 (the last product and the sum
 *             rounded once, as a fused multiply-add), then rounded to y's type
 *
 * so results are the same bits at every call and whatever the number of rows. A row that holds an
 * infinity or a NaN has that scale and non-finite results.
 *
 * All calls are asynchronous on `stream` (a hipStream_t; NULL = null stream), allocate nothing,
 * take device pointers of the current device and return FFAI_OK or a negative ffai_status
 * (ffai_attn.h), with the reason in ffai_attn_last_error(). Row strides are in elements.
 */
#ifndef FFAI_INT8_H
#define FFAI_INT8_H

#include <stddef.h>
#include <stdint.h>

#include "ffai_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of x (rows, dim; FFAI_F32, F16 or BF16, contiguous within a row, aligned to their element)
 * to int8 rows and scales by the formulas above. q: row stride q_row_stride, a multiple of 128 and
 * at least dim, base 16-byte aligned; the bytes from dim to the next multiple of 128 become zero.
 * rows >= 0. The same call quantizes weights (one scale per output channel). */
int ffai_int8_quantize_rows(const void* x, int32_t x_dtype, int32_t rows, int32_t dim,
                            int64_t x_row_stride, int8_t* q, int64_t q_row_stride, float* scale,
                            void* stream);

/* y = the product of quantized rows and weights, scaled. q, q_row_stride and scale as
 * ffai_int8_quantize_rows leaves them (the bytes past in_dim zero). w: (out_dim, in_dim) int8, row
 * stride w_row_stride a multiple of 16 and at least in_dim, 16-byte aligned; the bytes between
 * in_dim and the next multiple of 16 are read but count for nothing. w_scale (out_dim) f32; bias
 * (out_dim) f32 or NULL. y: y_dtype FFAI_F32, F16 or BF16, row stride y_row_stride >= out_dim.
 * Row strides of q and w at most 2^22. */
int ffai_int8_product(const int8_t* q, int64_t q_row_stride, const float* scale, int32_t rows,
                      int32_t in_dim, const int8_t* w, int64_t w_row_stride, const float* w_scale,
                      const float* bias, int32_t out_dim, void* y, int32_t y_dtype,
                      int64_t y_row_stride, void* stream);

/* Both of them: y from x. The workspace holds the quantized rows for the time of the call: it
 * needs no clearing; calls that may overlap need one each. 16-byte aligned. Few rows need none (0
 * bytes; then it may be NULL). */
int ffai_int8_linear(const void* x, int32_t x_dtype, int64_t x_row_stride, int32_t rows,
                     int32_t in_dim, const int8_t* w, int64_t w_row_stride, const float* w_scale,
                     const float* bias, int32_t out_dim, void* y, int32_t y_dtype,
                     int64_t y_row_stride, void* workspace, size_t workspace_bytes, void* stream);
int ffai_int8_linear_workspace_bytes(int32_t rows, int32_t in_dim, size_t* bytes);

/* Diagnostic: the tile that ffai_int8_product runs for these sizes: info[0]: rows of x, info[1]:
 * rows of w, info[2]: waves, info[3]: workgroups. */
int ffai_int8_plan_info(int32_t rows, int32_t in_dim, int32_t out_dim, int32_t* info);

#ifdef __cplusplus
}
#endif

#endif /* FFAI_INT8_H */
