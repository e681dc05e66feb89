/*
 * ffai_sample.h -- C ABI of sampling on MI355X (gfx950): one token per row of logits, with
 * temperature, top-k, min-p and top-p, from given uniform numbers.
 *
 * What follows the vocabulary projection (ffai_vocab_int8_logits, ffai_gemv.h) on the device. The
 * reference samples on the host (crates/ffai-mercury/src/asr/decoder.rs:650-847, its temperature
 * ladder); logits then cross to the host at every step.
 *
 * For a row of logits l (widened to f32; a NaN counts as -inf) with largest value m:
 *   w_i = exp((l_i - m) / T) in 64 bits (w_i = 1 where l_i = m, 0 where l_i = -inf);
 *   order: l descending, the lower index first among equals;
 *   S1: the first top_k tokens in that order (all of them when top_k <= 0) of weight >= min_p
 *       (min_p <= 0: all; above 1: as 1), so min_p is relative to the likeliest token;
 *   S2: the tokens of S1 whose predecessors in that order weigh less than top_p * W(S1) together
 *       (top_p >= 1 or NaN: all of S1), at least the first;
 *   token: the lowest index i such that the tokens of S2 up to i weigh more than u * W(S2)
 *       (u below 0 or NaN counts as 0, from 1 on as the largest f32 below 1).
 * T <= 0 or NaN: the first maximum, whatever the other settings. The other NaN settings: as if
 * off. A row without a finite or infinite maximum (all -inf or NaN) gives token -1.
 * logprob: log softmax(l)[token] at temperature 1 over the whole row, -inf for token -1.
 *
 * Token choices are exact to 64-bit rounding (below 1e-12 of the row's weight) and the same at
 * every call. All calls are asynchronous on `stream` (a hipStream_t; NULL = null stream), allocate
 * nothing, take device pointers of the current device and return FFAI_OK or a negative
 * ffai_status (ffai_attn.h), with the reason in ffai_attn_last_error().
 */
#ifndef FFAI_SAMPLE_H
#define FFAI_SAMPLE_H

#include <stddef.h>
#include <stdint.h>

#include "ffai_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* logits: (rows, vocab) FFAI_F32, F16 or BF16, row stride logits_row_stride (elements), contiguous
 * within a row, aligned to their element; vocab in [1, 2^20]. Each setting is a device array of
 * one value per row, or NULL for the one value that follows it. u: rows f32. tokens: rows int32;
 * logprobs: rows f32, or NULL. rows in [0, 65535]. The workspace needs no clearing; calls that
 * may overlap need one each. 16-byte aligned. */
int ffai_sample(const void* logits, int32_t logits_dtype, int32_t rows, int32_t vocab,
                int64_t logits_row_stride, const float* temperature, float temperature_all,
                const int32_t* top_k, int32_t top_k_all, const float* top_p, float top_p_all,
                const float* min_p, float min_p_all, const float* u, int32_t* tokens,
                float* logprobs, void* workspace, size_t workspace_bytes, void* stream);

int ffai_sample_workspace_bytes(int32_t rows, int32_t vocab, size_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* FFAI_SAMPLE_H */
