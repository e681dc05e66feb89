/*
 * ffai_prefix.h -- C ABI of attention over a shared prefix on MI355X (gfx950).
 *
 * No counterpart in the reference, whose beams each restore a whole DecoderState
 * (crates/ffai-mercury/src/asr/decoder.rs:559-583): here the keys that several sequences have in
 * common (a window's prompt under beam search or temperature sampling, a document under many
 * answers) are held once per group of slots, and each slot's own cache holds only what it has
 * generated since. One call attends every slot over both, as if they were one sequence; the
 * prefix is read once for all the slots of its group.
 *
 * All calls are asynchronous on `stream` (a hipStream_t; NULL = null stream), allocate nothing,
 * take device pointers of the current device, and return FFAI_OK, FFAI_DECLINED or a negative
 * ffai_status (ffai_attn.h); the reason is then in ffai_attn_last_error(). Strides are in elements.
 */
#ifndef FFAI_PREFIX_H
#define FFAI_PREFIX_H

#include <stddef.h>
#include <stdint.h>

#include "ffai_attn.h"
#include "ffai_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* out[s][h][i] = softmax over the visible keys of scale * q[s][h][i] . k, times their values.
 * `prefix` has one slot per group; own->slots is a multiple of it, and slot s belongs to group
 * s / (own->slots / prefix->slots). Query head h reads K/V head h / (heads_q / heads). Row i of
 * the q_len rows of slot s sees every key of its group's prefix (prefix->lens[group] of them) and
 * the slot's own keys j <= own->lens[s] - q_len + i: the rows are the slot's last q_len tokens,
 * whose K/V rows the cache already holds (ffai_kv_append runs first). Lengths are read on the
 * device and clamped to [0, capacity]; a row that sees no key gives 0. What masked positions
 * hold, NaN included, never reaches a result. The caches are not written; they may be views of
 * larger ones.
 *
 * Types: caches both FFAI_F16 or both FFAI_BF16 (f32 caches are declined: FFAI_DECLINED). q of
 * the caches' type or FFAI_F32; out of the caches' type (q of it too) or FFAI_F32. With a 16-bit
 * output the softmax weights are rounded to the caches' type before the second product; with an
 * f32 output they keep f32 accuracy (as several 16-bit parts), and so does an f32 q. head_dim 64 or 128
 * (others are declined). Cache bases 16-byte aligned and strides multiples of 8 elements, the
 * position stride at most 2^23. q and out: strides slot, head, row, head_dim contiguous, aligned
 * to their element.
 *
 * The workspace holds partial results only: it needs no clearing and is free again once the
 * call's work on `stream` is done; calls that may overlap need one each. 16-byte aligned. Short
 * sequences need none (0 bytes; then it may be NULL). Results are the same bits at every call. */
int ffai_prefix_attn_fwd(const ffai_kv_cache* prefix, const ffai_kv_cache* own, const void* q,
                         int32_t q_dtype, int32_t heads_q, int32_t q_len,
                         const int64_t* q_strides, float scale, void* out, int32_t out_dtype,
                         const int64_t* o_strides, void* workspace, size_t workspace_bytes,
                         void* stream);

/* Device workspace of that call, from the caches' slots, heads, capacities and head_dim alone. */
int ffai_prefix_attn_workspace_bytes(const ffai_kv_cache* prefix, const ffai_kv_cache* own,
                                     int32_t heads_q, int32_t q_len, size_t* bytes);

/* Diagnostic: the launch plan. info[0]: query rows that share a prefix K/V head, info[1]: pieces
 * the prefix is split into, info[2]: pieces of a slot's own keys, info[3]: workgroups of the
 * attention launch, info[4]: prefix rows per workgroup. */
int ffai_prefix_attn_plan_info(const ffai_kv_cache* prefix, const ffai_kv_cache* own,
                               int32_t heads_q, int32_t q_len, int32_t* info);

#ifdef __cplusplus
}
#endif

#endif /* FFAI_PREFIX_H */
