// Parameters and launchers of attention over a shared prefix (prefix_attn.cuh, prefix.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ffai {

// One cache side: K and V of (slot, head, position, head_dim), 16-bit.
struct PrefixSide {
  const void* k;
  const void* v;
  int64_t s_slot, s_head, s_pos;  // elements
  const int32_t* lens;
  int32_t capacity;
  int32_t pieces;      // key pieces of a unit
  int32_t row_blocks;  // row blocks of a unit
  int32_t items;       // workgroups
};

struct PrefixParams {
  const void* q;
  int64_t q_ss, q_sh, q_st;  // slot, head, row strides (elements)
  void* out;  // prefix_whole_kernel writes it; else the merge does
  int64_t o_ss, o_sh, o_st;
  PrefixSide pre, own;
  float* part;  // partial rows: O [row][piece][D], row = (slot * Hkv + head) * R + rr, pieces of
                // the prefix first, then the own ones
  float* ml;    // their (max, weight sum) pairs [row][piece][2]
  int32_t per;  // slots per group
  int32_t Hkv, rep, T;
  int32_t R;  // rows of a slot that read one K/V head: rep * T
  int32_t M;  // rows of a group that read one prefix K/V head: per * R
  int32_t block_slots;  // prefix_whole_kernel: slots of a workgroup
  int32_t many;    // the prefix's pieces in blocks of kPrefixManyRows rows (prefix_rows)
  float scale_log2;
};

struct PrefixMergeParams {
  const float* part;
  const float* ml;
  void* out;
  int64_t o_ss, o_sh, o_st;
  int32_t rows;  // slots * Hkv * R
  int32_t pieces;
  int32_t Hkv, rep, T, R;
};

// Parts: 16-bit parts that q (NQ) and the softmax weights (NP) are carried in.
enum PrefixParts : int {
  kPartsOne = 0,      // q and weights of the caches' type
  kPartsWeights = 1,  // q of the caches' type, weights to f32 accuracy
  kPartsBoth = 2      // f32 q, weights to f32 accuracy
};

hipError_t launch_prefix_f16(const PrefixParams& p, int head_dim, int parts, hipStream_t s);
hipError_t launch_prefix_bf16(const PrefixParams& p, int head_dim, int parts, hipStream_t s);
// The whole attention in one launch (p.block_slots, p.pre.row_blocks set; no workspace).
hipError_t launch_whole_f16(const PrefixParams& p, int groups, int head_dim, int parts, hipStream_t s);
hipError_t launch_whole_bf16(const PrefixParams& p, int groups, int head_dim, int parts, hipStream_t s);

constexpr int kPrefixWaves = 4;     // waves of a workgroup, a key tile each
// Rows of a workgroup of prefix_work: two 16-column MFMA blocks at head_dim 64. At 128 one: two need
// more than the 256 registers that leave room for two workgroups on a CU.
constexpr int prefix_row_block(int head_dim) { return head_dim == 64 ? 32 : 16; }
constexpr int kWholeWaves = 8;  // waves of a workgroup of prefix_whole_kernel
constexpr int kPrefixManyRows = 128;  // rows of a workgroup of prefix_rows: 32 a wave

}  // namespace ffai
