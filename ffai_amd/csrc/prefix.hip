// Attention over a shared prefix: the C ABI (include/ffai_prefix.h), its launch plan, and the
// kernel that joins a row's pieces. The attention kernel itself: prefix_attn.cuh.
#include "../../include/ffai_prefix.h"

#include <algorithm>
#include <cmath>

#include "attn_common.cuh"
#include "prefix_attn.h"

namespace ffai {
namespace {

// out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over a row's pieces, m = max m_i; 0 where no
// piece saw a key. One wave per row: D / 4 lanes cover O, the lane groups take pieces in turn
// (each its own running maximum) and join at the end, always in the same order. Bound by one
// round trip for the (m, l) pairs and one for O: the loads of four pieces go out together.
template <int OUTT, int D>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixMergeParams p) {
  constexpr int C4 = D / 4, NG = 64 / C4;
  const int lane = item_id() & 63;
  const int row = __builtin_amdgcn_readfirstlane(wg_id_x() * 4 + (item_id() >> 6));
  if (row >= p.rows) return;  // wave-uniform
  const int g = lane / C4, c = lane % C4;
  const float* ml = p.ml + (int64_t)row * p.pieces * 2;
  const float* po = p.part + (int64_t)row * p.pieces * D + 4 * c;
  float m = kNegInf, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
#pragma unroll 1
  for (int i0 = g; i0 < p.pieces; i0 += NG * U) {
    f32x2 a[U];
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + NG * u, p.pieces - 1);
      a[u] = *reinterpret_cast<const f32x2*>(ml + 2 * i);
      x[u] = *reinterpret_cast<const f32x4*>(po + (int64_t)i * D);
    }
    float mt = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + NG * u < p.pieces) mt = fmaxf(mt, a[u][0]);
    const float mc = mt == kNegInf ? 0.f : mt;
    const float old = fast_exp2(m - mc);
    acc *= old;
    l *= old;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float wt = i0 + NG * u < p.pieces ? fast_exp2(a[u][0] - mc) : 0.f;
      if (i0 + NG * u < p.pieces) {
        acc += wt * x[u];
        l = __builtin_fmaf(wt, a[u][1], l);
      }
    }
    m = mt;
  }
#pragma unroll
  for (int s = C4; s < 64; s *= 2) {
    const float m2 = __shfl_xor(m, s), l2 = __shfl_xor(l, s);
    f32x4 x2;
#pragma unroll
    for (int e = 0; e < 4; ++e) x2[e] = __shfl_xor(acc[e], s);
    const float mt = fmaxf(m, m2), mc = mt == kNegInf ? 0.f : mt;
    // lane pairs add the same two products, the lower group's first, so both hold the same bits
    const float w1 = fast_exp2(m - mc), w2 = fast_exp2(m2 - mc);
    const bool low = (lane & s) == 0;
    const float wa = low ? w1 : w2, wb = low ? w2 : w1;
    const float la = low ? l : l2, lb = low ? l2 : l;
    l = __builtin_fmaf(wb, lb, wa * la);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float xa = low ? acc[e] : x2[e], xb = low ? x2[e] : acc[e];
      acc[e] = __builtin_fmaf(wb, xb, wa * xa);
    }
    m = mt;
  }
  if (g == 0) {
    // (the sum's bits are tested: a NaN sum must reach the output, not become an empty row)
    const float inv = (__float_as_uint(l) & 0x7fffffffu) == 0 ? 0.f : 1.f / l;
    const int rr = row % p.R, sh = row / p.R;
    const int h = sh % p.Hkv, slot = sh / p.Hkv;
    const int hh = rr / p.T, t = rr - hh * p.T;
    store_t<OUTT>* o = reinterpret_cast<store_t<OUTT>*>(p.out) + (int64_t)slot * p.o_ss +
                       (int64_t)(h * p.rep + hh) * p.o_sh + (int64_t)t * p.o_st + 4 * c;
    st4<OUTT>(o, acc * inv);
  }
}

template <int OUTT>
void launch_merge(const PrefixMergeParams& p, int d, hipStream_t s) {
  const dim3 grid((unsigned)((p.rows + 3) / 4));
  if (d == 64) hipLaunchKernelGGL((prefix_merge_kernel<OUTT, 64>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((prefix_merge_kernel<OUTT, 128>), grid, dim3(256), 0, s, p);
}

int check_side(const ffai_kv_cache* c) {
  if (!c) return api_fail(FFAI_ERR_INVALID, "null cache");
  if (c->dtype != FFAI_F32 && c->dtype != FFAI_F16 && c->dtype != FFAI_BF16)
    return api_fail(FFAI_ERR_INVALID, "unknown cache dtype");
  if (c->slots < 1 || c->heads < 1 || c->capacity < 1 || c->capacity > (1 << 30) || c->head_dim < 1)
    return api_fail(FFAI_ERR_INVALID, "slots, heads, head_dim >= 1 and capacity in [1, 2^30]");
  return FFAI_OK;
}

// Sizes alone: what the workspace query and the call both need.
int check_sizes(const ffai_kv_cache* pre, const ffai_kv_cache* own, int32_t heads_q, int32_t q_len) {
  int rc = check_side(pre);
  if (rc != FFAI_OK) return rc;
  rc = check_side(own);
  if (rc != FFAI_OK) return rc;
  if (pre->dtype != own->dtype || pre->heads != own->heads || pre->head_dim != own->head_dim)
    return api_fail(FFAI_ERR_INVALID, "prefix and own cache differ in dtype, heads or head_dim");
  if (own->slots % pre->slots)
    return api_fail(FFAI_ERR_INVALID, "own slots must be a multiple of the prefix's (one prefix slot per group)");
  if (heads_q < 1 || heads_q % own->heads || q_len < 1)
    return api_fail(FFAI_ERR_INVALID, "heads_q must be a multiple of the cache's heads, q_len >= 1");
  if ((int64_t)own->slots * heads_q * q_len > (int64_t(1) << 24))
    return api_fail(FFAI_ERR_INVALID, "more than 2^24 query rows");
  if (own->dtype == FFAI_F32) return api_fail(FFAI_DECLINED, "f32 caches are not served");
  if (own->head_dim != 64 && own->head_dim != 128)
    return api_fail(FFAI_DECLINED, "head_dim must be 64 or 128");
  return FFAI_OK;
}

struct PrefixPlan {
  int R, M, pieces_p, pieces_o, blocks_p, blocks_o;
  bool many;
  int block_slots;  // > 0: the whole attention in one launch, this many slots a workgroup
  int64_t items_p, items_o, rows;
  size_t part_bytes, bytes;
};

// Tiles (by capacity, which is what the host knows) up to which a workgroup of eight waves attends
// whole slots: where such workgroups fill the GPU (one for most CUs, or tiles enough for pieces to
// fill it anyway), pieces win nothing but shorter chains; where they do not, pieces win the other
// CUs. Both ways, us (one slot a workgroup unless they exceed 256): head_dim
// 64, 5 slots x 16 heads, 3, 9 and 17 tiles 5.2 (7.0), 7.2 (7.3) and 9.1 (7.4); 32 x 16, 17 and 33
// tiles 10.2 (11.9) and 15.9 (16.2); head_dim 128, 5 x 16, 3 and 9 tiles 6.0 (7.3) and 9.7 (8.5);
// 32 x 16, 9 and 17 tiles 13.1 (13.5) and 18.8 (18.6).
constexpr int64_t whole_tiles(int64_t head_dim, bool full) {
  return head_dim == 64 ? (full ? 40 : 9) : (full ? 17 : 6);
}

PrefixPlan plan_prefix(const ffai_kv_cache* pre, const ffai_kv_cache* own, int heads_q, int q_len) {
  PrefixPlan p{};
  p.R = heads_q / own->heads * q_len;
  p.M = own->slots / pre->slots * p.R;
  const int block = prefix_row_block(own->head_dim);
  const int64_t units = (int64_t)pre->slots * own->heads;
  const int64_t units_o = (int64_t)own->slots * own->heads * ((p.R + block - 1) / block);
  const int64_t tiles_p = (pre->capacity + kBlockN - 1) / kBlockN;
  const int64_t tiles_o = (own->capacity + kBlockN - 1) / kBlockN;
  auto ceil_div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  // Few tiles for a block of whole slots: one launch, no partials (the launch and the round trip of a
  // merge cost as much as the attention of a short step).
  if (p.R <= block) {
    const int64_t per = own->slots / pre->slots;
    // As few slots to a workgroup as keep one workgroup or less to a CU (110 slots x 8 heads, 48 shared
    // and 5 own keys: 4 slots 8.4 us, 32 slots 18.2; 8 x 5 slots x 16 heads, 224 shared and 200 own
    // keys: 3 slots 10.1, 5 slots 11.0).
    const int64_t most = std::min<int64_t>(per, block / p.R);
    int64_t bs = 1;
    while (bs < most && units * ceil_div(per, bs) > 256) ++bs;
    const bool full = units * ceil_div(per, bs) >= 192 ||
                      units * tiles_p + own->slots * own->heads * tiles_o >= 8 * 256;
    if (tiles_p + bs * tiles_o <= whole_tiles(own->head_dim, full)) {
      p.block_slots = (int)bs;
      p.blocks_p = (int)ceil_div(per, bs);
      p.pieces_p = 1;
      p.items_p = (int64_t)pre->slots * own->heads * p.blocks_p;
      p.rows = (int64_t)own->slots * heads_q * q_len;
      return p;
    }
  }
  // Row blocks of 32 or 16 read the prefix once each, through the caches, and their waves run a tile's
  // whole chain alone: short, but far from the matrix cores' rate. Blocks of 128 share a tile among
  // four waves; they pay off once the products outweigh the chain.
  const int64_t wave_tiles = units * ceil_div(p.M, 32) * tiles_p;
  p.many = p.M > 64 && wave_tiles >= 4096;
  p.blocks_p = (int)ceil_div(p.M, p.many ? kPrefixManyRows : block);
  p.blocks_o = (p.R + block - 1) / block;
  const int64_t units_p = units * p.blocks_p;
  // Key pieces: enough workgroups for two on every CU, but no fewer than four tiles (one a wave)
  // to a piece, since every piece of a row is written once and read once by the merge. Blocks of
  // 128 rows: one workgroup on every CU, which leaves its other place to the own pieces' stream under
  // those products, eight tiles at least (128 slots x 32 heads, 16384 shared and 33 to 1024 own keys: 95
  // us; two workgroups on every CU, twice the pieces, 113; one and a half 103).
  constexpr int64_t kTarget = 512;
  auto pieces = [&](int64_t tiles, int64_t least, int64_t target, int64_t n) {
    return (int)std::min<int64_t>(std::min<int64_t>(ceil_div(tiles, least), 64),
                                  std::max<int64_t>(1, ceil_div(target, n)));
  };
  p.pieces_p = p.many ? pieces(tiles_p, 8, kTarget / 2, units_p)
                      : pieces(tiles_p, 4, std::max<int64_t>(kTarget - units_o, kTarget / 2), units_p);
  p.pieces_o = pieces(tiles_o, 4, kTarget - (p.many ? 0 : units_p * p.pieces_p), units_o);
  p.items_p = units_p * p.pieces_p;
  p.items_o = units_o * p.pieces_o;
  p.rows = (int64_t)own->slots * heads_q * q_len;
  const size_t n = (size_t)p.rows * (p.pieces_p + p.pieces_o);
  p.part_bytes = n * own->head_dim * sizeof(float);
  p.bytes = p.part_bytes + ((n * 2 * sizeof(float) + 15) & ~size_t(15));
  return p;
}

int check_operands(const ffai_kv_cache* c) {
  if (!c->k || !c->v || !c->lens) return api_fail(FFAI_ERR_INVALID, "null cache pointer");
  if (c->strides[0] < 0 || c->strides[1] < 0 || c->strides[2] < c->head_dim ||
      c->strides[2] > (1 << 23))
    return api_fail(FFAI_ERR_INVALID, "bad cache strides (position stride in [head_dim, 2^23])");
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || c->strides[0] % 8 || c->strides[1] % 8 ||
      c->strides[2] % 8 || (uintptr_t)c->lens % 4)
    return api_fail(FFAI_ERR_INVALID, "cache bases must be 16-byte aligned, strides multiples of 8 elements");
  return FFAI_OK;
}

}  // namespace
}  // namespace ffai

using namespace ffai;

extern "C" {

int ffai_prefix_attn_workspace_bytes(const ffai_kv_cache* prefix, const ffai_kv_cache* own,
                                     int32_t heads_q, int32_t q_len, size_t* bytes) {
  api_clear_error();
  if (!bytes) return api_fail(FFAI_ERR_INVALID, "null bytes pointer");
  const int rc = check_sizes(prefix, own, heads_q, q_len);
  if (rc != FFAI_OK) return rc;
  *bytes = plan_prefix(prefix, own, heads_q, q_len).bytes;
  return FFAI_OK;
}

int ffai_prefix_attn_plan_info(const ffai_kv_cache* prefix, const ffai_kv_cache* own,
                               int32_t heads_q, int32_t q_len, int32_t* info) {
  api_clear_error();
  if (!info) return api_fail(FFAI_ERR_INVALID, "null info pointer");
  const int rc = check_sizes(prefix, own, heads_q, q_len);
  if (rc != FFAI_OK) return rc;
  const PrefixPlan p = plan_prefix(prefix, own, heads_q, q_len);
  info[0] = p.M;
  info[1] = p.pieces_p;
  info[2] = p.pieces_o;
  info[3] = (int32_t)(p.items_p + p.items_o);
  info[4] = p.block_slots > 0 ? p.block_slots * p.R : std::min(p.M, p.many ? kPrefixManyRows : prefix_row_block(own->head_dim));
  return FFAI_OK;
}

int ffai_prefix_attn_fwd(const ffai_kv_cache* prefix, const ffai_kv_cache* own, const void* q,
                         int32_t q_dtype, int32_t heads_q, int32_t q_len,
                         const int64_t* q_strides, float scale, void* out, int32_t out_dtype,
                         const int64_t* o_strides, void* workspace, size_t workspace_bytes,
                         void* stream) {
  api_clear_error();
  int rc = check_sizes(prefix, own, heads_q, q_len);
  if (rc != FFAI_OK) return rc;
  rc = check_operands(prefix);
  if (rc != FFAI_OK) return rc;
  rc = check_operands(own);
  if (rc != FFAI_OK) return rc;
  if (!q || !out || !q_strides || !o_strides) return api_fail(FFAI_ERR_INVALID, "null pointer");
  const int dt = own->dtype;
  if (q_dtype != FFAI_F32 && q_dtype != dt)
    return api_fail(FFAI_ERR_INVALID, "q must be f32 or of the caches' type");
  if (out_dtype != FFAI_F32 && (out_dtype != dt || q_dtype != dt))
    return api_fail(FFAI_ERR_INVALID, "out must be f32, or of the caches' type when q is");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return api_fail(FFAI_ERR_INVALID, "scale must be finite and > 0");
  const size_t qe = q_dtype == FFAI_F32 ? 4 : 2, oe = out_dtype == FFAI_F32 ? 4 : 2;
  if ((uintptr_t)q % qe || (uintptr_t)out % oe)
    return api_fail(FFAI_ERR_INVALID, "q and out must be aligned to their element size");
  const int64_t ext[3] = {own->slots, heads_q, q_len};
  for (int i = 0; i < 3; ++i) {
    if (q_strides[i] < 0 || o_strides[i] < 0)
      return api_fail(FFAI_ERR_INVALID, "q and out strides must not be negative");
    if (ext[i] > 1 && o_strides[i] < own->head_dim)
      return api_fail(FFAI_ERR_INVALID, "out rows overlap (a stride below head_dim)");
  }
  const PrefixPlan pl = plan_prefix(prefix, own, heads_q, q_len);
  if (pl.items_p + pl.items_o > 0x7fffffff)
    return api_fail(FFAI_ERR_INVALID, "problem too large");
  if (pl.bytes > 0 && (!workspace || workspace_bytes < pl.bytes))
    return api_fail(FFAI_ERR_WORKSPACE, "workspace smaller than ffai_prefix_attn_workspace_bytes");
  if ((uintptr_t)workspace % 16)
    return api_fail(FFAI_ERR_INVALID, "workspace must be 16-byte aligned");
  rc = api_check_device();
  if (rc != FFAI_OK) return rc;

  PrefixParams p{};
  p.q = q;
  p.q_ss = q_strides[0]; p.q_sh = q_strides[1]; p.q_st = q_strides[2];
  p.out = out;
  p.o_ss = o_strides[0]; p.o_sh = o_strides[1]; p.o_st = o_strides[2];
  auto side = [](const ffai_kv_cache* c, int pieces, int blocks, int64_t items) {
    PrefixSide s{};
    s.k = c->k; s.v = c->v; s.lens = c->lens;
    s.s_slot = c->strides[0]; s.s_head = c->strides[1]; s.s_pos = c->strides[2];
    s.capacity = c->capacity; s.pieces = pieces; s.row_blocks = blocks; s.items = (int32_t)items;
    return s;
  };
  p.pre = side(prefix, pl.pieces_p, pl.blocks_p, pl.items_p);
  p.own = side(own, pl.pieces_o, pl.blocks_o, pl.items_o);
  p.part = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.part_bytes);
  p.per = own->slots / prefix->slots;
  p.Hkv = own->heads; p.rep = heads_q / own->heads; p.T = q_len; p.R = pl.R; p.M = pl.M;
  p.many = pl.many;
  p.scale_log2 = scale * 1.44269504088896340736f;
  const int parts = q_dtype == FFAI_F32     ? kPartsBoth
                    : out_dtype == FFAI_F32 ? kPartsWeights
                                            : kPartsOne;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (pl.block_slots > 0) {
    p.block_slots = pl.block_slots;
    if (parts != kPartsOne && p.R <= 16) {  // (the parts leave registers for 16 rows)
      p.block_slots = std::min(p.block_slots, 16 / p.R);
      p.pre.row_blocks = (p.per + p.block_slots - 1) / p.block_slots;
    }
    const hipError_t e = dt == FFAI_F16
                             ? launch_whole_f16(p, prefix->slots, own->head_dim, parts, st)
                             : launch_whole_bf16(p, prefix->slots, own->head_dim, parts, st);
    if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
    return FFAI_OK;
  }
  hipError_t e = dt == FFAI_F16 ? launch_prefix_f16(p, own->head_dim, parts, st)
                                : launch_prefix_bf16(p, own->head_dim, parts, st);
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  PrefixMergeParams m{};
  m.part = p.part; m.ml = p.ml; m.out = out;
  m.o_ss = o_strides[0]; m.o_sh = o_strides[1]; m.o_st = o_strides[2];
  m.rows = (int32_t)pl.rows; m.pieces = pl.pieces_p + pl.pieces_o;
  m.Hkv = p.Hkv; m.rep = p.rep; m.T = p.T; m.R = p.R;
  if (out_dtype == FFAI_F32) launch_merge<kF32>(m, own->head_dim, st);
  else if (dt == FFAI_F16) launch_merge<kF16>(m, own->head_dim, st);
  else launch_merge<kBF16>(m, own->head_dim, st);
  e = hipGetLastError();
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  return FFAI_OK;
}

}  // extern "C"
