// Attention of slots over a shared prefix and their own keys (include/ffai_prefix.h), gfx950.
//
// For a query row q with visible keys K_p (its group's prefix) and K_o (its slot's own):
//   o = (sum_p w_j v_j + sum_o w_j v_j) / (sum_p w_j + sum_o w_j),  w_j = 2^(c q.k_j - m),
// c = scale log2(e). Both sums may be cut anywhere: a piece over any set of keys is its own
// (m, l = sum w, O = sum w v), and pieces join by 2^(m_piece - m) (prefix_merge_kernel).
//
// prefix_unit_kernel, one launch: a workgroup takes one piece of keys and up to 32 query rows
// that read them. Prefix pieces come first (the rows of every slot and head of the group that
// read one K/V head are the columns of one S^T = K Q^T product, so the prefix leaves HBM once per
// 32 rows, and later row blocks find it in L2), then the slots' own pieces. Each of the four
// waves takes 64-key tiles of its own, by DMA into its own LDS region, so all the workgroup's
// loads are in flight at once and no wave waits for another until the four partial results meet
// in LDS.
//
// Products on 16x16x32 MFMA (A lane l: row l % 16, contraction 8 (l / 16) .. +7; B: the same of
// column l % 16; D: rows 4 (l / 16) .. +3 of column l % 16): S^T from K rows as they lie; its D
// layout holds, per lane, 4 consecutive keys of each 16-key block, which is P^T's B layout when
// the contraction slots of lane group q4 are named keys 32 ch + 4 q4 + e and 32 ch + 16 + 4 q4 + e,
// and V^T's A operand is read in that order by transposing LDS reads.
//
// Accuracy: with a 16-bit output the weights are rounded to 16 bits for the second product (the
// rounding is below the output's own); their sum is of the unrounded f32 weights. For an f32
// output a weight is carried in NP parts, w = w0 + w1 (+ w2), each the 16-bit rounding of what the
// earlier ones leave (f16: 2 parts, 22 bits; bf16: 3 parts, 24 bits), and an f32 q likewise in NQ
// (f16 after scaling the row by a power of two so that its largest element lies in [2^14, 2^15)):
// the part products are exact in f32 and sum in f32.
#pragma once

#include "attn_common.cuh"
#include "prefix_attn.h"

namespace ffai {
namespace {

// What one workgroup attends: its keys and its rows.
struct PrefixWork {
  const uint16_t* k;  // the K/V head's position 0
  const uint16_t* v;
  int64_t s_pos;
  int n_keys;          // keys from position 0
  int t_begin, t_end;  // its 64-key tiles
  int h;               // K/V head
  int slot0;           // slot of row 0
  int r0, rows;        // rows r0 .. r0 + rows - 1; row r is row r % R of slot slot0 + r / R
  int causal_last;     // own keys: row t sees keys <= causal_last + t; prefix: INT_MAX / 2
  int piece, pieces;   // index and number of a row's pieces
};

template <int DT>
__device__ __forceinline__ float hi_part(float x) {
  return to_f32<DT>(from_f32<DT>(x));
}

// Whether a pair of 16-bit values holds an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool not_finite2(uint32_t u) {
  constexpr uint32_t E = DT == kBF16 ? 0x7f80u : 0x7c00u;
  return (u & E) == E || ((u >> 16) & E) == E;
}

template <int DT, int D, int NQ, int NP, int NC>
__device__ __forceinline__ void prefix_work(const PrefixParams& p, const PrefixWork& w,
                                            uint16_t* lds) {
  constexpr int NWD = kPrefixWaves;
  constexpr int TILE = BN * D;        // elements of a K or V tile
  constexpr int WBUF = 2 * TILE;      // per wave
  constexpr int OROW = D + 4;         // merge area: rows of O, then maxima, then sums
  constexpr int CH = D / 8;           // 16-byte chunks of a row
  constexpr int RB = 64 / CH;         // rows of a 1 KB DMA block
  constexpr int KC = D / 32;          // contraction chunks of S^T
  static_assert((32 * OROW + 64) * 4 <= WBUF * 2, "the merge area fits in the wave's tile area");
  static_assert(NC * 16 * BN * 4 <= TILE * 2, "a tile's weights fit in the K region");
  const int tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q4 = lane >> 4, n16 = lane & 15;
  uint16_t* kl = lds + wave * WBUF;
  uint16_t* vl = kl + TILE;
  auto swz_k = [](int r, int c) { return D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); };
  auto swz_v = [](int r, int c) { return D == 64 ? c ^ (4 * ((r >> 1) & 1)) : c ^ (4 * (r & 3)); };
  const int tr_row = n16 >> 2, tr_col = 4 * (n16 & 3);

  // A tile by DMA: lane's 16-byte slot of each 1 KB block gets the chunk that the row's XOR
  // permutation assigns to it. Rows past the last key are not read past the block that holds it
  // (within the block the last key's row stands in): their scores are masked and their V rows
  // cleared below.
  const int lr = lane / CH, lc = lane % CH;
  auto issue = [&](int it) {
    const int valid = min(BN, w.n_keys - it * BN);
    const char* kb = reinterpret_cast<const char*>(w.k + (int64_t)it * BN * w.s_pos);
    const char* vb = reinterpret_cast<const char*>(w.v + (int64_t)it * BN * w.s_pos);
    const uint32_t ka = lds_addr(kl), va = lds_addr(vl);
#pragma unroll
    for (int j = 0; j < BN / RB; ++j) {
      const int r = j * RB + lr;
      const uint32_t row = (uint32_t)min(r, valid - 1) * (uint32_t)w.s_pos;
      if (j * RB < valid) lds_dma16_sbase(kb, 2 * (row + 8 * swz_k(r, lc)), ka + j * 1024);
    }
#pragma unroll
    for (int j = 0; j < BN / RB; ++j) {
      const int r = j * RB + lr;
      const uint32_t row = (uint32_t)min(r, valid - 1) * (uint32_t)w.s_pos;
      if (j * RB < valid) lds_dma16_sbase(vb, 2 * (row + 8 * swz_v(r, lc)), va + j * 1024);
    }
  };
  // the first tile's loads go out before anything else
  if (w.t_begin + wave < w.t_end) issue(w.t_begin + wave);

  // ---- Q: column 16 c + n16 is row r0 + that (past the last row: the last row again; such a
  //      column's results are not stored)
  u32x4 qf[NQ][NC][KC];
  int lim[NC];     // the last key the column's row sees
  float sl2[NC];   // scores to log2 units
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = w.r0 + min(16 * c + n16, w.rows - 1);
    const int ds = r / p.R, rr = r - ds * p.R;
    const int hh = rr / p.T, t = rr - hh * p.T;
    lim[c] = min(w.n_keys - 1, w.causal_last + t);
    const int64_t qo = (int64_t)(w.slot0 + ds) * p.q_ss + (int64_t)(w.h * p.rep + hh) * p.q_sh +
                       (int64_t)t * p.q_st;
    if constexpr (NQ == 1) {
#pragma unroll
      for (int h = 0; h < KC; ++h)
        qf[0][c][h] = ld16h(reinterpret_cast<const uint16_t*>(p.q) + qo + 32 * h + 8 * q4);
      sl2[c] = p.scale_log2;
    } else {
      const float* qr = reinterpret_cast<const float*>(p.q) + qo;
      float x[KC][8];
      float mx = 0.f;
#pragma unroll
      for (int h = 0; h < KC; ++h) {
        const f32x4 a = *reinterpret_cast<const f32x4_e*>(qr + 32 * h + 8 * q4);
        const f32x4 b = *reinterpret_cast<const f32x4_e*>(qr + 32 * h + 8 * q4 + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[h][e] = e < 4 ? a[e & 3] : b[e & 3];
          mx = fmaxf(mx, fabsf(x[h][e]));
        }
      }
      float sc = 1.f, inv = 1.f;
      if constexpr (DT == kF16) {
        mx = quad_max(mx);
        // max in [2^e, 2^(e+1)) to [2^14, 2^15): exponent field 127 + 14 - e
        const int sb = min(max(268 - (int)(__float_as_uint(mx) >> 23), 1), 253);
        sc = __uint_as_float((uint32_t)sb << 23);
        inv = __uint_as_float((uint32_t)(254 - sb) << 23);
      }
      sl2[c] = p.scale_log2 * inv;
#pragma unroll
      for (int h = 0; h < KC; ++h)
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) {
          float r0 = x[h][2 * e2] * sc, r1 = x[h][2 * e2 + 1] * sc;
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            const uint32_t pk = pack2<DT>(r0, r1);
            qf[q][c][h][e2] = pk;
            // (an infinite element stays in its first part: inf - inf would be NaN)
            const float h0 = to_f32<DT>(pk & 0xffffu), h1 = to_f32<DT>(pk >> 16);
            r0 = fabsf(h0) < __builtin_inff() ? r0 - h0 : 0.f;
            r1 = fabsf(h1) < __builtin_inff() ? r1 - h1 : 0.f;
          }
        }
    }
  }

  f32x4 oacc[NC][D / 16];  // O^T: d = 16 db + 4 q4 + r of column 16 c + n16
  float m_s[NC], l_run[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db) oacc[c][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_s[c] = kNegInf;
    l_run[c] = 0.f;
  }

#pragma unroll 1
  for (int it = w.t_begin + wave; it < w.t_end; it += NWD) {
    const int kb = it * BN;
    if (it != w.t_begin + wave) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the region's earlier reads are done
      issue(it);
    }
    vm_wait_all();
    asm volatile("" ::: "memory");
    const bool tail = kb + BN > w.n_keys;
    const bool band = p.T > 1 && kb + BN - 1 > w.causal_last;  // keys that some row does not see
    if (tail) {
      // V rows past the last key: a masked weight is 0, but 0 times what lies there need not be
      for (int u = (w.n_keys - kb) * CH + lane; u < BN * CH; u += 64)
        *reinterpret_cast<u32x4*>(&vl[8 * u]) = u32x4{0u, 0u, 0u, 0u};
    }
    // Keys that only later rows see may hold a non-finite V, which a weight of 0 would let into
    // the earlier rows: such a tile takes the slow second product.
    bool slow = false;
    if (band) {
      bool bad = false;
      for (int u = lane; u < BN * CH; u += 64) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(&vl[8 * u]);
        bad = bad || not_finite2<DT>(x[0]) || not_finite2<DT>(x[1]) || not_finite2<DT>(x[2]) ||
              not_finite2<DT>(x[3]);
      }
      slow = __ballot(bad) != 0;
    }

    f32x4 s[NC][4];  // S^T: key kb + 16 kb4 + 4 q4 + r of column 16 c + n16
#pragma unroll
    for (int kb4 = 0; kb4 < 4; ++kb4) {
#pragma unroll
      for (int c = 0; c < NC; ++c) s[c][kb4] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int r = 16 * kb4 + n16;
#pragma unroll
      for (int h = 0; h < KC; ++h) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(&kl[r * D + 8 * swz_k(r, 4 * h + q4)]);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int q = NQ - 1; q >= 0; --q) s[c][kb4] = mfma16x16<DT>(a, qf[q][c][h], s[c][kb4]);
      }
    }
    if (tail || band) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kb + 16 * kb4 + 4 * q4 + r > lim[c]) s[c][kb4][r] = kNegInf;
    }
    u32x4 pf[NP][NC][2];
    float corr[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = kNegInf;
#pragma unroll
      for (int kb4 = 0; kb4 < 4; ++kb4)
        mx = fmaxf(mx, fmaxf(fmaxf(s[c][kb4][0], s[c][kb4][1]), fmaxf(s[c][kb4][2], s[c][kb4][3])));
      const float m_new = fmaxf(m_s[c], quad_max(mx) * sl2[c]);
      const float mc = m_new == kNegInf ? 0.f : m_new;
      corr[c] = fast_exp2(m_s[c] - mc);  // 0 while nothing is seen
      m_s[c] = m_new;
      float rs = 0.f;
#pragma unroll
      for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[c][kb4][r] = fast_exp2(__builtin_fmaf(s[c][kb4][r], sl2[c], -mc));
          rs += s[c][kb4][r];
        }
      l_run[c] = __builtin_fmaf(l_run[c], corr[c], rs);
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float r0 = s[c][2 * ch + (k >> 1)][2 * (k & 1)];
          float r1 = s[c][2 * ch + (k >> 1)][2 * (k & 1) + 1];
#pragma unroll
          for (int q = 0; q < NP; ++q) {
            const uint32_t pk = pack2<DT>(r0, r1);
            pf[q][c][ch][k] = pk;
            r0 -= to_f32<DT>(pk & 0xffffu);
            r1 -= to_f32<DT>(pk >> 16);
          }
        }
#pragma unroll
      for (int db = 0; db < D / 16; ++db) oacc[c][db] *= corr[c];
    }
    if (!slow) {
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          const int r = 32 * ch + 4 * q4 + tr_row, col = 16 * db + tr_col;
          const uint16_t* base = &vl[r * D + 8 * swz_v(r, col >> 3) + (col & 7)];
          const u32x2 a0 = lds_tr(base), a1 = lds_tr(base + 16 * D);
          const u32x4 a = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int q = NP - 1; q >= 0; --q) oacc[c][db] = mfma16x16<DT>(a, pf[q][c][ch], oacc[c][db]);
        }
    } else {
      // key by key, only where the row sees it (the tile's weights through the K region, whose
      // reads are done)
      float* pl = reinterpret_cast<float*>(kl);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            pl[(16 * kb4 + 4 * q4 + r) * (16 * NC) + 16 * c + n16] = s[c][kb4][r];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
      for (int key = 0; key < min(BN, w.n_keys - kb); ++key)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float wt = pl[key * (16 * NC) + 16 * c + n16];
          const bool seen = kb + key <= lim[c];
#pragma unroll
          for (int db = 0; db < D / 16; ++db) {
            const int col = 16 * db + 4 * q4;
            const u32x2 x = *reinterpret_cast<const u32x2*>(
                &vl[key * D + 8 * swz_v(key, col >> 3) + (col & 7)]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float vv = to_f32<DT>((r & 1) ? x[r >> 1] >> 16 : x[r >> 1] & 0xffffu);
              if (seen) oacc[c][db][r] = __builtin_fmaf(wt, vv, oacc[c][db][r]);
            }
          }
        }
      __builtin_amdgcn_s_waitcnt(0xc07f);
    }
  }

  // ---- the waves' results meet in LDS (each wave's tile area is free once all pass here)
  __syncthreads();
  float* mbase = reinterpret_cast<float*>(lds);
  {
    float* mb = mbase + wave * (WBUF / 2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float l = quad_sum(l_run[c]);
      const int n = 16 * c + n16;
      if (n < w.rows) {
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          *reinterpret_cast<f32x4*>(&mb[n * OROW + 16 * db + 4 * q4]) = oacc[c][db];
        if (q4 == 0) {
          mb[32 * OROW + n] = m_s[c];
          mb[32 * OROW + 32 + n] = l;
        }
      }
    }
  }
  __syncthreads();
  constexpr int C4 = D / 4;
  const int np = p.pre.pieces + p.own.pieces;
#pragma unroll 1
  for (int i = tid; i < w.rows * C4; i += NWD * 64) {
    const int n = i / C4, c4 = i % C4;
    float mw[NWD], M = kNegInf;
#pragma unroll
    for (int x = 0; x < NWD; ++x) {
      mw[x] = mbase[x * (WBUF / 2) + 32 * OROW + n];
      M = fmaxf(M, mw[x]);
    }
    const float Mc = M == kNegInf ? 0.f : M;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
#pragma unroll
    for (int x = 0; x < NWD; ++x) {
      const float* mb = mbase + x * (WBUF / 2);
      const float wt = fast_exp2(mw[x] - Mc);
      acc += wt * *reinterpret_cast<const f32x4*>(&mb[n * OROW + 4 * c4]);
      L = __builtin_fmaf(wt, mb[32 * OROW + 32 + n], L);
    }
    const int r = w.r0 + n, ds = r / p.R, rr = r - ds * p.R;
    const int64_t row = ((int64_t)(w.slot0 + ds) * p.Hkv + w.h) * p.R + rr;
    const int64_t at = row * np + w.piece;
    *reinterpret_cast<f32x4*>(p.part + at * D + 4 * c4) = acc;
    if (c4 == 0) *reinterpret_cast<f32x2*>(p.ml + at * 2) = f32x2{M, L};
  }
}

template <int DT, int D, int NQ, int NP, int NCP, int NCO>
__global__ __launch_bounds__(kPrefixWaves * 64, D == 64 ? 2 : 1) void prefix_unit_kernel(
    PrefixParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[kPrefixWaves * 2 * BN * D];
  int item = wg_id_x();
  const bool pre = item < p.pre.items;
  const PrefixSide& sd = pre ? p.pre : p.own;
  if (!pre) item -= p.pre.items;
  // piece fastest, then K/V head, row block, slot (group): the row blocks of a prefix piece are
  // `pieces * Hkv` apart, a multiple of 8 in the large cases, so that they land on one XCD and
  // share its L2
  PrefixWork w;
  const int piece = item % sd.pieces;
  item /= sd.pieces;
  w.h = item % p.Hkv;
  item /= p.Hkv;
  const int rb = item % sd.row_blocks;
  const int slot = item / sd.row_blocks;
  w.piece = pre ? piece : p.pre.pieces + piece;
  w.pieces = p.pre.pieces + p.own.pieces;
  w.n_keys = __builtin_amdgcn_readfirstlane(min(max(sd.lens[slot], 0), sd.capacity));
  const int tiles = (w.n_keys + BN - 1) / BN;
  const int per_piece = (tiles + sd.pieces - 1) / sd.pieces;
  w.t_begin = min(piece * per_piece, tiles);
  w.t_end = min(tiles, w.t_begin + per_piece);
  w.s_pos = sd.s_pos;
  const int64_t base = (int64_t)slot * sd.s_slot + (int64_t)w.h * sd.s_head;
  w.k = reinterpret_cast<const uint16_t*>(sd.k) + base;
  w.v = reinterpret_cast<const uint16_t*>(sd.v) + base;
  w.slot0 = pre ? slot * p.per : slot;
  w.r0 = rb * kPrefixRowBlock;
  w.rows = min(kPrefixRowBlock, (pre ? p.M : p.R) - w.r0);
  w.causal_last = pre ? 0x3fffffff : w.n_keys - p.T;
  if constexpr (NCP == NCO) {
    prefix_work<DT, D, NQ, NP, NCP>(p, w, lds);
  } else {
    if (pre) prefix_work<DT, D, NQ, NP, NCP>(p, w, lds);
    else prefix_work<DT, D, NQ, NP, NCO>(p, w, lds);
  }
}

template <int DT, int D, int NQ, int NP>
hipError_t launch_prefix(const PrefixParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.pre.items + p.own.items)), block(kPrefixWaves * 64);
  if (p.M <= 16)
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, 1, 1>), grid, block, 0, s, p);
  else if (p.R <= 16)
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, 2, 1>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, 2, 2>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_prefix_type(const PrefixParams& p, int head_dim, int parts, hipStream_t s) {
  constexpr int N = DT == kBF16 ? 3 : 2;
  if (head_dim == 64)
    return parts == kPartsOne       ? launch_prefix<DT, 64, 1, 1>(p, s)
           : parts == kPartsWeights ? launch_prefix<DT, 64, 1, N>(p, s)
                                    : launch_prefix<DT, 64, N, N>(p, s);
  return parts == kPartsOne       ? launch_prefix<DT, 128, 1, 1>(p, s)
         : parts == kPartsWeights ? launch_prefix<DT, 128, 1, N>(p, s)
                                  : launch_prefix<DT, 128, N, N>(p, s);
}

}  // namespace
}  // namespace ffai
