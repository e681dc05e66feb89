// Attention of slots over a shared prefix and their own keys (include/ffai_prefix.h), gfx950.
//
// For a query row q with visible keys K_p (its group's prefix) and K_o (its slot's own):
//   o = (sum_p w_j v_j + sum_o w_j v_j) / (sum_p w_j + sum_o w_j),  w_j = 2^(c q.k_j - m),
// c = scale log2(e). Both sums may be cut anywhere: a piece over any set of keys is its own
// (m, l = sum w, O = sum w v), and pieces join by 2^(m_piece - m) (prefix_merge_kernel).
//
// Few tiles: prefix_whole_kernel, whole slots in one launch (below). Otherwise
// prefix_unit_kernel: a workgroup takes one piece of keys and up to 32 query rows that read them
// (128 of the prefix's where there are many: prefix_rows). Prefix pieces come first (the rows of every slot and head of the group that
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

// LDS elements of a wave: its V tiles (two at head_dim 64, see PrefixWave::AHEAD) and 2 KB, and no
// less than the merge area (32 rows of D + 4 floats, then their maxima and sums).
template <int D>
constexpr int kWaveLds = (D == 64 ? 2 : 1) * BN * D + 1024;

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
  int piece;           // index among a row's pieces
};

// Whether a pair of 16-bit values holds an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool not_finite2(uint32_t u) {
  constexpr uint32_t E = DT == kBF16 ? 0x7f80u : 0x7c00u;
  return (u & E) == E || ((u >> 16) & E) == E;
}

// One wave over tiles of 64 keys for 16 NC rows, column 16 c + n16 of the products each.
template <int DT, int D, int NQ, int NP, int NC>
struct PrefixWave {
  static constexpr int CH = D / 8;    // 16-byte chunks of a row
  static constexpr int RB = 64 / CH;  // rows of a 1 KB DMA block
  static constexpr int KC = D / 32;   // contraction chunks of S^T
  static constexpr int OROW = D + 4;  // merge area: rows of O, then maxima, then sums
  static_assert((32 * OROW + 64) * 4 <= kWaveLds<D> * 2, "the merge area fits in the wave's area");
  // The next tile is loaded under the current one, K into the registers that the scores have read, V
  // into a second buffer, where registers and LDS have room for it: at head_dim 64 with 16 rows. (At
  // 128 the buffer would leave room for one workgroup on a CU; two without it stream keys at 5.4 TB/s.)
  static constexpr bool AHEAD = D == 64 && NC == 1;
  static constexpr int VBUF = AHEAD ? BN * D : 0;  // from one V buffer to the other
  static_assert((VBUF + BN * D) * 2 + 32 * 16 * 4 <= kWaveLds<D> * 2, "V tiles and 32 keys' weights");

  uint16_t* base;  // the wave's LDS
  int cur;         // the V buffer of the tile issued last, elements from base
  bool careful;    // look for non-finite V before a product that rows share (always where !AHEAD)
  int lane, q4, n16;
  u32x4 qf[NQ][NC][KC];
  float sl2[NC];  // scores to log2 units
  u32x4 kf[4][KC];
  f32x4 oacc[NC][D / 16];  // O^T: d = 16 db + 4 q4 + r of column 16 c + n16
  float m_s[NC], l_run[NC];

  static __device__ __forceinline__ int swz_v(int r, int c) {
    return D == 64 ? c ^ (4 * ((r >> 1) & 1)) : c ^ (4 * (r & 3));
  }

  __device__ __forceinline__ void init(uint16_t* lds) {
    lane = item_id() & 63;
    q4 = lane >> 4;
    n16 = lane & 15;
    base = lds;
    cur = 0;
    careful = !AHEAD;
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int db = 0; db < D / 16; ++db) oacc[c][db] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_s[c] = kNegInf;
      l_run[c] = 0.f;
    }
  }

  // A tile's loads (k, v: its first key): V by DMA (a lane's 16-byte slot of each 1 KB block gets the
  // chunk that the row's XOR permutation assigns to it), K from memory straight into the A operand's
  // layout (per load 16 rows by 64 bytes). Rows past the last of `valid` keys are not read: the last
  // key's row stands in (their scores are masked, and their V rows cleared below).
  __device__ __forceinline__ void issue(const uint16_t* k, const uint16_t* v, int64_t s_pos,
                                        int valid) {
    const int lr = lane / CH, lc = lane % CH;
    const char* kb = reinterpret_cast<const char*>(k);
    const char* vb = reinterpret_cast<const char*>(v);
    cur ^= VBUF;
    const uint32_t va = lds_addr(base + cur);
#pragma unroll
    for (int kb4 = 0; kb4 < 4; ++kb4) {
      const char* kr = kb + 2 * ((uint32_t)min(16 * kb4 + n16, valid - 1) * (uint32_t)s_pos + 8 * q4);
#pragma unroll
      for (int h = 0; h < KC; ++h) kf[kb4][h] = ld16(kr + 64 * h);
    }
#pragma unroll
    for (int j = 0; j < BN / RB; ++j) {
      const int r = j * RB + lr;
      const uint32_t row = (uint32_t)min(r, valid - 1) * (uint32_t)s_pos;
      if (j * RB < valid) lds_dma16_sbase(vb, 2 * (row + 8 * swz_v(r, lc)), va + j * 1024);
    }
  }

  // Column block c's q from the row at element offset qo.
  __device__ __forceinline__ void load_q(const PrefixParams& p, int c, int64_t qo) {
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

  // The tile that was issued last, `valid` of its keys there; column block c's row sees its keys up to
  // lim[c] (all of the valid ones where `cut` is false). next() issues the tile after it: under this
  // one, or once its V is done with.
  template <class F>
  __device__ __forceinline__ void tile(int valid, bool cut, const int (&lim)[NC], F next) {
    vm_wait_all();
    asm volatile("" ::: "memory");
    uint16_t* vl = base + cur;
    if (valid < BN) {
      // V rows past the last key: a masked weight is 0, but 0 times what lies there need not be
      for (int u = valid * CH + lane; u < BN * CH; u += 64)
        *reinterpret_cast<u32x4*>(&vl[8 * u]) = u32x4{0u, 0u, 0u, 0u};
    }
    // Keys that only some of the rows see may hold a non-finite V, which a weight of 0 would let into
    // the other rows: such a tile takes the slow second product.
    bool slow = false;
    if (cut && careful) {
      bool bad = false;
#pragma unroll 2
      for (int u = lane; u < BN * CH; u += 64) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(&vl[8 * u]);
        bad = bad || not_finite2<DT>(x[0]) || not_finite2<DT>(x[1]) || not_finite2<DT>(x[2]) ||
              not_finite2<DT>(x[3]);
      }
      slow = __ballot(bad) != 0;
    }

    f32x4 s[NC][4];  // S^T: key 16 kb4 + 4 q4 + r of column 16 c + n16
#pragma unroll
    for (int kb4 = 0; kb4 < 4; ++kb4) {
#pragma unroll
      for (int c = 0; c < NC; ++c) s[c][kb4] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < KC; ++h)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int q = NQ - 1; q >= 0; --q)
            s[c][kb4] = mfma16x16<DT>(kf[kb4][h], qf[q][c][h], s[c][kb4]);
    }
    if constexpr (AHEAD) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the other buffer's reads are done
      next();
    }
    if (cut || valid < BN) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int last = cut ? min(lim[c], valid - 1) : valid - 1;
#pragma unroll
        for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * kb4 + 4 * q4 + r > last) s[c][kb4][r] = kNegInf;
      }
    }
    u32x4 pf[NP][NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = kNegInf;
#pragma unroll
      for (int kb4 = 0; kb4 < 4; ++kb4)
        mx = fmaxf(mx, fmaxf(fmaxf(s[c][kb4][0], s[c][kb4][1]), fmaxf(s[c][kb4][2], s[c][kb4][3])));
      const float m_new = fmaxf(m_s[c], quad_max(mx) * sl2[c]);
      const float mc = m_new == kNegInf ? 0.f : m_new;
      const float corr = fast_exp2(m_s[c] - mc);  // 0 while nothing is seen
      m_s[c] = m_new;
      float rs = 0.f;
#pragma unroll
      for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[c][kb4][r] = fast_exp2(__builtin_fmaf(s[c][kb4][r], sl2[c], -mc));
          rs += s[c][kb4][r];
        }
      l_run[c] = __builtin_fmaf(l_run[c], corr, rs);
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
      for (int db = 0; db < D / 16; ++db) oacc[c][db] *= corr;
    }
    if (!slow) {
      const int tr_row = n16 >> 2, tr_col = 4 * (n16 & 3);
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          const int r = 32 * ch + 4 * q4 + tr_row, col = 16 * db + tr_col;
          const uint16_t* at = &vl[r * D + 8 * swz_v(r, col >> 3) + (col & 7)];
          const u32x2 a0 = lds_tr(at), a1 = lds_tr(at + 16 * D);
          const u32x4 a = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int q = NP - 1; q >= 0; --q) oacc[c][db] = mfma16x16<DT>(a, pf[q][c][ch], oacc[c][db]);
        }
    } else {
      // key by key, only where the row sees it (the weights through LDS, 32 keys of 16 columns at a
      // time)
      float* pl = reinterpret_cast<float*>(base + VBUF + BN * D);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              pl[(16 * k2 + 4 * q4 + r) * 16 + n16] = s[c][2 * ch + k2][r];
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
          for (int key = 32 * ch; key < min(32 * ch + 32, valid); ++key) {
            const float wt = pl[(key & 31) * 16 + n16];
            const bool seen = key <= lim[c];
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
          asm volatile("" ::: "memory");
        }
    }
    if constexpr (!AHEAD) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this tile's V reads are done
      next();
    }
  }

  // Whether every result so far is finite (AHEAD: its registers allow a second go). A row that shares
  // a tile with a non-finite V that it does not see is not: then the wave starts again, carefully.
  // Results that are rightly non-finite come out the same from the second go.
  __device__ __forceinline__ bool finite() const {
    bool bad = false;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          bad = bad || (__float_as_uint(oacc[c][db][r]) & 0x7f800000u) == 0x7f800000u;
    return __ballot(bad) == 0;
  }

  // The wave's result to its merge area (after a barrier: tiles are done with).
  __device__ __forceinline__ void leave(float* mb, int rows) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float l = quad_sum(l_run[c]);
      const int n = 16 * c + n16;
      if (n < rows) {
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
  // Row n's elements 4 c4 .. +3 joined over NW waves' areas (WST floats apart).
  template <int NW>
  static __device__ __forceinline__ f32x4 join(const float* mbase, int n, int c4, float* M_,
                                               float* L_) {
    constexpr int WST = kWaveLds<D> / 2;
    float mw[NW], M = kNegInf;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      mw[x] = mbase[x * WST + 32 * OROW + n];
      M = fmaxf(M, mw[x]);
    }
    const float Mc = M == kNegInf ? 0.f : M;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float* mb = mbase + x * WST;
      const float wt = fast_exp2(mw[x] - Mc);
      acc += wt * *reinterpret_cast<const f32x4*>(&mb[n * OROW + 4 * c4]);
      L = __builtin_fmaf(wt, mb[32 * OROW + 32 + n], L);
    }
    *M_ = M;
    *L_ = L;
    return acc;
  }
};

// Element offset of q's (or out's) row rr of a slot's rows that read K/V head h.
__device__ __forceinline__ int64_t row_offset(const PrefixParams& p, int64_t ss, int64_t sh,
                                              int64_t st, int slot, int h, int rr) {
  const int hh = rr / p.T, t = rr - hh * p.T;
  return (int64_t)slot * ss + (int64_t)(h * p.rep + hh) * sh + (int64_t)t * st;
}

// A piece of keys for a block of rows: the waves take its tiles in turn and leave one partial.
template <int DT, int D, int NQ, int NP, int NC>
__device__ __forceinline__ void prefix_work(const PrefixParams& p, const PrefixWork& w,
                                            uint16_t* lds) {
  constexpr int NWD = kPrefixWaves;
  using Wave = PrefixWave<DT, D, NQ, NP, NC>;
  const int tid = item_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Wave x;
  x.init(lds + wave * kWaveLds<D>);
  auto issue = [&](int it) {
    const int64_t at = (int64_t)it * BN * w.s_pos;
    x.issue(w.k + at, w.v + at, w.s_pos, min(BN, w.n_keys - it * BN));
  };
  // the first tile's loads go out before anything else
  if (w.t_begin + wave < w.t_end) issue(w.t_begin + wave);
  // column 16 c + n16 is row r0 + that (past the last row: the last row again; such a column's
  // results are not stored)
  int see[NC];  // the last key the column's row sees
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = w.r0 + min(16 * c + x.n16, w.rows - 1);
    const int ds = r / p.R, rr = r - ds * p.R;
    see[c] = w.causal_last + rr % p.T;
    x.load_q(p, c, row_offset(p, p.q_ss, p.q_sh, p.q_st, w.slot0 + ds, w.h, rr));
  }
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int it = w.t_begin + wave; it < w.t_end; it += NWD) {
      const int kb = it * BN;
      int lim[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) lim[c] = see[c] - kb;
      // (one query token sees every key of the sequence)
      x.tile(min(BN, w.n_keys - kb), p.T > 1 && kb + BN - 1 > w.causal_last, lim, [&] {
        if (it + NWD < w.t_end) issue(it + NWD);
      });
    }
    if (!Wave::AHEAD || p.T == 1 || x.careful || x.finite()) break;
    x.clear();
    x.careful = true;
    if (w.t_begin + wave < w.t_end) issue(w.t_begin + wave);
  }
  // ---- the waves' results meet in LDS (each wave's area is free once all pass here)
  __syncthreads();
  float* mbase = reinterpret_cast<float*>(lds);
  x.leave(mbase + wave * (kWaveLds<D> / 2), w.rows);
  __syncthreads();
  constexpr int C4 = D / 4;
  const int np = p.pre.pieces + p.own.pieces;
#pragma unroll 1
  for (int i = tid; i < w.rows * C4; i += NWD * 64) {
    const int n = i / C4, c4 = i % C4;
    float M, L;
    const f32x4 acc = Wave::template join<NWD>(mbase, n, c4, &M, &L);
    const int r = w.r0 + n, ds = r / p.R, rr = r - ds * p.R;
    const int64_t row = ((int64_t)(w.slot0 + ds) * p.Hkv + w.h) * p.R + rr;
    const int64_t at = row * np + w.piece;
    *reinterpret_cast<f32x4*>(p.part + at * D + 4 * c4) = acc;
    if (c4 == 0) *reinterpret_cast<f32x2*>(p.ml + at * 2) = f32x2{M, L};
  }
}

// Short sequences, one launch and no partials: a workgroup takes a few slots of a group (their rows
// are the columns, whole slots only) with everything they see of one K/V head: the prefix's tiles,
// then each slot's own, dealt to the eight waves in turn. A slot's own tile is masked for the other
// slots' columns. Bound by
// the chain of a few tiles a wave (~2 us each) and the join.
template <int DT, int D, int NQ, int NP, int NC, int OUTT>
__global__ __launch_bounds__(kWholeWaves * 64, 2) void prefix_whole_kernel(PrefixParams p) {
  constexpr int NWD = kWholeWaves;
  using Wave = PrefixWave<DT, D, NQ, NP, NC>;
  extern __shared__ __attribute__((aligned(16))) uint16_t whole_lds[];
  const int tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int item = wg_id_x();
  const int h = item % p.Hkv;
  item /= p.Hkv;
  const int blocks = p.pre.row_blocks;  // of a group's slots, p.block_slots each
  const int group = item / blocks, s0 = (item - group * blocks) * p.block_slots;
  const int slots = min(p.block_slots, p.per - s0), slot0 = group * p.per + s0;
  const int rows = slots * p.R;

  // lane l: slot l's own length, and the tiles up to and with it (after the prefix's)
  const int n_pre = __builtin_amdgcn_readfirstlane(min(max(p.pre.lens[group], 0), p.pre.capacity));
  const int len = lane < slots ? min(max(p.own.lens[slot0 + lane], 0), p.own.capacity) : 0;
  const int t_pre = (n_pre + BN - 1) / BN;
  int upto = (len + BN - 1) / BN;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  upto += t_pre;
  const int tiles = __builtin_amdgcn_readfirstlane(__shfl(upto, 31));

  Wave x;
  x.init(whole_lds + wave * kWaveLds<D>);
  // where tile `it` lies: its slot among the block's (-1: the prefix), its first key, its keys
  int t_slot = -1, t_kb = 0, t_len = 0;
  auto issue = [&](int it) {
    if (it < t_pre) {
      t_slot = -1;
      t_kb = it * BN;
      t_len = n_pre;
      const int64_t at = (int64_t)group * p.pre.s_slot + (int64_t)h * p.pre.s_head + (int64_t)t_kb * p.pre.s_pos;
      x.issue(reinterpret_cast<const uint16_t*>(p.pre.k) + at,
              reinterpret_cast<const uint16_t*>(p.pre.v) + at, p.pre.s_pos, min(BN, t_len - t_kb));
    } else {
      t_slot = __builtin_ctzll(__ballot(lane < slots && it < upto));
      const int before = t_slot == 0 ? t_pre : __builtin_amdgcn_readfirstlane(__shfl(upto, max(t_slot - 1, 0)));
      t_kb = (it - before) * BN;
      t_len = __builtin_amdgcn_readfirstlane(__shfl(len, t_slot));
      const int64_t at = (int64_t)(slot0 + t_slot) * p.own.s_slot + (int64_t)h * p.own.s_head + (int64_t)t_kb * p.own.s_pos;
      x.issue(reinterpret_cast<const uint16_t*>(p.own.k) + at,
              reinterpret_cast<const uint16_t*>(p.own.v) + at, p.own.s_pos, min(BN, t_len - t_kb));
    }
  };
  if (wave < tiles) issue(wave);
  int my_slot[NC], my_t[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = min(16 * c + x.n16, rows - 1);
    my_slot[c] = r / p.R;
    const int rr = r - my_slot[c] * p.R;
    my_t[c] = rr % p.T;
    x.load_q(p, c, row_offset(p, p.q_ss, p.q_sh, p.q_st, slot0 + my_slot[c], h, rr));
  }
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int it = wave; it < tiles; it += NWD) {
      int lim[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c)
        lim[c] = my_slot[c] == t_slot ? t_len - p.T + my_t[c] - t_kb : -1;
      const bool cut = t_slot >= 0 && (slots > 1 || (p.T > 1 && t_kb + BN - 1 > t_len - p.T));
      x.tile(min(BN, t_len - t_kb), cut, lim, [&] {
        if (it + NWD < tiles) issue(it + NWD);
      });
    }
    if (!Wave::AHEAD || x.careful || x.finite()) break;
    x.clear();
    x.careful = true;
    if (wave < tiles) issue(wave);
  }
  __syncthreads();
  float* mbase = reinterpret_cast<float*>(whole_lds);
  x.leave(mbase + wave * (kWaveLds<D> / 2), rows);
  __syncthreads();
  constexpr int C4 = D / 4;
#pragma unroll 1
  for (int i = tid; i < rows * C4; i += NWD * 64) {
    const int n = i / C4, c4 = i % C4;
    float M, L;
    const f32x4 acc = Wave::template join<NWD>(mbase, n, c4, &M, &L);
    // (the sum's bits are tested: a NaN sum must reach the output, not become an empty row)
    const float inv = (__float_as_uint(L) & 0x7fffffffu) == 0 ? 0.f : 1.f / L;
    const int ds = n / p.R, rr = n - ds * p.R;
    store_t<OUTT>* o = reinterpret_cast<store_t<OUTT>*>(p.out) +
                       row_offset(p, p.o_ss, p.o_sh, p.o_st, slot0 + ds, h, rr) + 4 * c4;
    st4<OUTT>(o, acc * inv);
  }
}

// Many rows over one piece of a prefix: 128 rows a workgroup, 32 a wave, over tiles that the waves
// share. A tile's K and V come by DMA into one of two buffers while the other is worked on; one
// barrier a tile says that the next one's loads have landed and that every wave has read the buffer
// they are followed by. Products on 32x32x16 MFMA: S^T (A: 32 keys, B: the wave's 32 rows as
// columns), and O^T with P^T as it lies in S^T's layout: lane half hb holds keys 8 j + 4 hb + r of
// a 32-key block, so contraction chunk cc takes slots 4 hb + e (e < 4) and 8 + 4 hb + e - 4 of its 16
// keys, and V is read transposed in that order. Bound by LDS reads and MFMA alike (32 KB of K and V
// a wave and 2 MFLOP at head_dim 128: 1024 clocks of a CU's LDS for four waves, as many of each
// SIMD's matrix core), and by the softmax between them.
template <int DT, int D, int NQ, int NP>
__device__ __forceinline__ void prefix_rows(const PrefixParams& p, const PrefixWork& w,
                                            uint16_t* lds) {
  constexpr int NWD = kPrefixWaves;
  constexpr int TILE = BN * D;
  constexpr int CH = D / 8, RB = 64 / CH;
  constexpr int PB = BN / RB / NWD;  // 1 KB blocks of K (and of V) a wave loads
  constexpr int KC = D / 16;
  const int tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hb = lane >> 5, n32 = lane & 31, n16 = lane & 15;
  auto swz_k = [](int r, int c) { return D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15); };
  auto swz_v = [](int r, int c) { return D == 64 ? c ^ (4 * ((r >> 1) & 1)) : c ^ (4 * (r & 3)); };
  const int lr = lane / CH, lc = lane % CH;
  auto issue = [&](int it, int buf) {
    const int valid = min(BN, w.n_keys - it * BN);
    const char* kb = reinterpret_cast<const char*>(w.k + (int64_t)it * BN * w.s_pos);
    const char* vb = reinterpret_cast<const char*>(w.v + (int64_t)it * BN * w.s_pos);
    const uint32_t ka = lds_addr(lds) + buf * (4 * TILE), va = ka + 2 * TILE;
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      const int jb = wave * PB + j, r = jb * RB + lr;
      const uint32_t row = (uint32_t)min(r, valid - 1) * (uint32_t)w.s_pos;
      lds_dma16_sbase(kb, 2 * (row + 8 * swz_k(r, lc)), ka + jb * 1024);
      lds_dma16_sbase(vb, 2 * (row + 8 * swz_v(r, lc)), va + jb * 1024);
    }
  };
  if (w.t_begin < w.t_end) issue(w.t_begin, 0);

  const bool on = 32 * wave < w.rows;  // the wave has rows (wave-uniform)
  u32x4 qf[NQ][KC];
  float sl2 = p.scale_log2;
  const int r = w.r0 + min(32 * wave + n32, w.rows - 1);
  const int ds = r / p.R, rr = r - ds * p.R;
  {
    const int hh = rr / p.T, t = rr - hh * p.T;
    const int64_t qo = (int64_t)(w.slot0 + ds) * p.q_ss + (int64_t)(w.h * p.rep + hh) * p.q_sh +
                       (int64_t)t * p.q_st;
    if constexpr (NQ == 1) {
#pragma unroll
      for (int h = 0; h < KC; ++h)
        qf[0][h] = ld16h(reinterpret_cast<const uint16_t*>(p.q) + qo + 16 * h + 8 * hb);
    } else {
      const float* qr = reinterpret_cast<const float*>(p.q) + qo;
      float sc = 1.f;
      if constexpr (DT == kF16) {
        float mx = 0.f;
#pragma unroll
        for (int h = 0; h < KC; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const f32x4 a = *reinterpret_cast<const f32x4_e*>(qr + 16 * h + 8 * hb + 4 * e);
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(a[0]), fabsf(a[1])), fmaxf(fabsf(a[2]), fabsf(a[3]))));
          }
        mx = partner_max(mx);
        const int sb = min(max(268 - (int)(__float_as_uint(mx) >> 23), 1), 253);
        sc = __uint_as_float((uint32_t)sb << 23);
        sl2 *= __uint_as_float((uint32_t)(254 - sb) << 23);
      }
#pragma unroll
      for (int h = 0; h < KC; ++h) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 a = *reinterpret_cast<const f32x4_e*>(qr + 16 * h + 8 * hb + 4 * e);
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            float x0 = a[2 * e2] * sc, x1 = a[2 * e2 + 1] * sc;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              const uint32_t pk = pack2<DT>(x0, x1);
              qf[q][h][2 * e + e2] = pk;
              const float h0 = to_f32<DT>(pk & 0xffffu), h1 = to_f32<DT>(pk >> 16);
              x0 = fabsf(h0) < __builtin_inff() ? x0 - h0 : 0.f;
              x1 = fabsf(h1) < __builtin_inff() ? x1 - h1 : 0.f;
            }
          }
        }
      }
    }
  }
  f32x16 oacc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  float m_s = kNegInf, l_run = 0.f;

  int buf = 0;
#pragma unroll 1
  for (int it = w.t_begin; it < w.t_end; ++it, buf ^= 1) {
    const int kb = it * BN;
    uint16_t* kl = lds + buf * (2 * TILE);
    uint16_t* vl = kl + TILE;
    asm volatile("" ::: "memory");
    vm_wait_all();
    asm volatile("" ::: "memory");
    if (kb + BN > w.n_keys) {
      // V rows past the last key, each by the wave that loaded it
      for (int u = lane; u < PB * 64; u += 64) {
        const int row = wave * PB * RB + u / CH;
        if (row >= w.n_keys - kb)
          *reinterpret_cast<u32x4*>(&vl[(wave * PB * 64 + u) * 8]) = u32x4{0u, 0u, 0u, 0u};
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (it + 1 < w.t_end) issue(it + 1, buf ^ 1);
    if (!on) continue;

    f32x16 s[2];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[k2][e] = 0.f;
      const int row = 32 * k2 + n32;
#pragma unroll
      for (int h = 0; h < KC; ++h) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(&kl[row * D + 8 * swz_k(row, 2 * h + hb)]);
#pragma unroll
        for (int q = NQ - 1; q >= 0; --q) s[k2] = mfma16<DT>(a, qf[q][h], s[k2]);
      }
    }
    if (kb + BN > w.n_keys) {
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (kb + 32 * k2 + 8 * (e >> 2) + 4 * hb + (e & 3) >= w.n_keys) s[k2][e] = kNegInf;
    }
    float mx = kNegInf;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[k2][e]);
    const float m_new = fmaxf(m_s, partner_max(mx) * sl2);
    const float mc = m_new == kNegInf ? 0.f : m_new;
    const float corr = fast_exp2(m_s - mc);
    float rs = 0.f;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[k2][e] = fast_exp2(__builtin_fmaf(s[k2][e], sl2, -mc));
        rs += s[k2][e];
      }
    l_run = __builtin_fmaf(l_run, corr, rs);
    // (the running maximum settles after a few tiles: then nothing is scaled)
    if (__ballot(m_new != m_s)) {
#pragma unroll
      for (int db = 0; db < D / 32; ++db) oacc[db] *= corr;
    }
    m_s = m_new;
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
      u32x4 pf[NP];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x0 = s[cc >> 1][8 * (cc & 1) + 2 * k], x1 = s[cc >> 1][8 * (cc & 1) + 2 * k + 1];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const uint32_t pk = pack2<DT>(x0, x1);
          pf[q][k] = pk;
          x0 -= to_f32<DT>(pk & 0xffffu);
          x1 -= to_f32<DT>(pk >> 16);
        }
      }
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        const int row = 16 * cc + 4 * hb + (n16 >> 2);
        const int col = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (n16 & 3);
        const u32x2 a0 = lds_tr(&vl[row * D + 8 * swz_v(row, col >> 3) + (col & 7)]);
        const u32x2 a1 = lds_tr(&vl[(row + 8) * D + 8 * swz_v(row + 8, col >> 3) + (col & 7)]);
        const u32x4 a = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
        for (int q = NP - 1; q >= 0; --q) oacc[db] = mfma16<DT>(a, pf[q], oacc[db]);
      }
    }
  }
  const float l = partner_sum(l_run);
  if (on && 32 * wave + n32 < w.rows) {
    const int64_t row = ((int64_t)(w.slot0 + ds) * p.Hkv + w.h) * p.R + rr;
    const int64_t at = row * (p.pre.pieces + p.own.pieces) + w.piece;
    float* o = p.part + at * D;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = oacc[db][4 * j + e];
        *reinterpret_cast<f32x4*>(o + 32 * db + 8 * j + 4 * hb) = x;
      }
    if (hb == 0) *reinterpret_cast<f32x2*>(p.ml + at * 2) = f32x2{m_s, l};
  }
}

// ROWS: the prefix's pieces run as prefix_rows (many rows), else as prefix_work in blocks of 16 NCP
// rows; the own pieces always as prefix_work. The prefix's come first in the grid, one a CU where they
// are prefix_rows: the own ones then stream beside them. 128 slots x 32 heads, 16384 shared and 33 to
// 1024 own keys 95 us, of which the merge 6.
template <int DT, int D, int NQ, int NP, int NCP, int NCO, bool ROWS>
__global__ __launch_bounds__(kPrefixWaves * 64, NQ > 1 && (NCP > 1 || NCO > 1 || D == 128) ? 1 : 2) void
prefix_unit_kernel(PrefixParams p) {
  constexpr int LDS = kPrefixWaves * kWaveLds<D>;
  static_assert(!ROWS || LDS >= 4 * BN * D, "two tiles of K and V fit");
  __shared__ __attribute__((aligned(16))) uint16_t lds[LDS];
  int item = wg_id_x();
  const bool pre = item < p.pre.items;
  if (!pre) item -= p.pre.items;
  const PrefixSide& sd = pre ? p.pre : p.own;
  PrefixWork w;
  const int piece = item % sd.pieces;
  item /= sd.pieces;
  w.h = item % p.Hkv;
  item /= p.Hkv;
  const int rb = item % sd.row_blocks;
  const int slot = item / sd.row_blocks;
  w.piece = pre ? piece : p.pre.pieces + piece;
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
  w.causal_last = pre ? 0x3fffffff : w.n_keys - p.T;
  const int block = ROWS && pre ? kPrefixManyRows : prefix_row_block(D);
  w.r0 = rb * block;
  w.rows = min(block, (pre ? p.M : p.R) - w.r0);
  if constexpr (ROWS) {
    if (pre) prefix_rows<DT, D, NQ, NP>(p, w, lds);
    else prefix_work<DT, D, NQ, NP, NCO>(p, w, lds);
  } else if constexpr (NCP == NCO) {
    prefix_work<DT, D, NQ, NP, NCP>(p, w, lds);
  } else {
    if (pre) prefix_work<DT, D, NQ, NP, NCP>(p, w, lds);
    else prefix_work<DT, D, NQ, NP, NCO>(p, w, lds);
  }
}

template <int DT, int D, int NQ, int NP>
hipError_t launch_prefix(const PrefixParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.pre.items + p.own.items)), block(kPrefixWaves * 64);
  // 16-column blocks of rows on either side, one or two (head_dim 128: one, prefix_row_block)
  constexpr int NC = prefix_row_block(D) / 16;
  if (p.many && p.R <= 16)
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, 1, 1, true>), grid, block, 0, s, p);
  else if (p.many)
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, NC, NC, true>), grid, block, 0, s, p);
  else if (p.M <= 16)
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, 1, 1, false>), grid, block, 0, s, p);
  else if (p.R <= 16)
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, NC, 1, false>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((prefix_unit_kernel<DT, D, NQ, NP, NC, NC, false>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <int DT, int D, int NQ, int NP, int NC, int OUTT>
hipError_t launch_whole(const PrefixParams& p, int groups, hipStream_t s) {
  constexpr int lds = kWholeWaves * kWaveLds<D> * 2;
  auto kernel = prefix_whole_kernel<DT, D, NQ, NP, NC, OUTT>;
  static const hipError_t once = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (once != hipSuccess) return once;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(groups * p.pre.row_blocks * p.Hkv)),
                     dim3(kWholeWaves * 64), lds, s, p);
  return hipGetLastError();
}
template <int DT, int D, int NQ, int NP, int OUTT>
hipError_t launch_whole_rows(const PrefixParams& p, int groups, hipStream_t s) {
  if constexpr (prefix_row_block(D) == 32) {
    if (p.block_slots * p.R > 16) return launch_whole<DT, D, NQ, NP, 2, OUTT>(p, groups, s);
  }
  return launch_whole<DT, D, NQ, NP, 1, OUTT>(p, groups, s);
}
template <int DT>
hipError_t launch_whole_type(const PrefixParams& p, int groups, int head_dim, int parts,
                             hipStream_t s) {
  constexpr int N = DT == kBF16 ? 3 : 2;
  if (head_dim == 64)
    return parts == kPartsOne       ? launch_whole_rows<DT, 64, 1, 1, DT>(p, groups, s)
           : parts == kPartsWeights ? launch_whole_rows<DT, 64, 1, N, kF32>(p, groups, s)
                                    : launch_whole_rows<DT, 64, N, N, kF32>(p, groups, s);
  return parts == kPartsOne       ? launch_whole_rows<DT, 128, 1, 1, DT>(p, groups, s)
         : parts == kPartsWeights ? launch_whole_rows<DT, 128, 1, N, kF32>(p, groups, s)
                                  : launch_whole_rows<DT, 128, N, N, kF32>(p, groups, s);
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
