// Sampling of one token per row of logits (include/ffai_sample.h).
//
// One launch for small vocabularies; else two, three where a row may filter, four where it may by
// weight:
//   * sample_small_kernel, up to 8192 tokens (16384 with filters): all of it, a row in registers;
//   * sample_scan_kernel reads the logits, spread over the whole GPU: of every 1024 elements (a
//     wave's) the maximum, those of its quads of lanes, and the weights' sum;
//   * sample_gather_kernel: nearly always few tokens can be kept. The k-th largest group maximum
//     bounds the k-th largest logit from below, so a second spread pass lists everything from there
//     up (k and a few tokens more). Beside that, where there is no k: min_p's kept weight of each
//     group, and for a nucleus a histogram of weights;
//   * sample_spread_kernel, only where the list does not settle a nucleus: the bins that the limit
//     lies in are listed, the weights above them summed by group;
//   * sample_pick_kernel, one workgroup a row, finds the token. No filter, or min_p alone: the group
//     that holds u W by a scan of the groups' sums, then the token in it, an element a thread.
//     Filters: the list is ordered in LDS and the definition applied as it stands; a nucleus' bins
//     likewise, and then its token by the groups' sums. Where neither holds what can be kept
//     (top_k above 256, thousands of equal tokens) the workgroup finds the boundary by histograms of
//     counts or weights over the row, finer each time, down to a list or a single value.
// Weights are 64-bit throughout: a token's share may be 1e-5 of the row's, and with f32 sums the
// token at a given u would depend on the order of summation. f64 FMAs run at the f32 rate here;
// an exponential is 18 instructions. Only a histogram's weights are less (integers of f32
// exponentials: adding them in any order gives the same sum), and what they decide is confirmed
// with f64 sums.
//
// Few rows are bound by the launches and their chains of loads: 5 x 51865 f32 at a temperature
// 12 us, 64 x 51865 with top-k and top-p 26, one row of 51865 top-k 18, top-p over thousands of
// tokens 45 (81 with the histograms in the picking workgroup alone); 12 x 1906 top-k in one launch 17
// (56 in three), 26 x 1182 top-p 25 (44 in four). Many rows by instructions: 256 x
// 131072 bf16, settings of each row's own, 126 us (235): the scan 32, the gather 36, the nuclei's
// spread 32, the pick 27. The spread costs rows that need none 2 to 3 us.
#include "../../include/ffai_sample.h"

#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"

namespace ffai {
namespace {

constexpr int kGroup = 1024;  // elements whose maximum and sums a scan wave leaves
constexpr int kMaxVocab = 1 << 20;
constexpr int kPick = 1024;   // threads of a pick workgroup
constexpr int kWaves = kPick / 64;
constexpr int kSpread = 512;  // threads of a spread workgroup
constexpr int kShort = 256;   // tokens of a list that one wave finishes
constexpr int kList = 2048;   // tokens of an LDS list
constexpr int kBins = 4096;
constexpr int kChunk = 4096;  // elements of a gather workgroup's share
constexpr int kParts = 16;    // gather workgroups of a row, about
constexpr int kCutBins = 2048;  // bins of a nucleus' histogram
constexpr int kHeld = 1024;   // maxima that bound a list, at most
constexpr int kAhead = 4;     // steps of a pass over a row that a wave loads ahead

struct SampleParams {
  const void* logits;
  int64_t ls;
  int32_t rows, vocab, groups, chunks;
  const float* t;
  const int32_t* k;
  const float* p;
  const float* mp;
  float t_all, p_all, mp_all;
  int32_t k_all;
  const float* u;
  int32_t* tok;
  float* lp;
  double* sum_t;   // [row][group] sum of exp((l - group max) / T)
  double* sum_1;   // [row][group] sum of exp(l - group max)
  float* gmax;     // [row][group] maxima
  float* smax;     // [row][group][16] of the group's quads of lanes
  float* low;      // [row] the least logit that is listed; -inf: no list
  int32_t* count;  // [row][chunk] listed tokens (kShort at most are held)
  uint64_t* cand;  // [row][chunk][kShort] their ranks, in no order
  int32_t per, parts;  // chunks of a gather workgroup, and such workgroups of a row
  uint32_t* hist;   // [row][part][kCutBins] nuclei: weights by distance from the maximum
  double* sum_k;    // [row][group] minima: sum of the weights >= min_p
  double* sum_a;    // [row][group] nuclei: sum of the weights above the boundary's bins
  int32_t* count2;  // [row][chunk] tokens in the boundary's bins (kShort at most are held)
  uint64_t* cand2;  // [row][chunk][kShort] their ranks, in no order
  int32_t* cut;     // [row] nuclei that the list does not settle: whether the boundary's bins are listed
};

// The device code is compiled for numbers that are not NaN, so NaN is recognised by its bits, and
// NaN logits become -inf by an instruction (max of a NaN and a number is the number).
__device__ __forceinline__ bool is_nan(float x) {
  return (__float_as_uint(x) & 0x7fffffffu) > 0x7f800000u;
}
__device__ __forceinline__ float nan_to_low(float x) {
  float r;
  asm("v_max_f32 %0, 0xff800000, %1" : "=v"(r) : "v"(x));
  return r;
}

constexpr double kLog2e = 1.4426950408889634074;

struct RowSettings {
  bool greedy;
  double inv2;  // log2(e) / T
  bool t1;      // T is 1
  int k;        // 0: off
  float p;      // 1: off
  double mp;    // 0: off
  __device__ __forceinline__ bool filtered() const { return k > 0 || p < 1.f || mp > 0.0; }
};
__device__ __forceinline__ RowSettings settings(const SampleParams& p, int row) {
  RowSettings s;
  const float t = p.t ? p.t[row] : p.t_all;
  const uint32_t tb = __float_as_uint(t);
  s.greedy = !(tb > 0u && tb <= 0x7f800000u);  // positive, infinity included
  s.inv2 = __builtin_fmax(kLog2e / (double)t, 1e-300);  // (T = inf: -inf times it stays -inf)
  s.t1 = t == 1.f;
  const int k = p.k ? p.k[row] : p.k_all;
  s.k = k <= 0 || k >= p.vocab ? 0 : k;
  const float tp = p.p ? p.p[row] : p.p_all;
  s.p = is_nan(tp) || tp >= 1.f ? 1.f : tp;
  const float mp = p.mp ? p.mp[row] : p.mp_all;
  s.mp = is_nan(mp) || mp <= 0.f ? 0.0 : (double)fminf(mp, 1.f);
  return s;
}

// a b + c with c in scalar registers: one instruction. (The compiler's choice is an accumulating
// form that first copies c to vector registers, two instructions a term.)
__device__ __forceinline__ double fma_const(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}
// 2^y, y <= 0 (0 below -1000): 2^n times 2^f, n the whole number nearest to y, |f| <= 1/2 by the
// polynomial of degree 10 that equals it at the Chebyshev points (relative error below 3e-16; exactly
// 1 at 0). n comes as the low bits of y + 1.5 2^52, and goes into the exponent field: additions and
// FMAs, which run at the f32 rate. A weight's exponent carries the rounding of its own product,
// about |y| 2^-53: 1e-14 at most where it counts.
__device__ __forceinline__ double exp2_neg(double y) {
  constexpr double kMagic = 0x1.8p52;
  const double t = y + kMagic;
  const double f = y - (t - kMagic);
  double e = 0x1.e6063f7217bc6p-28;
  e = fma_const(e, f, 0x1.b675bca4eeebbp-24);
  e = fma_const(e, f, 0x1.62bfd47773353p-20);
  e = fma_const(e, f, 0x1.ffcb54062e698p-17);
  e = fma_const(e, f, 0x1.430913096fd9fp-13);
  e = fma_const(e, f, 0x1.5d87fe9d7a584p-10);
  e = fma_const(e, f, 0x1.3b2ab6fba1ddap-7);
  e = fma_const(e, f, 0x1.c6b08d703ce49p-5);
  e = fma_const(e, f, 0x1.ebfbdff82c598p-3);
  e = fma_const(e, f, 0x1.62e42fefa3a19p-1);
  e = __builtin_fma(e, f, 1.0);
  const uint64_t eb = __builtin_bit_cast(uint64_t, e), tb = __builtin_bit_cast(uint64_t, t);
  const uint32_t hi = (uint32_t)(eb >> 32) + ((uint32_t)tb << 20);
  // (negative numbers: the larger the bits, the lower the number; -inf too)
  const bool under = (uint32_t)(__builtin_bit_cast(uint64_t, y) >> 32) > 0xc08f4000u;
  const uint64_t r = ((uint64_t)(under ? 0u : hi) << 32) | (under ? 0u : (uint32_t)eb);
  return __builtin_bit_cast(double, r);
}
// A token's weight against the largest logit m (l <= m): 1 at m even where both are infinite.
__device__ __forceinline__ double weight(float l, float m, double inv2) {
  if (m == __builtin_inff()) return l >= m ? 1.0 : 0.0;  // uniform
  return exp2_neg(((double)l - (double)m) * inv2);
}

template <int DT>
__device__ __forceinline__ float load1(const store_t<DT>* x, int i) {
  if constexpr (DT == kF32) return nan_to_low(x[i]);
  else return nan_to_low(to_f32<DT>(x[i]));
}
// EPL consecutive logits from index i of a row of n (TINY: n < EPL); -inf from index `end` on. Loads
// have no branch: the address is clamped into the row, and a step that reaches past `end` puts its
// elements right afterwards (`fix`). A load on one side of a branch makes the compiler wait for all
// loads at the join: a pass over a row then had one step's loads in flight, 1.2 us a step.
template <int DT, bool TINY>
struct Lane {
  static constexpr int EPL = DT == kF32 ? 4 : 8;
  using S = store_t<DT>;
  float v[EPL];
  static __device__ __forceinline__ u32x4 raw(const S* x, int i, int n) {
    if constexpr (!TINY) {
      return ld16h(x + min(i, n - EPL));
    } else {
      u32x4 r = {0u, 0u, 0u, 0u};
      for (int e = 0; e < n; ++e) put(r, e, x[e]);
      return r;
    }
  }
  static __device__ __forceinline__ void put(u32x4& r, int e, S b) {
#pragma unroll
    for (int q = 0; q < EPL; ++q)
      if (q == e) {
        if constexpr (DT == kF32) r[q] = __float_as_uint(b);
        else r[q >> 1] = (q & 1) ? (r[q >> 1] & 0xffffu) | ((uint32_t)b << 16)
                                 : (r[q >> 1] & 0xffff0000u) | (uint32_t)b;
      }
  }
  // what raw(x, i, n) loaded, its elements at their places and -inf from `end` on
  static __device__ __forceinline__ u32x4 fix(u32x4 r, int i, int n, int end) {
    constexpr uint32_t LOW = DT == kF32 ? 0xff800000u : DT == kF16 ? 0xfc00u : 0xff80u;
    const int by = TINY ? 0 : i - min(i, n - EPL);  // places the load began too early
    u32x4 o = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      uint32_t b = LOW;
#pragma unroll
      for (int q = 0; q < EPL; ++q) {
        const uint32_t w = DT == kF32 ? r[q & 3] : (q & 1) ? r[q >> 1] >> 16 : r[q >> 1] & 0xffffu;
        if (q == e + by && i + e < end) b = w;
      }
      if constexpr (DT == kF32) o[e & 3] = b;
      else o[e >> 1] |= b << (16 * (e & 1));
    }
    return o;
  }
  static __device__ __forceinline__ float value(const u32x4& r, int e) {
    if constexpr (DT == kF32) return nan_to_low(__uint_as_float(r[e]));
    else return nan_to_low(to_f32<DT>((e & 1) ? r[e >> 1] >> 16 : r[e >> 1] & 0xffffu));
  }
  // `last`: the wave's last element, plus one
  __device__ __forceinline__ void take(u32x4 r, int i, int n, int end, int last) {
    if (TINY || last > end) r = fix(r, i, n, end);  // uniform
#pragma unroll
    for (int e = 0; e < EPL; ++e) v[e] = value(r, e);
  }
};

template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v += __shfl_xor(v, s);
  return v;
}
// Exclusive prefix sum over the wave's lanes, and the whole sum.
__device__ __forceinline__ double wave_scan(double v, double* total) {
  const int lane = item_id() & 63;
  double x = v;
#pragma unroll
  for (int s = 1; s < 64; s *= 2) {
    const double y = __shfl_up(x, s);
    if (lane >= s) x += y;
  }
  *total = __shfl(x, 63);
  const double e = __shfl_up(x, 1);
  return lane == 0 ? 0.0 : e;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v = min(v, __shfl_xor(v, s));
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v = max(v, __shfl_xor(v, s));
  return v;
}

// ---- scan --------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void sample_scan_kernel(SampleParams p) {
  constexpr int EPL = Lane<DT, false>::EPL, IT = kGroup / (64 * EPL);
  const int row = wg_id_y(), lane = item_id() & 63;
  const int group = __builtin_amdgcn_readfirstlane(wg_id_x() * 4 + (item_id() >> 6));
  if (group >= p.groups) return;
  const store_t<DT>* x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)row * p.ls;
  const int base = group * kGroup + lane * EPL;
  const int end = min((group + 1) * kGroup, p.vocab);
  u32x4 raw[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) raw[i] = Lane<DT, false>::raw(x, base + i * 64 * EPL, p.vocab);
  const RowSettings s = settings(p, row);
  Lane<DT, false> a[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
    a[i].take(raw[i], base + i * 64 * EPL, p.vocab, end, (group + 1) * kGroup);
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int e = 0; e < EPL; ++e) m = fmaxf(m, a[i].v[e]);
  m = fmaxf(m, dpp_mov<0xb1>(m));   // quad_perm [1,0,3,2]
  m = fmaxf(m, dpp_mov<0x4e>(m));   // quad_perm [2,3,0,1]
  if ((lane & 3) == 0) p.smax[((int64_t)row * p.groups + group) * 16 + (lane >> 2)] = m;
  m = fmaxf(m, dpp_mov<0x124>(m));  // row_ror:4
  m = fmaxf(m, dpp_mov<0x128>(m));  // row_ror:8: the row's maximum in each of its 16 lanes
  m = quad_max(m);
  // the weights' sum is needed unless top-k lists the kept tokens anyway (or the row is greedy)
  const bool need_t = !s.greedy && s.k == 0;
  double st = 0.0, s1 = 0.0;
  if (m != kNegInf && need_t) {  // uniform
    // the elements once more, from the caches: a loop of one load's exponentials instead of
    // sixteen in line (the code of a launch comes cold from memory)
#pragma unroll 1
    for (int i = 0; i < IT; ++i) {
      Lane<DT, false> b;
      const int j = base + i * 64 * EPL;
      b.take(Lane<DT, false>::raw(x, j, p.vocab), j, p.vocab, end, (group + 1) * kGroup);
#pragma unroll
      for (int e = 0; e < EPL; ++e) st += weight(b.v[e], m, s.inv2);
    }
    st = wave_sum(st);
  }
  if (need_t && s.t1) {
    s1 = st;
  } else if (p.lp && m != kNegInf) {
    // for the log-probability, an f32 number: f32 exponentials (off by about 2^-22 of their own
    // value, either way), 16 of them summed in f32, those sums in f64
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float d = a[i].v[e] >= m ? 0.f : a[i].v[e] - m;
        q += fast_exp2(d * 1.44269504088896340736f);
      }
    s1 = wave_sum((double)q);
  }
  if (lane == 0) {
    const int64_t at = (int64_t)row * p.groups + group;
    p.gmax[at] = m;
    p.sum_t[at] = st;
    p.sum_1[at] = s1;
  }
}

// ---- shared by gather and pick -----------------------------------------------------------------
// Order-preserving integers of floats (no NaN; -0 as +0), and the order of tokens as one number:
// larger is earlier.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t rank_of(float l, int i) {
  return ((uint64_t)key_of(l) << 32) | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float logit_of(uint64_t r) { return of_key((uint32_t)(r >> 32)); }
__device__ __forceinline__ int index_of(uint64_t r) { return (int)(0xffffffffu - (uint32_t)r); }

// LDS of a spread workgroup, and what the block functions below need of one.
struct SpreadShared {
  static constexpr int NW = kSpread / 64;
  uint64_t raw[kShort];  // ranks as collected
  double red[NW];
  double sums[2][kChunk / 256];
  int i[6];
};
// That of a pick workgroup: where no row filters, and where rows may.
struct DrawShared {
  static constexpr int NW = kWaves;
  double red[NW];
  double logz;
  int i[2];
};
struct PickShared {
  static constexpr int NW = kWaves;
  u32x4 ring[kWaves * kAhead * 64];
  uint64_t raw[kList];     // ranks as collected
  uint64_t sorted[kList];  // ranks, earliest first
  uint32_t bin[kBins];     // counts or weights
  double red[NW];
  uint32_t cnt[NW];
  double logz;
  int n;
  int i[8];
};

// The sum over the workgroup, the same bits in every thread.
template <class SH>
__device__ __forceinline__ double block_sum(SH& sh, double v) {
  v = wave_sum(v);
  __syncthreads();
  if ((item_id() & 63) == 0) sh.red[item_id() >> 6] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < SH::NW; ++w) t += sh.red[w];
  return t;
}
// Exclusive prefix sum over the workgroup's threads, and the whole sum.
template <class SH>
__device__ __forceinline__ double block_scan(SH& sh, double v, double* total) {
  const int wave = item_id() >> 6;
  double mine;
  const double e = wave_scan(v, &mine);
  __syncthreads();
  if ((item_id() & 63) == 0) sh.red[wave] = mine;
  __syncthreads();
  double before = 0.0, t = 0.0;
#pragma unroll
  for (int w = 0; w < SH::NW; ++w) {
    if (w == wave) before = t;
    t += sh.red[w];
  }
  *total = t;
  return before + e;
}
template <class F>
__device__ __forceinline__ uint32_t block_reduce_u32(PickShared& sh, uint32_t v, F f) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v = f(v, (uint32_t)__shfl_xor((int)v, s));
  __syncthreads();
  if ((item_id() & 63) == 0) sh.cnt[item_id() >> 6] = v;
  __syncthreads();
  uint32_t t = sh.cnt[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) t = f(t, sh.cnt[w]);
  return t;
}
// The smallest of the threads' `lo` (their wave first: a thousand atomics on one word took 17 us)
// and the largest of their `hi`, in sh.i[at] and sh.i[at + 1].
template <class SH>
__device__ __forceinline__ void block_min_max(SH& sh, int at, int lo, int hi) {
  if (item_id() == 0) {
    sh.i[at] = 0x7fffffff;
    sh.i[at + 1] = -0x7fffffff;
  }
  __syncthreads();
  lo = wave_min(lo);
  hi = wave_max(hi);
  if ((item_id() & 63) == 0) {
    atomicMin(&sh.i[at], lo);
    atomicMax(&sh.i[at + 1], hi);
  }
  __syncthreads();
}

// Descending bitonic sort of v[0 .. n), padded with zeros to a power of two (at most kList).
__device__ __forceinline__ void sort_list(uint64_t* v, int n) {
  int n2 = 2;
  while (n2 < n) n2 *= 2;
  const int tid = item_id();
  for (int i = n + tid; i < n2; i += kPick) v[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int size = 2; size <= n2; size *= 2)
#pragma unroll 1
    for (int stride = size / 2; stride > 0; stride /= 2) {
#pragma unroll 1
      for (int t = tid; t < n2 / 2; t += kPick) {
        const int lo = 2 * t - (t & (stride - 1)), hi = lo + stride;
        const uint64_t a = v[lo], b = v[hi];
        if ((a < b) == ((lo & size) == 0)) {
          v[lo] = b;
          v[hi] = a;
        }
      }
      __syncthreads();
    }
}

// A row, or a part of one: each wave owns a run of whole steps (64 lanes' loads).
template <int DT, bool TINY>
struct Row {
  static constexpr int EPL = Lane<DT, TINY>::EPL;
  static constexpr int STEP = 64 * EPL;
  const store_t<DT>* x;
  int n;
  u32x4* ring;  // LDS
  // the run of wave w when [from, to) is shared out: steps of it, the last waves' may be empty
  static __device__ __forceinline__ int run_of(int from, int to) {
    const int steps = (to - from + STEP - 1) / STEP;
    return (steps + kWaves - 1) / kWaves * STEP;
  }
  // f(this lane's first index, its EPL logits) over the wave's run of [from, to) in index order, a
  // step at a time, elements past `to` as -inf. kAhead steps are loaded while as many are worked on:
  // a CU alone reads a row (200 KB or so) from beyond its L2. The ones worked on lie in the wave's
  // part of `ring`, so that f is there once, in a loop over them (in registers every step would have
  // its own copy of f; turning registers round instead waits for the load just issued).
  template <class F>
  __device__ __forceinline__ void each(int from, int to, F f) const {
    const int run = run_of(from, to);
    const int wave = __builtin_amdgcn_readfirstlane(item_id() >> 6), lane = item_id() & 63;
    const int a = from + wave * run, b = min(to, a + run);
    const int off = lane * EPL;
    u32x4* mine = ring + wave * (kAhead * 64) + lane;
    u32x4 r[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) r[j] = Lane<DT, TINY>::raw(x, a + j * STEP + off, n);
#pragma unroll 1
    for (int i = a; i < b; i += kAhead * STEP) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) mine[j * 64] = r[j];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        r[j] = Lane<DT, TINY>::raw(x, i + (kAhead + j) * STEP + off, n);
#pragma unroll 1
      for (int j = 0; j < kAhead && i + j * STEP < b; ++j) {  // uniform
        Lane<DT, TINY> cur;
        cur.take(mine[j * 64], i + j * STEP + off, n, b, i + (j + 1) * STEP);
        f(i + j * STEP + off, cur);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each(0, n, f);
  }
};

// Appends the lanes' ranks where `take`, in no order; sh.n counts them, the first kList are held.
__device__ __forceinline__ void append(PickShared& sh, bool take, float l, int i) {
  const uint64_t v = __ballot(take);
  if (v == 0) return;  // uniform
  const int lane = item_id() & 63;
  int at = 0;
  if (lane == 0) at = atomicAdd(&sh.n, __popcll(v));
  at = __builtin_amdgcn_readfirstlane(at) + __popcll(v & ((uint64_t(1) << lane) - 1));
  if (take && at < kList) sh.raw[at] = rank_of(l, i);
}

// One wave: the position at which the running weight passes u times the whole, over positions
// PER * lane + e in order; the last one of any weight where rounding leaves none.
template <int PER>
__device__ __forceinline__ int wave_draw(const double (&w)[PER], double u) {
  double mine = 0.0, total;
#pragma unroll
  for (int e = 0; e < PER; ++e) mine += w[e];
  double run = wave_scan(mine, &total);
  const double target = u * total;
  const int lane = item_id() & 63;
  int hit = 0x7fffffff, last = -1;
#pragma unroll
  for (int e = PER - 1; e >= 0; --e)
    if (last < 0 && w[e] > 0.0) last = PER * lane + e;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    run += w[e];
    if (w[e] > 0.0 && run > target) hit = min(hit, PER * lane + e);
  }
  hit = wave_min(hit);
  last = wave_max(last);
  return hit != 0x7fffffff ? hit : last;
}

// The token of a row all of whose kept elements are among sh.raw[0 .. n), n <= kShort: the
// definition as it stands. whole: W(S1) where S1 reaches below the list, else negative. The
// result is wave 0's alone.
__device__ __forceinline__ int pick_short(PickShared& sh, int n, const RowSettings& s, float m,
                                          double whole, double u) {
  // both orders by counting: kPick / n2 threads an element (n2: n as a power of two), each a part of
  // the list; an element's place is the number of ranks above (indexes below) its own
  const int tid = item_id();
  int n2 = 64;
  while (n2 < n) n2 *= 2;
  const int parts = kPick / n2, part = tid / n2, me = tid % n2;  // parts 16, 8 or 4
  uint32_t* place = sh.bin;  // [part][me]: by rank (low half) and by index (high half)
  {
    const uint64_t mine = me < n ? sh.raw[me] : 0;
    const uint32_t my_i = (uint32_t)mine;
    const int len = n2 / parts, a = part * len, b = min(a + len, n);
    uint32_t c = 0;
#pragma unroll 4
    for (int j = a; j < b; ++j) {
      const uint64_t r = sh.raw[j];
      c += (r > mine ? 1u : 0u) + ((uint32_t)r > my_i ? 0x10000u : 0u);  // (indexes are inverted)
    }
    place[part * n2 + me] = c;
    __syncthreads();
    if (part == 0 && me < n) {
      c = 0;
      for (int q = 0; q < parts; ++q) c += place[q * n2 + me];
      sh.sorted[c & 0xffffu] = mine;
      sh.sorted[kShort + (c >> 16)] = mine;  // in index order
    }
    __syncthreads();
  }
  if (tid >= 64) return 0;
  constexpr int PER = kShort / 64;
  double w[PER];
  double sum = 0.0, total;
  bool in1[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int j = PER * tid + e;
    w[e] = j < n ? weight(logit_of(sh.sorted[j]), m, s.inv2) : 0.0;
    in1[e] = j < n && (s.k == 0 || j < s.k) && w[e] >= s.mp;
    if (!in1[e]) w[e] = 0.0;
    sum += w[e];
  }
  double run = wave_scan(sum, &total);
  const double limit = (double)s.p * (whole >= 0.0 ? whole : total);
  // the kept ranks are a run from the first: its last one
  int last = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (in1[e] && (s.p >= 1.f || run < limit)) last = PER * tid + e;
    run += w[e];
  }
  const uint64_t low = sh.sorted[wave_max(last)];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int j = PER * tid + e;
    const uint64_t r = j < n ? sh.sorted[kShort + j] : 0;
    w[e] = j < n && r >= low ? weight(logit_of(r), m, s.inv2) : 0.0;
  }
  return index_of(sh.sorted[kShort + wave_draw<PER>(w, u)]);
}

// The last rank that is kept when a row's ranks are cut at a count (by_count: the first `count`) or
// at a weight (those whose predecessors weigh less than `limit`). Histograms over the logits, first
// linear below m, then over ever smaller ranges of their integer keys, until the boundary's bin
// holds a list's worth of tokens or a single value. total_w: the row's weight.
// *listed (weights only): the boundary's bin is listed, sh.sorted[0 .. *listed), and `mine` is the
// weight of the ranks before that bin in the wave's run of the row; -1 where it is not.
template <int DT, bool TINY>
__device__ __forceinline__ uint64_t boundary(const Row<DT, TINY>& row, PickShared& sh, float m,
                                             double inv2, bool by_count, int count, double limit,
                                             double total_w, int* listed, double* mine_before) {
  constexpr int EPL = Row<DT, TINY>::EPL;
  const int tid = item_id();
  // linear bins: 1/256 of a natural-log unit of weight, or 1/128 of a logit
  const float scale = by_count ? 128.f : fminf((float)(inv2 * (256.0 / kLog2e)), 1e30f);
  const float inv2f = fminf((float)inv2, 1e30f);
  // histogram weights are integers whose sum over the row stays below 2^31
  const int wshift = 30 - (int)__builtin_ceil(log2(fmax(total_w, 1.0)));
  const float wscale = __builtin_ldexpf(1.f, wshift);
  uint32_t klo = key_of(kNegInf) + 1, khi = key_of(m);  // the range that holds the boundary
  int shift = -1;                                       // -1: linear bins
  *listed = -1;
#pragma unroll 1
  for (;;) {
    // bin 0 is the earliest; bins grow as logits fall
    auto linear_bin = [&](float l) -> int {
      return (int)(l >= m ? 0.f : fminf((m - l) * scale, (float)(kBins - 1)));
    };
    // the least key of bins [0, b]
    auto bin_floor = [&](int b) -> uint32_t {
      if (shift >= 0) {
        const uint64_t d = ((uint64_t)(b + 1) << shift) - 1;
        return d >= khi - klo ? klo : khi - (uint32_t)d;
      }
      uint32_t x = klo, y = khi;  // by bisection: the bin is monotone in the logit
      while (x < y) {
        const uint32_t mid = x + (y - x) / 2;
        if (linear_bin(of_key(mid)) <= b) y = mid;
        else x = mid + 1;
      }
      return x;
    };
    const bool counts = by_count || shift == 0;  // (a single value's weight is count * weight)
    const float fhi = of_key(khi), flo = of_key(klo);
    __syncthreads();
    for (int b = tid; b < kBins; b += kPick) sh.bin[b] = 0;
    __syncthreads();
    double above = 0.0;    // weight of the ranks before the range (integer bins only)
    uint32_t n_above = 0;  // and their number
    row.each([&](int, const Lane<DT, TINY>& a) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float l = a.v[e];
        if (shift >= 0) {  // uniform
          n_above += l > fhi ? 1u : 0u;
          if (!by_count && __ballot(l > fhi)) above += l > fhi ? weight(l, m, inv2) : 0.0;
        }
        // an f32 exponential, off by up to (|y| + 2) 2^-23: 2^-18 of it where it counts
        const float w = l >= m ? wscale : fast_exp2((l - m) * inv2f) * wscale;
        const int b = shift < 0 ? linear_bin(l) : (int)((khi - key_of(l)) >> (shift & 31));
        if (l >= flo && l <= fhi) atomicAdd(&sh.bin[b], counts ? 1u : (uint32_t)w);
      }
    });
    if (!by_count && shift >= 0) above = block_sum(sh, above);
    if (shift >= 0)
      n_above = block_reduce_u32(sh, n_above, [](uint32_t a, uint32_t b) { return a + b; });
    else __syncthreads();
    // ---- walk the bins from the earliest (thread t: bins PB t ..): by weight the boundary is in
    // bins [lo, hi], where the running weight passes the limit less and more what the histogram's
    // weights may be off by; at single-value bins the weights are exact
    constexpr int PB = kBins / kPick;
    double w[PB];
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < PB; ++e) {
      const int b = PB * tid + e;
      const double c = (double)sh.bin[b];
      w[e] = by_count     ? c
             : shift == 0 ? c * weight(of_key(khi - min((uint32_t)b, khi - klo)), m, inv2)
                          : __builtin_ldexp(c, -wshift);
      sum += w[e];
    }
    double total;
    double run = block_scan(sh, sum, &total);
    run += by_count ? (double)n_above : above;
    const double want = by_count ? (double)count : limit;
    // (an integer weight is truncated: one step an element)
    const double slack = counts ? 0.0 : (above + total) * 0x1p-17 + __builtin_ldexp(row.n, -wshift);
    if (tid == 0) {
      sh.i[0] = kBins;  // lo
      sh.i[1] = kBins;  // hi
      sh.i[2] = 0;      // the last bin with a weight
      sh.n = 0;
    }
    __syncthreads();
    {
      int b0 = kBins, b1 = kBins, b2 = 0;
#pragma unroll
      for (int e = 0; e < PB; ++e) {
        const int b = PB * tid + e;
        run += w[e];
        if (run >= want - slack) b0 = min(b0, b);
        if (run >= want + slack) b1 = min(b1, b);
        if (sh.bin[b]) b2 = b;
      }
      // (within a wave first: a thousand atomics on one word took 17 us)
      b0 = wave_min(b0);
      b1 = wave_min(b1);
      b2 = wave_max(b2);
      if ((tid & 63) == 0) {
        atomicMin(&sh.i[0], b0);
        atomicMin(&sh.i[1], b1);
        atomicMax(&sh.i[2], b2);
      }
    }
    __syncthreads();
    // (a count that the row does not reach ends at its last element; a limit that it does not
    // reach but for rounding, somewhere from the last bin of any weight on)
    int hi = sh.i[1] == kBins ? (counts ? sh.i[2] : kBins - 1) : sh.i[1];
    int lo = min(sh.i[0] == kBins ? sh.i[2] : sh.i[0], hi);

    // ---- what the bins hold is listed; the same pass sums what comes before
    uint32_t top = lo == 0 ? khi : bin_floor(lo - 1) - 1, bottom = bin_floor(hi);
    {
      const float ftop = of_key(top), fbottom = of_key(bottom);
      double x = 0.0;
      uint32_t pre = 0;
      row.each([&](int i, const Lane<DT, TINY>& a) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const float l = a.v[e];
          append(sh, l >= fbottom && l <= ftop, l, i + e);
          if (by_count) pre += l > ftop ? 1u : 0u;
          else if (__ballot(l > ftop)) x += l > ftop ? weight(l, m, inv2) : 0.0;
        }
      });
      if (by_count)
        pre = block_reduce_u32(sh, pre, [](uint32_t a, uint32_t b) { return a + b; });
      x = wave_sum(x);
      *mine_before = x;
      above = by_count ? (double)pre : block_sum(sh, (tid & 63) == 0 ? x : 0.0);
    }
    const int n = sh.n;
    if (n <= kList) {
      // ---- the boundary is one of these: ordered, and the definition applied to them
      __syncthreads();
      for (int j = tid; j < n; j += kPick) sh.sorted[j] = sh.raw[j];
      __syncthreads();
      sort_list(sh.sorted, n);
      if (!by_count) *listed = n;
      constexpr int PL = kList / kPick;
      double wl[PL];
      double mine = 0.0, tot;
#pragma unroll
      for (int e = 0; e < PL; ++e) {
        const int j = PL * tid + e;
        wl[e] = j >= n ? 0.0 : by_count ? 1.0 : weight(logit_of(sh.sorted[j]), m, inv2);
        mine += wl[e];
      }
      double before = above + block_scan(sh, mine, &tot);
      if (tid == 0) sh.i[3] = 0;
      __syncthreads();
      int at = 0;
#pragma unroll
      for (int e = 0; e < PL; ++e) {
        if (PL * tid + e < n && before < want) at = PL * tid + e;
        before += wl[e];
      }
      at = wave_max(at);
      if ((tid & 63) == 0) atomicMax(&sh.i[3], at);
      __syncthreads();
      const uint64_t r = sh.sorted[sh.i[3]];
      __syncthreads();
      return r;
    }
    if (top == bottom) {
      // ---- one value, more often than a list holds: its t-th occurrence in index order
      const float v = of_key(top);
      const double wv = by_count ? 1.0 : weight(v, m, inv2);
      // kept: occurrences j with above + j wv < want
      double t = above < want ? (double)n : 1.0;
      if (wv > 0.0) {
        t = fmin(fmax(__builtin_ceil((want - above) / wv), 1.0), (double)n);
        if (t > 1.0 && above + (t - 1.0) * wv >= want) t -= 1.0;
        else if (above + t * wv < want) t += 1.0;
      }
      const uint32_t nth = (uint32_t)fmin(fmax(t, 1.0), (double)n);
      // its index: the waves' counts, then the wave that holds it step by step
      uint32_t mine = 0;
      row.each([&](int, const Lane<DT, TINY>& a) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) mine += a.v[e] == v ? 1u : 0u;
      });
      double all, wave_all;
      const double wave_mine = wave_sum((double)mine);
      const double first = block_scan(sh, (tid & 63) == 0 ? wave_mine : 0.0, &all);
      // (the scan gives lane 0 of a wave the waves before it)
      uint32_t seen = (uint32_t)__shfl(first, 0);
      if (tid == 0) sh.i[4] = 0;
      __syncthreads();
      if (seen < nth && nth <= seen + (uint32_t)wave_mine)
        row.each([&](int i, const Lane<DT, TINY>& a) {
          uint32_t c = 0;
#pragma unroll
          for (int e = 0; e < EPL; ++e) c += a.v[e] == v ? 1u : 0u;
          uint32_t before = seen + (uint32_t)wave_scan((double)c, &wave_all);
#pragma unroll
          for (int e = 0; e < EPL; ++e)
            if (a.v[e] == v)
              if (++before == nth) sh.i[4] = i + e;
          seen += (uint32_t)wave_all;
        });
      __syncthreads();
      const uint64_t r = ((uint64_t)top << 32) | (0xffffffffu - (uint32_t)sh.i[4]);
      __syncthreads();
      return r;
    }
    // ---- a smaller range. First the one bin of [lo, hi], by exact sums (so that every round leaves
    // a bin of the last one's, and the rounds end)
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      const float fm = of_key(bin_floor(mid));
      double y = 0.0;
      row.each([&](int, const Lane<DT, TINY>& a) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (__ballot(a.v[e] >= fm)) y += a.v[e] >= fm ? weight(a.v[e], m, inv2) : 0.0;
      });
      if (block_sum(sh, y) >= want) hi = mid;
      else lo = mid + 1;
    }
    top = lo == 0 ? khi : bin_floor(lo - 1) - 1;
    klo = bin_floor(lo);
    khi = top;
    const int bits = 32 - __builtin_clz((khi - klo) | 1u);
    shift = max(0, bits - 12);
  }
}

// Any filters, any number of kept tokens. The result is every thread's.
template <int DT, bool TINY>
__device__ __forceinline__ int pick_wide(const Row<DT, TINY>& row, PickShared& sh, const RowSettings& s,
                                         float m, double W, double u) {
  constexpr int EPL = Row<DT, TINY>::EPL;
  const int tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint64_t low = 0;  // kept: ranks from here up, of weight >= mp
  int listed = -1;
  double mine = 0.0;
  auto kept_weight = [&](int i, float l) {
    const bool in = rank_of(l, i) >= low;
    if (!__ballot(in)) return 0.0;
    const double w = in ? weight(l, m, s.inv2) : 0.0;
    return w >= s.mp ? w : 0.0;
  };
  // the cut by count, then the one by weight (one loop, so that the code is there once)
#pragma unroll 1
  for (int by = s.k > 0 ? 0 : 1; by < (s.p < 1.f ? 2 : 1); ++by) {
    double limit = 0.0, all = 1.0;
    if (by == 1) {
      // W(S1) and the whole row's weight
      double w1 = all = W;
      if (s.k > 0 || s.mp > 0.0) {
        double x = 0.0, y = 0.0;
        row.each([&](int i, const Lane<DT, TINY>& a) {
#pragma unroll
          for (int e = 0; e < EPL; ++e) {
            const double w = weight(a.v[e], m, s.inv2);
            y += w;
            if (w >= s.mp && rank_of(a.v[e], i + e) >= low) x += w;
          }
        });
        w1 = block_sum(sh, x);
        all = block_sum(sh, y);
      }
      limit = (double)s.p * w1;
    }
    // S1 is a run from the first rank and weighs more than the limit (p < 1), so the boundary in
    // the whole row's order is the boundary in S1's; a limit of 0 or less keeps the first alone
    const uint64_t r = boundary(row, sh, m, s.inv2, by == 0, s.k, limit, all, &listed, &mine);
    if (r > low) low = r;
    else listed = -1;
  }
  // ---- the kept weight of each wave's run; then of the runs of the run that holds u times the
  // whole, down to 256 elements
  int from = 0, to = row.n;
  bool known = false;
  if (listed >= 0 && s.mp <= 0.0) {
    // what comes before the boundary's bin is known; its kept ranks join their runs
    const int run = Row<DT, TINY>::run_of(0, row.n);
    double x = 0.0;
#pragma unroll 1
    for (int j = lane; j < listed; j += 64) {
      const uint64_t r = sh.sorted[j];
      if (r >= low && index_of(r) / run == wave) x += weight(logit_of(r), m, s.inv2);
    }
    mine += wave_sum(x);
    known = true;
  }
  double left = 0.0;
  bool top = true;
#pragma unroll 1
  for (;;) {
    if (!known) {
      double x = 0.0;
      row.each(from, to, [&](int i, const Lane<DT, TINY>& a) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) x += kept_weight(i + e, a.v[e]);
      });
      mine = wave_sum(x);
    }
    known = false;
    __syncthreads();
    if (lane == 0) sh.red[wave] = mine;
    __syncthreads();
    double total = 0.0;
#pragma unroll 1
    for (int w = 0; w < kWaves; ++w) total += sh.red[w];
    if (top) left = u * total;
    top = false;
    // the first run whose running weight passes `left`, the last one of any weight where rounding
    // leaves none
    double run = 0.0, before = 0.0;
    int hit = 0;
    bool found = false;
#pragma unroll 1
    for (int w = 0; w < kWaves; ++w) {
      const double x = sh.red[w];
      if (!found && x > 0.0) {
        hit = w;
        before = run;
        found = run + x > left;
      }
      run += x;
    }
    left -= before;
    const int len = Row<DT, TINY>::run_of(from, to);
    from += hit * len;
    to = min(to, from + len);
    if (to - from <= Row<DT, TINY>::STEP) break;
  }
  // at most a step is left (every wave alike)
  Lane<DT, TINY> a;
  const int i0 = from + lane * EPL;
  a.take(Lane<DT, TINY>::raw(row.x, i0, row.n), i0, row.n, to, from + Row<DT, TINY>::STEP);
  double x[EPL];
  double sum = 0.0, all;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    x[e] = kept_weight(i0 + e, a.v[e]);
    sum += x[e];
  }
  double run = wave_scan(sum, &all);
  int hit = 0x7fffffff, lastk = -1;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    run += x[e];
    if (x[e] > 0.0) {
      if (run > left) hit = min(hit, i0 + e);
      lastk = i0 + e;
    }
  }
  hit = wave_min(hit);
  lastk = wave_max(lastk);
  return hit != 0x7fffffff ? hit : lastk;
}

// ---- gather ------------------------------------------------------------------------------------
// Which maxima bound a row's list: the `k`-th largest of `n`, of a group or a quarter or a sixteenth
// of one each (`span` of the sixteenths); n 0 for no list. k is top_k, or for nuclei and minima a
// guess at what they leave.
struct ListRule {
  int k, n, span;
};
__device__ __forceinline__ ListRule list_rule(const RowSettings& s, int groups) {
  ListRule r;
  r.k = s.k > 0 ? s.k : 96;
  // (with k near the number of maxima the bound falls far below the k-th logit)
  r.span = 4 * r.k <= 3 * groups ? 16 : r.k <= 3 * groups || groups > kHeld / 16 ? 4 : 1;
  r.n = groups * (16 / r.span);
  if (r.k > r.n || r.k > kShort || r.n > kHeld) r.n = 0;
  return r;
}

// A bound that the k-th largest of n maxima does not fall below, one wave: bisection of the keys'
// range, the maxima in registers (PER a lane). 20 steps leave a millionth of the range, which costs a
// few tokens more on the list. -inf where fewer than k are finite.
template <int PER, class F>
__device__ __forceinline__ float list_bound(F maximum, int n, int k) {
  const int lane = item_id() & 63;
  const uint32_t none = key_of(kNegInf);
  uint32_t key[PER], hi = none, least = 0xffffffffu;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int g = 64 * j + lane;
    key[j] = g < n ? key_of(maximum(g)) : none;
    hi = max(hi, key[j]);
    least = min(least, key[j] > none ? key[j] : 0xffffffffu);
  }
  auto at_least = [&](uint32_t t) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) c += __popcll(__ballot(key[j] >= t));
    return c;
  };
  if (at_least(none + 1) < k) return kNegInf;
  // (the signed order of keys with their top bit turned is their own)
  hi = (uint32_t)wave_max((int)(hi ^ 0x80000000u)) ^ 0x80000000u;
  uint32_t lo = (uint32_t)wave_min((int)(least ^ 0x80000000u)) ^ 0x80000000u;
#pragma unroll 1
  for (int step = 0; step < 20 && lo < hi; ++step) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const int c = at_least(mid);
    if (c >= k) lo = mid;
    else hi = mid - 1;
    if (c == k) break;
  }
  return of_key(lo);
}

// A row's largest logit, and its weight against that; each wave by itself.
__device__ __forceinline__ float row_max(const SampleParams& p, int row) {
  const float* gm = p.gmax + (int64_t)row * p.groups;
  float m = kNegInf;
#pragma unroll 2
  for (int g = item_id() & 63; g < p.groups; g += 64) m = fmaxf(m, gm[g]);
  return wave_max_all(m);
}
__device__ __forceinline__ double row_weight(const SampleParams& p, int row, float m, double inv2) {
  const int64_t at = (int64_t)row * p.groups;
  double w = 0.0;
#pragma unroll 1
  for (int g = item_id() & 63; g < p.groups; g += 64)
    w += p.sum_t[at + g] * weight(p.gmax[at + g], m, inv2);
  return wave_sum(w);
}

// A nucleus' histogram: bins of equal steps of the weight's logarithm below the maximum. They reach
// as far as the boundary may lie: n tokens of weight below (1 - p) W / n weigh less than (1 - p) W
// together (and 2^8 further they do not matter to what follows the boundary either), and none below
// min_p is kept. A bin's weights are integers of f32 exponentials (adding them in any order gives the
// same sum), in a unit of the bin's own, 2^-unit 2^-`bits` of the largest: each is off by less than
// `off` of itself, so that the sum over the bins up to one is known to that share of it, and what
// follows it to that share of what follows.
struct CutBins {
  float m = 0.f, scale = 0.f, inv2f = 0.f, step = 0.f;
  int bits = 0;
  CutBins() = default;
  __device__ __forceinline__ CutBins(float m, const RowSettings& s, int n, double whole) : m(m) {
    double reach = s.mp > 0.0 ? 0.25 - log2(s.mp)
                              : 8.25 + log2((double)n / ((1.0 - (double)s.p) * whole));
    reach = __builtin_fmin(__builtin_fmax(reach, 1.0), 120.0);
    scale = fminf((float)(s.inv2 * (kCutBins / reach)), 1e30f);
    inv2f = fminf((float)s.inv2, 1e30f);
    step = (float)reach * (1.f / kCutBins);
    bits = 31 - (32 - __builtin_clz((uint32_t)n));  // n times the largest stays below 2^32
  }
  // a bin where below kCutBins; it does not fall as logits do
  __device__ __forceinline__ float pos(float l) const {
    return l >= m ? 0.f : fminf((m - l) * scale, (float)kCutBins);
  }
  __device__ __forceinline__ float unit(int b) const { return floorf((float)b * step); }
  __device__ __forceinline__ uint32_t value(float l, int b) const {
    const float y = l >= m ? 0.f : (l - m) * inv2f;
    return (uint32_t)(fast_exp2(y + unit(b)) * __builtin_ldexpf(1.f, bits) + 0.5f);
  }
  __device__ __forceinline__ double weight_of(uint32_t c, int b) const {
    return __builtin_ldexp((double)c, -bits - (int)unit(b));
  }
  // (a value is 2^(bits - 1) units at least, rounded to one; an exponent is off by 2^-16)
  __device__ __forceinline__ double off() const { return __builtin_ldexp(1.0, -bits) + 0x1p-15; }
};

// Sums over the groups of a chunk from those of the waves' loads: entry n covers elements
// n * 64 EPL on. Called by the workgroup's first threads.
template <int EPL>
__device__ __forceinline__ void put_group_sums(const SampleParams& p, double* to, int row, int chunk,
                                               const double* red) {
  constexpr int PER = kGroup / (64 * EPL), N = kChunk / kGroup;
  const int t = item_id(), g = chunk * N + t;
  if (t >= N || g >= p.groups) return;
  double x = 0.0;
#pragma unroll
  for (int j = 0; j < PER; ++j) x += red[t * PER + j];
  to[(int64_t)row * p.groups + g] = x;
}

template <int DT>
__global__ __launch_bounds__(256) void sample_gather_kernel(SampleParams p) {
  constexpr int EPL = Lane<DT, false>::EPL, IT = kChunk / (256 * EPL);
  __shared__ float bound, top;
  __shared__ double whole;
  __shared__ int count[2];
  __shared__ double red[2][kChunk / (64 * EPL)];
  __shared__ __attribute__((aligned(16))) uint32_t hist[kCutBins];
  const int row = wg_id_y(), tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RowSettings s = settings(p, row);
  if (s.greedy || !s.filtered()) return;
  bool nucleus = s.k == 0 && s.p < 1.f;
  const bool minima = s.k == 0 && s.mp > 0.0;
  const ListRule rule = list_rule(s, p.groups);
  const bool listing = rule.n > 0;
  const int c0 = wg_id_x() * p.per, c1 = min(c0 + p.per, p.chunks);
  if (!listing && !nucleus && !minima) {
    if (c0 == 0 && tid == 0) p.low[row] = kNegInf;
    return;
  }
  const store_t<DT>* x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)row * p.ls;
  u32x4 a[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
    a[i] = Lane<DT, false>::raw(x, c0 * kChunk + (i * 256 + tid) * EPL, p.vocab);
  if (tid < 2) count[tid] = 0;
  if (nucleus)
    for (int b = tid; b < kCutBins; b += 256) hist[b] = 0;
  if (wave == 0) {
    float b = kNegInf;
    if (listing) {
      const float* gm = p.gmax + (int64_t)row * p.groups;
      const float* sm = p.smax + (int64_t)row * p.groups * 16;
      auto quarter = [&](int g) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(sm + 4 * g);
        return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      };
      if (rule.span == 16)
        b = rule.n <= 128 ? list_bound<2>([&](int g) { return gm[g]; }, rule.n, rule.k)
                          : list_bound<kHeld / 64>([&](int g) { return gm[g]; }, rule.n, rule.k);
      else if (rule.span == 4)
        b = rule.n <= 256 ? list_bound<4>(quarter, rule.n, rule.k)
                          : list_bound<kHeld / 64>(quarter, rule.n, rule.k);
      else
        b = list_bound<kHeld / 64>([&](int g) { return sm[g]; }, rule.n, rule.k);
    }
    if (lane == 0) bound = b;
  } else if (wave == 1 && (nucleus || minima)) {
    const float m = row_max(p, row);
    const double w = nucleus && m != kNegInf ? row_weight(p, row, m, s.inv2) : 0.0;
    if (lane == 0) {
      top = m;
      whole = w;
    }
  }
  __syncthreads();
  const float low = bound;
  if (c0 == 0 && tid == 0) p.low[row] = low;
  if (low == kNegInf && !nucleus && !minima) return;
  const float m = nucleus || minima ? top : 0.f;
  if (m == kNegInf) return;
  nucleus = nucleus && m != __builtin_inff();
  CutBins bins;
  if (nucleus) bins = CutBins(m, s, p.vocab, whole);
  const float inv2f = fminf((float)s.inv2, 1e30f);
  // (surely below min_p: no f64 weight)
  float min_y = 0.f;
  if (minima) min_y = (float)log2(s.mp) - 0.01f;
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    uint64_t* to = p.cand + ((int64_t)row * p.chunks + c) * kShort;
    int* n = &count[c & 1];
    if (nucleus || minima) {
      // (a loop of one load, from the caches: the code is there once)
#pragma unroll 1
      for (int i = 0; i < IT; ++i) {
        const int i0 = c * kChunk + (i * 256 + tid) * EPL;
        Lane<DT, false> cur;
        cur.take(Lane<DT, false>::raw(x, i0, p.vocab), i0, p.vocab, p.vocab,
                 c * kChunk + (i + 1) * 256 * EPL);
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const float l = cur.v[e];
          if (nucleus) {
            const float at = bins.pos(l);
            if (at < (float)kCutBins) atomicAdd(&hist[(int)at], bins.value(l, (int)at));
          }
          if (minima) {
            if (__ballot(l >= m || (l - m) * inv2f >= min_y)) {
              const double w = weight(l, m, s.inv2);
              sum += w >= s.mp ? w : 0.0;
            }
          }
        }
        if (minima) {
          sum = wave_sum(sum);
          if (lane == 0) red[c & 1][i * 4 + wave] = sum;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int i0 = c * kChunk + (i * 256 + tid) * EPL;
      Lane<DT, false> cur;
      cur.take(a[i], i0, p.vocab, p.vocab, c * kChunk + (i + 1) * 256 * EPL);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float l = cur.v[e];
        const bool take = l >= low && low != kNegInf;
        const uint64_t v = __ballot(take);
        if (v == 0) continue;  // uniform
        int at = 0;
        if (lane == 0) at = atomicAdd(n, __popcll(v));
        at = __builtin_amdgcn_readfirstlane(at) + __popcll(v & ((uint64_t(1) << lane) - 1));
        if (take && at < kShort) to[at] = rank_of(l, i0 + e);
      }
      // the next chunk's loads go out as this one's are done with
      a[i] = Lane<DT, false>::raw(x, i0 + kChunk, p.vocab);
    }
    __syncthreads();
    // (the next chunk uses the other word and row, and its barrier comes before these ones' reuse)
    if (tid == 0) {
      p.count[(int64_t)row * p.chunks + c] = *n;
      *n = 0;
    }
    if (minima) put_group_sums<EPL>(p, p.sum_k, row, c, red[c & 1]);
  }
  if (nucleus) {
    u32x4* to = reinterpret_cast<u32x4*>(p.hist + ((int64_t)row * p.parts + wg_id_x()) * kCutBins);
    for (int b = tid; b < kCutBins / 4; b += 256) to[b] = reinterpret_cast<const u32x4*>(hist)[b];
  }
}

// ---- pick --------------------------------------------------------------------------------------
// The token by the groups' weights: the group that holds u times the whole (each wave by itself),
// then its elements, one a thread. sums(g): a group's weight; keep(i, l): an element's.
static_assert(kGroup == kPick, "one element of a group per thread");
template <int DT, class SH, class F, class G>
__device__ __forceinline__ int draw_groups(SH& sh, const store_t<DT>* x, int vocab, int groups,
                                           double u, F sums, G keep) {
  const int tid = item_id(), lane = tid & 63;
  if (tid == 0) {
    sh.i[0] = 0x7fffffff;
    sh.i[1] = 0;
  }
  // lane: the groups from lane * per
  const int per = (groups + 63) / 64, g0 = lane * per, g1 = min(g0 + per, groups);
  double mine = 0.0, total;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) mine += sums(g);
  double run = wave_scan(mine, &total);
  const double target = u * total;
  const uint64_t pass = __ballot(mine > 0.0 && run + mine > target);
  const uint64_t any = __ballot(mine > 0.0);
  const int who = pass ? __builtin_ctzll(pass) : any ? 63 - __builtin_clzll(any) : 0;
  int g_hit = 0;
  double left = 0.0;
  if (per == 1) {
    g_hit = lane;
    left = target - run;
  } else if (lane == who) {
    bool done = false;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {
      const double w = sums(g);
      if (!done && w > 0.0) {  // (the last one of any weight where rounding leaves none)
        g_hit = g;
        left = target - run;
        done = run + w > target;
      }
      run += w;
    }
  }
  g_hit = __builtin_amdgcn_readfirstlane(__shfl(g_hit, who));
  left = __shfl(left, who);
  const int i = g_hit * kGroup + tid;
  const double w = i < vocab ? keep(i, load1<DT>(x, i)) : 0.0;
  run = block_scan(sh, w, &total);
  const int hit = wave_min(w > 0.0 && run + w > left ? i : 0x7fffffff);
  const int last = wave_max(w > 0.0 ? i : 0);
  if (lane == 0) {
    atomicMin(&sh.i[0], hit);
    atomicMax(&sh.i[1], last);
  }
  __syncthreads();
  return sh.i[0] != 0x7fffffff ? sh.i[0] : sh.i[1];
}

// Collects a row's listed ranks, `held` at most (first: the lane's chunk's count); how many there are (more where a chunk's list is cut).
template <class SH>
__device__ __forceinline__ int collect(SH& sh, const int32_t* counts, int first,
                                       const uint64_t* cand, int chunks, int held) {
  const int lane = item_id() & 63;
  const int wave = __builtin_amdgcn_readfirstlane(item_id() >> 6);
  // chunk counts by lane (every wave alike), places by their running sum
  int n = 0;
  bool over = false;
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const int c = c0 + lane >= chunks ? 0 : c0 == 0 ? first : counts[c0 + lane];
    over = over || __ballot(c > kShort) != 0;
    int before = c;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(before, d);
      if (lane >= d) before += y;
    }
    const int all = __shfl(before, 63);
    before += n - c;
    // waves take the chunks in turn
    for (int j = wave; j < min(64, chunks - c0); j += SH::NW) {
      const int cj = min(__shfl(c, j), kShort), at0 = __shfl(before, j);
      const uint64_t* from = cand + (int64_t)(c0 + j) * kShort;
      for (int q = lane; q < cj; q += 64)
        if (at0 + q < held) sh.raw[at0 + q] = from[q];
    }
    n += all;
  }
  __syncthreads();
  return over ? max(n, held + 1) : n;
}

// Whether the gathered list (from `low` on) settles the row: sh.raw[0 .. *n), and W(S1) in *whole where
// S1 reaches below the list (else -1). first: the count of chunk `lane`.
template <class SH>
__device__ __forceinline__ bool settled(const SampleParams& p, SH& sh, int row, const RowSettings& s,
                                        float low, int first, float m, double W, int* n,
                                        double* whole) {
  *whole = -1.0;
  if (low == kNegInf) return false;
  *n = collect(sh, p.count + (int64_t)row * p.chunks, first, p.cand + (int64_t)row * p.chunks * kShort,
               p.chunks, kShort);
  if (*n > kShort) return false;
  // every kept token is listed when the k-th, the least weight or the limit ends inside
  if (s.k > 0 || (s.mp > 0.0 && weight(low, m, s.inv2) < s.mp)) return true;
  if (s.mp > 0.0 || s.p >= 1.f) return false;
  const int tid = item_id();
  double x = tid < *n ? weight(logit_of(sh.raw[tid]), m, s.inv2) : 0.0;
  x = block_sum(sh, x);
  *whole = W;
  // (a limit so near the list's end that rounding decides goes the long way)
  return x * (1.0 - 1e-12) >= (double)s.p * W;
}

// The logits [*bottom, *top] of the bins that the boundary may lie in, by as much as the histogram may be
// off; c: the bins PB t .. of thread t. False where the bins do not reach it.
template <int PB, class SH>
__device__ __forceinline__ bool cut_range(SH& sh, const CutBins& bins, const RowSettings& s,
                                          const uint32_t (&c)[PB], double W, double want, float* top,
                                          float* bottom) {
  const int tid = item_id(), lane = tid & 63;
  double w[PB], sum = 0.0, total;
#pragma unroll
  for (int e = 0; e < PB; ++e) {
    w[e] = bins.weight_of(c[e], PB * tid + e);
    sum += w[e];
  }
  double run = block_scan(sh, sum, &total);
  const double off = bins.off(), eps = W * 1e-13, rest = (1.0 - (double)s.p) * W * 0x1p-8;
  int b0 = kCutBins, b1 = kCutBins;
#pragma unroll
  for (int e = 0; e < PB; ++e) {
    run += w[e];
    // the weight up to this bin's end: by what it is, or (all the row reached) by what follows
    double least = run * (1.0 - off), most = run * (1.0 + off);
    if (s.mp <= 0.0) {
      const double after = total - run;
      least = __builtin_fmax(least, W - after * (1.0 + off) - rest);
      most = __builtin_fmin(most, W - after * (1.0 - off));
    }
    if (most + eps >= want) b0 = min(b0, PB * tid + e);
    if (least - eps >= want) b1 = min(b1, PB * tid + e);
  }
  block_min_max(sh, 0, b0, -b1);
  // (with min_p the bins reach past all of S1, which the boundary is in)
  const int hi = min(-sh.i[1], s.mp > 0.0 ? kCutBins - 1 : kCutBins), lo = min(sh.i[0], hi);
  if (hi >= kCutBins) return false;
  // the bins' ends by bisection: the least key of bins [0, lo - 1] (lanes 0 .. 31) and of [0, hi]
  uint32_t kx = key_of(kNegInf) + 1, ky = key_of(bins.m);
  const float b = (float)(lane < 32 ? lo : hi + 1);
  auto probe = [&](uint32_t k) {
    if (bins.pos(of_key(k)) < b) ky = k;
    else kx = k + 1;
  };
  // (the first two next to where the end must lie: a few steps then, 30 without)
  const float far = b / bins.scale, near = far * 0x1p-20f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t k = key_of(bins.m - far + (j ? near : -near));
    if (k >= kx && k < ky) probe(k);
  }
  while (__ballot(kx < ky))
    if (kx < ky) probe(kx + (ky - kx) / 2);
  const uint32_t k_lo = (uint32_t)__shfl((int)kx, 0), k_hi = (uint32_t)__shfl((int)kx, 32);
  *top = lo == 0 ? bins.m : of_key(k_lo - 1);
  *bottom = of_key(k_hi);
  return true;
}

// An open nucleus, spread over the row's chunks: the bins of the histogram that the limit may lie
// in, by as much as its integers may be off; the tokens in them are listed, the weights above them
// summed by group; the pick finishes the row.
template <int DT>
__global__ __launch_bounds__(kSpread) void sample_spread_kernel(SampleParams p) {
  constexpr int EPL = Lane<DT, false>::EPL, IT = kChunk / (kSpread * EPL);
  __shared__ SpreadShared sh;
  const int part = wg_id_x(), row = wg_id_y();
  const int tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const RowSettings s = settings(p, row);
  if (s.greedy || s.k > 0 || s.p >= 1.f) return;
  const float low = p.low[row];
  const int first = p.count[(int64_t)row * p.chunks + min(lane, p.chunks - 1)];
  const float m = row_max(p, row);
  if (m == kNegInf) return;
  const double W = row_weight(p, row, m, s.inv2);
  int n;
  double w1;
  if (m == __builtin_inff() || settled(p, sh, row, s, low, first, m, W, &n, &w1)) {
    if (part == 0 && tid == 0) p.cut[row] = 0;
    return;
  }
  w1 = W;
  if (s.mp > 0.0) {  // W(S1)
    w1 = 0.0;
#pragma unroll 1
    for (int g = lane; g < p.groups; g += 64) w1 += p.sum_k[(int64_t)row * p.groups + g];
    w1 = wave_sum(w1);
  }
  const double want = (double)s.p * w1;
  const CutBins bins(m, s, p.vocab, W);
  // ---- thread t: bins PB t ..
  constexpr int PB = kCutBins / kSpread;
  static_assert(PB == 4, "a 16-byte load of bins");
  u32x4 c = {0u, 0u, 0u, 0u};
  {
    const u32x4* h = reinterpret_cast<const u32x4*>(p.hist + (int64_t)row * p.parts * kCutBins) + tid;
#pragma unroll 4
    for (int j = 0; j < p.parts; ++j) c += h[(int64_t)j * (kCutBins / 4)];
  }
  uint32_t cb[PB] = {c[0], c[1], c[2], c[3]};
  float ftop, fbottom;
  const bool cut = cut_range<PB>(sh, bins, s, cb, W, want, &ftop, &fbottom);
  if (part == 0 && tid == 0) p.cut[row] = cut ? 1 : 0;
  if (!cut) return;
  // ---- list what the bins hold, sum what lies above them
  const store_t<DT>* x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)row * p.ls;
  const int c0 = part * p.per, c1 = min(c0 + p.per, p.chunks);
  int* count = &sh.i[4];  // two, by turns
  u32x4 r[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
    r[i] = Lane<DT, false>::raw(x, c0 * kChunk + (i * kSpread + tid) * EPL, p.vocab);
  if (tid < 2) count[tid] = 0;
  __syncthreads();
#pragma unroll 1
  for (int ch = c0; ch < c1; ++ch) {
    uint64_t* to = p.cand2 + ((int64_t)row * p.chunks + ch) * kShort;
    int* held = &count[ch & 1];
    double* rd = sh.sums[ch & 1];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int i0 = ch * kChunk + (i * kSpread + tid) * EPL;
      Lane<DT, false> cur;
      cur.take(r[i], i0, p.vocab, p.vocab, ch * kChunk + (i + 1) * kSpread * EPL);
      double above = 0.0;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float l = cur.v[e];
        const bool take = l >= fbottom && l <= ftop;
        const uint64_t v = __ballot(take);
        if (v != 0) {  // uniform
          int at = 0;
          if (lane == 0) at = atomicAdd(held, __popcll(v));
          at = __builtin_amdgcn_readfirstlane(at) + __popcll(v & ((uint64_t(1) << lane) - 1));
          if (take && at < kShort) to[at] = rank_of(l, i0 + e);
        }
        if (__ballot(l > ftop)) above += l > ftop ? weight(l, m, s.inv2) : 0.0;
      }
      r[i] = Lane<DT, false>::raw(x, i0 + kChunk, p.vocab);
      above = wave_sum(above);
      if (lane == 0) rd[i * SpreadShared::NW + wave] = above;
    }
    __syncthreads();
    // (the next chunk uses the other word and row, and its barrier comes before these ones' reuse)
    if (tid == 0) {
      p.count2[(int64_t)row * p.chunks + ch] = *held;
      *held = 0;
    }
    put_group_sums<EPL>(p, p.sum_a, row, ch, rd);
  }
}

// The list sh.sorted[0 .. n) of a nucleus' bins, ordered; the place of the last kept token in it. above:
// the weight of what comes before the list.
__device__ __forceinline__ int cut_list(PickShared& sh, int n, const RowSettings& s, float m,
                                        double above, double want) {
  const int tid = item_id();
  sort_list(sh.sorted, n);
  constexpr int PL = kList / kPick;
  double w[PL], mine = 0.0, total;
#pragma unroll
  for (int e = 0; e < PL; ++e) {
    w[e] = PL * tid + e < n ? weight(logit_of(sh.sorted[PL * tid + e]), m, s.inv2) : 0.0;
    mine += w[e];
  }
  double before = above + block_scan(sh, mine, &total);
  int last = 0;
#pragma unroll
  for (int e = 0; e < PL; ++e) {
    if (PL * tid + e < n && before < want) last = PL * tid + e;
    before += w[e];
  }
  block_min_max(sh, 0, 0, last);
  return sh.i[1];
}

// A nucleus whose boundary's bins are listed (n tokens, sh.raw): ordered, the definition applied;
// then the token by the groups' weights.
template <int DT>
__device__ __forceinline__ int finish_cut(const SampleParams& p, const Row<DT, false>& row,
                                          PickShared& sh, int rowi, int n, const RowSettings& s,
                                          float m, double W, double u) {
  const int tid = item_id(), lane = tid & 63;
  const int64_t at = (int64_t)rowi * p.groups;
  double above = 0.0, w1 = W;
  if (s.mp > 0.0) w1 = 0.0;
#pragma unroll 1
  for (int g = lane; g < p.groups; g += 64) {
    above += p.sum_a[at + g];
    if (s.mp > 0.0) w1 += p.sum_k[at + g];
  }
  above = wave_sum(above);
  if (s.mp > 0.0) w1 = wave_sum(w1);
  const double want = (double)s.p * w1;
  for (int j = tid; j < n; j += kPick) sh.sorted[j] = sh.raw[j];
  __syncthreads();
  const int last = cut_list(sh, n, s, m, above, want);
  const uint64_t low = sh.sorted[last];
  // the listed tokens that are kept join their groups, as multiples of 2^-52 of the largest weight
  // (adding integers in any order gives the same sum)
  uint64_t* sums = reinterpret_cast<uint64_t*>(sh.ring);
  for (int g = tid; g < p.groups; g += kPick) sums[g] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kList / kPick; ++e) {
    const int j = kList / kPick * tid + e;
    if (j <= last) {
      const uint64_t r = sh.sorted[j];
      atomicAdd(reinterpret_cast<unsigned long long*>(&sums[index_of(r) / kGroup]),
                (unsigned long long)(weight(logit_of(r), m, s.inv2) * 0x1p52));
    }
  }
  __syncthreads();
  return draw_groups<DT>(
      sh, row.x, p.vocab, p.groups, u, [&](int g) { return p.sum_a[at + g] + (double)sums[g] * 0x1p-52; },
      [&](int i, float l) { return rank_of(l, i) >= low ? weight(l, m, s.inv2) : 0.0; });
}
static_assert(sizeof(PickShared::ring) >= kMaxVocab / kGroup * sizeof(double), "a sum per group");

// FILTER: rows may filter. (Without, a kernel of a tenth of the code, which comes cold from memory.)
template <int DT, bool FILTER>
__global__ __launch_bounds__(kPick) void sample_pick_kernel(SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) char pick_lds[];
  using SH = std::conditional_t<FILTER, PickShared, DrawShared>;
  SH& sh = *reinterpret_cast<SH*>(pick_lds);
  const int rowi = wg_id_x(), tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Row<DT, false> row;
  row.x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)rowi * p.ls;
  row.n = p.vocab;
  if constexpr (FILTER) row.ring = sh.ring;
  const RowSettings s = settings(p, rowi);
  if (s.greedy && wave > 0) return;  // one wave's work, no barrier
  const float uf = p.u[rowi];
  const double u = is_nan(uf) || uf < 0.f ? 0.0 : (double)fminf(uf, 0x1.fffffep-1f);
  const int64_t at = (int64_t)rowi * p.groups;
  const float* gm = p.gmax + at;
  // (on their way while the maximum is found; of rows that filter, the list's bound and counts)
  const int first = min(lane, p.groups - 1);
  const double sum_1 = p.sum_1[at + first], sum_t = p.sum_t[at + first];
  float low = kNegInf;
  int count = 0;
  if constexpr (FILTER) {
    low = p.low[rowi];
    count = p.count[(int64_t)rowi * p.chunks + min(lane, p.chunks - 1)];
  }
  const float m = row_max(p, rowi);
  if (m == kNegInf) {  // nothing to choose from (uniform)
    if (tid == 0) {
      p.tok[rowi] = -1;
      if (p.lp) p.lp[rowi] = kNegInf;
    }
    return;
  }
  // log of the row's sum at temperature 1 (m apart): the last wave's, beside the others' work
  if (p.lp && (s.greedy || wave == kWaves - 1)) {
    double r = 0.0;
#pragma unroll 1
    for (int g = lane; g < p.groups; g += 64)
      r += (g == lane ? sum_1 : p.sum_1[at + g]) * weight(gm[g], m, kLog2e);
    r = log(wave_sum(r));
    if (lane == 0) sh.logz = r;
  }
  int token = 0;
  if (s.greedy) {
    // the first group that holds the maximum, then its first element of that value
    int g0 = 0x7fffffff;
#pragma unroll 1
    for (int g = lane; g < p.groups; g += 64)
      if (gm[g] == m) g0 = min(g0, g);
    g0 = wave_min(g0);
    constexpr int EPL = Row<DT, false>::EPL;
    int f = 0x7fffffff;
#pragma unroll 1
    for (int i = g0 * kGroup + (kGroup / 64 - EPL) + kGroup / 64 * lane; i >= g0 * kGroup + kGroup / 64 * lane; i -= EPL) {
      Lane<DT, false> a;
      a.take(Lane<DT, false>::raw(row.x, i, row.n), i, row.n, row.n, (g0 + 1) * kGroup);
#pragma unroll
      for (int e = EPL - 1; e >= 0; --e)
        if (a.v[e] == m) f = i + e;
    }
    token = wave_min(f);
  } else if (!FILTER || !s.filtered()) {
    token = draw_groups<DT>(
        sh, row.x, p.vocab, p.groups, u,
        [&](int g) {
          return (p.groups <= 64 ? sum_t : p.sum_t[at + g]) * weight(gm[g], m, s.inv2);
        },
        [&](int, float l) { return weight(l, m, s.inv2); });
  } else if constexpr (FILTER) {
    const double W = s.k == 0 ? row_weight(p, rowi, m, s.inv2) : 0.0;
    int n = 0;
    double whole = -1.0;
    if (settled(p, sh, rowi, s, low, count, m, W, &n, &whole)) {
      token = pick_short(sh, n, s, m, whole, u);
    } else if (s.k == 0 && s.p >= 1.f) {
      // the tokens of weight >= min_p
      token = draw_groups<DT>(
          sh, row.x, p.vocab, p.groups, u, [&](int g) { return p.sum_k[at + g]; },
          [&](int, float l) {
            const double w = weight(l, m, s.inv2);
            return w >= s.mp ? w : 0.0;
          });
    } else {
      n = kList + 1;
      if (s.k == 0 && p.cut[rowi] != 0) {
        __syncthreads();  // (the list that did not settle it is done with)
        const int32_t* counts = p.count2 + (int64_t)rowi * p.chunks;
        n = collect(sh, counts, counts[min(lane, p.chunks - 1)],
                    p.cand2 + (int64_t)rowi * p.chunks * kShort, p.chunks, kList);
      }
      token = n > 0 && n <= kList ? finish_cut(p, row, sh, rowi, n, s, m, W, u)
                                  : pick_wide(row, sh, s, m, W, u);
    }
  }
  // (every way here but the greedy one has passed barriers since sh.logz was written)
  if (tid == 0) {
    p.tok[rowi] = token;
    if (p.lp) {
      const float l = load1<DT>(row.x, token);
      const double d = l >= m ? 0.0 : (double)l - (double)m;
      p.lp[rowi] = (float)(d - sh.logz);
    }
  }
}

// ---- small vocabularies ------------------------------------------------------------------------
// A row in the registers of one workgroup, 8 or 16 logits a thread: one launch. top_k: the k-th largest of
// the threads' maxima bounds the list, as in the gather; a nucleus: its histogram in LDS, then the
// boundary's bins listed.
constexpr int kSmall = 16 * kPick;
static_assert(sizeof(PickShared::bin) >= kCutBins * 4 && sizeof(PickShared::bin) >= kPick * 4, "");

template <int DT, bool TINY, int PER>
__global__ __launch_bounds__(kPick) void sample_small_kernel(SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) char pick_lds[];
  PickShared& sh = *reinterpret_cast<PickShared*>(pick_lds);
  constexpr int EPL = Lane<DT, TINY>::EPL;
  const int rowi = wg_id_x(), tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Row<DT, TINY> row;
  row.x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)rowi * p.ls;
  row.n = p.vocab;
  row.ring = sh.ring;
  const int i0 = PER * tid;
  u32x4 raw[PER / EPL];
#pragma unroll
  for (int j = 0; j < PER / EPL; ++j) raw[j] = Lane<DT, TINY>::raw(row.x, i0 + j * EPL, p.vocab);
  const RowSettings s = settings(p, rowi);
  const float uf = p.u[rowi];
  const double u = is_nan(uf) || uf < 0.f ? 0.0 : (double)fminf(uf, 0x1.fffffep-1f);
  float v[PER];
  float mine = kNegInf;
#pragma unroll
  for (int j = 0; j < PER / EPL; ++j) {
    Lane<DT, TINY> a;
    a.take(raw[j], i0 + j * EPL, p.vocab, p.vocab, (wave + 1) * 64 * PER);
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      v[j * EPL + e] = a.v[e];
      mine = fmaxf(mine, a.v[e]);
    }
  }
  {
    const float x = wave_max_all(mine);
    if (lane == 0) sh.red[wave] = x;
    __syncthreads();
  }
  float m = kNegInf;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, (float)sh.red[w]);
  if (m == kNegInf) {  // nothing to choose from (uniform)
    if (tid == 0) {
      p.tok[rowi] = -1;
      if (p.lp) p.lp[rowi] = kNegInf;
    }
    return;
  }
  double logz = 0.0;
  if (p.lp) {  // f32 exponentials, as in the scan
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      x += fast_exp2((v[e] >= m ? 0.f : v[e] - m) * 1.44269504088896340736f);
    logz = block_sum(sh, (double)x);
  }
  int token = -1;
  uint64_t low = 0;  // kept: ranks from here up, of weight >= min_p
  if (s.greedy) {
    int f = 0x7fffffff;
#pragma unroll
    for (int e = PER - 1; e >= 0; --e)
      if (v[e] == m) f = i0 + e;
    block_min_max(sh, 0, f, 0);
    token = sh.i[0];
  } else {
    if (s.k > 0) {
      // ---- a list of the first k (sh.n: how many are listed)
      float* top = reinterpret_cast<float*>(sh.bin);
      top[tid] = mine;
      if (tid == 0) sh.n = 0;
      __syncthreads();
      const int n_top = (p.vocab + PER - 1) / PER;
      if (wave == 0) {
        const float b = s.k <= n_top ? list_bound<kPick / 64>([&](int g) { return top[g]; }, n_top, s.k) : kNegInf;
        if (lane == 0) sh.logz = (double)b;
      }
      __syncthreads();
      const float bound = (float)sh.logz;
#pragma unroll
      for (int e = 0; e < PER; ++e) append(sh, v[e] >= bound && v[e] > kNegInf, v[e], i0 + e);
      __syncthreads();
      const int n = sh.n;
      if (n <= kShort) {
        token = pick_short(sh, n, s, m, -1.0, u);
      } else if (n <= kList) {
        for (int j = tid; j < n; j += kPick) sh.sorted[j] = sh.raw[j];
        __syncthreads();
        sort_list(sh.sorted, n);
        constexpr int PL = kList / kPick;
        double w[PL], sum = 0.0, total;
        bool in1[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) {
          const int j = PL * tid + e;
          w[e] = j < min(n, s.k) ? weight(logit_of(sh.sorted[j]), m, s.inv2) : 0.0;
          in1[e] = j < min(n, s.k) && w[e] >= s.mp;
          if (!in1[e]) w[e] = 0.0;
          sum += w[e];
        }
        double run = block_scan(sh, sum, &total);
        const double limit = (double)s.p * total;
        int last = 0;
#pragma unroll
        for (int e = 0; e < PL; ++e) {
          if (in1[e] && (s.p >= 1.f || run < limit)) last = PL * tid + e;
          run += w[e];
        }
        block_min_max(sh, 0, 0, last);
        low = sh.sorted[sh.i[1]];
      } else {
        token = pick_wide(row, sh, s, m, 0.0, u);
      }
    } else if (s.p < 1.f) {
      double x = 0.0, y = 0.0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const double w = weight(v[e], m, s.inv2);
        x += w;
        y += w >= s.mp ? w : 0.0;
      }
      const double W = block_sum(sh, x), w1 = s.mp > 0.0 ? block_sum(sh, y) : W;
      const double want = (double)s.p * w1;
      bool cut = m != __builtin_inff();
      if (cut) {  // uniform
        for (int b = tid; b < kCutBins; b += kPick) sh.bin[b] = 0;
        if (tid == 0) sh.n = 0;
        __syncthreads();
        const CutBins bins(m, s, p.vocab, W);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const float at = bins.pos(v[e]);
          if (at < (float)kCutBins) atomicAdd(&sh.bin[(int)at], bins.value(v[e], (int)at));
        }
        __syncthreads();
        constexpr int PB = kCutBins / kPick;
        uint32_t c[PB];
#pragma unroll
        for (int e = 0; e < PB; ++e) c[e] = sh.bin[PB * tid + e];
        float ftop, fbottom;
        cut = cut_range<PB>(sh, bins, s, c, W, want, &ftop, &fbottom);
        if (cut) {
          x = 0.0;
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            append(sh, v[e] >= fbottom && v[e] <= ftop, v[e], i0 + e);
            if (__ballot(v[e] > ftop)) x += v[e] > ftop ? weight(v[e], m, s.inv2) : 0.0;
          }
          const double above = block_sum(sh, x);
          const int n = sh.n;
          cut = n > 0 && n <= kList;
          if (cut) {
            for (int j = tid; j < n; j += kPick) sh.sorted[j] = sh.raw[j];
            __syncthreads();
            low = sh.sorted[cut_list(sh, n, s, m, above, want)];
          }
        }
      }
      if (!cut) token = pick_wide(row, sh, s, m, W, u);
    }
    if (token < 0) {
      // ---- the kept weights in index order
      double w[PER], sum = 0.0, total;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        w[e] = rank_of(v[e], i0 + e) >= low ? weight(v[e], m, s.inv2) : 0.0;
        if (!(w[e] >= s.mp)) w[e] = 0.0;
        sum += w[e];
      }
      double run = block_scan(sh, sum, &total);
      const double target = u * total;
      int hit = 0x7fffffff, last = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (w[e] > 0.0) {
          last = i0 + e;
          if (run + w[e] > target) hit = min(hit, last);
        }
        run += w[e];
      }
      block_min_max(sh, 0, hit, last);
      token = sh.i[0] != 0x7fffffff ? sh.i[0] : sh.i[1];
    }
  }
  if (tid == 0) {
    p.tok[rowi] = token;
    if (p.lp) {
      const float l = load1<DT>(row.x, token);
      const double d = l >= m ? 0.0 : (double)l - (double)m;
      p.lp[rowi] = (float)(d - log(logz));
    }
  }
}

template <class K>
hipError_t large_lds(K kernel) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PickShared));
}

// (TINY: fewer tokens than a lane's load)
template <int DT, bool TINY, int PER>
hipError_t launch_small(const SampleParams& p, hipStream_t st) {
  static const hipError_t once = large_lds(sample_small_kernel<DT, TINY, PER>);
  if (once != hipSuccess) return once;
  hipLaunchKernelGGL((sample_small_kernel<DT, TINY, PER>), dim3((unsigned)p.rows), dim3(kPick),
                     sizeof(PickShared), st, p);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_sample(const SampleParams& p, hipStream_t st) {
  if (p.vocab < Lane<DT, false>::EPL) return launch_small<DT, true, 8>(p, st);
  if (p.vocab <= kSmall / 2) return launch_small<DT, false, 8>(p, st);
  // what rows may do, as far as the host knows
  const bool counts = p.k || p.k_all > 0, nuclei = p.p || p.p_all < 1.f;
  const bool minima = p.mp || p.mp_all > 0.f, all_count = !p.k && p.k_all > 0 && p.k_all < p.vocab;
  const bool filter = counts || nuclei || minima;
  // (16 logits a thread: 113 x 10101 top-p 38 us, 52 in four launches; 31 x 8691 without a filter 14.5
  // us, 12.9 in two)
  if (p.vocab <= kSmall && filter) return launch_small<DT, false, 16>(p, st);
  static const hipError_t once = large_lds(sample_pick_kernel<DT, true>);
  if (once != hipSuccess) return once;
  const unsigned rows = (unsigned)p.rows;
  hipLaunchKernelGGL(sample_scan_kernel<DT>, dim3((unsigned)((p.groups + 3) / 4), rows), dim3(256), 0,
                     st, p);
  if (!filter) {
    hipLaunchKernelGGL((sample_pick_kernel<DT, false>), dim3(rows), dim3(kPick), sizeof(DrawShared), st,
                       p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(sample_gather_kernel<DT>, dim3((unsigned)p.parts, rows), dim3(256), 0, st, p);
  if (nuclei && !all_count)
    hipLaunchKernelGGL(sample_spread_kernel<DT>, dim3((unsigned)p.parts, rows), dim3(kSpread), 0, st, p);
  hipLaunchKernelGGL((sample_pick_kernel<DT, true>), dim3(rows), dim3(kPick), sizeof(PickShared), st, p);
  return hipGetLastError();
}

int check_sample_sizes(int32_t rows, int32_t vocab) {
  if (rows < 0 || rows > 65535) return api_fail(FFAI_ERR_INVALID, "rows must be in [0, 65535]");
  if (vocab < 1 || vocab > kMaxVocab) return api_fail(FFAI_ERR_INVALID, "vocab must be in [1, 2^20]");
  return FFAI_OK;
}
// Chunks of a gather workgroup: four where that leaves enough of them (each finds the row's bound by
// itself), and so many that a row has kParts at most (a nucleus reads all their histograms).
int32_t sample_per(int32_t rows, int32_t chunks) {
  const int32_t per = (int64_t)chunks * rows >= 4096 ? 4 : 1;
  return std::max(per, (chunks + kParts - 1) / kParts);
}
// The workspace's parts, in order, each 16-byte aligned.
struct SampleSpace {
  size_t sum_t, sum_1, sum_k, sum_a, cand, cand2, hist, gmax, smax, low, count, count2, cut,
      bytes;
};
SampleSpace sample_space(int32_t rows, int32_t vocab) {
  const size_t g = (size_t)rows * ((vocab + kGroup - 1) / kGroup);
  const int32_t chunks = (vocab + kChunk - 1) / kChunk;
  const size_t c = (size_t)rows * chunks;
  const int32_t per = sample_per(rows, chunks);
  SampleSpace s{};
  auto take = [&](size_t n) {
    const size_t at = s.bytes;
    s.bytes += (n + 15) & ~size_t(15);
    return at;
  };
  s.sum_t = take(g * 8);
  s.sum_1 = take(g * 8);
  s.sum_k = take(g * 8);
  s.sum_a = take(g * 8);
  s.cand = take(c * kShort * 8);
  s.cand2 = take(c * kShort * 8);
  s.hist = take((size_t)rows * ((chunks + per - 1) / per) * kCutBins * 4);
  s.gmax = take(g * 4);
  s.smax = take(g * 64);
  s.low = take((size_t)rows * 4);
  s.count = take(c * 4);
  s.count2 = take(c * 4);
  s.cut = take((size_t)rows * 4);
  return s;
}

}  // namespace
}  // namespace ffai

using namespace ffai;

extern "C" {

int ffai_sample_workspace_bytes(int32_t rows, int32_t vocab, size_t* bytes) {
  api_clear_error();
  if (!bytes) return api_fail(FFAI_ERR_INVALID, "null bytes pointer");
  const int rc = check_sample_sizes(rows, vocab);
  if (rc != FFAI_OK) return rc;
  *bytes = sample_space(rows, vocab).bytes;
  return FFAI_OK;
}

int ffai_sample(const void* logits, int32_t logits_dtype, int32_t rows, int32_t vocab,
                int64_t logits_row_stride, const float* temperature, float temperature_all,
                const int32_t* top_k, int32_t top_k_all, const float* top_p, float top_p_all,
                const float* min_p, float min_p_all, const float* u, int32_t* tokens,
                float* logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  api_clear_error();
  int rc = check_sample_sizes(rows, vocab);
  if (rc != FFAI_OK) return rc;
  if (logits_dtype != FFAI_F32 && logits_dtype != FFAI_F16 && logits_dtype != FFAI_BF16)
    return api_fail(FFAI_ERR_INVALID, "unknown logits dtype");
  if (rows == 0) return FFAI_OK;
  if (!logits || !u || !tokens) return api_fail(FFAI_ERR_INVALID, "null pointer");
  if ((uintptr_t)logits % (logits_dtype == FFAI_F32 ? 4 : 2))
    return api_fail(FFAI_ERR_INVALID, "logits must be aligned to their element size");
  if ((uintptr_t)temperature % 4 || (uintptr_t)top_k % 4 || (uintptr_t)top_p % 4 ||
      (uintptr_t)min_p % 4 || (uintptr_t)u % 4 || (uintptr_t)tokens % 4 || (uintptr_t)logprobs % 4)
    return api_fail(FFAI_ERR_INVALID, "settings, u and outputs must be 4-byte aligned");
  if (logits_row_stride < 0)
    return api_fail(FFAI_ERR_INVALID, "logits row stride must not be negative");
  if (!workspace || workspace_bytes < sample_space(rows, vocab).bytes)
    return api_fail(FFAI_ERR_WORKSPACE, "workspace smaller than ffai_sample_workspace_bytes");
  if ((uintptr_t)workspace % 16) return api_fail(FFAI_ERR_INVALID, "workspace must be 16-byte aligned");
  rc = api_check_device();
  if (rc != FFAI_OK) return rc;
  SampleParams p{};
  p.logits = logits; p.ls = logits_row_stride; p.rows = rows; p.vocab = vocab;
  p.groups = (vocab + kGroup - 1) / kGroup;
  p.t = temperature; p.t_all = temperature_all;
  p.k = top_k; p.k_all = top_k_all;
  p.p = top_p; p.p_all = top_p_all;
  p.mp = min_p; p.mp_all = min_p_all;
  p.u = u; p.tok = tokens; p.lp = logprobs;
  p.chunks = (vocab + kChunk - 1) / kChunk;
  const SampleSpace sp = sample_space(rows, vocab);
  char* ws = static_cast<char*>(workspace);
  p.sum_t = reinterpret_cast<double*>(ws + sp.sum_t);
  p.sum_1 = reinterpret_cast<double*>(ws + sp.sum_1);
  p.cand = reinterpret_cast<uint64_t*>(ws + sp.cand);
  p.gmax = reinterpret_cast<float*>(ws + sp.gmax);
  p.smax = reinterpret_cast<float*>(ws + sp.smax);
  p.low = reinterpret_cast<float*>(ws + sp.low);
  p.count = reinterpret_cast<int32_t*>(ws + sp.count);
  p.sum_k = reinterpret_cast<double*>(ws + sp.sum_k);
  p.sum_a = reinterpret_cast<double*>(ws + sp.sum_a);
  p.cand2 = reinterpret_cast<uint64_t*>(ws + sp.cand2);
  p.hist = reinterpret_cast<uint32_t*>(ws + sp.hist);
  p.count2 = reinterpret_cast<int32_t*>(ws + sp.count2);
  p.cut = reinterpret_cast<int32_t*>(ws + sp.cut);
  p.per = sample_per(rows, p.chunks);
  p.parts = (p.chunks + p.per - 1) / p.per;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = logits_dtype == FFAI_F32   ? launch_sample<kF32>(p, st)
                       : logits_dtype == FFAI_F16 ? launch_sample<kF16>(p, st)
                                                  : launch_sample<kBF16>(p, st);
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  return FFAI_OK;
}

}  // extern "C"
