// Sampling of one token per row of logits (include/ffai_sample.h).
//
// Two launches. sample_scan_kernel reads the logits once, spread over the whole GPU: per chunk of
// a row its maximum and weight sums, per 1024 elements their maximum. sample_pick_kernel, one
// workgroup a row, joins them and finds the token:
//   * no filter: the chunk that holds u W by a scan of the chunks' sums, then the token in it;
//   * filters: nearly always few tokens can be kept. The k-th largest of the 1024-element maxima
//     bounds the k-th largest logit from below, so one pass collects everything from there up
//     (k + a few tokens) in LDS, where it is sorted and the definition is applied as it stands;
//   * otherwise (thousands of tokens kept, many equal ones): the boundary is found by histograms
//     of counts or weights, finer each time, down to a list or a single value.
// Weights are 64-bit throughout: a token's share may be 1e-5 of the row's, and with f32 sums the
// token at a given u would depend on the order of summation. f64 FMAs run at the f32 rate here;
// an exponential is 20 of them. Histogram weights alone are integers (2^-43 steps: adding them in
// any order gives the same sum), and what they decide is confirmed with f64 sums.
#include "../../include/ffai_sample.h"

#include <algorithm>

#include "attn_common.cuh"

namespace ffai {
namespace {

constexpr int kChunk = 4096;  // elements of a scan workgroup
constexpr int kGroup = 1024;  // elements of one of its waves
constexpr int kMaxVocab = 1 << 20;
constexpr int kPick = 1024;  // threads of a pick workgroup
constexpr int kList = 2048;  // tokens of an LDS list
constexpr int kBins = 2048;
constexpr int kSegs = 4096;  // ordered segments of a row at most (kMaxVocab / (64 * 4))

struct SampleParams {
  const void* logits;
  int64_t ls;
  int32_t rows, vocab, chunks;
  const float* t;
  const int32_t* k;
  const float* p;
  const float* mp;
  float t_all, p_all, mp_all;
  int32_t k_all;
  const float* u;
  int32_t* tok;
  float* lp;
  double* sum_t;   // [row][chunk] sum of exp((l - chunk max) / T)
  double* sum_1;   // [row][chunk] sum of exp(l - chunk max)
  float* gmax;     // [row][chunk * 4 + wave] maxima
  int32_t* first;  // [row][chunk] index of the chunk's first maximum
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

struct RowSettings {
  bool greedy;
  double inv;  // 1 / T
  int k;       // 0: off
  float p;     // 1: off
  double mp;   // 0: off
  __device__ bool filtered() const { return k > 0 || p < 1.f || mp > 0.0; }
};
__device__ __forceinline__ RowSettings settings(const SampleParams& p, int row) {
  RowSettings s;
  const float t = p.t ? p.t[row] : p.t_all;
  const uint32_t tb = __float_as_uint(t);
  s.greedy = !(tb > 0u && tb <= 0x7f800000u);  // positive, infinity included
  s.inv = 1.0 / (double)t;
  const int k = p.k ? p.k[row] : p.k_all;
  s.k = k <= 0 || k >= p.vocab ? 0 : k;
  const float tp = p.p ? p.p[row] : p.p_all;
  s.p = is_nan(tp) || tp >= 1.f ? 1.f : tp;
  const float mp = p.mp ? p.mp[row] : p.mp_all;
  s.mp = is_nan(mp) || mp <= 0.f ? 0.0 : (double)fminf(mp, 1.f);
  return s;
}

// exp(z), z <= 0: z = n ln 2 + r, |r| <= ln 2 / 2, by two-part reduction, exp(r) by its Taylor sum
// to r^13 / 13! (the next term is below 2^-58), times 2^n.
__device__ __forceinline__ double exp_neg(double z) {
  if (z < -745.0) return 0.0;
  const double n = __builtin_rint(z * 1.4426950408889634074);
  double r = __builtin_fma(-n, 0x1.62e42fefa3800p-1, z);  // ln 2, its leading 42 bits
  r = __builtin_fma(-n, 0x1.ef35793c76730p-45, r);        // and the rest
  double e = 1.0 / 6227020800.0;
  e = __builtin_fma(e, r, 1.0 / 479001600.0);
  e = __builtin_fma(e, r, 1.0 / 39916800.0);
  e = __builtin_fma(e, r, 1.0 / 3628800.0);
  e = __builtin_fma(e, r, 1.0 / 362880.0);
  e = __builtin_fma(e, r, 1.0 / 40320.0);
  e = __builtin_fma(e, r, 1.0 / 5040.0);
  e = __builtin_fma(e, r, 1.0 / 720.0);
  e = __builtin_fma(e, r, 1.0 / 120.0);
  e = __builtin_fma(e, r, 1.0 / 24.0);
  e = __builtin_fma(e, r, 1.0 / 6.0);
  e = __builtin_fma(e, r, 0.5);
  e = __builtin_fma(e, r, 1.0);
  e = __builtin_fma(e, r, 1.0);
  return __builtin_ldexp(e, (int)n);
}
// A token's weight against the largest logit m. (l < m strictly below: 1 at m even where both
// are infinite.)
__device__ __forceinline__ double weight(float l, float m, double inv) {
  if (l >= m) return l == kNegInf ? 0.0 : 1.0;
  if (l == kNegInf || m == __builtin_inff()) return 0.0;
  return exp_neg(((double)l - (double)m) * inv);
}

template <int DT>
__device__ __forceinline__ float load1(const store_t<DT>* x, int i) {
  if constexpr (DT == kF32) return nan_to_low(x[i]);
  else return nan_to_low(to_f32<DT>(x[i]));
}
// EPL consecutive logits from index i; -inf past the row's end.
template <int DT>
struct Lane {
  static constexpr int EPL = DT == kF32 ? 4 : 8;
  float v[EPL];
  __device__ __forceinline__ void load(const store_t<DT>* x, int i, int n) {
    if (i + EPL <= n) {
      if constexpr (DT == kF32) {
        const f32x4 a = *reinterpret_cast<const f32x4_e*>(x + i);
#pragma unroll
        for (int e = 0; e < EPL; ++e) v[e] = nan_to_low(a[e]);
      } else {
        const u32x4 a = ld16h(x + i);
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          v[e] = nan_to_low(to_f32<DT>((e & 1) ? a[e >> 1] >> 16 : a[e >> 1] & 0xffffu));
      }
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = i + e < n ? load1<DT>(x, i + e) : kNegInf;
    }
  }
};

template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v += __shfl_xor(v, s);
  return v;
}

// ---- scan --------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void sample_scan_kernel(SampleParams p) {
  constexpr int EPL = Lane<DT>::EPL, IT = kGroup / (64 * EPL);
  const int row = wg_id_y(), chunk = wg_id_x(), tid = item_id();
  const int lane = tid & 63, wave = tid >> 6;
  const store_t<DT>* x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)row * p.ls;
  const int base = chunk * kChunk + wave * kGroup;
  Lane<DT> a[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) a[i].load(x, base + (i * 64 + lane) * EPL, p.vocab);
  const RowSettings s = settings(p, row);
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int e = 0; e < EPL; ++e) m = fmaxf(m, a[i].v[e]);
  m = wave_max_all(m);
  __shared__ float wm[4];
  __shared__ int wf[4];
  __shared__ double wt[4], w1[4];
  if (lane == 0) {
    wm[wave] = m;
    p.gmax[((int64_t)row * p.chunks + chunk) * 4 + wave] = m;
  }
  int first = 0x7fffffff;
#pragma unroll
  for (int i = IT - 1; i >= 0; --i)
#pragma unroll
    for (int e = EPL - 1; e >= 0; --e)
      if (a[i].v[e] == m) first = base + (i * 64 + lane) * EPL + e;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d));
  if (lane == 0) wf[wave] = first;
  __syncthreads();
  const float cm = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  // the weights' sum is needed unless the kept tokens are listed anyway (top-k) or the row is
  // greedy; the sum at temperature 1 for the log-probability
  const bool need_t = !s.greedy && s.k == 0 && s.inv != 1.0;
  double st = 0.0, s1 = 0.0;
  if (cm != kNegInf) {
    if (need_t) {
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < EPL; ++e) st += weight(a[i].v[e], cm, s.inv);
    }
    if (!s.greedy && s.k == 0 && s.inv == 1.0) {
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < EPL; ++e) s1 += weight(a[i].v[e], cm, 1.0);
    } else if (p.lp) {
      // f32 exponentials (relative error about 2^-22 each, of either sign) summed in f64: the
      // log-probability is an f32 number
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const float d = a[i].v[e] >= cm ? 0.f : a[i].v[e] - cm;
          q += fast_exp2(d * 1.44269504088896340736f);
        }
      s1 = (double)q;
    }
  }
  st = wave_sum(st);
  s1 = wave_sum(s1);
  if (lane == 0) {
    wt[wave] = st;
    w1[wave] = s1;
  }
  __syncthreads();
  if (tid == 0) {
    const int64_t at = (int64_t)row * p.chunks + chunk;
    const double b = (w1[0] + w1[1]) + (w1[2] + w1[3]);
    p.sum_1[at] = b;
    p.sum_t[at] = need_t ? (wt[0] + wt[1]) + (wt[2] + wt[3]) : b;
    int f = 0x7fffffff;
#pragma unroll
    for (int w = 3; w >= 0; --w)
      if (wm[w] == cm) f = wf[w];
    p.first[at] = f;
  }
}

// ---- pick --------------------------------------------------------------------------------------
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

struct PickShared {
  uint64_t list[kList];    // ranks in index order
  uint64_t sorted[kList];  // ranks, earliest first
  uint64_t wbin[kBins];    // weights in 2^-43 steps
  uint32_t cbin[kBins];
  double seg[kSegs];
  double red[16];
  int cnt[2][4][16];
  double d[4];
  uint64_t r[2];
  uint32_t q[4];
  int i[8];
};

// The sum over the workgroup, the same bits in every thread.
__device__ __forceinline__ double block_sum(PickShared& sh, double v) {
  v = wave_sum(v);
  __syncthreads();
  if ((item_id() & 63) == 0) sh.red[item_id() >> 6] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) t += sh.red[w];
  return t;
}
// Exclusive prefix sum over the workgroup's threads, and the whole sum.
__device__ __forceinline__ double block_scan(PickShared& sh, double v, double* total) {
  const int lane = item_id() & 63, wave = item_id() >> 6;
  double x = v;
#pragma unroll
  for (int s = 1; s < 64; s *= 2) {
    const double y = __shfl_up(x, s);
    if (lane >= s) x += y;
  }
  double e = __shfl_up(x, 1);
  if (lane == 0) e = 0.0;
  __syncthreads();
  if (lane == 63) sh.red[wave] = x;
  __syncthreads();
  double before = 0.0, t = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
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
  if ((item_id() & 63) == 0) sh.cnt[0][0][item_id() >> 6] = (int)v;
  __syncthreads();
  uint32_t t = (uint32_t)sh.cnt[0][0][0];
#pragma unroll
  for (int w = 1; w < 16; ++w) t = f(t, (uint32_t)sh.cnt[0][0][w]);
  return t;
}

// Descending bitonic sort of sorted[0 .. n) padded with zeros (below every rank) to a power of two.
__device__ __forceinline__ void sort_list(PickShared& sh, int n) {
  int n2 = 2;
  while (n2 < n) n2 *= 2;
  const int tid = item_id();
  for (int i = n + tid; i < n2; i += kPick) sh.sorted[i] = 0;
  __syncthreads();
  auto step = [&](int size, int stride, int t) {
    const int lo = 2 * t - (t & (stride - 1)), hi = lo + stride;
    const uint64_t a = sh.sorted[lo], b = sh.sorted[hi];
    const bool down = (lo & size) == 0;
    if ((a < b) == down) {
      sh.sorted[lo] = b;
      sh.sorted[hi] = a;
    }
  };
  if (n2 <= 128) {  // one wave, whose LDS accesses are in order
    if (tid < 64)
      for (int size = 2; size <= n2; size *= 2)
        for (int stride = size / 2; stride > 0; stride /= 2) {
          if (tid < n2 / 2) step(size, stride, tid);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
    __syncthreads();
  } else {
    for (int size = 2; size <= n2; size *= 2)
      for (int stride = size / 2; stride > 0; stride /= 2) {
        for (int t = tid; t < n2 / 2; t += kPick) step(size, stride, t);
        __syncthreads();
      }
  }
}

template <int DT>
struct Row {
  static constexpr int EPL = Lane<DT>::EPL;
  static constexpr int TILE = kPick * EPL;
  const store_t<DT>* x;
  int n;
  // f(index, logit) of every element, in no order
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int U = 4;  // tiles whose loads are in flight together
#pragma unroll 1
    for (int b = item_id() * EPL; b < n; b += U * TILE) {
      Lane<DT> a[U];
#pragma unroll
      for (int j = 0; j < U; ++j) a[j].load(x, min(b + j * TILE, n), n);
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) f(b + j * TILE + e, a[j].v[e]);
    }
  }
};

// The ranks of the elements that `take` chooses, in index order, to sh.list (the first kList of
// them) and sh.sorted alike. Returns how many there are. One barrier per U tiles: each wave says
// how many it keeps of each tile, and every thread adds up what lies before its own.
template <int DT, class F>
__device__ __forceinline__ int collect(const Row<DT>& row, PickShared& sh, F take) {
  constexpr int EPL = Row<DT>::EPL, TILE = Row<DT>::TILE, U = 4;
  const int tid = item_id(), lane = tid & 63, wave = tid >> 6;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  int n = 0, flip = 0;
  __syncthreads();
#pragma unroll 1
  for (int b0 = 0; b0 < row.n; b0 += U * TILE) {
    Lane<DT> a[U];
#pragma unroll
    for (int j = 0; j < U; ++j) a[j].load(row.x, min(b0 + j * TILE + tid * EPL, row.n), row.n);
    uint32_t mine = 0;  // bit j * EPL + e
    int before[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      int all = 0;
      before[j] = 0;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float l = a[j].v[e];
        const bool t = l != kNegInf && take(b0 + j * TILE + tid * EPL + e, l);
        const uint64_t v = __ballot(t);
        before[j] += __popcll(v & below);
        all += __popcll(v);
        mine |= (uint32_t)t << (j * EPL + e);
      }
      if (lane == 0) sh.cnt[flip][j][wave] = all;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < U; ++j) {
      int at = n + before[j];
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const int c = sh.cnt[flip][j][w];
        if (w < wave) at += c;
        n += c;
      }
      if ((mine >> (j * EPL)) & ((1u << EPL) - 1)) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if ((mine >> (j * EPL + e)) & 1) {
            if (at < kList) {
              const uint64_t r = rank_of(a[j].v[e], b0 + j * TILE + tid * EPL + e);
              sh.list[at] = r;
              sh.sorted[at] = r;
            }
            ++at;
          }
      }
    }
    flip ^= 1;
  }
  __syncthreads();
  return n;
}

// The element at which the running weight passes u times the whole, over elements in order: `w`
// (0 for one that is not kept) of PER consecutive positions per thread. Every thread returns the
// position (threads' elements are PER * tid + e).
template <int PER>
__device__ __forceinline__ int draw(PickShared& sh, const double (&w)[PER], double u) {
  double mine = 0.0, total;
#pragma unroll
  for (int e = 0; e < PER; ++e) mine += w[e];
  double run = block_scan(sh, mine, &total);
  const double target = u * total;
  if (item_id() == 0) {
    sh.i[6] = 0x7fffffff;
    sh.i[7] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    run += w[e];
    if (w[e] > 0.0) {
      if (run > target) atomicMin(&sh.i[6], PER * (int)item_id() + e);
      atomicMax(&sh.i[7], PER * (int)item_id() + e);
    }
  }
  __syncthreads();
  // (rounding may leave every running sum at or below u times the whole: then the last one)
  const int at = sh.i[6];
  const int last = sh.i[7];
  __syncthreads();
  return at != 0x7fffffff ? at : last;
}

// What is kept of a row: ranks from `low` up, of weight at least mp.
struct Kept {
  uint64_t low;
  double mp;
};

// The token of a row whose every kept element is in sh.list[0 .. n): the definition as it stands.
// whole: W(S1) where S1 reaches below the list (top_k and min_p off), else negative.
__device__ int pick_from_list(PickShared& sh, int n, const RowSettings& s, float m, double whole,
                              double u) {
  sort_list(sh, n);
  const int tid = item_id();
  double w[2];
  bool in1[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int j = 2 * tid + e;
    w[e] = j < n ? weight(logit_of(sh.sorted[j]), m, s.inv) : 0.0;
    in1[e] = j < n && (s.k == 0 || j < s.k) && w[e] >= s.mp;
    if (!in1[e]) w[e] = 0.0;
  }
  double total;
  const double before = block_scan(sh, w[0] + w[1], &total);
  const double limit = (double)s.p * (whole >= 0.0 ? whole : total);
  // the last rank that is kept (in1 and the running weight make it a run from the first)
  if (tid == 0) sh.i[5] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const double b = e == 0 ? before : before + w[0];
    if (in1[e] && (s.p >= 1.f || b < limit)) atomicMax(&sh.i[5], 2 * tid + e);
  }
  __syncthreads();
  const uint64_t low = sh.sorted[sh.i[5]];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int j = 2 * tid + e;
    const uint64_t r = j < n ? sh.list[j] : 0;
    w[e] = r >= low && j < n ? weight(logit_of(r), m, s.inv) : 0.0;
  }
  return index_of(sh.list[draw<2>(sh, w, u)]);
}

// The last rank that is kept when ranks `from` and earlier of weight >= mp are cut at a count
// (by_count: the first `count`) or at a weight (those whose predecessors weigh less than `limit`).
// Histograms over the logits, first linear below m, then over ever smaller ranges of their integer
// keys, until the boundary's bin holds a list's worth of tokens or a single value.
template <int DT>
__device__ uint64_t boundary(const Row<DT>& row, PickShared& sh, float m, double inv, Kept from,
                             bool by_count, int count, double limit) {
  const int tid = item_id();
  // linear bins: 1/64 of a natural-log unit of weight, or of a logit
  const float scale = by_count ? 64.f : fminf(64.f * (float)inv, 1e30f);
  uint32_t klo = key_of(kNegInf) + 1, khi = key_of(m);  // the range that holds the boundary
  int shift = -1;                                       // -1: linear bins
  // a bin index grows towards earlier ranks for integer bins, towards later ones for linear bins;
  // `bin` below is turned so that 0 is always the earliest
  auto member = [&](int i, float l) {
    if (rank_of(l, i) < from.low) return false;
    return from.mp <= 0.0 || weight(l, m, inv) >= from.mp;
  };
#pragma unroll 1
  for (;;) {
    auto bin_of = [&](float l) -> int {
      if (shift < 0) {
        const float d = (m - l) * scale;  // NaN only for two infinities: l = m then
        return l >= m ? 0 : d >= (float)(kBins - 1) ? kBins - 1 : (int)d;
      }
      return (int)((khi - key_of(l)) >> shift);
    };
    auto inside = [&](float l) {
      const uint32_t k = key_of(l);
      return k >= klo && k <= khi;
    };
    __syncthreads();
    for (int b = tid; b < kBins; b += kPick) {
      sh.wbin[b] = 0;
      sh.cbin[b] = 0;
    }
    __syncthreads();
    double above = 0.0;     // weight of the earlier ranks, past the range
    uint32_t n_above = 0;   // and their number
    row.each([&](int i, float l) {
      if (l == kNegInf || !member(i, l)) return;
      if (key_of(l) > khi) {
        ++n_above;
        if (!by_count) above += weight(l, m, inv);
      } else if (inside(l)) {
        const int b = bin_of(l);
        atomicAdd(&sh.cbin[b], 1u);
        if (!by_count)
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.wbin[b]),
                    (unsigned long long)(weight(l, m, inv) * 0x1p43));
      }
    });
    if (!by_count) above = block_sum(sh, above);
    n_above = block_reduce_u32(sh, n_above, [](uint32_t a, uint32_t b) { return a + b; });
    // ---- walk the bins from the earliest (thread t: bins 2 t, 2 t + 1): by weight the boundary is
    // in bins [lo, hi], where the running weight passes the limit less and more the integers'
    // possible error (2^-43 an element) and the sums' own; at single-value bins the weights are
    // count * weight, exact
    double w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = 2 * tid + e;
      const uint32_t c = sh.cbin[b];
      w[e] = by_count     ? (double)c
             : shift == 0 ? (double)c * weight(of_key(khi - (uint32_t)min((uint32_t)b, khi - klo)), m, inv)
                          : (double)sh.wbin[b] * 0x1p-43;
    }
    double total;
    double run = block_scan(sh, w[0] + w[1], &total);
    run += by_count ? (double)n_above : above;
    const double want = by_count ? (double)count : limit;
    const double slack = by_count || shift == 0 ? 0.0 : (above + total + 1.0) * 1e-12 + row.n * 0x1p-42;
    if (tid == 0) {
      sh.i[0] = kBins;  // lo
      sh.i[1] = kBins;  // hi
      sh.i[2] = 0;      // the last bin with a member
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = 2 * tid + e;
      run += w[e];
      if (sh.cbin[b]) {
        if (run >= want - slack) atomicMin(&sh.i[0], b);
        if (run >= want + slack) atomicMin(&sh.i[1], b);
        atomicMax(&sh.i[2], b);
      }
    }
    __syncthreads();
    const int last = sh.i[2];
    const int hi = min(sh.i[1], last), lo = min(sh.i[0], hi);
    uint32_t pop = 0, pre = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = 2 * tid + e;
      if (b >= lo && b <= hi) pop += sh.cbin[b];
      if (b < lo) pre += sh.cbin[b];
    }
    pop = block_reduce_u32(sh, pop, [](uint32_t a, uint32_t b) { return a + b; });
    pre = block_reduce_u32(sh, pre, [](uint32_t a, uint32_t b) { return a + b; });

    if (pop <= (uint32_t)kList) {
      // ---- the boundary is one of these: sorted, and the definition applied to them
      double ab = 0.0;
      if (!by_count) {
        row.each([&](int i, float l) {
          if (l == kNegInf || !member(i, l)) return;
          if (key_of(l) > khi || (inside(l) && bin_of(l) < lo)) ab += weight(l, m, inv);
        });
        ab = block_sum(sh, ab);
      }
      const int n = collect(row, sh, [&](int i, float l) {
        if (!inside(l) || !member(i, l)) return false;
        const int b = bin_of(l);
        return b >= lo && b <= hi;
      });
      sort_list(sh, n);
      double wl[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 2 * tid + e;
        wl[e] = j >= n ? 0.0 : by_count ? 1.0 : weight(logit_of(sh.sorted[j]), m, inv);
      }
      double tot;
      const double before = block_scan(sh, wl[0] + wl[1], &tot) +
                            (by_count ? (double)(n_above + pre) : ab);
      if (tid == 0) sh.i[3] = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const double b = e == 0 ? before : before + wl[0];
        if (2 * tid + e < n && b < want) atomicMax(&sh.i[3], 2 * tid + e);
      }
      __syncthreads();
      const uint64_t r = sh.sorted[sh.i[3]];
      __syncthreads();
      return r;
    }
    if (shift == 0 && lo == hi) {
      // ---- one value, more often than a list holds: its t-th occurrence in index order
      const uint32_t key = khi - (uint32_t)lo;
      const float v = of_key(key);
      const double wv = by_count ? 1.0 : weight(v, m, inv);
      double ab = (double)n_above + (double)pre;
      if (!by_count) {
        // above + the earlier bins, in the walk's arithmetic
        double x = 0.0;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * tid + e < lo) x += w[e];
        ab = above + block_sum(sh, x);
      }
      // kept: occurrences j with ab + j wv < want
      double t = ab < want ? (double)pop : 1.0;
      if (wv > 0.0) {
        t = fmin(fmax(__builtin_ceil((want - ab) / wv), 1.0), (double)pop);
        if (t > 1.0 && ab + (t - 1.0) * wv >= want) t -= 1.0;
        else if (ab + t * wv < want) t += 1.0;
      }
      const uint32_t nth = (uint32_t)fmin(fmax(t, 1.0), (double)pop);
      // its index: counted tile by tile
      constexpr int EPL = Row<DT>::EPL, TILE = Row<DT>::TILE;
      const int lane = tid & 63, wave = tid >> 6;
      uint32_t seen = 0;
      if (tid == 0) sh.i[4] = 0;
#pragma unroll 1
      for (int b = 0; b < row.n; b += TILE) {
        Lane<DT> a;
        const int i0 = b + tid * EPL;
        a.load(row.x, min(i0, row.n), row.n);
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          mine += i0 + e < row.n && a.v[e] != kNegInf && key_of(a.v[e]) == key && member(i0 + e, a.v[e]);
        uint32_t inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const uint32_t y = (uint32_t)__shfl_up((int)inc, d);
          if (lane >= d) inc += y;
        }
        __syncthreads();
        if (lane == 63) sh.cnt[0][0][wave] = (int)inc;
        __syncthreads();
        uint32_t before = seen + inc - mine, all = 0;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          if (x < wave) before += (uint32_t)sh.cnt[0][0][x];
          all += (uint32_t)sh.cnt[0][0][x];
        }
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (i0 + e < row.n && a.v[e] != kNegInf && key_of(a.v[e]) == key && member(i0 + e, a.v[e]))
            if (++before == nth) sh.i[4] = i0 + e;
        seen += all;
        if (seen >= nth) break;  // uniform
      }
      __syncthreads();
      const uint64_t r = ((uint64_t)key << 32) | (0xffffffffu - (uint32_t)sh.i[4]);
      __syncthreads();
      return r;
    }
    // ---- a smaller range: the keys of bins [lo, hi]
    uint32_t a = 0xffffffffu, b = 0;
    row.each([&](int i, float l) {
      if (l == kNegInf || !inside(l) || !member(i, l)) return;
      const int bb = bin_of(l);
      if (bb >= lo && bb <= hi) {
        a = min(a, key_of(l));
        b = max(b, key_of(l));
      }
    });
    a = block_reduce_u32(sh, a, [](uint32_t x, uint32_t y) { return min(x, y); });
    b = block_reduce_u32(sh, b, [](uint32_t x, uint32_t y) { return max(x, y); });
    klo = a;
    khi = b;
    const int bits = 32 - __builtin_clz((khi - klo) | 1u);
    shift = max(0, bits - 11);
  }
}

template <int DT>
__global__ __launch_bounds__(kPick) void sample_pick_kernel(SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) char pick_lds[];
  PickShared& sh = *reinterpret_cast<PickShared*>(pick_lds);
  const int rowi = wg_id_x(), tid = item_id();
  Row<DT> row;
  row.x = reinterpret_cast<const store_t<DT>*>(p.logits) + (int64_t)rowi * p.ls;
  row.n = p.vocab;
  const RowSettings s = settings(p, rowi);
  const float uf = p.u[rowi];
  const double u = is_nan(uf) || uf < 0.f ? 0.0 : (double)fminf(uf, 0x1.fffffep-1f);

  // ---- the row's maximum and sums, a thread per chunk
  const bool on = tid < p.chunks;
  const int64_t at = (int64_t)rowi * p.chunks + (on ? tid : 0);
  const f32x4 g = *reinterpret_cast<const f32x4*>(p.gmax + at * 4);
  const float cm = on ? fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3])) : kNegInf;
  const double ct = p.sum_t[at], c1 = p.sum_1[at];
  const uint32_t mk = block_reduce_u32(sh, key_of(cm), [](uint32_t a, uint32_t b) { return max(a, b); });
  const float m = of_key(mk);
  if (m == kNegInf) {  // nothing to choose from (uniform)
    if (tid == 0) {
      p.tok[rowi] = -1;
      if (p.lp) p.lp[rowi] = kNegInf;
    }
    return;
  }
  const double r1 = block_sum(sh, on ? c1 * weight(cm, m, 1.0) : 0.0);
  const int first = (int)block_reduce_u32(sh, on && cm == m ? (uint32_t)p.first[at] : 0xffffffffu,
                                          [](uint32_t a, uint32_t b) { return min(a, b); });
  int token = first;
  if (!s.greedy && !s.filtered()) {
    double w[1] = {on ? ct * weight(cm, m, s.inv) : 0.0};
    // the chunk, then the token in it by what is left of u W
    double total;
    const double before = block_scan(sh, w[0], &total);
    const int c = draw<1>(sh, w, u);
    if (tid == c) sh.d[0] = u * total - before;
    __syncthreads();
    const double left = sh.d[0];
    double e[4];
    const int i0 = c * kChunk + 4 * tid;
    double mine = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      e[j] = i0 + j < row.n ? weight(load1<DT>(row.x, i0 + j), m, s.inv) : 0.0;
      mine += e[j];
    }
    double run = block_scan(sh, mine, &total);
    if (tid == 0) {
      sh.i[0] = 0x7fffffff;
      sh.i[1] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      run += e[j];
      if (e[j] > 0.0) {
        if (run > left) atomicMin(&sh.i[0], i0 + j);
        atomicMax(&sh.i[1], i0 + j);
      }
    }
    __syncthreads();
    token = sh.i[0] != 0x7fffffff ? sh.i[0] : sh.i[1];
  } else if (!s.greedy) {
    const double W = s.k == 0 ? block_sum(sh, on ? ct * weight(cm, m, s.inv) : 0.0) : 0.0;
    // ---- a list of everything from the k-th largest group maximum up
    const int groups = 4 * p.chunks;
    const int k = s.k > 0 ? s.k : min(groups, 96);
    bool done = false;
    if (k <= groups && groups <= kList) {
      __syncthreads();
      if (on)
#pragma unroll
        for (int e = 0; e < 4; ++e) sh.sorted[4 * tid + e] = rank_of(g[e], 4 * tid + e);
      __syncthreads();
      sort_list(sh, groups);
      const float low = logit_of(sh.sorted[k - 1]);
      if (low != kNegInf) {
        const int n = collect(row, sh, [&](int, float l) { return l >= low; });
        if (n <= kList) {
          // every kept token is listed when the k-th, the least weight or the limit ends inside
          const bool by_mp = s.mp > 0.0 && weight(low, m, s.inv) < s.mp;
          double whole = -1.0;
          done = s.k > 0 || by_mp;
          if (!done && s.mp <= 0.0 && s.p < 1.f) {
            double x = 0.0;
            for (int j = tid; j < n; j += kPick) x += weight(logit_of(sh.list[j]), m, s.inv);
            x = block_sum(sh, x);
            // (a limit so near the list's end that rounding decides goes to the general way)
            done = x * (1.0 - 1e-12) >= (double)s.p * W;
            whole = W;
          }
          if (done) token = pick_from_list(sh, n, s, m, whole, u);
        }
      }
    }
    if (!done) {
      // ---- the general way
      Kept kept = {0, s.mp};
      if (s.k > 0) kept.low = boundary(row, sh, m, s.inv, Kept{0, 0.0}, true, s.k, 0.0);
      if (s.p < 1.f) {
        double w1 = W;
        if (s.k > 0 || s.mp > 0.0) {
          w1 = 0.0;
          row.each([&](int i, float l) {
            if (l == kNegInf || rank_of(l, i) < kept.low) return;
            const double w = weight(l, m, s.inv);
            if (w >= kept.mp) w1 += w;
          });
          w1 = block_sum(sh, w1);
        }
        // (a limit of 0 or less keeps the first alone)
        kept.low = boundary(row, sh, m, s.inv, kept, false, 0, (double)s.p * w1);
      }
      // sums of the kept weights by segments in index order: a wave's share of a tile
      constexpr int EPL = Row<DT>::EPL, TILE = Row<DT>::TILE, SEG = 64 * EPL;
      auto kept_weight = [&](int i, float l) {
        if (l == kNegInf || rank_of(l, i) < kept.low) return 0.0;
        const double w = weight(l, m, s.inv);
        return w >= kept.mp ? w : 0.0;
      };
      const int segs = (row.n + SEG - 1) / SEG;
      __syncthreads();
#pragma unroll 1
      for (int b = tid * EPL; b < (row.n + TILE - 1) / TILE * TILE; b += TILE) {
        Lane<DT> a;
        a.load(row.x, min(b, row.n), row.n);
        double x = 0.0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) x += kept_weight(b + e, a.v[e]);
        x = wave_sum(x);
        if ((tid & 63) == 0 && b / SEG < segs) sh.seg[b / SEG] = x;
      }
      __syncthreads();
      double w[4];
      double mine = 0.0, total;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = 4 * tid + e < segs ? sh.seg[4 * tid + e] : 0.0;
        mine += w[e];
      }
      double before = block_scan(sh, mine, &total);
      const int sg = draw<4>(sh, w, u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (4 * tid + e == sg) sh.d[0] = u * total - before;
        before += w[e];
      }
      __syncthreads();
      const double left = sh.d[0];
      // the segment, one wave
      if (tid < 64) {
        Lane<DT> a;
        const int i0 = sg * SEG + tid * EPL;
        a.load(row.x, min(i0, row.n), row.n);
        double x[EPL];
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          x[e] = kept_weight(i0 + e, a.v[e]);
          sum += x[e];
        }
        double inc = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const double y = __shfl_up(inc, d);
          if (tid >= d) inc += y;
        }
        double run = __shfl_up(inc, 1);
        if (tid == 0) run = 0.0;
        int hit = 0x7fffffff, lastk = -1;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          run += x[e];
          if (x[e] > 0.0) {
            if (run > left) hit = min(hit, i0 + e);
            lastk = i0 + e;
          }
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          hit = min(hit, __shfl_xor(hit, d));
          lastk = max(lastk, __shfl_xor(lastk, d));
        }
        token = hit != 0x7fffffff ? hit : lastk;
      }
    }
  }
  if (tid == 0) {
    p.tok[rowi] = token;
    if (p.lp) {
      const float l = load1<DT>(row.x, token);
      const double d = l >= m ? 0.0 : (double)l - (double)m;
      p.lp[rowi] = (float)(d - log(r1));
    }
  }
}

template <int DT>
hipError_t launch_sample(const SampleParams& p, hipStream_t st) {
  static const hipError_t once = hipFuncSetAttribute(
      reinterpret_cast<const void*>(sample_pick_kernel<DT>),
      hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PickShared));
  if (once != hipSuccess) return once;
  hipLaunchKernelGGL(sample_scan_kernel<DT>, dim3((unsigned)p.chunks, (unsigned)p.rows), dim3(256), 0,
                     st, p);
  hipLaunchKernelGGL(sample_pick_kernel<DT>, dim3((unsigned)p.rows), dim3(kPick), sizeof(PickShared),
                     st, p);
  return hipGetLastError();
}

int check_sample_sizes(int32_t rows, int32_t vocab) {
  if (rows < 0 || rows > 65535) return api_fail(FFAI_ERR_INVALID, "rows must be in [0, 65535]");
  if (vocab < 1 || vocab > kMaxVocab) return api_fail(FFAI_ERR_INVALID, "vocab must be in [1, 2^20]");
  return FFAI_OK;
}
size_t sample_bytes(int32_t rows, int32_t vocab) {
  const size_t n = (size_t)rows * ((vocab + kChunk - 1) / kChunk);
  return n * (16 + 8 + 8) + ((n * 4 + 15) & ~size_t(15));
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
  *bytes = sample_bytes(rows, vocab);
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
  if (!workspace || workspace_bytes < sample_bytes(rows, vocab))
    return api_fail(FFAI_ERR_WORKSPACE, "workspace smaller than ffai_sample_workspace_bytes");
  if ((uintptr_t)workspace % 16) return api_fail(FFAI_ERR_INVALID, "workspace must be 16-byte aligned");
  rc = api_check_device();
  if (rc != FFAI_OK) return rc;
  SampleParams p{};
  p.logits = logits; p.ls = logits_row_stride; p.rows = rows; p.vocab = vocab;
  p.chunks = (vocab + kChunk - 1) / kChunk;
  p.t = temperature; p.t_all = temperature_all;
  p.k = top_k; p.k_all = top_k_all;
  p.p = top_p; p.p_all = top_p_all;
  p.mp = min_p; p.mp_all = min_p_all;
  p.u = u; p.tok = tokens; p.lp = logprobs;
  const size_t n = (size_t)rows * p.chunks;
  char* ws = static_cast<char*>(workspace);
  p.gmax = reinterpret_cast<float*>(ws);
  p.sum_t = reinterpret_cast<double*>(ws + n * 16);
  p.sum_1 = reinterpret_cast<double*>(ws + n * 24);
  p.first = reinterpret_cast<int32_t*>(ws + n * 32);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = logits_dtype == FFAI_F32   ? launch_sample<kF32>(p, st)
                       : logits_dtype == FFAI_F16 ? launch_sample<kF16>(p, st)
                                                  : launch_sample<kBF16>(p, st);
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  return FFAI_OK;
}

}  // extern "C"
