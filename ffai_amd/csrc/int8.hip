// Linear layers in 8-bit integers (include/ffai_int8.h): the quantization of rows and the product
// of quantized rows with weights on the int8 matrix instructions.
#include "../../include/ffai_int8.h"

#include <algorithm>

#include "attn_common.cuh"

namespace ffai {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;  // contraction elements (bytes) of a product step

// ---- quantization ----------------------------------------------------------------------------
// Two passes over a row that stays in registers, as it lies in memory: its largest magnitude, then
// the quotients. The magnitude is taken on the bit patterns (sign cleared, as integers: the order of
// non-negative floats, with NaN above infinity), so that a NaN becomes the scale.
//
// The quotient's rounding, of the IEEE f32 quotient x / s, decides which integer a value near a half
// goes to. Away from one the product with 1 / s gives the same integer: for |x / s| <= 127 its
// error is below 127 (2^-24 + 2^-24) (1 / s rounded, the sum below exact before its one rounding) and
// the quotient's own rounding below 127 2^-24, together 2.3e-5. So: n = round(x (1 / s)) by a sum
// with 1.5 * 2^23, whose low bits are n in two's complement, four instructions a value; eight
// values of which one lies within 3e-5 of a half (one in 2000), and rows whose 1 / s or s is not
// finite, are divided (25 instructions a value).
// 24000 x 5120 bf16: 65 us, 5.6 TB/s; with every value divided 125.
__device__ __forceinline__ int quant1(float x, float s) {
  const float r = __builtin_rintf(x / s);
  // NaN (of a non-finite row) to 0: the clamps compare bits of ordinary numbers only
  const bool nan = (__float_as_uint(r) & 0x7fffffffu) > 0x7f800000u;
  return nan ? 0 : (int)fminf(fmaxf(r, -127.f), 127.f);
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, s));
  return v;
}
__device__ __forceinline__ bool finite_bits(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// Eight elements of a row as they lie in memory.
template <int DT>
struct Raw8 {
  u32x4 u[DT == kF32 ? 2 : 1];
  __device__ __forceinline__ void load(const store_t<DT>* p) {
    u[0] = ld16h(p);
    if constexpr (DT == kF32) u[1] = ld16h(p + 4);
  }
  __device__ __forceinline__ void load_first(const store_t<DT>* p, int n) {  // n < 8, zeros behind
    for (auto& x : u) x = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) {
        if constexpr (DT == kF32) u[e >> 2][e & 3] = __float_as_uint(p[e]);
        else u[0][e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
      }
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (DT == kF32) return __uint_as_float(u[e >> 2][e & 3]);
    else return to_f32<DT>((uint16_t)((u[0][e >> 1] >> (16 * (e & 1))) & 0xffffu));
  }
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// The largest magnitude so far: f32 bits, or two 16-bit ones.
template <int DT>
struct Top {
  uint32_t t = 0;
  __device__ __forceinline__ void add(const Raw8<DT>& r) {
#pragma unroll
    for (int i = 0; i < (DT == kF32 ? 8 : 4); ++i) {
      const uint32_t x = r.u[i >> 2][i & 3];
      if constexpr (DT == kF32)
        t = max(t, x & 0x7fffffffu);
      else
        t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
                                             __builtin_bit_cast(u16x2, t),
                                             __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
    }
  }
  __device__ __forceinline__ uint32_t bits() const {  // of the magnitude in f32
    if constexpr (DT == kF32) return t;
    else return __float_as_uint(to_f32<DT>((uint16_t)max(t & 0xffffu, t >> 16)));
  }
};

struct RowScale {
  float s, inv;
  bool fast;
  __device__ __forceinline__ RowScale(uint32_t top) {
    s = top == 0 ? 1.f : __uint_as_float(top) * (1.f / 127.f);
    inv = 1.f / s;
    fast = finite_bits(s) && finite_bits(inv);
  }
};

template <int DT>
__device__ __forceinline__ uint64_t quant8(const Raw8<DT>& r, const RowScale& sc) {
  constexpr float MAGIC = 12582912.f;
  uint32_t y[8];
  float off = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = r.at(e);
    const float z = __builtin_fmaf(x, sc.inv, MAGIC);
    off = fmaxf(off, fabsf(__builtin_fmaf(x, sc.inv, MAGIC - z)));
    y[e] = __float_as_uint(z);
  }
  if (__builtin_expect(!sc.fast || off > 0.49997f, 0)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (uint32_t)quant1(r.at(e), sc.s);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[4 * h + 3], y[4 * h + 2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(y[4 * h + 1], y[4 * h], 0x0c0c0400u),
                                 0x05040100u);
  return (uint64_t)w[1] << 32 | w[0];
}
// The eight results at k, from the eight elements at kl = min(k, dim - 8): zeros from dim on.
__device__ __forceinline__ void put8(int8_t* q, int k, int kl, uint64_t w) {
  const int sh = k - kl;
  *reinterpret_cast<uint64_t*>(q + k) = sh >= 8 ? 0ull : w >> (8 * sh);
}

// WPR waves a row (1: a wave per row, four rows a workgroup; 4: the workgroup's four waves share
// a row, for few rows); NC > 0: the row fits NC chunks of 8 elements a lane and stays in
// registers; NC == 0: any length, read twice. Bound by reading x and writing q. The row's last chunk
// is read as its last eight elements; only a row of fewer is read by element.
template <int DT, int WPR, int NC>
__global__ __launch_bounds__(256) void int8_quantize_kernel(const void* xv, int64_t xs, int rows,
                                                            int dim, int8_t* q, int64_t qs,
                                                            float* scale) {
  __shared__ uint32_t tops[4];
  const int wave = item_id() >> 6;
  const int t = WPR == 1 ? item_id() & 63 : item_id();
  const int row = WPR == 1 ? wg_id_x() * 4 + wave : wg_id_x();
  if (row >= rows) return;  // the whole wave (WPR 1); never with WPR 4
  const store_t<DT>* x = reinterpret_cast<const store_t<DT>*>(xv) + (int64_t)row * xs;
  int8_t* qr = q + (int64_t)row * qs;
  const int end = (dim + kStep - 1) / kStep * kStep;  // q is zero from dim to here
  constexpr int SPAN = WPR * 64 * 8;
  const int last = max(dim - 8, 0);
  Top<DT> top;
  Raw8<DT> v[NC > 0 ? NC : 1];
  if constexpr (NC > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c].load(x + min(c * SPAN + 8 * t, last));
#pragma unroll
    for (int c = 0; c < NC; ++c) top.add(v[c]);
  } else if (dim >= 8) {
    for (int k = 8 * t; k < dim; k += SPAN) {
      v[0].load(x + min(k, last));
      top.add(v[0]);
    }
  } else {
    v[0].load_first(x, dim);
    top.add(v[0]);
  }
  uint32_t m = wave_umax(top.bits());
  if constexpr (WPR == 4) {
    if ((t & 63) == 0) tops[wave] = m;
    __syncthreads();
    m = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  const RowScale sc(m);
  if (t == 0) scale[row] = sc.s;
  if constexpr (NC > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = c * SPAN + 8 * t;
      if (k < end) put8(qr, k, min(k, last), quant8(v[c], sc));
    }
  } else {
    for (int k = 8 * t; k < end; k += SPAN) {
      if (dim >= 8) v[0].load(x + min(k, last));
      put8(qr, k, min(k, last), quant8(v[0], sc));
    }
  }
}

template <int DT>
void launch_quantize(const void* x, int64_t xs, int rows, int dim, int8_t* q, int64_t qs,
                     float* scale, hipStream_t st) {
  const int end = (dim + kStep - 1) / kStep * kStep;
  auto go = [&](auto kernel, int wpr) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(wpr == 1 ? (rows + 3) / 4 : rows)), dim3(256), 0, st,
                       x, xs, rows, dim, q, qs, scale);
  };
  if (dim < 8) return go(int8_quantize_kernel<DT, 1, 0>, 1);
  // few rows: a row's loads over four waves shorten its latency
  if (rows <= 1024) {
    if (end <= 2048) go(int8_quantize_kernel<DT, 4, 1>, 4);
    else if (end <= 4096) go(int8_quantize_kernel<DT, 4, 2>, 4);
    else if (end <= 8192) go(int8_quantize_kernel<DT, 4, 4>, 4);
    else go(int8_quantize_kernel<DT, 4, 0>, 4);
  } else {
    if (end <= 512) go(int8_quantize_kernel<DT, 1, 1>, 1);
    else if (end <= 1024) go(int8_quantize_kernel<DT, 1, 2>, 1);
    else if (end <= 2048) go(int8_quantize_kernel<DT, 1, 4>, 1);
    else if (end <= 4096) go(int8_quantize_kernel<DT, 1, 8>, 1);
    else if (end <= 8192) go(int8_quantize_kernel<DT, 1, 16>, 1);
    else go(int8_quantize_kernel<DT, 1, 0>, 1);
  }
}

// ---- product ---------------------------------------------------------------------------------
struct Int8Params {
  const int8_t* x;
  int64_t xs;
  const float* sx;
  const int8_t* w;
  int64_t ws;
  const float* sw;
  const float* bias;
  void* y;
  int64_t ys;
  int32_t rows, out_dim;
  int32_t steps;  // kStep-byte contraction steps
  int32_t w_last;  // the last 16-byte chunk of a row of w
  int32_t tx, tw;  // tiles over the rows of x and of w
};

// s_waitcnt vmcnt(N) lgkmcnt(0)
template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
}

// One tile of BX rows of x by BW rows of w per workgroup, waves in a grid of GX by GW, on
// v_mfma_i32_32x32x32_i8 (lane l: row l % 32, 16 bytes at 16 (l / 32) of the 32): the weights are
// the A operand, so a lane's results are four consecutive outputs of one row of x. Steps of 128
// bytes of the contraction arrive by DMA in a ring of STAGES buffers, rows unpadded with their eight
// 16-byte chunks XOR-permuted by the row's number / 2, so that the DMA's lanes read whole 128-byte
// rows and the sixteen lanes of one cycle of a fragment read cover all 64 banks (by the row's low
// bits instead, rows r and r + 8 collide: half of all LDS cycles). One barrier a step, before its last
// products: it says that the next step's loads of every wave have landed and that every wave has
// read this step's buffer, which the loads begun there overwrite; the next step's first fragments
// are read under those products. Rows past the operands' ends are clamped (their results are not
// stored); contraction bytes past in_dim are zero in x, so whatever w's clamped chunk holds there
// counts for nothing.
//
// Bound by the matrix cores at the clock that their power leaves: 24000 x 10240 x 1280 takes 295 us
// (2.1 POPS), 233 of them with the loop's loads left out; 24000 x 5120 x 1280 155 us, 24000 x 1280 x
// 1280 51 (its 61 MB of results and the tiles' first loads are 20 of them).
template <int BX, int BW, int GX, int GW, int STAGES, int OCC, int OUT>
__global__ __launch_bounds__((GX * GW) * 64, OCC) void int8_product_kernel(Int8Params p) {
  constexpr int NW = GX * GW;
  constexpr int FX = BX / GX / 32, FW = BW / GW / 32;  // fragments of a wave
  constexpr int BUF = (BX + BW) * kStep;
  constexpr int PB = (BX + BW) / 8 / NW;  // 1 KB DMA blocks of a wave and step
  static_assert((BX + BW) % (8 * NW) == 0, "whole blocks per wave");
  static_assert(PB * (STAGES - 1) <= 63, "outstanding loads fit the counter");
  extern __shared__ __attribute__((aligned(16))) int8_t int8_lds[];
  const int lane = item_id() & 63;
  const int wave = __builtin_amdgcn_readfirstlane(item_id() >> 6);
  const int gx = wave % GX, gw = wave / GX;

  // Workgroups go to the eight XCDs in turn: each XCD takes a run of consecutive tiles, w fastest,
  // so that its L2 serves a few row blocks of x against all of w.
  const int n = p.tx * p.tw;
  int tile = wg_id_x();
  {
    const int per = n / 8, more = n % 8, xcd = tile & 7, at = tile >> 3;
    tile = xcd * per + min(xcd, more) + at;
  }
  const int x0 = tile / p.tw * BX, w0 = tile % p.tw * BW;

  const char* xb = reinterpret_cast<const char*>(p.x + (int64_t)x0 * p.xs);
  const char* wb = reinterpret_cast<const char*>(p.w + (int64_t)w0 * p.ws);
  const int lr = lane >> 3;
  const int chunk[2] = {16 * ((lane & 7) ^ (lr >> 1)), 16 * ((lane & 7) ^ (4 + (lr >> 1)))};
  static_assert(PB % 2 == 0 && BW % 16 == 0, "a wave's blocks begin at even ones");
  uint32_t off[PB];
#pragma unroll
  for (int b = 0; b < PB; ++b) {
    const int r = (wave * PB + b) * 8 + lr;
    off[b] = r < BW ? (uint32_t)min(r, p.out_dim - 1 - w0) * (uint32_t)p.ws
                    : (uint32_t)min(r - BW, p.rows - 1 - x0) * (uint32_t)p.xs;
  }
  const uint32_t lds0 = lds_addr(int8_lds) + wave * PB * 1024;
  auto issue = [&](int step, int buf, int b0, int b1) {  // blocks b0 .. b1 - 1 of the wave's PB
#pragma unroll
    for (int b = b0; b < b1; ++b) {
      const bool of_w = (wave * PB + b) * 8 < BW;  // wave-uniform
      const uint32_t kx = (uint32_t)(step * kStep + chunk[b & 1]);
      lds_dma16_sbase(of_w ? wb : xb, off[b] + (of_w ? min(kx, (uint32_t)p.w_last) : kx),
                      lds0 + buf * BUF + b * 1024);
    }
  };

  i32x16 acc[FW][FX];
#pragma unroll
  for (int i = 0; i < FW; ++i)
#pragma unroll
    for (int j = 0; j < FX; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < p.steps) issue(s, s, 0, PB);
  const int row = lane & 31, half = lane >> 5;
  constexpr int KS = kStep / 32;
  i32x4 a[2][FW], b[2][FX];
  auto frags = [&](int buf, int ks, i32x4 (&fa)[FW], i32x4 (&fb)[FX]) {
    const int8_t* base = int8_lds + buf * BUF;
    const int8_t* wl = base + (gw * FW * 32 + row) * kStep;
    const int8_t* xl = base + (BW + gx * FX * 32 + row) * kStep;
    const int c = 16 * ((2 * ks + half) ^ ((row >> 1) & 7));
#pragma unroll
    for (int i = 0; i < FW; ++i) fa[i] = *reinterpret_cast<const i32x4*>(wl + i * 32 * kStep + c);
#pragma unroll
    for (int j = 0; j < FX; ++j) fb[j] = *reinterpret_cast<const i32x4*>(xl + j * 32 * kStep + c);
  };
  // the loads of `step` of every wave have landed, and every wave's reads so far are done
  auto meet = [&](int step) {
    asm volatile("" ::: "memory");
    if (STAGES > 2 && step + STAGES - 2 < p.steps) wait_vm<PB*(STAGES - 2)>();
    else wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (STAGES <= p.steps) wait_vm<PB*(STAGES - 1)>();
  else wait_vm<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  frags(0, 0, a[0], b[0]);
  int buf = 0;
#pragma unroll 1
  for (int step = 0; step < p.steps; ++step) {
    const int nbuf = buf + 1 == STAGES ? 0 : buf + 1;
    constexpr int NM = FX * FW;
    const bool more = step + STAGES < p.steps;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS) {
        frags(buf, ks + 1, a[(ks + 1) & 1], b[(ks + 1) & 1]);
      } else if (step + 1 < p.steps) {
        meet(step + 1);
        frags(nbuf, 0, a[0], b[0]);
      }
#pragma unroll
      for (int n = 0; n < NM; ++n) {
        const int i = n / FX, j = n % FX;
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[ks & 1][i], b[ks & 1][j], acc[i][j],
                                                          0, 0, 0);
        if (ks + 1 == KS && more) {
          issue(step + STAGES, buf, n * PB / NM, (n + 1) * PB / NM);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    buf = nbuf;
  }

  // ---- D lane l, element 4 q + r: w row 8 q + 4 (l / 32) + r, x row l % 32. Through the wave's
  // share of LDS (16-byte chunks XOR-permuted so that eight rows cover all banks) into whole rows of
  // the wave's tile: 16 bytes a lane, 64 to 256 a row. (Stored straight from here, 8 bytes a lane to 32
  // rows at a time: 24000 x 5120 x 1280 to bf16 187 us, so 158.)
  constexpr int ES = OUT == kF32 ? 4 : 2;
  constexpr int P = FW * 32 * ES;  // bytes of a row of the wave's tile
  constexpr int AREA = BUF * STAGES / NW;
  constexpr int JP = FX < AREA / (32 * P) ? FX : AREA / (32 * P);  // row blocks at a time
  static_assert(JP >= 1 && FX % JP == 0 && P >= 64 && P <= 512, "");
  constexpr int LPR = P / 16, RPI = 64 / LPR;  // lanes of a row, rows of a store
  auto key = [](int r) { return P == 64 ? (r >> 1) & 3 : r & 7; };
  int8_t* area = int8_lds + wave * AREA;
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();  // every wave has read its last fragments
  asm volatile("" ::: "memory");
  const int wx0 = x0 + gx * FX * 32, ww0 = w0 + gw * FW * 32;
#pragma unroll
  for (int jp = 0; jp < FX; jp += JP) {
    float sx[JP];
#pragma unroll
    for (int j = 0; j < JP; ++j) sx[j] = p.sx[min(wx0 + (jp + j) * 32 + row, p.rows - 1)];
#pragma unroll
    for (int i = 0; i < FW; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int o = ww0 + i * 32 + 8 * q + 4 * half;
        float sw[4], bias[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int oc = min(o + r, p.out_dim - 1);
          sw[r] = p.sw[oc];
          bias[r] = p.bias ? p.bias[oc] : 0.f;
        }
        const int chunk = ES == 2 ? 4 * i + q : 8 * i + 2 * q + half;
        int8_t* at = area + row * P + 16 * (chunk ^ key(row)) + (ES == 2 ? 8 * half : 0);
#pragma unroll
        for (int j = 0; j < JP; ++j) {
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float t = (float)acc[i][jp + j][4 * q + r] * sx[j];
            v[r] = p.bias ? __builtin_fmaf(t, sw[r], bias[r]) : t * sw[r];
          }
          st4<OUT>(reinterpret_cast<store_t<OUT>*>(at + j * 32 * P), v);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    asm volatile("" ::: "memory");  // (a wave's LDS accesses stay in order)
#pragma unroll 4
    for (int r0 = 0; r0 < JP * 32; r0 += RPI) {
      const int r = r0 + lane / LPR, c = lane % LPR;
      const u32x4 d = *reinterpret_cast<const u32x4*>(area + r * P + 16 * (c ^ key(r)));
      const int m = wx0 + jp * 32 + r, o = ww0 + c * (16 / ES);
      if (m >= p.rows) continue;
      store_t<OUT>* y = reinterpret_cast<store_t<OUT>*>(p.y) + (int64_t)m * p.ys + o;
      if (o + 16 / ES <= p.out_dim) {
        *reinterpret_cast<u32x4_h*>(y) = d;
      } else {
#pragma unroll
        for (int e = 0; e < 16 / ES; ++e)
          if (o + e < p.out_dim) {
            if constexpr (OUT == kF32) y[e] = __uint_as_float(d[e]);
            else y[e] = (store_t<OUT>)(d[e >> 1] >> (16 * (e & 1)));
          }
      }
    }
    asm volatile("" ::: "memory");
  }
}

// ---- few rows --------------------------------------------------------------------------------
// At most 16 rows, quantization and product in one launch: a workgroup takes 16 outputs, quantizes
// all the rows itself into LDS (they are a few KB, from L2) under its weights' loads, and its eight
// waves share out the contraction, 64 bytes a step in turn, on v_mfma_i32_16x16x64_i8 (A: the
// weights' rows, B: the rows of x; lane l: row l % 16, 16 bytes at 16 (l / 16)). LDS rows are padded
// by 16 bytes, so that the 16 rows of a fragment read cover all banks. The waves' partial sums are
// integers: their order does not matter. Bound by the launch and the chain of two round trips; a
// second launch for the quantization alone costs more than doing it in every workgroup.
constexpr int kFewRows = 16;
constexpr int kFewWaves = 8;
constexpr int kFewAhead = 2;            // steps of weights loaded before the rows are quantized
constexpr int kFewLds = 64 * 1024;      // quantized rows at most
constexpr int64_t few_lds(int rows, int in_dim) {
  return (int64_t)rows * ((in_dim + kStep - 1) / kStep * kStep + 16);
}

template <int DT, int OUT>
__global__ __launch_bounds__(kFewWaves * 64) void int8_few_kernel(Int8Params p, const void* xv,
                                                                  int64_t xs, int dim) {
  extern __shared__ __attribute__((aligned(16))) int8_t few_x[];
  __shared__ float scales[kFewRows];
  __shared__ int part[kFewWaves][256];
  const int tid = item_id(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int o0 = wg_id_x() * 16, r16 = lane & 15, q4 = lane >> 4;
  const int8_t* wr = p.w + (int64_t)min(o0 + r16, p.out_dim - 1) * p.ws;
  const int steps = 2 * p.steps;  // of 64 bytes
  const int pitch = p.steps * kStep + 16;
  auto load_w = [&](int s) {
    return *reinterpret_cast<const i32x4*>(wr + min(64 * s + 16 * q4, p.w_last));
  };
  i32x4 a[kFewAhead];
#pragma unroll
  for (int j = 0; j < kFewAhead; ++j) a[j] = load_w(wave + kFewWaves * j);
  // ---- a wave per row: its largest magnitude, then its quotients (from the caches, or registers)
  for (int m = wave; m < p.rows; m += kFewWaves) {
    const store_t<DT>* x = reinterpret_cast<const store_t<DT>*>(xv) + (int64_t)m * xs;
    const int end = p.steps * kStep, last = max(dim - 8, 0);
    int8_t* q = few_x + m * pitch;
    Raw8<DT> v[2];
    Top<DT> top;
#pragma unroll 1
    for (int k = 8 * lane; k < end; k += 1024) {
      if (dim >= 8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h].load(x + min(k + 512 * h, last));
      } else {
        v[0].load_first(x, dim);
        v[1] = v[0];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) top.add(v[h]);
    }
    const RowScale sc(wave_umax(top.bits()));
    if (lane == 0) scales[m] = sc.s;
#pragma unroll 1
    for (int k = 8 * lane; k < end; k += 1024) {
      if (end > 1024) {
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h].load(x + min(k + 512 * h, last));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int kk = k + 512 * h;
        if (kk < end) put8(q, kk, min(kk, last), quant8(v[h], sc));
      }
    }
  }
  __syncthreads();
  i32x4 acc = {0, 0, 0, 0};
  const int8_t* xl = few_x + min(r16, p.rows - 1) * pitch + 16 * q4;
#pragma unroll
  for (int j = 0; j < kFewAhead; ++j) {
    const int s = wave + kFewWaves * j;
    if (s < steps)  // uniform
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], *reinterpret_cast<const i32x4*>(xl + 64 * s),
                                                  acc, 0, 0, 0);
  }
#pragma unroll 1
  for (int s0 = wave + kFewWaves * kFewAhead; s0 < steps; s0 += 4 * kFewWaves) {
    i32x4 b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = load_w(s0 + kFewWaves * j);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = s0 + kFewWaves * j;
      if (s < steps)  // uniform
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j], *reinterpret_cast<const i32x4*>(xl + 64 * s),
                                                    acc, 0, 0, 0);
    }
  }
  // D lane l: outputs 4 (l / 16) .. +3 of row l % 16
  *reinterpret_cast<i32x4*>(&part[wave][4 * lane]) = acc;
  __syncthreads();
  if (tid < 256) {
    const int m = tid >> 4, o = tid & 15;  // rows outermost: 16 outputs of a row in a row
    if (m < p.rows && o0 + o < p.out_dim) {
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) sum += part[w][4 * (16 * (o >> 2) + m) + (o & 3)];
      const float t = (float)sum * scales[m];
      const float v = p.bias ? __builtin_fmaf(t, p.sw[o0 + o], p.bias[o0 + o]) : t * p.sw[o0 + o];
      store_t<OUT>* y = reinterpret_cast<store_t<OUT>*>(p.y) + (int64_t)m * p.ys + o0 + o;
      if constexpr (OUT == kF32) *y = v;
      else *y = from_f32<OUT>(v);
    }
  }
}

template <int DT, int OUT>
hipError_t launch_few(const Int8Params& p, const void* x, int64_t xs, int dim, hipStream_t st) {
  auto kernel = int8_few_kernel<DT, OUT>;
  static const hipError_t once = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kFewLds);
  if (once != hipSuccess) return once;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.out_dim + 15) / 16)), dim3(kFewWaves * 64),
                     (size_t)few_lds(p.rows, dim), st, p, x, xs, dim);
  return hipGetLastError();
}
template <int DT>
hipError_t launch_few_out(const Int8Params& p, int32_t y_dtype, const void* x, int64_t xs, int dim,
                          hipStream_t st) {
  return y_dtype == FFAI_F32   ? launch_few<DT, kF32>(p, x, xs, dim, st)
         : y_dtype == FFAI_F16 ? launch_few<DT, kF16>(p, x, xs, dim, st)
                               : launch_few<DT, kBF16>(p, x, xs, dim, st);
}

struct Int8Tile {
  int bx, bw, waves, stages;
};
constexpr Int8Tile kTiles[] = {{256, 256, 8, 2}, {128, 128, 8, 2}, {64, 64, 4, 4}};

// The tile of least cost, in rounds of one 256^2 tile on each of the 256 CUs: two 128^2 tiles a CU take
// 0.62 of that, two 64^2 ones 0.26 (24000 x 5120 x 1280: 145, 171 and 296 us), and one where a CU has no
// second 0.6 of two. A larger tile within 5%, since it wins with the length of the contraction.
// 1500 x 1280 x 3840: 128^2 16 us, 256^2 24, 64^2 25; 1500 x 1280 x 1280: 64^2 8.6, 128^2 9.4; 4000 x 1000 x
// 6000: 128^2 42, 256^2 45; 3000 x 4000 x 3000: 256^2 54, 128^2 59.
int int8_tile(int rows, int out_dim) {
  auto tiles = [&](int t) {
    return (int64_t)((rows + kTiles[t].bx - 1) / kTiles[t].bx) *
           ((out_dim + kTiles[t].bw - 1) / kTiles[t].bw);
  };
  auto pairs = [&](int t, double two) {
    const int64_t n = tiles(t), rest = n % 512;
    return two * ((double)(n / 512) + (rest == 0 ? 0.0 : rest <= 256 ? 0.6 : 1.0));
  };
  const double large = (double)((tiles(0) + 255) / 256), middle = pairs(1, 0.62), small = pairs(2, 0.26);
  if (large <= 1.05 * std::min(middle, small)) return 0;
  return middle <= 1.05 * small ? 1 : 2;
}

template <int BX, int BW, int GX, int GW, int STAGES, int OCC, int OUT>
hipError_t launch_tile(const Int8Params& p, hipStream_t st) {
  constexpr int lds = (BX + BW) * kStep * STAGES;
  auto kernel = int8_product_kernel<BX, BW, GX, GW, STAGES, OCC, OUT>;
  static const hipError_t once = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (once != hipSuccess) return once;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(p.tx * p.tw)), dim3(GX * GW * 64), lds, st, p);
  return hipGetLastError();
}

template <int OUT>
hipError_t launch_product(Int8Params p, hipStream_t st) {
  const int t = int8_tile(p.rows, p.out_dim);
  p.tx = (p.rows + kTiles[t].bx - 1) / kTiles[t].bx;
  p.tw = (p.out_dim + kTiles[t].bw - 1) / kTiles[t].bw;
  if (t == 0) return launch_tile<256, 256, 2, 4, 2, 2, OUT>(p, st);
  if (t == 1) return launch_tile<128, 128, 2, 4, 2, 4, OUT>(p, st);
  return launch_tile<64, 64, 2, 2, 4, 2, OUT>(p, st);
}

bool known_dtype(int32_t d) { return d == FFAI_F32 || d == FFAI_F16 || d == FFAI_BF16; }
size_t esize(int32_t d) { return d == FFAI_F32 ? 4 : 2; }
constexpr int kMaxIn = 131072;  // 127 * 127 * in_dim stays below 2^31

int check_dims(int32_t rows, int32_t in_dim) {
  if (rows < 0) return api_fail(FFAI_ERR_INVALID, "rows must be >= 0");
  if (in_dim < 1 || in_dim > kMaxIn) return api_fail(FFAI_ERR_INVALID, "in_dim must be in [1, 131072]");
  return FFAI_OK;
}
int check_rows_of_x(const void* x, int32_t dt, int32_t rows, int32_t dim, int64_t xs) {
  const int rc = check_dims(rows, dim);
  if (rc != FFAI_OK) return rc;
  if (!known_dtype(dt)) return api_fail(FFAI_ERR_INVALID, "unknown x dtype");
  if (rows == 0) return FFAI_OK;
  if (!x) return api_fail(FFAI_ERR_INVALID, "null x");
  if ((uintptr_t)x % esize(dt)) return api_fail(FFAI_ERR_INVALID, "x must be aligned to its element size");
  if (xs < 0 || (rows > 1 && xs < dim)) return api_fail(FFAI_ERR_INVALID, "x rows overlap");
  return FFAI_OK;
}
int check_weights(const int8_t* w, int64_t ws, const float* sw, const float* bias, int32_t out_dim,
                  int32_t in_dim, const void* y, int32_t y_dtype, int64_t ys, int32_t rows) {
  if (!w || !sw || (rows > 0 && !y)) return api_fail(FFAI_ERR_INVALID, "null pointer");
  if (out_dim < 1 || out_dim > (1 << 28)) return api_fail(FFAI_ERR_INVALID, "out_dim must be in [1, 2^28]");
  if ((uintptr_t)w % 16 || ws % 16 || ws < in_dim || ws > (1 << 22))
    return api_fail(FFAI_ERR_INVALID, "w must be 16-byte aligned with a row stride that is a multiple of 16 in [in_dim, 2^22]");
  if ((uintptr_t)sw % 4 || (uintptr_t)bias % 4) return api_fail(FFAI_ERR_INVALID, "w_scale and bias must be 4-byte aligned");
  if (!known_dtype(y_dtype)) return api_fail(FFAI_ERR_INVALID, "unknown y dtype");
  if ((uintptr_t)y % esize(y_dtype)) return api_fail(FFAI_ERR_INVALID, "y must be aligned to its element size");
  if (ys < 0 || (rows > 1 && ys < out_dim)) return api_fail(FFAI_ERR_INVALID, "y rows overlap");
  if ((int64_t)((rows + 63) / 64) * ((out_dim + 63) / 64) > 0x7fffffff)
    return api_fail(FFAI_ERR_INVALID, "problem too large");
  return FFAI_OK;
}

hipError_t quantize(const void* x, int32_t dt, int32_t rows, int32_t dim, int64_t xs, int8_t* q,
                    int64_t qs, float* scale, hipStream_t st) {
  if (dt == FFAI_F32) launch_quantize<kF32>(x, xs, rows, dim, q, qs, scale, st);
  else if (dt == FFAI_F16) launch_quantize<kF16>(x, xs, rows, dim, q, qs, scale, st);
  else launch_quantize<kBF16>(x, xs, rows, dim, q, qs, scale, st);
  return hipGetLastError();
}

Int8Params product_params(const int8_t* q, int64_t qs, const float* sx, int32_t rows,
                          int32_t in_dim, const int8_t* w, int64_t ws, const float* sw,
                          const float* bias, int32_t out_dim, void* y, int64_t ys) {
  Int8Params p{};
  p.x = q; p.xs = qs; p.sx = sx; p.w = w; p.ws = ws; p.sw = sw; p.bias = bias;
  p.y = y; p.ys = ys; p.rows = rows; p.out_dim = out_dim;
  p.steps = (in_dim + kStep - 1) / kStep;
  p.w_last = (in_dim + 15) / 16 * 16 - 16;
  return p;
}
hipError_t product(const Int8Params& p, int32_t y_dtype, hipStream_t st) {
  return y_dtype == FFAI_F32   ? launch_product<kF32>(p, st)
         : y_dtype == FFAI_F16 ? launch_product<kF16>(p, st)
                               : launch_product<kBF16>(p, st);
}
bool few(int32_t rows, int32_t in_dim) {
  return rows <= kFewRows && few_lds(rows, in_dim) <= kFewLds;
}

int64_t row_bytes(int32_t dim) { return ((int64_t)dim + kStep - 1) / kStep * kStep; }

}  // namespace
}  // namespace ffai

using namespace ffai;

extern "C" {

int ffai_int8_quantize_rows(const void* x, int32_t x_dtype, int32_t rows, int32_t dim,
                            int64_t x_row_stride, int8_t* q, int64_t q_row_stride, float* scale,
                            void* stream) {
  api_clear_error();
  int rc = check_rows_of_x(x, x_dtype, rows, dim, x_row_stride);
  if (rc != FFAI_OK) return rc;
  if (rows == 0) return FFAI_OK;
  if (!q || !scale) return api_fail(FFAI_ERR_INVALID, "null pointer");
  if ((uintptr_t)q % 16 || q_row_stride % kStep || q_row_stride < dim || q_row_stride > (1 << 22))
    return api_fail(FFAI_ERR_INVALID, "q must be 16-byte aligned with a row stride that is a multiple of 128 in [dim, 2^22]");
  if ((uintptr_t)scale % 4) return api_fail(FFAI_ERR_INVALID, "scale must be 4-byte aligned");
  rc = api_check_device();
  if (rc != FFAI_OK) return rc;
  const hipError_t e = quantize(x, x_dtype, rows, dim, x_row_stride, q, q_row_stride, scale,
                                static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  return FFAI_OK;
}

int ffai_int8_product(const int8_t* q, int64_t q_row_stride, const float* scale, int32_t rows,
                      int32_t in_dim, const int8_t* w, int64_t w_row_stride, const float* w_scale,
                      const float* bias, int32_t out_dim, void* y, int32_t y_dtype,
                      int64_t y_row_stride, void* stream) {
  api_clear_error();
  int rc = check_dims(rows, in_dim);
  if (rc != FFAI_OK) return rc;
  rc = check_weights(w, w_row_stride, w_scale, bias, out_dim, in_dim, y, y_dtype, y_row_stride, rows);
  if (rc != FFAI_OK) return rc;
  if (rows == 0) return FFAI_OK;
  if (!q || !scale) return api_fail(FFAI_ERR_INVALID, "null pointer");
  if ((uintptr_t)q % 16 || q_row_stride % kStep || q_row_stride < in_dim || q_row_stride > (1 << 22))
    return api_fail(FFAI_ERR_INVALID, "q must be 16-byte aligned with a row stride that is a multiple of 128 in [in_dim, 2^22]");
  if ((uintptr_t)scale % 4) return api_fail(FFAI_ERR_INVALID, "scale must be 4-byte aligned");
  rc = api_check_device();
  if (rc != FFAI_OK) return rc;
  const hipError_t e = product(product_params(q, q_row_stride, scale, rows, in_dim, w, w_row_stride,
                                              w_scale, bias, out_dim, y, y_row_stride),
                               y_dtype, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  return FFAI_OK;
}

int ffai_int8_linear_workspace_bytes(int32_t rows, int32_t in_dim, size_t* bytes) {
  api_clear_error();
  if (!bytes) return api_fail(FFAI_ERR_INVALID, "null bytes pointer");
  const int rc = check_dims(rows, in_dim);
  if (rc != FFAI_OK) return rc;
  *bytes = few(rows, in_dim)
               ? 0 : (size_t)rows * row_bytes(in_dim) + (((size_t)rows * 4 + 15) & ~size_t(15));
  return FFAI_OK;
}

int ffai_int8_linear(const void* x, int32_t x_dtype, int64_t x_row_stride, int32_t rows,
                     int32_t in_dim, const int8_t* w, int64_t w_row_stride, const float* w_scale,
                     const float* bias, int32_t out_dim, void* y, int32_t y_dtype,
                     int64_t y_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  api_clear_error();
  int rc = check_rows_of_x(x, x_dtype, rows, in_dim, x_row_stride);
  if (rc != FFAI_OK) return rc;
  rc = check_weights(w, w_row_stride, w_scale, bias, out_dim, in_dim, y, y_dtype, y_row_stride, rows);
  if (rc != FFAI_OK) return rc;
  if (rows == 0) return FFAI_OK;
  size_t need = 0;
  ffai_int8_linear_workspace_bytes(rows, in_dim, &need);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return api_fail(FFAI_ERR_WORKSPACE, "workspace smaller than ffai_int8_linear_workspace_bytes");
  if ((uintptr_t)workspace % 16) return api_fail(FFAI_ERR_INVALID, "workspace must be 16-byte aligned");
  rc = api_check_device();
  if (rc != FFAI_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int8_t* q = static_cast<int8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(q + (size_t)rows * row_bytes(in_dim));
  const Int8Params p = product_params(q, row_bytes(in_dim), sx, rows, in_dim, w, w_row_stride, w_scale,
                                      bias, out_dim, y, y_row_stride);
  hipError_t e;
  if (few(rows, in_dim)) {
    e = x_dtype == FFAI_F32   ? launch_few_out<kF32>(p, y_dtype, x, x_row_stride, in_dim, st)
        : x_dtype == FFAI_F16 ? launch_few_out<kF16>(p, y_dtype, x, x_row_stride, in_dim, st)
                              : launch_few_out<kBF16>(p, y_dtype, x, x_row_stride, in_dim, st);
  } else {
    e = quantize(x, x_dtype, rows, in_dim, x_row_stride, q, row_bytes(in_dim), sx, st);
    if (e == hipSuccess) e = product(p, y_dtype, st);
  }
  if (e != hipSuccess) return api_fail(FFAI_ERR_HIP, hipGetErrorString(e));
  return FFAI_OK;
}

int ffai_int8_plan_info(int32_t rows, int32_t in_dim, int32_t out_dim, int32_t* info) {
  api_clear_error();
  if (!info) return api_fail(FFAI_ERR_INVALID, "null info pointer");
  const int rc = check_dims(rows, in_dim);
  if (rc != FFAI_OK) return rc;
  if (rows < 1 || out_dim < 1 || out_dim > (1 << 28)) return api_fail(FFAI_ERR_INVALID, "rows >= 1 and out_dim in [1, 2^28]");
  const Int8Tile t = kTiles[int8_tile(rows, out_dim)];
  info[0] = t.bx;
  info[1] = t.bw;
  info[2] = t.waves;
  info[3] = ((rows + t.bx - 1) / t.bx) * ((out_dim + t.bw - 1) / t.bw);
  return FFAI_OK;
}

}  // extern "C"
