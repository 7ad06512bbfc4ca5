// 8-bit integers on MI355X (gfx950): rows to codes with a scale each, and products of such rows
// with packed weights, dense or grouped by expert, alone or as the SwiGLU layers.
//
// For a row v with a = max(max |v|, 127 * 2^-126), the fp32 numbers r = 127 / a and s = a / 127
// (so that neither leaves the normal range), the codes are q = v r rounded once to the nearest
// integer, ties to even, |q| <= 127, and stand for q s. A row with an infinity or a NaN has the
// scale NaN and zero codes. For the rows of expert e (sorted by expert, counts [E] on the device;
// a dense product has one expert with all rows) and weight rows n, quantized the same way:
//
//   linear    y_n = s s_n (q . q_n) + b_n, written in bf16 or fp32:      rows x N, k = K
//   gate_up   g, u as y of w1 and w3, h = act(g, u), written in fp32:    rows x 2H, k = D
//
// with act(g, u) = silu(g) u, or gpt-oss's on interleaved rows with biases:
//   g' = min(g + b, L), u' = clamp(u + b, -L, L), g' sigmoid(1.702 g') (u' + 1).
//
// v_mfma_i32_16x16x64_i8: lane (row, q), q = lane / 16, holds 16 consecutive k of its row; the sums
// are exact (K <= 131072: 2^17 * 127 * 128 < 2^31), and what is done with them is the same in every
// kernel and tile, so that a row's results do not depend on which of them it went through. (On
// random codes that instruction alone runs at 4.1 POP/s on this card, v_mfma_i32_32x32x32_i8 at 3.5: the
// clock goes by the power they take.)
#include <algorithm>
#include <atomic>

#include "grouped.h"
#include "mx.h"

namespace moe {
namespace int8 {

using namespace grouped;

typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kMaxK = 131072;
constexpr int kMaxCols = 1 << 30;  // of rows by themselves, so that a column and a step fit 32 bits
constexpr float kLeast = 127.0f * 0x1p-126f;

// The columns of a row operand: whole stages of 128, so that every copy of a stage lies inside its
// row, and zeros behind the contraction meet whatever is read of a weight row there; kLeastStages
// at least, behind which everything that a tile's first stage asked for has landed.
constexpr int kLeastStages = 3;
__host__ __device__ constexpr int padded(int cols) {
  return cols <= kLeastStages * 128 ? kLeastStages * 128 : (cols + 127) / 128 * 128;
}

// ---------------------------------------------------------------------------
// quantization and its inverse
// ---------------------------------------------------------------------------

// Eight elements of a bf16 or fp32 row.
template <typename T> struct Eight;
template <> struct Eight<uint16_t> {
  uint4 v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = *(const uint4*)p; }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&a)[8]) const { Chunk<uint16_t>::unpack(v, a); }
};
template <> struct Eight<float> {
  float4 lo, hi;
  __device__ __forceinline__ void load(const float* p) { lo = *(const float4*)p; hi = *(const float4*)(p + 4); }
  __device__ __forceinline__ void zero() { lo = hi = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&a)[8]) const {
    a[0] = lo.x; a[1] = lo.y; a[2] = lo.z; a[3] = lo.w;
    a[4] = hi.x; a[5] = hi.y; a[6] = hi.z; a[7] = hi.w;
  }
};
template <typename T>
__device__ __forceinline__ uint32_t amax8(const Eight<T>& e) {
  float a[8];
  e.get(a);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, mx::abs_bits(a[i]));
  return m;
}
// the maximum over the wave's lanes: turns within rows of 16, then two lane swaps
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror 8, 4, 2, 1
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
  return mx::row_max(v);
}

// A row's multiplier and scale from the bits of its max |v| taken over integers (bits of |v| order
// as the values do, with infinities and NaN on top). r = 0 stands for a row without a scale.
struct RowScale { float r, s; };
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return {0.f, __uint_as_float(0x7fc00000u)};
  const float a = fmaxf(__uint_as_float(amax_bits), kLeast);
  return {127.0f / a, a / 127.0f};
}
// v r rounded once: the fused sum with 1.5 * 2^23, whose unit in the last place is 1, has the code
// in its low byte (two's complement; the constant is even, so ties go to even codes).
__device__ __forceinline__ uint32_t code(float v, float r) { return __float_as_uint(fmaf(v, r, 12582912.0f)); }
__device__ __forceinline__ uint32_t codes4(const float* v, float r) {
  const uint32_t lo = __builtin_amdgcn_perm(code(v[1], r), code(v[0], r), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code(v[3], r), code(v[2], r), 0x04000c0cu);
  return lo | hi;
}
template <typename T>
__device__ __forceinline__ uint2 codes8(const Eight<T>& e, float r) {
  float v[8];
  e.get(v);
  return r == 0.f ? make_uint2(0, 0) : make_uint2(codes4(v, r), codes4(v + 4, r));
}

// Rows of cols elements, ld apart, to rows of q_cols >= cols codes, zeros behind. W waves a row,
// up to 8 chunks of eight elements a lane in registers between the maximum and the codes; longer
// rows are read again. A code is one fused operation and a byte move. Bound by HBM, 3 bytes an
// element from bf16: 131072 x 2304 in 150 to 176 us, 5.2 to 6.0 TB/s; 16384 x 7168 (four waves a row) 69 us, 5.1;
// from fp32 131072 x 1024 115 us, 5.8. 64 x 2304 3.2 us, a launch's latency.
template <typename T, int W>
__global__ __launch_bounds__(256) void quant_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols,
                                                    int q_cols, int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int C = 8;
  __shared__ uint32_t s_max[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, sub = W == 1 ? 0 : wv;
  const int64_t row = W == 1 ? (int64_t)workgroup() * 4 + wv : (int64_t)workgroup();
  if (row >= rows) return;  // (W == 4: of the whole workgroup)
  const T* xr = x + row * ld;
  const int cpr = cols / 8, c0 = sub * 64 + lane;
  Eight<T> v[C];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = c0 + i * 64 * W;
    if (c < cpr) v[i].load(xr + 8 * (int64_t)c);
    else v[i].zero();
  }
#pragma unroll
  for (int i = 0; i < C; ++i) m = max(m, amax8(v[i]));
  for (int c = c0 + C * 64 * W; c < cpr; c += 64 * W) {
    Eight<T> e;
    e.load(xr + 8 * (int64_t)c);
    m = max(m, amax8(e));
  }
  m = wave_max(m);
  if (W > 1) {
    if (lane == 0) s_max[wv] = m;
    __syncthreads();
    m = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
  }
  const RowScale rs = row_scale(m);
  int8_t* qr = q + row * (int64_t)q_cols;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = c0 + i * 64 * W;
    if (c < cpr) *(uint2*)(qr + 8 * (int64_t)c) = codes8(v[i], rs.r);
  }
  for (int c = c0 + C * 64 * W; c < cpr; c += 64 * W) {
    Eight<T> e;
    e.load(xr + 8 * (int64_t)c);
    *(uint2*)(qr + 8 * (int64_t)c) = codes8(e, rs.r);
  }
  for (int c = cpr + c0; c < q_cols / 8; c += 64 * W) *(uint2*)(qr + 8 * (int64_t)c) = make_uint2(0, 0);
  if (lane == 0 && sub == 0) scale[row] = rs.s;
}

__device__ __forceinline__ float element(const uint16_t* p) { return bf2f(*p); }
__device__ __forceinline__ float element(const float* p) { return *p; }

// Rows whose pieces of eight are not aligned: an element at a time, a wave a row, read twice. Far from HBM's
// rate with 2 or 4 bytes a lane and load: 16384 x 2303 54 us from bf16 and 57 from fp32, where 2304 columns
// take 19 and 28; 131072 x 2303 568 and 625 (162 and 277); 64 x 8001 35 us, a wave's 126 steps twice.
template <typename T>
__global__ __launch_bounds__(256) void quant_any_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int cols,
                                                        int8_t* __restrict__ q, float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)workgroup() * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const T* xr = x + row * ld;
  uint32_t m = 0;
  for (int c = lane; c < cols; c += 64) m = max(m, mx::abs_bits(element(xr + c)));
  const RowScale rs = row_scale(wave_max(m));
  int8_t* qr = q + row * (int64_t)cols;
  for (int c = lane; c < cols; c += 64) qr[c] = rs.r == 0.f ? (int8_t)0 : (int8_t)code(element(xr + c), rs.r);
  if (lane == 0) scale[row] = rs.s;
}

__device__ __forceinline__ void put(uint16_t* p, float v) { *p = (uint16_t)f2bf(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

// Codes back to values: a wave a row, in pieces of eight where they are aligned. Bound by HBM:
// 131072 x 2304 to bf16 145 us, 6.2 TB/s; to fp32 386, 3.9 (16384 rows of it 29 us, 6.5). By elements 131072 x
// 2303 312 and 521 us, 16384 x 2303 22 and 33.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dequant_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                                      int64_t rows, int cols, T* __restrict__ x) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)workgroup() * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const float s = scale[row];
  const int8_t* qr = q + row * (int64_t)cols;
  T* xr = x + row * (int64_t)cols;
  if constexpr (VEC) {
    for (int c = lane; c < cols / 8; c += 64) {
      const uint2 w = *(const uint2*)(qr + 8 * (int64_t)c);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = (float)(int8_t)(w.x >> (8 * i)) * s;
        v[4 + i] = (float)(int8_t)(w.y >> (8 * i)) * s;
      }
      if constexpr (sizeof(T) == 2) {
        *(uint4*)(xr + 8 * (int64_t)c) = Chunk<uint16_t>::pack(v);
      } else {
        *(float4*)(xr + 8 * (int64_t)c) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(xr + 8 * (int64_t)c + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  } else {
    for (int c = lane; c < cols; c += 64) put(xr + c, (float)qr[c] * s);
  }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
enum Mode : int { kGateUp = 0, kLinear = 1 };
enum Act : int { kSwiGLU = 0, kOssGLU = 1 };
constexpr float kOssAlpha = 1.702f;

struct Params {
  const int64_t* counts;  // [E]; null: one expert with all rows
  int64_t R;              // rows; segments are clamped to them
  int E, K, N;            // contraction, and the output's columns (gate_up: H)
  const void* x;          // narrow: the rows [R, K] in bf16 or (x_f32) fp32
  int x_f32;
  const int8_t* q;        // wide: rows of padded(K) codes, zeros past K, and their scales
  const float* s;
  const int8_t* wa;       // weights: gate rows, or linear's
  const float* sa;
  const int8_t* wb;       // up rows
  const float* sb;
  int64_t e_rows;         // row n of expert e is row e * e_rows + n * r_rows of wa and wb
  int r_rows;
  const void* bias;       // in bf16 or (bias_f32) fp32: linear [E, N] or null, gpt-oss's b1 [E, 2H] (glu 2j, linear 2j + 1)
  int bias_f32;
  float limit;
  float* h;               // gate_up: [R, N]
  void* y;                // linear: [R, N] in bf16 or (y_f32) fp32; rows past the last expert's are zeroed
  int y_f32;
};

__device__ __forceinline__ int64_t count_of(const Params& p, int e) { return p.counts ? p.counts[e] : p.R; }

// A product's arguments in one go (asked for where they are used, each batch of them is a wait of its
// own), and its segments: by one wave and without a scan where there are no counts. (With scans by
// the whole workgroup and no such shortcut the wide kernel took 1.6 to 2 us longer.)
template <typename F>
__device__ __forceinline__ void begin(const Params& p, int* s_seg, int* s_tile, F tiles_of) {
  asm volatile("" ::"s"(p.counts), "s"(p.R), "s"(p.x), "s"(p.q), "s"(p.s), "s"(p.wa), "s"(p.sa), "s"(p.wb), "s"(p.sb),
               "s"(p.e_rows), "s"(p.r_rows), "s"(p.bias), "s"(p.h), "s"(p.y));
  if (!p.counts) {  // (every thread writes the same)
    s_seg[0] = s_tile[0] = 0;
    s_seg[1] = (int)p.R;
    s_tile[1] = tiles_of((int)p.R);
  } else {
    segments_wave(p, s_seg, s_tile, tiles_of);
  }
}

__device__ __forceinline__ float activation(int act, float g, float u, float limit) {
  if (act == kSwiGLU) return g * mx::sigmoid(g) * u;
  const float a = g > limit ? limit : g, b = u < -limit ? -limit : (u > limit ? limit : u);  // NaN passes
  return a * mx::sigmoid(kOssAlpha * a) * (b + 1.0f);
}

// Sums s of a row by four columns, in their scales. A sum's product with one scale may leave fp32's
// range where the whole does not: with the row's first if that is below 2^97 (a sum is below 2^31),
// else with the column's, which leaves it only where the whole does. Neither goes below the
// normal range. (Rows of the second kind are rare: a branch of the whole wave, not two choices a sum.)
__device__ __forceinline__ void scaled(const i32x4_t& s, float rs, const float (&c)[4], float (&v)[4]) {
#pragma clang fp contract(off)  // (a bias is added to what is rounded here, in every kernel)
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)s[i] * rs * c[i];
  const bool high = rs >= 0x1p97f;
  if (__any(high)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = high ? (float)s[i] * c[i] * rs : v[i];
  }
}

// scales of weight rows n .. n + 3 of expert e (uniform), linear's biases, gpt-oss's of gate and up
// (the last row's past the end)
__device__ __forceinline__ void col_scales(const float* s, const Params& p, int e, int n, float (&v)[4]) {
  const float* se = s + e * p.e_rows;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = se[(uint32_t)(min(n + i, p.N - 1) * p.r_rows)];
}
__device__ __forceinline__ float bias_at(const Params& p, int64_t row0, uint32_t i) {
  return p.bias_f32 ? ((const float*)p.bias + row0)[i] : bf2f(((const uint16_t*)p.bias + row0)[i]);
}
__device__ __forceinline__ void col_bias(const Params& p, int e, int n, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = 0.f;
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = bias_at(p, e * (int64_t)p.N, (uint32_t)min(n + i, p.N - 1));
  }
}
__device__ __forceinline__ void glu_bias(const Params& p, int e, int n, float (&a)[4], float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t at = 2u * (uint32_t)min(n + i, p.N - 1);
    a[i] = bias_at(p, 2 * e * (int64_t)p.N, at);
    b[i] = bias_at(p, 2 * e * (int64_t)p.N, at + 1);
  }
}

// columns n .. n + 3 of row r of y
__device__ __forceinline__ void store4(const Params& p, int64_t r, int n, const float (&v)[4]) {
  if (p.y_f32) {
    float* y = (float*)p.y + r * p.N + n;
    if (p.N % 4 == 0) {
      if (n < p.N) *(float4*)y = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) if (n + i < p.N) y[i] = v[i];
    }
  } else {
    uint16_t* y = (uint16_t*)p.y + r * p.N + n;
    if (p.N % 4 == 0) {
      if (n < p.N) *(uint2*)y = pack4_mid(v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) if (n + i < p.N) y[i] = (uint16_t)f2bf(v[i]);
    }
  }
}
// rows [from, R) of y zeroed by all workgroups together
__device__ __forceinline__ void zero_rest(const Params& p, int from) {
  const int64_t S = (int64_t)gridDim.x * blockDim.x, i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int es = p.y_f32 ? 4 : 2;
  const int64_t at = (int64_t)from * p.N * es, n = (p.R - from) * p.N * es;
  uint8_t* y = (uint8_t*)p.y + at;
  if (at % 16 == 0 && n % 16 == 0)
    for (int64_t i = i0; i < n / 16; i += S) ((uint4*)y)[i] = make_uint4(0, 0, 0, 0);
  else
    for (int64_t i = i0; i < n / 2; i += S) ((uint16_t*)y)[i] = 0;
}

// Many rows per expert: tiles of up to BM rows x BN columns by WM x WN waves of 16 TM x 16 TN, k in
// stages of 128 (a cache line), S stages in LDS, persistent workgroups. Operands reach LDS by
// direct-to-LDS copies, S - 1 stages ahead and across tile boundaries. gate_up's columns alternate
// in blocks of 16 between gate and up, so that a lane holds both. An expert's rows are shared
// evenly by its tiles, a tile's by its waves, in blocks of 16, and a wave's stages are compiled for
// each number of blocks. The scales and biases of a tile come into LDS with its first stage: loads
// of them behind the sums waited for every copy on its way, 4 % of the whole.
//
// What bounds it. Dense, 16384 x 7168 x 7168 on 256 x 256: 650 to 684 us, 2.46 to 2.59 POP/s (the library's int8 product of
// 8192 cubed runs at 1.99, its fp8 one at 2.58): MFMAs 58 % busy at 1.85 GHz, where they alone come to 4.1; no
// bank conflicts (chunk 4 step + g4 of a row: 2 g4 + step met every bank twice). 131072 rows on 256
// experts of 2304 / 1024, on 128 x 256: gate_up 731 us, down 453, 1.7 and 1.4 POP/s: they also move 2.2 and 1.5 GB; without
// their stores they take 240 us less, without the experts' weights from memory 90.
// Measured and not kept: a touch of the lines three stages ahead (7 % slower, 64 x 128 tiles 40 %: the
// copies' path is the narrow place); a tile's results kept in registers and stored between the
// next one's MFMAs (20 % slower, 250 registers); s_setprio for one of a SIMD's two waves (the same);
// rows in two, four, eight passes of all kernels so that codes and h stay in the cache (1479, 1531,
// 1655 us for 1456). For the smallest tile, 1003 x 2880 x 1008 17.5 us with its quantization: eight stages in
// place of four 18.9, k shared by two groups of waves 18.3, a stage's fragments all read at once 17.6.
template <int MODE, int ACT, int WM, int WN, int TM, int TN, int S>
__global__ __launch_bounds__(64 * WM * WN, 2) void wide_kernel(Params p) {
  constexpr int NW = WM * WN, BM = 16 * WM * TM, BN = 16 * WN * TN;
  constexpr int RB = 128, RPC = 8, CPR = 8;                // bytes of a stage's row; rows of a 1 KB copy; chunks of a row
  constexpr int PW = BM / RPC / NW, QC = BN / RPC / NW;    // a wave's copies a stage: of P, of Q
  constexpr int NCOPY = PW + QC, GM = 8;
  static_assert(PW * RPC * NW == BM && QC * RPC * NW == BN && TN % 2 == 0 && 64 * NW >= 256, "whole copies");
  static_assert(NCOPY * (S - 2) < 64, "vmcnt");
  static_assert(S - 1 <= kLeastStages, "the copies are in the next tile at most");
  static_assert(BM % 64 == 0 && BN % 64 == 0 && (BM + BN) / 64 <= NW, "a wave's scales");
  static_assert(S * (BM + BN) * RB + kTileList * 16 + (2 * BN + BM) * 4 + 2 * (kMaxE + 1) * 4 <= 160 * 1024, "LDS, most experts");
  __shared__ __attribute__((aligned(1024))) uint8_t sP[S][BM * RB];
  __shared__ __attribute__((aligned(1024))) uint8_t sQ[S][BN * RB];
  __shared__ int4 s_list[kTileList];  // this workgroup's first tiles: first row, end of its rows, expert, column tile
  // of the tile's columns and rows: scales, and biases as they are stored
  __shared__ __attribute__((aligned(16))) float s_col[BN], s_row[BM];
  __shared__ __attribute__((aligned(16))) uint32_t s_bias[BN];
  extern __shared__ __attribute__((aligned(16))) int s_dyn_i[];
  int* s_seg = s_dyn_i;           // E + 1
  int* s_tile = s_seg + p.E + 1;  // E + 1

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv / WN, wn = wv % WN, ml = lane & 15, g4 = lane >> 4;
  const int E = p.E, K = p.K, N = p.N, KC = K / 16;
  const int NT = MODE == kGateUp ? (N + BN / 2 - 1) / (BN / 2) : (N + BN - 1) / BN;
  const int nk = padded(K) / RB;
  auto tiles_of = [&](int rows) { return (rows + BM - 1) / BM * NT; };
  begin(p, s_seg, s_tile, tiles_of);
  // Each XCD works on a contiguous window of tiles, and with fewer of them than workgroups all XCDs do.
  const int total_tiles = s_tile[E], G = min((int)gridDim.x, (total_tiles + 7) & ~7);
  const int lb = G % 8 == 0 ? (int)(blockIdx.x & 7) * (G >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;

  // An expert's tiles run over its rows first, in groups of GM row tiles, so that the tiles that an
  // XCD works on at a time share rows and columns.
  auto search = [&](int t) {
    const int e = find(s_tile, E, t), local = t - s_tile[e], seg0 = s_seg[e], seg1 = s_seg[e + 1];
    const int blocks = (seg1 - seg0 + 15) >> 4, mtiles = (seg1 - seg0 + BM - 1) / BM;
    const int grp = local / (GM * NT), gm = min(GM, mtiles - grp * GM), in = local - grp * GM * NT, nt = in / gm;
    const int mt = grp * GM + in - nt * gm, per = blocks / mtiles, more = blocks - per * mtiles;
    const int first = mt * per + min(mt, more), end = first + per + (mt < more ? 1 : 0);
    return make_int4(seg0 + 16 * first, min(seg1, seg0 + 16 * end), e, nt);
  };
  if (tid < kTileList && lb + (int64_t)tid * G < total_tiles) s_list[tid] = search(lb + tid * G);
  if (!p.bias)
    for (int i = tid; i < BN; i += 64 * NW) s_bias[i] = 0;
  __syncthreads();
  struct TileRef { int row0, end, e, nt; };
  auto decode = [&](int i) {  // this workgroup's i-th tile
    int4 v;
    if (i < kTileList) v = s_list[i];
    else v = search(lb + i * G);
    return TileRef{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y),
                   __builtin_amdgcn_readfirstlane(v.z), __builtin_amdgcn_readfirstlane(v.w)};
  };
  const int my_tiles = (int)blockIdx.x < G && lb < total_tiles ? (total_tiles - lb + G - 1) / G : 0;

  // ---- copies. One fills RPC rows, lane i row i / 8, chunk i % 8 with the row's chunk
  // (i % 8) ^ ((row >> 1) & 7) (eight lanes that read one chunk of eight rows meet no bank
  // twice). Rows past the tile's or the last column repeat the last one inside (what they give is
  // not stored), chunks past a weight row's end the last one of the row (the other operand has
  // zeros there), and behind the last stage of a workgroup the last tile's first are copied once
  // more. ----
  auto swz = [](int row) { return (row >> 1) & 7; };
  auto q_col = [](int n) { return MODE == kGateUp ? (n >> 5) * 16 + (n & 15) : n; };  // in the tile's columns
  const int p_ld = padded(K);
  const uint8_t *baseP, *baseQ[2];  // of the tile being copied: P, gate (or linear) and up
  uint32_t offP[PW], offQ[QC];
  auto setup = [&](const TileRef& r) {
    int ln = lane;
    asm volatile("" : "+v"(ln));  // what a tile's offsets come from is made again, not kept in registers
    const int crow = ln / CPR, cbit = ln % CPR;
    const int last = r.end - 1 - r.row0, col0 = r.nt * (MODE == kGateUp ? BN / 2 : BN), last_col = N - 1 - col0;
    baseP = (const uint8_t*)p.q + (int64_t)r.row0 * p_ld;
    const int64_t wr = r.e * p.e_rows + (int64_t)col0 * p.r_rows;
    baseQ[0] = (const uint8_t*)p.wa + wr * K;
    if (MODE == kGateUp) baseQ[1] = (const uint8_t*)p.wb + wr * K;
#pragma unroll
    for (int b = 0; b < PW; ++b) {
      const int m = (wv * PW + b) * RPC + crow;
      offP[b] = __umul24(min(m, last), p_ld) + (cbit ^ swz(m)) * 16;
    }
#pragma unroll
    for (int b = 0; b < QC; ++b)
      offQ[b] = __umul24(min(q_col((wv * QC + b) * RPC + crow), last_col), p.r_rows * K);
  };
  auto copy = [&](auto c_c, int kt, int s) {  // copy c of stage kt into buffer s
    constexpr int c = decltype(c_c)::value;
    if constexpr (c < PW) {
      dma16(baseP + kt * RB, offP[c], lds_addr(sP[0] + s * (BM * RB) + (wv * PW + c) * 1024));
    } else {
      constexpr int b = c - PW;
      const uint8_t* base = MODE == kGateUp && (((wv * QC + b) * RPC >> 4) & 1) ? baseQ[1] : baseQ[0];
      const int chunk = min(kt * CPR + (lane % CPR ^ swz((wv * QC + b) * RPC + lane / CPR)), KC - 1);
      dma16(base, offQ[b] + chunk * 16, lds_addr(sQ[0] + s * (BN * RB) + (wv * QC + b) * 1024));
    }
  };
  int ct = 0, ik = 0, bi = 0, bc = 0;  // copy cursor: tile ct, its stage ik, buffer bi; the buffer bc that is read next
  auto advance = [&]() {
    bi = bi + 1 == S ? 0 : bi + 1;
    if (++ik == nk) {
      ik = 0;
      if (++ct < my_tiles) setup(decode(ct));
    }
  };
  if (my_tiles) {
    setup(decode(0));
    for_each<NCOPY>([&](auto c) { copy(c, 0, 0); });
#pragma unroll
    for (int s = 1; s < S - 1; ++s) {
      advance();
      for_each<NCOPY>([&](auto c) { copy(c, ik, s); });
    }
  }
  // The stage that is read next has landed (behind its copies only those of the S - 2 stages after
  // it need still be on their way; an epilogue's loads and stores make the wait longer, not
  // shorter), and every read of the buffer that is filled next is done.
  auto stage_in = [&]() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NCOPY * (S - 2)) : "memory");
  };
  // scales and biases of tile r, a slot a lane
  auto bring = [&](const TileRef& r) {
    if (wv < BN / 64) {
      const int n = wv * 64 + lane, col0 = r.nt * (MODE == kGateUp ? BN / 2 : BN);
      const int col = col0 + min(q_col(n), N - 1 - col0), up = MODE == kGateUp ? (n >> 4) & 1 : 0;
      const int64_t at = r.e * p.e_rows + (int64_t)col * p.r_rows;
      dma4((up ? p.sb : p.sa) + at, lds_addr((const uint8_t*)&s_col[wv * 64]));
      if (p.bias) {
        const uint32_t lds = lds_addr((const uint8_t*)&s_bias[wv * 64]);
        if (p.bias_f32) dma4((const float*)p.bias + (at + up), lds);
        else dma2((const uint16_t*)p.bias + (at + up), lds);
      }
    } else if (wv < (BM + BN) / 64) {
      const int w = wv - BN / 64;
      dma4(p.s + r.row0 + min(w * 64 + lane, r.end - 1 - r.row0), lds_addr((const uint8_t*)&s_row[w * 64]));
    }
  };

  i32x4_t acc[TM][TN];
  int wave_row = 0;
  // A tile's stages by a wave with MB blocks of rows: 2 TN blocks of 16 columns by 64 k each, the
  // fragments read two blocks ahead. The barrier between two stages lies ahead of the last two
  // blocks, whose fragments are there by then, so that MFMAs cover the wait and the next stage's
  // first reads; copies go between the MFMAs of a stage's first half, to land within it.
  auto stages = [&](auto mb_c, const TileRef& cur) {
    constexpr int MB = decltype(mb_c)::value, NB = 2 * TN;
    const uint8_t *cP, *cQ;
    auto enter = [&]() {
      stage_in();
      cP = sP[0] + bc * (BM * RB);
      cQ = sQ[0] + bc * (BN * RB);
      bc = bc + 1 == S ? 0 : bc + 1;
    };
    auto frag = [&](const uint8_t* tile, int row, int step) {
      return *(const i32x4_t*)(tile + row * RB + (((4 * step + g4) ^ swz(row)) << 4));
    };
    i32x4_t af[2][MB > 0 ? MB : 1], bq[4];
    auto read_q = [&](auto n_c) {
      constexpr int n = decltype(n_c)::value % NB;
      bq[n % 4] = frag(cQ, (wn * TN + n % TN) * 16 + ml, n / TN);
    };
    auto read_first = [&]() {
      read_q(std::integral_constant<int, 0>{});
#pragma unroll
      for (int i = 0; i < MB; ++i) af[0][i] = frag(cP, (wave_row + i) * 16 + ml, 0);
      read_q(std::integral_constant<int, 1>{});
    };
    enter();
    bring(cur);
    if constexpr (MB > 0) read_first();
    for (int kt = 0; kt < nk; ++kt) {
      advance();  // ahead of the MFMAs, which the compiler would otherwise sink behind its branches
      if constexpr (MB == 0) {
        for_each<NCOPY>([&](auto c) { copy(c, ik, bi); });
        if (kt + 1 < nk) enter();
      } else {
        for_each<NB>([&](auto n_c) {
          constexpr int n = decltype(n_c)::value, st = n / TN, j = n % TN, first = TN > MB ? TN - MB : 0;
          if constexpr (n + 2 < NB) {
            read_q(std::integral_constant<int, n + 2>{});
          } else if constexpr (n + 2 == NB) {
            if (kt + 1 < nk) {
              enter();
              read_first();
            }
          }
          if constexpr (st == 0 && j >= first) {
#pragma unroll
            for (int i = (j - first) * MB / (TN - first); i < (j - first + 1) * MB / (TN - first); ++i)
              af[1][i] = frag(cP, (wave_row + i) * 16 + ml, 1);
          }
#pragma unroll
          for (int i = 0; i < MB; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bq[n % 4], af[st][i], acc[i][j], 0, 0, 0);
          for_each<NCOPY>([&](auto c) {
            if constexpr (decltype(c)::value * TN / NCOPY == n) copy(c, ik, bi);
          });
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    }
  };

  for (int t = 0; t < my_tiles; ++t) {
    const TileRef cur = decode(t);
    const int blocks = (cur.end - cur.row0 + 15) >> 4, each = (blocks + WM - 1) / WM;
    wave_row = wm * each;  // this wave's first block, and their number
    const int tmv = max(0, min(each, blocks - wave_row));
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
    bool done = false;
    for_each<TM + 1>([&](auto mb) {
      if (!done && tmv == decltype(mb)::value) {
        stages(mb, cur);
        done = true;
      }
    });

    // ---- epilogue: lane holds C[m = .. + ml][n = .. + 4 g4 .. + 3] of each 16-column block ----
#pragma unroll
    for (int b = 0; b < TN / 2; ++b) {
      const int n0 = cur.nt * (MODE == kGateUp ? BN / 2 : BN) + (wn * TN / 2 + b) * (MODE == kGateUp ? 16 : 32);
      if (n0 >= N) continue;
      const int at = (wn * TN + 2 * b) * 16 + 4 * g4;
      float ca[4], cb[4];
      *(float4*)ca = *(const float4*)&s_col[at];
      *(float4*)cb = *(const float4*)&s_col[at + 16];
      float ba[4], bb[4];  // (no biases: zeros)
      if constexpr (MODE == kLinear || ACT == kOssGLU) {
        const int sh = p.bias_f32 ? 0 : 16;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          ba[k] = __uint_as_float(s_bias[at + k] << sh);
          bb[k] = __uint_as_float(s_bias[at + 16 + k] << sh);
        }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i >= tmv) continue;
        const int m = (wave_row + i) * 16 + ml, r = cur.row0 + m;
        const float rs = s_row[m];
        const i32x4_t sa = acc[i][2 * b], sb = acc[i][2 * b + 1];
        float lo[4], hi[4];
        scaled(sa, rs, ca, lo);
        scaled(sb, rs, cb, hi);
        if constexpr (MODE == kLinear || ACT == kOssGLU) {
#pragma unroll
          for (int k = 0; k < 4; ++k) { lo[k] += ba[k]; hi[k] += bb[k]; }
        }
        if (MODE == kGateUp) {
          float h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) h[k] = activation(ACT, lo[k], hi[k], p.limit);
          if (r < cur.end) *(float4*)(p.h + (int64_t)r * N + n0 + 4 * g4) = make_float4(h[0], h[1], h[2], h[3]);
        } else if (p.y_f32 || N % 8) {
          if (r < cur.end) {
            store4(p, r, n0 + 4 * g4, lo);
            store4(p, r, n0 + 16 + 4 * g4, hi);
          }
        } else {
          const uint4 v = span64(pack4_mid(lo), pack4_mid(hi), lane);
          if (r < cur.end && n0 + 8 * g4 < N) *(uint4*)((uint16_t*)p.y + (int64_t)r * N + n0 + 8 * g4) = v;
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last copies write LDS that is not this workgroup's later
  if (MODE == kLinear) zero_rest(p, s_seg[E]);
}

// Few rows per expert: the weights are read once and decide the time, so every byte goes straight
// from memory into the MFMAs' registers. A unit is NB blocks of 16 weight rows (gate_up: 8 gate and
// 8 up rows each) by up to 16 TM rows of one expert; of eight waves, NB take a block each, and 8 / NB
// of them share its k, stages of 128 in turn. A wave multiplies a stage while the next one is on its
// way, through to the following unit. A workgroup's units are consecutive, so
// the rows, which are quantized on the way into LDS, are prepared once per expert and workgroup.
// The columns' scales and biases are asked for ahead of the unit's first stages: loads come back in
// order, so that one asked for where it is used would wait for the stages behind it.
//
// What bounds it: 128 rows on 32 experts of 2880 x 2880 52 us, 265 MB of weights at 5.1 TB/s. One row
// of 7168 x 2048 8.5 us, of which the weights are 3: 0.2 until the arguments are there, 0.7 to the first
// loads, 1.9 until the row is quantized, 4.1 for its weights, 115 KB into each of 128 CUs (28 KB/us is
// what a CU takes in from memory); one token's 8 experts of 256 of 2304 / 1024 11.3 and 8.6 us. Measured
// otherwise: two stages in flight 1 to 15 % slower, more spill; x behind the first weights 1 us
// later; arguments asked for where they are used 0.5 us.
__host__ __device__ constexpr int narrow_stride(int K) { return padded(K) + 16; }  // rows 16 bytes apart mod 128
__host__ __device__ constexpr int64_t narrow_lds(int K, int E, int TM) {  // rows, two units' sums, row scales and maxima, segments
  return 16 * (int64_t)TM * narrow_stride(K) + 2 * 8 * TM * 64 * 16 + 16 * TM * 4 + 8 * 4 + 2 * (E + 1) * (int)sizeof(int);
}

template <int MODE, int ACT, typename T, int NB, int TM>
__global__ __launch_bounds__(512, 4) void narrow_kernel(Params p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_dyn[];
  constexpr int kRows = 16 * TM, KS = 8 / NB, COLS = MODE == kGateUp ? 8 : 16;  // COLS: columns of a block
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = wv % NB, ks = wv / NB, ml = lane & 15, g4 = lane >> 4;
  const int E = p.E, K = p.K, N = p.N, KC = K / 16, nst = (K + 127) / 128;
  const int stride = narrow_stride(K);
  uint8_t* sP = s_dyn;
  i32x4_t* sums = (i32x4_t*)(s_dyn + kRows * stride);  // [2 units][KS][NB][TM][64]
  float* s_scale = (float*)(sums + 2 * 8 * TM * 64);    // [kRows]
  uint32_t* s_max = (uint32_t*)(s_scale + kRows);       // [8]
  int* s_seg = (int*)(s_max + 8);
  int* s_tile = s_seg + E + 1;
  const int nblk = (N + COLS - 1) / COLS, NCB = (nblk + NB - 1) / NB;
  auto tiles_of = [&](int rows) { return (rows + kRows - 1) / kRows * NCB; };
  begin(p, s_seg, s_tile, tiles_of);
  // consecutive units, of which the first workgroups have one more
  const uint32_t total = (uint32_t)__builtin_amdgcn_readfirstlane(s_tile[E]), per = total / gridDim.x, more = total - per * gridDim.x;
  const int u0 = (int)(blockIdx.x * per + min(blockIdx.x, more)), u1 = u0 + (int)per + (blockIdx.x < more ? 1 : 0);
  const int mine = (nst + KS - 1) / KS;  // a wave's stages: ks, ks + KS, ...

  struct Unit { int e, rt, cb; };
  auto decode = [&](int u) {
    Unit r{0, 0, u};
    if (p.counts) {
      r.e = __builtin_amdgcn_readfirstlane(find_wave(s_tile, E, u));
      r.cb = __builtin_amdgcn_readfirstlane(u - s_tile[r.e]);
    }
    if (r.cb >= NCB) {
      r.rt = r.cb / NCB;
      r.cb -= r.rt * NCB;
    }
    return r;
  };
  // this lane's weight row of a unit (blocks past the last one repeat it, rows past N the last row)
  const int8_t* lane_row = MODE == kGateUp ? (ml < 8 ? p.wa : p.wb) + (uint32_t)((ml & 7) * p.r_rows * K) : p.wa;
  auto weight_row = [&](const Unit& u) {
    const int first = min(u.cb * NB + nb, nblk - 1) * COLS;
    const int8_t* row = lane_row + (u.e * p.e_rows + (int64_t)first * p.r_rows) * K;
    return MODE == kGateUp ? row : row + (uint32_t)(min(ml, N - 1 - first) * K);
  };
  struct Stage { i32x4_t w[2]; };
  // chunks past a row's end repeat its last one, against zeros in LDS
  auto load = [&](Stage& g, const int8_t* row, int i) {
    const int c = 8 * (ks + KS * i) + g4;
    g.w[0] = *(const i32x4_t*)(row + (uint32_t)(min(c, KC - 1) * 16));
    g.w[1] = *(const i32x4_t*)(row + (uint32_t)(min(c + 4, KC - 1) * 16));
  };
  // A thread's part of a unit's results: columns 4 fc .. of block fb, row fr.
  constexpr int kQuads = MODE == kGateUp ? 2 : 4;
  const int fl = tid % (16 * kQuads), fi = tid / (16 * kQuads) % TM, fb = tid / (16 * kQuads * TM);
  const int fc = fl >> 4, fr = 16 * fi + (fl & 15);
  struct Cols { float a[4], b[4], ba[4], bb[4]; };  // scales (of gate and up) and biases
  auto first_col = [&](const Unit& u) { return (u.cb * NB + fb) * COLS + 4 * fc; };
  auto load_cols = [&](Cols& c, const Unit& u) {
    if (fb >= NB) return;  // (whole waves, but for gate and up with one block of each: half of the first)
    const int n = min(first_col(u), N - 1);
    col_scales(p.sa, p, u.e, n, c.a);
    if (MODE == kGateUp) col_scales(p.sb, p, u.e, n, c.b);
    if (MODE == kGateUp && ACT == kOssGLU) glu_bias(p, u.e, n, c.ba, c.bb);
    if (MODE == kLinear) col_bias(p, u.e, n, c.ba);
  };

  // Rows row0 .. of x into LDS as codes: a wave a row, or with few rows 2, 4 or 8 waves. A lane's first
  // four chunks are asked for ahead of the unit's weights, behind which they would come back.
  const int cpr = K / 8;
  auto waves_log = [](int rows) { return rows == 1 ? 3 : rows == 2 ? 2 : rows <= 4 ? 1 : 0; };
  auto load_row = [&](Eight<T> (&v)[4], int row0, int rows, int r, int lw) {
    const T* xr = (const T*)p.x + (int64_t)(row0 + r) * K;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = (wv & ((1 << lw) - 1)) * 64 + lane + (k << (6 + lw));
      if (r < rows && c < cpr) v[k].load(xr + 8 * (int64_t)c);
      else v[k].zero();
    }
  };
  auto fill = [&](Eight<T> (&v)[4], int row0, int rows) {
    const int lw = waves_log(rows), W = 1 << lw, sub = wv & (W - 1);
    for (int r = wv >> lw; r < kRows; r += 8 >> lw) {  // (one pass where W > 1)
      const bool on = r < rows;
      const T* xr = (const T*)p.x + (int64_t)(row0 + r) * K;
      uint32_t m = 0;
      if (r >= 8) load_row(v, row0, rows, r, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) m = max(m, amax8(v[k]));
      if (on) {
        for (int c = sub * 64 + lane + 4 * 64 * W; c < cpr; c += 64 * W) {
          Eight<T> e;
          e.load(xr + 8 * (int64_t)c);
          m = max(m, amax8(e));
        }
      }
      m = wave_max(m);
      if (lw) {
        if (lane == 0) s_max[wv] = m;
        __syncthreads();
        for (int k = 0; k < W; ++k) m = max(m, s_max[(wv & ~(W - 1)) + k]);
      }
      if (on) {
        const RowScale rs = row_scale(m);
        uint8_t* row = sP + r * stride;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = sub * 64 + lane + k * 64 * W;
          if (c < cpr) *(uint2*)(row + 8 * c) = codes8(v[k], rs.r);
        }
        for (int c = sub * 64 + lane + 4 * 64 * W; c < cpr; c += 64 * W) {
          Eight<T> e;
          e.load(xr + 8 * (int64_t)c);
          *(uint2*)(row + 8 * c) = codes8(e, rs.r);
        }
        if (sub == 0) {
          for (int c = cpr + lane; c < nst * 16; c += 64) *(uint2*)(row + 8 * c) = make_uint2(0, 0);
          if (lane == 0) s_scale[r] = rs.s;
        }
      }
      if (lw) break;
    }
  };
  auto unit_rows = [&](const Unit& w, int& rows) {
    const int row0 = s_seg[w.e] + w.rt * kRows;
    rows = min(kRows, s_seg[w.e + 1] - row0);
    return row0;
  };

  Stage ga, gb;
  Cols cols{};
  Unit u{};
  const int8_t* wrow = nullptr;
  Eight<T> x[4];
  int at = 0, t = u0, row0 = 0, rows = 0;
  if (u0 < u1) {
    u = decode(u0);
    row0 = unit_rows(u, rows);
    load_row(x, row0, rows, wv >> waves_log(rows), waves_log(rows));
    wrow = weight_row(u);
    load_cols(cols, u);
    load(ga, wrow, 0);
  }
  i32x4_t acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) acc[i] = i32x4_t{0, 0, 0, 0};
  auto multiply = [&](const Stage& g) {
    const int st = ks + KS * at;
    if (st >= nst) return;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if (i > 0 && rows <= 16 * i) continue;
      const uint8_t* a = sP + (16 * i + ml) * stride + st * 128 + g4 * 16;
      acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(g.w[0], *(const i32x4_t*)a, acc[i], 0, 0, 0);
      acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(g.w[1], *(const i32x4_t*)(a + 64), acc[i], 0, 0, 0);
    }
  };
  // stage `at` of unit t from `cur`, with the next one's loads on their way into `nxt`; false where
  // that one is of other rows, or there is none
  auto step = [&](Stage& cur, Stage& nxt) __attribute__((always_inline)) {
    const bool last = at + 1 == mine;
    Unit to = u;
    Cols next{};
    if (last && t + 1 == u1) {
      multiply(cur);
    } else {
      if (last) {
        to = decode(t + 1);
        wrow = weight_row(to);
        load_cols(next, to);
      }
      load(nxt, wrow, last ? 0 : at + 1);
      multiply(cur);
    }
    if (!last) {
      ++at;
      return true;
    }
    at = 0;
    // one barrier a unit: the waves that read these sums come to the next one before anyone
    // writes over them
    i32x4_t* red = sums + (t & 1) * 8 * TM * 64;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      red[((ks * NB + nb) * TM + i) * 64 + lane] = acc[i];
      acc[i] = i32x4_t{0, 0, 0, 0};
    }
    __syncthreads();
    const int n = first_col(u);
    if (fb < NB && fr < rows && n < N) {
      auto sum = [&](int l) {
        i32x4_t v = red[(fb * TM + fi) * 64 + l];
#pragma unroll
        for (int k = 1; k < KS; ++k) {
          const i32x4_t o = red[((k * NB + fb) * TM + fi) * 64 + l];
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] += o[q];
        }
        return v;
      };
      const float s = s_scale[fr];
      float v[4];
      scaled(sum(fl), s, cols.a, v);
      if (MODE == kGateUp) {
        float up[4];
        scaled(sum(fl + 32), s, cols.b, up);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (ACT == kOssGLU) { v[q] += cols.ba[q]; up[q] += cols.bb[q]; }
          v[q] = activation(ACT, v[q], up[q], p.limit);
        }
        *(float4*)(p.h + (int64_t)(row0 + fr) * N + n) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += cols.ba[q];
        store4(p, row0 + fr, n, v);
      }
    }
    const bool same = to.e == u.e && to.rt == u.rt;
    u = to;
    cols = next;
    return ++t < u1 && same;
  };
  while (t < u1) {
    if (t > u0) {
      row0 = unit_rows(u, rows);
      load_row(x, row0, rows, wv >> waves_log(rows), waves_log(rows));
      __syncthreads();  // every wave is done with the rows before
    }
    fill(x, row0, rows);
    __syncthreads();
    while (step(ga, gb)) {
      if (!step(gb, ga)) {
        gb = ga;
        break;
      }
    }
    ga = gb;
  }
  if (MODE == kLinear) zero_rest(p, s_seg[E]);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int kLdsMost = 156 * 1024;  // dynamic LDS of the narrow kernel

static bool aligned16(const void* a) { return ((uintptr_t)a & 15) == 0; }
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// The wide kernel's tiles, with what a stage of 128 k and the rest of a tile take in 10 ns, measured
// where they fill the chip (16384 rows by 7168 x 7168), and the workgroups a CU holds. Experts' weights
// come from memory, which the largest tile, with one stage on its way, waits for: `of_experts`.
struct Tile { int bm, bn, per_cu, stage, of_experts, rest; };
constexpr Tile kTiles[] = {{256, 256, 1, 145, 165, 550}, {128, 256, 1, 90, 90, 280}, {64, 128, 2, 65, 65, 150}, {64, 64, 2, 43, 43, 100}};

// The tile with the least time by that count: as many rounds of the chip as its tiles take, half a
// tile more for each expert that can have rows. Measured against the others (us, 256 x 256 / 128 x
// 256 / 64 x 128 / 64 x 64): 16384 x 7168 x 7168 736 / 796 / 1076 / 1469; 2048 x 2304 x 2304 38 / 27
// / 33 / 32; 1024 x 2304 x 2304 35 / 24 / 20 / 24; 1003 x 2880 x 1008 41 / 27 / 19 / 16; 131072 rows
// on 256 experts of 2304 x 1024 548 / 527 / 698 / 848; 8192 on 32 of 7168 x 2048 250 / 204 / 275 / 294; 16384 on
// 32 of 2880 x 2880 213 / 218; layers of experts 131072 on 256 of 2304 / 1024 1480 / 1451, half as many 850 / 798.
static int pick_tile(int64_t R, int64_t E, int64_t K, int64_t cols, int64_t cus) {
  const int64_t nk = (K + 127) / 128, used = R < E ? R : E;
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = 0; i < 4; ++i) {
    const Tile& t = kTiles[i];
    const int64_t mt = E == 1 ? (R + t.bm - 1) / t.bm : std::max(used, R / t.bm + (used + 1) / 2);
    const int64_t tiles = mt * ((cols + t.bn - 1) / t.bn);
    const int64_t time = (tiles + cus * t.per_cu - 1) / (cus * t.per_cu) * (nk * (E == 1 ? t.stage : t.of_experts) + t.rest);
    if (time < least) { least = time; best = i; }
  }
  return best;
}

template <int MODE, int ACT, int WM, int WN, int TM, int TN, int S>
static void launch_tiles(const Params& p, int per_cu, hipStream_t stream) {
  constexpr int BM = 16 * WM * TM, BN = 16 * WN * TN;
  const int64_t nt = MODE == kGateUp ? (p.N + BN / 2 - 1) / (BN / 2) : (p.N + BN - 1) / BN;
  const int64_t mt = p.E == 1 ? (p.R + BM - 1) / BM : p.R / BM + std::min(p.R, (int64_t)p.E);
  const int64_t g = std::min((mt * nt + 7) / 8 * 8, (int64_t)cu_count() * per_cu);
  hipLaunchKernelGGL((wide_kernel<MODE, ACT, WM, WN, TM, TN, S>), dim3((unsigned)g), dim3(64 * WM * WN),
                     2 * (p.E + 1) * sizeof(int), stream, p);
}
template <int MODE, int ACT>
static void launch_wide(const Params& p, hipStream_t stream) {
  const int tile = pick_tile(p.R, p.E, p.K, MODE == kGateUp ? 2 * (int64_t)p.N : p.N, cu_count());
  const int per_cu = kTiles[tile].per_cu;
  switch (tile) {
    case 0: return launch_tiles<MODE, ACT, 4, 2, 4, 8, 2>(p, per_cu, stream);
    case 1: return launch_tiles<MODE, ACT, 2, 4, 4, 4, 3>(p, per_cu, stream);
    case 2: return launch_tiles<MODE, ACT, 2, 2, 2, 4, 3>(p, per_cu, stream);
    default: return launch_tiles<MODE, ACT, 2, 2, 2, 2, 4>(p, per_cu, stream);
  }
}

// Blocks of 16 rows in a unit of the narrow kernel: two with more than eight rows an expert, where two
// workgroups share a CU's LDS still, else one, where that fits; 0: neither does. With few rows the
// second block is code and LDS for nothing: 16 experts of 2304 / 1024 with 8 rows each 39 us with two in
// their second product, 35 with one; 64 of 1024 / 512 with two rows 32 / 28.
static int narrow_blocks(int64_t R, int64_t E, int K) {
  if (R > 8 * (R < E ? R : E) && narrow_lds(K, (int)E, 2) <= 80 * 1024) return 2;
  return narrow_lds(K, (int)E, 1) <= kLdsMost ? 1 : 0;
}
// The limit of dynamic LDS is a kernel's on a device: raised at its first launch there that needs it.
template <auto Kernel>
static void launch_units(const Params& p, int64_t units, int64_t lds, hipStream_t stream) {
  static std::atomic<uint64_t> raised{0};
  if (lds > 64 * 1024) {
    int dev = 64;
    const uint64_t bit = hipGetDevice(&dev) == hipSuccess && dev < 64 ? (uint64_t)1 << dev : 0;
    if (!bit || !(raised.load() & bit)) {
      if (hipFuncSetAttribute((const void*)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsMost) == hipSuccess)
        raised.fetch_or(bit);
    }
  }
  hipLaunchKernelGGL(Kernel, dim3((unsigned)std::min(units, (int64_t)cu_count() * 2)), dim3(512), (unsigned)lds, stream, p);
}
template <int MODE, int ACT, typename T>
static void launch_narrow_of(const Params& p, hipStream_t stream) {
  const int tm = narrow_blocks(p.R, p.E, p.K);
  const int64_t nblk = MODE == kGateUp ? p.N / 8 : (p.N + 15) / 16, tiles = p.R / (16 * tm) + (p.R < p.E ? p.R : p.E);
  const int64_t lds = narrow_lds(p.K, p.E, tm);
  // One block of weight rows a unit, its k shared by all eight waves, where those do not fill the chip
  // twice (us, one / two / four blocks: 7168 x 2048 9 / 11 / 18, 2304 x 2304 7 / 7 / 9); else four, whose
  // waves read longer runs (64 tokens' rows on 32 experts of 2880 x 2880 65 / 60 / 58, on 256 of 2304 x 2048
  // 228 / 190 / 187).
  const bool small = tiles * nblk <= (int64_t)cu_count() * 2;
  const int64_t units = small ? tiles * nblk : tiles * ((nblk + 3) / 4);
  if (tm == 1) {
    if (small) launch_units<narrow_kernel<MODE, ACT, T, 1, 1>>(p, units, lds, stream);
    else launch_units<narrow_kernel<MODE, ACT, T, 4, 1>>(p, units, lds, stream);
  } else {
    if (small) launch_units<narrow_kernel<MODE, ACT, T, 1, 2>>(p, units, lds, stream);
    else launch_units<narrow_kernel<MODE, ACT, T, 4, 2>>(p, units, lds, stream);
  }
}
template <int MODE, int ACT>
static void launch_narrow(const Params& p, hipStream_t stream) {
  if (MODE == kLinear && p.x_f32) launch_narrow_of<kLinear, kSwiGLU, float>(p, stream);
  else launch_narrow_of<MODE, ACT, uint16_t>(p, stream);
}

// Whether a product with `cols` weight rows (gate_up: of both) goes to the narrow kernel: where it reads
// little and has up to 128 rows an expert, or where there are up to eight, less work in quantizing
// them, which every workgroup does, than in its weights (1024 bytes of a row's two in each of 512
// workgroups a weight row), and not so many weights that more bytes on their way count. Where long
// rows leave a CU one workgroup, half the rows and a fifth of the bytes. us, narrow / wide with its
// quantization: 16 rows of 7168 x 2048 17.3 / 18.1, 48 rows 34 / 20; 96 rows of 2304 x 2304 11.5 / 11.4;
// 16 8.2 / 10.2; 32 of 2880 x 2880 13.2 / 12.2, 16 9.0 / 11.5 (a wide call, of two launches, takes the host 4 us
// more); past 16 rows, weights from memory: 24 rows of 7168 x 2048 16.6 / 19.0, 32 17.5 / 19.0, 40 27.5 / 19.9; 24 of
// 2880 x 2880 10.4 / 11.6, 32 12.7 / 11.8; 32 of 2304 x 2304 10.3 / 10.4; one of 7168 x 7168 19.8 / 21.8, four 22.1 /
// 22.1, seven 28.6 / 22.1; on 32 experts of 2880 x 2880 64 rows 48.8 / 51.9, 256 58.1 / 57.4, of 5760 x 2880 8 rows
// 26.9 / 31.8, 128 112 / 101; on 64 of 2304 x 2048 64 rows 45.6 / 47.5, 256 62.9 / 57.2; on 256 of it 8 10.7 / 12.5, 64
// 47 / 51, 256 142 / 140; on 256 of 1024 x 2304 64 27 / 30, 256 78 / 74; on 32 of 7168 x 4096 8 rows 57 / 38.
static bool takes_narrow(int64_t R, int64_t E, int K, int64_t cols) {
  const int tm = narrow_blocks(R, E, K);
  if (!tm) return false;
  const int64_t used = R < E ? R : E, tiles = E == 1 ? (R + 16 * tm - 1) / (16 * tm) : R / (16 * tm) + used;
  const int64_t bytes = tiles * cols * K;
  const bool two = narrow_lds(K, (int)E, tm) <= 80 * 1024;  // workgroups a CU
  return (R <= 128 * used && bytes <= 30000000) ||
         (R <= (two ? 8 : 4) * used && 1024 * R <= cols * used * used && bytes <= (two ? 330000000 : 60000000));
}

static int check_shape(int64_t R, int E, int K, int N) {
  if (R < 0 || E < 1 || E > kMaxE || K < 16 || N < 1) return kErrInvalidArgument;
  if (K % 16 || K > kMaxK || N > (1 << 22)) return kErrUnsupportedShape;
  if (R >= (int64_t)INT32_MAX / 2) return kErrUnsupportedShape;
  // tiles and units are counted in 32 bits
  if ((R / 16 + E) * ((int64_t)N / 8 + 1) >= (int64_t)0x3fffffff) return kErrUnsupportedShape;
  return kOk;
}

// rows without codes behind theirs where q_cols is cols; x 16-byte aligned rows or not
template <typename T>
static void launch_quant(const T* x, int64_t ld, int64_t rows, int cols, int q_cols, int8_t* q, float* scale,
                         hipStream_t stream) {
  const bool vec = cols % 8 == 0 && aligned16(x) && ld * (int64_t)sizeof(T) % 16 == 0 && ((uintptr_t)q & 7) == 0;
  const int64_t four = (rows + 3) / 4;
  if (!vec) hipLaunchKernelGGL(quant_any_kernel<T>, sliced(four), dim3(256), 0, stream, x, ld, rows, cols, q, scale);
  else if (cols <= 4096)
    hipLaunchKernelGGL((quant_kernel<T, 1>), sliced(four), dim3(256), 0, stream, x, ld, rows, cols, q_cols, q, scale);
  else
    hipLaunchKernelGGL((quant_kernel<T, 4>), sliced(rows), dim3(256), 0, stream, x, ld, rows, cols, q_cols, q, scale);
}

// The rows of a wide product in codes: [R, padded(K)] and [R] scales.
static int64_t row_bytes(int64_t R, int K) { return up256(R * padded(K)) + up256(R * 4); }
struct Rows { int8_t* q; float* s; };
static Rows rows_at(uint8_t* ws, int64_t R, int K) { return {(int8_t*)ws, (float*)(ws + up256(R * padded(K)))}; }

// y = x w^T + b from rows in bf16 or fp32: at x in the workspace or the caller's.
static void product(Params& p, uint8_t* ws, hipStream_t stream) {
  if (takes_narrow(p.R, p.E, p.K, p.N)) return launch_narrow<kLinear, kSwiGLU>(p, stream);
  const Rows rows = rows_at(ws, p.R, p.K);
  if (p.x_f32) launch_quant((const float*)p.x, p.K, p.R, p.K, padded(p.K), rows.q, rows.s, stream);
  else launch_quant((const uint16_t*)p.x, p.K, p.R, p.K, padded(p.K), rows.q, rows.s, stream);
  p.q = rows.q;
  p.s = rows.s;
  launch_wide<kLinear, kSwiGLU>(p, stream);
}

template <int ACT>
static int layer(const uint16_t* x, const int8_t* qw1, const float* sw1, const int8_t* qw2, const float* sw2,
                 const int8_t* qw3, const float* sw3, const void* b1, const void* b2, int bias_f32, float limit,
                 const int64_t* counts, int64_t R, int E, int D, int H, uint8_t* ws, int64_t ws_bytes, uint16_t* y,
                 hipStream_t stream) {
  if (H > (1 << 21)) return kErrUnsupportedShape;
  for (const int st : {check_shape(R, E, D, 2 * H), check_shape(R, E, H, D)})
    if (st) return st;
  if (!counts && E != 1) return kErrInvalidArgument;
  if (R == 0) return kOk;
  if (!x || !qw1 || !sw1 || !qw2 || !sw2 || !qw3 || !sw3 || !ws || !y) return kErrInvalidArgument;
  for (const void* q : {(const void*)x, (const void*)qw1, (const void*)qw2, (const void*)qw3, (const void*)ws, (const void*)y})
    if (!aligned16(q)) return kErrInvalidArgument;
  if (ws_bytes < moe_int8_layer_workspace_bytes(R, E, D, H)) return kErrWorkspace;
  float* h = (float*)ws;
  uint8_t* rows_ws = ws + up256(R * 4 * (int64_t)H);  // x's rows, then h's
  Params p{};
  p.counts = counts; p.R = R; p.E = E; p.K = D; p.N = H;
  p.x = x;
  p.wa = qw1; p.sa = sw1; p.wb = qw3; p.sb = sw3;
  p.e_rows = ACT == kOssGLU ? 2 * (int64_t)H : H;
  p.r_rows = ACT == kOssGLU ? 2 : 1;
  p.bias = b1; p.bias_f32 = bias_f32; p.limit = limit;
  p.h = h;
  if (takes_narrow(R, E, D, 2 * (int64_t)H)) {
    launch_narrow<kGateUp, ACT>(p, stream);
  } else {
    const Rows rows = rows_at(rows_ws, R, D);
    launch_quant(x, D, R, D, padded(D), rows.q, rows.s, stream);
    p.q = rows.q; p.s = rows.s;
    launch_wide<kGateUp, ACT>(p, stream);
  }
  p.K = H; p.N = D;
  p.x = h; p.x_f32 = 1;
  p.wa = qw2; p.sa = sw2; p.e_rows = D; p.r_rows = 1;
  p.bias = b2; p.y = y;
  product(p, rows_ws, stream);
  return launch_status();
}

}  // namespace int8
}  // namespace moe

using namespace moe;
using namespace moe::int8;

MOE_API int moe_int8_quant_rows(const void* x, int64_t ld, int64_t rows, int32_t cols, int32_t dtype, int8_t* q,
                                float* scale, hipStream_t stream) {
  if (rows < 0 || cols < 1 || ld < cols || (dtype != 0 && dtype != 1)) return kErrInvalidArgument;
  if (rows >= kMaxGrid || cols > kMaxCols) return kErrUnsupportedShape;
  if (rows == 0) return kOk;
  if (!x || !q || !scale) return kErrInvalidArgument;
  if (dtype == 0) launch_quant((const uint16_t*)x, ld, rows, cols, cols, q, scale, stream);
  else launch_quant((const float*)x, ld, rows, cols, cols, q, scale, stream);
  return launch_status();
}

MOE_API int moe_int8_dequant_rows(const int8_t* q, const float* scale, int64_t rows, int32_t cols, int32_t dtype, void* x,
                                  hipStream_t stream) {
  if (rows < 0 || cols < 1 || (dtype != 0 && dtype != 1)) return kErrInvalidArgument;
  if (rows >= kMaxGrid || cols > kMaxCols) return kErrUnsupportedShape;
  if (rows == 0) return kOk;
  if (!q || !scale || !x) return kErrInvalidArgument;
  const bool vec = cols % 8 == 0 && aligned16(x) && ((uintptr_t)q & 7) == 0;
  const dim3 grid = sliced((rows + 3) / 4);
  auto launch = [&](auto kernel, auto* out) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, q, scale, rows, cols, out);
  };
  if (dtype == 0) vec ? launch(dequant_kernel<uint16_t, true>, (uint16_t*)x) : launch(dequant_kernel<uint16_t, false>, (uint16_t*)x);
  else vec ? launch(dequant_kernel<float, true>, (float*)x) : launch(dequant_kernel<float, false>, (float*)x);
  return launch_status();
}

MOE_API int moe_int8_tile(int64_t n_rows, int32_t n_experts, int32_t in_features, int32_t columns, int32_t n_cus) {
  const int st = check_shape(n_rows, n_experts, in_features, columns);
  if (st) return st;
  if (n_cus < 1) return kErrInvalidArgument;
  return takes_narrow(n_rows, n_experts, in_features, columns) ? 4 : pick_tile(n_rows, n_experts, in_features, columns, n_cus);
}

MOE_API int64_t moe_int8_linear_workspace_bytes(int64_t n_rows, int32_t n_experts, int32_t in_features, int32_t out_features) {
  const int st = check_shape(n_rows, n_experts, in_features, out_features);
  if (st) return st;
  return takes_narrow(n_rows, n_experts, in_features, out_features) ? 0 : row_bytes(n_rows, in_features);
}

MOE_API int moe_int8_linear(const void* x, int32_t dtype, const int8_t* qw, const float* sw, const void* bias,
                            int32_t bias_dtype, const int64_t* counts, int64_t n_rows, int32_t n_experts,
                            int32_t in_features, int32_t out_features, uint8_t* workspace, int64_t workspace_bytes, void* y,
                            hipStream_t stream) {
  const int st = check_shape(n_rows, n_experts, in_features, out_features);
  if (st) return st;
  if ((dtype != 0 && dtype != 1) || (bias_dtype != 0 && bias_dtype != 1) || (!counts && n_experts != 1))
    return kErrInvalidArgument;
  if (n_rows == 0) return kOk;
  if (!x || !qw || !sw || !y) return kErrInvalidArgument;
  for (const void* q : {x, (const void*)qw, (const void*)workspace, (const void*)y})
    if (!aligned16(q)) return kErrInvalidArgument;
  const int64_t need = moe_int8_linear_workspace_bytes(n_rows, n_experts, in_features, out_features);
  if (need && !workspace) return kErrInvalidArgument;
  if (workspace_bytes < need) return kErrWorkspace;
  Params p{};
  p.counts = counts; p.R = n_rows; p.E = n_experts; p.K = in_features; p.N = out_features;
  p.x = x; p.x_f32 = dtype;
  p.wa = qw; p.sa = sw; p.e_rows = out_features; p.r_rows = 1;
  p.bias = bias; p.bias_f32 = bias_dtype;
  p.y = y; p.y_f32 = dtype;
  product(p, workspace, stream);
  return launch_status();
}

MOE_API int64_t moe_int8_layer_workspace_bytes(int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden) {
  if (n_rows < 0 || n_experts < 1 || dim < 16 || hidden < 16 || dim % 16 || hidden % 16) return kErrInvalidArgument;
  return up256(n_rows * 4 * (int64_t)hidden) + std::max(row_bytes(n_rows, dim), row_bytes(n_rows, hidden));
}

MOE_API int moe_int8_swiglu(const uint16_t* x, const int8_t* qw1, const float* sw1, const int8_t* qw2, const float* sw2,
                            const int8_t* qw3, const float* sw3, const int64_t* counts, int64_t n_rows, int32_t n_experts,
                            int32_t dim, int32_t hidden, uint8_t* workspace, int64_t workspace_bytes, uint16_t* y,
                            hipStream_t stream) {
  return layer<kSwiGLU>(x, qw1, sw1, qw2, sw2, qw3, sw3, nullptr, nullptr, 0, 0.f, counts, n_rows, n_experts, dim, hidden,
                        workspace, workspace_bytes, y, stream);
}

MOE_API int moe_int8_oss(const uint16_t* x, const int8_t* qmlp1, const float* smlp1, const void* mlp1_bias,
                         const int8_t* qmlp2, const float* smlp2, const void* mlp2_bias, int32_t bias_dtype,
                         const int64_t* counts, int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden,
                         float swiglu_limit, uint8_t* workspace, int64_t workspace_bytes, uint16_t* y,
                         hipStream_t stream) {
  if (bias_dtype != 0 && bias_dtype != 1) return kErrInvalidArgument;
  if (n_rows > 0 && (!qmlp1 || !smlp1 || !mlp1_bias || !mlp2_bias)) return kErrInvalidArgument;
  if (dim < 16 || dim % 16) return dim < 16 ? kErrInvalidArgument : kErrUnsupportedShape;
  return layer<kOssGLU>(x, qmlp1, smlp1, qmlp2, smlp2, qmlp1 ? qmlp1 + dim : nullptr, smlp1 ? smlp1 + 1 : nullptr,
                        mlp1_bias, mlp2_bias, bias_dtype, swiglu_limit, counts, n_rows, n_experts, dim, hidden, workspace,
                        workspace_bytes, y, stream);
}
