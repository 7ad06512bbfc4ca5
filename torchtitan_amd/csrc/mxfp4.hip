// MXFP4 on MI355X (gfx950): quantization, and the SwiGLU experts' products of 4-bit operands.
//
// Rows are packed along the contraction, two e2m1 elements per byte, with one e8m0 scale per
// 32 (mx.h). For the rows r of expert e (sorted by expert, counts [E] on the device):
//
//   gate_up   g = xq w1^T, u = xq w3^T, h = act(g, u), written in MXFP4:  rows x 2H, k = D
//   down      y = hq w2^T, written in bf16:                               rows x D,  k = H
//
// with act(g, u) = silu(g) u, or gpt-oss's on interleaved rows with biases b1, b2:
//   g' = min(g + b, L), u' = clamp(u + b, -L, L), g' sigmoid(1.702 g') (u' + 1); y + b2.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 on e2m1 operands: lane (row, q), q = lane / 16, holds 32
// consecutive k of its row, which is one scaling block, and passes that block's scale.
#include <algorithm>

#include "grouped.h"
#include "mx.h"

namespace moe {
namespace mxfp4 {

using mx::kBlock;
using namespace grouped;

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// The columns of a row operand: whole stages of 256, so that every copy of a stage lies inside
// its row, and zeros behind the contraction meet whatever is read of a weight row there.
__host__ __device__ constexpr int padded(int cols) { return (cols + 255) / 256 * 256; }

// ---------------------------------------------------------------------------
// quantization and its inverse
// ---------------------------------------------------------------------------

// Eight elements of a bf16 or fp32 row.
template <typename T> struct Eight;
template <> struct Eight<uint16_t> {
  uint4 v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = *(const uint4*)p; }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&a)[4], float (&b)[4]) const {
    unpack4(make_uint2(v.x, v.y), a);
    unpack4(make_uint2(v.z, v.w), b);
  }
};
template <> struct Eight<float> {
  float4 lo, hi;
  __device__ __forceinline__ void load(const float* p) { lo = *(const float4*)p; hi = *(const float4*)(p + 4); }
  __device__ __forceinline__ void zero() { lo = hi = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&a)[4], float (&b)[4]) const {
    a[0] = lo.x; a[1] = lo.y; a[2] = lo.z; a[3] = lo.w;
    b[0] = hi.x; b[1] = hi.y; b[2] = hi.z; b[3] = hi.w;
  }
};

// Four consecutive lanes hold a block, eight elements each: its scale byte and this lane's
// eight codes.
template <typename T>
__device__ __forceinline__ uint32_t quad_block4(const Eight<T>& x, uint32_t& q) {
  float a[4], b[4];
  x.get(a, b);
  uint32_t m = max(mx::amax4(a), mx::amax4(b));
  m = max(m, (uint32_t)__shfl_xor((int)m, 1));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2));
  const uint32_t s = mx::scale_byte4(m);
  const float f = mx::multiplier(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) { a[i] *= f; b[i] *= f; }
  q = mx::e2m1x8(a, b);
  return s;
}

// Rows of cpr chunks of eight elements to rows of ocpr >= cpr, zeros behind (ocpr == cpr: one
// flat run of chunks). Chunk c's codes are the word q[c], its block's scale scale[c / 4]. One
// pass, bound by HBM (2.53 bytes an element from bf16): 65536 x 2304 in 75 us, 5.1 TB/s (fp32 136
// us, 5.0), 94 behind a kernel that leaves its own 300 MB in the caches; 131072 rows before the
// products 166 us. Eight elements a lane are one 16-byte load and two lane exchanges a block;
// four loads are in flight before the first is used.
template <typename T>
__global__ __launch_bounds__(256) void quant_kernel(const T* __restrict__ x, int64_t n_chunks, int cpr, int ocpr,
                                                    uint32_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const int64_t S = (int64_t)gridDim.x * 256;
  for (int64_t c0 = (int64_t)blockIdx.x * 256 + threadIdx.x; c0 - threadIdx.x < n_chunks; c0 += 4 * S) {
    Eight<T> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * S;
      int64_t at = c;
      bool in = c < n_chunks;
      if (ocpr != cpr) {
        const int64_t r = c / ocpr;
        const int k = (int)(c - r * ocpr);
        at = r * cpr + k;
        in = in && k < cpr;
      }
      if (in) v[u].load(x + 8 * at);
      else v[u].zero();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * S;
      uint32_t w;
      const uint32_t s = quad_block4(v[u], w);
      if (c < n_chunks) {
        q[c] = w;
        if ((c & 3) == 0) scale[c >> 2] = (uint8_t)s;
      }
    }
  }
}

// rows of n scale bytes, each to ld bytes apart with 1.0 behind it
__global__ __launch_bounds__(256) void pad_scales_kernel(const uint8_t* __restrict__ src, int64_t rows, int n, int ld,
                                                         uint8_t* __restrict__ dst) {
  const int64_t total = rows * (ld / 8), S = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += S) {
    const int64_t r = i / (ld / 8);
    const int c = (int)(i - r * (ld / 8)) * 8;
    uint64_t w = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) w |= (uint64_t)(c + k < n ? src[r * n + c + k] : 0x7f) << (8 * k);
    *(uint64_t*)(dst + r * ld + c) = w;
  }
}

// codes back to values: rows of cpr chunks of eight from rows of icpr >= cpr. A product of a
// code and a power of two is exact in bf16 too (two bits of mantissa). Bound by HBM, mostly its
// writes: 65536 x 2304 to bf16 in 64 us, 6.0 TB/s, with the codes partly in the cache still, 73
// without, 5.2 TB/s; to fp32 182 us, 3.8 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void dequant_kernel(const uint32_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                      int64_t n_chunks, int cpr, int icpr, T* __restrict__ x) {
  const int64_t S = (int64_t)gridDim.x * 256;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < n_chunks; c += S) {
    int64_t at = c;
    if (icpr != cpr) {
      const int64_t r = c / cpr;
      at = r * icpr + (c - r * cpr);
    }
    const uint32_t w = q[at];
    const float s = mx::scale_value(scale[at >> 2]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w >> (8 * i), 1.0f, 0);
      v[2 * i] = p[0] * s;
      v[2 * i + 1] = p[1] * s;
    }
    if constexpr (sizeof(T) == 2) {
      *(uint4*)(x + 8 * c) = Chunk<uint16_t>::pack(v);
    } else {
      *(float4*)(x + 8 * c) = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(x + 8 * c + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
}

// ---------------------------------------------------------------------------
// grouped products
// ---------------------------------------------------------------------------
enum Mode : int { kGateUp = 0, kDown = 1 };
enum Act : int { kSwiGLU = 0, kOssGLU = 1 };
constexpr float kOssAlpha = 1.702f;

struct Params {
  const int64_t* counts;  // [E]
  int64_t R;              // rows; segments are clamped to them
  int E, K, N;            // contraction, and the output's columns (gate_up: H)
  const uint16_t* x;      // narrow gate_up: the rows in bf16 [R, K]
  const uint8_t* qp;      // else rows of padded(K) columns in MXFP4, zeros past K, and their scales
  const uint8_t* sp;
  const uint8_t* qa;      // weights: gate rows, or down's
  const uint8_t* sa;
  const uint8_t* qb;      // up rows
  const uint8_t* sb;
  int w_ld;               // bytes between the scales of two weight rows
  int64_t e_rows;         // row n of expert e is row e * e_rows + n * r_rows of qa and qb
  int r_rows;
  const uint16_t* bias;   // gpt-oss: b1 [E, 2H] (glu 2j, linear 2j + 1), b2 [E, D]
  float limit;
  uint8_t* qh;            // gate_up: h, rows of padded(H) columns
  uint8_t* sh;
  uint8_t* g8;            // gate_up with KEEP: g and u in MXFP8 [R, H], scales [R, H / 32]
  uint8_t* gs;
  uint8_t* u8;
  uint8_t* us;
  uint16_t* y;            // down: [R, N]; rows past the last expert's are zeroed
};

__device__ __forceinline__ float activation(int act, float g, float u, float limit) {
  if (act == kSwiGLU) return g * mx::sigmoid(g) * u;
  const float a = g > limit ? limit : g, b = u < -limit ? -limit : (u > limit ? limit : u);  // NaN passes
  return a * mx::sigmoid(kOssAlpha * a) * (b + 1.0f);
}

// rows [from, R) of y zeroed by all workgroups together
__device__ __forceinline__ void zero_rest(const Params& p, int from) {
  const int64_t per_row = p.N / 8, n = (p.R - from) * per_row;
  uint4* y = (uint4*)(p.y + (int64_t)from * p.N);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    y[i] = make_uint4(0, 0, 0, 0);
}

// One row's 32 columns from the accumulators (ga, ua: this lane's columns 4 g .. of the first
// 16, gb, ub: of the second): the activation, quantized, at column hc of row r; with KEEP also
// g and u in MXFP8. gpt-oss's biases: (glu, linear) pairs of this lane's columns.
template <int ACT, bool KEEP>
__device__ __forceinline__ void store_hidden(const Params& p, int64_t r, int hc, int lane, bool valid, float (&ga)[4],
                                             float (&gb)[4], float (&ua)[4], float (&ub)[4], uint4 bias_a,
                                             uint4 bias_b) {
  const int g4 = lane >> 4;
  if constexpr (ACT == kOssGLU) {
    const uint32_t ba[4] = {bias_a.x, bias_a.y, bias_a.z, bias_a.w}, bb[4] = {bias_b.x, bias_b.y, bias_b.z, bias_b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ga[i] += bf_lo(ba[i]); ua[i] += bf_hi(ba[i]);
      gb[i] += bf_lo(bb[i]); ub[i] += bf_hi(bb[i]);
    }
  }
  float ha[4], hb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ha[i] = activation(ACT, ga[i], ua[i], p.limit);
    hb[i] = activation(ACT, gb[i], ub[i], p.limit);
  }
  uint32_t q;
  const uint32_t s = mx::block4(ha, hb, q);
  const int cols = padded(p.N);
  if (valid) {
    uint32_t* row = (uint32_t*)(p.qh + r * (cols / 2));
    row[hc / 8 + g4] = q;
    if (g4 == 0) p.sh[r * (cols / kBlock) + hc / kBlock] = (uint8_t)s;
    if (hc + kBlock == p.N) {  // the row's padding
      for (int i = p.N / 8 + g4; i < cols / 8; i += 4) row[i] = 0;
      for (int i = p.N / kBlock + g4; i < cols / kBlock; i += 4) p.sh[r * (cols / kBlock) + i] = 0;
    }
  }
  if constexpr (KEEP) {
    uint2 kg, ku;
    const uint32_t sg = mx::block8(ga, gb, kg), su = mx::block8(ua, ub, ku);
    if (valid) {
      *(uint2*)(p.g8 + r * p.N + hc + 8 * g4) = kg;
      *(uint2*)(p.u8 + r * p.N + hc + 8 * g4) = ku;
      if (g4 == 0) {
        p.gs[r * (p.N / kBlock) + hc / kBlock] = (uint8_t)sg;
        p.us[r * (p.N / kBlock) + hc / kBlock] = (uint8_t)su;
      }
    }
  }
}

// Many rows per expert: tiles of 256 rows x 256 columns by eight waves of 64 x 128, k in stages of
// 256 (128 bytes a row, a cache line where rows are whole lines), two stages in LDS, persistent
// workgroups, one per CU. Operands and scales reach LDS by direct-to-LDS copies, a stage ahead
// and across tile boundaries. PAIR: the weights' scale rows are only 2-byte aligned (w_ld even
// but not a multiple of 4) and are copied as pairs; odd ones come here padded
// (pad_scales_kernel). gate_up's columns alternate in blocks of 16 between gate and up, so that a
// lane holds both.
//
// What bounds it (131072 rows on 256 experts of 2304 / 1024, call upon call: gate_up 435 us = 2.8
// PFLOP/s, down 302; 547 and 347 in the first calls after a pause): of a tile's 43000 cycles the MFMAs take 18400 and the LDS reads beside them as many, the
// epilogue 7500 (an exponential and a reciprocal, at a quarter of the rate, per element). Measured
// and slower: four waves of 128 x 128 with the fragments a step ahead in registers (569 us: one
// wave per SIMD leaves the epilogue alone on it), two workgroups of 128 x 256 per CU on 64-byte
// rows (521: half again the copies per MFMA), all copies right behind the barrier (538).
template <int MODE, int ACT, bool KEEP, bool PAIR>
__global__ __launch_bounds__(512, 2) void wide_kernel(Params p) {
  constexpr int NW = 8, WGN = 2, TM = 4, TN = 8, BM = 256, BN = 256;  // waves, their columns, blocks of 16 a wave, tile
  constexpr int RB = 128, RPC = 1024 / RB, CPR = RB / 16;             // bytes of a stage's row; rows of a 1 KB copy; chunks of a row
  constexpr int PW = BM / RPC / NW, QC = BN / RPC / NW;               // a wave's copies a stage: of P, of Q,
  constexpr int SUB = PAIR ? 4 : 2, SQC = BN * SUB / 64 / NW;         // and of their scales (P's: one), a dword or a pair a lane
  constexpr int NCOPY = 1 + PW + SQC + QC;
  __shared__ __attribute__((aligned(1024))) uint8_t sP[2][BM * RB];
  __shared__ __attribute__((aligned(1024))) uint8_t sQ[2][BN * RB];
  // scales: a lane's, for each of its 16-row blocks a word (a dword has two lanes' pairs of a
  // stage's steps, PAIR one in its low half), side by side, so that it reads them four at a time
  __shared__ __attribute__((aligned(16))) uint8_t sSP[2][BM * 8];
  __shared__ __attribute__((aligned(16))) uint8_t sSQ[2][SQC * NW * 256];
  __shared__ int4 s_list[kTileList];  // this workgroup's first tiles: first row, end of the segment, expert, column tile
  __shared__ int s_tmp[8];
  extern __shared__ __attribute__((aligned(16))) int s_dyn_i[];
  int* s_seg = s_dyn_i;           // E + 1
  int* s_tile = s_seg + p.E + 1;  // E + 1

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv / WGN, wn = wv % WGN, ml = lane & 15, g4 = lane >> 4;
  const int E = p.E, K = p.K, N = p.N, KB = K / kBlock, kbytes = K / 2;
  const int NT = MODE == kGateUp ? (N + BN / 2 - 1) / (BN / 2) : (N + BN - 1) / BN;
  const int nk = (kbytes + RB - 1) / RB;
  segments(p, s_seg, s_tile, s_tmp, [&](int rows) { return (rows + BM - 1) / BM * NT; });
  const int total_tiles = s_tile[E], G = gridDim.x;
  // each XCD works on a contiguous window of tiles
  const int lb = G % 8 == 0 ? (int)(blockIdx.x & 7) * (G >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;

  // tile t: a search over the experts and a division, 2000 cycles of dependent LDS reads if a wave
  // does it between its MFMAs, so the list is made first, a tile a thread
  auto search = [&](int t) {
    const int e = find(s_tile, E, t), local = t - s_tile[e], seg0 = s_seg[e], seg1 = s_seg[e + 1];
    const int mtiles = (seg1 - seg0 + BM - 1) / BM, nt = local / mtiles;
    return make_int4(seg0 + (local - nt * mtiles) * BM, seg1, e, nt);
  };
  if (tid < kTileList && lb + (int64_t)tid * G < total_tiles) s_list[tid] = search(lb + tid * G);
  __syncthreads();
  struct TileRef { int row0, seg1, e, nt; };
  auto decode = [&](int i) {  // this workgroup's i-th tile
    int4 v;
    if (i < kTileList) v = s_list[i];
    else v = search(lb + i * G);
    return TileRef{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y),
                   __builtin_amdgcn_readfirstlane(v.z), __builtin_amdgcn_readfirstlane(v.w)};
  };
  const int my_tiles = lb < total_tiles ? (total_tiles - lb + G - 1) / G : 0;

  // ---- copies. One fills RPC rows, lane i row i / 8, chunk i % 8 with the row's chunk
  // (i % 8) ^ ((row >> 1) & 7) (eight lanes that read one chunk of eight rows meet no bank
  // twice). A source is a base of the tile and stage in scalar registers and a 32-bit offset per
  // lane. Nothing branches: rows past a segment or the last column repeat the last one inside
  // (what they give is not stored), chunks past a weight row's end the last one of the row (the
  // other operand has zeros there), and behind the last stage of a workgroup the last tile's
  // first is copied once more. ----
  auto swz = [](int row) { return (row >> 1) & 7; };
  auto q_col = [](int n) { return MODE == kGateUp ? (n >> 5) * 16 + (n & 15) : n; };  // in the tile's columns
  // Word i of the scale copies: for a wave row (of P) or column (of Q), row of a 16-row block
  // and part of its stage's scales (a dword of four or PAIR two), the T blocks.
  auto scale_row = [](int i, int t, int sub) { return (i / (16 * sub * t) * t + i % t) * 16 + i / (t * sub) % 16; };
  auto sq_off = [&](int b) { return ((wv * SQC + b) * 64 + lane) / TN % SUB * (PAIR ? 2 : 4); };
  const int p_ld = padded(K) / 2, sp_ld = padded(K) / kBlock;
  const uint8_t *baseP, *baseSP, *baseQ[2];  // of the tile being copied: P, its scales, gate (or down) and up
  uint32_t offP[PW], offQ[QC], offSP;
  const uint8_t* srcSQ[SQC];
  auto setup = [&](const TileRef& r) {
    int ln = lane;
    asm volatile("" : "+v"(ln));  // what a tile's offsets come from is made again, not kept in registers
    const int crow = ln / CPR, cbit = ln % CPR;
    const int last = r.seg1 - 1 - r.row0, col0 = r.nt * (MODE == kGateUp ? BN / 2 : BN), last_col = N - 1 - col0;
    baseP = p.qp + (int64_t)r.row0 * p_ld;
    baseSP = p.sp + (int64_t)r.row0 * sp_ld;
    const int64_t wr = r.e * p.e_rows + (int64_t)col0 * p.r_rows;
    baseQ[0] = p.qa + wr * kbytes;
    if (MODE == kGateUp) baseQ[1] = p.qb + wr * kbytes;
#pragma unroll
    for (int b = 0; b < PW; ++b) {
      const int m = (wv * PW + b) * RPC + crow;
      offP[b] = __umul24(min(m, last), p_ld) + (cbit ^ swz(m)) * 16;
    }
#pragma unroll
    for (int b = 0; b < QC; ++b)
      offQ[b] = __umul24(min(q_col((wv * QC + b) * RPC + crow), last_col), p.r_rows * kbytes);
    const int sp_at = wv * 64 + ln;
    offSP = __umul24(min(scale_row(sp_at, TM, 2), last), sp_ld) + sp_at / TM % 2 * 4;
#pragma unroll
    for (int b = 0; b < SQC; ++b) {
      const int n = scale_row((wv * SQC + b) * 64 + ln, TN, SUB);
      const uint8_t* base = (MODE == kGateUp && ((n >> 4) & 1) ? p.sb : p.sa) + wr * p.w_ld;
      srcSQ[b] = base + __umul24(min(q_col(n), last_col), p.r_rows * p.w_ld);
    }
  };
  auto copy = [&](auto c_c, int kt, int s) {  // copy c of stage kt into buffer s
    constexpr int c = decltype(c_c)::value;
    if constexpr (c == 0) {
      dma4(baseSP + kt * CPR, offSP, lds_addr(&sSP[s][wv * 256]));
    } else if constexpr (c < 1 + PW) {
      constexpr int b = c - 1;
      dma16(baseP + kt * RB, offP[b], lds_addr(&sP[s][(wv * PW + b) * 1024]));
    } else if constexpr (c < 1 + PW + SQC) {
      constexpr int b = c - 1 - PW;
      const uint32_t lds = lds_addr(&sSQ[s][(wv * SQC + b) * 256]);
      if constexpr (PAIR) dma2(srcSQ[b] + min(kt * CPR + sq_off(b), p.w_ld - 2), lds);
      else dma4(srcSQ[b] + min(kt * CPR + sq_off(b), p.w_ld - 4), lds);
    } else {
      constexpr int b = c - 1 - PW - SQC;
      const uint8_t* base = MODE == kGateUp && (((wv * QC + b) * RPC >> 4) & 1) ? baseQ[1] : baseQ[0];
      const int chunk = min(kt * CPR + (lane % CPR ^ swz((wv * QC + b) * RPC + lane / CPR)), KB - 1);
      dma16(base, offQ[b] + chunk * 16, lds_addr(&sQ[s][(wv * QC + b) * 1024]));
    }
  };
  int ct = 0, ik = 0, bi = 0, bc = 0;  // copy cursor: tile ct, its stage ik, buffer bi; the buffer bc that is read next
  auto advance = [&]() {
    bi ^= 1;
    if (++ik == nk) {
      ik = 0;
      if (++ct < my_tiles) setup(decode(ct));
    }
  };
  if (my_tiles) {
    setup(decode(0));
    for_each<NCOPY>([&](auto c) { copy(c, 0, 0); });
  }

  for (int t = 0; t < my_tiles; ++t) {
    const TileRef cur = decode(t);
    const int row0 = cur.row0, seg1 = cur.seg1;
    // the stage that is read next has landed (its copies are the last there are; an epilogue's
    // stores are waited for too), and every read of the buffer that is filled next is done
    auto stage_in = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // 16-row blocks of this wave with rows in them; a wave without any only copies
    const int tmv = min(TM, max(0, (seg1 - (row0 + wm * TM * 16) + 15) >> 4));
    if (tmv == 0) {
      for (int kt = 0; kt < nk; ++kt) {
        advance();
        stage_in();
        bc ^= 1;
        for_each<NCOPY>([&](auto c) { copy(c, ik, bi); });
      }
      continue;
    }
    f32x4_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    for (int kt = 0; kt < nk; ++kt) {
      advance();  // ahead of the MFMAs, which the compiler would otherwise sink behind its branches
      stage_in();
      const uint8_t *cP = sP[bc], *cQ = sQ[bc], *cSP = sSP[bc], *cSQ = sSQ[bc];
      bc ^= 1;
      // lane row g4 takes a row's chunk 2 g4 + step, so that its two scales of a stage lie side by side
      int scp[TM], scq[TN];
      v8i_t af[TM], bq[2];
      auto frag = [&](const uint8_t* tile, int row, int step) {
        const uint4 v = *(const uint4*)(tile + row * RB + (((2 * g4 + step) ^ swz(row)) << 4));
        return v8i_t{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
      };
      const int sh_p = 16 * (g4 & 1), sh_q = PAIR ? 0 : sh_p;
      {
        const uint4 w = *(const uint4*)(cSP + ((wm * 16 + ml) * 2 + (g4 >> 1)) * TM * 4);
        scp[0] = w.x >> sh_p; scp[1] = w.y >> sh_p; scp[2] = w.z >> sh_p; scp[3] = w.w >> sh_p;
      }
#pragma unroll
      for (int j = 0; j < TN; j += 4) {
        const uint4 w = *(const uint4*)(cSQ + (((wn * 16 + ml) * SUB + (PAIR ? g4 : g4 >> 1)) * TN + j) * 4);
        scq[j] = w.x >> sh_q; scq[j + 1] = w.y >> sh_q; scq[j + 2] = w.z >> sh_q; scq[j + 3] = w.w >> sh_q;
      }
      // the next stage's copies go between the MFMAs, one behind each of the first blocks of
      // columns: issued together right behind the barrier they hold every wave up at once (a
      // copy takes the CU's address path 16 cycles)
      auto step = [&](auto s_c) {
        constexpr int st = decltype(s_c)::value;
#pragma unroll
        for (int i = 0; i < TM; ++i) af[i] = frag(cP, (wm * TM + i) * 16 + ml, st);
        bq[0] = frag(cQ, wn * TN * 16 + ml, st);
        for_each<TN>([&](auto j_c) {
          constexpr int j = decltype(j_c)::value;
          if constexpr (j + 1 < TN) bq[(j + 1) & 1] = frag(cQ, (wn * TN + j + 1) * 16 + ml, st);
#pragma unroll
          for (int i = 0; i < TM; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bq[j & 1], af[i], acc[i][j], 4, 4, st, scq[j],
                                                                         st, scp[i]);
          constexpr int slot = st * TN + j, slots = 2 * TN;
          for_each<NCOPY>([&](auto c) {
            if constexpr (decltype(c)::value * slots / NCOPY == slot) copy(c, ik, bi);
          });
          __builtin_amdgcn_sched_barrier(0);
        });
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
    }

    // ---- epilogue: lane holds C[m = .. + ml][n = .. + 4 g4 .. + 3] of each 16-column block ----
    if (MODE == kGateUp) {
#pragma unroll
      for (int b = 0; b < TN / 4; ++b) {
        const int hc = cur.nt * (BN / 2) + wn * (TN * 8) + b * 32;
        if (hc >= N) continue;
        uint4 bias_a{}, bias_b{};
        if constexpr (ACT == kOssGLU) {
          const uint16_t* bp = p.bias + (int64_t)cur.e * 2 * N + 2 * (hc + 4 * g4);
          bias_a = *(const uint4*)bp;
          bias_b = *(const uint4*)(bp + 32);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (i >= tmv) continue;
          const int r = row0 + (wm * TM + i) * 16 + ml;
          float v[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) v[j][q] = acc[i][4 * b + j][q];
          store_hidden<ACT, KEEP>(p, r, hc, lane, r < seg1, v[0], v[2], v[1], v[3], bias_a, bias_b);
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < TN / 2; ++b) {
        const int n0 = cur.nt * BN + wn * TN * 16 + b * 32;
        if (n0 >= N) continue;
        float ba[4] = {0.f, 0.f, 0.f, 0.f}, bb[4] = {0.f, 0.f, 0.f, 0.f};
        if constexpr (ACT == kOssGLU) {
          const uint16_t* bp = p.bias + (int64_t)cur.e * N + n0 + 4 * g4;
          unpack4(*(const uint2*)bp, ba);
          unpack4(*(const uint2*)(bp + 16), bb);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (i >= tmv) continue;
          const int r = row0 + (wm * TM + i) * 16 + ml;
          float lo[4], hi[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            lo[q] = acc[i][2 * b][q] + ba[q];
            hi[q] = acc[i][2 * b + 1][q] + bb[q];
          }
          const uint4 v = span64(pack4(lo), pack4(hi), lane);
          if (r < seg1) *(uint4*)(p.y + (int64_t)r * N + n0 + 8 * g4) = v;
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last copies write LDS that is not this workgroup's later
  if (MODE == kDown) zero_rest(p, s_seg[E]);
}

// Few rows per expert: the weights are read once and decide the time, so every byte goes
// straight from memory into the MFMAs' registers. A unit is 64 weight rows (gate_up: 32 gate and
// 32 up rows, one scaling block of h; down: 64 columns) by up to 16 TM rows of one expert; eight
// waves take four blocks of 16 weight rows by the even and the odd 256-k stages. A wave keeps two
// stages in registers, in turn, one's loads in flight while the other multiplies, through to the
// following unit. A workgroup's units are consecutive, so the rows, which gate_up quantizes from
// bf16 on the way into LDS, are prepared once per expert and workgroup. The weights' scales come
// through LDS, a unit ahead: 64 rows of them are one or two runs of memory, of which each thread
// brings two bytes a stage.
//
// What bounds it: the weights' bytes. One row on each of 57 experts of 7168 / 2048 takes 236 us, 5.6
// TB/s; four rows each on 256 of 2304 / 1024 189 us, 5.1 TB/s; eight each on 32 of gpt-oss's 2880 / 2880
// 101 us, 4.2 TB/s (rows of 1440 bytes: a stage of 128 straddles two cache lines). One token's 8
// experts of 256 take 17 us, of which the 30 MB are 6: two launches that each wait for the counts,
// then for the weights.
// Measured otherwise: scales loaded where they are multiplied, two bytes a lane from 16 rows, 248, 203
// and 123 us (a load costs by the cache lines it touches, and these were as many as the weights');
// a register copy of the stage in flight (the loop not in pairs) waits for its loads: 220 and 139
// us. More in flight was slower: groups of two stages 206 and 125 us, three or four single ones in
// turn 199 to 219 and 126 to 134; loads past the caches 223 and 160.
__host__ __device__ constexpr int narrow_stride(int K) { return (K + 255) / 256 * 128 + 16; }  // rows 16 bytes apart mod 128
__host__ __device__ constexpr int64_t narrow_lds(int K, int E, int TM) {  // rows and their scales, sums, the weights' scales, segments
  return 16 * (int64_t)TM * (narrow_stride(K) + (K + 255) / 256 * 8) + 2 * 8 * 64 * 16 + 2 * 64 * (K / kBlock) +
         2 * (E + 1) * (int)sizeof(int);
}

template <int MODE, int ACT, bool ODD, int TM>
__global__ __launch_bounds__(512, 4) void narrow_kernel(Params p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_dyn[];
  constexpr int kRows = 16 * TM;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = wv & 3, ks = wv >> 2, ml = lane & 15, g4 = lane >> 4;
  const int E = p.E, K = p.K, N = p.N, KB = K / kBlock, kbytes = K / 2, nst = (K + 255) / 256;
  const int stride = narrow_stride(K), sld = nst * 8;
  uint8_t* sP = s_dyn;
  f32x4_t* sums = (f32x4_t*)(s_dyn + kRows * (stride + sld));  // [2 units or row blocks][2 ks][4 nb][64]
  uint8_t* sc = s_dyn + kRows * stride;
  uint8_t* sW = (uint8_t*)(sums + 2 * 8 * 64);  // two units' weight scales, 64 rows of KB
  int* s_seg = (int*)(sW + 2 * 64 * KB);
  int* s_tile = s_seg + E + 1;
  const int NCB = MODE == kGateUp ? N / 32 : (N + 63) / 64;
  segments_wave(p, s_seg, s_tile, [&](int rows) { return (rows + kRows - 1) / kRows * NCB; });
  const int64_t total = s_tile[E];
  const int u0 = (int)(total * blockIdx.x / gridDim.x), u1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
  const int mine = (nst + 1) / 2;  // stages of a half: ks, ks + 2, ...

  struct Stage { uint4 w[2]; uint16_t s; };  // s: a pair of the next unit's scales
  struct Unit { int e, rt, cb; };
  auto decode = [&](int u) {
    Unit r;
    r.e = __builtin_amdgcn_readfirstlane(find_wave(s_tile, E, u));
    const int local = __builtin_amdgcn_readfirstlane(u - s_tile[r.e]);
    r.rt = local / NCB;
    r.cb = local - r.rt * NCB;
    return r;
  };
  // The 64 weight rows' scales of a unit, in the order of their addresses (gate_up of separate
  // weights: 32 gate rows, then 32 up rows): bytes o .. of them, o at most n from the end.
  auto scales = [&](const Unit& u, int o, int n) {
    if (MODE == kGateUp && ACT == kSwiGLU) {
      const int64_t row = u.e * p.e_rows + u.cb * 32;
      o = min(o, 64 * KB - n);
      return o < 32 * KB ? p.sa + row * KB + o : p.sb + row * KB + (o - 32 * KB);
    }
    const int64_t row = u.e * p.e_rows + u.cb * 64;
    return p.sa + row * KB + min(o, (MODE == kGateUp ? 64 : min(64, N - u.cb * 64)) * KB - n);
  };
  const int srow = MODE == kDown ? nb * 16 + ml : ACT == kSwiGLU ? (nb & 1) * 16 + ml + (nb >= 2 ? 32 : 0)
                                                                : 2 * ((nb & 1) * 16 + ml) + (nb >= 2 ? 1 : 0);
  // Stage i of unit u, and the thread's pair of the scales of unit `then` behind it. Without
  // branches, so that the compiler's waits leave the other stage in flight: chunks past the row
  // repeat its last ones, against zeros in LDS; columns past N repeat the last block's (nothing
  // is stored of them); and behind the last unit one piece is loaded again.
  auto load = [&](Stage& g, const Unit& u, const Unit& then, int i, bool on) {
    const int col = MODE == kGateUp ? u.cb * 32 + (nb & 1) * 16 : min(u.cb * 64 + nb * 16, N - 16);
    const bool up = MODE == kGateUp && nb >= 2;
    const uint8_t* wq = (up ? p.qb : p.qa) + (u.e * p.e_rows + (int64_t)col * p.r_rows) * kbytes;
    const uint32_t lq = on ? (uint32_t)(ml * p.r_rows) * (uint32_t)kbytes : 0u;
    const int c = on ? 8 * (ks + 2 * i) + 2 * g4 : 0;  // this lane's chunks of 32 k: c, c + 1
    if constexpr (ODD) {
      g.w[0] = *(const uint4*)(wq + (lq + (uint32_t)min(c, KB - 1) * 16));
      g.w[1] = *(const uint4*)(wq + (lq + (uint32_t)min(c + 1, KB - 1) * 16));
    } else {
      const uint32_t at = lq + (uint32_t)min(c, KB - 2) * 16;
      g.w[0] = *(const uint4*)(wq + at);
      g.w[1] = *(const uint4*)(wq + (at + 16));
    }
    g.s = *(const uint16_t*)scales(then, 2 * (i * 512 + tid), 2);
  };
  struct Rows { Eight<uint16_t> v[4]; };
  auto load_rows = [&](Rows& x, int row0, int rows, int c0) {
    const int n = rows * (K / 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + 512 * k;
      if (c < n) x.v[k].load(p.x + (int64_t)row0 * K + (int64_t)c * 8);
      else x.v[k].zero();
    }
  };
  auto fill = [&](Rows& x, int row0, int rows) {  // x: the thread's first chunks, which are there already
    if (MODE == kGateUp) {
      const int cpr = K / 8, n = rows * cpr;
      for (int c0 = tid; c0 - tid < n; c0 += 4 * 512) {
        if (c0 != tid) load_rows(x, row0, rows, c0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = c0 + 512 * k;
          uint32_t w;
          const uint32_t s = quad_block4(x.v[k], w);
          if (c < n) {
            const int r = c / cpr, at = c - r * cpr;
            *(uint32_t*)(sP + r * stride + at * 4) = w;
            if ((at & 3) == 0) sc[r * sld + (at >> 2)] = (uint8_t)s;
          }
        }
      }
      for (int i = tid; i < rows * (sld - KB); i += 512) {
        const int r = i / (sld - KB), c = KB + i % (sld - KB);
        *(uint4*)(sP + r * stride + c * 16) = make_uint4(0, 0, 0, 0);
        sc[r * sld + c] = 0x7f;
      }
    } else {
      for (int i = tid; i < rows * sld; i += 512) {
        const int r = i / sld, c = i - r * sld;
        *(uint4*)(sP + r * stride + c * 16) = *(const uint4*)(p.qp + (int64_t)(row0 + r) * (padded(K) / 2) + c * 16);
      }
      for (int i = tid; i < rows * nst; i += 512) {
        const int r = i / nst, st = i - r * nst;
        *(uint2*)(sc + r * sld + st * 8) = *(const uint2*)(p.sp + (int64_t)(row0 + r) * (padded(K) / kBlock) + st * 8);
      }
    }
  };

  Stage ga, gb;
  Unit u{}, un{};
  Rows x;
  auto unit_rows = [&](const Unit& w, int& rows) {
    const int row0 = s_seg[w.e] + w.rt * kRows;
    rows = min(kRows, s_seg[w.e + 1] - row0);
    return row0;
  };
  if (u0 < u1) {
    u = decode(u0);
    if (MODE == kGateUp) {  // ahead of the weights: the rows are waited for first
      int rows;
      const int row0 = unit_rows(u, rows);
      load_rows(x, row0, rows, tid);
    }
    un = u0 + 1 < u1 ? decode(u0 + 1) : u;
    uint8_t* own = sW + (u0 & 1) * 64 * KB;
    const uint4 first = *(const uint4*)scales(u, tid * 16, 16);
    load(ga, u, un, 0, true);
    *(uint4*)(own + min(tid * 16, 64 * KB - 16)) = first;
    for (int o = (tid + 512) * 16; o < 64 * KB; o += 512 * 16) *(uint4*)(own + o) = *(const uint4*)scales(u, o, 16);
  }
  int at = 0, t = u0, row0 = 0, rows = 0;
  f32x4_t acc[TM] = {};
  // unit t's stage `at` from `cur`, with the next one's loads on their way into `nxt`; false
  // where that one is of other rows, or there is none
  auto step = [&](Stage& cur, Stage& nxt) __attribute__((always_inline)) {
    const bool last = at + 1 == mine;
    const Unit to = last ? un : u, then = last && t + 2 < u1 ? decode(t + 2) : un;
    load(nxt, to, then, last ? 0 : at + 1, !last || t + 1 < u1);
    const int st = ks + 2 * at;
    *(uint16_t*)(sW + ((t + 1) & 1) * 64 * KB + min(2 * (at * 512 + tid), 64 * KB - 2)) = cur.s;
    if (st < nst) {
      const uint8_t* ws = sW + (t & 1) * 64 * KB + srow * KB;
      const int c = 8 * st + 2 * g4;
      const uint32_t sw = ODD ? ws[min(c, KB - 1)] | (ws[min(c + 1, KB - 1)] << 8) : *(const uint16_t*)(ws + min(c, KB - 2));
      const uint4 b0 = cur.w[0], b1 = cur.w[1];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i > 0 && rows <= 16 * i) continue;
        const int r = 16 * i + ml;
        const uint32_t sp = *(const uint16_t*)(sc + r * sld + st * 8 + 2 * g4);
        const uint4 a0 = *(const uint4*)(sP + r * stride + st * 128 + g4 * 32);
        const uint4 a1 = *(const uint4*)(sP + r * stride + st * 128 + g4 * 32 + 16);
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            v8i_t{(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, 0, 0, 0, 0},
            v8i_t{(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, 0, 0, 0, 0}, acc[i], 4, 4, 0, (int)sw, 0, (int)sp);
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            v8i_t{(int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w, 0, 0, 0, 0},
            v8i_t{(int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w, 0, 0, 0, 0}, acc[i], 4, 4, 1, (int)sw, 1, (int)sp);
      }
    }
    if (!last) {
      ++at;
      return true;
    }
    at = 0;
    // one barrier a unit: the waves that read these sums come to the next one before anyone
    // writes over them; they take turns, so that none is behind the others for good
    // (with two blocks of rows in the two buffers: with a barrier for that)
    f32x4_t* red = sums + (TM == 1 ? t & 1 : 0) * 8 * 64;
    if (TM > 1) __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i) red[((i * 2 + ks) * 4 + nb) * 64 + lane] = acc[i];
    __syncthreads();
    const int turn = (wv + t) & 7, blk = MODE == kGateUp ? turn : turn >> 1;  // this wave's block of rows
    auto sum = [&](int b, float (&v)[4]) {
      const f32x4_t a = red[(blk * 8 + b) * 64 + lane], c = red[(blk * 8 + 4 + b) * 64 + lane];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = a[q] + c[q];
    };
    if (MODE == kGateUp) {
      if (blk < TM && 16 * blk < rows) {
        float ha[4], hb[4], ua[4], ub[4];
        sum(0, ha);
        sum(1, hb);
        sum(2, ua);
        sum(3, ub);
        const int hc = u.cb * 32, r = 16 * blk + ml;
        uint4 bias_a{}, bias_b{};
        if constexpr (ACT == kOssGLU) {
          const uint16_t* bp = p.bias + (int64_t)u.e * 2 * N + 2 * (hc + 4 * g4);
          bias_a = *(const uint4*)bp;
          bias_b = *(const uint4*)(bp + 32);
        }
        store_hidden<ACT, false>(p, row0 + r, hc, lane, r < rows, ha, hb, ua, ub, bias_a, bias_b);
      }
    } else if (blk < TM && 16 * blk < rows) {
      const int pr = turn & 1, n0 = u.cb * 64 + pr * 32, r = 16 * blk + ml;
      if (n0 < N) {
        float lo[4], hi[4];
        sum(2 * pr, lo);
        sum(2 * pr + 1, hi);
        if constexpr (ACT == kOssGLU) {
          float ba[4], bb[4];
          const uint16_t* bp = p.bias + (int64_t)u.e * N + n0 + 4 * g4;
          unpack4(*(const uint2*)bp, ba);
          unpack4(*(const uint2*)(bp + 16), bb);
#pragma unroll
          for (int q = 0; q < 4; ++q) { lo[q] += ba[q]; hi[q] += bb[q]; }
        }
        const uint4 v = span64(pack4(lo), pack4(hi), lane);
        if (r < rows) *(uint4*)(p.y + (int64_t)(row0 + r) * N + n0 + 8 * g4) = v;
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const bool same = to.e == u.e && to.rt == u.rt;
    u = to;
    un = then;
    return ++t < u1 && same;
  };
  while (t < u1) {
    row0 = unit_rows(u, rows);
    if (t > u0) {
      if (MODE == kGateUp) load_rows(x, row0, rows, tid);
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
  if (MODE == kDown) zero_rest(p, s_seg[E]);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int kLdsMost = 156 * 1024;  // dynamic LDS of the narrow kernel

template <int MODE, int ACT, bool KEEP>
static void launch_wide(const Params& p, hipStream_t stream) {
  const int64_t nt = MODE == kGateUp ? (p.N + 127) / 128 : (p.N + 255) / 256;
  int64_t g = (p.R / 256 + (p.R < p.E ? p.R : p.E)) * nt;
  const int64_t most = cu_count();
  if (g > most) g = most;
  if (g >= 8) g -= g % 8;
  const unsigned lds = 2 * (p.E + 1) * sizeof(int);
  if (p.w_ld % 4 == 0)
    hipLaunchKernelGGL((wide_kernel<MODE, ACT, KEEP, false>), dim3((unsigned)g), dim3(512), lds, stream, p);
  else
    hipLaunchKernelGGL((wide_kernel<MODE, ACT, KEEP, true>), dim3((unsigned)g), dim3(512), lds, stream, p);
}
// Blocks of 16 rows in a unit of the narrow kernel on a contraction of K: two where two workgroups
// share a CU's LDS still, else one, where that fits; 0: neither does. With up to eight rows per
// expert one and two take the same time (189 / 189 us at 4 of 256 experts of 2304 / 1024, 210 / 200 at 8);
// with more, one reads the weights more often (16 rows 275 / 219, gpt-oss 129 / 111), and two without
// the second workgroup lose what they win (192 us instead of 161 at 8 rows of 32 of 7168 / 2048).
static int narrow_blocks(int K, int64_t E) {
  return narrow_lds(K, (int)E, 2) <= 80 * 1024 ? 2 : narrow_lds(K, (int)E, 1) <= kLdsMost ? 1 : 0;
}

template <int MODE, int ACT>
static void launch_narrow(const Params& p, hipStream_t stream) {
  const int tm = narrow_blocks(p.K, p.E);
  const int64_t ncb = MODE == kGateUp ? p.N / 32 : (p.N + 63) / 64;
  int64_t g = (p.R / (16 * tm) + (p.R < p.E ? p.R : p.E)) * ncb;
  const int64_t most = (int64_t)cu_count() * 2;
  if (g > most) g = most;
  const int64_t lds = narrow_lds(p.K, p.E, tm);
  auto launch = [&](auto kernel) {
    if (lds > 64 * 1024)
      (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsMost);
    hipLaunchKernelGGL(kernel, dim3((unsigned)g), dim3(512), (unsigned)lds, stream, p);
  };
  const bool odd = p.K / kBlock % 2;
  if (tm == 1) odd ? launch(narrow_kernel<MODE, ACT, true, 1>) : launch(narrow_kernel<MODE, ACT, false, 1>);
  else odd ? launch(narrow_kernel<MODE, ACT, true, 2>) : launch(narrow_kernel<MODE, ACT, false, 2>);
}

// The narrow kernel takes up to 20 rows per expert that can have one (12 with units of one block),
// and small work, where the wide kernel's tiles leave most of the chip idle, where its rows fit
// into LDS (us, narrow / wide with its quantization; rows per expert): 256 experts of 2304 / 1024 one
// token 18 / 30, 4 rows 189 / 220, 16 rows 219 / 238, 24 rows 247 / 247, 31 rows 292 / 268; 32 of
// gpt-oss's 2880 / 2880 8 rows 101 / 152, 16 rows 111 / 156, 24 rows 132 / 159, 50 rows 176 / 168; 32 of 7168 /
// 2048 8 rows 161 / 191, 12 rows 192 / 194, 16 rows 218 / 198; 16 of 2304 / 1024 16 rows 29 / 32, 24 rows 39 /
// 33. Small: 8 experts of 2048 / 1408 16 rows 22 / 32; 16 of 320 / 704 19 rows 16 / 24; one of 512 / 512 128
// rows 13 / 22. One bound in rows fits 256 experts and misses on few wide ones: gpt-oss's cross near
// 45 rows, and between 21 and there take the wide kernel, 159 us where the narrow one took 132.
static bool takes_narrow(int64_t R, int64_t E, int D, int H) {
  const int tm = std::min(narrow_blocks(D, E), narrow_blocks(H, E));
  const int64_t cols = 2 * (int64_t)H > D ? 2 * (int64_t)H : D;
  return tm && (R <= (tm == 2 ? 20 : 12) * (R < E ? R : E) || R * ((cols + 255) / 256) <= 1536);
}

static int check_shape(int64_t R, int E, int D, int H) {
  if (R < 0 || E < 1 || E > kMaxE || D < kBlock || H < kBlock) return kErrInvalidArgument;
  if (D % kBlock || H % kBlock || D > (1 << 22) || H > (1 << 22)) return kErrUnsupportedShape;
  if (R >= (int64_t)INT32_MAX / 2) return kErrUnsupportedShape;
  // tiles and units are counted in 32 bits
  if ((R / 16 + E) * ((int64_t)(D > H ? D : H) / 32 + 1) >= (int64_t)0x3fffffff) return kErrUnsupportedShape;
  return kOk;
}
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
static int padded_blocks(int cols) { return padded(cols) / kBlock; }
static int64_t row_bytes(int64_t rows, int cols) { return up256(rows * (padded(cols) / 2)); }
static int64_t row_scales(int64_t rows, int cols) { return up256(rows * padded_blocks(cols)); }
static bool aligned16(const void* a) { return ((uintptr_t)a & 15) == 0; }

template <typename T>
static void launch_quant(const void* x, int64_t rows, int cols, int out_cols, uint8_t* q, uint8_t* scale, hipStream_t stream) {
  const int64_t chunks = rows * (out_cols / 8);
  int64_t g = (chunks + 1023) / 1024;
  if (g > 16384) g = 16384;
  hipLaunchKernelGGL(quant_kernel<T>, dim3((unsigned)g), dim3(256), 0, stream, (const T*)x, chunks, cols / 8, out_cols / 8,
                     (uint32_t*)q, scale);
}

}  // namespace mxfp4
}  // namespace moe

using namespace moe;
using namespace moe::mxfp4;

MOE_API int moe_mxfp4_padded_cols(int32_t cols) {
  return cols < kBlock || cols % kBlock || cols > (1 << 30) ? kErrInvalidArgument : padded(cols);
}

static int check_rows(const void* x, int64_t rows, int32_t cols, int32_t q_cols, int32_t dtype, const void* q, const void* scale) {
  if (rows < 0 || cols < kBlock || cols % kBlock || q_cols < cols || q_cols % kBlock || (dtype != 0 && dtype != 1))
    return kErrInvalidArgument;
  if (rows && (!x || !q || !scale || !aligned16(x) || !aligned16(q))) return kErrInvalidArgument;
  return kOk;
}

MOE_API int moe_mxfp4_quant_rows(const void* x, int64_t rows, int32_t cols, int32_t q_cols, int32_t dtype, uint8_t* q,
                                 uint8_t* scale, hipStream_t stream) {
  const int st = check_rows(x, rows, cols, q_cols, dtype, q, scale);
  if (st || rows == 0) return st;
  if (dtype == 0) launch_quant<uint16_t>(x, rows, cols, q_cols, q, scale, stream);
  else launch_quant<float>(x, rows, cols, q_cols, q, scale, stream);
  return launch_status();
}

MOE_API int moe_mxfp4_dequant_rows(const uint8_t* q, const uint8_t* scale, int64_t rows, int32_t cols, int32_t q_cols,
                                   int32_t dtype, void* x, hipStream_t stream) {
  const int st = check_rows(x, rows, cols, q_cols, dtype, q, scale);
  if (st || rows == 0) return st;
  const int64_t chunks = rows * (cols / 8);
  int64_t g = (chunks + 255) / 256;
  if (g > 16384) g = 16384;
  if (dtype == 0)
    hipLaunchKernelGGL(dequant_kernel<uint16_t>, dim3((unsigned)g), dim3(256), 0, stream, (const uint32_t*)q, scale, chunks,
                       cols / 8, q_cols / 8, (uint16_t*)x);
  else
    hipLaunchKernelGGL(dequant_kernel<float>, dim3((unsigned)g), dim3(256), 0, stream, (const uint32_t*)q, scale, chunks,
                       cols / 8, q_cols / 8, (float*)x);
  return launch_status();
}

// bytes of scales of the weights' rows that take a padded copy: odd rows, for the wide kernel
static int64_t odd_scales(int64_t rows, int cols) { return cols / kBlock % 2 ? up256(rows * padded_blocks(cols)) : 0; }

// workspace of the experts' forward: x in MXFP4 with its scales, h with its scales, and padded
// copies of odd scale rows
MOE_API int64_t moe_mxfp4_workspace_bytes(int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden) {
  if (n_rows < 0 || n_experts < 1 || dim < kBlock || hidden < kBlock || dim % kBlock || hidden % kBlock)
    return kErrInvalidArgument;
  const int64_t rows = row_bytes(n_rows, dim) + row_scales(n_rows, dim) + row_bytes(n_rows, hidden) + row_scales(n_rows, hidden);
  return rows + (takes_narrow(n_rows, n_experts, dim, hidden)
                     ? 0 : odd_scales(2 * (int64_t)n_experts * hidden, dim) + odd_scales((int64_t)n_experts * dim, hidden));
}

namespace moe {
namespace mxfp4 {
template <int ACT>
static int experts_fwd(const uint16_t* x, const uint8_t* qw1, const uint8_t* sw1, const uint8_t* qw2, const uint8_t* sw2,
                       const uint8_t* qw3, const uint8_t* sw3, const uint16_t* b1, const uint16_t* b2, float limit,
                       const int64_t* counts, int64_t R, int E, int D, int H, uint8_t* ws, int64_t ws_bytes, uint16_t* y,
                       hipStream_t stream) {
  const int st = check_shape(R, E, D, H);
  if (st) return st;
  if (!counts) return kErrInvalidArgument;
  if (R == 0) return kOk;
  if (!x || !qw1 || !sw1 || !qw2 || !sw2 || !qw3 || !sw3 || !ws || !y) return kErrInvalidArgument;
  for (const void* q : {(const void*)x, (const void*)qw1, (const void*)qw2, (const void*)qw3, (const void*)sw1,
                        (const void*)sw2, (const void*)ws, (const void*)y, (const void*)b1, (const void*)b2})
    if (!aligned16(q)) return kErrInvalidArgument;
  if (ws_bytes < moe_mxfp4_workspace_bytes(R, E, D, H)) return kErrWorkspace;
  uint8_t* qx = ws;
  uint8_t* sx = qx + row_bytes(R, D);
  uint8_t* qh = sx + row_scales(R, D);
  uint8_t* sh = qh + row_bytes(R, H);
  uint8_t* pads = sh + row_scales(R, H);
  const bool oss = ACT == kOssGLU;
  const bool narrow = takes_narrow(R, E, D, H);
  // odd scale rows, padded for the wide kernel: the copy, and its row stride
  auto pad_scales = [&](const uint8_t* src, int64_t rows, int cols, int& ld) {
    ld = cols / kBlock;
    if (narrow || ld % 2 == 0) return src;
    ld = padded_blocks(cols);
    int64_t g = (rows * (ld / 8) + 255) / 256;
    if (g > 16384) g = 16384;
    hipLaunchKernelGGL(pad_scales_kernel, dim3((unsigned)g), dim3(256), 0, stream, src, rows, cols / kBlock, ld, pads);
    const uint8_t* got = pads;
    pads += rows * ld;
    return got;
  };
  Params p{};
  p.counts = counts; p.R = R; p.E = E; p.K = D; p.N = H;
  p.x = x; p.qp = qx; p.sp = sx;
  p.qa = qw1; p.qb = qw3;
  if (oss) {
    p.sa = pad_scales(sw1, 2 * (int64_t)E * H, D, p.w_ld);
    p.sb = p.sa + p.w_ld;
  } else {
    p.sa = pad_scales(sw1, (int64_t)E * H, D, p.w_ld);
    p.sb = pad_scales(sw3, (int64_t)E * H, D, p.w_ld);
  }
  pads = ws + up256(pads - ws);
  p.e_rows = oss ? 2 * (int64_t)H : H;
  p.r_rows = oss ? 2 : 1;
  p.bias = b1; p.limit = limit;
  p.qh = qh; p.sh = sh;
  if (narrow) {
    launch_narrow<kGateUp, ACT>(p, stream);
  } else {
    launch_quant<uint16_t>(x, R, D, padded(D), qx, sx, stream);
    launch_wide<kGateUp, ACT, false>(p, stream);
  }
  p.K = H; p.N = D;
  p.qp = qh; p.sp = sh;
  p.qa = qw2; p.sa = pad_scales(sw2, (int64_t)E * D, H, p.w_ld); p.e_rows = D; p.r_rows = 1;
  p.bias = b2; p.y = y;
  if (narrow) launch_narrow<kDown, ACT>(p, stream);
  else launch_wide<kDown, ACT, false>(p, stream);
  return launch_status();
}
}  // namespace mxfp4
}  // namespace moe

MOE_API int moe_mxfp4_swiglu_fwd(const uint16_t* x, const uint8_t* qw1, const uint8_t* sw1, const uint8_t* qw2,
                                 const uint8_t* sw2, const uint8_t* qw3, const uint8_t* sw3, const int64_t* counts,
                                 int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden, uint8_t* workspace,
                                 int64_t workspace_bytes, uint16_t* y, hipStream_t stream) {
  if (sw3 && !aligned16(sw3)) return kErrInvalidArgument;
  return experts_fwd<kSwiGLU>(x, qw1, sw1, qw2, sw2, qw3, sw3, nullptr, nullptr, 0.f, counts, n_rows, n_experts, dim,
                              hidden, workspace, workspace_bytes, y, stream);
}

MOE_API int moe_mxfp4_oss_fwd(const uint16_t* x, const uint8_t* qmlp1, const uint8_t* smlp1, const uint16_t* mlp1_bias,
                              const uint8_t* qmlp2, const uint8_t* smlp2, const uint16_t* mlp2_bias,
                              const int64_t* counts, int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden,
                              float swiglu_limit, uint8_t* workspace, int64_t workspace_bytes, uint16_t* y,
                              hipStream_t stream) {
  if (n_rows > 0 && (!qmlp1 || !smlp1 || !mlp1_bias || !mlp2_bias)) return kErrInvalidArgument;
  if (dim < kBlock || dim % kBlock) return kErrInvalidArgument;
  return experts_fwd<kOssGLU>(x, qmlp1, smlp1, qmlp2, smlp2, qmlp1 ? qmlp1 + dim / 2 : nullptr,
                              smlp1 ? smlp1 + dim / kBlock : nullptr, mlp1_bias, mlp2_bias, swiglu_limit, counts,
                              n_rows, n_experts, dim, hidden, workspace, workspace_bytes, y, stream);
}

// The training step's forward products, one at a time.
MOE_API int moe_mxfp4_gemm_gate_up_keep(const uint8_t* qx, const uint8_t* sx, const uint8_t* qw1, const uint8_t* sw1,
                                        const uint8_t* qw3, const uint8_t* sw3, const int64_t* counts, int64_t n_rows,
                                        int32_t n_experts, int32_t dim, int32_t hidden, uint8_t* qh, uint8_t* sh,
                                        uint8_t* g8, uint8_t* gs, uint8_t* u8, uint8_t* us, hipStream_t stream) {
  const int st = check_shape(n_rows, n_experts, dim, hidden);
  if (st) return st;
  if (dim / kBlock % 2) return kErrUnsupportedShape;
  if (!counts) return kErrInvalidArgument;
  if (n_rows == 0) return kOk;
  if (!qx || !sx || !qw1 || !sw1 || !qw3 || !sw3 || !qh || !sh || !g8 || !gs || !u8 || !us) return kErrInvalidArgument;
  for (const void* q : {(const void*)qx, (const void*)sx, (const void*)qw1, (const void*)qw3, (const void*)sw1,
                        (const void*)sw3, (const void*)qh, (const void*)g8, (const void*)u8})
    if (!aligned16(q)) return kErrInvalidArgument;
  Params p{};
  p.counts = counts; p.R = n_rows; p.E = n_experts; p.K = dim; p.N = hidden;
  p.qp = qx; p.sp = sx;
  p.qa = qw1; p.sa = sw1; p.qb = qw3; p.sb = sw3; p.e_rows = hidden; p.r_rows = 1; p.w_ld = dim / kBlock;
  p.qh = qh; p.sh = sh;
  p.g8 = g8; p.gs = gs; p.u8 = u8; p.us = us;
  launch_wide<kGateUp, kSwiGLU, true>(p, stream);
  return launch_status();
}

MOE_API int moe_mxfp4_gemm_down(const uint8_t* qh, const uint8_t* sh, const uint8_t* qw2, const uint8_t* sw2,
                                const int64_t* counts, int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden,
                                uint16_t* y, hipStream_t stream) {
  const int st = check_shape(n_rows, n_experts, dim, hidden);
  if (st) return st;
  if (hidden / kBlock % 2) return kErrUnsupportedShape;
  if (!counts) return kErrInvalidArgument;
  if (n_rows == 0) return kOk;
  if (!qh || !sh || !qw2 || !sw2 || !y) return kErrInvalidArgument;
  for (const void* q : {(const void*)qh, (const void*)sh, (const void*)qw2, (const void*)sw2, (const void*)y})
    if (!aligned16(q)) return kErrInvalidArgument;
  Params p{};
  p.counts = counts; p.R = n_rows; p.E = n_experts; p.K = hidden; p.N = dim;
  p.qp = qh; p.sp = sh;
  p.qa = qw2; p.sa = sw2; p.qb = qw2; p.sb = sw2; p.e_rows = dim; p.r_rows = 1; p.w_ld = hidden / kBlock;
  p.y = y;
  launch_wide<kDown, kSwiGLU, false>(p, stream);
  return launch_status();
}
