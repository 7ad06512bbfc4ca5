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
#include <type_traits>

#include "mx.h"

namespace moe {
namespace mxfp4 {

using mx::kBlock;

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kMaxE = 1024;

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

// x as n_chunks chunks of eight elements; chunk c's codes are the word q[c], its block's scale
// scale[c / 4], or, with rows of cpr chunks whose scales lie s_ld apart (s_ld > 0), in their row.
template <typename T>
__global__ __launch_bounds__(256) void quant_kernel(const T* __restrict__ x, int64_t n_chunks, int cpr, int s_ld,
                                                    uint32_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const int64_t S = (int64_t)gridDim.x * 256;
  for (int64_t c0 = (int64_t)blockIdx.x * 256 + threadIdx.x; c0 - threadIdx.x < n_chunks; c0 += 4 * S) {
    Eight<T> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * S;
      if (c < n_chunks) v[u].load(x + 8 * c);
      else v[u].zero();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * S;
      uint32_t w;
      const uint32_t s = quad_block4(v[u], w);
      if (c < n_chunks) {
        q[c] = w;
        if ((c & 3) == 0) {
          int64_t at = c >> 2;
          if (s_ld) {
            const int64_t r = c / cpr;
            at = r * s_ld + ((c - r * cpr) >> 2);
          }
          scale[at] = (uint8_t)s;
        }
      }
    }
  }
}

// codes back to values: chunk c's eight elements from the word q[c] and its block's scale, which
// lies as in quant_kernel
template <typename T>
__global__ __launch_bounds__(256) void dequant_kernel(const uint32_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                      int64_t n_chunks, int cpr, int s_ld, T* __restrict__ x) {
  const int64_t S = (int64_t)gridDim.x * 256;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < n_chunks; c += S) {
    const uint32_t w = q[c];
    int64_t at = c >> 2;
    if (s_ld) {
      const int64_t r = c / cpr;
      at = r * s_ld + ((c - r * cpr) >> 2);
    }
    const float s = mx::scale_value(scale[at]);
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
  const uint8_t* qp;      // else rows [R, K / 2], their scales [R, p_ld], p_ld a multiple of 8
  const uint8_t* sp;
  int p_ld;
  const uint8_t* qa;      // weights: gate rows, or down's
  const uint8_t* sa;
  const uint8_t* qb;      // up rows
  const uint8_t* sb;
  int64_t e_rows;         // row n of expert e is row e * e_rows + n * r_rows of qa and qb
  int r_rows;
  const uint16_t* bias;   // gpt-oss: b1 [E, 2H] (glu 2j, linear 2j + 1), b2 [E, D]
  float limit;
  uint8_t* qh;            // gate_up: h [R, H / 2], its scales [R, h_ld]
  uint8_t* sh;
  int h_ld;
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

#define LDSP __attribute__((address_space(3)))
// One wave-wide direct-to-LDS copy: lane i's 16 bytes at g land at LDS byte address
// lds + 16 i; waited for with vmcnt.
__device__ __forceinline__ void dma16(const void* g, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, off" :: "v"(g), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const uint8_t* ptr) { return (uint32_t)(size_t)((LDSP const uint8_t*)ptr); }

// Row-major LDS tile of 128-byte rows (256 k): byte offset of 16-byte chunk c of row r;
// conflict-free where eight lanes read one chunk of eight rows.
__device__ __forceinline__ int rm_off(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }

__device__ const uint4 kZeroRow[8] = {};  // source of rows and k past an edge
constexpr uint32_t kUnitScales = 0x7f7f7f7fu;

// Exclusive prefix sums of up to 1024 non-negative ints, four per thread of the first 256,
// that stop at `most` (saturating sums are associative, and with most < 2^30 no step passes
// 2^31 whatever the values). Returns the total. Called by every thread; tmp: one int per wave.
__device__ __forceinline__ int saturating_scan4(const int (&v)[4], int (&out)[4], int* tmp, int most) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = blockDim.x >> 6;
  auto add = [&](int a, int b) { return min(a + b, most); };
  const int local = add(add(min(v[0], most), min(v[1], most)), add(min(v[2], most), min(v[3], most)));
  int incl = local;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off);
    if (lane >= off) incl = add(incl, o);
  }
  if (lane == 63) tmp[wv] = incl;
  __syncthreads();
  int run = 0, total = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < wv) run = add(run, tmp[w]);
    total = add(total, tmp[w]);
  }
  __syncthreads();
  const int before = __shfl_up(incl, 1);
  if (lane) run = add(run, before);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i] = run;
    run = add(run, min(v[i], most));
  }
  return total;
}

// Expert e's rows [seg[e], seg[e + 1]), clamped to R, and the exclusive sums of
// tiles_of(rows) in `tile`, both of E + 1 ints in LDS. Called by every thread of a workgroup of
// at least 256; negative counts count as none.
template <typename F>
__device__ __forceinline__ void segments(const Params& p, int* seg, int* tile, int* tmp, F tiles_of) {
  const int tid = threadIdx.x, R = (int)p.R;
  int cnt[4], sg[4], tl[4], ts[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    const int64_t c = e < p.E ? p.counts[e] : 0;
    cnt[i] = c < 0 ? 0 : (c > p.R ? R : (int)c);
  }
  const int rows = saturating_scan4(cnt, sg, tmp, R);
#pragma unroll
  for (int i = 0; i < 4; ++i) tl[i] = tid * 4 + i < p.E ? tiles_of(min(cnt[i], R - sg[i])) : 0;
  const int tiles = saturating_scan4(tl, ts, tmp, 0x3fffffff);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    if (e < p.E) { seg[e] = sg[i]; tile[e] = ts[i]; }
  }
  if (tid == 0) { seg[p.E] = rows; tile[p.E] = tiles; }
  __syncthreads();
}
__device__ __forceinline__ int find(const int* start, int E, int t) {  // the last e with start[e] <= t
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
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
  if (valid) {
    *(uint32_t*)(p.qh + r * (p.N / 2) + hc / 2 + 4 * g4) = q;
    if (g4 == 0) p.sh[r * p.h_ld + hc / kBlock] = (uint8_t)s;
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

// Eight scale bytes of which `left` belong to the row (the others: 1.0).
__device__ __forceinline__ uint2 masked_scales(uint2 v, int left) {
  if (left >= 8) return v;
  const uint64_t keep = (1ull << (8 * left)) - 1, unit = 0x7f7f7f7f7f7f7f7full;
  const uint64_t m = ((((uint64_t)v.y << 32) | v.x) & keep) | (unit & ~keep);
  return make_uint2((uint32_t)m, (uint32_t)(m >> 32));
}

// Many rows per expert: 256 x 256 outputs of eight 64 x 128 wave tiles, k in stages of 256 (128
// bytes a row, as 128 k of 8-bit operands), two stages in LDS, persistent workgroups. The
// operands reach LDS by direct-to-LDS copies, issued one stage ahead across tile boundaries;
// the scales (8 bytes a row and stage) through registers, since a row of K / 32 scale bytes has
// any alignment. MFMA step s of a stage takes chunk 2 q + s of a row in lane row q, so that a
// lane's two scales are one 16-bit read. gate_up's columns alternate in blocks of 16 between
// gate and up, so that a lane holds both.
template <int MODE, int ACT, bool KEEP>
__global__ __launch_bounds__(512, 1) void wide_kernel(Params p) {
  constexpr int TM = 4, TN = 8, WGN = 2, BM = 256, BN = 256, CPW = 4;
  __shared__ __attribute__((aligned(1024))) uint8_t sP[2][BM * 128];
  __shared__ __attribute__((aligned(1024))) uint8_t sQ[2][BN * 128];
  __shared__ __attribute__((aligned(16))) uint2 sS[2][BM + BN];
  __shared__ int s_seg[kMaxE + 1];
  __shared__ int s_tile[kMaxE + 1];
  __shared__ int s_tmp[8];

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv / WGN, wn = wv % WGN, ml = lane & 15, g4 = lane >> 4;
  const int E = p.E, K = p.K, N = p.N, KB = K / kBlock, kbytes = K / 2;
  const int NT = MODE == kGateUp ? (N + BN / 2 - 1) / (BN / 2) : (N + BN - 1) / BN;
  const int nk = (K + 255) / 256;
  segments(p, s_seg, s_tile, s_tmp, [&](int rows) { return (rows + BM - 1) / BM * NT; });
  const int total_tiles = s_tile[E], G = gridDim.x;
  // each XCD works on a contiguous window of tiles
  const int lb = G % 8 == 0 ? (int)(blockIdx.x & 7) * (G >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;

  struct TileRef { int e, seg0, seg1, mt, nt; };
  auto decode = [&](int t) {
    TileRef r;
    r.e = find(s_tile, E, t);
    const int local = t - s_tile[r.e];
    r.seg0 = s_seg[r.e];
    r.seg1 = s_seg[r.e + 1];
    const int mtiles = (r.seg1 - r.seg0 + BM - 1) / BM;
    r.nt = local / mtiles;
    r.mt = local - r.nt * mtiles;
    return r;
  };
  // row n of the tile's weight columns: its tensor, row number, and whether it is inside
  auto weight_row = [&](const TileRef& r, int n, bool& up, bool& in) -> int64_t {
    int col;
    if (MODE == kGateUp) {
      const int blk = n >> 4;
      col = r.nt * (BN / 2) + (blk >> 1) * 16 + (n & 15);
      up = blk & 1;
    } else {
      col = r.nt * BN + n;
      up = false;
    }
    in = col < N;
    return r.e * p.e_rows + (int64_t)col * p.r_rows;
  };

  // ---- sources of the tile being copied: copy b of this wave fills rows 8 (4 wv + b) .. + 7,
  // lane i row i / 8, chunk i % 8 with the row's chunk (i % 8) ^ ((row >> 1) & 7) ----
  const int crow = lane >> 3;
  const uint8_t* srcP[CPW];
  const uint8_t* srcQ[CPW];
  int ch[CPW];
  bool okP[CPW], okQ[CPW];
#pragma unroll
  for (int b = 0; b < CPW; ++b) ch[b] = (lane & 7) ^ ((((wv * CPW + b) * 8 + crow) >> 1) & 7);
  const uint8_t* srcS = nullptr;  // this thread's row of scales: tid < 256 P row tid, else Q row tid - 256
  bool okS = false;
  auto setup = [&](const TileRef& r) {
    const int row0 = r.seg0 + r.mt * BM;
#pragma unroll
    for (int b = 0; b < CPW; ++b) {
      const int m = (wv * CPW + b) * 8 + crow;
      okP[b] = row0 + m < r.seg1;
      srcP[b] = p.qp + (int64_t)(row0 + m) * kbytes + ch[b] * 16;
      bool up;
      const int64_t wr = weight_row(r, m, up, okQ[b]);
      srcQ[b] = (up ? p.qb : p.qa) + wr * kbytes + ch[b] * 16;
    }
    if (tid < BM) {
      okS = row0 + tid < r.seg1;
      srcS = p.sp + (int64_t)(row0 + tid) * p.p_ld;
    } else {
      bool up;
      const int64_t wr = weight_row(r, tid - BM, up, okS);
      srcS = (up ? p.sb : p.sa) + wr * KB;
    }
  };
  const bool p_side = tid < BM;
  uint2 scales;  // of the stage in flight
  auto issue = [&](int kt, int s) {
#pragma unroll
    for (int b = 0; b < CPW; ++b) {
      const bool in = kt * 8 + ch[b] < KB;
      dma16(okP[b] && in ? (const void*)(srcP[b] + kt * 128) : (const void*)kZeroRow, lds_addr(&sP[s][(wv * CPW + b) * 1024]));
    }
#pragma unroll
    for (int b = 0; b < CPW; ++b) {
      const bool in = kt * 8 + ch[b] < KB;
      dma16(okQ[b] && in ? (const void*)(srcQ[b] + kt * 128) : (const void*)kZeroRow, lds_addr(&sQ[s][(wv * CPW + b) * 1024]));
    }
    const int left = KB - kt * 8;  // scale bytes of this stage and after it
    uint32_t w0 = kUnitScales, w1 = kUnitScales;
    if (okS) {
      const uint8_t* src = srcS + kt * 8;
      if (p_side || KB % 8 == 0) {
        const uint2 v = masked_scales(*(const uint2*)src, left);  // rows of P's scales are padded to whole words
        w0 = v.x;
        w1 = v.y;
      } else if (KB % 2 == 0) {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = 2 * i < left ? *(const uint16_t*)(src + 2 * i) : 0x7f7fu;
        w0 = h[0] | (h[1] << 16);
        w1 = h[2] | (h[3] << 16);
      } else {
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = i < left ? src[i] : 0x7fu;
        w0 = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
        w1 = c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24);
      }
    }
    scales = make_uint2(w0, w1);
  };
  int ct = lb, ik = 0, gi = 0, gc = 0;  // copy cursor: tile ct, its stage ik; stage gi goes to buffer gi % 2
  auto seek = [&](int t) {
    ct = t;
    ik = 0;
    if (ct < total_tiles) setup(decode(ct));
  };
  auto issue_next = [&]() {
    issue(ik, gi & 1);
    ++gi;
    if (++ik == nk) seek(ct + G);
  };
  seek(lb);
  if (ct < total_tiles) issue_next();

  for (int t = lb; t < total_tiles; t += G) {
    const TileRef cur = decode(t);
    const int row0 = cur.seg0 + cur.mt * BM, seg1 = cur.seg1;
    f32x4_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    for (int kt = 0; kt < nk; ++kt) {
      // this stage's copies and scales have landed; its scales go to LDS (the buffer's last
      // readers are two stages back); the barrier also retires every read of the buffer
      // that is filled next
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      sS[gc & 1][tid] = scales;
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (ct < total_tiles) issue_next();
      __builtin_amdgcn_sched_barrier(0);
      const int sl = gc & 1;
      ++gc;
      int scp[TM], scq[TN];
      const uint8_t* ss = (const uint8_t*)sS[sl];
#pragma unroll
      for (int i = 0; i < TM; ++i) scp[i] = *(const uint16_t*)(ss + (wm * 64 + i * 16 + ml) * 8 + 2 * g4);
#pragma unroll
      for (int j = 0; j < TN; ++j) scq[j] = *(const uint16_t*)(ss + (BM + wn * 128 + j * 16 + ml) * 8 + 2 * g4);
      auto frag = [&](const uint8_t* tile, int row, int s) {
        const uint4 v = *(const uint4*)(tile + rm_off(row, 2 * g4 + s));
        return v8i_t{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
      };
      auto step = [&](auto s_c) {
        constexpr int s = decltype(s_c)::value;
        v8i_t af[TM], bq[2];
#pragma unroll
        for (int i = 0; i < TM; ++i) af[i] = frag(sP[sl], wm * 64 + i * 16 + ml, s);
        bq[0] = frag(sQ[sl], wn * 128 + ml, s);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if (j + 1 < TN) bq[(j + 1) & 1] = frag(sQ[sl], wn * 128 + (j + 1) * 16 + ml, s);
#pragma unroll
          for (int i = 0; i < TM; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bq[j & 1], af[i], acc[i][j], 4, 4, s, scq[j],
                                                                         s, scp[i]);
        }
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
    }

    // ---- epilogue: lane holds C[m = .. + ml][n = .. + 4 g4 .. + 3] of each 16-column block ----
    if (MODE == kGateUp) {
#pragma unroll
      for (int b = 0; b < TN / 4; ++b) {
        const int hc = cur.nt * (BN / 2) + wn * 64 + b * 32;
        if (hc >= N) continue;
        uint4 bias_a{}, bias_b{};
        if constexpr (ACT == kOssGLU) {
          const uint16_t* bp = p.bias + (int64_t)cur.e * 2 * N + 2 * (hc + 4 * g4);
          bias_a = *(const uint4*)bp;
          bias_b = *(const uint4*)(bp + 32);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = row0 + wm * 64 + i * 16 + ml;
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
        const int n0 = cur.nt * BN + wn * 128 + b * 32;
        if (n0 >= N) continue;
        float ba[4] = {0.f, 0.f, 0.f, 0.f}, bb[4] = {0.f, 0.f, 0.f, 0.f};
        if constexpr (ACT == kOssGLU) {
          const uint16_t* bp = p.bias + (int64_t)cur.e * N + n0 + 4 * g4;
          unpack4(*(const uint2*)bp, ba);
          unpack4(*(const uint2*)(bp + 16), bb);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = row0 + wm * 64 + i * 16 + ml;
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
  if (MODE == kDown) zero_rest(p, s_seg[E]);
}

// Few rows per expert: the weights are read once and decide the time, so every byte goes
// straight from memory into the MFMAs' registers. A unit is 64 weight rows (gate_up: 32 gate and
// 32 up rows, one scaling block of h; down: 64 columns) by up to 16 TM rows of one expert;
// eight waves take four blocks of 16 weight rows by the even and the odd 256-k stages. A wave
// keeps two groups of kAhead stages in registers, the next group's loads in flight while
// this group multiplies, through to the following unit. A workgroup's units are consecutive,
// so the rows, which gate_up quantizes from bf16 on the way into LDS, are prepared once per
// expert and workgroup.
constexpr int kAhead = 4;
__host__ __device__ constexpr int narrow_stride(int K) { return (K + 255) / 256 * 128 + 16; }  // rows 16 bytes apart mod 128
__host__ __device__ constexpr int64_t narrow_lds(int K, int TM) {
  return (int64_t)TM * 16 * (narrow_stride(K) + (K + 255) / 256 * 8) + (int64_t)TM * 8 * 64 * 16;
}

template <int MODE, int ACT, int TM>
__global__ __launch_bounds__(512, 2) void narrow_kernel(Params p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_dyn[];
  __shared__ int s_seg[kMaxE + 1];
  __shared__ int s_tile[kMaxE + 1];
  __shared__ int s_tmp[8];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = wv & 3, ks = wv >> 2, ml = lane & 15, g4 = lane >> 4;
  const int E = p.E, K = p.K, N = p.N, KB = K / kBlock, kbytes = K / 2, nst = (K + 255) / 256;
  const int stride = narrow_stride(K), sld = nst * 8;
  uint8_t* sP = s_dyn;
  f32x4_t* red = (f32x4_t*)(s_dyn + TM * 16 * (stride + sld));  // [2 ks][4 nb][TM][64]
  uint8_t* sc = s_dyn + TM * 16 * stride;
  const int NCB = MODE == kGateUp ? N / 32 : (N + 63) / 64;
  segments(p, s_seg, s_tile, s_tmp, [&](int rows) { return (rows + 16 * TM - 1) / (16 * TM) * NCB; });
  const int64_t total = s_tile[E];
  const int u0 = (int)(total * blockIdx.x / gridDim.x), u1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
  const int mine = (nst - ks + 1) / 2;  // this wave's stages: ks, ks + 2, ...

  struct Group { uint4 w[kAhead][2]; uint32_t s[kAhead]; };
  struct Unit { int e, rt, cb; };
  auto decode = [&](int u) {
    Unit r;
    r.e = find(s_tile, E, u);
    const int local = u - s_tile[r.e];
    r.rt = local / NCB;
    r.cb = local - r.rt * NCB;
    return r;
  };
  auto load = [&](Group& g, const Unit& u, int base) {
    const int col = MODE == kGateUp ? u.cb * 32 + (nb & 1) * 16 + ml : u.cb * 64 + nb * 16 + ml;
    const bool up = MODE == kGateUp && nb >= 2, in = col < N;
    const int64_t row = u.e * p.e_rows + (int64_t)col * p.r_rows;
    const uint8_t* wq = (up ? p.qb : p.qa) + row * kbytes;
    const uint8_t* ws = (up ? p.sb : p.sa) + row * KB;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = 8 * (ks + 2 * (base + i)) + 2 * g4;  // this lane's first chunk of 32 k
      g.w[i][0] = *(const uint4*)(in && c < KB ? wq + c * 16 : (const uint8_t*)kZeroRow);
      g.w[i][1] = *(const uint4*)(in && c + 1 < KB ? wq + c * 16 + 16 : (const uint8_t*)kZeroRow);
      if (KB % 2 == 0) {
        g.s[i] = in && c < KB ? *(const uint16_t*)(ws + c) : 0x7f7fu;
      } else {
        const uint32_t lo = in && c < KB ? ws[c] : 0x7fu, hi = in && c + 1 < KB ? ws[c + 1] : 0x7fu;
        g.s[i] = lo | (hi << 8);
      }
    }
  };
  auto fill = [&](int row0, int rows) {
    if (MODE == kGateUp) {
      const int cpr = K / 8, n = rows * cpr;
      for (int c0 = tid; c0 - tid < n; c0 += 4 * 512) {
        Eight<uint16_t> v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = c0 + 512 * k;
          if (c < n) v[k].load(p.x + (int64_t)row0 * K + (int64_t)c * 8);
          else v[k].zero();
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = c0 + 512 * k;
          uint32_t w;
          const uint32_t s = quad_block4(v[k], w);
          if (c < n) {
            const int r = c / cpr, at = c - r * cpr;
            *(uint32_t*)(sP + r * stride + at * 4) = w;
            if ((at & 3) == 0) sc[r * sld + (at >> 2)] = (uint8_t)s;
          }
        }
      }
      for (int i = tid; i < rows * (sld - KB); i += 512) sc[i / (sld - KB) * sld + KB + i % (sld - KB)] = 0x7f;
    } else {
      for (int i = tid; i < rows * KB; i += 512) {
        const int r = i / KB, c = i - r * KB;
        *(uint4*)(sP + r * stride + c * 16) = *(const uint4*)(p.qp + (int64_t)(row0 + r) * kbytes + c * 16);
      }
      for (int i = tid; i < rows * nst; i += 512) {
        const int r = i / nst, st = i - r * nst;
        *(uint2*)(sc + r * sld + st * 8) =
            masked_scales(*(const uint2*)(p.sp + (int64_t)(row0 + r) * p.p_ld + st * 8), KB - st * 8);
      }
    }
  };

  Group cur, nxt;
  Unit u{};
  if (u0 < u1) {
    u = decode(u0);
    load(cur, u, 0);
  }
  int have_e = -1, have_rt = -1;
  for (int t = u0; t < u1; ++t) {
    const int row0 = s_seg[u.e] + u.rt * 16 * TM, rows = min(16 * TM, s_seg[u.e + 1] - row0);
    if (u.e != have_e || u.rt != have_rt) {
      __syncthreads();  // every wave is done with the rows before
      fill(row0, rows);
      __syncthreads();
      have_e = u.e;
      have_rt = u.rt;
    }
    const Unit un = t + 1 < u1 ? decode(t + 1) : u;
    f32x4_t acc[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int base = 0; base < mine; base += kAhead) {
      if (base + kAhead < mine) load(nxt, u, base + kAhead);
      else if (t + 1 < u1) load(nxt, un, 0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int st = ks + 2 * (base + i);
        if (st < nst) {
#pragma unroll
          for (int m = 0; m < TM; ++m) {
            const int row = m * 16 + ml;
            const uint32_t sp = *(const uint16_t*)(sc + row * sld + st * 8 + 2 * g4);
            const uint4 a0 = *(const uint4*)(sP + row * stride + st * 128 + g4 * 32);
            const uint4 a1 = *(const uint4*)(sP + row * stride + st * 128 + g4 * 32 + 16);
            const uint4 b0 = cur.w[i][0], b1 = cur.w[i][1];
            acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                v8i_t{(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, 0, 0, 0, 0},
                v8i_t{(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, 0, 0, 0, 0}, acc[m], 4, 4, 0, (int)cur.s[i], 0, (int)sp);
            acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                v8i_t{(int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w, 0, 0, 0, 0},
                v8i_t{(int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w, 0, 0, 0, 0}, acc[m], 4, 4, 1, (int)cur.s[i], 1, (int)sp);
          }
        }
      }
      cur = nxt;
    }
    if (mine == 0 && t + 1 < u1) load(cur, un, 0);
    __syncthreads();  // the sums of the unit before have been read
#pragma unroll
    for (int m = 0; m < TM; ++m) red[((ks * 4 + nb) * TM + m) * 64 + lane] = acc[m];
    __syncthreads();
    auto sum = [&](int b, int m, float (&v)[4]) {
      const f32x4_t a = red[(b * TM + m) * 64 + lane], c = red[((4 + b) * TM + m) * 64 + lane];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = a[q] + c[q];
    };
    if (MODE == kGateUp) {
      if (wv < TM) {
        float ga[4], gb[4], ua[4], ub[4];
        sum(0, wv, ga);
        sum(1, wv, gb);
        sum(2, wv, ua);
        sum(3, wv, ub);
        const int hc = u.cb * 32, r = wv * 16 + ml;
        uint4 bias_a{}, bias_b{};
        if constexpr (ACT == kOssGLU) {
          const uint16_t* bp = p.bias + (int64_t)u.e * 2 * N + 2 * (hc + 4 * g4);
          bias_a = *(const uint4*)bp;
          bias_b = *(const uint4*)(bp + 32);
        }
        store_hidden<ACT, false>(p, row0 + r, hc, lane, r < rows, ga, gb, ua, ub, bias_a, bias_b);
      }
    } else if (wv < 2 * TM) {
      const int m = wv >> 1, pr = wv & 1, n0 = u.cb * 64 + pr * 32, r = m * 16 + ml;
      if (n0 < N) {
        float lo[4], hi[4];
        sum(2 * pr, m, lo);
        sum(2 * pr + 1, m, hi);
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
    u = un;
  }
  if (MODE == kDown) zero_rest(p, s_seg[E]);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int g_cus[64];
static int cu_count() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!g_cus[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    g_cus[dev] = n;
  }
  return g_cus[dev];
}

constexpr int kLdsMost = 144 * 1024;  // dynamic LDS of the narrow kernel (160 KB less its static part)

template <int MODE, int ACT, bool KEEP>
static void launch_wide(const Params& p, hipStream_t stream) {
  const int64_t nt = MODE == kGateUp ? (p.N + 127) / 128 : (p.N + 255) / 256;
  int64_t g = (p.R / 256 + p.E) * nt, cus = cu_count();
  if (g > cus) g = cus;
  if (g >= 8) g -= g % 8;
  hipLaunchKernelGGL((wide_kernel<MODE, ACT, KEEP>), dim3((unsigned)g), dim3(512), 0, stream, p);
}
template <int MODE, int ACT, int TM>
static void launch_narrow_tm(const Params& p, hipStream_t stream) {
  const int64_t ncb = MODE == kGateUp ? p.N / 32 : (p.N + 63) / 64;
  int64_t g = (p.R / (16 * TM) + (p.R < p.E ? p.R : p.E)) * ncb;
  const int64_t most = cu_count();
  if (g > most) g = most;
  if (narrow_lds(p.K, TM) > 64 * 1024)
    (void)hipFuncSetAttribute((const void*)narrow_kernel<MODE, ACT, TM>, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsMost);
  hipLaunchKernelGGL((narrow_kernel<MODE, ACT, TM>), dim3((unsigned)g), dim3(512), (unsigned)narrow_lds(p.K, TM), stream, p);
}
// rows an expert with rows has on average decide the row blocks a unit holds
static int narrow_rows(int64_t R, int64_t E, int K) {
  const int64_t used = R < E ? R : E, avg = (R + used - 1) / used;
  int tm = avg <= 8 ? 1 : avg <= 24 ? 2 : 4;
  while (tm > 1 && narrow_lds(K, tm) > kLdsMost) tm >>= 1;
  return tm;
}
template <int MODE, int ACT>
static void launch_narrow(const Params& p, hipStream_t stream) {
  const int tm = narrow_rows(p.R, p.E, p.K);
  if (tm == 1) launch_narrow_tm<MODE, ACT, 1>(p, stream);
  else if (tm == 2) launch_narrow_tm<MODE, ACT, 2>(p, stream);
  else launch_narrow_tm<MODE, ACT, 4>(p, stream);
}

static bool takes_narrow(int64_t R, int64_t E, int D, int H) {
  const int64_t used = R < E ? R : E;
  return R <= 64 * used && narrow_lds(D, 1) <= kLdsMost && narrow_lds(H, 1) <= kLdsMost;
}

static int check_shape(int64_t R, int E, int D, int H) {
  if (R < 0 || E < 1 || E > kMaxE || D < kBlock || H < kBlock) return kErrInvalidArgument;
  if (D % kBlock || H % kBlock || D > (1 << 24) || H > (1 << 24)) return kErrUnsupportedShape;
  if (R >= (int64_t)INT32_MAX / 2) return kErrUnsupportedShape;
  // tiles and units are counted in 32 bits
  if ((R / 16 + E) * ((int64_t)(D > H ? D : H) / 32 + 1) >= (int64_t)0x3fffffff) return kErrUnsupportedShape;
  return kOk;
}
static int padded_blocks(int cols) { return (cols / kBlock + 7) / 8 * 8; }
static bool aligned16(const void* a) { return ((uintptr_t)a & 15) == 0; }
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

template <typename T>
static void launch_quant(const void* x, int64_t rows, int cols, int s_ld, uint8_t* q, uint8_t* scale, hipStream_t stream) {
  const int64_t chunks = rows * (cols / 8);
  int64_t g = (chunks + 1023) / 1024;
  if (g > 16384) g = 16384;
  hipLaunchKernelGGL(quant_kernel<T>, dim3((unsigned)g), dim3(256), 0, stream, (const T*)x, chunks, cols / 8,
                     s_ld == cols / kBlock ? 0 : s_ld, (uint32_t*)q, scale);
}

}  // namespace mxfp4
}  // namespace moe

using namespace moe;
using namespace moe::mxfp4;

MOE_API int moe_mxfp4_quant_rows(const void* x, int64_t rows, int32_t cols, int32_t dtype, int32_t scale_ld,
                                 uint8_t* q, uint8_t* scale, hipStream_t stream) {
  if (rows < 0 || cols < kBlock || cols % kBlock || scale_ld < cols / kBlock || (dtype != 0 && dtype != 1))
    return kErrInvalidArgument;
  if (rows == 0) return kOk;
  if (!x || !q || !scale || !aligned16(x) || !aligned16(q)) return kErrInvalidArgument;
  if (dtype == 0) launch_quant<uint16_t>(x, rows, cols, scale_ld, q, scale, stream);
  else launch_quant<float>(x, rows, cols, scale_ld, q, scale, stream);
  return launch_status();
}

MOE_API int moe_mxfp4_dequant_rows(const uint8_t* q, const uint8_t* scale, int64_t rows, int32_t cols,
                                   int32_t scale_ld, int32_t dtype, void* x, hipStream_t stream) {
  if (rows < 0 || cols < kBlock || cols % kBlock || scale_ld < cols / kBlock || (dtype != 0 && dtype != 1))
    return kErrInvalidArgument;
  if (rows == 0) return kOk;
  if (!x || !q || !scale || !aligned16(x) || !aligned16(q)) return kErrInvalidArgument;
  const int64_t chunks = rows * (cols / 8);
  int64_t g = (chunks + 255) / 256;
  if (g > 16384) g = 16384;
  const int s_ld = scale_ld == cols / kBlock ? 0 : scale_ld;
  if (dtype == 0)
    hipLaunchKernelGGL(dequant_kernel<uint16_t>, dim3((unsigned)g), dim3(256), 0, stream, (const uint32_t*)q, scale, chunks, cols / 8, s_ld, (uint16_t*)x);
  else
    hipLaunchKernelGGL(dequant_kernel<float>, dim3((unsigned)g), dim3(256), 0, stream, (const uint32_t*)q, scale, chunks, cols / 8, s_ld, (float*)x);
  return launch_status();
}

MOE_API int moe_mxfp4_scale_ld(int32_t cols) { return cols < kBlock || cols % kBlock ? kErrInvalidArgument : padded_blocks(cols); }

// workspace of the experts' forward: x in MXFP4 with its scales, h with its scales
MOE_API int64_t moe_mxfp4_workspace_bytes(int64_t n_rows, int32_t dim, int32_t hidden) {
  if (n_rows < 0 || dim < kBlock || hidden < kBlock || dim % kBlock || hidden % kBlock) return kErrInvalidArgument;
  return up256(n_rows * (dim / 2)) + up256(n_rows * padded_blocks(dim)) + up256(n_rows * (hidden / 2)) +
         up256(n_rows * padded_blocks(hidden));
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
  if (ws_bytes < moe_mxfp4_workspace_bytes(R, D, H)) return kErrWorkspace;
  uint8_t* qx = ws;
  uint8_t* sx = qx + up256(R * (D / 2));
  uint8_t* qh = sx + up256(R * padded_blocks(D));
  uint8_t* sh = qh + up256(R * (H / 2));
  const bool oss = ACT == kOssGLU;
  Params p{};
  p.counts = counts; p.R = R; p.E = E; p.K = D; p.N = H;
  p.x = x; p.qp = qx; p.sp = sx; p.p_ld = padded_blocks(D);
  p.qa = qw1; p.sa = sw1; p.qb = qw3; p.sb = sw3;
  p.e_rows = oss ? 2 * (int64_t)H : H;
  p.r_rows = oss ? 2 : 1;
  p.bias = b1; p.limit = limit;
  p.qh = qh; p.sh = sh; p.h_ld = padded_blocks(H);
  const bool narrow = takes_narrow(R, E, D, H);
  if (narrow) {
    launch_narrow<kGateUp, ACT>(p, stream);
  } else {
    launch_quant<uint16_t>(x, R, D, p.p_ld, qx, sx, stream);
    launch_wide<kGateUp, ACT, false>(p, stream);
  }
  p.K = H; p.N = D;
  p.qp = qh; p.sp = sh; p.p_ld = padded_blocks(H);
  p.qa = qw2; p.sa = sw2; p.e_rows = D; p.r_rows = 1;
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
  if (!counts) return kErrInvalidArgument;
  if (n_rows == 0) return kOk;
  if (!qx || !sx || !qw1 || !sw1 || !qw3 || !sw3 || !qh || !sh || !g8 || !gs || !u8 || !us) return kErrInvalidArgument;
  for (const void* q : {(const void*)qx, (const void*)sx, (const void*)qw1, (const void*)qw3, (const void*)sw1,
                        (const void*)sw3, (const void*)qh, (const void*)g8, (const void*)u8})
    if (!aligned16(q)) return kErrInvalidArgument;
  Params p{};
  p.counts = counts; p.R = n_rows; p.E = n_experts; p.K = dim; p.N = hidden;
  p.qp = qx; p.sp = sx; p.p_ld = padded_blocks(dim);
  p.qa = qw1; p.sa = sw1; p.qb = qw3; p.sb = sw3; p.e_rows = hidden; p.r_rows = 1;
  p.qh = qh; p.sh = sh; p.h_ld = padded_blocks(hidden);
  p.g8 = g8; p.gs = gs; p.u8 = u8; p.us = us;
  launch_wide<kGateUp, kSwiGLU, true>(p, stream);
  return launch_status();
}

MOE_API int moe_mxfp4_gemm_down(const uint8_t* qh, const uint8_t* sh, const uint8_t* qw2, const uint8_t* sw2,
                                const int64_t* counts, int64_t n_rows, int32_t n_experts, int32_t dim, int32_t hidden,
                                uint16_t* y, hipStream_t stream) {
  const int st = check_shape(n_rows, n_experts, dim, hidden);
  if (st) return st;
  if (!counts) return kErrInvalidArgument;
  if (n_rows == 0) return kOk;
  if (!qh || !sh || !qw2 || !sw2 || !y) return kErrInvalidArgument;
  for (const void* q : {(const void*)qh, (const void*)sh, (const void*)qw2, (const void*)sw2, (const void*)y})
    if (!aligned16(q)) return kErrInvalidArgument;
  Params p{};
  p.counts = counts; p.R = n_rows; p.E = n_experts; p.K = hidden; p.N = dim;
  p.qp = qh; p.sp = sh; p.p_ld = padded_blocks(hidden);
  p.qa = qw2; p.sa = sw2; p.qb = qw2; p.sb = sw2; p.e_rows = dim; p.r_rows = 1;
  p.y = y;
  launch_wide<kDown, kSwiGLU, false>(p, stream);
  return launch_status();
}
