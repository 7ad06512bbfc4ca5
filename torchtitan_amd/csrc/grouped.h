// Products grouped by expert: rows sorted by expert, counts [E] on the device. Direct-to-LDS copies,
// the experts' segments of rows and tiles, and searches in them.
#pragma once

#include <type_traits>

#include "common.h"

namespace moe {
namespace grouped {

constexpr int kMaxE = 1024;

#define LDSP __attribute__((address_space(3)))
// One wave-wide direct-to-LDS copy: lane i's 4 bytes at g land at LDS byte address lds + 4 i;
// waited for with vmcnt. s_nop: a copy may read m0 one wait state after a scalar instruction
// wrote it at the earliest, and the compiler, which keeps to that elsewhere, does not look into
// the asm.
__device__ __forceinline__ void dma4(const void* g, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(g), "{m0}"(lds) : "memory");
}
// The same with lane i's 2 bytes there, zeros above them.
__device__ __forceinline__ void dma2(const void* g, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_ushort %0, off" :: "v"(g), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const uint8_t* ptr) { return (uint32_t)(size_t)((LDSP const uint8_t*)ptr); }

// Copies from a scalar base and a 32-bit offset per lane, 16 bytes a lane at lds + 16 i or 4 at
// lds + 4 i. (readfirstlane: under pressure the compiler keeps uniform values in vector registers,
// which the instruction does not take there. s_nop: a scalar register that a vector instruction
// has just written may be read by a memory instruction five wait states later at the earliest;
// m0's one lies within them.)
__device__ __forceinline__ uint64_t scalar(const uint8_t* p) {
  const uint64_t v = (uint64_t)p;
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
         ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(scalar(base)), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void dma4(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" :: "v"(off), "s"(scalar(base)), "{m0}"(lds) : "memory");
}

template <int N, typename F>
__device__ __forceinline__ void for_each(F f) {  // f(0), ..., f(N - 1) with compile-time indices
  if constexpr (N > 0) {
    for_each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}
constexpr int kTileList = 64;

// What segments() takes for expert e's count.
template <typename P>
__device__ __forceinline__ int64_t count_of(const P& p, int e) { return p.counts[e]; }

// Expert e's rows [seg[e], seg[e + 1]), clamped to R, and the exclusive sums of
// tiles_of(rows) in `tile`, both of E + 1 ints in LDS. Called by every thread of a workgroup of
// at least 256; negative counts count as none.
template <typename P, typename F>
__device__ __forceinline__ void segments(const P& p, int* seg, int* tile, int* tmp, F tiles_of) {
  const int tid = threadIdx.x, R = (int)p.R;
  int cnt[4], sg[4], tl[4], ts[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = tid * 4 + i;
    const int64_t c = e < p.E ? count_of(p, e) : 0;
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
// Inclusive sums over the wave's lanes that stop at `most`, of non-negative ints: four steps in
// rows of 16 lanes, then the last lanes of the rows before. Cross-lane operands of vector
// instructions: a step costs a few cycles where one through LDS costs a hundred.
__device__ __forceinline__ int wave_scan(int v, int most) {
  v = min(v, most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false), most);  // row_shr 1, 2, 4, 8
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false), most);
  v = min(v + __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false), most);  // lane 15 of the row before
  return min(v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false), most);  // lane 31
}
// the sums over the lanes below
__device__ __forceinline__ int wave_scan_below(int v, int most) {
  return __builtin_amdgcn_update_dpp(0, wave_scan(v, most), 0x138, 0xf, 0xf, false);  // wave_shr 1
}

// segments() by the first wave alone (lane l the experts l n .. l n + n - 1, n = ceil(E / 64) <= MOST),
// where a launch is so short that the barriers of the scans above are a third of it. One barrier.
template <int MOST, typename P, typename F>
__device__ __forceinline__ void segments_of_lanes(const P& p, int* seg, int* tile, F tiles_of) {
  const int lane = threadIdx.x, R = (int)p.R, n = (p.E + 63) / 64;
  int64_t raw[MOST];
  int cnt[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) {  // all of them on their way before the first is used
    const int e = lane * n + i;
    raw[i] = i < n && e < p.E ? count_of(p, e) : 0;
  }
  int rows = 0;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    cnt[i] = raw[i] < 0 ? 0 : (raw[i] > p.R ? R : (int)raw[i]);
    rows = min(rows + cnt[i], R);
  }
  int at = wave_scan_below(rows, R), tiles = 0;
  const int at0 = at;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    cnt[i] = min(cnt[i], R - at);
    at += cnt[i];
    tiles += tiles_of(cnt[i]);
  }
  int run = at0, tl = wave_scan_below(tiles, 0x3fffffff);
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int e = lane * n + i;
    if (i < n && e < p.E) { seg[e] = run; tile[e] = tl; }
    run += cnt[i];
    tl += tiles_of(cnt[i]);
  }
  if (lane == 63) { seg[p.E] = run; tile[p.E] = tl; }
}
template <typename P, typename F>
__device__ __forceinline__ void segments_wave(const P& p, int* seg, int* tile, F tiles_of) {
  if (threadIdx.x < 64) {
    if (p.E <= 256) segments_of_lanes<4>(p, seg, tile, tiles_of);
    else segments_of_lanes<kMaxE / 64>(p, seg, tile, tiles_of);
  }
  __syncthreads();
}
// find() by a wave at once: the last e with start[e] <= t
__device__ __forceinline__ int find_wave(const int* start, int E, int t) {
  const int lane = threadIdx.x & 63, n = (E + 63) / 64;
  const int blk = __popcll(__ballot(lane * n < E && start[min(lane * n, E - 1)] <= t)) - 1;
  const int e = blk * n + lane;
  return blk * n + __popcll(__ballot(lane < n && e < E && start[min(e, E - 1)] <= t)) - 1;
}
__device__ __forceinline__ int find(const int* start, int E, int t) {  // the last e with start[e] <= t
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// compute units of the current device
inline int cu_count() {
  static int g_cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!g_cus[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    g_cus[dev] = n;
  }
  return g_cus[dev];
}

}  // namespace grouped
}  // namespace moe
