// Block-scaled (MX) formats on MI355X (gfx950): 32 consecutive elements along a row share one
// power-of-two scale, kept as an e8m0 byte k + 127. For a format whose largest value is M the
// scale is the least 2^k, k in [-127, 127], with max |x| <= M 2^k (rounded up: no element
// saturates), and an element is x 2^-k rounded to the nearest of the format's values, ties to
// the even code. A block that holds an infinity or a NaN gets the scale byte 255 (NaN), with
// which all of its 32 values are NaN: neither format has infinities, e2m1 no NaN either. A
// block of zeros has k = -127.
//
//   MXFP4: e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6), M = 6 = 1.5 * 2^2, two elements per byte, the
//          first in the low half
//   MXFP8: e4m3 (OCP e4m3fn), M = 448 = 1.75 * 2^8
#pragma once

#include "common.h"

namespace moe {
namespace mx {

constexpr int kBlock = 32;

// Scale byte of a block from the bits of its max |x| taken over integers (bits of |x| order
// as the values do, with infinities and NaN on top, which a float maximum would drop). With
// max = m 2^a, m in [1, 2), and M = m' 2^b: k = a - b, one more where m > m'.
template <uint32_t kMantissa, int kExponent>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - kExponent + ((amax_bits & 0x7fffffu) > kMantissa ? 1 : 0);
  return amax_bits >= 0x7f800000u ? 255u : (uint32_t)max(e, 0);
}
__device__ __forceinline__ uint32_t scale_byte4(uint32_t amax_bits) { return scale_byte<0x400000u, 2>(amax_bits); }
__device__ __forceinline__ uint32_t scale_byte8(uint32_t amax_bits) { return scale_byte<0x600000u, 8>(amax_bits); }

// 2^-k, the elements' multiplier (exact: k <= 126 for finite blocks); 0 for a NaN block, whose
// scale byte makes all of its values NaN: its codes, conversions of zeros and NaN then, are not
// defined
__device__ __forceinline__ float multiplier(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
// 2^k, what a code's value is multiplied by
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u) : byte == 0u ? __uint_as_float(0x400000u) : __uint_as_float(byte << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t amax4(const float (&v)[4]) {
  return max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
}

// The maximum over the four lanes of a row in an accumulator tile (lane l, l ^ 16, l ^ 32,
// l ^ 48): two lane swaps, no LDS.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}

// Four or eight floats, each at most 6 in magnitude, to e2m1 codes, the first in the lowest
// half byte (v_cvt_scalef32_pk_fp4_f32 with a scale of 1: round to nearest even; checked on
// the GPU against the definition for every fp32 value up to 6).
__device__ __forceinline__ uint32_t e2m1x8(const float (&a)[4], const float (&b)[4]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[0], a[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[2], a[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, b[0], b[1], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, b[2], b[3], 1.0f, 3);
}

// Four floats, each at most 448 in magnitude, to e4m3 bytes (v_cvt_pk_fp8_f32).
__device__ __forceinline__ uint32_t e4m3x4(const float (&v)[4]) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
}
__device__ __forceinline__ void from_e4m3x4(uint32_t w, float s, float (&v)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo[0] * s; v[1] = lo[1] * s; v[2] = hi[0] * s; v[3] = hi[1] * s;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Lane (row, g) holds words 4 g .. 4 g + 3 of its row and gets words g, 4 + g, 8 + g, 12 + g.
__device__ __forceinline__ uint4 transpose4(uint4 v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v.x, v.z, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(v.y, v.w, false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return make_uint4(c[0], c[1], d[0], d[1]);
}

// One row's block of 32 columns in an accumulator tile: lane (row, g) holds columns 4 g .. of
// the first 16 (a) and of the second (b). Returns the scale byte (in all four lanes) and in
// `q` this lane's eight consecutive columns 8 g .. 8 g + 7 of the block, MXFP4 in one word,
// MXFP8 in two, exchanged between the row's lanes as span64 exchanges bf16 pieces.
__device__ __forceinline__ uint32_t block4(const float (&a)[4], const float (&b)[4], uint32_t& q) {
  const uint32_t s = scale_byte4(row_max(max(amax4(a), amax4(b))));
  const float m = multiplier(s);
  const float am[4] = {a[0] * m, a[1] * m, a[2] * m, a[3] * m}, bm[4] = {b[0] * m, b[1] * m, b[2] * m, b[3] * m};
  const uint32_t w = e2m1x8(am, bm);
  const auto x32 = __builtin_amdgcn_permlane32_swap(w & 0xffffu, w >> 16, false, false);
  const auto x16 = __builtin_amdgcn_permlane16_swap(x32[0], x32[1], false, false);
  q = (uint32_t)x16[0] | ((uint32_t)x16[1] << 16);
  return s;
}
__device__ __forceinline__ uint32_t block8(const float (&a)[4], const float (&b)[4], uint2& q) {
  const uint32_t s = scale_byte8(row_max(max(amax4(a), amax4(b))));
  const float m = multiplier(s);
  const float am[4] = {a[0] * m, a[1] * m, a[2] * m, a[3] * m}, bm[4] = {b[0] * m, b[1] * m, b[2] * m, b[3] * m};
  const auto x32 = __builtin_amdgcn_permlane32_swap(e4m3x4(am), e4m3x4(bm), false, false);
  const auto x16 = __builtin_amdgcn_permlane16_swap(x32[0], x32[1], false, false);
  q = make_uint2(x16[0], x16[1]);
  return s;
}

// sigmoid(z) = 1 / (1 + 2^(-z log2 e)) on the hardware's exponential and reciprocal, each
// within about one unit of fp32's last place: for |z| <= 20 the result is within 2e-6 of
// its own size, far inside the spacing of the formats it goes into. z below -88 gives 0.
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

}  // namespace mx
}  // namespace moe
