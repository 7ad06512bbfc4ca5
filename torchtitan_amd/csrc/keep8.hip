// Rows kept in MXFP8 between a forward and its backward (gfx950): e4m3 elements, one e8m0 scale
// per 32 along the row (mx.h). Streaming kernels, bound by HBM: 3.03 bytes per element each way.
// In a training step 131072 rows of 2304 are kept in 175 us (5.2 TB/s) and restored in 152 us
// (6.0 TB/s).
#include "mx.h"

namespace moe {
namespace keep8 {

// x as n_chunks chunks of eight bf16: four consecutive lanes hold a block. Chunk c's bytes are
// q[c], its block's scale scale[c / 4]. Four chunks per thread are loaded before any is processed.
__global__ __launch_bounds__(256) void keep_kernel(const uint4* __restrict__ x, int64_t n_chunks,
                                                   uint2* __restrict__ q, uint8_t* __restrict__ scale) {
  const int64_t S = (int64_t)gridDim.x * 256;
  for (int64_t c0 = (int64_t)blockIdx.x * 256 + threadIdx.x; c0 - threadIdx.x < n_chunks; c0 += 4 * S) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * S;
      v[u] = c < n_chunks ? x[c] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * S;
      float a[4], b[4];
      unpack4(make_uint2(v[u].x, v[u].y), a);
      unpack4(make_uint2(v[u].z, v[u].w), b);
      uint32_t m = max(mx::amax4(a), mx::amax4(b));
      m = max(m, (uint32_t)__shfl_xor((int)m, 1));
      m = max(m, (uint32_t)__shfl_xor((int)m, 2));
      const uint32_t s = mx::scale_byte8(m);
      const float f = mx::multiplier(s);
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] *= f; b[i] *= f; }
      if (c < n_chunks) {
        q[c] = make_uint2(mx::e4m3x4(a), mx::e4m3x4(b));
        if ((c & 3) == 0) scale[c >> 2] = (uint8_t)s;
      }
    }
  }
}

__global__ __launch_bounds__(256) void restore_kernel(const uint2* __restrict__ q, const uint8_t* __restrict__ scale,
                                                      int64_t n_chunks, uint4* __restrict__ x) {
  const int64_t S = (int64_t)gridDim.x * 256;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < n_chunks; c += S) {
    const uint2 w = q[c];
    const float s = mx::scale_value(scale[c >> 2]);
    float a[4], b[4];
    mx::from_e4m3x4(w.x, s, a);
    mx::from_e4m3x4(w.y, s, b);
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    x[c] = Chunk<uint16_t>::pack(v);
  }
}

static int check(const void* x, int64_t rows, int32_t cols, const void* q, const void* scale) {
  if (rows < 0 || cols < mx::kBlock || cols % mx::kBlock) return kErrInvalidArgument;
  if (rows && (!x || !q || !scale || ((uintptr_t)x & 15) || ((uintptr_t)q & 7))) return kErrInvalidArgument;
  return kOk;
}

}  // namespace keep8
}  // namespace moe

using namespace moe;

MOE_API int moe_keep8_rows(const uint16_t* x, int64_t rows, int32_t cols, uint8_t* q, uint8_t* scale,
                           hipStream_t stream) {
  const int st = keep8::check(x, rows, cols, q, scale);
  if (st || rows == 0) return st;
  const int64_t chunks = rows * (cols / 8);
  int64_t g = (chunks + 1023) / 1024;
  if (g > 16384) g = 16384;
  hipLaunchKernelGGL(keep8::keep_kernel, dim3((unsigned)g), dim3(256), 0, stream, (const uint4*)x, chunks, (uint2*)q, scale);
  return launch_status();
}

MOE_API int moe_restore8_rows(const uint8_t* q, const uint8_t* scale, int64_t rows, int32_t cols, uint16_t* x,
                              hipStream_t stream) {
  const int st = keep8::check(x, rows, cols, q, scale);
  if (st || rows == 0) return st;
  const int64_t chunks = rows * (cols / 8);
  int64_t g = (chunks + 255) / 256;
  if (g > 16384) g = 16384;
  hipLaunchKernelGGL(keep8::restore_kernel, dim3((unsigned)g), dim3(256), 0, stream, (const uint2*)q, scale, chunks, (uint4*)x);
  return launch_status();
}
