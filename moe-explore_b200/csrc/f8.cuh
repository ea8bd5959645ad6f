// 8-bit rows: e4m3 values with one fp32 scale per row and block of 128 columns.
//   scale = max(max |v|, 2^-80) / 448,  q = e4m3(v / scale)     (448 is the largest e4m3 value)
// The floor keeps the scale of an empty block a normal number; a block's NaN stays a NaN in place, an infinity makes the block's
// scale infinite (the row's products are then NaN).
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace moe {

constexpr int kF8Block = 128;
constexpr float kF8Top = 448.0f;
constexpr float kF8Least = 8.271806125530277e-25f;  // 2^-80

// The wait of the kernels in this family for the one they are chained to: nothing before it touches global memory, and what was
// said about such kernels at grid_wait() holds for them (no __restrict__, no __ldg).
__device__ __forceinline__ void await_predecessor() { grid_wait(); }

__device__ __forceinline__ uint32_t f8x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Largest |v| over the 16 lanes that share a block (8 values each).
__device__ __forceinline__ float block_most(const float (&v)[8]) {
  float m = kF8Least;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
  return m;
}

// v * 448 / most.  16-bit values often lie exactly in the middle between two 8-bit ones; with one rounding (7/8 v is exact, and so
// is the factor 512) they stay there and go to the even one, whoever computes it.
__device__ __forceinline__ float f8_exact(float v, float most) { return __fdiv_rn(v * 0.875f, most) * 512.0f; }

}  // namespace moe
