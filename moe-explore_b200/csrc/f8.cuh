// 8-bit rows: e4m3 values with one fp32 scale per row and block of 128 columns.
//   scale = max(max |v|, 2^-80) / 448,  q = e4m3(v / scale)     (448 is the largest e4m3 value)
// 16-bit rows get the quotient rounded once (f8_quotients).  The norm's results and the activated products exist as fp32 sums and products
// with roundings of their own; they are multiplied by the rounded 448 / max, one unit of fp32 more, which for a value next to the middle
// between two 8-bit ones may decide.  (The one rounding there: 8192 x 7168 from the norm 90 us instead of 82.5, 3001 uneven tokens
// through 64 experts 311 instead of 297, one token through 8 experts 91 instead of 86.)
// The floor keeps the scale of an empty block a normal number; a block's NaN stays a NaN in place, an infinity makes the block's
// scale infinite (the row's products are then NaN).
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace moe {

constexpr int kF8Block = 128;
constexpr float kF8Top = 448.0f;
constexpr float kF8Least = 8.271806125530277e-25f;  // 2^-80

// grid_wait() of the kernels in this family.  They may read the maps before it where a kernel before their predecessor wrote them
// (F8Args::maps_before), past L1; otherwise what is said at grid_wait() holds for them, no __restrict__ and no __ldg included.
// (tests/test_synchronisation_sources.py finds the kernels that wait by what they call, not by the name.)
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

// f[i] * 448 / most.  16-bit values often lie exactly in the middle between two 8-bit ones; with one rounding (7/8 v is exact, and so
// is the factor 512) they stay there and go to the even one, whoever computes it.  The quotients share their divisor: one rounded
// reciprocal, and per value a product, its remainder and a correction, which rounds as a division does (Markstein's theorem, in
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  Both sides are first brought by a power of two
// to where reciprocal and remainder are normal numbers; a value that is not normal then is far below the least 8-bit one.
// (Eight divisions of their own were 100 instructions per thread, and the kernel of the rows was bound by them.)
template <int N> __device__ __forceinline__ void f8_quotients(float (&f)[N], float most) {
  if (!(most <= 3.0e38f)) {  // infinite, or nothing is left to spare: as the formula says
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __fdiv_rn(f[i] * 0.875f, most) * 512.0f;
    return;
  }
  const float near1 = most >= 1.0f ? 0x1p-60f : 0x1p60f;  // d: 2^-60 to 2^68, or 2^-20 to 2^60
  const float d = most * near1, r = __frcp_rn(d);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float v = f[i] * (0.875f * near1);
    const float q = v * r;
    f[i] = copysignf(fmaf(fmaf(-q, d, v), r, q) * 512.0f, v);  // (the correction makes -0 a 0)
  }
}

}  // namespace moe
