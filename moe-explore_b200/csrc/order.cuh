// An order of floating-point values that whole numbers have, for choices among scores.
#pragma once

#include "common.cuh"

#include <math_constants.h>

namespace moe {

// Values as unsigned integers in the same order; NaN below all of them, 0 below NaN (no candidate).
template <typename V> struct Order;
template <> struct Order<float> {
  typedef uint32_t Key;
  __device__ static __forceinline__ Key key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and 0 are equal
    return v != v ? 1u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  }
  __device__ static __forceinline__ float value(Key k) {
    return k <= 1u ? CUDART_NAN_F : __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
  }
  __device__ static __forceinline__ Key warp_max(Key k) { return __reduce_max_sync(0xFFFFFFFFu, k); }
  __device__ static __forceinline__ Key warp_min(Key k) { return __reduce_min_sync(0xFFFFFFFFu, k); }
};
template <> struct Order<double> {
  typedef unsigned long long Key;
  __device__ static __forceinline__ Key key(double v) {
    const Key u = static_cast<Key>(__double_as_longlong(v + 0.0));
    return v != v ? 1ull : (u >> 63) ? ~u : u | (1ull << 63);
  }
  __device__ static __forceinline__ double value(Key k) {
    return k <= 1ull ? CUDART_NAN : __longlong_as_double(static_cast<long long>((k >> 63) ? k & ~(1ull << 63) : ~k));
  }
  __device__ static __forceinline__ Key warp_max(Key k) {
    const uint32_t hi = static_cast<uint32_t>(k >> 32);
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, hi);
    const uint32_t low = __reduce_max_sync(0xFFFFFFFFu, hi == top ? static_cast<uint32_t>(k) : 0u);
    return (static_cast<Key>(top) << 32) | low;
  }
  __device__ static __forceinline__ Key warp_min(Key k) { return ~warp_max(~k); }
};

}  // namespace moe
