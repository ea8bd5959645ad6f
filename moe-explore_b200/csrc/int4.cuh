// Products of a few 16-bit rows with 4-bit weights: element [n, k] = (value - zero) * scale, a value of 0 to 15, scale (in the rows' type)
// and zero (8 where there is none) per row n and group of 32, 64 or 128 columns.
//
// Layout.  A matrix [N, K] is cut into tiles of 16 rows and steps of 128 columns; a step of a tile is 1 KB, the steps of a tile lie one
// behind the other, so that a warp's loads are whole lines of one stream.  Byte (half * 32 + lane) * 16 + i * 4 + b of a step belongs to
// row (lane / 4) + 8 half and word i of that lane: columns 32 i + 8 (lane % 4) + 0..7, the even ones in the word's low half and the odd
// ones in the high half, lowest column lowest.  Scales (and zeros) of a step: [16 rows][groups of the step].  Rows behind N and columns
// behind K hold zeros, values and scales.
//
// A step's fragments.  m16n8k16 with the weights as its 16 rows and eight tokens as its columns: the sums over k may take the columns in
// any order, as long as both operands do, and in the order above (word >> 4 j) & 0x000F000F is the pair of columns 2 j, 2 j + 1 of a
// fragment, and a token's 16 consecutive bytes are the other operand's as they are.  The pair becomes two numbers by setting the exponent
// bits of 128 (bf16) or 1024 (fp16), whose last mantissa bits it then is, and subtracting 128 + zero (1024 + zero), exactly.  Word i
// holds columns of one group of 32 for all lanes, so the scale is applied to the fp32 sums of a group: no weight is ever rounded.
//
// Bound by HBM for up to 16 rows.  (Tensor cores by mma.sync because the weights are made in registers and M is 16: per KB of weights a
// warp issues 88 instructions to make them and 8 to multiply.)
#pragma once

#include "common.cuh"

namespace moe {

constexpr int kQ4Step = 128;    // columns
constexpr int kQ4Rows = 16;
constexpr int kQ4Words = 64;    // 16-byte pieces of a step of a tile

template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes to shared memory, past L1; they are there for this thread after copies_wait, and for the warp after __syncwarp().
__device__ __forceinline__ void copy_16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last N groups of this thread's copies have landed.
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One matrix, as the kernels see it.
struct Q4Matrix {
  const uint4* data;     // [tiles][steps][64]
  const void* scales;    // [tiles][steps][16][NG], NG = 128 / group
  const uint8_t* zeros;  // the same, or null
  int64_t tiles;         // of the whole matrix (a matrix per expert follows)
  int steps;
};

template <typename T> struct Q4Magic;
template <> struct Q4Magic<__nv_bfloat16> {
  static constexpr uint32_t kBits = 0x43004300u, kEight = 0x43084308u;
};
template <> struct Q4Magic<__half> {
  static constexpr uint32_t kBits = 0x64006400u, kEight = 0x64086408u;
};
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b, __half) {
  const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A step in shared memory: the words, each lane's copied by itself, then scales and zeros, copied by the first lanes.
template <int NG, bool ZEROS> struct Q4Stage {
  static constexpr int kScales = 1024, kZeros = kScales + 32 * NG, kBytes = kZeros + (ZEROS ? 16 * NG : 0);
};
template <int NG, bool ZEROS>
__device__ __forceinline__ void q4_copy(uint32_t stage, const uint4* data, const uint16_t* scales, const uint8_t* zeros, int step, int lane) {
  using S = Q4Stage<NG, ZEROS>;
  const uint4* from = data + static_cast<int64_t>(step) * kQ4Words + lane;
  copy_16(stage + lane * 16, from);
  copy_16(stage + 512 + lane * 16, from + 32);
  const int64_t at = static_cast<int64_t>(step) * (kQ4Rows * NG);
  if (lane < 2 * NG) copy_16(stage + S::kScales + lane * 16, scales + at + lane * 8);
  else if (ZEROS && lane < 3 * NG) copy_16(stage + S::kZeros + (lane - 2 * NG) * 16, zeros + at + (lane - 2 * NG) * 16);
}
// What a lane takes of a step: its words of rows g and g + 8, and their scales and zeros.
template <int NG, bool ZEROS> struct Q4Piece {
  uint4 w[2];
  uint32_t scale[2][NG == 4 ? 2 : 1];
  uint32_t zero[2];
};
__device__ __forceinline__ uint32_t lds_32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds_16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds_8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds_128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
template <int NG, bool ZEROS> __device__ __forceinline__ void q4_take(Q4Piece<NG, ZEROS>& p, uint32_t stage, int lane) {
  using S = Q4Stage<NG, ZEROS>;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    p.w[h] = lds_128(stage + h * 512 + lane * 16);
    const uint32_t row = (lane >> 2) + 8 * h;
    if constexpr (NG == 4) {
      p.scale[h][0] = lds_32(stage + S::kScales + row * 8);
      p.scale[h][1] = lds_32(stage + S::kScales + row * 8 + 4);
      if constexpr (ZEROS) p.zero[h] = lds_32(stage + S::kZeros + row * 4);
    } else if constexpr (NG == 2) {
      p.scale[h][0] = lds_32(stage + S::kScales + row * 4);
      if constexpr (ZEROS) p.zero[h] = lds_16(stage + S::kZeros + row * 2);
    } else {
      p.scale[h][0] = lds_16(stage + S::kScales + row * 2);
      if constexpr (ZEROS) p.zero[h] = lds_8(stage + S::kZeros + row);
    }
  }
}
template <typename T> __device__ __forceinline__ float q4_scale(const uint32_t* s, int j) {
  const uint16_t bits = static_cast<uint16_t>(s[j >> 1] >> (16 * (j & 1)));
  return Elem<T>::to_float(*reinterpret_cast<const T*>(&bits));
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// The other operand of word i: eight columns of token 8 m + lane / 4.  x: that token's row, or null.
__device__ __forceinline__ uint4 q4_row(const uint16_t* x, int K, int step, int i, int lane) {
  const int k = step * kQ4Step + 32 * i + 8 * (lane & 3);
  return x != nullptr && k < K ? *reinterpret_cast<const uint4*>(x + k) : make_uint4(0, 0, 0, 0);
}

// acc[m][..] += the tile's product over one step, by groups.
template <typename T, int NG, bool ZEROS, int MT>
__device__ __forceinline__ void q4_step(float (&acc)[MT][4], const Q4Piece<NG, ZEROS>& p, const uint16_t* const (&x)[MT], int K, int step, int lane) {
  constexpr int kPerGroup = 4 / NG;  // words
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    float sum[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) sum[m][0] = sum[m][1] = sum[m][2] = sum[m][3] = 0.0f;
    uint32_t bias[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (ZEROS) {
        const uint32_t z = (p.zero[h] >> (8 * j)) & 15u;
        bias[h] = Q4Magic<T>::kBits | z | (z << 16);
      } else {
        bias[h] = Q4Magic<T>::kEight;
      }
    }
#pragma unroll
    for (int n = 0; n < kPerGroup; ++n) {
      const int i = j * kPerGroup + n;
      uint32_t a[2][4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // pair q of the words of rows g and g + 8: fragment q / 2, its first or second eight columns
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t bits = ((word_of(p.w[h], i) >> (4 * q)) & 0x000F000Fu) | Q4Magic<T>::kBits;
          a[q >> 1][2 * (q & 1) + h] = sub2(bits, bias[h], T());
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 b = q4_row(x[m], K, step, i, lane);
        mma_16x8x16<T>(sum[m], a[0], b.x, b.y);
        mma_16x8x16<T>(sum[m], a[1], b.z, b.w);
      }
    }
    const float s0 = q4_scale<T>(p.scale[0], j), s1 = q4_scale<T>(p.scale[1], j);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      acc[m][0] = fmaf(sum[m][0], s0, acc[m][0]);
      acc[m][1] = fmaf(sum[m][1], s0, acc[m][1]);
      acc[m][2] = fmaf(sum[m][2], s1, acc[m][2]);
      acc[m][3] = fmaf(sum[m][3], s1, acc[m][3]);
    }
  }
}

// Steps first, first + stride, ... of a tile, DEPTH - 1 of them on their way while one is computed.  `ring`: DEPTH stages of this warp's
// own in shared memory.
template <typename T, int NG, bool ZEROS, int MT, int DEPTH>
__device__ __forceinline__ void q4_tile(float (&acc)[MT][4], const Q4Matrix& w, int64_t tile, const uint16_t* const (&x)[MT], int K, int first, int stride,
                                        uint32_t ring, int lane) {
  constexpr int kStage = Q4Stage<NG, ZEROS>::kBytes;
  const uint4* data = w.data + tile * w.steps * kQ4Words;
  const uint16_t* scales = static_cast<const uint16_t*>(w.scales) + tile * w.steps * (kQ4Rows * NG);
  const uint8_t* zeros = ZEROS ? w.zeros + tile * w.steps * (kQ4Rows * NG) : nullptr;
  int ahead = first;
#pragma unroll
  for (int s = 0; s < DEPTH - 1; ++s, ahead += stride) {
    if (ahead < w.steps) q4_copy<NG, ZEROS>(ring + s * kStage, data, scales, zeros, ahead, lane);
    copies_commit();
  }
  uint32_t stage = ring, free_stage = ring + (DEPTH - 1) * kStage;
  for (int step = first; step < w.steps; step += stride, ahead += stride) {
    copies_wait<DEPTH - 2>();
    __syncwarp();  // every lane's copies of this step, and every lane is through with the stage that is filled next
    if (ahead < w.steps) q4_copy<NG, ZEROS>(free_stage, data, scales, zeros, ahead, lane);
    copies_commit();
    Q4Piece<NG, ZEROS> p;
    q4_take<NG, ZEROS>(p, stage, lane);
    q4_step<T, NG, ZEROS, MT>(acc, p, x, K, step, lane);
    free_stage = stage;
    stage = stage == ring + (DEPTH - 1) * kStage ? ring : stage + kStage;
  }
  copies_wait<0>();
  __syncwarp();  // the ring is free again
}

}  // namespace moe
