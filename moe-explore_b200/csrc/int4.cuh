// Products of a few 16-bit rows with 4-bit weights: element [n, k] = (value - zero) * scale, a value of 0 to 15, scale (in the rows' type)
// and zero (8 where there is none) per row n and group of 32, 64 or 128 columns.
//
// Layout.  A matrix [N, K] is cut into tiles of 16 rows and steps of 128 columns; a step of a tile is one block, 1 KB of values, then the
// scales, then the zeros, and the steps of a tile lie one behind the other, so that a warp reads one stream.  Byte (half * 32 + lane) * 16
// + i * 4 + b of the values belongs to row (lane / 4) + 8 half and word i of that lane: columns 32 i + 8 (lane % 4) + 0..7, the even ones in
// the word's low half and the odd ones in the high half, lowest column lowest.  Scales and zeros: [16 rows][groups of the step].  Rows
// behind N and columns behind K hold zeros, values and scales.
//
// A step's fragments.  m16n8k16 with the weights as its 16 rows and eight tokens as its columns: the sums over k may take the columns in
// any order, as long as both operands do, and in the order above (word >> 4 j) & 0x000F000F is the pair of columns 2 j, 2 j + 1 of a
// fragment, and a token's 16 consecutive bytes are the other operand's as they are.  The pair becomes two numbers by setting the exponent
// bits of 128 (bf16) or 1024 (fp16), whose last mantissa bits it then is, and subtracting 128 + zero (1024 + zero), exactly.  Word i
// holds columns of one group of 32 for all lanes, so the scale is applied to the fp32 sums of a group: no weight is ever rounded.
//
// Tensor cores by mma.sync, because the weights are made in registers and there are only 16 of their rows: per KB of weights a warp issues 88
// instructions to make them and 8 to multiply; the 56 integer ones among them are what bounds the rate beside HBM.
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
// The same, or 16 zero bytes (nothing is read then).
__device__ __forceinline__ void copy_16_or_zeros(uint32_t to, const void* from, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last N groups of this thread's copies have landed.
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One matrix (a matrix per expert follows), as the kernels see it: [tiles][steps][block].
struct Q4Matrix {
  const uint8_t* data;
  int64_t tiles;
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

// A step in shared memory: its block, then the same columns of eight tokens' rows, 256 bytes each, their 16-byte pieces turned by four in
// every second row (so that the eight lanes of a load that are served at once read two rows without a conflict).
template <int NG, bool ZEROS> struct Q4Stage {
  static constexpr int kScales = 1024, kZeros = kScales + 32 * NG, kBlock = kZeros + (ZEROS ? 16 * NG : 0), kRows = kBlock, kBytes = kRows + 2048;
};
template <int NG, bool ZEROS> __device__ __forceinline__ void q4_copy(uint32_t stage, const uint8_t* block, int lane) {
  const uint8_t* from = block + lane * 16;
  const uint32_t to = stage + lane * 16;
  copy_16(to, from);
  copy_16(to + 512, from + 512);
  if (lane < (ZEROS ? 3 : 2) * NG) copy_16(to + 1024, from + 1024);
}
// The rows' part: row(r) gives row r < count, for lanes 0..15 even rows, for the others odd ones.
template <int NG, bool ZEROS, typename Row>
__device__ __forceinline__ void q4_copy_rows(uint32_t stage, Row row, int count, int K, int step, int lane) {
  const int piece = lane & 15, odd = lane >> 4, k = step * kQ4Step + 8 * piece;
  const bool real = k < K;
  const uint32_t to = stage + Q4Stage<NG, ZEROS>::kRows + odd * 256 + ((piece ^ (odd << 2)) << 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (2 * i >= count) break;
    if (2 * i + odd < count) {
      const uint16_t* x = row(i);
      copy_16_or_zeros(to + i * 512, real ? x + k : x, real);
    }
  }
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

// Where a lane finds the other operand of word 0: eight columns of token lane / 4 (of the first one behind the last: its products are
// nobody's); of word i at this ^ 64 (i & 1) + 128 (i / 2).
__device__ __forceinline__ uint32_t q4_row_at(int count, int lane) {
  const int g = lane >> 2, r = g < count ? g : 0;
  return r * 256 + (((lane & 3) ^ ((r & 1) << 2)) << 4);
}

// acc += the tile's product with up to eight rows over one step, by groups.
template <typename T, int NG, bool ZEROS>
__device__ __forceinline__ void q4_step(float (&acc)[4], uint32_t stage, uint32_t row_at, int lane) {
  constexpr int kPerGroup = 4 / NG;  // words
  Q4Piece<NG, ZEROS> p;
  q4_take<NG, ZEROS>(p, stage, lane);
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    float sum[4] = {};
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
      const uint4 b = lds_128(stage + Q4Stage<NG, ZEROS>::kRows + (row_at ^ (64 * (i & 1))) + 128 * (i >> 1));
      mma_16x8x16<T>(sum, a[0], b.x, b.y);
      mma_16x8x16<T>(sum, a[1], b.z, b.w);
    }
    const float s0 = q4_scale<T>(p.scale[0], j), s1 = q4_scale<T>(p.scale[1], j);
    acc[0] = fmaf(sum[0], s0, acc[0]);
    acc[1] = fmaf(sum[1], s0, acc[1]);
    acc[2] = fmaf(sum[2], s1, acc[2]);
    acc[3] = fmaf(sum[3], s1, acc[3]);
  }
}

}  // namespace moe
