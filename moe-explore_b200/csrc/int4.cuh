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
// Tensor cores by mma.sync, because the weights are made in registers and a tile has only 16 of their rows: per KB of weights a warp issues 88
// instructions to make them (56 of them on the integer pipe, which takes one every other cycle), 8 to multiply and about 70 around them.  So
// long streams are bound by issuing, at 3.5 to 4 TB/s of weights.  (Two tiles per warp instead of one: 382 us instead of 420 for 64
// experts of 7168 x 2048; the pair of numbers masked and given its exponent by one lop3, which the compiler makes two of: 320; four
// tiles: no gain.)
#pragma once

#include "common.cuh"

namespace moe {

constexpr int kQ4Step = 128;    // columns
constexpr int kQ4Rows = 16;

template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same onto zeros.
template <typename T> __device__ __forceinline__ void mma_16x8x16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16_first<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <> __device__ __forceinline__ void mma_16x8x16_first<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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

// A warp works on two tiles at a time: the rows' operands are fetched for both, and what a step costs besides its numbers is shared.
// A step in shared memory: the tiles' blocks, then the same columns of eight tokens' rows, 256 bytes each, their 16-byte pieces turned by four
// in every second row (so that the eight lanes of a load that are served at once read two rows without a conflict).
constexpr int kQ4Tiles = 2, kQ4Cols = kQ4Tiles * kQ4Rows;
template <int NG, bool ZEROS> struct Q4Stage {
  static constexpr int kScales = 1024, kZeros = kScales + 32 * NG, kBlock = kZeros + (ZEROS ? 16 * NG : 0), kRows = kQ4Tiles * kBlock, kBytes = kRows + 2048;
};
// `block`: the lane's first 16 bytes of the first tile's; the second tile's lies `apart` bytes behind (0: there is none).
template <int NG, bool ZEROS> __device__ __forceinline__ void q4_copy(uint32_t stage, const uint8_t* block, int64_t apart, int lane) {
  constexpr int kBlock = Q4Stage<NG, ZEROS>::kBlock;
  const uint32_t to = stage + lane * 16;
  copy_16(to, block);
  copy_16(to + 512, block + 512);
  if (apart != 0) {
    copy_16(to + kBlock, block + apart);
    copy_16(to + kBlock + 512, block + apart + 512);
  }
  if (lane < (ZEROS ? 3 : 2) * NG) {
    copy_16(to + 1024, block + 1024);
    if (apart != 0) copy_16(to + kBlock + 1024, block + apart + 1024);
  }
}
// The rows' part.  Lanes 0..15 copy the even rows, the others the odd ones: x[i] is the lane's piece of row 2 i + lane / 16, `at` the step's
// first column.
template <int NG, bool ZEROS>
__device__ __forceinline__ void q4_copy_rows(uint32_t stage, const uint16_t* const (&x)[4], int count, int K, int at, int lane) {
  const int piece = lane & 15, odd = lane >> 4;
  const uint32_t to = stage + Q4Stage<NG, ZEROS>::kRows + odd * 256 + ((piece ^ (odd << 2)) << 4);
  if (at + kQ4Step <= K) {
    if (odd < count) copy_16(to, x[0] + at);
    if (count > 2) {
      if (2 + odd < count) copy_16(to + 512, x[1] + at);
      if (count > 4) {
        if (4 + odd < count) copy_16(to + 1024, x[2] + at);
        if (6 + odd < count) copy_16(to + 1536, x[3] + at);
      }
    }
  } else {
    const bool real = at + 8 * piece < K;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (2 * i + odd < count) copy_16_or_zeros(to + i * 512, real ? x[i] + at : x[i] - 8 * piece, real);
  }
}

// Loads from shared memory, in order with the copies and waits around them (volatile), free to move among the arithmetic.
__device__ __forceinline__ uint4 lds_128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds_64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

// What a lane takes of a tile's step: its words of rows g and g + 8, and their scales and zeros.
template <int NG, bool ZEROS> struct Q4Piece {
  uint4 w[2];
  uint32_t scale[2][NG == 4 ? 2 : 1];
  uint32_t zero[2];
};
template <int NG, bool ZEROS> __device__ __forceinline__ void q4_take(Q4Piece<NG, ZEROS>& p, uint32_t block, int lane) {
  using S = Q4Stage<NG, ZEROS>;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    p.w[h] = lds_128(block + lane * 16 + h * 512);
    const uint32_t row = lane >> 2;
    if constexpr (NG == 4) {
      const uint2 both = lds_64(block + row * 8 + S::kScales + 64 * h);
      p.scale[h][0] = both.x;
      p.scale[h][1] = both.y;
      if constexpr (ZEROS) p.zero[h] = lds_32(block + row * 4 + S::kZeros + 32 * h);
    } else if constexpr (NG == 2) {
      p.scale[h][0] = lds_32(block + row * 4 + S::kScales + 32 * h);
      if constexpr (ZEROS) p.zero[h] = lds_16(block + row * 2 + S::kZeros + 16 * h);
    } else {
      p.scale[h][0] = lds_16(block + row * 2 + S::kScales + 16 * h);
      if constexpr (ZEROS) p.zero[h] = lds_8(block + row + S::kZeros + 8 * h);
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

// (word & 0x000F000F) | magic as the one instruction that it is.
__device__ __forceinline__ uint32_t q4_pair(uint32_t word, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r) : "r"(word), "r"(magic));
  return r;
}

// Word i of a tile as the two fragments of its products.
template <typename T, int NG, bool ZEROS> __device__ __forceinline__ void q4_numbers(uint32_t (&a)[2][4], const Q4Piece<NG, ZEROS>& p, int i) {
  const int j = i * NG / 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t bias = Q4Magic<T>::kEight;
    if constexpr (ZEROS) {
      const uint32_t z = (p.zero[h] >> (8 * j)) & 15u;
      bias = Q4Magic<T>::kBits | z | (z << 16);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)  // pair q of the words of rows g and g + 8: fragment q / 2, its first or second eight columns
      a[q >> 1][2 * (q & 1) + h] = sub2(q4_pair(word_of(p.w[h], i) >> (4 * q), Q4Magic<T>::kBits), bias, T());
  }
}

// acc[tile] += the tiles' products with up to eight rows over one step, by groups.
template <typename T, int NG, bool ZEROS>
__device__ __forceinline__ void q4_step(float (&acc)[kQ4Tiles][4], uint32_t stage, uint32_t row_at, int lane) {
  constexpr int kPerGroup = 4 / NG;  // words
  Q4Piece<NG, ZEROS> p[kQ4Tiles];
#pragma unroll
  for (int t = 0; t < kQ4Tiles; ++t) q4_take<NG, ZEROS>(p[t], stage + t * Q4Stage<NG, ZEROS>::kBlock, lane);
  float sum[kQ4Tiles][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = i / kPerGroup;
    const uint4 b = lds_128(stage + (row_at ^ (64 * (i & 1))) + Q4Stage<NG, ZEROS>::kRows + 128 * (i >> 1));
#pragma unroll
    for (int t = 0; t < kQ4Tiles; ++t) {
      uint32_t a[2][4];
      q4_numbers<T, NG, ZEROS>(a, p[t], i);
      if (i % kPerGroup == 0) mma_16x8x16_first<T>(sum[t], a[0], b.x, b.y);
      else mma_16x8x16<T>(sum[t], a[0], b.x, b.y);
      mma_16x8x16<T>(sum[t], a[1], b.z, b.w);
      if (i % kPerGroup == kPerGroup - 1) {
        const float s0 = q4_scale<T>(p[t].scale[0], j), s1 = q4_scale<T>(p[t].scale[1], j);
        acc[t][0] = fmaf(sum[t][0], s0, acc[t][0]);
        acc[t][1] = fmaf(sum[t][1], s0, acc[t][1]);
        acc[t][2] = fmaf(sum[t][2], s1, acc[t][2]);
        acc[t][3] = fmaf(sum[t][3], s1, acc[t][3]);
      }
    }
  }
}

}  // namespace moe
