// A few 16-bit rows by one matrix of 4-bit weights (int4.cuh): out [rows, N] = x [rows, K] @ w [N, K]^T.
//
// A CTA takes two tiles, 32 weight rows, and up to eight rows of x; its eight warps share the steps of K, and where there are few tiles,
// so do the CTAs of a cluster.  Their sums are joined in a fixed order, through shared memory and then the cluster's.  1 and 8 rows of 7168
// by 4096 columns (15 MB) take 7.5 and 8.2 us on the device: launch, first loads and joining; 1 row of 4096 by 28672 19 (3.3 TB/s).
#include "int4.cuh"

#include <atomic>

namespace moe {

constexpr int kQ4Warps = 8;
constexpr int kQ4Depth = 3;   // steps that a warp has room for: 2 CTAs per SM ask for 68 KB of weights at a time
template <int NG, bool ZEROS> constexpr int kQ4Ring = kQ4Depth * Q4Stage<NG, ZEROS>::kBytes;

struct Q4Args {
  Q4Matrix w;
  const uint16_t* x;
  uint16_t* out;
  int rows, K, N, ranks;
};

__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T, int NG, bool ZEROS>
__global__ void __launch_bounds__(kQ4Warps * 32, 2) q4_rows_kernel(const Q4Args a) {
  constexpr int kStage = Q4Stage<NG, ZEROS>::kBytes, TOKENS = 8;
  extern __shared__ __align__(128) uint8_t rings[];
  __shared__ float parts[kQ4Warps][TOKENS][kQ4Cols];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = a.ranks > 1 ? static_cast<int>(blockIdx.x) % a.ranks : 0;
  const int64_t tile = static_cast<int64_t>(blockIdx.x / a.ranks) * kQ4Tiles;
  const int row0 = blockIdx.y * TOKENS, count = min(a.rows - row0, TOKENS);
  constexpr int kBlock = Q4Stage<NG, ZEROS>::kBlock;
  const uint8_t* data = a.w.data + tile * a.w.steps * kBlock + lane * 16;
  const int64_t apart = tile + 1 < a.w.tiles ? static_cast<int64_t>(a.w.steps) * kBlock : 0;
  const uint16_t* x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 2 * i + (lane >> 4);
    x[i] = a.x + static_cast<int64_t>(row0 + (r < count ? r : 0)) * a.K + 8 * (lane & 15);
  }
  const uint32_t row_at = q4_row_at(count, lane);
  const int stride = a.ranks * kQ4Warps;
  int step = rank * kQ4Warps + warp, ahead = step;
  const uint32_t ring = smem_u32(rings) + warp * kQ4Ring<NG, ZEROS>;
  uint32_t to = ring, from = ring;
  const auto copy = [&]() {
    if (ahead < a.w.steps) {
      q4_copy<NG, ZEROS>(to, data + static_cast<int64_t>(ahead) * kBlock, apart, lane);
      q4_copy_rows<NG, ZEROS>(to, x, count, a.K, ahead * kQ4Step, lane);
    }
    copies_commit();
    ahead += stride;
    to = to == ring + (kQ4Depth - 1) * kStage ? ring : to + kStage;
  };
#pragma unroll
  for (int s = 0; s < kQ4Depth - 1; ++s) copy();
  float acc[kQ4Tiles][4] = {};
  for (; step < a.w.steps; step += stride) {
    copies_wait<kQ4Depth - 2>();
    __syncwarp();  // every lane's copies of this step, and every lane is through with the stage that is filled next
    copy();
    q4_step<T, NG, ZEROS>(acc, from, row_at, lane);
    from = from == ring + (kQ4Depth - 1) * kStage ? ring : from + kStage;
  }
  copies_wait<0>();
#pragma unroll
  for (int t = 0; t < kQ4Tiles; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) parts[warp][2 * (lane & 3) + (c & 1)][kQ4Rows * t + (lane >> 2) + 8 * (c >> 1)] = acc[t][c];
  __syncthreads();
  static_assert(TOKENS * kQ4Cols == kQ4Warps * 32, "a sum per thread");
  float sum = 0.0f;
  float* const mine = &parts[0][0][0] + tid;
#pragma unroll
  for (int v = 0; v < kQ4Warps; ++v) sum += mine[v * TOKENS * kQ4Cols];
  if (a.ranks > 1) {  // the same for the whole grid
    *mine = sum;
    __syncthreads();
    cluster_sync_all();
    if (rank == 0)
      for (int r = 1; r < a.ranks; ++r) sum += load_cluster(mapa_shared(smem_u32(mine), r));
    __syncthreads();
    cluster_sync_all();  // the others' shared memory lives until it has been read
    if (rank != 0) return;
  }
  const int r = tid / kQ4Cols, n = static_cast<int>(tile) * kQ4Rows + tid % kQ4Cols;
  if (r < count && n < a.N) {
    const T v = Elem<T>::from_float(sum);
    a.out[static_cast<int64_t>(row0 + r) * a.N + n] = *reinterpret_cast<const uint16_t*>(&v);
  }
}

// More rows, 8 MT at a time.  A CTA takes eight tiles, two per warp, and the rows; its warps go through the steps together, so that a step's
// columns of the rows lie in shared memory once, and the numbers made of a word are used for all rows.  16, 32, 64 rows of 4096 by 28672: 28,
// 43, 78 us (by eights: 36, 70, 134), the tensor pipe busy for 40 % of it with two warps per scheduler; 9 and 16 rows of 7168 by 4096
// 9.1 and 9.4 (by eights 13.7 and 14.8).  With one tile per warp and twice the CTAs an SM, which read the rows out of shared memory twice as
// often, 84 us for the 64 rows and 10.7 for the 16.  64 and 32 rows take all registers that two (three) CTAs per SM leave, 255 (168), and
// spill 32 to 144 (4 to 32) bytes.
constexpr int kQ4ManyWarps = 4, kQ4ManyDepth = 3;
template <int NG, bool ZEROS, int MT> struct Q4Many {
  static constexpr int kBlock = Q4Stage<NG, ZEROS>::kBlock, kRows = kQ4ManyWarps * kQ4Tiles * kBlock, kStage = kRows + MT * 2048;
  static constexpr int kCols = kQ4ManyWarps * kQ4Cols, kTokens = 8 * MT;
  static constexpr int kSums = kTokens * kCols * 4;  // [token][column], where the stages were
  static constexpr int kTotal = kQ4ManyDepth * kStage > kSums ? kQ4ManyDepth * kStage : kSums;
};
template <typename T, int NG, bool ZEROS, int MT>
__global__ void __launch_bounds__(kQ4ManyWarps * 32, MT == 8 ? 2 : 3) q4_many_kernel(const Q4Args a) {
  using P = Q4Many<NG, ZEROS, MT>;
  extern __shared__ __align__(128) uint8_t stages[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = a.ranks > 1 ? static_cast<int>(blockIdx.x) % a.ranks : 0;
  const int64_t tile = static_cast<int64_t>(blockIdx.x / a.ranks) * (kQ4ManyWarps * kQ4Tiles) + warp * kQ4Tiles;
  const int row0 = blockIdx.y * P::kTokens, count = min(a.rows - row0, P::kTokens);
  const uint8_t* data = a.w.data + tile * a.w.steps * P::kBlock + lane * 16;
  const int64_t apart = tile + 1 < a.w.tiles ? static_cast<int64_t>(a.w.steps) * P::kBlock : 0;
  const int piece = tid & 15, r8 = tid >> 4;  // of the rows: this thread copies one 16-byte piece of rows r8, r8 + 8, ...
  const uint16_t* x = a.x + static_cast<int64_t>(row0 + (r8 < count ? r8 : 0)) * a.K + 8 * piece;
  const uint32_t base = smem_u32(stages), row_to = P::kRows + r8 * 256 + ((piece ^ ((r8 & 1) << 2)) << 4);
  const uint32_t row_at = P::kRows + (lane >> 2) * 256 + (((lane & 3) ^ (((lane >> 2) & 1) << 2)) << 4);
  const auto copy = [&](uint32_t stage, int step) {
    if (step < a.w.steps) {
      if (tile < a.w.tiles) q4_copy<NG, ZEROS>(stage + warp * kQ4Tiles * P::kBlock, data + static_cast<int64_t>(step) * P::kBlock, apart, lane);
      const int at = step * kQ4Step;
      const bool real = at + 8 * piece < a.K;
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (r8 + 8 * m < count) copy_16_or_zeros(stage + row_to + m * 2048, real ? x + static_cast<int64_t>(8 * m) * a.K + at : a.x, real);
    }
    copies_commit();
  };
  float acc[kQ4Tiles][MT][4];
#pragma unroll
  for (int t = 0; t < kQ4Tiles; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m][0] = acc[t][m][1] = acc[t][m][2] = acc[t][m][3] = 0.0f;
#pragma unroll
  for (int s = 0; s < kQ4ManyDepth - 1; ++s) copy(base + s * P::kStage, rank + s * a.ranks);
  uint32_t from = base, spent = base + (kQ4ManyDepth - 1) * P::kStage;
#pragma unroll 1
  for (int step = rank; step < a.w.steps; step += a.ranks) {
    copies_wait<kQ4ManyDepth - 2>();
    __syncthreads();  // everybody's copies of this step, and everybody is through with the stage that is filled next
    copy(spent, step + (kQ4ManyDepth - 1) * a.ranks);
    Q4Piece<NG, ZEROS> p[kQ4Tiles];
#pragma unroll
    for (int t = 0; t < kQ4Tiles; ++t) q4_take<NG, ZEROS>(p[t], from + (warp * kQ4Tiles + t) * P::kBlock, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t n[kQ4Tiles][2][4];
      float scale[kQ4Tiles][2];
#pragma unroll
      for (int t = 0; t < kQ4Tiles; ++t) {
        q4_numbers<T, NG, ZEROS>(n[t], p[t], i);
        scale[t][0] = q4_scale<T>(p[t].scale[0], i * NG / 4);
        scale[t][1] = q4_scale<T>(p[t].scale[1], i * NG / 4);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 b = lds_128(from + (row_at ^ (64 * (i & 1))) + 128 * (i >> 1) + m * 2048);
#pragma unroll
        for (int t = 0; t < kQ4Tiles; ++t) {
          float sum[4];
          mma_16x8x16_first<T>(sum, n[t][0], b.x, b.y);
          mma_16x8x16<T>(sum, n[t][1], b.z, b.w);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[t][m][c] = fmaf(sum[c], scale[t][c >> 1], acc[t][m][c]);
        }
      }
    }
    spent = from;
    from = from == base + (kQ4ManyDepth - 1) * P::kStage ? base : from + P::kStage;
  }
  copies_wait<0>();
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(stages);
#pragma unroll
  for (int t = 0; t < kQ4Tiles; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        sums[(8 * m + 2 * (lane & 3) + (c & 1)) * P::kCols + warp * kQ4Cols + t * kQ4Rows + (lane >> 2) + 8 * (c >> 1)] = acc[t][m][c];
  __syncthreads();
  if (a.ranks > 1) cluster_sync_all();
  // the ranks share out the tokens
  const int n = static_cast<int>(blockIdx.x / a.ranks) * P::kCols + tid;
  for (int t = rank; t < count; t += a.ranks) {
    float v = 0.0f;
    if (a.ranks > 1) {
      for (int r = 0; r < a.ranks; ++r) v += load_cluster(mapa_shared(smem_u32(&sums[t * P::kCols + tid]), r));
    } else {
      v = sums[t * P::kCols + tid];
    }
    if (n < a.N) {
      const T w = Elem<T>::from_float(v);
      a.out[static_cast<int64_t>(row0 + t) * a.N + n] = *reinterpret_cast<const uint16_t*>(&w);
    }
  }
  __syncthreads();
  if (a.ranks > 1) cluster_sync_all();  // the others' shared memory lives until it has been read
}

template <typename Kernel> static int launch_q4(Kernel kernel, std::atomic<bool> (&prepared)[64], const Q4Args& a, int64_t groups, int rows_at_once, int warps,
                                                int smem, cudaStream_t s) {
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !prepared[dev].load(std::memory_order_acquire)) {
    MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) prepared[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * a.ranks), static_cast<unsigned>((a.rows + rows_at_once - 1) / rows_at_once), 1);
  cfg.blockDim = dim3(static_cast<unsigned>(warps * 32), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(a.ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.ranks > 1 ? 1 : 0;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return MOE_OK;
}
// CTAs share a group of tiles while SMs would stay idle and each of them has `least` steps.
static int q4_ranks(int64_t ctas, int64_t wanted, int steps, int least) {
  int ranks = 1;
  while (ranks < 8 && ctas * ranks < wanted && steps >= 2 * least * ranks) ranks *= 2;
  return ranks;
}
template <typename T, int NG, bool ZEROS, int MT> static int launch_q4_many(Q4Args a, cudaStream_t s) {
  static std::atomic<bool> prepared[64];
  const int64_t groups = (a.w.tiles + kQ4ManyWarps * kQ4Tiles - 1) / (kQ4ManyWarps * kQ4Tiles);
  a.ranks = q4_ranks(groups * ((a.rows + 8 * MT - 1) / (8 * MT)), sm_count(), a.w.steps, 2);
  return launch_q4(q4_many_kernel<T, NG, ZEROS, MT>, prepared, a, groups, 8 * MT, kQ4ManyWarps, Q4Many<NG, ZEROS, MT>::kTotal, s);
}
template <typename T, int NG, bool ZEROS> static int launch_q4_rows(Q4Args a, cudaStream_t s) {
  if (a.rows > 32) return launch_q4_many<T, NG, ZEROS, 8>(a, s);
  if (a.rows > 16) return launch_q4_many<T, NG, ZEROS, 4>(a, s);
  if (a.rows > 8) return launch_q4_many<T, NG, ZEROS, 2>(a, s);
  static std::atomic<bool> prepared[64];
  const int64_t pairs = (a.w.tiles + kQ4Tiles - 1) / kQ4Tiles;
  a.ranks = q4_ranks(pairs * ((a.rows + 7) / 8), 2 * sm_count(), a.w.steps, 2 * kQ4Warps);
  return launch_q4(q4_rows_kernel<T, NG, ZEROS>, prepared, a, pairs, 8, kQ4Warps, kQ4Warps * kQ4Ring<NG, ZEROS>, s);
}
template <typename T> static int launch_q4_groups(const Q4Args& a, int group, bool z, cudaStream_t s) {
  if (group == 128) return z ? launch_q4_rows<T, 1, true>(a, s) : launch_q4_rows<T, 1, false>(a, s);
  if (group == 64) return z ? launch_q4_rows<T, 2, true>(a, s) : launch_q4_rows<T, 2, false>(a, s);
  return z ? launch_q4_rows<T, 4, true>(a, s) : launch_q4_rows<T, 4, false>(a, s);
}

// The weights as 16-bit matrices [K, N] (N contiguous), each value times its scale rounded once: for passes of so many rows that 16-bit
// products of whole tiles are cheaper than making the numbers again for every few of them.  GATED: eight rows of the gate and eight of
// the up matrix in turn become columns in turn.  A CTA takes a step of four tiles: 128 rows of the result, 64 columns.
template <typename T, int NG, bool ZEROS, bool GATED>
__global__ void __launch_bounds__(256) q4_expand_kernel(const uint8_t* data, int64_t tiles, int steps, int K, int N, uint16_t* out) {
  constexpr int kBlock = Q4Stage<NG, ZEROS>::kBlock, TILES = 4;
  __shared__ __align__(16) uint8_t blocks[TILES][kBlock];
  const int step = blockIdx.x;
  const int64_t tile0 = static_cast<int64_t>(blockIdx.y) * TILES, matrix = blockIdx.z;
  for (int at = threadIdx.x; at < TILES * (kBlock / 16); at += 256) {
    const int t = at / (kBlock / 16), p = at - t * (kBlock / 16);
    if (tile0 + t < tiles)
      reinterpret_cast<uint4*>(blocks[t])[p] = __ldg(reinterpret_cast<const uint4*>(data + ((matrix * tiles + tile0 + t) * steps + step) * kBlock) + p);
  }
  __syncthreads();
  for (int item = threadIdx.x; item < kQ4Step * TILES * 2; item += 256) {
    const int k = item / (TILES * 2), eight = item % (TILES * 2), t = eight / 2;  // row of the result, eight of its columns
    const int64_t column = tile0 * kQ4Rows + eight * 8;
    if (step * kQ4Step + k >= K || column >= N) continue;
    const int low = k % 8, j = k * NG / kQ4Step;
    const int byte = (k % 32 / 8) * 16 + 4 * (k / 32) + (low % 2) * 2 + low / 4, shift = low % 4 / 2 * 4;
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int of16 = 8 * (eight % 2) + c, row = GATED ? of16 / 2 + 8 * (of16 % 2) : of16;
      const int value = blocks[t][(row / 8 * 32 + 4 * (row % 8)) * 16 + byte] >> shift & 15;
      const int zero = ZEROS ? blocks[t][1024 + 32 * NG + row * NG + j] : 8;
      v[c] = static_cast<float>(value - zero) * Elem<T>::to_float(reinterpret_cast<const T*>(blocks[t] + 1024)[row * NG + j]);
    }
    *reinterpret_cast<uint4*>(out + (matrix * K + step * kQ4Step + k) * N + column) =
        make_uint4(Elem<T>::pack2(v[0], v[1]), Elem<T>::pack2(v[2], v[3]), Elem<T>::pack2(v[4], v[5]), Elem<T>::pack2(v[6], v[7]));
  }
}
template <typename T, int NG, bool ZEROS>
static void launch_q4_expand(const void* data, int64_t matrices, int K, int N, bool gated, void* out, cudaStream_t s) {
  const int64_t tiles = (N + kQ4Rows - 1) / kQ4Rows;
  const int steps = (K + kQ4Step - 1) / kQ4Step;
  const dim3 grid(static_cast<unsigned>(steps), static_cast<unsigned>((tiles + 3) / 4), static_cast<unsigned>(matrices));
  const uint8_t* from = static_cast<const uint8_t*>(data);
  uint16_t* to = static_cast<uint16_t*>(out);
  if (gated) q4_expand_kernel<T, NG, ZEROS, true><<<grid, 256, 0, s>>>(from, tiles, steps, K, N, to);
  else q4_expand_kernel<T, NG, ZEROS, false><<<grid, 256, 0, s>>>(from, tiles, steps, K, N, to);
}
template <typename T> static void launch_q4_expand_groups(const void* data, int64_t matrices, int K, int N, int group, bool z, bool gated, void* out, cudaStream_t s) {
  if (group == 128) z ? launch_q4_expand<T, 1, true>(data, matrices, K, N, gated, out, s) : launch_q4_expand<T, 1, false>(data, matrices, K, N, gated, out, s);
  else if (group == 64) z ? launch_q4_expand<T, 2, true>(data, matrices, K, N, gated, out, s) : launch_q4_expand<T, 2, false>(data, matrices, K, N, gated, out, s);
  else z ? launch_q4_expand<T, 4, true>(data, matrices, K, N, gated, out, s) : launch_q4_expand<T, 4, false>(data, matrices, K, N, gated, out, s);
}

}  // namespace moe

using namespace moe;

extern "C" int moe_int4_matmul(const void* x, const void* data, void* out, int64_t rows, int k_dim, int n_dim, int group, int zeros, int dtype,
                               void* stream) {
  MOE_CHECK_ARG(rows >= 0 && rows <= (1 << 21) && k_dim > 0 && n_dim > 0, "moe_int4_matmul: %lld rows (at most 2^21), K=%d, N=%d",
                static_cast<long long>(rows), k_dim, n_dim);
  MOE_CHECK_ARG(group == 32 || group == 64 || group == 128, "moe_int4_matmul: groups of 32, 64 or 128 columns, got %d", group);
  MOE_CHECK_ARG(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16, "moe_int4_matmul: unknown dtype %d", dtype);
  if (k_dim % 8 != 0 || n_dim % 8 != 0 || k_dim > (1 << 27) || n_dim > (1 << 27)) {
    set_error("moe_int4_matmul: K=%d and N=%d must be multiples of 8 up to 2^27", k_dim, n_dim);
    return MOE_ERR_UNSUPPORTED;
  }
  if (rows == 0) return MOE_OK;
  MOE_CHECK_ARG(x && data && out, "moe_int4_matmul: null pointer argument");
  MOE_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(data)) & 15) == 0, "moe_int4_matmul: pointers must be 16-byte aligned");
  Q4Args a{};
  a.w.data = static_cast<const uint8_t*>(data);
  a.w.tiles = (n_dim + kQ4Rows - 1) / kQ4Rows;
  a.w.steps = (k_dim + kQ4Step - 1) / kQ4Step;
  a.x = static_cast<const uint16_t*>(x);
  a.out = static_cast<uint16_t*>(out);
  a.rows = static_cast<int>(rows);
  a.K = k_dim;
  a.N = n_dim;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_DTYPE_BF16 ? launch_q4_groups<__nv_bfloat16>(a, group, zeros != 0, s) : launch_q4_groups<__half>(a, group, zeros != 0, s);
}

extern "C" int moe_int4_expand(const void* data, void* out, int64_t matrices, int k_dim, int n_dim, int group, int zeros, int gated, int dtype,
                               void* stream) {
  MOE_CHECK_ARG(matrices >= 0 && matrices <= 65535 && k_dim > 0 && n_dim > 0, "moe_int4_expand: %lld matrices (at most 65535), K=%d, N=%d",
                static_cast<long long>(matrices), k_dim, n_dim);
  MOE_CHECK_ARG(group == 32 || group == 64 || group == 128, "moe_int4_expand: groups of 32, 64 or 128 columns, got %d", group);
  MOE_CHECK_ARG(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16, "moe_int4_expand: unknown dtype %d", dtype);
  if (k_dim % 8 != 0 || n_dim % (gated ? 16 : 8) != 0 || k_dim > (1 << 21) || n_dim > (1 << 21)) {
    set_error("moe_int4_expand: K=%d must be a multiple of 8 and N=%d of 8 (gated: 16), up to 2^21", k_dim, n_dim);
    return MOE_ERR_UNSUPPORTED;
  }
  if (matrices == 0) return MOE_OK;
  MOE_CHECK_ARG(data && out, "moe_int4_expand: null pointer argument");
  MOE_CHECK_ARG(((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(out)) & 15) == 0, "moe_int4_expand: pointers must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_DTYPE_BF16) launch_q4_expand_groups<__nv_bfloat16>(data, matrices, k_dim, n_dim, group, zeros != 0, gated != 0, out, s);
  else launch_q4_expand_groups<__half>(data, matrices, k_dim, n_dim, group, zeros != 0, gated != 0, out, s);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}
