// A few 16-bit rows by one matrix of 4-bit weights (int4.cuh): out [rows, N] = x [rows, K] @ w [N, K]^T.
//
// A CTA takes two tiles, 32 weight rows, and up to eight rows of x; its eight warps share the steps of K, and where there are few tiles,
// so do the CTAs of a cluster.  Their sums are joined in a fixed order, through shared memory and then the cluster's.
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

template <typename T, int NG, bool ZEROS> static int launch_q4_rows(const Q4Args& a, cudaStream_t s) {
  const auto kernel = q4_rows_kernel<T, NG, ZEROS>;
  constexpr int smem = kQ4Warps * kQ4Ring<NG, ZEROS>;
  static std::atomic<bool> prepared[64];
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !prepared[dev].load(std::memory_order_acquire)) {
    MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) prepared[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.w.tiles + kQ4Tiles - 1) / kQ4Tiles * a.ranks), static_cast<unsigned>((a.rows + 7) / 8), 1);
  cfg.blockDim = dim3(kQ4Warps * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
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
template <typename T> static int launch_q4_groups(const Q4Args& a, int group, bool z, cudaStream_t s) {
  if (group == 128) return z ? launch_q4_rows<T, 1, true>(a, s) : launch_q4_rows<T, 1, false>(a, s);
  if (group == 64) return z ? launch_q4_rows<T, 2, true>(a, s) : launch_q4_rows<T, 2, false>(a, s);
  return z ? launch_q4_rows<T, 4, true>(a, s) : launch_q4_rows<T, 4, false>(a, s);
}

}  // namespace moe

using namespace moe;

extern "C" int moe_int4_matmul(const void* x, const void* data, void* out, int64_t rows, int k_dim, int n_dim, int group, int zeros, int dtype,
                               void* stream) {
  MOE_CHECK_ARG(rows >= 0 && rows <= (1 << 19) && k_dim > 0 && n_dim > 0, "moe_int4_matmul: %lld rows (at most 2^19), K=%d, N=%d",
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
  // CTAs share a pair of tiles while SMs would stay idle and each of their warps has two steps
  const int64_t row_blocks = (rows + 7) / 8;
  a.ranks = 1;
  while (a.ranks < 8 && (a.w.tiles + kQ4Tiles - 1) / kQ4Tiles * row_blocks * a.ranks < 2ll * sm_count() && a.w.steps >= 4 * kQ4Warps * a.ranks) a.ranks *= 2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_DTYPE_BF16 ? launch_q4_groups<__nv_bfloat16>(a, group, zeros != 0, s) : launch_q4_groups<__half>(a, group, zeros != 0, s);
}
