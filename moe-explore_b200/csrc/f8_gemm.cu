// Host side of the 8-bit products: checks, tensor maps, the choice between the two kernels (f8_gemm.cuh), and the row movement
// around them (rows to 8 bits, dispatch to the experts, gather).
#define MOE_GEMM_DEFINE_LAUNCH
#include "f8_gemm.cuh"

namespace moe {

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int CTAS, typename Kernel, typename... Args>
static int launch_f8(Kernel kernel, int threads, int smem, std::atomic<int> (&grids)[64], cudaStream_t s, const Args&... args) {
  LaunchParams lp;
  lp.stream = s;
  lp.max_ctas = 0;
  lp.chained = chained_launches();
  PersistentLaunch l;
  const int rc = configure<CTAS>(l, kernel, smem, grids, lp);
  if (rc != MOE_OK) return rc;
  l.cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  MOE_CUDA(cudaLaunchKernelEx(&l.cfg, kernel, args...));
  return MOE_OK;
}

template <typename T, int OUT, int CTAS>
static int launch_f8_wide_on(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& to, const F8Args& args, cudaStream_t s) {
  static std::atomic<int> grids[64];
  return launch_f8<CTAS>(f8_wide_kernel<T, OUT, CTAS>, kF8Threads, F8WidePlan<CTAS>::kTotal, grids, s, tx, tw, to, args);
}
template <typename T, int OUT>
static int launch_f8_wide(bool pairs, const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& to, const F8Args& args, cudaStream_t s) {
  return pairs ? launch_f8_wide_on<T, OUT, 2>(tx, tw, to, args, s) : launch_f8_wide_on<T, OUT, 1>(tx, tw, to, args, s);
}
// One cluster of `ranks` CTAs per item.
template <typename T, int OUT>
static int launch_f8_lanes(const CUtensorMap& tx, const CUtensorMap& tw, const F8Args& args, int items, int ranks, cudaStream_t s) {
  const auto kernel = f8_lanes_kernel<T, OUT>;
  constexpr int smem = F8LanesPlan<OUT == F8_GLU_QUANT>::kTotal;
  static std::atomic<bool> prepared[64];
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !prepared[dev].load(std::memory_order_acquire)) {
    MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) prepared[dev].store(true, std::memory_order_release);
  }
  PersistentLaunch l;
  l.cfg.gridDim = dim3(static_cast<unsigned>(items * ranks), 1, 1);
  l.cfg.blockDim = dim3(kF8Threads, 1, 1);
  l.cfg.dynamicSmemBytes = smem;
  l.cfg.stream = s;
  l.attr[0].id = cudaLaunchAttributeClusterDimension;
  l.attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  l.attr[0].val.clusterDim.y = 1;
  l.attr[0].val.clusterDim.z = 1;
  l.attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  l.attr[1].val.programmaticStreamSerializationAllowed = 1;
  l.cfg.attrs = l.attr;
  l.cfg.numAttrs = chained_launches() ? 2 : 1;
  MOE_CUDA(cudaLaunchKernelEx(&l.cfg, kernel, tx, tw, args));
  return MOE_OK;
}

// Rows [rows, K] and weights [mats, N, K] in bytes, described as pairs of bytes.
static int f8_maps(CUtensorMap* tx, CUtensorMap* tw, const void* x, int64_t rows, const void* w, int64_t mats, int N, int K, uint32_t row_box) {
  const uint64_t dx[2] = {static_cast<uint64_t>(K / 2), static_cast<uint64_t>(rows)};
  const uint32_t bx[2] = {kF8K / 2, row_box};
  int rc = make_tmap(tx, MOE_DTYPE_BF16, x, 2, dx, bx);
  if (rc != MOE_OK) return rc;
  const uint64_t dw[3] = {static_cast<uint64_t>(K / 2), static_cast<uint64_t>(N), static_cast<uint64_t>(mats)};
  const uint32_t bw[3] = {kF8K / 2, BM, 1};
  return make_tmap(tw, MOE_DTYPE_BF16, w, 3, dw, bw);
}

// The kernel with the weights on the lanes: how many items there can be (an expert each, in blocks of 128 columns) and how many
// CTAs share one; none where it does not serve.  It does for 64 rows in all (what its accumulators hold beside the ring) and no more
// items than SMs: 29 MB of one matrix (7168 x 4096) take 12 us with 1 to 16 rows, 13 with 32 and 16 with 64, and 31 to 32 with rows on
// the lanes, 65 of them or 600; the 2 x 32 items of one token's down products (14336 x 4096) 31
// instead of 63 (as a part of the pass, waiting for the up products included).
struct F8Lanes {
  int items, ranks;
};
static F8Lanes f8_lanes(const F8Product& p) {
  if (p.routed_rows > kF8LaneRows) return {0, 0};
  const int64_t experts = p.dense ? 1 : p.routed_rows < p.num_experts ? p.routed_rows : p.num_experts;
  const int64_t items = experts * ((p.N + 127) / 128);
  if (items > sm_count()) return {0, 0};
  const int kiters = (p.K + kF8K - 1) / kF8K;
  // as many CTAs as leave every one an SM (a cluster lies within a processing cluster of 16 to 20 SMs, so that some stay without)
  int ranks = kF8MostRanks;
  while (ranks > 1 && (items * ranks * 8 > sm_count() * 7 || kiters < ranks * kF8LeastSteps)) ranks /= 2;
  return {static_cast<int>(items), ranks};
}
// Rows on the lanes: pairs of CTAs or single ones.  A pair's 256 rows are more often partly empty, a single CTA takes half as much again
// from L2, and more where rows of K bytes begin inside a line of 128.  Time of single CTAs over that of pairs by rows per expert, the
// geometric mean over shapes (8 to 64 experts, K 720 to 14336, N 1024 to 14336); loads: all the same / 0.5 to 1.5 of the mean /
// exponential, as an unbalanced router leaves them:
//                                   64              128              192              256              384              448              768
//   8 shapes of K % 128 == 0   .78 .74 .76     .79 .91 .84    1.06 .92 .86    1.08 .94 .92     .88 .96 .96    1.07 .97 .99    1.09 1.00 .97
//   6 others                   .81 .77 .82     .85 1.06 .98   1.25 1.11 1.03  1.24 1.16 1.14   1.09 1.19 1.16 1.29 1.21 1.23  1.34 1.31 1.29
// Over the three loads they meet at about 430 (.94 at 384, 1.01 at 448) and 144 (.96 at 128, 1.13 at 192) rows per expert.  One matrix
// of 7168 x 4096 takes 35 / 29 us with 128 rows and 36 / 31 with 512.
static bool f8_in_pairs(const F8Product& p) {
  const int64_t mean = p.routed_rows / p.num_experts;
  return mean > (p.num_experts == 1 ? 64 : p.K % 128 == 0 ? 432 : 144);
}

int f8_product(const char* name, const F8Product& p, void* stream) {
  MOE_CHECK_ARG(p.x && p.x_scales && p.w && p.w_scales && p.out, "%s: null pointer argument", name);
  MOE_CHECK_ARG(aligned16(p.x) && aligned16(p.w) && aligned16(p.out), "%s: pointers must be 16-byte aligned", name);
  MOE_CHECK_ARG(p.K > 0 && p.N > 0 && p.num_experts > 0 && p.x_rows > 0, "%s: K=%d N=%d E=%d and %lld rows must be positive", name, p.K,
                p.N, p.num_experts, static_cast<long long>(p.x_rows));
  const bool glu = p.kind == F8_GLU_QUANT;
  if (p.K % 16 != 0 || p.N % (p.kind == F8_ROWS ? 8 : 16) != 0 || p.x_rows > 0x7FFFFF00) {
    set_error("%s: K=%d must be a multiple of 16 and N=%d of 8 (of 16 for 8-bit results): rows are 16-byte aligned", name, p.K, p.N);
    return MOE_ERR_UNSUPPORTED;
  }
  MOE_CHECK_ARG(p.dtype == MOE_DTYPE_BF16 || p.dtype == MOE_DTYPE_F16, "%s: unknown dtype %d", name, p.dtype);
  MOE_CHECK_ARG(glu ? (p.act == MOE_ACT_SWIGLU || p.act == MOE_ACT_GEGLU)
                    : (p.act == MOE_ACT_NONE || p.act == MOE_ACT_SILU || p.act == MOE_ACT_GELU || p.act == MOE_ACT_GELU_TANH),
                "%s: activation %d does not fit the weights", name, p.act);
  MOE_CHECK_ARG(p.kind == F8_ROWS || p.out_scales != nullptr, "%s: 8-bit results have scales", name);
  MOE_CHECK_ARG(p.dense || (p.mtile_expert && p.tile_pairs && p.num_mtiles && p.pad_offsets && p.group_indices),
                "%s: null pointer argument", name);
  F8Args a{};
  a.mtile_expert = p.mtile_expert;
  a.tile_pairs = p.tile_pairs;
  a.num_mtiles = p.num_mtiles;
  a.pad_offsets = p.pad_offsets;
  a.group_indices = p.group_indices;
  a.dense_rows = p.dense ? p.x_rows : -1;
  a.compact = p.compact;
  a.padded = !p.compact && !p.dense;
  a.total_rows = p.x_rows;
  a.x_scales = p.x_scales;
  a.w_scales = p.w_scales;
  a.out = p.out;
  a.out_scales = p.out_scales;
  a.out_perm = p.out_perm;
  a.out_rows = p.out_perm != nullptr ? p.out_rows : p.x_rows;
  a.n_dim = p.N;
  a.k_dim = p.K;
  a.act = p.act;
  a.group_m = kDefaultGroupM;
  a.wait_limit = wait_limit_cycles();
  a.status = p.status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  a.maps_before = p.dense || p.maps_before;
  const F8Lanes lanes = f8_lanes(p);
  const bool pairs = f8_in_pairs(p);
  CUtensorMap tx, tw;
  const int rc = f8_maps(&tx, &tw, p.x, p.x_rows, p.w, static_cast<int64_t>(p.num_experts) * (glu ? 2 : 1), p.N, p.K,
                         lanes.items > 0 ? 16 : f8_row_box(pairs ? 2 : 1));
  if (rc != MOE_OK) return rc;
  const bool bf16 = p.dtype == MOE_DTYPE_BF16;
  if (lanes.items == 0) {
    CUtensorMap to = tx;
    if (p.kind == F8_ROWS && p.out_perm == nullptr) {
      const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.x_rows)};
      const uint32_t box[2] = {64, 32};
      const int rc2 = make_tmap(&to, p.dtype, p.out, 2, dims, box);
      if (rc2 != MOE_OK) return rc2;
    }
    if (p.kind == F8_GLU_QUANT) return launch_f8_wide<__nv_bfloat16, F8_GLU_QUANT>(pairs, tx, tw, to, a, s);
    if (p.kind == F8_QUANT) return launch_f8_wide<__nv_bfloat16, F8_QUANT>(pairs, tx, tw, to, a, s);
    return bf16 ? launch_f8_wide<__nv_bfloat16, F8_ROWS>(pairs, tx, tw, to, a, s) : launch_f8_wide<__half, F8_ROWS>(pairs, tx, tw, to, a, s);
  }
  if (p.kind == F8_GLU_QUANT) return launch_f8_lanes<__nv_bfloat16, F8_GLU_QUANT>(tx, tw, a, lanes.items, lanes.ranks, s);
  if (p.kind == F8_QUANT) return launch_f8_lanes<__nv_bfloat16, F8_QUANT>(tx, tw, a, lanes.items, lanes.ranks, s);
  return bf16 ? launch_f8_lanes<__nv_bfloat16, F8_ROWS>(tx, tw, a, lanes.items, lanes.ranks, s)
              : launch_f8_lanes<__half, F8_ROWS>(tx, tw, a, lanes.items, lanes.ranks, s);
}

// ---- rows to 8 bits, and their way to the experts ----
// Eight lanes share a block of 128 columns (16 each).  Every source block is read once and written to `copies` rows:
//   dst_row == nullptr: row t;  otherwise rows dst_row[t * copies + s] (negative: none).
template <typename T> __device__ __forceinline__ void to_floats(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Elem<T>::unpack2(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// T: a 16-bit type (rows are converted) or uint8_t (8-bit rows with `scales_in` are copied).
// A warp takes four blocks of a row at a time, 16 values per lane, so that the row and where it goes are the whole warp's; the next ones
// are on their way meanwhile.  Everything that counts is 32 bits wide (the host keeps rows x blocks below 2^31) and advances by
// additions.
constexpr int kF8RowsCtas = 4;  // per SM
template <typename T>
__global__ void __launch_bounds__(256, kF8RowsCtas)
f8_rows_kernel(const T* x, const float* scales_in, const int32_t* dst_row, int copies, uint4* out, float* scales, int rows, int cols) {
  await_predecessor();  // before the release: what comes up next reads the routing metadata
  grid_release();
  const int blocks = (cols + kF8Block - 1) / kF8Block;
  const int units = (blocks + 3) / 4;
  const int vecs = cols / 16;
  const int lane = threadIdx.x & 31;
  const int stride = static_cast<int>(gridDim.x) * 8;
  const int stride_rows = stride / units, stride_units = stride - stride_rows * units;
  const int first = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  int row = first / units, unit = first - row * units;
  struct Piece {
    uint4 a, b;
  };
  const auto load = [&](int r, int v) {
    Piece p{};
    if (r < rows && v < vecs) {
      const int64_t at = static_cast<int64_t>(r) * vecs + v;
      if constexpr (sizeof(T) == 2) {
        p.a = reinterpret_cast<const uint4*>(x)[2 * at];
        p.b = reinterpret_cast<const uint4*>(x)[2 * at + 1];
      } else {
        p.a = reinterpret_cast<const uint4*>(x)[at];
      }
    }
    return p;
  };
  Piece next = load(row, unit * 32 + lane);
  while (row < rows) {
    const Piece u = next;
    const int this_row = row, v = unit * 32 + lane;
    row += stride_rows;
    if ((unit += stride_units) >= units) {
      unit -= units;
      ++row;
    }
    next = load(row, unit * 32 + lane);
    const int block = v >> 3;
    const bool ok = v < vecs, has_scale = (lane & 7) == 0 && block < blocks;
    uint4 q;
    float scale;
    if constexpr (sizeof(T) == 2) {
      float f[16];
      to_floats<T>(u.a, f);
      to_floats<T>(u.b, f + 8);
      float most = kF8Least;
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(f[i]));
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
      f8_quotients(f, most);
      q = make_uint4(f8x4(f[0], f[1], f[2], f[3]), f8x4(f[4], f[5], f[6], f[7]), f8x4(f[8], f[9], f[10], f[11]),
                     f8x4(f[12], f[13], f[14], f[15]));
      scale = most / kF8Top;
    } else {
      q = u.a;
      scale = has_scale ? scales_in[static_cast<int64_t>(this_row) * blocks + block] : 0.0f;
    }
    const auto put = [&](int to) {
      if (ok) out[static_cast<int64_t>(to) * vecs + v] = q;
      if (has_scale) scales[static_cast<int64_t>(to) * blocks + block] = scale;
    };
    if (dst_row == nullptr) {
      put(this_row);
      continue;
    }
    // the rows it goes to, one per lane: asked for at once
    for (int s0 = 0; s0 < copies; s0 += 32) {
      const int mine = s0 + lane < copies ? dst_row[static_cast<int64_t>(this_row) * copies + s0 + lane] : -1;
      const int some = min(copies - s0, 32);
      for (int s = 0; s < some; ++s) {
        const int to = __shfl_sync(0xFFFFFFFFu, mine, s);
        if (to >= 0) put(to);
      }
    }
  }
}

// Row r of the result is row index[r] / div of the 8-bit source (zeros where negative or past its end).
__global__ void __launch_bounds__(256)
f8_gather_kernel(const uint2* x, const float* scales_in, const int64_t* index, int div, int64_t x_rows, uint2* out, float* scales, int64_t rows,
                 int cols) {
  await_predecessor();
  grid_release();
  const int blocks = (cols + kF8Block - 1) / kF8Block;
  const int vecs = cols / 8;
  const int lane16 = threadIdx.x & 15;
  const int64_t total = rows * blocks;
  for (int64_t g = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / 16; g < total; g += static_cast<int64_t>(gridDim.x) * 16) {
    const int64_t r = g / blocks;
    const int b = static_cast<int>(g - r * blocks);
    const int v = b * 16 + lane16;
    const int64_t j = index[r];
    const int64_t from = j < 0 || j / div >= x_rows ? -1 : j / div;
    if (v < vecs) out[r * vecs + v] = from >= 0 ? x[from * vecs + v] : make_uint2(0, 0);
    if (lane16 == 0) scales[r * blocks + b] = from >= 0 ? scales_in[from * blocks + b] : 0.0f;
  }
}

static int f8_row_grid(int64_t rows, int cols) {
  const int64_t want = (rows * ((cols + kF8Block - 1) / kF8Block) + 15) / 16;
  const int64_t most = 8ll * sm_count();
  return static_cast<int>(want < most ? want : most);
}

int f8_rows(const char* name, const void* x, const float* x_scales, const int32_t* dst_row, int copies, void* out, float* scales,
            int64_t rows, int cols, int dtype, void* stream) {
  MOE_CHECK_ARG(rows >= 0 && cols > 0 && copies > 0, "%s: negative or zero size", name);
  if (cols % 16 != 0) {
    set_error("%s: 8-bit rows have a multiple of 16 columns, got %d", name, cols);
    return MOE_ERR_UNSUPPORTED;
  }
  if (rows == 0) return MOE_OK;
  if (rows * ((cols + kF8Block - 1) / kF8Block) > 0x7FFFFFFF - kF8RowsCtas * 16ll * sm_count()) {
    set_error("%s: at most 2^31 blocks of 128 columns are supported, got %lld rows of %d", name, static_cast<long long>(rows), cols);
    return MOE_ERR_UNSUPPORTED;
  }
  MOE_CHECK_ARG(x && out && scales, "%s: null pointer argument", name);
  MOE_CHECK_ARG(aligned16(x) && aligned16(out), "%s: pointers must be 16-byte aligned", name);
  MOE_CHECK_ARG(x_scales != nullptr || dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16, "%s: unknown dtype %d", name, dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t want = (rows * ((cols + 4 * kF8Block - 1) / (4 * kF8Block)) + 7) / 8, most = static_cast<int64_t>(kF8RowsCtas) * sm_count();
  const int grid = static_cast<int>(want < most ? want : most);
  uint4* o = static_cast<uint4*>(out);
  if (x_scales != nullptr)
    MOE_CUDA(launch_kernel(f8_rows_kernel<uint8_t>, grid, 256, s, static_cast<const uint8_t*>(x), x_scales, dst_row, copies, o, scales, static_cast<int>(rows), cols));
  else if (dtype == MOE_DTYPE_BF16)
    MOE_CUDA(launch_kernel(f8_rows_kernel<__nv_bfloat16>, grid, 256, s, static_cast<const __nv_bfloat16*>(x), x_scales, dst_row, copies, o, scales, static_cast<int>(rows), cols));
  else
    MOE_CUDA(launch_kernel(f8_rows_kernel<__half>, grid, 256, s, static_cast<const __half*>(x), x_scales, dst_row, copies, o, scales, static_cast<int>(rows), cols));
  return MOE_OK;
}

static bool glu(int act) { return act == MOE_ACT_SWIGLU || act == MOE_ACT_GEGLU; }

}  // namespace moe

using namespace moe;

extern "C" int moe_f8_quantize_rows(const void* x, void* q, float* scales, int64_t num_rows, int cols, int dtype, void* stream) {
  return f8_rows("moe_f8_quantize_rows", x, nullptr, nullptr, 1, q, scales, num_rows, cols, dtype, stream);
}

extern "C" size_t moe_f8_pass_size(void) { return sizeof(moe_f8_pass); }

extern "C" int moe_f8_expert_forward(const moe_f8_pass* p, int steps, void* stream) {
  MOE_CHECK_ARG(p != nullptr, "moe_f8_expert_forward: null pointer argument");
  MOE_CHECK_ARG(p->num_tokens > 0 && p->topk > 0 && p->num_experts > 0 && p->d > 0 && p->inter > 0, "moe_f8_expert_forward: bad sizes");
  const int64_t rows = p->num_tokens * p->topk;
  MOE_CHECK_ARG(p->padded_rows == moe_padded_rows_bound(rows, p->num_experts), "moe_f8_expert_forward: padded_rows is not the bound of %lld rows",
                static_cast<long long>(rows));
  if (p->d % 16 != 0 || p->inter % 16 != 0) {
    set_error("moe_f8_expert_forward: d=%d and inter=%d must be multiples of 16", p->d, p->inter);
    return MOE_ERR_UNSUPPORTED;
  }
  // (the steps by themselves take a null map for "rows stay where they are")
  MOE_CHECK_ARG(p->dst_row != nullptr || !(steps & (MOE_F8_ROUTE | MOE_F8_DISPATCH | MOE_F8_FOLD)), "moe_f8_expert_forward: null pointer argument");
  const Chain chain;
  if (steps & MOE_F8_ROUTE)
    MOE_STEP(routing_metadata(p->expert_idx, rows, p->num_experts, p->group_indices, nullptr, p->pad_offsets, p->row_src, p->dst_row,
                              p->mtile_expert, p->tile_pairs, p->num_mtiles, p->status, p->workspace, p->workspace_bytes, false, stream));
  if (steps & MOE_F8_DISPATCH)
    MOE_STEP(f8_rows("moe_f8_expert_forward", p->x, p->x_scales, p->dst_row, p->topk, p->xs, p->xs_scales, p->num_tokens, p->d, p->dtype,
                     stream));
  F8Product g{};
  g.x_rows = p->padded_rows;
  g.routed_rows = rows;
  g.num_experts = p->num_experts;
  g.dtype = p->dtype;
  g.mtile_expert = p->mtile_expert;
  g.tile_pairs = p->tile_pairs;
  g.num_mtiles = p->num_mtiles;
  g.pad_offsets = p->pad_offsets;
  g.group_indices = p->group_indices;
  g.status = p->status;
  if (steps & MOE_F8_UP) {
    g.kind = glu(p->act) ? F8_GLU_QUANT : F8_QUANT;
    g.maps_before = !(steps & MOE_F8_ROUTE) || (steps & MOE_F8_DISPATCH);  // by an earlier call, or with a kernel between
    g.x = p->xs;
    g.x_scales = p->xs_scales;
    g.w = p->w1;
    g.w_scales = p->w1_scales;
    g.out = p->hidden;
    g.out_scales = p->hidden_scales;
    g.K = p->d;
    g.N = p->inter;
    g.act = p->act;
    MOE_STEP(f8_product("moe_f8_expert_forward", g, stream));
  }
  if (steps & MOE_F8_DOWN) {
    g.kind = F8_ROWS;
    g.maps_before = !(steps & MOE_F8_ROUTE) || (steps & (MOE_F8_DISPATCH | MOE_F8_UP));
    g.x = p->hidden;
    g.x_scales = p->hidden_scales;
    g.w = p->w2;
    g.w_scales = p->w2_scales;
    g.out = p->ys;
    g.out_scales = nullptr;
    g.K = p->inter;
    g.N = p->d;
    g.act = MOE_ACT_NONE;
    MOE_STEP(f8_product("moe_f8_expert_forward", g, stream));
  }
  if (steps & MOE_F8_FOLD)
    MOE_STEP(combine_topk(p->ys, p->scores, p->dst_row, p->out, p->num_tokens, p->topk, p->d, p->dtype, p->addend, nullptr, nullptr,
                          nullptr, stream));
  return MOE_OK;
}

extern "C" size_t moe_f8_rows_pass_size(void) { return sizeof(moe_f8_rows_pass); }

extern "C" int moe_f8_rows_gemm(const moe_f8_rows_pass* p, int steps, void* stream) {
  MOE_CHECK_ARG(p != nullptr, "moe_f8_rows_gemm: null pointer argument");
  MOE_CHECK_ARG(p->num_rows > 0 && p->x_rows > 0 && p->num_experts > 0 && p->k_dim > 0 && p->topk > 0, "moe_f8_rows_gemm: bad sizes");
  const bool dense = p->group_indices == nullptr;
  MOE_CHECK_ARG(!dense || (p->num_experts == 1 && !p->gather && !p->scatter && p->x_rows == p->num_rows),
                "moe_f8_rows_gemm: rows without a group prefix are those of one expert, in their order");
  MOE_CHECK_ARG(p->gather || p->x_rows >= p->num_rows, "moe_f8_rows_gemm: %lld rows of %lld", static_cast<long long>(p->num_rows),
                static_cast<long long>(p->x_rows));
  MOE_CHECK_ARG(dense || (p->pad_offsets && p->mtile_expert && p->tile_pairs && p->num_mtiles), "moe_f8_rows_gemm: null pointer argument");
  MOE_CHECK_ARG(!(p->gather || p->scatter) || p->perm != nullptr, "moe_f8_rows_gemm: null pointer argument");
  MOE_CHECK_ARG(!p->gather || (p->gathered != nullptr && p->gathered_scales != nullptr && p->x != nullptr && p->x_scales != nullptr),
                "moe_f8_rows_gemm: null pointer argument");
  const Chain chain;
  if ((steps & MOE_ROWS_LAYOUT) && !dense)
    MOE_STEP(moe_layout_from_groups(p->group_indices, p->num_rows, p->num_experts, p->pad_offsets, nullptr, nullptr, p->mtile_expert,
                                    p->tile_pairs, p->num_mtiles, p->status, stream));
  if ((steps & MOE_ROWS_GATHER) && p->gather) {
    if (p->k_dim % 16 != 0) {
      set_error("moe_f8_rows_gemm: 8-bit rows have a multiple of 16 columns, got %d", p->k_dim);
      return MOE_ERR_UNSUPPORTED;
    }
    MOE_CHECK_ARG(aligned16(p->x) && aligned16(p->gathered), "moe_f8_rows_gemm: pointers must be 16-byte aligned");
    MOE_CUDA(launch_kernel(f8_gather_kernel, f8_row_grid(p->num_rows, p->k_dim), 256, static_cast<cudaStream_t>(stream),
                           static_cast<const uint2*>(p->x), p->x_scales, p->perm, p->topk, p->x_rows, static_cast<uint2*>(p->gathered),
                           p->gathered_scales, p->num_rows, p->k_dim));
    chained_launches() = true;
  }
  if (steps & MOE_ROWS_GEMM) {
    F8Product g{};
    g.kind = F8_ROWS;
    g.x = p->gather ? p->gathered : p->x;
    g.x_scales = p->gather ? p->gathered_scales : p->x_scales;
    g.x_rows = p->num_rows;
    g.routed_rows = p->num_rows;
    g.w = p->w;
    g.w_scales = p->w_scales;
    g.out = p->out;
    g.K = p->k_dim;
    g.N = p->n_dim;
    g.num_experts = p->num_experts;
    g.act = p->act;
    g.dtype = p->dtype;
    g.dense = dense;
    g.compact = 1;
    g.out_perm = p->scatter ? p->perm : nullptr;
    g.out_rows = p->num_rows;
    g.mtile_expert = p->mtile_expert;
    g.tile_pairs = p->tile_pairs;
    g.num_mtiles = p->num_mtiles;
    g.pad_offsets = p->pad_offsets;
    g.group_indices = p->group_indices;
    g.status = p->status;
    MOE_STEP(f8_product("moe_f8_rows_gemm", g, stream));
  }
  return MOE_OK;
}
