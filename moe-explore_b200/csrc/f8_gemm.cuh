// Grouped products of 8-bit rows and 8-bit weights on the tensor cores, a scale per row and 128 columns on one side and per 128 x 128
// block on the other:
//
//   out[r, n] = sum over the blocks b of K:  sx[r, b] * sw[n / 128, b] * sum over k in b: x[r, k] * w[e][n, k]
//
// The inner sums are tcgen05.mma (kind::f8f6f4, e4m3 x e4m3) over one 128-byte-deep stage into an accumulator of their own in TMEM; the
// epilogue warps fetch it, multiply by the two scales and add in fp32 registers while the tensor cores work on the next block.
// (The scales are fp32, not powers of two, so the tensor cores' own block scaling cannot apply them.)
//
// Two kernels, chosen by the sizes (f8_gemm.cu):
//   f8_wide_kernel   rows on the accumulator's lanes: a CTA covers 128 rows x 256 weight rows of one expert, a CTA pair twice the rows
//   f8_lanes_kernel  weights on the lanes: a cluster covers 128 weight rows (of gate AND up where gated) and up to 64 rows of
//                    one expert, each of its CTAs a part of K; for calls with so few of these that SMs would be idle
//
// Operands are described to the copy engine as pairs of bytes (16-bit elements, 64 to a 128-byte swizzle row); loads past an edge
// read zeros, which are zeros in e4m3 too.
#pragma once

#include "f8.cuh"
#include "gemm_kernel.cuh"

#include <type_traits>

namespace moe {

// What a product's results become.
enum F8Out : int {
  F8_ROWS = 0,       // 16-bit rows, element-wise activation
  F8_QUANT = 1,      // 8-bit rows with scales, element-wise activation
  F8_GLU_QUANT = 2,  // 8-bit rows with scales of act(gate) * up; w holds [E][gate, up][I][K]
};

// A product as the host asks for it (f8_gemm.cu).
struct F8Product {
  int kind;  // F8Out
  const void* x;            // [x_rows, K]
  const float* x_scales;    // [x_rows, ceil(K / 128)]
  int64_t x_rows;
  const void* w;            // [E, N, K], gated [E, 2, N, K]
  const float* w_scales;    // [E(, 2), ceil(N / 128), ceil(K / 128)]
  void* out;
  float* out_scales;
  int K, N, num_experts, act, dtype;
  int64_t routed_rows;      // about how many rows there are
  bool maps_before;         // F8Args
  bool dense;
  int compact;
  const int64_t* out_perm;
  int64_t out_rows;
  const int32_t *mtile_expert, *tile_pairs, *num_mtiles, *pad_offsets, *group_indices;
  int32_t* status;
};
int f8_product(const char* name, const F8Product& p, void* stream);

struct F8Args {
  // The rows of the experts: maps of the padded layout, or dense_rows >= 0: one expert, rows 0 .. dense_rows - 1, no maps.
  const int32_t *mtile_expert, *tile_pairs, *num_mtiles, *pad_offsets, *group_indices;
  int64_t dense_rows;
  int32_t padded;        // out has rows for whole tiles: what is stored past an expert's last row is read by nobody
  int32_t compact;       // x and out hold the rows without padding, expert by expert
  int64_t total_rows;    // rows of x
  const float* x_scales;
  const float* w_scales;
  void* out;
  float* out_scales;
  const int64_t* out_perm;  // F8_ROWS: row r of x goes to row out_perm[r] of out (negative: nowhere)
  int64_t out_rows;
  int32_t n_dim;            // columns of out
  int32_t k_dim;
  int32_t act;
  int32_t group_m;
  int32_t maps_before;    // the maps were complete when the kernel before began
  long long wait_limit;
  int32_t* status;
};

// One work item of a CTA: `rows` rows of x from a_row on (0: nothing to do for this CTA of a pair), result columns from n0 on.
struct F8Item {
  int a_row, n0, expert, rows;
  bool valid;
};

// The items of one worker, decoded 32 at a time, one per lane (a chain of dependent loads each), and taken from the lanes in turn.
// Row units (two row tiles of one expert for a CTA pair, one otherwise) are walked in groups of group_m, inside a group column
// tile by column tile, so that the workers running at one time share weight and row tiles in L2.
template <int CTAS> struct F8Walk {
  F8Item mine;
  int first, stride, count, units, nt, rank;
  __device__ __forceinline__ F8Walk(const F8Args& a, int worker, int workers, int cols_per_tile, int rank_)
      : mine{}, first(worker), stride(workers), rank(rank_) {
    nt = (a.n_dim + cols_per_tile - 1) / cols_per_tile;
    units = a.dense_rows >= 0 ? static_cast<int>((a.dense_rows + CTAS * BM - 1) / (CTAS * BM)) : map_word(a.num_mtiles + (CTAS == 2 ? 1 : 0));
    count = units * nt;
  }
  __device__ __forceinline__ F8Item decode(int t, const F8Args& a, int cols_per_tile) const {
    const int groups = (units + a.group_m - 1) / a.group_m;
    const int group_m = (units + groups - 1) / groups;
    const int g = t / (group_m * nt);
    const int rem = t - g * group_m * nt;
    const int gm = min(group_m, units - g * group_m);
    const int n_idx = rem / gm;
    const int unit = g * group_m + rem - n_idx * gm;
    F8Item c;
    c.n0 = n_idx * cols_per_tile;
    c.valid = true;
    if (a.dense_rows >= 0) {
      c.expert = 0;
      c.a_row = (unit * CTAS + rank) * BM;
      const int64_t left = a.dense_rows - c.a_row;
      c.rows = left < 0 ? 0 : left < BM ? static_cast<int>(left) : BM;
      return c;
    }
    int tile = unit;
    bool active = true;
    if (CTAS == 2) {
      const uint32_t info = static_cast<uint32_t>(map_word(a.tile_pairs + unit));
      tile = static_cast<int>(info & 0xFFFFFu);
      c.expert = static_cast<int>((info >> 20) & 0x7FFu);
      if (rank == 1) {
        if (info >> 31) ++tile;
        else active = false;  // reads no rows and stores nothing
      }
    } else {
      c.expert = map_word(a.mtile_expert + unit);
    }
    const int base = map_word(a.pad_offsets + c.expert);
    const int begin = map_word(a.group_indices + c.expert), end = map_word(a.group_indices + c.expert + 1);
    const int inside = tile * BM - base;
    c.a_row = a.compact ? begin + inside : tile * BM;
    int rows = end - begin - inside;
    if (rows > BM) rows = BM;
    if (rows > a.total_rows - c.a_row) rows = static_cast<int>(a.total_rows - c.a_row);  // (whatever the prefix says)
    c.rows = active && rows > 0 && c.a_row >= 0 ? rows : 0;
    return c;
  }
  // What lane `src` decoded.
  __device__ __forceinline__ F8Item held(int src) const {
    F8Item c;
    c.valid = true;
    c.a_row = __shfl_sync(0xFFFFFFFFu, mine.a_row, src);
    c.n0 = __shfl_sync(0xFFFFFFFFu, mine.n0, src);
    c.expert = __shfl_sync(0xFFFFFFFFu, mine.expert, src);
    c.rows = __shfl_sync(0xFFFFFFFFu, mine.rows, src);
    return c;
  }
  __device__ __forceinline__ F8Item get(int i, const F8Args& a, int cols_per_tile) {
    if ((i & 31) == 0) {
      const int t = first + (i + static_cast<int>(threadIdx.x & 31)) * stride;
      if (t < count) mine = decode(t, a, cols_per_tile);
      __syncwarp();
    }
    F8Item c = held(i & 31);
    c.valid = first + i * stride < count;
    return c;
  }
};

// e4m3 x e4m3 -> fp32, both operands K-major: the instruction descriptor without the extents.
constexpr uint32_t kF8Idesc = 1u << 4;
__host__ __device__ constexpr uint32_t f8_idesc(int m, int n) {
  return kF8Idesc | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 lanes x 16 consecutive fp32 columns.
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// Waits for the warp's TMEM loads; the registers pass through, so that nothing that reads them is moved before the wait.
__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
// The same for 32 columns (tmem_ld_32x32 loads them).
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
// The element-wise activation of N registers of a row; the choice is made once, so that the elements interleave.
template <int N, int M> __device__ __forceinline__ void act_row(float (&v)[M], int act, int from = 0) {
  if (act == MOE_ACT_SILU || act == MOE_ACT_SWIGLU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[from + i] = silu_f(v[from + i]);
  } else if (act == MOE_ACT_GELU || act == MOE_ACT_GEGLU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[from + i] = gelu_f(v[from + i]);
  } else if (act == MOE_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[from + i] = gelu_tanh_f(v[from + i]);
  }
}
// Warps: 0 producer, 1 MMA issuer, 2 and 3 none, 4 to 11 epilogue: whole warpgroups, so that the epilogue's take the registers that
// the first one gives back (its own and twice theirs make 3 * 168, what the launch has).
constexpr int kF8Threads = 384;
constexpr int kF8LaunchRegs = 168;
template <int FEW> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW)); }
template <int FEW> __device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"((3 * kF8LaunchRegs - FEW) / 2));
}

constexpr int kF8K = 128;                    // bytes (= elements) of K in one stage: one swizzle row
constexpr int kF8Tile = BM * kF8K;           // 16 KB: 128 rows of an operand
constexpr int kF8MmaK = 32;                  // K of one instruction

// ------------------------------------------------------------------------------------------------------------------
// Rows on the lanes, CTA pairs or CTAs by themselves.
//
// A pair's tile is 256 rows x 256 weight rows (128 gate + 128 up rows where gated); per 128 of K each CTA loads 16 KB of rows and
// 16 KB of weights, and the leader's four instructions (M 256, N 256, K 32) fill one of the two accumulator stages.  A CTA by itself
// has 128 rows x 256 weight rows: as many products and 32 KB of weights; 64 rows or fewer take instructions of M 64.  Either loads no
// more of the rows than there are.  Each of the eight epilogue warps of a CTA owns 32 rows x 128 of the columns: 128 fp32 sums per
// thread, fetched from TMEM 32 at a time, the next 32 on their way while the last are added.  A thread's row is its lane, so a step's
// factor is one register (two where gated).
//
// Bound by TMEM, which the accumulators' writes and the epilogue's reads share, and between 24 and 400 rows per expert by what L2
// hands out: pairs take 2.0 to 2.1 PFLOP/s at 8192 rows (a step of 256 x 256 x 128 in 0.55 us), 1.7 in long runs under the power limit.
// ------------------------------------------------------------------------------------------------------------------
__host__ __device__ constexpr int f8_row_box(int ctas) { return ctas == 2 ? 32 : 16; }  // rows of one copy
template <int CTAS> struct F8WidePlan {
  static constexpr int kStageBytes = (CTAS == 2 ? 2 : 3) * kF8Tile;
  static constexpr int kStages = CTAS == 2 ? 6 : 4;
  static constexpr int kStagingTile = 32 * 128;
  static constexpr int kStagingBytes = kEpilogueWarps * kStagingTile;
  static constexpr int kBarrierBytes = 1024;
  static constexpr int kTotal = kStages * kStageBytes + kStagingBytes + kBarrierBytes + 1024;
  static_assert(kTotal <= 232448, "shared memory");
};

template <typename T, int OUT, int CTAS>
__global__ void __launch_bounds__(kF8Threads, 1)
f8_wide_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
               const __grid_constant__ CUtensorMap tmap_out, const F8Args args) {
  using Plan = F8WidePlan<CTAS>;
  constexpr int kStages = Plan::kStages;
  constexpr bool kGlu = OUT == F8_GLU_QUANT;
  constexpr int kCols = kGlu ? 128 : 256;  // result columns of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t tiles_addr = (raw_addr + 1023u) & ~1023u;
  uint8_t* tiles = smem_raw + (tiles_addr - raw_addr);
  const uint32_t staging_addr = tiles_addr + kStages * Plan::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kStages * Plan::kStageBytes + Plan::kStagingBytes);
  const uint32_t full_bar = smem_u32(bars);                      // [kStages]  (used in the leader CTA)
  const uint32_t empty_bar = smem_u32(bars + kStages);           // [kStages]  (one set per CTA)
  const uint32_t tfull_bar = smem_u32(bars + 2 * kStages);       // [2]        (one set per CTA)
  const uint32_t tempty_bar = smem_u32(bars + 2 * kStages + 2);  // [2]        (used in the leader CTA)
  const uint32_t meet_bar = smem_u32(bars + 2 * kStages + 4);    // [4]        the two warps of a quadrant
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  constexpr bool kPair = CTAS == 2;
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;
  WaitCtx wctx;
  wctx.abort_flag = abort_flag;
  wctx.peer_abort = kPair ? mapa_shared(smem_u32(const_cast<int*>(abort_flag)), static_cast<uint32_t>(rank ^ 1)) : 0;
  wctx.status = args.status;
  wctx.limit = args.wait_limit;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar + 8 * s, CTAS);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar + 8 * a, 1);
      mbar_init(tempty_bar + 8 * a, kEpilogueWarps * CTAS);
    }
    for (int q = 0; q < 4; ++q) mbar_init(meet_bar + 8 * q, 2);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
    if (OUT == F8_ROWS) tma_prefetch_desc(&tmap_out);
  }
  if constexpr (!kPair) {
    // Rows that are not there are multiplied too.  As zeros they cost the least power, which is what a long run of products that stream
    // their weights is short of: 128 tokens x 8 on 64 experts of 7168 x 2048 at the 1000 W limit 558 us per pass at 1.25 GHz with what
    // the memory held, 543 with zeros, 536 with copies of 16 rows instead of 32, 522 at 1.59 GHz with products of 64 rows.
    for (int i = threadIdx.x; i < kStages * kF8Tile / 16; i += kF8Threads) {
      const int st = i / (kF8Tile / 16), at = i % (kF8Tile / 16);
      reinterpret_cast<uint4*>(tiles + st * Plan::kStageBytes)[at] = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int kiters = (args.k_dim + kF8K - 1) / kF8K;

  if (warp >= 4) {
    more_registers<40>();
    await_predecessor();
    F8Walk<CTAS> walk(args, blockIdx.x / CTAS, gridDim.x / CTAS, kCols, rank);
    // ------------------------------ epilogue ----------------------------------
    const int quad = warp & 3;
    const int half = (warp - 4) >> 2;
    const uint32_t tempty_leader = kPair ? mapa_shared(tempty_bar, 0) : tempty_bar;
    // An accumulator stage goes back when this warp has fetched its sums: by an arrival that releases, the same as in the 16-bit
    // kernels, so that the reads before it are over for whoever the barrier lets on.
    const auto give_back = [&](int stage) {
      if constexpr (kPair) mbar_arrive_cluster(tempty_leader + 8 * stage);
      else mbar_arrive(tempty_leader + 8 * stage);
    };
    const uint32_t stage_base = staging_addr + (warp - 4) * Plan::kStagingTile;
    const int kblocks = kiters;
    // first accumulator column of the thread's two groups of 64
    const int col_a = kGlu ? 64 * half : 128 * half;
    const int col_b = kGlu ? 128 + 64 * half : 128 * half + 64;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const int nblocks = (args.n_dim + kF8Block - 1) / kF8Block;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    F8Item c = walk.get(0, args, kCols);
    // The thread's row of the tile.  Products of at most 64 rows leave rows 16 q to 16 q + 15 on the first 16 lanes of quadrant q.
    const auto is_small = [&]() { return !kPair && c.rows <= 64; };
    int r = 0;
    bool here = false, live = false;  // the row exists; some of this warp's rows do
    const auto place = [&]() {
      r = is_small() ? quad * 16 + (lane & 15) : quad * 32 + lane;
      here = r < c.rows && (!is_small() || lane < 16);
      live = (is_small() ? quad * 16 : quad * 32) < c.rows;
    };
    const float *xs = args.x_scales, *wa = args.w_scales, *wb = args.w_scales;
    float x0 = 0.0f, a0 = 0.0f, b0 = 0.0f, x1 = 0.0f, a1 = 0.0f, b1 = 0.0f;
    const auto begin = [&]() {  // the scales of the first two steps of item c
      if (!c.valid) return;
      place();
      if (!live) return;
      const int64_t row = static_cast<int64_t>(c.a_row) + (r < c.rows ? r : c.rows - 1);
      xs = args.x_scales + row * kblocks;
      // (a tile's second block of columns may lie past the last one: its products are zeros, any scale serves)
      const int nb = kGlu ? c.n0 / kF8Block : min(c.n0 / kF8Block + half, nblocks - 1);
      wa = args.w_scales + (static_cast<int64_t>(c.expert) * (kGlu ? 2 : 1) * nblocks + nb) * kblocks;
      wb = wa + static_cast<int64_t>(nblocks) * kblocks;
      x0 = xs[0];
      a0 = wa[0];
      if (kGlu) b0 = wb[0];
      if (kiters > 1) {
        x1 = xs[1];
        a1 = wa[1];
        if (kGlu) b1 = wb[1];
      }
    };
    begin();
    F8Item next;
    for (int i = 0; ok && c.valid; ++i, c = next) {
      place();
      float sum[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
      for (int kb = 0; kb < kiters; ++kb) {
        const float fa = x0 * a0, fb = kGlu ? x0 * b0 : fa;
        x0 = x1;
        a0 = a1;
        b0 = b1;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(tfull_bar + 8 * acc, acc_phase, wctx, DS_TIMEOUT_EPILOGUE))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (live) {
          const uint32_t t0 = tmem_base + lanes + acc * 256;
          uint32_t v[2][32];
          tmem_ld_32x32(t0 + col_a, v[0]);
          tmem_ld_wait32(v[0]);
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            if (ch < 3) {
              tmem_ld_32x32(t0 + (ch == 0 ? col_a + 32 : ch == 1 ? col_b : col_b + 32), v[(ch + 1) & 1]);
            } else {
              // before the last additions: the stage is in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) give_back(acc);
              // (loads behind the arrival, which would wait for them: they are not needed before the step after the next.  8192 rows of
              // 4096 by 14336 columns take 489 us, as with an arrival that releases nothing)
              if (kb + 2 < kiters) {
                x1 = xs[kb + 2];
                a1 = wa[kb + 2];
                if (kGlu) b1 = wb[kb + 2];
              }
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[ch * 32 + j] = fmaf(__uint_as_float(v[ch & 1][j]), ch < 2 ? fa : fb, sum[ch * 32 + j]);
            if (ch < 3) tmem_ld_wait32(v[(ch + 1) & 1]);
          }
        } else {
          if (lane == 0) give_back(acc);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (!ok) break;
      // the next item's scales come while this one's results go (waiting for them then took as long as two steps)
      const F8Item done = c;
      next = walk.get(i + 1, args, kCols);
      c = next;
      begin();
      c = done;
      place();
      if constexpr (OUT == F8_ROWS) {
        if (!live) continue;
        // 64 columns at a time through the warp's staging tile: a tensor copy where all 32 rows are this expert's own (in the padded
        // layout they always are), else, or by a row map, stores of whole 128-byte row segments
        const bool whole = !is_small() && args.out_perm == nullptr && (args.padded || quad * 32 + 32 <= c.rows);
        long long out_row = -1;
        if (!whole && here) {
          out_row = args.out_perm != nullptr ? args.out_perm[c.a_row + r] : c.a_row + r;
          if (out_row >= args.out_rows) out_row = -1;
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int col0 = c.n0 + 128 * half + 64 * g;
          if (col0 >= args.n_dim) break;
          act_row<64>(sum, args.act, g * 64);
          if (lane == 0) bulk_wait_read_all();  // the copy that last read the tile
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint4 u = pack8<T>(sum + g * 64 + 8 * q);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage_base + lane * 128 + ((q ^ (lane & 7)) << 4)), "r"(u.x),
                         "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
          }
          if (whole) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_out, col0, c.a_row + quad * 32, stage_base);
              bulk_commit();
            }
            continue;
          }
          __syncwarp();
          const int ck = lane & 7;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int rr = j * 4 + (lane >> 3);
            const long long to = __shfl_sync(0xFFFFFFFFu, out_row, rr);
            uint4 u;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                         : "r"(stage_base + rr * 128 + ((ck ^ (rr & 7)) << 4)));
            const int col = col0 + ck * 8;
            if (to >= 0 && col < args.n_dim) *reinterpret_cast<uint4*>(static_cast<T*>(args.out) + to * args.n_dim + col) = u;
          }
          __syncwarp();
        }
      } else {
        // 8-bit rows: the block's largest value is this thread's (128 columns of its own), or its and its partner's (64 each)
        uint8_t* out = static_cast<uint8_t*>(args.out);
        const int blocks = nblocks;
        float most = kF8Least;
        constexpr int kMine = kGlu ? 64 : 128;
        if (live) {
          act_row<kMine>(sum, args.act);
          if (kGlu) {
#pragma unroll
            for (int j = 0; j < kMine; ++j) sum[j] *= sum[(64 + j) & 127];
          }
#pragma unroll
          for (int j = 0; j < kMine; ++j) most = fmaxf(most, fabsf(sum[j]));
        }
        if (kGlu) {
          // two places used in turn, so that one meeting of the quadrant's warps is enough
          float* mine = reinterpret_cast<float*>(tiles + kStages * Plan::kStageBytes) + (i & 1) * 256;
          mine[half * 128 + quad * 32 + lane] = most;
          __syncwarp();
          if (lane == 0) mbar_arrive(meet_bar + 8 * quad);
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(meet_bar + 8 * quad, i & 1, wctx, DS_TIMEOUT_EPILOGUE))) break;
          most = fmaxf(most, mine[(half ^ 1) * 128 + quad * 32 + lane]);
        }
        if (here) {
          const float inv = kF8Top / most;
          const int col0 = kGlu ? c.n0 + 64 * half : c.n0 + 128 * half;
          const int64_t to = static_cast<int64_t>(c.a_row) + r;
#pragma unroll
          for (int q = 0; q < kMine / 16; ++q) {
            const int col = col0 + 16 * q;
            if (col < args.n_dim)
              *reinterpret_cast<uint4*>(out + to * args.n_dim + col) =
                  make_uint4(f8x4(sum[16 * q] * inv, sum[16 * q + 1] * inv, sum[16 * q + 2] * inv, sum[16 * q + 3] * inv),
                             f8x4(sum[16 * q + 4] * inv, sum[16 * q + 5] * inv, sum[16 * q + 6] * inv, sum[16 * q + 7] * inv),
                             f8x4(sum[16 * q + 8] * inv, sum[16 * q + 9] * inv, sum[16 * q + 10] * inv, sum[16 * q + 11] * inv),
                             f8x4(sum[16 * q + 12] * inv, sum[16 * q + 13] * inv, sum[16 * q + 14] * inv, sum[16 * q + 15] * inv));
          }
          if ((!kGlu || half == 0) && col0 < args.n_dim) args.out_scales[to * blocks + col0 / kF8Block] = most / kF8Top;
        }
      }
    }
    if (OUT == F8_ROWS && lane == 0) bulk_wait_all();
  } else {
    fewer_registers<40>();
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      // Where the maps are complete before the kernel before (which waited for them itself) lets this one up, the first weights are
      // asked for before the wait for it: that one writes the rows.
      if (!args.maps_before) await_predecessor();
      F8Walk<CTAS> walk(args, blockIdx.x / CTAS, gridDim.x / CTAS, kCols, rank);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t pol = l2_policy_evict_normal();
      const uint32_t full_leader = kPair ? mapa_shared(full_bar, 0) : full_bar;
      constexpr int kBox = f8_row_box(CTAS);
      const auto groups_of = [](const F8Item& c) { return (c.rows + kBox - 1) / kBox; };
      const auto load_weights = [&](int st, int kb, const F8Item& c) {
        const uint32_t sw = tiles_addr + st * Plan::kStageBytes + kF8Tile, fb = full_leader + 8 * st;
        const int wz = kGlu ? 2 * c.expert + rank : c.expert;
        const int wrow = kGlu ? c.n0 : c.n0 + rank * BM;
        if constexpr (kPair) {
          mbar_arrive_expect_tx_cluster(fb, kF8Tile + groups_of(c) * kBox * kF8K);
          tma_load_3d_pair(sw, &tmap_w, kb * (kF8K / 2), wrow, wz, fb, pol);
        } else {
          mbar_arrive_expect_tx(fb, 2 * kF8Tile + groups_of(c) * kBox * kF8K);
          tma_load_3d(sw, &tmap_w, kb * (kF8K / 2), wrow, wz, fb, pol);
          tma_load_3d(sw + kF8Tile, &tmap_w, kb * (kF8K / 2), kGlu ? wrow : wrow + BM, kGlu ? wz + 1 : wz, fb, pol);
        }
      };
      const auto load_rows = [&](int st, int kb, const F8Item& c) {
        const uint32_t sx = tiles_addr + st * Plan::kStageBytes, fb = full_leader + 8 * st;
        // (what the products make of rows that are not there is not stored)
        for (int g = 0; g < groups_of(c); ++g) {
          if constexpr (kPair) tma_load_2d_pair(sx + g * kBox * kF8K, &tmap_x, kb * (kF8K / 2), c.a_row + g * kBox, fb, pol);
          else tma_load_2d(sx + g * kBox * kF8K, &tmap_x, kb * (kF8K / 2), c.a_row + g * kBox, fb, pol);
        }
      };
      for (int i = 0; ok; ++i) {
        const F8Item c = walk.get(i, args, kCols);
        int kb = 0;
        if (i == 0) {
          const int ahead = c.valid ? min(kiters, kStages) : 0;
          if (elect_one())
            for (int st = 0; st < ahead; ++st) load_weights(st, st, c);
          __syncwarp();
          if (args.maps_before) await_predecessor();
          if (elect_one())
            for (int st = 0; st < ahead; ++st) load_rows(st, st, c);
          __syncwarp();
          kb = ahead;
          if ((stage = ahead) == kStages) { stage = 0; phase = 1; }
        }
        if (!c.valid) break;
        for (; kb < kiters; ++kb) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(empty_bar + 8 * stage, phase ^ 1, wctx, DS_TIMEOUT_PRODUCER))) {
            ok = false;
            break;
          }
          if (elect_one()) {
            load_weights(stage, kb, c);
            load_rows(stage, kb, c);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
      grid_release();
      if (!ok || *abort_flag) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies already issued land before the CTA ends
      }
    } else if (warp == 1) {
      // ------------------------------ MMA issuer (leader CTA only) --------------
      if (rank == 0) {
        await_predecessor();
        F8Walk<CTAS> walk(args, blockIdx.x / CTAS, gridDim.x / CTAS, kCols, rank);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int i = 0; ok; ++i) {
          const F8Item c = walk.get(i, args, kCols);
          if (!c.valid) break;
          const uint32_t idesc = f8_idesc(!kPair && c.rows <= 64 ? 64 : CTAS * BM, 256);  // (half the work where half will do)
          for (int kb = 0; kb < kiters; ++kb) {
            // (the operands first: they are there before the accumulator stage is, and a wait that passes takes its 100 cycles too)
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(full_bar + 8 * stage, phase, wctx, DS_TIMEOUT_MMA)) ||
                !__all_sync(0xFFFFFFFFu, mbar_wait(tempty_bar + 8 * acc, acc_phase ^ 1, wctx, DS_TIMEOUT_MMA))) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              const uint32_t sx = tiles_addr + stage * Plan::kStageBytes;
#pragma unroll
              for (int k = 0; k < kF8K / kF8MmaK; ++k) {
                const uint64_t dx = make_desc(sx + k * kF8MmaK, 16, 1024), dw = make_desc(sx + kF8Tile + k * kF8MmaK, 16, 1024);
                if constexpr (kPair) umma_f8_pair(tmem_base + acc * 256, dx, dw, idesc, k != 0 ? 1u : 0u);
                else umma_f8(tmem_base + acc * 256, dx, dw, idesc, k != 0 ? 1u : 0u);
              }
              if constexpr (kPair) {
                umma_commit_pair_both(tfull_bar + 8 * acc);
                umma_commit_pair_both(empty_bar + 8 * stage);
              } else {
                umma_commit(tfull_bar + 8 * acc);
                umma_commit(empty_bar + 8 * stage);
              }
            }
            __syncwarp();
            if (++stage == kStages) { stage = 0; phase ^= 1; }
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
          }
        }
        if (!ok || *abort_flag) {
          for (int i = 0; i < 2000; ++i) __nanosleep(1000);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync_all();  // neither CTA may end while its peer can still touch its memory or barriers
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, kTmemCols);
    else tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Weights on the lanes, K split over a cluster.
//
// An item is 128 result columns (weight rows on the lanes; gate and up rows where gated: two accumulators) x the rows of one expert,
// kF8LaneRows of them at most.  The instruction's N is the rows there are, in steps of 16, and so are the rows loaded per stage:
// with one token a stage is 16 (32) KB of weights and 2 KB of rows.  The CTAs of a cluster have equal parts of K; each leaves its sums
// in its shared memory, and after a meeting of the cluster they share out the rows of the results, adding in the order of K.  Nothing
// goes through global memory, and nobody waits but for its own cluster.
//
// For the smallest calls: few items, which by themselves would leave most SMs without work.  64 rows of 7168 by 4096 columns (32
// items, clusters of 4): 15 us, 29 MB of weights at 2 TB/s; of that 6 us are the launch, the first loads' way and the joining.
// (Items cut wherever a worker's equal share of all steps ended, their parts joined through global memory and a counter: 30 us.)
//
// Epilogue warp w owns the 32 lanes of quadrant w % 4 and every other group of 16 rows.
// ------------------------------------------------------------------------------------------------------------------
constexpr int kF8LaneRows = 64;
constexpr int kF8MostRanks = 8;   // CTAs of a cluster
constexpr int kF8LeastSteps = 4;  // of a CTA; with fewer, what the joining costs is more than the streaming

template <bool GLU> struct F8LanesPlan {
  static constexpr int R = kF8LaneRows;
  static constexpr int kWBytes = (GLU ? 2 : 1) * kF8Tile;
  static constexpr int kStageBytes = kWBytes + R * kF8K;
  static constexpr int kAccCols = (GLU ? 2 : 1) * R;
  static constexpr int kAccs = 4;
  // the scales of as many steps as fit: [step][row], and [matrix][step] of the weights
  static constexpr int kTable = 2048;
  static constexpr int kTableSteps = 128;
  static constexpr int kExtra = (kTable + 2 * kTableSteps) * 4;
  static constexpr int kBarrierBytes = 1024;
  static constexpr int kBudget = 232448 - 1024 - kBarrierBytes - kExtra;
  static constexpr int kStages = kBudget / kStageBytes > 10 ? 10 : kBudget / kStageBytes;
  static constexpr int kTotal = kStages * kStageBytes + kExtra + kBarrierBytes + 1024;
  static_assert(kAccs * kAccCols <= static_cast<int>(kTmemCols), "tensor memory");
  static_assert(kTable >= 16 * R, "scales of 16 steps at least");
  static_assert((GLU ? 2 : 1) * R * 128 * 4 <= kStages * kStageBytes, "the sums lie where the ring was");
};

template <typename T, int OUT>
__global__ void __launch_bounds__(kF8Threads, 1)
f8_lanes_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const F8Args args) {
  constexpr bool kGlu = OUT == F8_GLU_QUANT;
  constexpr int R = kF8LaneRows;
  using Plan = F8LanesPlan<kGlu>;
  constexpr int kStages = Plan::kStages, kAccs = Plan::kAccs;
  constexpr int kMats = kGlu ? 2 : 1;
  constexpr int kChunks = R / 32;  // groups of 16 rows whose sums a warp sees to
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t tiles_addr = (raw_addr + 1023u) & ~1023u;
  uint8_t* tiles = smem_raw + (tiles_addr - raw_addr);
  float* const table = reinterpret_cast<float*>(tiles + kStages * Plan::kStageBytes);
  float* const weight_table = table + Plan::kTable;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kStages * Plan::kStageBytes + Plan::kExtra);
  const uint32_t full_bar = smem_u32(bars);
  const uint32_t empty_bar = smem_u32(bars + kStages);
  const uint32_t tfull_bar = smem_u32(bars + 2 * kStages);
  const uint32_t tempty_bar = smem_u32(bars + 2 * kStages + kAccs);
  const uint32_t meet_bar = smem_u32(bars + 2 * kStages + 2 * kAccs);  // the epilogue warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 2 * kAccs + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  WaitCtx wctx;
  wctx.abort_flag = abort_flag;
  wctx.peer_abort = 0;
  wctx.status = args.status;
  wctx.limit = args.wait_limit;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < kAccs; ++a) {
      mbar_init(tfull_bar + 8 * a, 1);
      mbar_init(tempty_bar + 8 * a, kEpilogueWarps);
    }
    mbar_init(meet_bar, kEpilogueWarps);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int kiters = (args.k_dim + kF8K - 1) / kF8K;
  const int ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int kb0 = kiters * rank / ranks, kb1 = kiters * (rank + 1) / ranks;
  // (the grid has a cluster for every item there could be)
  const auto find_item = [&]() {
    const F8Walk<1> walk(args, 0, 1, 128, 0);
    const int item = static_cast<int>(blockIdx.x) / ranks;
    F8Item c{};
    if (item < walk.count) c = walk.decode(item, args, 128);
    c.rows = min(c.rows, R);
    return c;
  };

  if (warp >= 4) {
    more_registers<72>();
    // ------------------------------ epilogue ----------------------------------
    const int quad = warp & 3;
    const int half = (warp - 4) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const int nblocks = (args.n_dim + kF8Block - 1) / kF8Block;
    int acc = 0, meets = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const auto meet = [&]() {  // of the epilogue warps
      __syncwarp();
      if (lane == 0) mbar_arrive(meet_bar);
      return __all_sync(0xFFFFFFFFu, mbar_wait(meet_bar, meets++ & 1, wctx, DS_TIMEOUT_EPILOGUE));
    };
    await_predecessor();
    const F8Item c = find_item();
    if (c.rows > 0) {
      const float* ws = args.w_scales + (static_cast<int64_t>(c.expert) * kMats * nblocks + c.n0 / kF8Block) * kiters;
      const int rows16 = (c.rows + 15) & ~15;
      float sum[kMats][kChunks][16];
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
        for (int m = 0; m < kMats; ++m)
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[m][ch][j] = 0.0f;
      const int most = min(Plan::kTable / rows16, Plan::kTableSteps);
      int filled = kb0, base = kb0;  // the table holds the scales of steps [base, filled)
      for (int kb = kb0; kb < kb1;) {
        if (kb == filled) {
          if (!meet()) {  // (everyone is done with what it held)
            ok = false;
            break;
          }
          base = kb;
          const int steps = min(kb1 - kb, most);
          filled = kb + steps;
#pragma unroll 1
          for (int rr = warp - 4; rr < c.rows; rr += kEpilogueWarps)
            for (int s = lane; s < steps; s += 32) table[s * rows16 + rr] = args.x_scales[(static_cast<int64_t>(c.a_row) + rr) * kiters + kb + s];
          if (warp < 4 + kMats)
            for (int s = lane; s < steps; s += 32)
              weight_table[(warp - 4) * Plan::kTableSteps + s] = ws[static_cast<int64_t>(warp - 4) * nblocks * kiters + kb + s];
          if (!meet()) {
            ok = false;
            break;
          }
        }
        // Two steps at a time where there are two: a step is a chain of waits (sums there, sums fetched) of about 350 ns, which is what
        // 16 KB of weights take to arrive.
        const int together = kb + 1 < filled && (acc & 1) == 0 ? 2 : 1;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (t < together && ok && !__all_sync(0xFFFFFFFFu, mbar_wait(tfull_bar + 8 * (acc + t), acc_phase, wctx, DS_TIMEOUT_EPILOGUE)))
            ok = false;
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
          const int col = 16 * (2 * ch + half);
          if (col < c.rows) {
            uint32_t v[2][kMats][16];
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (t < together) {
#pragma unroll
                for (int m = 0; m < kMats; ++m) tmem_ld_32x16(tmem_base + lanes + (acc + t) * Plan::kAccCols + m * R + col, v[t][m]);
              }
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (t < together) {
                const float* xs = table + (kb + t - base) * rows16 + col;
                const float a0 = weight_table[kb + t - base], b0 = kGlu ? weight_table[Plan::kTableSteps + kb + t - base] : 0.0f;
                float x[16];
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  const float4 q = *reinterpret_cast<const float4*>(xs + j);
                  x[j] = q.x;
                  x[j + 1] = q.y;
                  x[j + 2] = q.z;
                  x[j + 3] = q.w;
                }
#pragma unroll
                for (int m = 0; m < kMats; ++m) tmem_ld_wait16(v[t][m]);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  sum[0][ch][j] = fmaf(__uint_as_float(v[t][0][j]), x[j] * a0, sum[0][ch][j]);
                  if (kGlu) sum[kMats - 1][ch][j] = fmaf(__uint_as_float(v[t][kMats - 1][j]), x[j] * b0, sum[kMats - 1][ch][j]);
                }
              }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane < together) mbar_arrive(tempty_bar + 8 * (acc + lane));
        kb += together;
        acc += together;
        if (acc == kAccs) { acc = 0; acc_phase ^= 1; }
      }
      if (ok) {
        // (every product that read the ring is complete; its memory takes the sums: [matrix][row][column])
        float* to = reinterpret_cast<float*>(tiles) + quad * 32 + lane;
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
          const int col = 16 * (2 * ch + half);
          if (col >= c.rows) continue;
#pragma unroll
          for (int m = 0; m < kMats; ++m)
#pragma unroll
            for (int j = 0; j < 16; ++j) to[(m * R + col + j) * 128] = sum[m][ch][j];
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // every CTA's sums are there
    // a part of the rows for each CTA, a row (a block of 128 columns) per warp
    const int end = c.rows * (rank + 1) / ranks;
    const int col = c.n0 + 4 * lane;
#pragma unroll 1
    for (int rr = c.rows * rank / ranks + warp - 4; ok && rr < end; rr += kEpilogueWarps) {
      float f[kMats][4];
#pragma unroll
      for (int m = 0; m < kMats; ++m) {
        float4 v[kF8MostRanks];
#pragma unroll
        for (int w = 0; w < kF8MostRanks; ++w)
          if (w < ranks) v[w] = ld_cluster_v4(mapa_shared(tiles_addr + ((m * R + rr) * 128 + 4 * lane) * 4, static_cast<uint32_t>(w)));
#pragma unroll
        for (int j = 0; j < 4; ++j) f[m][j] = 0.0f;
#pragma unroll
        for (int w = 0; w < kF8MostRanks; ++w)
          if (w < ranks) {
            f[m][0] += v[w].x;
            f[m][1] += v[w].y;
            f[m][2] += v[w].z;
            f[m][3] += v[w].w;
          }
      }
      act_row<4>(f[0], args.act);
      if (kGlu) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[0][j] *= f[kMats - 1][j];
      }
      int64_t row = static_cast<int64_t>(c.a_row) + rr;
      if constexpr (OUT == F8_ROWS) {
        if (args.out_perm != nullptr) row = args.out_perm[row];
        if (row >= 0 && row < args.out_rows && col < args.n_dim)
          *reinterpret_cast<uint2*>(static_cast<T*>(args.out) + row * args.n_dim + col) =
              make_uint2(Elem<T>::pack2(f[0][0], f[0][1]), Elem<T>::pack2(f[0][2], f[0][3]));
      } else {
        float most = kF8Least;
#pragma unroll
        for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(f[0][j]));
        most = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most)));  // (non-negative: ordered as integers)
        const float inv = kF8Top / most;
        if (col < args.n_dim)
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(args.out) + row * args.n_dim + col) =
              f8x4(f[0][0] * inv, f[0][1] * inv, f[0][2] * inv, f[0][3] * inv);
        if (lane == 0) args.out_scales[row * nblocks + c.n0 / kF8Block] = most / kF8Top;
      }
    }
  } else {
    fewer_registers<72>();
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      bool ok = true;
      const uint64_t pol = l2_policy_evict_normal();
      // Where the maps are complete before the kernel before (which waited for them itself) lets this one up, the first weights are
      // asked for before the wait for it: that one writes the rows.
      if (!args.maps_before) await_predecessor();
      const F8Item c = find_item();
      const int groups = (c.rows + 15) >> 4;
      const int ahead = c.rows > 0 ? min(kb1 - kb0, kStages) : 0;
      const auto load_weights = [&](int st, int kb) {
        const uint32_t sw = tiles_addr + st * Plan::kStageBytes;
        mbar_arrive_expect_tx(full_bar + 8 * st, Plan::kWBytes + groups * 16 * kF8K);
#pragma unroll
        for (int m = 0; m < kMats; ++m)
          tma_load_3d(sw + m * kF8Tile, &tmap_w, kb * (kF8K / 2), c.n0, kMats * c.expert + m, full_bar + 8 * st, pol);
      };
      const auto load_rows = [&](int st, int kb) {
        const uint32_t sx = tiles_addr + st * Plan::kStageBytes + Plan::kWBytes;
        for (int g = 0; g < groups; ++g) tma_load_2d(sx + g * 16 * kF8K, &tmap_x, kb * (kF8K / 2), c.a_row + 16 * g, full_bar + 8 * st, pol);
      };
      if (elect_one())
        for (int st = 0; st < ahead; ++st) load_weights(st, kb0 + st);
      __syncwarp();
      if (args.maps_before) await_predecessor();
      if (elect_one())
        for (int st = 0; st < ahead; ++st) load_rows(st, kb0 + st);
      __syncwarp();
      int stage = ahead == kStages ? 0 : ahead;
      uint32_t phase = ahead == kStages ? 1 : 0;
      if (c.rows > 0)
        for (int kb = kb0 + ahead; kb < kb1; ++kb) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(empty_bar + 8 * stage, phase ^ 1, wctx, DS_TIMEOUT_PRODUCER))) {
            ok = false;
            break;
          }
          if (elect_one()) {
            load_weights(stage, kb);
            load_rows(stage, kb);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      grid_release();
      if (!ok || *abort_flag) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies already issued land before the CTA ends
      }
    } else if (warp == 1) {
      // ------------------------------ MMA issuer --------------------------------
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      await_predecessor();  // (the limits of the waits below are not to run out on the kernel before)
      const F8Item c = find_item();
      const uint32_t idesc = f8_idesc(BM, (c.rows + 15) & ~15);
      if (c.rows > 0)
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(tempty_bar + 8 * acc, acc_phase ^ 1, wctx, DS_TIMEOUT_MMA)) ||
              !__all_sync(0xFFFFFFFFu, mbar_wait(full_bar + 8 * stage, phase, wctx, DS_TIMEOUT_MMA))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t sw = tiles_addr + stage * Plan::kStageBytes;
#pragma unroll
            for (int m = 0; m < kMats; ++m)
#pragma unroll
              for (int k = 0; k < kF8K / kF8MmaK; ++k)
                umma_f8(tmem_base + acc * Plan::kAccCols + m * R, make_desc(sw + m * kF8Tile + k * kF8MmaK, 16, 1024),
                        make_desc(sw + Plan::kWBytes + k * kF8MmaK, 16, 1024), idesc, k != 0 ? 1u : 0u);
            umma_commit(empty_bar + 8 * stage);
            umma_commit(tfull_bar + 8 * acc);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1; }
          if (++acc == kAccs) { acc = 0; acc_phase ^= 1; }
        }
      if (!ok || *abort_flag) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
      }
    }
    __syncwarp();
    cluster_sync_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA ends while another reads its sums
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace moe
