// A whole layer for up to 16 tokens in two kernels, with experts in 16 or 4 bits:
//
//   first:   h = round(x + residual), r = 1 / sqrt(mean h^2 + eps), y = round(h r w);  logits = (h r w) W_router, in fp32
//   second:  scores and experts of every token (each CTA for itself);  hidden = round(act(y W1[e])) for the chosen experts;
//            rows = hidden W2[e] in fp32;  out = round(sum over the slots of score * row + addend)
//
// Bound by reading the chosen experts' weights once.  The second kernel is one resident wave (a cooperative launch, so that its CTAs may
// wait for one another): between its three phases they meet at a counter in global memory that the first kernel has set to zero.
// Every sum has a fixed order: nothing depends on timing.
//
// The logits are not rounded to 16 bits, nor are an expert's rows before the fold; y and the activated product are, because they are
// operands of 16-bit products.
#include "int4.cuh"

#include <atomic>

namespace moe {

constexpr int kFewTokens = 16;
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewSlots = 512;      // tokens x slots
constexpr int kFewExperts = 1024, kFewGroups = 64;
constexpr int kFewCtas = 2;         // per SM
constexpr int kFewParts = 4;        // shares of the down product's depth, at most

// ---------------------------------------------------------------------------------------------------- norm and logits
constexpr int kHeadRanks = 8;       // CTAs of a cluster share the hidden size
constexpr int kHeadCols = 32;       // experts of a cluster
constexpr int kHeadRows = 256;      // hidden columns at a time

struct HeadArgs {
  const void *x, *residual, *norm;  // residual, norm: or null
  const void* router;               // [d, E] or null: no logits
  void *stream, *y;                 // [T, d] or null
  float* logits;                    // [T, E]
  uint32_t* meeting;                // words of the second kernel, set to zero
  int T, d, E, norm_fp32;
  float eps;
};

__device__ __forceinline__ float cluster_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ double cluster_load_double(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T> __device__ __forceinline__ float to_f32(T v) { return Elem<T>::to_float(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }

// Four weights of a router row (fewer at its end), one load where rows are aligned for it.
template <typename W> __device__ __forceinline__ void router_row(const W* p, int left, bool whole, float (&f)[4]) {
  if (whole) {
    if constexpr (sizeof(W) == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p));
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      const float2 a = Elem<W>::unpack2(v.x), b = Elem<W>::unpack2(v.y);
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) f[c] = c < left ? to_f32<W>(p[c]) : 0.0f;
  }
}

// A cluster takes 32 experts' columns, its CTAs an eighth of the hidden size each; a thread four columns and every 32nd hidden row.
// Norm and logits in one pass over x: the logits are linear in r, which is known when all have met.
template <typename T, typename W, int TT>
__global__ void __launch_bounds__(kFewThreads) few_head_kernel(const HeadArgs a) {
  __shared__ float rows[TT][kHeadRows];
  __shared__ float parts[kFewWarps][TT][kHeadCols];
  __shared__ float joined[TT][kHeadCols];
  __shared__ double squares[kFewTokens], square_parts[kFewWarps][TT];
  __shared__ float scale[kFewTokens];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int col0 = static_cast<int>(blockIdx.x / kHeadRanks) * kHeadCols;
  const bool first = blockIdx.x < kHeadRanks;  // the cluster that writes stream and y
  if (blockIdx.x == 0 && tid < 2) a.meeting[tid] = 0;
  const int share = (a.d + kHeadRanks * 8 - 1) / (kHeadRanks * 8) * 8;
  const int k_begin = min(rank * share, a.d), k_end = min(k_begin + share, a.d);
  const T* x = static_cast<const T*>(a.x);
  const T* residual = static_cast<const T*>(a.residual);
  const int cv = tid & 7, kl = tid >> 3;  // columns col0 + 4 cv + 0..3, hidden rows kl + 32 i
  const int left = a.E - (col0 + 4 * cv);
  const bool whole = left >= 4 && (a.E & 3) == 0;
  const auto norm_weight = [&](int k) {
    return a.norm == nullptr ? 1.0f : a.norm_fp32 ? static_cast<const float*>(a.norm)[k] : to_f32<T>(static_cast<const T*>(a.norm)[k]);
  };
  float acc[TT][4];
  double sq[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.0f;
    sq[t] = 0.0;
  }
  for (int k0 = k_begin; k0 < k_end; k0 += kHeadRows) {
    float w[kHeadRows / 32][4];
#pragma unroll
    for (int i = 0; i < kHeadRows / 32; ++i) {
      const int k = k0 + kl + 32 * i;
      if (a.router != nullptr && k < k_end && left > 0) router_row<W>(static_cast<const W*>(a.router) + static_cast<int64_t>(k) * a.E + col0 + 4 * cv, left, whole, w[i]);
      else w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0.0f;
    }
    const int k = k0 + tid;
    const float g = k < k_end ? norm_weight(k) : 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float h = 0.0f;
      if (t < a.T && k < k_end) {
        h = to_f32<T>(x[static_cast<int64_t>(t) * a.d + k]);
        if (residual != nullptr) {
          const T v = Elem<T>::from_float(h + to_f32<T>(residual[static_cast<int64_t>(t) * a.d + k]));
          if (first) static_cast<T*>(a.stream)[static_cast<int64_t>(t) * a.d + k] = v;
          h = to_f32<T>(v);
        }
        sq[t] += static_cast<double>(h) * h;  // (bf16 values' squares may leave fp32)
      }
      rows[t][tid] = h * g;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kHeadRows / 32; ++i) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float h = rows[t][kl + 32 * i];
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[t][c] = fmaf(h, w[i][c], acc[t][c]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      acc[t][c] += __shfl_xor_sync(0xFFFFFFFFu, acc[t][c], 8);
      acc[t][c] += __shfl_xor_sync(0xFFFFFFFFu, acc[t][c], 16);
      if (lane < 8) parts[warp][t][4 * cv + c] = acc[t][c];
    }
    if (a.norm != nullptr) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sq[t] += __shfl_xor_sync(0xFFFFFFFFu, sq[t], off);
      if (lane == 0) square_parts[warp][t] = sq[t];
    }
  }
  __syncthreads();
  for (int at = tid; at < TT * kHeadCols; at += kFewThreads) {
    float v = 0.0f;
    for (int w = 0; w < kFewWarps; ++w) v += (&parts[w][0][0])[at];
    (&joined[0][0])[at] = v;
  }
  if (a.norm != nullptr && tid < TT) {
    double v = 0.0;
    for (int w = 0; w < kFewWarps; ++w) v += square_parts[w][tid];
    squares[tid] = v;
  }
  __syncthreads();
  cluster_sync_all();
  if (tid < TT) {
    float r = 1.0f;
    if (a.norm != nullptr) {
      double v = 0.0;
      for (int q = 0; q < kHeadRanks; ++q) v += cluster_load_double(mapa_shared(smem_u32(&squares[tid]), q));
      r = static_cast<float>(1.0 / sqrt(v / a.d + static_cast<double>(a.eps)));
    }
    scale[tid] = r;
  }
  __syncthreads();
  if (rank == 0 && a.router != nullptr) {
    for (int at = tid; at < TT * kHeadCols; at += kFewThreads) {
      const int t = at / kHeadCols, e = col0 + at % kHeadCols;
      if (t >= a.T || e >= a.E) continue;
      float v = 0.0f;
      for (int q = 0; q < kHeadRanks; ++q) v += cluster_load(mapa_shared(smem_u32(&(&joined[0][0])[at]), q));
      a.logits[static_cast<int64_t>(t) * a.E + e] = v * scale[t];
    }
  }
  __syncthreads();
  cluster_sync_all();  // the others' shared memory lives until it has been read
  if (!first || a.norm == nullptr) return;
  for (int t = 0; t < a.T; ++t) {
    for (int k = k_begin + tid; k < k_end; k += kFewThreads) {
      float h = to_f32<T>(x[static_cast<int64_t>(t) * a.d + k]);
      if (residual != nullptr) h = to_f32<T>(Elem<T>::from_float(h + to_f32<T>(residual[static_cast<int64_t>(t) * a.d + k])));
      static_cast<T*>(a.y)[static_cast<int64_t>(t) * a.d + k] = Elem<T>::from_float(h * scale[t] * norm_weight(k));
    }
  }
}

// -------------------------------------------------------------------------------------------------------- the experts
struct FewArgs {
  const void* x;           // [T, d]: what the experts read
  const float* logits;     // [T, E], or null: ids and scores are given
  const float* bias;       // [E], or null
  const int64_t* ids;      // [T, k]
  const void* given;       // scores [T, k]
  const void *w1, *w2;     // 16 bits
  Q4Matrix up, down;       // 4 bits
  uint16_t* hidden;        // [slots, I]
  float* rows;             // [kFewParts][slots, d]
  const void* addend;      // [T, d], or null
  void* out;               // [T, d]
  uint32_t* meeting;
  int* status;
  long long limit;
  int T, d, I, E, k, act;
  // the router's tail
  int sigmoid, softmax_after, normalize, groups, keep, best;
  float scale;
};

struct FewRouting {
  float score[kFewSlots];
  int16_t id[kFewSlots];
  int16_t expert[kFewSlots];       // of an entry: up to 16 slots of one expert
  uint8_t count[kFewSlots];
  int16_t slot[kFewSlots][kFewTokens];
  int entries;
  int go_on;
};

// All CTAs of the grid; false (and a status code) when one has not come in time.
__device__ __forceinline__ bool meet(const FewArgs& a, int turn, int* go_on) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(a.meeting, 1u);
    const uint32_t all = static_cast<uint32_t>(turn) * gridDim.x;
    const long long t0 = clock64();
    int ok = 1;
    while (true) {
      uint32_t seen;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(a.meeting) : "memory");
      if (seen >= all) break;
      if (clock64() - t0 > a.limit) {
        if (a.status != nullptr) atomicCAS(a.status, 0, DS_TIMEOUT_GRID);
        ok = 0;
        break;
      }
    }
    __threadfence();
    *go_on = ok;
  }
  __syncthreads();
  return *go_on != 0;
}

// One warp, one token: keys [E] is scratch of this warp's own.
__device__ __forceinline__ void choose(const FewArgs& a, int t, float* keys, FewRouting& r, int lane) {
  const float* logits = a.logits + static_cast<int64_t>(t) * a.E;
  const bool by_probability = a.bias != nullptr || a.groups > 1;
  float most = -INFINITY, sum = 0.0f;
  for (int e = lane; e < a.E; e += 32) most = fmaxf(most, logits[e]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
  const bool softmax = !a.sigmoid && !a.softmax_after;
  if (softmax) {
    for (int e = lane; e < a.E; e += 32) sum += expf(logits[e] - most);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  }
  const auto probability = [&](float l) { return a.sigmoid ? 1.0f / (1.0f + expf(-l)) : softmax ? expf(l - most) / sum : l; };
  // open experts' keys stay above -inf (NaN and -inf come last, lowest index first); taken and closed ones are -inf
  constexpr float kLast = -3.402823466e38f;
  for (int e = lane; e < a.E; e += 32) {
    float key = logits[e];
    if (by_probability) key = probability(key) + (a.bias != nullptr ? a.bias[e] : 0.0f);
    keys[e] = key > kLast ? key : kLast;
  }
  __syncwarp();
  if (a.groups > 1) {
    const int width = a.E / a.groups;
    float* worth = keys + a.E;  // [groups]
    for (int g = lane; g < a.groups; g += 32) {
      float b0 = -INFINITY, b1 = -INFINITY;
      for (int i = 0; i < width; ++i) {
        const float v = keys[g * width + i];
        b1 = fmaxf(b1, fminf(b0, v));
        b0 = fmaxf(b0, v);
      }
      worth[g] = a.best == 2 && width > 1 ? b0 + b1 : b0;
    }
    __syncwarp();
    for (int g = lane; g < a.groups; g += 32) {
      const float mine = worth[g];
      int before = 0;
      for (int o = 0; o < a.groups; ++o) before += worth[o] > mine || (worth[o] == mine && o < g);
      if (before >= a.keep)
        for (int i = 0; i < width; ++i) keys[g * width + i] = -INFINITY;
    }
    __syncwarp();
  }
  // k times the best; a lane looks again only when its own best was taken
  float best = -INFINITY;
  int at = a.E;
  const auto look = [&]() {
    best = -INFINITY;
    at = a.E;
    for (int e = lane; e < a.E; e += 32)
      if (keys[e] > best) best = keys[e], at = e;
  };
  look();
  float total = 0.0f, top = 0.0f;
  for (int s = 0; s < a.k; ++s) {
    float v = best;
    int e = at;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float ov = __shfl_xor_sync(0xFFFFFFFFu, v, off);
      const int oe = __shfl_xor_sync(0xFFFFFFFFu, e, off);
      if (ov > v || (ov == v && oe < e)) v = ov, e = oe;
    }
    if (e == at && e < a.E) {
      keys[e] = -INFINITY;
      look();
    }
    float p = e < a.E ? logits[e] : 0.0f;
    if (a.softmax_after) {
      if (s == 0) top = p;  // the largest selected logit comes first (no bias, no groups)
      p = expf(p - top);
    } else {
      p = probability(p);
    }
    total += p;
    if (lane == 0) {
      r.id[t * a.k + s] = static_cast<int16_t>(e < a.E ? e : -1);
      r.score[t * a.k + s] = p;
    }
  }
  __syncwarp();
  if (a.softmax_after) {
    for (int s = lane; s < a.k; s += 32) r.score[t * a.k + s] /= total;
  } else if (a.normalize) {
    const float by = a.normalize == 2 ? fmaxf(total, 1e-12f) : total + 1e-20f;
    for (int s = lane; s < a.k; s += 32) r.score[t * a.k + s] = r.score[t * a.k + s] / by * a.scale;
  } else {
    for (int s = lane; s < a.k; s += 32) r.score[t * a.k + s] *= a.scale;
  }
}

// Scores, experts, and the list of entries: up to 16 slots of one expert each, in the order of their first slots.
template <typename T> __device__ __forceinline__ void route(const FewArgs& a, FewRouting& r, float* scratch) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slots = a.T * a.k;
  if (a.logits != nullptr) {
    for (int t = warp; t < a.T; t += kFewWarps) choose(a, t, scratch + warp * (a.E + a.groups), r, lane);
  } else {
    for (int j = tid; j < slots; j += kFewThreads) {
      const int64_t e = a.ids[j];
      const bool ok = e >= 0 && e < a.E;
      if (!ok && a.status != nullptr) atomicCAS(a.status, 0, DS_BAD_EXPERT_ID);
      r.id[j] = static_cast<int16_t>(ok ? e : -1);
      r.score[j] = to_f32<T>(static_cast<const T*>(a.given)[j]);
    }
  }
  __syncthreads();
  __shared__ int starts[kFewSlots / 32];
  int rank[kFewSlots / kFewThreads];
  bool begins[kFewSlots / kFewThreads];
#pragma unroll
  for (int i = 0; i < kFewSlots / kFewThreads; ++i) {
    const int j = tid + i * kFewThreads;
    const int e = j < slots ? r.id[j] : -1;
    rank[i] = 0;
    if (e >= 0)
      for (int o = 0; o < j; ++o) rank[i] += r.id[o] == e;
    begins[i] = e >= 0 && rank[i] % kFewTokens == 0;
    const unsigned mine = __ballot_sync(0xFFFFFFFFu, begins[i]);
    if (lane == 0) starts[i * kFewWarps + warp] = static_cast<int>(mine);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kFewSlots / kFewThreads; ++i) {
    const int j = tid + i * kFewThreads;
    if (begins[i]) {
      int n = __popc(static_cast<unsigned>(starts[i * kFewWarps + warp]) & ((1u << lane) - 1));
      for (int w = 0; w < i * kFewWarps + warp; ++w) n += __popc(static_cast<unsigned>(starts[w]));
      int left = 0;
      for (int o = j; o < slots; ++o) left += r.id[o] == r.id[j];
      r.expert[n] = r.id[j];
      r.count[n] = static_cast<uint8_t>(min(left, kFewTokens));
      for (int o = j, c = 0; o < slots && c < kFewTokens; ++o)
        if (r.id[o] == r.id[j]) r.slot[n][c++] = static_cast<int16_t>(o);
    }
  }
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kFewSlots / 32; ++w) n += __popc(static_cast<unsigned>(starts[w]));
    r.entries = n;
  }
  __syncthreads();
}

__device__ __forceinline__ float few_act(float x, int act) {
  switch (act) {
    case MOE_ACT_SWIGLU:
    case MOE_ACT_SILU: return silu_f(x);
    case MOE_ACT_GEGLU:
    case MOE_ACT_GELU: return gelu_f(x);
    case MOE_ACT_GELU_TANH: return gelu_tanh_f(x);
    default: return x;
  }
}

// ---- 16-bit weights [K, N] (N contiguous) by up to 16 rows: a warp's step is 16 rows of K by 64 columns ----
// Tokens are the 16 rows of m16n8k16 and column 8 g + j of the tile is column g of its j-th product, so that a lane's 16-byte pieces are
// eight products' columns; slots (2 t, 2 t + 1) and (2 t + 8, 2 t + 9) of K stand for rows 4 t .. 4 t + 3.
constexpr int kWideCols = 64, kWideStep = 16;
constexpr int kWideStage = kWideStep * kWideCols * 2;
constexpr int kWideDepth = 5;

template <typename T>
__device__ __forceinline__ void wide_tile(float (&acc)[8][4], const uint16_t* w, int K, int N, int col0, const uint16_t* x0, const uint16_t* x1, int first,
                                          int end, int stride, uint32_t ring, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const bool inside = col0 + 8 * g < N;
  const uint16_t* from = w + static_cast<int64_t>(4 * t) * N + col0 + 8 * g;
  const auto copy = [&](uint32_t stage, int step) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = step * kWideStep + 4 * t + j;
      if (inside && k < K) copy_16(stage + j * 512 + lane * 16, from + (static_cast<int64_t>(step) * kWideStep + j) * N);
    }
  };
  int ahead = first;
#pragma unroll
  for (int s = 0; s < kWideDepth - 1; ++s, ahead += stride) {
    if (ahead < end) copy(ring + s * kWideStage, ahead);
    copies_commit();
  }
  uint32_t stage = ring, free_stage = ring + (kWideDepth - 1) * kWideStage;
  for (int step = first; step < end; step += stride, ahead += stride) {
    copies_wait<kWideDepth - 2>();
    if (ahead < end) copy(free_stage, ahead);  // (a lane reads what it has copied itself, and has read what this replaces)
    copies_commit();
    const int k = step * kWideStep + 4 * t;
    uint2 a0 = make_uint2(0, 0), a1 = a0;
    if (k < K) {
      if (x0 != nullptr) a0 = *reinterpret_cast<const uint2*>(x0 + k);
      if (x1 != nullptr) a1 = *reinterpret_cast<const uint2*>(x1 + k);
    }
    const uint32_t a[4] = {a0.x, a1.x, a0.y, a1.y};
    uint4 r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = inside && k < K ? lds_128(stage + j * 512 + lane * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t pick = j & 1 ? 0x7632u : 0x5410u;
      mma_16x8x16<T>(acc[j], a, __byte_perm(word_of(r[0], j >> 1), word_of(r[1], j >> 1), pick),
                     __byte_perm(word_of(r[2], j >> 1), word_of(r[3], j >> 1), pick));
    }
    free_stage = stage;
    stage = stage == ring + (kWideDepth - 1) * kWideStage ? ring : stage + kWideStage;
  }
  copies_wait<0>();
  __syncwarp();  // the ring is free again, for other lanes' words too
}

template <int BITS, int NG, bool ZEROS> struct FewPlan {
  static constexpr int kDepth = BITS == 4 ? 6 : kWideDepth;
  static constexpr int kStage = BITS == 4 ? Q4Stage<NG, ZEROS>::kBytes : kWideStage;
  static constexpr int kRing = kDepth * kStage;
  static constexpr int kCols = BITS == 4 ? kQ4Rows : kWideCols;       // of a tile of a product
  static constexpr int kTotal = kFewWarps * kRing;
  // a warp's ring also holds its sums of a unit, when the copies are through, and before all that the router's keys
  static_assert(kFewTokens * kCols * 4 <= kRing && kFewWarps * (kFewExperts + kFewGroups) * 4 <= kTotal, "the rings are large enough");
};

template <typename T, int BITS, int NG, bool ZEROS>
__global__ void __launch_bounds__(kFewThreads, kFewCtas) few_experts_kernel(const FewArgs a) {
  using P = FewPlan<BITS, NG, ZEROS>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ FewRouting r;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * P::kRing;
  const auto part = [&](int w, int row, int col) -> float& { return reinterpret_cast<float*>(smem + w * P::kRing)[row * P::kCols + col]; };
  route<T>(a, r, reinterpret_cast<float*>(smem));
  const bool gated = a.act == MOE_ACT_SWIGLU || a.act == MOE_ACT_GEGLU;
  const int slots = a.T * a.k;

  // One unit: entry n's rows by a tile of its expert's matrix over steps [begin, end); `source` gives the row of a slot.  Leaves the
  // warps' sums in their rings.
  const auto product = [&](int n, int tile, const void* w16, const Q4Matrix& w4, int64_t tiles4, int K, int N, int begin, int end, auto source) {
    const int count = r.count[n];
    const int e = r.expert[n];
    const uint16_t* x0 = g < count ? source(r.slot[n][g]) : nullptr;
    const uint16_t* x1 = g + 8 < count ? source(r.slot[n][g + 8]) : nullptr;
    if constexpr (BITS == 4) {
      Q4Matrix w = w4;
      w.steps = end;
      const int64_t at = e * tiles4 + tile;
      const uint4* data = w4.data + at * w4.steps * kQ4Words;
      w.data = data;
      w.scales = static_cast<const uint16_t*>(w4.scales) + at * w4.steps * (kQ4Rows * NG);
      w.zeros = ZEROS ? w4.zeros + at * w4.steps * (kQ4Rows * NG) : nullptr;
      const auto leave = [&](const auto& acc, int m) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = 8 * m + 2 * t4 + (c & 1);
          if (row < count) part(warp, row, g + 8 * (c >> 1)) = acc[c];
        }
      };
      if (count <= 8) {
        float acc[1][4] = {};
        const uint16_t* const x[1] = {x0};
        q4_tile<T, NG, ZEROS, 1, P::kDepth>(acc, w, 0, x, K, begin + warp, kFewWarps, ring, lane);
        leave(acc[0], 0);
      } else {
        float acc[2][4] = {};
        const uint16_t* const x[2] = {x0, x1};
        q4_tile<T, NG, ZEROS, 2, P::kDepth>(acc, w, 0, x, K, begin + warp, kFewWarps, ring, lane);
        leave(acc[0], 0);
        leave(acc[1], 1);
      }
    } else {
      float acc[8][4] = {};
      wide_tile<T>(acc, static_cast<const uint16_t*>(w16) + static_cast<int64_t>(e) * K * N, K, N, tile * kWideCols, x0, x1, begin + warp, end, kFewWarps, ring,
                   lane);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = g + 8 * (c >> 1);
          if (row < count) part(warp, row, 8 * (2 * t4 + (c & 1)) + j) = acc[j][c];
        }
    }
    __syncthreads();
  };
  const auto total = [&](int row, int col) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) v += part(w, row, col);
    return v;
  };

  {  // up: units (entry, tile)
    const int N = gated ? 2 * a.I : a.I;
    const int tiles = (N + P::kCols - 1) / P::kCols;
    const int steps = BITS == 4 ? a.up.steps : (a.d + kWideStep - 1) / kWideStep;
    for (int unit = blockIdx.x; unit < r.entries * tiles; unit += gridDim.x) {
      const int n = unit / tiles, tile = unit - n * tiles;
      product(n, tile, a.w1, a.up, a.up.tiles, a.d, N, 0, steps,
              [&](int slot) { return static_cast<const uint16_t*>(a.x) + static_cast<int64_t>(slot / a.k) * a.d; });
      const int cols = gated ? P::kCols / 2 : P::kCols;
      for (int at = tid; at < r.count[n] * cols; at += kFewThreads) {
        const int row = at / cols, c = at - row * cols;
        const int i = tile * cols + c;
        if (i >= a.I) continue;
        float v;
        if (gated) v = BITS == 4 ? few_act(total(row, c), a.act) * total(row, c + 8) : few_act(total(row, 2 * c), a.act) * total(row, 2 * c + 1);
        else v = few_act(total(row, c), a.act);
        const T h = Elem<T>::from_float(v);
        a.hidden[static_cast<int64_t>(r.slot[n][row]) * a.I + i] = *reinterpret_cast<const uint16_t*>(&h);
      }
      __syncthreads();
    }
  }
  if (!meet(a, 1, &r.go_on)) return;

  int shares = 1;  // of the depth of the down product: enough units for every CTA to have some
  {
    const int tiles = (a.d + P::kCols - 1) / P::kCols;
    const int steps = BITS == 4 ? a.down.steps : (a.I + kWideStep - 1) / kWideStep;
    while (shares < kFewParts && r.entries * tiles * shares < 2 * static_cast<int>(gridDim.x) && steps >= 2 * kFewWarps * shares) shares *= 2;
    for (int unit = blockIdx.x; unit < r.entries * tiles * shares; unit += gridDim.x) {
      const int n = unit / (tiles * shares), rest = unit - n * tiles * shares;
      const int share = rest / tiles, tile = rest - share * tiles;
      product(n, tile, a.w2, a.down, a.down.tiles, a.I, a.d, steps * share / shares, steps * (share + 1) / shares,
              [&](int slot) { return a.hidden + static_cast<int64_t>(slot) * a.I; });
      for (int at = tid; at < r.count[n] * P::kCols; at += kFewThreads) {
        const int row = at / P::kCols, c = at - row * P::kCols;
        const int i = tile * P::kCols + c;
        if (i < a.d) a.rows[(static_cast<int64_t>(share) * slots + r.slot[n][row]) * a.d + i] = total(row, c);
      }
      __syncthreads();
    }
  }
  if (!meet(a, 2, &r.go_on)) return;

  for (int at = blockIdx.x * kFewThreads + tid; at < a.T * a.d; at += gridDim.x * kFewThreads) {
    const int t = at / a.d, i = at - t * a.d;
    float v = a.addend != nullptr ? to_f32<T>(static_cast<const T*>(a.addend)[at]) : 0.0f;
    for (int s = 0; s < a.k; ++s) {
      const int slot = t * a.k + s;
      if (r.id[slot] < 0) continue;
      float row = 0.0f;
      for (int p = 0; p < shares; ++p) row += a.rows[(static_cast<int64_t>(p) * slots + slot) * a.d + i];
      v = fmaf(r.score[slot], row, v);
    }
    static_cast<T*>(a.out)[at] = Elem<T>::from_float(v);
  }
}

template <typename T, typename W, int TT> static int launch_head(const HeadArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int tiles = a.router == nullptr ? 1 : (a.E + kHeadCols - 1) / kHeadCols;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * kHeadRanks), 1, 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kHeadRanks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, few_head_kernel<T, W, TT>, a));
  return MOE_OK;
}
template <typename T, typename W> static int launch_head_tokens(const HeadArgs& a, cudaStream_t s) {
  if (a.T == 1) return launch_head<T, W, 1>(a, s);
  if (a.T <= 4) return launch_head<T, W, 4>(a, s);
  return launch_head<T, W, 16>(a, s);
}

// One wave: what of the grid's CTAs fit at once, at most kFewCtas per SM.
template <typename T, int BITS, int NG, bool ZEROS> static int launch_experts(const FewArgs& a, cudaStream_t s) {
  using P = FewPlan<BITS, NG, ZEROS>;
  const auto kernel = few_experts_kernel<T, BITS, NG, ZEROS>;
  static std::atomic<int> resident[64];
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  int ctas = dev < 64 ? resident[dev].load(std::memory_order_acquire) : 0;
  if (ctas == 0) {
    MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kTotal));
    MOE_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, kFewThreads, P::kTotal));
    MOE_CHECK_ARG(ctas > 0, "moe_few_tokens: the kernel does not fit on an SM");
    if (ctas > kFewCtas) ctas = kFewCtas;
    if (dev < 64) resident[dev].store(ctas, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * sm_count()), 1, 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.dynamicSmemBytes = P::kTotal;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return MOE_OK;
}
template <typename T> static int launch_experts_of(const FewArgs& a, int bits, int group, cudaStream_t s) {
  if (bits == 16) return launch_experts<T, 16, 1, false>(a, s);
  const bool z = a.up.zeros != nullptr;
  if (group == 128) return z ? launch_experts<T, 4, 1, true>(a, s) : launch_experts<T, 4, 1, false>(a, s);
  if (group == 64) return z ? launch_experts<T, 4, 2, true>(a, s) : launch_experts<T, 4, 2, false>(a, s);
  return z ? launch_experts<T, 4, 4, true>(a, s) : launch_experts<T, 4, 4, false>(a, s);
}

static int64_t few_up(int64_t n) { return (n + 255) / 256 * 256; }
struct FewSpace {
  int64_t meeting, logits, y, hidden, rows, total;
};
static FewSpace few_space(int64_t T, int64_t d, int64_t I, int64_t E, int64_t k) {
  FewSpace s;
  s.meeting = 0;
  s.logits = 256;
  s.y = s.logits + few_up(4 * T * E);
  s.hidden = s.y + few_up(2 * T * d);
  s.rows = s.hidden + few_up(2 * T * k * I);
  s.total = s.rows + few_up(4 * T * k * d * kFewParts);
  return s;
}

}  // namespace moe

using namespace moe;

extern "C" size_t moe_few_pass_size(void) { return sizeof(moe_few_pass); }

extern "C" size_t moe_few_workspace_bytes(int num_tokens, int d, int inter, int num_experts, int topk) {
  if (num_tokens < 0 || d < 0 || inter < 0 || num_experts < 0 || topk < 0) return 0;
  return static_cast<size_t>(few_space(num_tokens, d, inter, num_experts, topk).total);
}

extern "C" int moe_few_tokens(const moe_few_pass* p, void* stream) {
  MOE_CHECK_ARG(p != nullptr, "moe_few_tokens: null pointer argument");
  MOE_CHECK_ARG(p->num_tokens >= 0 && p->d > 0 && p->inter > 0 && p->num_experts > 0 && p->topk > 0, "moe_few_tokens: T=%d d=%d I=%d E=%d k=%d", p->num_tokens,
                p->d, p->inter, p->num_experts, p->topk);
  if (p->num_tokens > kFewTokens || p->num_tokens * static_cast<int64_t>(p->topk) > kFewSlots || p->num_experts > kFewExperts || p->d > (1 << 20) ||
      p->inter > (1 << 20) || (p->router_w != nullptr && p->num_groups > kFewGroups)) {
    set_error("moe_few_tokens: at most %d tokens, %d slots, %d experts in %d groups, rows of 2^20; got %d, %lld, %d in %d, %d and %d", kFewTokens, kFewSlots,
              kFewExperts, kFewGroups, p->num_tokens, static_cast<long long>(p->num_tokens) * p->topk, p->num_experts, p->num_groups, p->d, p->inter);
    return MOE_ERR_UNSUPPORTED;
  }
  if (p->d % 8 != 0 || p->inter % 8 != 0) {
    set_error("moe_few_tokens: d=%d and inter=%d must be multiples of 8", p->d, p->inter);
    return MOE_ERR_UNSUPPORTED;
  }
  MOE_CHECK_ARG(p->dtype == MOE_DTYPE_BF16 || p->dtype == MOE_DTYPE_F16, "moe_few_tokens: unknown dtype %d", p->dtype);
  MOE_CHECK_ARG(p->act >= MOE_ACT_NONE && p->act <= MOE_ACT_GELU_TANH, "moe_few_tokens: unknown activation %d", p->act);
  MOE_CHECK_ARG(p->bits == 16 || (p->bits == 4 && (p->group == 32 || p->group == 64 || p->group == 128)),
                "moe_few_tokens: weights of 16 bits, or of 4 in groups of 32, 64 or 128, got %d and %d", p->bits, p->group);
  const bool routed = p->router_w != nullptr;
  MOE_CHECK_ARG(routed || (p->expert_idx != nullptr && p->scores != nullptr), "moe_few_tokens: a router, or experts and scores");
  MOE_CHECK_ARG(!routed || (p->num_groups > 0 && p->num_experts % p->num_groups == 0 && p->topk_groups > 0 && p->topk_groups <= p->num_groups &&
                            (p->group_best == 1 || p->group_best == 2) &&
                            p->topk <= static_cast<int64_t>(p->topk_groups) * (p->num_experts / p->num_groups)),
                "moe_few_tokens: %d experts in %d groups, %d of them open, best %d, do not give %d", p->num_experts, p->num_groups, p->topk_groups,
                p->group_best, p->topk);
  MOE_CHECK_ARG(!routed || !(p->score_function == 2 && (p->router_bias != nullptr || p->num_groups > 1)),
                "moe_few_tokens: a softmax over the selected logits goes without bias and groups");
  MOE_CHECK_ARG(!routed || (p->score_function >= 0 && p->score_function <= 2 && p->normalize >= 0 && p->normalize <= 2 &&
                            (p->router_dtype == 2 || p->router_dtype == p->dtype)),
                "moe_few_tokens: unknown router options");
  if (p->num_tokens == 0) return MOE_OK;
  MOE_CHECK_ARG(p->x && p->w1 && p->w2 && p->out && p->workspace, "moe_few_tokens: null pointer argument");
  MOE_CHECK_ARG(p->bits == 16 || (p->w1_scales && p->w2_scales && (p->w1_zeros == nullptr) == (p->w2_zeros == nullptr)),
                "moe_few_tokens: 4-bit weights have scales, and both zero points or none");
  MOE_CHECK_ARG(p->residual == nullptr || (p->norm_w != nullptr && p->stream_out != nullptr), "moe_few_tokens: a residual goes with a norm and the stream");
  uintptr_t all = 0;
  for (const void* q : {p->x, p->residual, p->norm_w, p->w1, p->w1_scales, p->w1_zeros, p->w2, p->w2_scales, p->w2_zeros, p->router_w, p->addend,
                        static_cast<const void*>(p->out), static_cast<const void*>(p->stream_out), static_cast<const void*>(p->workspace)})
    all |= reinterpret_cast<uintptr_t>(q);
  MOE_CHECK_ARG((all & 15) == 0, "moe_few_tokens: pointers must be 16-byte aligned");
  const FewSpace sp = few_space(p->num_tokens, p->d, p->inter, p->num_experts, p->topk);
  MOE_CHECK_ARG(p->workspace_bytes >= static_cast<size_t>(sp.total), "moe_few_tokens: the workspace has %zu of %lld bytes", p->workspace_bytes,
                static_cast<long long>(sp.total));
  uint8_t* const ws = static_cast<uint8_t*>(p->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = p->dtype == MOE_DTYPE_BF16;

  FewArgs a{};
  a.meeting = reinterpret_cast<uint32_t*>(ws + sp.meeting);
  if (routed || p->norm_w != nullptr) {
    HeadArgs h{};
    h.x = p->x;
    h.residual = p->residual;
    h.norm = p->norm_w;
    h.router = p->router_w;
    h.stream = p->stream_out;
    h.y = ws + sp.y;
    h.logits = reinterpret_cast<float*>(ws + sp.logits);
    h.meeting = a.meeting;
    h.T = p->num_tokens;
    h.d = p->d;
    h.E = p->num_experts;
    h.norm_fp32 = p->norm_dtype == 2;
    h.eps = p->eps;
    const bool wide = p->router_dtype == 2;
    const int rc = bf16 ? wide ? launch_head_tokens<__nv_bfloat16, float>(h, s) : launch_head_tokens<__nv_bfloat16, __nv_bfloat16>(h, s)
                        : wide ? launch_head_tokens<__half, float>(h, s) : launch_head_tokens<__half, __half>(h, s);
    if (rc != MOE_OK) return rc;
  } else {
    MOE_CUDA(cudaMemsetAsync(a.meeting, 0, 2 * sizeof(uint32_t), s));
  }
  a.x = p->norm_w != nullptr ? static_cast<const void*>(ws + sp.y) : p->x;
  a.logits = routed ? reinterpret_cast<const float*>(ws + sp.logits) : nullptr;
  a.bias = p->router_bias;
  a.ids = p->expert_idx;
  a.given = p->scores;
  a.w1 = p->w1;
  a.w2 = p->w2;
  if (p->bits == 4) {
    const bool glu = p->act == MOE_ACT_SWIGLU || p->act == MOE_ACT_GEGLU;
    const auto matrix = [&](const void* data, const void* scales, const void* zeros, int n, int k) {
      return Q4Matrix{static_cast<const uint4*>(data), scales, static_cast<const uint8_t*>(zeros), (n + kQ4Rows - 1) / kQ4Rows, (k + kQ4Step - 1) / kQ4Step};
    };
    a.up = matrix(p->w1, p->w1_scales, p->w1_zeros, glu ? 2 * p->inter : p->inter, p->d);
    a.down = matrix(p->w2, p->w2_scales, p->w2_zeros, p->d, p->inter);
  }
  a.hidden = reinterpret_cast<uint16_t*>(ws + sp.hidden);
  a.rows = reinterpret_cast<float*>(ws + sp.rows);
  a.addend = p->addend;
  a.out = p->out;
  a.status = p->status;
  a.limit = wait_limit_cycles();
  a.T = p->num_tokens;
  a.d = p->d;
  a.I = p->inter;
  a.E = p->num_experts;
  a.k = p->topk;
  a.act = p->act;
  a.sigmoid = p->score_function == 1;
  a.softmax_after = p->score_function == 2;
  a.normalize = p->normalize;
  a.groups = routed ? p->num_groups : 1;
  a.keep = p->topk_groups;
  a.best = p->group_best;
  a.scale = p->scale;
  return bf16 ? launch_experts_of<__nv_bfloat16>(a, p->bits, p->group, s) : launch_experts_of<__half>(a, p->bits, p->group, s);
}
