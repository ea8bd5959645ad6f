// A whole layer for up to 16 tokens in two kernels, with experts in 16 or 4 bits:
//
//   first:   h = round(x + residual), r = 1 / sqrt(mean h^2 + eps), y = round(h r w);  logits = (h r w) W_router, in fp32
//   second:  scores and experts of every token (each CTA for itself);  hidden = round(act(y W1[e])) for the chosen experts;
//            rows = hidden W2[e] in fp32;  out = round(sum over the slots of score * row + addend)
//
// Bound by reading the chosen experts' weights (16 bits: 16 tokens x 8 on 64 experts of 2048 x 1024, 711 MB, in 136 us, the up product's
// part at 6.7 TB/s), by what it costs to make numbers of 4-bit ones (64 experts of 7168 x 2048, 1.2 GB, 318 us), and for one token by what
// is not reading: of 36 us for 69 MB the first kernel and the way to the second are 8, choosing 4, meeting twice 4.  The second kernel
// is one resident wave (a cooperative launch, so that its CTAs may wait for one another): between its three phases they meet at a counter
// in global memory that the first kernel has set to zero.  Weights are copied once per entry, eight slots of an expert: twice for
// an expert that 9 to 16 slots chose.
// Every sum has a fixed order: nothing depends on timing.
//
// The logits are not rounded to 16 bits, nor are an expert's rows before the fold; y and the activated product are, because they are
// operands of 16-bit products.
#include "int4.cuh"
#include "order.cuh"

#include <atomic>

namespace moe {

constexpr int kFewTokens = 16;
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewSlots = 256;      // tokens x slots
constexpr int kFewRows = 8;         // of an entry: slots of one expert that share its weights
constexpr int kFewExperts = 1024, kFewGroups = 64;
constexpr int kFewCtas = 2;         // per SM
constexpr int kFewParts = 4;        // shares of the down product's depth, at most (1, 2 or 4)

// ---------------------------------------------------------------------------------------------------- norm and logits
constexpr int kHeadRanks = 8;           // CTAs of a cluster share the hidden size
constexpr int kHeadCols = 16;           // experts of a cluster
constexpr int kHeadMost = 16384;        // hidden size: a CTA keeps its eighth of all rows in fp32
constexpr int kHeadLanes = kFewThreads / (kHeadCols / 4);

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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

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
template <typename T> __device__ __forceinline__ void eight(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Elem<T>::unpack2(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// A cluster takes 16 experts' columns, its CTAs an eighth of the hidden size each; a thread four columns and every 64th hidden row.  One
// look at x: the logits are linear in r, which is known when the sums of squares have met, while the products are computed.
template <typename T, typename W, int TT>
__global__ void __launch_bounds__(kFewThreads) few_head_kernel(const HeadArgs a) {
  extern __shared__ __align__(16) float rows[];  // [TT][share]: h w
  __shared__ float parts[kFewWarps][TT][kHeadCols];
  __shared__ float joined[TT][kHeadCols];
  __shared__ float2 squares[kFewTokens];  // sum of squares, and whether it is in units of 2^144 (the rows of this share then in ones of 2^72)
  __shared__ float scale[kFewTokens], part_scale[kFewTokens], logit_scale[kFewTokens];  // of the share's rows, its logits, and their sums
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int group = static_cast<int>(blockIdx.x / kHeadRanks), groups = static_cast<int>(gridDim.x / kHeadRanks);
  const int col0 = group * kHeadCols;
  if (blockIdx.x == 0 && tid < 2) a.meeting[tid] = 0;
  const int share = (a.d + kHeadRanks * 8 - 1) / (kHeadRanks * 8) * 8;
  const int k_begin = min(rank * share, a.d), count = min(share, a.d - k_begin);
  const int cv = tid % (kHeadCols / 4), kl = tid / (kHeadCols / 4);  // columns col0 + 4 cv + 0..3, hidden rows kl + 64 i
  const int left = a.E - (col0 + 4 * cv);
  const bool whole = left >= 4 && (a.E & 3) == 0, mine = a.router != nullptr && left > 0;
  const W* router = static_cast<const W*>(a.router) + static_cast<int64_t>(k_begin) * a.E + col0 + 4 * cv;
  constexpr int AHEAD = 2;
  float w[AHEAD][4];
  const auto ask = [&](int i, float (&f)[4]) {
    if (mine && i < count) router_row<W>(router + static_cast<int64_t>(i) * a.E, left, whole, f);
    else f[0] = f[1] = f[2] = f[3] = 0.0f;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) ask(kl + i * kHeadLanes, w[i]);  // on their way while the rows are made

  // rows: a warp per token, eight columns per lane at a time
  for (int t = warp; t < TT; t += kFewWarps) {
    if (t >= a.T) {
      for (int i = lane; i < share; i += 32) rows[t * share + i] = 0.0f;
      if (lane == 0) squares[t] = make_float2(0.0f, 0.0f);
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(t) * a.d + k_begin;
    const T* residual = a.residual == nullptr ? nullptr : static_cast<const T*>(a.residual) + static_cast<int64_t>(t) * a.d + k_begin;
    float sum = 0.0f, large = 0.0f, most = 0.0f;
    // h w, times `units`, to shared memory
    const auto make = [&](float units, bool first) {
#pragma unroll 1
      for (int i = lane * 8; i < share; i += 256) {
        float h[8] = {}, g[8];
        if (i < count) {
          eight<T>(*reinterpret_cast<const uint4*>(x + i), h);
          if (residual != nullptr) {
            float o[8];
            eight<T>(*reinterpret_cast<const uint4*>(residual + i), o);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] += o[j];
            const uint4 v = make_uint4(Elem<T>::pack2(h[0], h[1]), Elem<T>::pack2(h[2], h[3]), Elem<T>::pack2(h[4], h[5]), Elem<T>::pack2(h[6], h[7]));
            if (first && t % groups == group) *reinterpret_cast<uint4*>(static_cast<T*>(a.stream) + static_cast<int64_t>(t) * a.d + k_begin + i) = v;
            eight<T>(v, h);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (first) {
              sum = fmaf(h[j], h[j], sum);
              large = fmaf(h[j] * 0x1p-72f, h[j] * 0x1p-72f, large);  // bf16 values from 2^57 on have squares whose sum may leave fp32
              most = fmaxf(most, fabsf(h[j]));
            } else {
              h[j] *= units;
            }
            g[j] = a.norm == nullptr ? 1.0f : a.norm_fp32 ? static_cast<const float*>(a.norm)[k_begin + i + j] : 0.0f;
          }
          if (a.norm != nullptr && !a.norm_fp32) eight<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.norm) + k_begin + i), g);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] *= g[j];
        }
        float4* out = reinterpret_cast<float4*>(rows + t * share + i);
        out[0] = make_float4(h[0], h[1], h[2], h[3]);
        out[1] = make_float4(h[4], h[5], h[6], h[7]);
      }
    };
    make(1.0f, true);
    if (a.norm != nullptr) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
        large += __shfl_xor_sync(0xFFFFFFFFu, large, off);
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
      }
      if (lane == 0) squares[t] = most > 0x1p50f ? make_float2(large, 1.0f) : make_float2(sum, 0.0f);
      if (most > 0x1p50f) make(0x1p-72f, false);  // h w, and its sums with the router's weights, may leave fp32 where h r w is of order 1
    }
  }
  __syncthreads();
  cluster_arrive();  // the squares
  float acc[TT][4];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.0f;
  if (a.router != nullptr) {
    for (int i0 = kl; i0 < count; i0 += AHEAD * kHeadLanes) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int k = i0 + i * kHeadLanes;
        float f[4] = {w[i][0], w[i][1], w[i][2], w[i][3]};
        ask(k + AHEAD * kHeadLanes, w[i]);
        if (k < count) {
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            const float h = rows[t * share + k];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[t][c] = fmaf(h, f[c], acc[t][c]);
          }
        }
      }
    }
  }
  __syncwarp();
  cluster_wait();
  if (tid < TT) {
    float r = 1.0f, parts_by = 1.0f, logits_by = 1.0f;
    if (a.norm != nullptr) {
      float2 all[kHeadRanks];
#pragma unroll
      for (int q = 0; q < kHeadRanks; ++q) {
        const uint32_t at = mapa_shared(smem_u32(&squares[tid]), q);
        all[q] = make_float2(cluster_load(at), cluster_load(at + 4));
      }
      bool wide = false;
#pragma unroll
      for (int q = 0; q < kHeadRanks; ++q) wide |= all[q].y != 0.0f;
      float v = 0.0f;
#pragma unroll
      for (int q = 0; q < kHeadRanks; ++q) v += all[q].y == 0.0f && wide ? all[q].x * 0x1p-72f * 0x1p-72f : all[q].x;
      v /= static_cast<float>(a.d);
      // (beside such squares eps is nothing.)  The logits of a row that is large somewhere are summed in units of 2^72.
      const bool own = squares[tid].y != 0.0f;
      logits_by = wide ? rsqrtf(v) : rsqrtf(v + a.eps);
      r = wide && !own ? logits_by * 0x1p-72f : logits_by;
      parts_by = wide && !own ? 0x1p-72f : 1.0f;
    }
    scale[tid] = r;
    part_scale[tid] = parts_by;
    logit_scale[tid] = logits_by;
  }
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int off = kHeadCols / 4; off < 32; off <<= 1) acc[t][c] += __shfl_xor_sync(0xFFFFFFFFu, acc[t][c], off);
      if (lane < kHeadCols / 4) parts[warp][t][4 * cv + c] = acc[t][c];
    }
  __syncthreads();
  for (int at = tid; at < TT * kHeadCols; at += kFewThreads) {
    float v = 0.0f;
#pragma unroll
    for (int w8 = 0; w8 < kFewWarps; ++w8) v += (&parts[w8][0][0])[at];
    (&joined[0][0])[at] = v * part_scale[at / kHeadCols];
  }
  __syncthreads();
  cluster_arrive();  // the logits
  if (a.norm != nullptr) {
    for (int t = group; t < a.T; t += groups) {
      for (int i = tid * 8; i < count; i += kFewThreads * 8) {
        const float4 u = *reinterpret_cast<const float4*>(rows + t * share + i), v = *reinterpret_cast<const float4*>(rows + t * share + i + 4);
        const float r = scale[t];
        *reinterpret_cast<uint4*>(static_cast<T*>(a.y) + static_cast<int64_t>(t) * a.d + k_begin + i) =
            make_uint4(Elem<T>::pack2(u.x * r, u.y * r), Elem<T>::pack2(u.z * r, u.w * r), Elem<T>::pack2(v.x * r, v.y * r), Elem<T>::pack2(v.z * r, v.w * r));
      }
    }
  }
  __syncwarp();
  cluster_wait();
  if (a.router != nullptr) {
    // each CTA joins its share of the cluster's logits
    for (int at = tid * kHeadRanks + rank; at < TT * kHeadCols; at += kFewThreads * kHeadRanks) {
      const int t = at / kHeadCols, e = col0 + at % kHeadCols;
      if (t >= a.T || e >= a.E) continue;
      float part[kHeadRanks], v = 0.0f;
#pragma unroll
      for (int q = 0; q < kHeadRanks; ++q) part[q] = cluster_load(mapa_shared(smem_u32(&(&joined[0][0])[at]), q));
#pragma unroll
      for (int q = 0; q < kHeadRanks; ++q) v += part[q];
      a.logits[static_cast<int64_t>(t) * a.E + e] = v * logit_scale[t];
    }
  }
  __syncthreads();
  cluster_sync_all();  // the others' shared memory lives until it has been read
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
  int16_t expert[kFewSlots], first[kFewSlots];  // of an entry: its slots are slot[first] .. slot[first + count - 1]
  int16_t slot[kFewSlots], token[kFewSlots];    // and these slots' tokens
  uint8_t count[kFewSlots];
  int starts[kFewSlots / 32];
  uint32_t sums[kFewWarps];        // where a warp's sums of a unit are
  int entries;
  int go_on;
};

// All CTAs of the grid; false (and a status code) when one has not come in time.
__device__ __forceinline__ bool meet(const FewArgs& a, int turn, int* go_on) {
  __syncthreads();
  if (threadIdx.x == 0) {
    // what this CTA has written is published by the barrier above and this addition, what the others have is acquired by the last load
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(a.meeting) : "memory");
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
    *go_on = ok;
  }
  __syncthreads();
  return *go_on != 0;
}

template <typename V> __device__ __forceinline__ V share_of(float logit, bool sigmoid, float most, V sum) {
  if (sigmoid) return V(1) / (V(1) + exp(-static_cast<V>(logit)));
  return exp(static_cast<V>(logit) - static_cast<V>(most)) / sum;
}

// What a group is worth by the keys of its best two: the best one, or half the sum of both (which ranks as the sum does, and does not
// overflow).  Without a bias the keys are those of logits.  `size`: of the members, for what fp32 is off by.
template <typename V>
__device__ __forceinline__ V group_worth(const FewArgs& a, bool both, typename Order<V>::Key b0, typename Order<V>::Key b1, float most, V sum, V& size) {
  V v = Order<V>::value(b0), w = V(0);
  if (both) {
    w = Order<V>::value(b1);
    if (a.bias == nullptr) {
      v = share_of<V>(static_cast<float>(v), a.sigmoid != 0, most, sum);
      w = share_of<V>(static_cast<float>(w), a.sigmoid != 0, most, sum);
    }
    v *= V(0.5);
    w *= V(0.5);
  }
  size = fabs(v) + fabs(w);
  return v + w;
}

// The choice in 64 bits, all of it in shared memory: for the rare token whose values fp32 does not tell apart (one token, 64 experts in 8 groups: 7
// us more for the call, 256: 10, 1024: 20; all of 16 tokens 14, 23 and 70).  Leaves the experts and their shares; the lane's part of their sum.
__device__ __forceinline__ float choose_exactly(const FewArgs& a, int t, unsigned long long* keys, FewRouting& r, float most, int lane) {
  typedef Order<double> O;
  const float* from = a.logits + static_cast<int64_t>(t) * a.E;
  const bool sigmoid = a.sigmoid != 0;
  __syncwarp();  // the keys in 32 bits, which lie here, have been read
  double sum = 0.0;
  if (!sigmoid) {
    for (int e = lane; e < a.E; e += 32) sum += exp(static_cast<double>(from[e]) - static_cast<double>(most));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  }
  for (int e = lane; e < a.E; e += 32)
    keys[e] = O::key(a.bias != nullptr ? share_of<double>(from[e], sigmoid, most, sum) + static_cast<double>(a.bias[e]) : static_cast<double>(from[e]));
  __syncwarp();
  if (a.keep < a.groups) {
    const int width = a.E / a.groups;
    unsigned long long* const worth = keys + a.E;
    for (int g = lane; g < a.groups; g += 32) {
      unsigned long long b0 = 0, b1 = 0;
      for (int i = 0; i < width; ++i) {
        const unsigned long long k = keys[g * width + i], lower = k < b0 ? k : b0;
        b1 = lower > b1 ? lower : b1;
        b0 = k > b0 ? k : b0;
      }
      double size;
      worth[g] = O::key(group_worth<double>(a, a.best == 2 && width > 1, b0, b1, most, sum, size));
    }
    __syncwarp();
    for (int g = lane; g < a.groups; g += 32) {
      int before = 0;
      for (int o = 0; o < a.groups; ++o) before += worth[o] > worth[g] || (worth[o] == worth[g] && o < g);
      if (before >= a.keep)
        for (int i = 0; i < width; ++i) keys[g * width + i] = 0;
    }
    __syncwarp();
  }
  unsigned long long best = 0;
  int at = lane;
  const auto look = [&]() {
    best = 0;
    for (int e = lane; e < a.E; e += 32)
      if (keys[e] > best) best = keys[e], at = e;
  };
  look();
  float total = 0.0f;
  for (int s = 0; s < a.k; ++s) {
    const unsigned long long v = O::warp_max(best);
    const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == v ? static_cast<uint32_t>(at) : 0xFFFFu);
    if (e == static_cast<uint32_t>(at) && best == v) {
      const float share = static_cast<float>(share_of<double>(from[e], sigmoid, most, sum));
      r.id[t * a.k + s] = static_cast<int16_t>(e);
      r.score[t * a.k + s] = share;
      total += share;
      keys[e] = 0;
      look();
    }
  }
  return total;
}

// One warp, one token; expert lane + 32 i is the lane's i-th of up to EACH.  `keys`: scratch of this warp's own, [E] and [groups].  Leaves
// the experts, their shares, the largest logit and the lane's part of the shares' sum; false where the choice is to be made exactly.
//
// The logits decide where they are all that does (shares grow with them).  Where shares with a bias, or sums of two, are compared, the choice
// is that of exact arithmetic on the fp32 logits: values closer than what fp32 can be off by are decided again in 64 bits -- but for
// the router whose definition is in 32 bits (normalize 2).  Equal values by ascending index.  NaN is taken after everything else, or,
// where the softmax runs over the selected logits, before (the row is NaN then, as it is behind torch.topk).
template <int EACH> __device__ __forceinline__ bool choose(const FewArgs& a, int t, uint32_t* keys, FewRouting& r, float& most, float& total, int lane) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  typedef Order<float> O;
  const float* from = a.logits + static_cast<int64_t>(t) * a.E;
  const bool biased = a.bias != nullptr;
  float p[EACH];        // logit, then its share before normalisation
  float bias[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = lane + 32 * i;
    p[i] = e < a.E ? from[e] : -INFINITY;
    bias[i] = e < a.E && biased ? a.bias[e] : 0.0f;
  }
  uint32_t key[EACH];   // 0: no expert, or taken, or in a closed group
  float sum = 0.0f;
  most = -3.402823466e38f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    most = fmaxf(most, p[i]);
    key[i] = lane + 32 * i < a.E ? a.softmax_after && p[i] != p[i] ? kAll : O::key(p[i]) : 0u;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(kAll, most, off));
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    p[i] = a.sigmoid ? 1.0f / (1.0f + expf(-p[i])) : expf(p[i] - most);
    if (lane + 32 * i < a.E) sum += p[i];
  }
  if (!a.sigmoid && !a.softmax_after) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kAll, sum, off);
#pragma unroll
    for (int i = 0; i < EACH; ++i) p[i] /= sum;
  }
  if (biased) {
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (lane + 32 * i < a.E) key[i] = O::key(p[i] + bias[i]);
  }
  // How far a share can be off.  Sigmoid: the exponential by two units of 2^-23, which count with p (1 - p) <= 1/4, sum and quotient by
  // half a unit each.  Softmax: the same, a rounding per addition, and that of logit - most, which counts most (1/e) where it is -1.
  const float slack = a.sigmoid ? 3e-7f : (8e-7f + 1.2e-7f * EACH) / sum + 3e-8f;
  const bool exact = a.normalize != 2;
  bool sure = true;
  if (a.keep < a.groups) {
    const int width = a.E / a.groups;
    const bool both = a.best == 2 && width > 1;
    uint32_t* const worth = keys + a.E;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (lane + 32 * i < a.E) keys[lane + 32 * i] = key[i];
    __syncwarp();
    float off_by[2] = {};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int g = lane + 32 * j;
      if (g >= a.groups) continue;
      uint32_t b0 = 0, b1 = 0;
#pragma unroll 4
      for (int i = 0; i < width; ++i) {
        const uint32_t k = keys[g * width + i];
        b1 = max(b1, min(b0, k));
        b0 = max(b0, k);
      }
      float size;
      worth[g] = O::key(group_worth<float>(a, both, b0, b1, most, sum, size));
      // each member's slack and its rounding by 2^-24 of its size, the addition's and that of the bounds below by 2^-24 of the sum (an
      // infinite member is exact)
      off_by[j] = size < INFINITY ? slack + 2.4e-7f * size : 0.0f;
    }
    __syncwarp();
    uint32_t open[2] = {};  // groups 0..31, 32..63
    uint32_t worst = kAll, next = 0;  // the least that an open group can be worth, and the most that a closed one can
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int g = lane + 32 * j;
      bool is_open = false;
      if (g < a.groups) {
        const uint32_t mine = worth[g];
        int before = 0;
        for (int o = 0; o < a.groups; ++o) before += worth[o] > mine || (worth[o] == mine && o < g);
        is_open = before < a.keep;
        const float v = O::value(mine);
        if (is_open) worst = min(worst, O::key(v - off_by[j]));
        else next = max(next, O::key(v + off_by[j]));
      }
      open[j] = __ballot_sync(kAll, is_open);
    }
    if (exact && (biased || both)) {  // (closed groups of minus infinity or NaN are exact)
      worst = O::warp_min(worst);
      next = O::warp_max(next);
      sure = !(worst <= next && next > O::key(-INFINITY));
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int g = (lane + 32 * i) / width;
      if (((g < 32 ? open[0] : open[1]) >> (g & 31) & 1) == 0) key[i] = 0u;
    }
  }
  // k times the best of the lanes' best; only the lane that had it looks again
  uint32_t best;
  int at;
  float share;
  const auto look = [&]() {
    best = key[0], at = lane, share = p[0];
#pragma unroll
    for (int i = 1; i < EACH; ++i)
      if (key[i] > best) best = key[i], at = lane + 32 * i, share = p[i];
  };
  look();
  total = 0.0f;
  uint32_t last = 0;
  for (int s = 0; s < a.k; ++s) {
    last = __reduce_max_sync(kAll, best);
    const uint32_t e = __reduce_min_sync(kAll, best == last ? static_cast<uint32_t>(at) : 0xFFFFu);
    if (e == static_cast<uint32_t>(at)) {
      r.id[t * a.k + s] = static_cast<int16_t>(e);
      r.score[t * a.k + s] = share;
      total += share;
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (at == lane + 32 * i) key[i] = 0u;
      look();
    }
  }
  if (exact && biased) {  // the last that was taken and the first that was not
    const uint32_t next = O::warp_max(best);
    const float above = O::value(last), below = O::value(next);
    sure = sure && !(next != 0 && above - below <= 2.0f * slack + 1.2e-7f * (fabsf(above) + fabsf(below)));
  }
  return sure;
}

// Scores, experts, and the list of entries: up to eight slots of one expert each.  Entries of one expert follow one another (they read
// the same weights at the same time), experts by their first slots.  A function of its own, so that its registers are not the products': 1
// token on 8 experts of 4096 x 14336 in 4 bits 77 us on the device instead of 84, 16 of 64 of 7168 x 2048 318 instead of 322.
template <typename T> __device__ __noinline__ void route(const FewArgs& a, FewRouting& r, uint32_t* scratch) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slots = a.T * a.k;
  if (a.logits != nullptr) {
    uint32_t* const keys = scratch + warp * 2 * (a.E + a.groups);  // (room for 64-bit ones)
    for (int t = warp; t < a.T; t += kFewWarps) {
      float most, total;
      const bool sure = a.E <= 64 ? choose<2>(a, t, keys, r, most, total, lane) : a.E <= 256 ? choose<8>(a, t, keys, r, most, total, lane)
                                                                                 : choose<32>(a, t, keys, r, most, total, lane);
      if (!sure) total = choose_exactly(a, t, reinterpret_cast<unsigned long long*>(keys), r, most, lane);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
      __syncwarp();
      const float by = a.softmax_after ? total : a.normalize == 2 ? fmaxf(total, 1e-12f) : a.normalize == 1 ? total + 1e-20f : 1.0f;
      for (int s = lane; s < a.k; s += 32) r.score[t * a.k + s] = r.score[t * a.k + s] / by * (a.softmax_after ? 1.0f : a.scale);
      __syncwarp();
    }
  } else if (tid < slots) {
    const int64_t e = a.ids[tid];
    const bool ok = e >= 0 && e < a.E;
    if (!ok && a.status != nullptr) atomicCAS(a.status, 0, DS_BAD_EXPERT_ID);
    r.id[tid] = static_cast<int16_t>(ok ? e : -1);
    r.score[tid] = to_f32<T>(static_cast<const T*>(a.given)[tid]);
  }
  __syncthreads();
  // slots of an expert per warp, then where its slots and entries begin
  static_assert(kFewSlots == kFewThreads, "a slot per thread");
  uint8_t* const counts = reinterpret_cast<uint8_t*>(scratch);                               // [warp][E]
  int* const begins = reinterpret_cast<int*>(counts + kFewWarps * ((a.E + 15) / 16 * 16));   // [E]
  const int pitch = (a.E + 15) / 16 * 16;
  for (int i = tid; i < kFewWarps * pitch / 4; i += kFewThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0;
  __syncthreads();
  const int e = tid < slots ? r.id[tid] : -1;
  const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
  const int before = __popc(same & ((1u << lane) - 1));
  if (e >= 0 && before == 0) counts[warp * pitch + e] = static_cast<uint8_t>(__popc(same));
  __syncthreads();
  int rank = before, all = 0;  // among the slots of its expert
  if (e >= 0) {
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const int n = counts[w * pitch + e];
      all += n;
      if (w < warp) rank += n;
    }
  }
  const bool first = e >= 0 && rank == 0;
  int sum = first ? (all + kFewRows - 1) / kFewRows << 16 | all : 0;  // entries and slots up to here, then before
  const int own = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xFFFFFFFFu, sum, off);
    if (lane >= off) sum += o;
  }
  if (lane == 31) r.starts[warp] = sum;
  __syncthreads();
  int base = 0, everything = 0;
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    if (w < warp) base += r.starts[w];
    everything += r.starts[w];
  }
  if (first) begins[e] = base + sum - own;
  if (tid == 0) r.entries = everything >> 16;
  __syncthreads();
  if (e >= 0) {
    const int entry = begins[e] >> 16, at = begins[e] & 0xFFFF;
    r.slot[at + rank] = static_cast<int16_t>(tid);
    r.token[at + rank] = static_cast<int16_t>(tid / a.k);
    if (rank % kFewRows == 0) {
      const int n = entry + rank / kFewRows;
      r.expert[n] = static_cast<int16_t>(e);
      r.first[n] = static_cast<int16_t>(at + rank);
      r.count[n] = static_cast<uint8_t>(min(all - rank, kFewRows));
    }
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

// A format of weights: how a warp copies one step of a tile with the same columns of an entry's rows to shared memory, and multiplies them.
// A unit is an entry's rows by a tile of its expert's matrix, over a share of its steps.  It belongs to a team of 1, 2, 4 or 8 warps of a
// CTA; a team's warps take its steps in turn and join their sums.
struct FewMatrix {
  const void* w16;
  Q4Matrix w4;
  int K, N, steps;
  int cols, team, shares;  // columns of a tile; see share_out
};

// What gives the least to the team that has the most: `rounds` units of the steps of a warp and the joining, which costs about as much as
// `cost` steps.  Where the format has a choice, tiles of fewer columns (in eights, 16 to kCols; a step costs as much as eight columns more) make
// more units where there are few; shares of the depth, up to `most`, do too, and leave partial sums to the fold.  A lane per choice.
template <typename F> __device__ __forceinline__ void share_out(FewMatrix& m, int entries, int most, int lane) {
  constexpr int kWidths = (F::kCols - F::kNarrowest) / 8 + 1, kTeams = F::kLeastTeam == 8 ? 1 : 4, kAll = kWidths * kTeams * 3;
  uint32_t least = 0xFFFFFFFFu;
  for (int i = lane; i < kAll; i += 32) {
    const int cols = F::kCols - 8 * (i % kWidths), team = kFewWarps >> (i / kWidths % kTeams), shares = 1 << (i / kWidths / kTeams);
    if (shares > most) continue;
    const int tiles = (m.N + cols - 1) / cols, teams = static_cast<int>(gridDim.x) * (kFewWarps / team);
    const int rounds = (entries * tiles * shares + teams - 1) / teams;
    const uint32_t work = static_cast<uint32_t>(rounds) * ((m.steps + shares * team - 1) / (shares * team) + F::kCost + (shares > 1)) * (kWidths > 1 ? cols + 8 : 1);
    least = min(least, min(work, 0x1FFFFFFu) << 7 | i);
  }
  const int i = static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, least) & 127u);
  m.cols = F::kCols - 8 * (i % kWidths);
  m.team = kFewWarps >> (i / kWidths % kTeams);
  m.shares = 1 << (i / kWidths / kTeams);
}

// 16 bits, [K, N] with N contiguous: 16 rows of K by up to 64 columns.  The weights are the 16 rows of m16n8k16, transposed on their way from
// shared memory (ldmatrix); product q has columns 16 q .. 16 q + 15.  Eight lanes copy 128 bytes of one row (lanes in the order of the
// products, four rows to a quarter of a warp, made a request of every 16 bytes: 2.2 TB/s); in shared memory the 16-byte pieces of a row
// are turned by its number, so that the eight rows of a matrix lie in different banks.
template <typename T> struct FewWide {
  static constexpr int kCols = 64, kNarrowest = 16, kStep = 16, kDepth = 5, kProducts = 4, kCost = 4, kLeastTeam = 8;
  static constexpr int kRowsAt = kStep * kCols * 2, kStage = kRowsAt + kFewRows * kStep * 2;
  const uint16_t* w;   // the copy's: this lane's piece of the unit's first rows
  const uint16_t* x;   // this lane's piece of its row
  int64_t row;
  int K;
  bool inside;
  // the product's
  uint32_t weight_at, row_at;
  __device__ __forceinline__ void read(int count, int lane) {
    const int mine = lane & 7, k = mine + 8 * (lane >> 4);
    weight_at = k * 128 + ((((lane >> 3) & 1) ^ mine) << 4);   // product q: ^ 32 q
    const int g = lane >> 2;
    row_at = kRowsAt + (g < count ? g : 0) * 32 + (lane & 3) * 4;  // (rows behind the last give products that are nobody's)
  }
  template <typename Row> __device__ __forceinline__ void set(const FewMatrix& m, int expert, int tile, Row rows, int count, int lane) {
    const int piece = lane & 7, col = tile * m.cols + 8 * piece;
    inside = 8 * piece < m.cols && col < m.N;
    row = m.N;
    K = m.K;
    w = static_cast<const uint16_t*>(m.w16) + (static_cast<int64_t>(expert) * K + (lane >> 3)) * row + col;
    x = (lane >> 1) < count ? rows(lane >> 1) + 8 * (lane & 1) : nullptr;
  }
  __device__ __forceinline__ void copy(uint32_t stage, int step, int lane) const {
    if (!inside) return;
    const int r = lane >> 3;
    const uint32_t to = stage + r * 128;
    const uint16_t* from = w + step * kStep * row;
    if (step * kStep + kStep <= K) {
#pragma unroll
      for (int j = 0; j < 4; ++j) copy_16(to + j * 512 + (((lane & 7) ^ ((r + 4 * j) & 7)) << 4), from + 4 * j * row);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool real = step * kStep + r + 4 * j < K;
        copy_16_or_zeros(to + j * 512 + (((lane & 7) ^ ((r + 4 * j) & 7)) << 4), real ? from + 4 * j * row : w, real);
      }
    }
  }
  __device__ __forceinline__ void copy_rows(uint32_t stage, int, int step, int lane) const {
    const int k = step * kStep;
    const bool real = k + 8 * (lane & 1) < K;
    if (x != nullptr) copy_16_or_zeros(stage + kRowsAt + lane * 16, real ? x + k : x - 8 * (lane & 1), real);
  }
  __device__ __forceinline__ void multiply(float (&acc)[kProducts][4], uint32_t stage, int) const {
    const uint32_t b0 = lds_32(stage + row_at), b1 = lds_32(stage + row_at + 16);
#pragma unroll
    for (int q = 0; q < kProducts; ++q) {
      uint32_t a[4];
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                   : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                   : "r"(stage + (weight_at ^ (32 * q))));
      mma_16x8x16<T>(acc[q], a, b0, b1);
    }
  }
  // column of the tile that value c of product q belongs to
  __device__ static __forceinline__ int column(int q, int c, int lane) { return 16 * q + (lane >> 2) + 8 * (c >> 1); }
};

// 4 bits (int4.cuh): 32 rows of the weight by 128 columns.
template <typename T, int NG, bool ZEROS> struct FewFour {
  static constexpr int kCols = kQ4Cols, kNarrowest = kCols, kStep = kQ4Step, kDepth = 3, kProducts = kQ4Tiles, kCost = 2, kLeastTeam = 1;
  static constexpr int kStage = Q4Stage<NG, ZEROS>::kBytes, kBlock = Q4Stage<NG, ZEROS>::kBlock;
  const uint8_t* block;
  int64_t apart;
  const uint16_t* x[4];
  int K;
  uint32_t row_at;
  __device__ __forceinline__ void read(int count, int lane) { row_at = q4_row_at(count, lane); }
  template <typename Row> __device__ __forceinline__ void set(const FewMatrix& m, int expert, int tile, Row rows, int count, int lane) {
    block = m.w4.data + (expert * m.w4.tiles + kQ4Tiles * tile) * m.w4.steps * kBlock + lane * 16;
    apart = kQ4Tiles * tile + 1 < m.w4.tiles ? static_cast<int64_t>(m.w4.steps) * kBlock : 0;
    K = m.K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 2 * i + (lane >> 4);
      if (2 * i < count) x[i] = rows(r < count ? r : 0) + 8 * (lane & 15);
    }
  }
  __device__ __forceinline__ void copy(uint32_t stage, int step, int lane) const {
    q4_copy<NG, ZEROS>(stage, block + static_cast<int64_t>(step) * kBlock, apart, lane);
  }
  __device__ __forceinline__ void copy_rows(uint32_t stage, int count, int step, int lane) const {
    q4_copy_rows<NG, ZEROS>(stage, x, count, K, step * kStep, lane);
  }
  __device__ __forceinline__ void multiply(float (&acc)[kProducts][4], uint32_t stage, int lane) const {
    q4_step<T, NG, ZEROS>(acc, stage, row_at, lane);
  }
  __device__ static __forceinline__ int column(int q, int c, int lane) { return kQ4Rows * q + (lane >> 2) + 8 * (c >> 1); }
};

template <typename F> struct FewPlan {
  static constexpr int kRing = F::kDepth * F::kStage;
  static constexpr int kTotal = kFewWarps * kRing;
  static_assert(kFewRows * F::kCols * 4 <= F::kStage, "a warp's sums of a unit, [row][column], lie in the stage that it has read last");
  static_assert(kFewWarps * (kFewExperts + kFewGroups) * 8 <= kTotal && kFewWarps * kFewExperts + 4 * kFewExperts <= kTotal,
                "the router's keys lie where the rings will be");
};

// The warps of a team (of a CTA's; more than one warp).
__device__ __forceinline__ void team_sync(int team, int warp) {
  if (team == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / team), "r"(32 * team) : "memory");
}

// The units of one product.  A warp's copies run ahead of its products by up to kDepth - 1 steps, into the next units, so that nothing
// waits for memory while a unit's sums are joined.
template <typename F> struct FewWalk {
  const FewMatrix m;
  const FewRouting& r;
  const uint16_t* source;  // the rows, and which of them belong to the entries' slots
  const int16_t* which;
  int tiles, units, teams;
  int warp, lane;
  // where the copies are
  F f;
  int unit, step, end, count;

  __device__ __forceinline__ int first_unit() const { return warp / m.team * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x); }  // CTAs in turn
  __device__ __forceinline__ void place(int u, int& entry, int& tile, int& share) const {
    entry = u / (tiles * m.shares);
    const int rest = u - entry * tiles * m.shares;
    share = rest / tiles;
    tile = rest - share * tiles;
  }
  // this warp's steps of a share
  __device__ __forceinline__ int begin_of(int share) const { return m.steps * share / m.shares + warp % m.team; }
  __device__ __forceinline__ int end_of(int share) const { return m.steps * (share + 1) / m.shares; }
  __device__ __forceinline__ void seek() {  // the unit's first step of this warp's, or the next unit that has one
    while (unit < units) {
      int n, tile, share;
      place(unit, n, tile, share);
      step = begin_of(share);
      end = end_of(share);
      if (step < end) {
        count = r.count[n];
        const int first = r.first[n];
        f.set(m, r.expert[n], tile, [&](int i) { return source + static_cast<int64_t>(which[first + i]) * m.K; }, count, lane);
        return;
      }
      unit += teams;
    }
  }
  __device__ __forceinline__ void start() {
    unit = first_unit();
    seek();
  }
  __device__ __forceinline__ void advance() {
    step += m.team;
    if (step >= end) {
      unit += teams;
      seek();
    }
  }
  __device__ __forceinline__ void copy(uint32_t to, bool weights, bool rows) {  // one step, and on to the next
    if (unit >= units) return;
    if (weights) f.copy(to, step, lane);
    if (rows) f.copy_rows(to, count, step, lane);
    advance();
  }
};

template <typename T, typename F>
__global__ void __launch_bounds__(kFewThreads, kFewCtas) few_experts_kernel(const __grid_constant__ FewArgs a) {
  using P = FewPlan<F>;
  constexpr bool WIDE = F::kCols == 64;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ FewRouting r;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(smem), ring = warp * P::kRing;  // the ring's place in it
  route<T>(a, r, reinterpret_cast<uint32_t*>(smem));
  const bool gated = a.act == MOE_ACT_SWIGLU || a.act == MOE_ACT_GEGLU;
  const int slots = a.T * a.k;
  // All units of a product whose first copies are under way; `give` takes a unit's sums: (entry, tile, share, thread of the team,
  // the team's threads, total(row, column)).
  const auto walk = [&](FewWalk<F>& c, auto give) {
    F f;
    uint32_t from = ring, spent = ring + (F::kDepth - 1) * F::kStage;
    const int team = c.m.team, mine = warp % team * 32 + lane;
    const uint32_t* const sums = r.sums + (warp - warp % team);
#pragma unroll 1
    for (int unit = c.first_unit(); unit < c.units; unit += c.teams) {
      int n, tile, share;
      c.place(unit, n, tile, share);
      const int count = r.count[n], end = c.end_of(share);
      f.read(count, lane);
      float acc[F::kProducts][4] = {};
#pragma unroll 1
      for (int step = c.begin_of(share); step < end; step += team) {
        copies_wait<F::kDepth - 2>();
        __syncwarp();  // every lane's copies of this step, and every lane is through with the stage that is filled next
        c.copy(base + spent, true, true);
        copies_commit();
        f.multiply(acc, base + from, lane);
        spent = from;
        from = from == ring + (F::kDepth - 1) * F::kStage ? ring : from + F::kStage;
      }
      __syncwarp();  // every lane is through with the last stage, where the sums go
#pragma unroll
      for (int q = 0; q < F::kProducts; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 2 * (lane & 3) + (i & 1);
          if (row < count) reinterpret_cast<float*>(smem + spent)[row * F::kCols + F::column(q, i, lane)] = acc[q][i];
        }
      if (lane == 0) r.sums[warp] = spent;
      team_sync(team, warp);
      give(n, tile, share, mine, team * 32, [&](int row, int col) {
        float v = 0.0f;
        for (int w = 0; w < team; ++w) v += reinterpret_cast<const float*>(smem + sums[w])[row * F::kCols + col];
        return v;
      });
      team_sync(team, warp);
    }
    copies_wait<0>();
    __syncwarp();
  };
  const auto open = [&](const FewMatrix& m, const uint16_t* source, const int16_t* which) {
    const int tiles = (m.N + m.cols - 1) / m.cols;
    FewWalk<F> c{m, r, source, which, tiles, r.entries * tiles * m.shares, static_cast<int>(gridDim.x) * (kFewWarps / m.team), warp, lane};
    c.start();
    return c;
  };

  {
    FewMatrix up{a.w1, a.up, a.d, gated ? 2 * a.I : a.I, (a.d + F::kStep - 1) / F::kStep, F::kCols, kFewWarps, 1};
    share_out<F>(up, r.entries, 1, lane);
    auto c = open(up, static_cast<const uint16_t*>(a.x), r.token);
#pragma unroll 1
    for (int s = 0; s < F::kDepth - 1; ++s) {
      c.copy(base + ring + s * F::kStage, true, true);
      copies_commit();
    }
    const int cols = gated ? up.cols / 2 : up.cols;
    walk(c, [&](int n, int tile, int, int thread, int threads, auto total) {
      const int count = r.count[n];
      for (int at = thread; at < count * cols; at += threads) {
        const int row = at / cols, col = at - row * cols;
        const int i = tile * cols + col;
        if (i >= a.I) continue;
        // gate and up columns in turn, or (4 bits) in eights
        const int gate = !gated ? col : WIDE ? 2 * col : 2 * col - col % 8;
        float v = few_act(total(row, gate), a.act);
        if (gated) v *= total(row, gate + (WIDE ? 1 : 8));
        const T h = Elem<T>::from_float(v);
        a.hidden[static_cast<int64_t>(r.slot[r.first[n] + row]) * a.I + i] = *reinterpret_cast<const uint16_t*>(&h);
      }
    });
  }

  FewMatrix down{a.w2, a.down, a.I, a.d, (a.I + F::kStep - 1) / F::kStep, F::kCols, kFewWarps, 1};
  share_out<F>(down, r.entries, kFewParts, lane);
  const int shares = down.shares;
  {
    // the first weights of the down product are asked for before the wait for the rows that they multiply
    auto ahead = open(down, a.hidden, r.slot);
    auto c = ahead;
#pragma unroll 1
    for (int s = 0; s < F::kDepth - 1; ++s) ahead.copy(base + ring + s * F::kStage, true, false);
    if (!meet(a, 1, &r.go_on)) {
      copies_wait<0>();
      return;
    }
#pragma unroll 1
    for (int s = 0; s < F::kDepth - 1; ++s) {
      c.copy(base + ring + s * F::kStage, false, true);
      copies_commit();
    }
    walk(c, [&](int n, int tile, int share, int thread, int threads, auto total) {
      const int count = r.count[n], cols = down.cols;
      for (int at = thread; at < count * cols; at += threads) {
        const int row = at / cols, col = at - row * cols;
        const int i = tile * cols + col;
        if (i < a.d) a.rows[(static_cast<int64_t>(share) * slots + r.slot[r.first[n] + row]) * a.d + i] = total(row, col);
      }
    });
  }
  if (!meet(a, 2, &r.go_on)) return;

  for (int at = blockIdx.x * kFewThreads + tid; at < a.T * a.d; at += gridDim.x * kFewThreads) {
    const int t = at / a.d, i = at - t * a.d;
    float v = a.addend != nullptr ? to_f32<T>(static_cast<const T*>(a.addend)[at]) : 0.0f;
    const float* from = a.rows + static_cast<int64_t>(t) * a.k * a.d + i;
    const int64_t share = static_cast<int64_t>(slots) * a.d;
    for (int s0 = 0; s0 < a.k; s0 += 4) {  // four slots' loads at once
      float part[4][kFewParts];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int p = 0; p < kFewParts; ++p)
          part[s][p] = s0 + s < a.k && p < shares && r.id[t * a.k + s0 + s] >= 0 ? from[(s0 + s) * static_cast<int64_t>(a.d) + p * share] : 0.0f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float row = part[s][0];
#pragma unroll
        for (int p = 1; p < kFewParts; ++p) row += part[s][p];
        if (s0 + s < a.k && r.id[t * a.k + s0 + s] >= 0) v = fmaf(r.score[t * a.k + s0 + s], row, v);
      }
    }
    static_cast<T*>(a.out)[at] = Elem<T>::from_float(v);
  }
}

template <typename T, typename W, int TT> static int launch_head(const HeadArgs& a, cudaStream_t s) {
  const auto kernel = few_head_kernel<T, W, TT>;
  static std::atomic<bool> prepared[64];
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !prepared[dev].load(std::memory_order_acquire)) {
    MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TT * kHeadMost / kHeadRanks * 4));
    if (dev < 64) prepared[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  const int tiles = a.router == nullptr ? 1 : (a.E + kHeadCols - 1) / kHeadCols;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * kHeadRanks), 1, 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(TT) * ((a.d + kHeadRanks * 8 - 1) / (kHeadRanks * 8) * 8) * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kHeadRanks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return MOE_OK;
}
template <typename T, typename W> static int launch_head_tokens(const HeadArgs& a, cudaStream_t s) {
  if (a.T == 1) return launch_head<T, W, 1>(a, s);
  if (a.T <= 4) return launch_head<T, W, 4>(a, s);
  return launch_head<T, W, 16>(a, s);
}

// One wave: what of the grid's CTAs fit at once, at most kFewCtas per SM.
template <typename T, typename F> static int launch_experts(const FewArgs& a, cudaStream_t s) {
  constexpr int smem = FewPlan<F>::kTotal;
  const auto kernel = few_experts_kernel<T, F>;
  static std::atomic<int> resident[64];
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  int ctas = dev < 64 ? resident[dev].load(std::memory_order_acquire) : 0;
  if (ctas == 0) {
    MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    MOE_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, kFewThreads, smem));
    MOE_CHECK_ARG(ctas > 0, "moe_few_tokens: the kernel does not fit on an SM");
    if (ctas > kFewCtas) ctas = kFewCtas;
    if (dev < 64) resident[dev].store(ctas, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * sm_count()), 1, 1);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return MOE_OK;
}
template <typename T> static int launch_experts_of(const FewArgs& a, int bits, int group, bool z, cudaStream_t s) {
  if (bits == 16) return launch_experts<T, FewWide<T>>(a, s);
  if (group == 128) return z ? launch_experts<T, FewFour<T, 1, true>>(a, s) : launch_experts<T, FewFour<T, 1, false>>(a, s);
  if (group == 64) return z ? launch_experts<T, FewFour<T, 2, true>>(a, s) : launch_experts<T, FewFour<T, 2, false>>(a, s);
  return z ? launch_experts<T, FewFour<T, 4, true>>(a, s) : launch_experts<T, FewFour<T, 4, false>>(a, s);
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
  if ((p->router_w != nullptr || p->norm_w != nullptr) && p->d > kHeadMost) {
    set_error("moe_few_tokens: norm and router take rows of at most %d, got %d", kHeadMost, p->d);
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
  MOE_CHECK_ARG(p->norm_w == nullptr || p->norm_dtype == 2 || p->norm_dtype == p->dtype, "moe_few_tokens: norm_w is in fp32 or the rows' type, got %d",
                p->norm_dtype);
  if (p->num_tokens == 0) return MOE_OK;
  MOE_CHECK_ARG(p->x && p->w1 && p->w2 && p->out && p->workspace, "moe_few_tokens: null pointer argument");
  MOE_CHECK_ARG(p->residual == nullptr || (p->norm_w != nullptr && p->stream_out != nullptr), "moe_few_tokens: a residual goes with a norm and the stream");
  uintptr_t all = 0;
  for (const void* q : {p->x, p->residual, p->norm_w, p->w1, p->w2, p->router_w, p->addend,
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
    const auto matrix = [&](const void* data, int n, int k) {
      return Q4Matrix{static_cast<const uint8_t*>(data), (n + kQ4Rows - 1) / kQ4Rows, (k + kQ4Step - 1) / kQ4Step};
    };
    a.up = matrix(p->w1, glu ? 2 * p->inter : p->inter, p->d);
    a.down = matrix(p->w2, p->d, p->inter);
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
  return bf16 ? launch_experts_of<__nv_bfloat16>(a, p->bits, p->group, p->zeros != 0, s)
              : launch_experts_of<__half>(a, p->bits, p->group, p->zeros != 0, s);
}
