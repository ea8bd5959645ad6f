// Routing of tokens to experts that live in groups: scores, a bias for balance, the best groups, top-k inside them,
// renormalised weights -- and the gradient of the logits.
//
//   p = sigmoid(l) or softmax(l);  c = p + bias (selection only);  a group's score = sum of its best one or two c;
//   the `keep` best groups stay open;  the k best c of the open groups;  w = scale * p / (sum of the k p + 1e-20) or scale * p
//
// One warp per token, one launch; the logits are read once.  The experts of a group lie on neighbouring lanes in ascending order
// (group g on lanes [g*L, (g+1)*L), L the largest power of two that gives every group its lanes), so a group's best two are log2(L)
// exchanges, its rank one comparison with every other group's score, and "the lowest index of equal values" is "the lowest
// lane, then the lowest register".
//
// THE CHOICE IS THAT OF EXACT ARITHMETIC.  Values whose fp32 images are closer than what the evaluation in fp32 can be off by
// are decided again in 64 bits, by the warp that met them: about one token in 1500 for 256 sigmoid scores with a bias, but every
// token that has equal values among those that decide, as a third have with 16-bit logits and a bias of zeros.  Indices then
// depend neither on the order of a softmax's sum nor on the exponential's last bit.  Without a bias the logits
// themselves are compared (p grows with l), and only sums over two members of a group can be that close.
// Ties go to the lowest index, the k results come in descending order, NaN is taken after everything else.
//
// Bound by the instructions, about 1100 per token: 16384 tokens with 256 experts in 8 groups and a bias take 24 to 28 us (the logits
// pass HBM in 3), one token 5 us, most of which are the launch and the chain of the rounds.  A token that is decided again in 64
// bits takes 5 us more, beside the others: 16384 tokens with 16-bit logits 27 us, 45 where the bias is zeros, 22 without one.
#include "order.cuh"

namespace moe {

constexpr int kTopkWarps = 4;  // warps (tokens) per CTA: small, so that few tokens spread over the SMs
constexpr unsigned kAll = 0xFFFFFFFFu;

struct TopkArgs {
  const void* logits;
  const float* bias;
  void* scores;
  int64_t* indices;
  int64_t num_tokens;
  int num_experts, group_size, num_groups, keep, best, topk;
  int lanes_log2;  // lanes of a group
  int per_lane;    // experts of a lane (the last lanes of a group may have fewer)
  int sigmoid, normalize, scores_dtype;
  float scale;
};

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

template <typename T> __device__ __forceinline__ float load_elem(const T* p) { return Elem<T>::to_float(*p); }
template <> __device__ __forceinline__ float load_elem<float>(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ void store_elem(T* p, float v) { *p = Elem<T>::from_float(v); }
template <> __device__ __forceinline__ void store_elem<float>(float* p, float v) { *p = v; }

template <typename V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(kAll, v, off);
  return v;
}

// p of one logit; `top` and `sum` are the softmax's.
template <typename V> __device__ __forceinline__ V score_of(float x, bool sigmoid, float top, V sum) {
  if (sigmoid) return V(1) / (V(1) + exp_of(-static_cast<V>(x)));
  return exp_of(static_cast<V>(x) - static_cast<V>(top)) / sum;
}

// p as the choice in fp32 takes it: a sigmoid of the hardware's power of two and reciprocal, one instruction each.  The power is off by
// 2 units of 2^-23, its rounded argument -x log2(e) by another 0.6 |x|, the sum by half a unit and the reciprocal by one; the first
// two count with p (1 - p), and p (1 - p) (2 + 0.6 |x|) < 0.6: off by less than (0.6 + 1.5) 2^-23 < 2.6e-7.  (A softmax would add E
// such errors up: it does not use them.)
constexpr float kSigmoidSlack = 4e-7f;
__device__ __forceinline__ float key_score(float x, bool sigmoid, float top, float sum) {
  if (!sigmoid) return score_of<float>(x, false, top, sum);
  float e, p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.0f + e));
  return p;
}
__device__ __forceinline__ double key_score(float x, bool sigmoid, float top, double sum) { return score_of<double>(x, sigmoid, top, sum); }

// The logits (or biases) of a lane.
template <typename T, int PER>
__device__ __forceinline__ void load_logits(const TopkArgs& a, const T* row, int first, int count, float (&x)[PER]) {
  constexpr int kVec = 16 / sizeof(T);
  // whole 16-byte pieces where every lane's experts begin on one (a multiple of per_lane = PER elements from the row's beginning)
  if constexpr (PER % kVec == 0) {
    if (a.per_lane == PER && a.group_size % kVec == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0 && count == PER) {
#pragma unroll
      for (int i = 0; i < PER; i += kVec) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + first + i);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[i + j] = load_elem(e + j);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = i < count ? load_elem(row + first + i) : 0.0f;
}

// The best two of a lane's keys, the lower index first where they are equal.
template <typename Key, int PER>
__device__ __forceinline__ void best_two(const Key (&key)[PER], Key& m1, int& i1, Key& m2, int& i2) {
  m1 = m2 = 0;
  i1 = i2 = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool first = key[i] > m1, second = key[i] > m2;
    m2 = first ? m1 : second ? key[i] : m2;
    i2 = first ? i1 : second ? i : i2;
    m1 = first ? key[i] : m1;
    i1 = first ? i : i1;
  }
}
// The key after (last, last_at) in the order of the results: value descending, index ascending.
template <typename Key, int PER>
__device__ __forceinline__ void best_after(const Key (&key)[PER], Key last, int last_at, Key& m, int& at) {
  m = 0;
  at = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const Key below = last + (i > last_at ? 1 : 0);  // (no key is the type's largest number)
    if (key[i] < below && key[i] > m) {
      m = key[i];
      at = i;
    }
  }
}

// The choice: lane s < topk gets the s-th expert and its p.  False (fp32 only): two values that decide are too close to tell.
// Each lane holds its best two; a round takes the largest of the lanes' first ones, and a lane that has given both looks through
// its keys again (with 8 of 256 about every fourth token has such a lane).
template <typename T, typename V, int PER>
__device__ __forceinline__ bool choose(const TopkArgs& a, const T* row, int first, int count, float top, int& my_expert, V& my_p,
                                       const float (&x)[PER], int* taken) {
  typedef Order<V> O;
  typedef typename O::Key Key;
  const int lane = threadIdx.x & 31;
  const bool sigmoid = a.sigmoid != 0;
  const bool biased = a.bias != nullptr;
  constexpr bool kFirst = sizeof(V) == 4;
  V sum = V(0);
  if (!sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < count) sum += exp_of(static_cast<V>(x[i]) - static_cast<V>(top));
    sum = warp_sum(sum);
  }
  // how far p in fp32 may be off: exp, sum and division at a few units each, the sum of the softmax by one more per addition, and
  // the rounding of l - max, whose effect on p is largest (1/e) where l - max is -1
  const float p_top = sigmoid ? 1.0f : 1.0f / static_cast<float>(sum);
  const float slack = sigmoid ? kSigmoidSlack : p_top * (8e-7f + 1.2e-7f * PER) + 3e-8f;
  Key key[PER];
  if (biased) {
    float b[PER];
    load_logits<float, PER>(a, a.bias, first, count, b);
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = i < count ? O::key(key_score(x[i], sigmoid, top, sum) + static_cast<V>(b[i])) : Key(0);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = i < count ? O::key(static_cast<V>(x[i])) : Key(0);
  }
  bool sure = true;
  Key m1, m2;
  int i1, i2;
  best_two(key, m1, i1, m2, i2);
  if (a.keep < a.num_groups) {
    Key g1 = m1, g2 = m2;
    for (int off = (1 << a.lanes_log2) >> 1; off > 0; off >>= 1) {
      const Key o1 = __shfl_xor_sync(kAll, g1, off), o2 = __shfl_xor_sync(kAll, g2, off);
      const Key lower = o1 < g1 ? o1 : g1;
      g2 = g2 > o2 ? g2 : o2;
      g2 = lower > g2 ? lower : g2;
      g1 = o1 > g1 ? o1 : g1;
    }
    const int group = lane >> a.lanes_log2;
    Key mine = 0;
    float off_by = 0.0f;  // what the group's score in fp32 may be off by
    if (group < a.num_groups) {
      V v = O::value(g1);
      if (a.best == 2) {
        V w = O::value(g2);
        if (!biased) {
          v = key_score(static_cast<float>(v), sigmoid, top, sum);
          w = key_score(static_cast<float>(w), sigmoid, top, sum);
        }
        // (half the sum ranks as the sum does, and does not overflow)
        v = V(0.5) * v;
        w = V(0.5) * w;
        if (kFirst) {
          // each member's slack and its rounding to fp32 by 2^-24 of ITS size, the addition's and that of the bounds below by 2^-24 of
          // the sum: members that cancel leave a small sum with the large ones' roundings.  (An infinite member is exact.)
          const float size = fabsf(static_cast<float>(v)) + fabsf(static_cast<float>(w));
          off_by = size < CUDART_INF_F ? slack + 2.4e-7f * size : 0.0f;
        }
        v += w;
      } else if (kFirst) {
        const float size = fabsf(static_cast<float>(v));
        off_by = size < CUDART_INF_F ? slack + 2.4e-7f * size : 0.0f;
      }
      mine = O::key(v);
    }
    // groups before this one; the comparisons are shared out to its lanes
    int rank = 0;
    const int lanes = 1 << a.lanes_log2;
    for (int g0 = 0; g0 < a.num_groups; g0 += lanes) {
      const int g = g0 + (lane & (lanes - 1));
      const Key other = __shfl_sync(kAll, mine, g << a.lanes_log2);
      rank += g < a.num_groups && (other > mine || (other == mine && g < group));
    }
    for (int off = lanes >> 1; off > 0; off >>= 1) rank += __shfl_xor_sync(kAll, rank, off);
    const bool open = group < a.num_groups && rank < a.keep;
    if (kFirst && (biased || a.best == 2)) {
      // the least that an open group can have, and the most that a closed one can; closed ones of minus infinity (masked) or NaN
      // are exact: what they are compared with is larger, or equal and decided by index
      const Key worst = O::warp_min(open ? O::key(static_cast<V>(static_cast<float>(O::value(mine)) - off_by)) : ~Key(0));
      const Key next = O::warp_max(open || group >= a.num_groups ? Key(0) : O::key(static_cast<V>(static_cast<float>(O::value(mine)) + off_by)));
      if (worst <= next && next > O::key(static_cast<V>(-CUDART_INF_F))) sure = false;
    }
    if (!open) m1 = m2 = 0;
  }
  // k rounds of the largest value left, and one more to see how close the next one came
  Key mine = 0, last = 0;  // lane s: the s-th largest
  int left = count;
  const unsigned before = (1u << lane) - 1u;
  const int rounds = kFirst && biased ? a.topk + 1 : a.topk;
  for (int s = 0; s < rounds; ++s) {
    last = O::warp_max(m1);
    const unsigned equal = __ballot_sync(kAll, m1 == last);
    if (lane == s) mine = last;
    const int at = i1;
    bool again = false;
    if (m1 == last && (equal & before) == 0) {  // the first lane that has it
      if (s < a.topk) taken[s] = first + i1;
      m1 = m2;
      i1 = i2;
      m2 = 0;
      again = --left > 0 && m1 == 0 && last != 0;
    }
    if (__any_sync(kAll, again)) {
      Key next;
      int next_at;
      best_after(key, last, at, next, next_at);
      if (again) {
        m1 = next;
        i1 = next_at;
      }
    }
  }
  __syncwarp();
  if (lane < a.topk) my_expert = taken[lane];
  __syncwarp();  // (it is written again by the choice in 64 bits)
  if (kFirst && biased) {
    Key next = __shfl_down_sync(kAll, mine, 1);
    if (lane == a.topk - 1) next = last;
    const float above = static_cast<float>(O::value(mine)), below = static_cast<float>(O::value(next));
    const bool close = lane < a.topk && next != 0 && above - below <= 2.0f * slack + 1.2e-7f * (fabsf(above) + fabsf(below));
    sure = sure && !__any_sync(kAll, close);
  }
  my_p = V(0);
  if (lane < a.topk) my_p = score_of<V>(load_elem(row + my_expert), sigmoid, top, sum);
  return sure;
}

// The rare token again, in 64 bits; a function of its own, so that its registers are not everyone's.
template <typename T, int PER>
__device__ __noinline__ double choose_exactly(const TopkArgs& a, const T* row, int first, int count, float top, int* expert,
                                              int* taken) {
  float x[PER];
  load_logits<T, PER>(a, row, first, count, x);
  double p;
  int e = 0;
  choose<T, double, PER>(a, row, first, count, top, e, p, x, taken);
  *expert = e;
  return p;
}

template <typename V>
__device__ __forceinline__ void store_weight(const TopkArgs& a, int64_t token, int expert, V p) {
  const int lane = threadIdx.x & 31;
  const V sum = warp_sum(lane < a.topk ? p : V(0)) + V(1e-20);
  if (lane >= a.topk) return;
  const float w = static_cast<float>((a.normalize ? p / sum : p) * static_cast<V>(a.scale));
  const int64_t at = token * a.topk + lane;
  if (a.scores_dtype == MOE_DTYPE_F32) static_cast<float*>(a.scores)[at] = w;
  else if (a.scores_dtype == MOE_DTYPE_BF16) static_cast<__nv_bfloat16*>(a.scores)[at] = __float2bfloat16_rn(w);
  else static_cast<__half*>(a.scores)[at] = __float2half_rn(w);
  a.indices[at] = expert;
}

template <typename T, int PER>
__global__ void __launch_bounds__(kTopkWarps * 32) grouped_topk_kernel(const __grid_constant__ TopkArgs a) {
  __shared__ int all_taken[kTopkWarps][32];
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kTopkWarps + (threadIdx.x >> 5);
  if (token >= a.num_tokens) return;
  const int lane = threadIdx.x & 31;
  int* taken = all_taken[threadIdx.x >> 5];
  const T* row = static_cast<const T*>(a.logits) + token * a.num_experts;
  const int group = lane >> a.lanes_log2;
  const int member = (lane & ((1 << a.lanes_log2) - 1)) * a.per_lane;
  const int left = group < a.num_groups ? a.group_size - member : 0;
  const int count = left < 0 ? 0 : left < a.per_lane ? left : a.per_lane;
  const int first = count > 0 ? group * a.group_size + member : 0;
  float x[PER];
  load_logits<T, PER>(a, row, first, count, x);
  float top = 0.0f;
  if (!a.sigmoid) {
    top = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < count) top = fmaxf(top, x[i]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, off));
  }
  int expert = 0;
  float p;
  if (choose<T, float, PER>(a, row, first, count, top, expert, p, x, taken)) {
    store_weight(a, token, expert, p);
  } else {
    int exact = 0;
    const double q = choose_exactly<T, PER>(a, row, first, count, top, &exact, taken);
    store_weight(a, token, exact, q);
  }
}

// d_logits of d_scores, given the selection.  With s_i = p_i of the selection, S = sum s + 1e-20:
//   d_p_i = scale * (g_i - sum_j g_j s_j / S) / S (normalised) or scale * g_i;  0 outside the selection
//   sigmoid: d_l = d_p p (1 - p);   softmax: d_l = p (d_p - sum_j d_p_j p_j)
// The few values of the selection are worked out in 64 bits: their differences cancel.  Bound by the write of d_logits.
template <typename T>
__global__ void __launch_bounds__(kTopkWarps * 32)
grouped_topk_backward_kernel(const T* logits, const int64_t* indices, const void* d_scores, T* d_logits, int64_t num_tokens,
                             int num_experts, int topk, int sigmoid, int normalize, float scale, int scores_dtype) {
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kTopkWarps + (threadIdx.x >> 5);
  if (token >= num_tokens) return;
  const int lane = threadIdx.x & 31;
  const T* row = logits + token * num_experts;
  T* out = d_logits + token * num_experts;
  const int64_t at = token * topk + lane;
  int64_t expert = 0;
  double g = 0.0;
  if (lane < topk) {
    expert = indices[at];
    if (scores_dtype == MOE_DTYPE_F32) g = static_cast<const float*>(d_scores)[at];
    else if (scores_dtype == MOE_DTYPE_BF16) g = __bfloat162float(static_cast<const __nv_bfloat16*>(d_scores)[at]);
    else g = __half2float(static_cast<const __half*>(d_scores)[at]);
    g *= static_cast<double>(scale);
  }
  float top = 0.0f, sum = 0.0f;
  if (!sigmoid) {
    top = -CUDART_INF_F;
    for (int e = lane; e < num_experts; e += 32) top = fmaxf(top, load_elem(row + e));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, off));
    for (int e = lane; e < num_experts; e += 32) sum += expf(load_elem(row + e) - top);
    sum = warp_sum(sum);
  }
  double p = 0.0;
  if (lane < topk) p = score_of<double>(load_elem(row + expert), sigmoid != 0, top, static_cast<double>(sum));
  if (normalize) {
    const double total = warp_sum(p) + 1e-20;
    const double along = warp_sum(g * (p / total));
    g = (g - along) / total;
  }
  const float along = sigmoid ? 0.0f : static_cast<float>(warp_sum(g * p));
  for (int e = lane; e < num_experts; e += 32) {
    float v = 0.0f;
    if (!sigmoid) v = -along * (expf(load_elem(row + e) - top) / sum);
    store_elem(out + e, v);
  }
  __syncwarp();  // the selected entries are written again
  if (lane < topk) {
    const double d = sigmoid ? g * p * (1.0 - p) : p * (g - static_cast<double>(along));
    store_elem(out + expert, static_cast<float>(d));
  }
}

template <typename T>
static int launch_topk(const TopkArgs& a, cudaStream_t s) {
  const int blocks = static_cast<int>((a.num_tokens + kTopkWarps - 1) / kTopkWarps);
#define MOE_TOPK(PER) grouped_topk_kernel<T, PER><<<blocks, kTopkWarps * 32, 0, s>>>(a)
  if (a.per_lane <= 1) MOE_TOPK(1);
  else if (a.per_lane <= 2) MOE_TOPK(2);
  else if (a.per_lane <= 4) MOE_TOPK(4);
  else if (a.per_lane <= 8) MOE_TOPK(8);
  else if (a.per_lane <= 16) MOE_TOPK(16);
  else if (a.per_lane <= 32) MOE_TOPK(32);
  else MOE_TOPK(64);
#undef MOE_TOPK
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

}  // namespace moe

using namespace moe;

static int check_topk(const char* name, int64_t num_tokens, int num_experts, int topk, int dtype, int scores_dtype) {
  MOE_CHECK_ARG(num_tokens >= 0 && num_experts > 0 && topk > 0, "%s: negative or zero size", name);
  MOE_CHECK_ARG(dtype >= MOE_DTYPE_BF16 && dtype <= MOE_DTYPE_F32 && scores_dtype >= MOE_DTYPE_BF16 && scores_dtype <= MOE_DTYPE_F32,
                "%s: unknown dtype", name);
  if (num_experts > 1024 || topk > 32 || num_tokens > (1ll << 31)) {
    set_error("%s: E <= 1024, k <= 32 and at most 2^31 tokens are supported (E = %d, k = %d)", name, num_experts, topk);
    return MOE_ERR_UNSUPPORTED;
  }
  return MOE_OK;
}

extern "C" int moe_grouped_topk(const void* logits, const float* bias, void* scores, int64_t* indices, int64_t num_tokens,
                                int num_experts, int num_groups, int topk_groups, int group_best, int topk, int sigmoid,
                                int normalize, float scale, int dtype, int scores_dtype, void* stream) {
  const int rc = check_topk("moe_grouped_topk", num_tokens, num_experts, topk, dtype, scores_dtype);
  if (rc != MOE_OK) return rc;
  MOE_CHECK_ARG(num_groups > 0 && num_groups <= 32 && num_experts % num_groups == 0,
                "moe_grouped_topk: the experts must divide into 1 to 32 equal groups (%d experts, %d groups)", num_experts, num_groups);
  const int size = num_experts / num_groups;
  MOE_CHECK_ARG(topk_groups > 0 && topk_groups <= num_groups && topk <= topk_groups * size,
                "moe_grouped_topk: %d of %d groups of %d experts hold no %d experts", topk_groups, num_groups, size, topk);
  MOE_CHECK_ARG(group_best >= 1 && group_best <= 2 && group_best <= size,
                "moe_grouped_topk: a group's score is the sum of its best one or two, got %d of %d", group_best, size);
  if (num_tokens == 0) return MOE_OK;
  MOE_CHECK_ARG(logits != nullptr && scores != nullptr && indices != nullptr, "moe_grouped_topk: null pointer argument");
  TopkArgs a{logits, bias, scores, indices, num_tokens, num_experts, size, num_groups, topk_groups, group_best, topk,
             0, 0, sigmoid, normalize, scores_dtype, scale};
  int lanes_log2 = 5;
  while ((num_groups << lanes_log2) > 32) --lanes_log2;
  a.lanes_log2 = lanes_log2;
  a.per_lane = (size + (1 << lanes_log2) - 1) >> lanes_log2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_DTYPE_F32 ? launch_topk<float>(a, s) : dtype == MOE_DTYPE_BF16 ? launch_topk<__nv_bfloat16>(a, s) : launch_topk<__half>(a, s);
}

extern "C" int moe_grouped_topk_backward(const void* logits, const int64_t* indices, const void* d_scores, void* d_logits,
                                         int64_t num_tokens, int num_experts, int topk, int sigmoid, int normalize, float scale,
                                         int dtype, int scores_dtype, void* stream) {
  const int rc = check_topk("moe_grouped_topk_backward", num_tokens, num_experts, topk, dtype, scores_dtype);
  if (rc != MOE_OK) return rc;
  if (num_tokens == 0) return MOE_OK;
  MOE_CHECK_ARG(logits != nullptr && indices != nullptr && d_scores != nullptr && d_logits != nullptr,
                "moe_grouped_topk_backward: null pointer argument");
  const int blocks = static_cast<int>((num_tokens + kTopkWarps - 1) / kTopkWarps);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define MOE_TOPK_BWD(T)                                                                                                      \
  grouped_topk_backward_kernel<T><<<blocks, kTopkWarps * 32, 0, s>>>(static_cast<const T*>(logits), indices, d_scores,        \
                                                                     static_cast<T*>(d_logits), num_tokens, num_experts, topk, \
                                                                     sigmoid, normalize, scale, scores_dtype)
  if (dtype == MOE_DTYPE_F32) MOE_TOPK_BWD(float);
  else if (dtype == MOE_DTYPE_BF16) MOE_TOPK_BWD(__nv_bfloat16);
  else MOE_TOPK_BWD(__half);
#undef MOE_TOPK_BWD
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}
