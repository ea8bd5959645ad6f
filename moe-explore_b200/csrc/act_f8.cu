// Activations whose un-activated product is kept in 8 bits for the backward pass, e4m3 with one fp32 scale per row and block of 128
// columns (f8.cuh).  z: the 16-bit product, gated ones with gate and up in turn (z[2i], z[2i + 1]); z~: what 8 bits give back of it.
//
//   forward:   h_i = act(z_2i) z_2i+1   (ungated: act(z_i)),   from z, not from z~;   kept: q = e4m3(z / scale), scale = max |z| / 448
//   backward:  dz_2i = dh_i z~_2i+1 act'(z~_2i),  dz_2i+1 = dh_i act(z~_2i)   (ungated: dh_i act'(z~_i))
//   as a step of the experts' backward pass, with u = dOut W2^T (not yet weighted) and the slot's weight s:
//              dh = s u,   d_s = sum_i u_i h~_i,   and s h~ for the gradient of W2;   padding rows get zeros
//
// The kept values are quotients of 16-bit values rounded once to fp32 and once to e4m3 (f8_quotients); everything else is fp32,
// rounded once to 16 bits.
//
// Bound by HBM beside instructions (the forward pass issues about 300 per 16 columns: exponentials, reciprocals and exactly rounded quotients;
// 72 % of the issue slots): 65536 x 2816 swiglu 132 us forward and 129 back, 114 each at the copy's rate; geglu 182 and 188 (erff).
// A lane takes 16 columns of a row, eight lanes share a block and ask for their next one before they compute.  The backward pass walks
// a row (or, where there are few rows, a share of one) 512 columns at a time: the gradient of a slot's weight is a sum over its row.  (That
// of a layer spills 4 to 52 bytes to stay within the 64 registers of four CTAs per SM.)
#include "f8.cuh"

namespace moe {

constexpr int kActThreads = 256, kActCtas = 4;

struct ActArgs {
  const void* z;         // [rows, cols]                                   (forward)
  const void* u;         // [rows, inter]: dh, or u of a layer             (backward)
  uint8_t* q;            // [rows, q_cols], q_cols = cols rounded up to 16
  float* scales;         // [rows, blocks]
  void* h;               // [rows, inter]: h (forward); s h~ of a layer (backward)
  void* dz;              // [rows, cols]                                   (backward)
  int64_t rows;          // of a layer: the bound that its padded layout was built for
  int cols, q_cols, split;
  // of a layer, else null: the padded layout, and the slots' weights and their gradients (backward)
  const int32_t *row_src, *num_mtiles, *dst_row;
  const void* scores;
  void* d_scores;
  int64_t slots;
};

__host__ __device__ constexpr bool act_gated(int act) { return act == MOE_ACT_SWIGLU || act == MOE_ACT_GEGLU; }

// act(x) and act'(x)
template <int ACT> __device__ __forceinline__ void act_both(float x, float& y, float& slope) {
  if constexpr (ACT == MOE_ACT_SWIGLU || ACT == MOE_ACT_SILU) {
    const float p = sigmoidf_fast(x);
    y = x * p;
    slope = p * (1.0f + x * (1.0f - p));
  } else if constexpr (ACT == MOE_ACT_GEGLU || ACT == MOE_ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(x * 0.70710678118654752f));
    y = x * cdf;
    slope = cdf + x * 0.3989422804014327f * __expf(-0.5f * x * x);
  } else if constexpr (ACT == MOE_ACT_GELU_TANH) {
    y = gelu_tanh_f(x);
    slope = dgelu_tanh_f(x);
  } else {
    y = x;
    slope = 1.0f;
  }
}
template <int ACT> __device__ __forceinline__ float act_only(float x) {
  if constexpr (ACT == MOE_ACT_SWIGLU || ACT == MOE_ACT_SILU) return silu_f(x);
  else if constexpr (ACT == MOE_ACT_GEGLU || ACT == MOE_ACT_GELU) return gelu_f(x);
  else if constexpr (ACT == MOE_ACT_GELU_TANH) return gelu_tanh_f(x);
  else return x;
}

template <typename T> __device__ __forceinline__ void act_unpack(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Elem<T>::unpack2(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T> __device__ __forceinline__ uint4 act_pack(const float* f) {
  return make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]), Elem<T>::pack2(f[4], f[5]), Elem<T>::pack2(f[6], f[7]));
}

// 16 columns of a row (the last eight may be behind its end: columns come in eights)
struct Wide {
  uint4 a, b;
};
__device__ __forceinline__ Wide wide_load(const void* base, int64_t row, int cols, int at) {
  Wide w{};
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + row * cols + at);
  if (at < cols) w.a = p[0];
  if (at + 8 < cols) w.b = p[1];
  return w;
}

// Two fp32 numbers in one register pair.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
// f8_quotients, two at a time: the same operations, the same bits.
__device__ __forceinline__ void act_quotients(float (&f)[16], float most) {
  if (!(most <= 3.0e38f)) {
    f8_quotients(f, most);
    return;
  }
  const float near1 = most >= 1.0f ? 0x1p-60f : 0x1p60f;
  const float d = most * near1, r = __frcp_rn(d);
  const uint64_t c2 = pair_of(0.875f * near1, 0.875f * near1), r2 = pair_of(r, r), d2 = pair_of(-d, -d), top2 = pair_of(512.0f, 512.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t v = mul_pair(pair_of(f[2 * i], f[2 * i + 1]), c2);
    const uint64_t q = mul_pair(v, r2);
    const uint64_t o = mul_pair(fma_pair(fma_pair(q, d2, v), r2, q), top2);
    float o0, o1, v0, v1;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o0), "=f"(o1) : "l"(o));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v0), "=f"(v1) : "l"(v));
    f[2 * i] = copysignf(o0, v0);
    f[2 * i + 1] = copysignf(o1, v1);
  }
}

// A warp takes four blocks at a time, wherever rows end (where a row's last piece was half a warp's, 65536 x 2816 took 168 us).
template <typename T, int ACT, bool LAYER>
__global__ void __launch_bounds__(kActThreads, kActCtas) act_f8_forward_kernel(const ActArgs a) {
  constexpr bool GATED = act_gated(ACT);
  const int lane = threadIdx.x & 31;
  const int blocks = (a.cols + kF8Block - 1) / kF8Block;
  const int inter = GATED ? a.cols / 2 : a.cols;
  int64_t rows = a.rows;
  if constexpr (LAYER) rows = min(rows, static_cast<int64_t>(*a.num_mtiles) * MOE_TILE_M);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (kActThreads / 8);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kActThreads / 8) + threadIdx.x / 8;
  const int64_t stride_rows = stride / blocks;
  const int stride_blocks = static_cast<int>(stride - stride_rows * blocks);
  int64_t row = first / blocks;
  int block = static_cast<int>(first - row * blocks);
  const auto load = [&](int64_t r, int b) {
    Wide w{};
    if (r >= rows) return w;
    if constexpr (LAYER)
      if (a.row_src[r] < 0) return w;
    return wide_load(a.z, r, a.cols, b * kF8Block + (lane & 7) * 16);
  };
  Wide next = load(row, block);
  while (__any_sync(0xFFFFFFFFu, row < rows)) {
    const Wide u = next;
    const int64_t this_row = row;
    const int at = block * kF8Block + (lane & 7) * 16;
    bool ok = row < rows && at < a.cols;
    if constexpr (LAYER) ok = ok && a.row_src[this_row] >= 0;
    row += stride_rows;
    if ((block += stride_blocks) >= blocks) {
      block -= blocks;
      ++row;
    }
    next = load(row, block);
    float f[16];
    act_unpack<T>(u.a, f);
    act_unpack<T>(u.b, f + 8);
    if (ok) {
      float h[16];
      if constexpr (GATED) {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = act_only<ACT>(f[2 * i]) * f[2 * i + 1];
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + this_row * inter + at / 2) = act_pack<T>(h);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = act_only<ACT>(f[i]);
        uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + this_row * inter + at);
        out[0] = act_pack<T>(h);
        if (at + 8 < a.cols) out[1] = act_pack<T>(h + 8);
      }
    }
    if (a.q == nullptr) continue;
    float most = kF8Least;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(f[i]));
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, off));
    act_quotients(f, most);
    if (ok) {
      *reinterpret_cast<uint4*>(a.q + this_row * a.q_cols + at) =
          make_uint4(f8x4(f[0], f[1], f[2], f[3]), f8x4(f[4], f[5], f[6], f[7]), f8x4(f[8], f[9], f[10], f[11]), f8x4(f[12], f[13], f[14], f[15]));
      if ((lane & 7) == 0) a.scales[this_row * blocks + at / kF8Block] = most / kF8Top;
    }
  }
}

template <typename T, int ACT, bool LAYER>
__global__ void __launch_bounds__(kActThreads, kActCtas) act_f8_backward_kernel(const ActArgs a) {
  constexpr bool GATED = act_gated(ACT);
  const int lane = threadIdx.x & 31;
  const int blocks = (a.cols + kF8Block - 1) / kF8Block;
  const int inter = GATED ? a.cols / 2 : a.cols;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kActThreads / 32);
  const int64_t first_warp = static_cast<int64_t>(blockIdx.x) * (kActThreads / 32) + (threadIdx.x >> 5);
  int64_t rows = a.rows;
  if constexpr (LAYER) {
    rows = min(rows, static_cast<int64_t>(*a.num_mtiles) * MOE_TILE_M);
    // slots that the routing dropped are no row's
    for (int64_t j = first_warp * 32 + lane; j < a.slots; j += warps * 32)
      if (a.dst_row[j] < 0) static_cast<T*>(a.d_scores)[j] = Elem<T>::from_float(0.0f);
  }
  struct Piece {
    uint4 q;
    float scale;
    Wide u;
  };
  for (int64_t item = first_warp; item < rows * a.split; item += warps) {
    const int64_t row = item / a.split;
    const int step = 512 * a.split;
    const int first = static_cast<int>(item - row * a.split) * 512;
    int src = 0;
    float weight = 1.0f;
    if constexpr (LAYER) {
      src = a.row_src[row];
      if (src < 0) {  // the gradients of the weights contract over it
        for (int at = lane * 8; at < a.cols; at += 256) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + row * a.cols + at) = make_uint4(0, 0, 0, 0);
        for (int at = lane * 8; at < inter; at += 256) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + row * inter + at) = make_uint4(0, 0, 0, 0);
        continue;
      }
      weight = Elem<T>::to_float(static_cast<const T*>(a.scores)[src]);
    }
    float d_score = 0.0f;
    const auto load = [&](int at) {
      Piece p{};
      if (at < a.cols) {
        p.q = *reinterpret_cast<const uint4*>(a.q + row * a.q_cols + at);
        p.scale = a.scales[row * blocks + at / kF8Block];
        p.u = GATED ? wide_load(a.u, row, inter, at / 2) : wide_load(a.u, row, inter, at);
      }
      return p;
    };
    Piece next = load(first + lane * 16);
    for (int c0 = first; c0 < a.cols; c0 += step) {
      const Piece p = next;
      const int at = c0 + lane * 16;
      next = load(at + step);
      if (at >= a.cols) continue;
      const uint32_t words[4] = {p.q.x, p.q.y, p.q.z, p.q.w};
      float z[16], u[16], dz[16], h[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2_raw v = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(words[i / 2] >> (16 * (i & 1))), __NV_E4M3);
        const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(&v));
        z[2 * i] = pair.x * p.scale;
        z[2 * i + 1] = pair.y * p.scale;
      }
      act_unpack<T>(p.u.a, u);
      if constexpr (!GATED) act_unpack<T>(p.u.b, u + 8);
      constexpr int N = GATED ? 8 : 16;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float dh = LAYER ? weight * u[i] : u[i];
        float y, slope;
        act_both<ACT>(z[GATED ? 2 * i : i], y, slope);
        if constexpr (GATED) {
          dz[2 * i] = dh * z[2 * i + 1] * slope;
          dz[2 * i + 1] = dh * y;
          y *= z[2 * i + 1];
        } else {
          dz[i] = dh * slope;
        }
        if constexpr (LAYER) {
          if (GATED || i < 8 || at + 8 < a.cols) d_score = fmaf(u[i], y, d_score);
          h[i] = weight * y;
        }
      }
      uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dz) + row * a.cols + at);
      out[0] = act_pack<T>(dz);
      if (at + 8 < a.cols) out[1] = act_pack<T>(dz + 8);
      if constexpr (LAYER) {
        uint4* hs = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + row * inter + (GATED ? at / 2 : at));
        hs[0] = act_pack<T>(h);
        if (!GATED && at + 8 < a.cols) hs[1] = act_pack<T>(h + 8);
      }
    }
    if constexpr (LAYER) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) d_score += __shfl_xor_sync(0xFFFFFFFFu, d_score, off);
      if (lane == 0) static_cast<T*>(a.d_scores)[src] = Elem<T>::from_float(d_score);
    }
  }
}

template <typename T, bool LAYER, bool BACKWARD> static int launch_act(int act, const ActArgs& a, int grid, cudaStream_t s) {
  const auto go = [&](auto code) {
    constexpr int ACT = decltype(code)::value;
    if constexpr (BACKWARD) act_f8_backward_kernel<T, ACT, LAYER><<<grid, kActThreads, 0, s>>>(a);
    else act_f8_forward_kernel<T, ACT, LAYER><<<grid, kActThreads, 0, s>>>(a);
  };
  switch (act) {
    case MOE_ACT_SILU: go(std::integral_constant<int, MOE_ACT_SILU>()); break;
    case MOE_ACT_GELU: go(std::integral_constant<int, MOE_ACT_GELU>()); break;
    case MOE_ACT_GELU_TANH: go(std::integral_constant<int, MOE_ACT_GELU_TANH>()); break;
    case MOE_ACT_SWIGLU: go(std::integral_constant<int, MOE_ACT_SWIGLU>()); break;
    case MOE_ACT_GEGLU: go(std::integral_constant<int, MOE_ACT_GEGLU>()); break;
    default: go(std::integral_constant<int, MOE_ACT_NONE>()); break;
  }
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

static bool act_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int run_act(const char* name, bool backward, ActArgs a, int inter, int act, int dtype, void* stream) {
  MOE_CHECK_ARG(act >= MOE_ACT_NONE && act <= MOE_ACT_GELU_TANH, "%s: unknown activation %d", name, act);
  MOE_CHECK_ARG(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16, "%s: unknown dtype %d", name, dtype);
  MOE_CHECK_ARG(a.rows >= 0 && inter > 0 && inter <= (1 << 29), "%s: %lld rows of %d", name, static_cast<long long>(a.rows), inter);
  if (inter % 8 != 0) {
    set_error("%s: rows have a multiple of 8 columns, got %d", name, inter);
    return MOE_ERR_UNSUPPORTED;
  }
  if (a.rows == 0) return MOE_OK;
  const bool layer = a.row_src != nullptr;
  MOE_CHECK_ARG(backward ? a.q && a.scales && a.u && a.dz : a.z && a.h && (a.q == nullptr) == (a.scales == nullptr), "%s: null pointer argument", name);
  MOE_CHECK_ARG(!layer || (a.num_mtiles && (!backward || (a.dst_row && a.scores && a.d_scores && a.h))), "%s: null pointer argument", name);
  MOE_CHECK_ARG(act_aligned(a.z) && act_aligned(a.u) && act_aligned(a.q) && act_aligned(a.h) && act_aligned(a.dz),
                "%s: pointers must be 16-byte aligned", name);
  a.cols = act_gated(act) ? 2 * inter : inter;
  a.q_cols = (a.cols + 15) / 16 * 16;
  // a warp per row, or as many as there are pieces of 512 columns where that leaves SMs without work (a layer's row is one warp's:
  // the gradient of its weight is a sum over the row)
  const int units = (a.cols + 511) / 512;
  const int64_t resident = static_cast<int64_t>(sm_count()) * kActCtas * (kActThreads / 32);
  a.split = 1;
  if (!layer)
    while (a.split < units && a.rows * a.split < resident) ++a.split;
  const int64_t pieces = backward ? a.rows * a.split : (a.rows * ((a.cols + kF8Block - 1) / kF8Block) + 3) / 4;
  const int64_t want = (pieces + kActThreads / 32 - 1) / (kActThreads / 32);
  const int64_t most = static_cast<int64_t>(sm_count()) * kActCtas;
  const int grid = static_cast<int>(want < most ? want : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto type) {
    using T = decltype(type);
    if (layer) return backward ? launch_act<T, true, true>(act, a, grid, s) : launch_act<T, true, false>(act, a, grid, s);
    return backward ? launch_act<T, false, true>(act, a, grid, s) : launch_act<T, false, false>(act, a, grid, s);
  };
  return dtype == MOE_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
}

// The steps of an experts' pass (layer.cu).
int act_f8_layer_forward(const moe_expert_pass* p, void* stream) {
  ActArgs a{};
  a.z = p->pre_act;
  a.q = static_cast<uint8_t*>(p->pre_q);
  a.scales = p->pre_scales;
  a.h = p->hidden;
  a.rows = p->padded_rows;
  a.row_src = p->row_src;
  a.num_mtiles = p->num_mtiles;
  MOE_CHECK_ARG(a.row_src != nullptr && a.q != nullptr, "moe_expert_forward: null pointer argument");
  return run_act("moe_expert_forward", false, a, p->inter, p->act, p->dtype, stream);
}
int act_f8_layer_backward(const moe_expert_pass* p, void* stream) {
  ActArgs a{};
  a.u = p->dh;
  a.q = static_cast<uint8_t*>(p->pre_q);
  a.scales = p->pre_scales;
  a.h = p->hidden;
  a.dz = p->d_pre;
  a.rows = p->padded_rows;
  a.row_src = p->row_src;
  a.num_mtiles = p->num_mtiles;
  a.dst_row = p->dst_row;
  a.scores = p->scores;
  a.d_scores = p->d_scores;
  a.slots = p->num_tokens * p->topk;
  MOE_CHECK_ARG(a.row_src != nullptr, "moe_expert_backward: null pointer argument");
  return run_act("moe_expert_backward", true, a, p->inter, p->act, p->dtype, stream);
}

}  // namespace moe

using namespace moe;

extern "C" int moe_act_f8_forward(const void* z, void* h, void* q, float* scales, int64_t rows, int inter, int act, int dtype, void* stream) {
  ActArgs a{};
  a.z = z;
  a.h = h;
  a.q = static_cast<uint8_t*>(q);
  a.scales = scales;
  a.rows = rows;
  return run_act("moe_act_f8_forward", false, a, inter, act, dtype, stream);
}

extern "C" int moe_act_f8_backward(const void* q, const float* scales, const void* dh, void* dz, int64_t rows, int inter, int act, int dtype,
                                   void* stream) {
  ActArgs a{};
  a.q = static_cast<uint8_t*>(const_cast<void*>(q));
  a.scales = const_cast<float*>(scales);
  a.u = dh;
  a.dz = dz;
  a.rows = rows;
  return run_act("moe_act_f8_backward", true, a, inter, act, dtype, stream);
}
