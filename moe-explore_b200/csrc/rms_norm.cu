// Root-mean-square norm with the residual's addition, its result in 16 bits and / or in 8 bits with a scale per 128 columns, and its
// backward pass.
//
//   h = round(x + residual);  r = 1 / sqrt(mean h^2 + eps);  y = h r w;  per 128 columns: scale = max |y| / 448, q = e4m3(y / scale)
//   backward, with g = dy w and n = h r:  dx = dh + r (g - n mean(g n)),  dw = sum over the rows of dy n
//
// The norm is taken of the ROUNDED sum: it is the stream that the next layer reads, so the fused and the separate form, and the
// forward and the backward pass, see the same h.  Everything else is fp32, rounded once.
//
// Bound by HBM: 8192 rows of 7168 with a residual and both results (530 MB) in 82 us, 6.4 TB/s.  One pass over the rows, each thread
// keeping its 16-byte pieces of a row in registers between the sum and the scaling.  A row of at most 1024 columns belongs to a
// warp, a longer one to a CTA.
#include "f8.cuh"

#include <type_traits>

namespace moe {

constexpr int kNormVec = 8;  // elements of a 16-byte piece

template <typename W> __device__ __forceinline__ void load_weight8(const W* w, int at, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(w + at);
  const uint32_t p[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Elem<W>::unpack2(p[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <> __device__ __forceinline__ void load_weight8<float>(const float* w, int at, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(w + at), b = *reinterpret_cast<const float4*>(w + at + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <typename T> __device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t p[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Elem<T>::unpack2(p[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <typename T> __device__ __forceinline__ uint4 packed8(const float (&f)[8]) {
  return make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]), Elem<T>::pack2(f[4], f[5]), Elem<T>::pack2(f[6], f[7]));
}

// Sum over the threads of a row: a warp (THREADS == 32) or the CTA; `parts` [2][32], used in turn so that one barrier is enough.
template <int THREADS> __device__ __forceinline__ float row_sum(float v, float (*parts)[32], int turn) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  if constexpr (THREADS > 32) {
    float* p = parts[turn & 1];
    if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = v;
    __syncthreads();
    v = p[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
    for (int off = THREADS / 64; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  }
  return v;
}

struct NormArgs {
  const void *x, *residual, *weight;
  int64_t x_stride, residual_stride;  // elements
  void *h, *y;
  uint2* q;
  float *scales, *rstd;
  int64_t rows;
  int cols;
  float eps;
};

// CTAs per SM that the wide forms are compiled for: 64 registers per thread, 56 for the 128-thread form without 8 bits (what the
// compiler takes by itself, 72 to 91, leaves fewer rows under way: 4096 x 16384 in 8 and 16 bits 115 us instead of 95).
constexpr int norm_ctas(int threads, int vecs, bool quant) {
  return vecs == 1 ? 1 : threads >= 256 ? 1024 / threads : threads == 128 && !quant ? 9 : 1;
}

template <typename T, typename W, int THREADS, int VECS, bool QUANT>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS, norm_ctas(THREADS, VECS, QUANT))
    rms_norm_kernel(const NormArgs a) {
  __shared__ float parts[2][32];
  const int tid = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = THREADS == 32 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (THREADS == 32 && row >= a.rows) return;
  const int vecs = a.cols / kNormVec;
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.x_stride);
  const uint4* res = a.residual == nullptr ? nullptr : reinterpret_cast<const uint4*>(static_cast<const T*>(a.residual) + row * a.residual_stride);
  uint4 u[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = i * THREADS + tid;
    u[i] = v < vecs ? x[v] : make_uint4(0, 0, 0, 0);
  }
  if (res != nullptr) {
    uint4 r[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = i * THREADS + tid;
      r[i] = v < vecs ? res[v] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = i * THREADS + tid;
      float f[8], g[8];
      unpack8<T>(u[i], f);
      unpack8<T>(r[i], g);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += g[j];
      u[i] = packed8<T>(f);
      if (v < vecs && a.h != nullptr) reinterpret_cast<uint4*>(a.h)[row * vecs + v] = u[i];
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    float f[8];
    unpack8<T>(u[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(f[j], f[j], sum);
  }
  sum = row_sum<THREADS>(sum, parts, 0);
  float r = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
  // bf16 values from 2^57 on have squares whose sum may leave fp32: such a row again in units of 2^72, beside which eps is nothing.
  // (A row that holds an infinity is infinite again.  The branch is the whole row's; fp16 rows cannot get here.)
  if (!std::is_same<T, __half>::value && sum > 3.0e38f) {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      float f[8];
      unpack8<T>(u[i], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(f[j] * 0x1p-72f, f[j] * 0x1p-72f, sum);
    }
    sum = row_sum<THREADS>(sum, parts, 1);
    r = rsqrtf(sum / static_cast<float>(a.cols)) * 0x1p-72f;
  }
  if (a.rstd != nullptr && tid == 0) a.rstd[row] = r;
  const int blocks = (a.cols + kF8Block - 1) / kF8Block;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = i * THREADS + tid;
    if (i * THREADS + (tid & ~31) >= vecs) break;  // by whole warps: the block maxima are exchanged
    float f[8], w[8];
    unpack8<T>(u[i], f);
    if (v < vecs) load_weight8<W>(static_cast<const W*>(a.weight), v * kNormVec, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v < vecs ? f[j] * r * w[j] : 0.0f;
    if (v < vecs && a.y != nullptr) reinterpret_cast<uint4*>(a.y)[row * vecs + v] = packed8<T>(f);
    if constexpr (QUANT) {
      const float most = block_most(f);
      const float inv = kF8Top / most;
      if (v < vecs) {
        a.q[row * vecs + v] = make_uint2(f8x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                                         f8x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        if ((v & 15) == 0) a.scales[row * blocks + (v >> 4)] = most / kF8Top;
      }
    }
  }
}

struct NormBackArgs {
  const void *dy, *dh, *h, *weight;
  int64_t h_stride;
  const float* rstd;
  void* dx;
  float* partials;  // [gridDim.x, cols]
  int64_t rows;
  int cols;
};

// A CTA takes every gridDim.x-th row (a warp of the 32-thread form every row of its own stride) and keeps the weight gradient of
// its columns in registers; the partial sums are joined by the next kernel in a fixed order.  The next row's loads are issued before
// the row's one reduction.  8191 rows of 2048 with a residual: 28 to 31 us, 4.3 to 4.8 TB/s, with the sums of dw (42 us with the
// residual's gradient fetched in the row's own turn).  Up to 2048 columns all CTAs are resident at once; wider rows leave room for two
// or one per SM, so that they come in two to four waves and begin anew in each: 8192 x 4096 51 us (5.2 TB/s), 4096 x 7168 56 (4.2),
// 4096 x 16384 143 (3.8; two pieces per thread in 64 registers spill).
template <typename T, typename W, int THREADS, int VECS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : VECS == 1 ? 4 : 512 / THREADS)
    rms_norm_backward_kernel(const NormBackArgs a) {
  __shared__ float parts[2][32];
  const int tid = threadIdx.x;
  const int vecs = a.cols / kNormVec;
  // (with 64 registers per thread there is room for neither the weight nor the next row)
  constexpr bool kAhead = THREADS < 1024;
  float dw[VECS][8], held[kAhead ? VECS : 1][8];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = i * THREADS + tid;
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.0f;
    if (kAhead) {
#pragma unroll
      for (int j = 0; j < 8; ++j) held[i][j] = 0.0f;
      if (v < vecs) load_weight8<W>(static_cast<const W*>(a.weight), v * kNormVec, held[i]);
    }
  }
  const auto weights = [&](int i, float (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = kAhead ? held[i][j] : 0.0f;
    const int v = i * THREADS + tid;
    if (!kAhead && v < vecs) load_weight8<W>(static_cast<const W*>(a.weight), v * kNormVec, w);
  };
  const uint4* dy = static_cast<const uint4*>(a.dy);
  uint4 uy[VECS], uh[VECS], ud[VECS];
  const auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = i * THREADS + tid;
      const bool ok = v < vecs;
      uy[i] = ok ? dy[row * vecs + v] : make_uint4(0, 0, 0, 0);
      uh[i] = ok ? reinterpret_cast<const uint4*>(static_cast<const T*>(a.h) + row * a.h_stride)[v] : make_uint4(0, 0, 0, 0);
      ud[i] = ok && a.dh != nullptr ? static_cast<const uint4*>(a.dh)[row * vecs + v] : make_uint4(0, 0, 0, 0);
    }
  };
  int64_t row = blockIdx.x;
  if (kAhead && row < a.rows) load(row);
  for (int turn = 0; row < a.rows; row += gridDim.x, ++turn) {
    uint4 cy[VECS], ch[VECS], cr[VECS];
    if (!kAhead) load(row);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      cy[i] = uy[i];
      ch[i] = uh[i];
      cr[i] = ud[i];
    }
    const float r = a.rstd[row];
    if (kAhead && row + gridDim.x < a.rows) load(row + gridDim.x);
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      float y[8], h[8], w[8];
      unpack8<T>(cy[i], y);
      unpack8<T>(ch[i], h);
      weights(i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = h[j] * r;
        dw[i][j] = fmaf(y[j], n, dw[i][j]);
        dot = fmaf(y[j] * w[j], n, dot);
      }
    }
    dot = row_sum<THREADS>(dot, parts, turn) / static_cast<float>(a.cols);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = i * THREADS + tid;
      if (v >= vecs) continue;
      float y[8], h[8], d[8], w[8];
      unpack8<T>(cy[i], y);
      unpack8<T>(ch[i], h);
      unpack8<T>(cr[i], d);
      weights(i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += r * (y[j] * w[j] - h[j] * r * dot);
      static_cast<uint4*>(a.dx)[row * vecs + v] = packed8<T>(d);
    }
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = i * THREADS + tid;
    if (v >= vecs) continue;
    float4* p = reinterpret_cast<float4*>(a.partials + static_cast<int64_t>(blockIdx.x) * a.cols + v * kNormVec);
    p[0] = make_float4(dw[i][0], dw[i][1], dw[i][2], dw[i][3]);
    p[1] = make_float4(dw[i][4], dw[i][5], dw[i][6], dw[i][7]);
  }
}

// dw[c] = sum of the partial sums of column c: 32 columns and 32 slices of the partials per CTA.
template <typename W>
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* partials, W* dw, int count, int cols) {
  __shared__ float tile[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < cols)
    for (int p = threadIdx.y; p < count; p += 32) s += partials[static_cast<int64_t>(p) * cols + c];
  tile[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = tile[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
  const int out = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && out < cols) {
    if constexpr (sizeof(W) == 4) dw[out] = s;
    else dw[out] = Elem<W>::from_float(s);
  }
}

template <typename T, typename W, bool QUANT>
static int launch_norm(const NormArgs& a, cudaStream_t s) {
  const int vecs = a.cols / kNormVec;
#define MOE_NORM(THREADS, VECS)                                                                          \
  do {                                                                                                   \
    const int64_t grid = THREADS == 32 ? (a.rows + 3) / 4 : a.rows;                                      \
    const int block = THREADS == 32 ? 128 : THREADS;                                                     \
    MOE_CUDA(launch_kernel(rms_norm_kernel<T, W, THREADS, VECS, QUANT>, static_cast<int>(grid), block, s, a)); \
  } while (0)
  // few rows: as many threads per row as have a piece of it; many rows: a few pieces per thread
  const bool few = a.rows < 2 * sm_count();
  if (vecs <= 32) MOE_NORM(32, 1);
  else if (vecs <= 128 && !few) MOE_NORM(32, 4);
  else if (vecs <= 128) MOE_NORM(128, 1);
  else if (vecs <= 512 && !few) MOE_NORM(128, 4);
  else if (vecs <= 512) MOE_NORM(512, 1);
  else if (vecs <= 1024 && !few) MOE_NORM(256, 4);
  else if (vecs <= 1024) MOE_NORM(1024, 1);
  else MOE_NORM(512, 4);
#undef MOE_NORM
  return MOE_OK;
}

constexpr int kNormMaxCols = 16384;
constexpr int kNormPartials = 592;  // four CTAs on each of 148 SMs, at every width

template <typename T, typename W>
static int launch_norm_backward(const NormBackArgs& a, W* dw, cudaStream_t s) {
  const int vecs = a.cols / kNormVec;
  const int grid = static_cast<int>(a.rows < kNormPartials ? a.rows : kNormPartials);
#define MOE_NORM_BWD(THREADS, VECS) MOE_CUDA(launch_kernel(rms_norm_backward_kernel<T, W, THREADS, VECS>, grid, THREADS, s, a))
  if (vecs <= 64) MOE_NORM_BWD(64, 1);
  else if (vecs <= 128) MOE_NORM_BWD(128, 1);
  else if (vecs <= 256) MOE_NORM_BWD(256, 1);
  else if (vecs <= 512) MOE_NORM_BWD(256, 2);
  else if (vecs <= 1024) MOE_NORM_BWD(512, 2);
  else MOE_NORM_BWD(1024, 2);
#undef MOE_NORM_BWD
  norm_weight_grad_kernel<W><<<(a.cols + 31) / 32, dim3(32, 32), 0, s>>>(a.partials, dw, grid, a.cols);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

static int check_norm(const char* name, int64_t rows, int cols, int dtype, int weight_dtype) {
  MOE_CHECK_ARG(rows >= 0 && cols > 0, "%s: negative or zero size", name);
  MOE_CHECK_ARG(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16, "%s: unknown dtype %d", name, dtype);
  MOE_CHECK_ARG(weight_dtype == dtype || weight_dtype == MOE_DTYPE_F32, "%s: the weight is of the rows' dtype or fp32", name);
  if (cols % 8 != 0 || cols > kNormMaxCols || rows > 0x7FFFFFFF) {
    set_error("%s: rows of a multiple of 8 up to %d columns are supported, at most 2^31 of them, got %lld x %d", name, kNormMaxCols,
              static_cast<long long>(rows), cols);
    return MOE_ERR_UNSUPPORTED;
  }
  return MOE_OK;
}
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace moe

using namespace moe;

extern "C" int moe_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                            int weight_dtype, void* h, void* y, void* q, float* scales, float* rstd, int64_t num_rows, int cols,
                            float eps, int dtype, void* stream) {
  const int rc = check_norm("moe_rms_norm", num_rows, cols, dtype, weight_dtype);
  if (rc != MOE_OK) return rc;
  if (num_rows == 0) return MOE_OK;
  MOE_CHECK_ARG(x != nullptr && weight != nullptr && (y != nullptr || q != nullptr), "moe_rms_norm: null pointer argument");
  MOE_CHECK_ARG((q == nullptr) == (scales == nullptr), "moe_rms_norm: 8-bit rows and their scales come together");
  MOE_CHECK_ARG(aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(h) && aligned16(y) && aligned16(q) &&
                    x_stride % 8 == 0 && residual_stride % 8 == 0, "moe_rms_norm: pointers and row strides must be 16-byte aligned");
  const NormArgs a{x, residual, weight, x_stride, residual_stride, h, y, static_cast<uint2*>(q), scales, rstd, num_rows, cols, eps};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define MOE_NORM_OF(T, W) (q != nullptr ? launch_norm<T, W, true>(a, s) : launch_norm<T, W, false>(a, s))
  if (dtype == MOE_DTYPE_BF16) return weight_dtype == MOE_DTYPE_F32 ? MOE_NORM_OF(__nv_bfloat16, float) : MOE_NORM_OF(__nv_bfloat16, __nv_bfloat16);
  return weight_dtype == MOE_DTYPE_F32 ? MOE_NORM_OF(__half, float) : MOE_NORM_OF(__half, __half);
#undef MOE_NORM_OF
}

extern "C" int64_t moe_rms_norm_partials(int64_t num_rows) { return num_rows < kNormPartials ? num_rows : kNormPartials; }

extern "C" int moe_rms_norm_backward(const void* dy, const void* dh, const void* h, int64_t h_stride, const void* weight, int weight_dtype,
                                     const float* rstd, void* dx, void* dw, float* partials, int64_t num_rows, int cols, int dtype,
                                     void* stream) {
  const int rc = check_norm("moe_rms_norm_backward", num_rows, cols, dtype, weight_dtype);
  if (rc != MOE_OK) return rc;
  MOE_CHECK_ARG(dw != nullptr, "moe_rms_norm_backward: null pointer argument");
  if (num_rows == 0) {
    MOE_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(cols) * (weight_dtype == MOE_DTYPE_F32 ? 4 : 2), static_cast<cudaStream_t>(stream)));
    return MOE_OK;
  }
  MOE_CHECK_ARG(dy != nullptr && h != nullptr && weight != nullptr && rstd != nullptr && dx != nullptr && partials != nullptr,
                "moe_rms_norm_backward: null pointer argument");
  MOE_CHECK_ARG(aligned16(dy) && aligned16(dh) && aligned16(h) && aligned16(weight) && aligned16(dx) && aligned16(partials) && h_stride % 8 == 0,
                "moe_rms_norm_backward: pointers and row strides must be 16-byte aligned");
  const NormBackArgs a{dy, dh, h, weight, h_stride, rstd, dx, partials, num_rows, cols};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_DTYPE_BF16)
    return weight_dtype == MOE_DTYPE_F32 ? launch_norm_backward<__nv_bfloat16>(a, static_cast<float*>(dw), s)
                                         : launch_norm_backward<__nv_bfloat16>(a, static_cast<__nv_bfloat16*>(dw), s);
  return weight_dtype == MOE_DTYPE_F32 ? launch_norm_backward<__half>(a, static_cast<float*>(dw), s)
                                       : launch_norm_backward<__half>(a, static_cast<__half*>(dw), s);
}
