// RMSNorm with the residual's addition and an e4m3 output with one scale per row:
//   h = round(x + residual)  (stored: the new residual stream)        f = h (or x without a residual)
//   y = f * rsqrt(mean(f^2) + eps) * w  in fp32
//   s = max(max |y|, 2^-100) / 448,   q = e4m3(y / s)
// No rounding between the sum's and the output's: y stays in fp32 until it is divided by the scale (the bf16 kernel of
// emk_rmsnorm.cu rounds the normalised value as the eager module does; here the only consumer is the 8-bit rounding).
//
// Bound by HBM: x, residual in, h, q out, one pass, the row in registers across both reductions (sum of squares, then
// the maximum of |y|, which needs the first). A warp holds a row where there are many rows and they fit one warp's
// registers, eight warps hold it otherwise; rows longer than 8 vectors a thread are re-read (L2) instead.
#include "emk_common.cuh"

#include <cuda_fp8.h>

namespace {

using namespace emk;

constexpr float E4M3_MAX = 448.f;
constexpr float AMAX_FLOOR = 7.888609052210118e-31f;  // 2^-100: the scale of a row of zeros stays a normal number

// maximum that keeps a NaN: a row with one comes out as a row of NaN codes with a NaN scale, as y / s would
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements: V * sizeof(T) is 16 bytes (aligned rows), 4 bytes, or one element.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float* f) {
  Pack<T, V> a;
  if constexpr (sizeof(a) == 16) {
    *reinterpret_cast<uint4*>(&a) = __ldcs(reinterpret_cast<const uint4*>(p));
  } else {
    a = *reinterpret_cast<const Pack<T, V>*>(p);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f<T>(a.e[i]);
}
// the weight row: read by every row, so with the default caching
template <typename T, int V>
__device__ __forceinline__ void load_weight(const T* p, float* f) {
  const Pack<T, V> a = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f<T>(a.e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float* f) {
  Pack<T, V> a;
#pragma unroll
  for (int i = 0; i < V; ++i) a.e[i] = from_f<T>(f[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = a;
}
template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* y, float inv) {
  if constexpr (V == 1) {
    *p = __nv_cvt_float_to_fp8(y[0] * inv, __NV_SATFINITE, __NV_E4M3);
  } else {
    Pack<uint16_t, V / 2> o;
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      o.e[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * inv, y[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<Pack<uint16_t, V / 2>*>(p) = o;
  }
}

// One element pack of the normalised input: the residual is added in fp32 and rounded once to T, and that rounded sum
// is both what is stored and what is normalised.
template <typename T, int V>
__device__ __forceinline__ void load_sum(const T* x, const T* residual, T* hidden, int64_t at, float* f) {
  load_pack<T, V>(x + at, f);
  if (residual != nullptr) {
    float r[V];
    load_pack<T, V>(residual + at, r);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f<T>(from_f<T>(f[i] + r[i]));
    store_pack<T, V>(hidden + at, f);
  }
}

__device__ __forceinline__ float row_scale(float amax) { return max_nan(amax, AMAX_FLOOR) / E4M3_MAX; }

// WPR warps hold a row (1 or 8), NV packs of V elements a thread.
template <typename T, int V, int NV, int WPR>
__global__ void __launch_bounds__(256) rmsnorm_e4m3_kernel(const T* x, const T* residual, const T* __restrict__ w,
                                                           uint8_t* __restrict__ q, float* __restrict__ scale, T* hidden,
                                                           int64_t rows, int cols, float eps) {
  constexpr int TPR = WPR * 32;
  __shared__ float red_sum[8], red_max[8];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int tid = WPR == 1 ? lane : (int)threadIdx.x;
  const int64_t first = WPR == 1 ? (int64_t)blockIdx.x * 8 + wid : blockIdx.x;
  const int64_t step = WPR == 1 ? (int64_t)gridDim.x * 8 : gridDim.x;
  const int nvec = cols / V;
  for (int64_t row = first; row < rows; row += step) {
    const int64_t base = row * cols;
    float f[NV][V];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * TPR + tid;
      if (vi < nvec) {
        load_sum<T, V>(x, residual, hidden, base + (int64_t)vi * V, f[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fmaf(f[i][e], f[i][e], ss);
      }
    }
    ss = warp_sum(ss);
    if (WPR > 1) {
      if (lane == 0) red_sum[wid] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) ss += red_sum[i];
    }
    const float r = 1.0f / sqrtf(ss / (float)cols + eps);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * TPR + tid;
      if (vi < nvec) {
        float wv[V];
        load_weight<T, V>(w + (int64_t)vi * V, wv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          f[i][e] = (f[i][e] * r) * wv[e];
          amax = max_nan(amax, fabsf(f[i][e]));
        }
      }
    }
    amax = warp_max_nan(amax);
    if (WPR > 1) {
      // the sums of the next row are written after this barrier, when all have read this row's; likewise the maxima
      if (lane == 0) red_max[wid] = amax;
      __syncthreads();
      amax = red_max[0];
#pragma unroll
      for (int i = 1; i < WPR; ++i) amax = max_nan(amax, red_max[i]);
    }
    const float s = row_scale(amax);
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * TPR + tid;
      if (vi < nvec) store_codes<V>(q + base + (int64_t)vi * V, f[i], inv);
    }
    if (tid == 0) scale[row] = s;
  }
}

// Rows too long for eight packs a thread: one CTA per row, the row re-read (from L2) for the maximum and the codes. With
// a residual the later sweeps read the stored sum, each element by the thread that wrote it.
template <typename T, int V>
__global__ void __launch_bounds__(256) rmsnorm_e4m3_long_kernel(const T* x, const T* residual,
                                                                const T* __restrict__ w, uint8_t* __restrict__ q,
                                                                float* __restrict__ scale, T* hidden, int64_t rows,
                                                                int64_t cols, float eps) {
  __shared__ float red_sum[8], red_max[8];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * cols;
    const T* src = residual != nullptr ? hidden : x;
    float f[V], wv[V];
    float ss = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += 256 * V) {
      load_sum<T, V>(x, residual, hidden, base + c, f);
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(f[e], f[e], ss);
    }
    ss = warp_sum(ss);
    if (lane == 0) red_sum[wid] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += red_sum[i];
    const float r = 1.0f / sqrtf(ss / (float)cols + eps);
    float amax = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += 256 * V) {
      load_weight<T, V>(src + base + c, f);
      load_weight<T, V>(w + c, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) amax = max_nan(amax, fabsf((f[e] * r) * wv[e]));
    }
    amax = warp_max_nan(amax);
    if (lane == 0) red_max[wid] = amax;
    __syncthreads();
    amax = red_max[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) amax = max_nan(amax, red_max[i]);
    const float s = row_scale(amax);
    const float inv = 1.0f / s;
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += 256 * V) {
      load_weight<T, V>(src + base + c, f);
      load_weight<T, V>(w + c, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = (f[e] * r) * wv[e];
      store_codes<V>(q + base + c, f, inv);
    }
    if (threadIdx.x == 0) scale[row] = s;
  }
}

template <typename T, int V>
int launch_vec(emk_handle_t h, const T* x, const T* residual, const T* w, uint8_t* q, float* scale, T* hidden,
               int64_t rows, int64_t cols, float eps, cudaStream_t s) {
  const int64_t nvec = cols / V;
  const int64_t cap = (int64_t)h->sm_count * 16;
  // A warp a row needs enough rows to fill the machine; below that the row's latency counts and eight warps share it.
  if (nvec <= 32 * 8 && rows >= (int64_t)h->sm_count * 8) {
    const int64_t ctas = (rows + 7) / 8;
    const unsigned grid = (unsigned)(ctas < cap ? ctas : cap);
    if (nvec <= 32) rmsnorm_e4m3_kernel<T, V, 1, 1><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else if (nvec <= 64) rmsnorm_e4m3_kernel<T, V, 2, 1><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else if (nvec <= 128) rmsnorm_e4m3_kernel<T, V, 4, 1><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else rmsnorm_e4m3_kernel<T, V, 8, 1><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
  } else {
    const unsigned grid = (unsigned)(rows < cap ? rows : cap);
    if (nvec <= 256) rmsnorm_e4m3_kernel<T, V, 1, 8><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else if (nvec <= 512) rmsnorm_e4m3_kernel<T, V, 2, 8><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else if (nvec <= 1024) rmsnorm_e4m3_kernel<T, V, 4, 8><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else if (nvec <= 2048) rmsnorm_e4m3_kernel<T, V, 8, 8><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, (int)cols, eps);
    else rmsnorm_e4m3_long_kernel<T, V><<<grid, 256, 0, s>>>(x, residual, w, q, scale, hidden, rows, cols, eps);
  }
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}

template <typename T>
int launch(emk_handle_t h, const void* x, const void* residual, const void* w, void* q, float* scale, void* hidden,
           int64_t rows, int64_t cols, float eps, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const uintptr_t at = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)w | (uintptr_t)hidden;
  const T *xt = (const T*)x, *rt = (const T*)residual, *wt = (const T*)w;
  if (cols % V == 0 && (at & 15u) == 0 && ((uintptr_t)q & (V - 1)) == 0)
    return launch_vec<T, V>(h, xt, rt, wt, (uint8_t*)q, scale, (T*)hidden, rows, cols, eps, s);
  return launch_vec<T, 1>(h, xt, rt, wt, (uint8_t*)q, scale, (T*)hidden, rows, cols, eps, s);
}

}  // namespace

extern "C" int emk_rmsnorm_e4m3(emk_handle_t h, const void* x, const void* residual, const void* w, void* q, float* scale,
                                void* hidden, int64_t rows, int64_t cols, float eps, int dtype, emk_stream_t stream) {
  if (!h || !x || !w || !q || !scale || (residual != nullptr) != (hidden != nullptr)) return EMK_ERR_ARG;
  if (rows <= 0 || cols <= 0 || cols > 0x7fffffff) return EMK_ERR_SHAPE;
  if (dtype != EMK_F32 && dtype != EMK_BF16) return EMK_ERR_DTYPE;
  const unsigned mask = dtype == EMK_F32 ? 3u : 1u;
  if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)w | (uintptr_t)hidden) & mask) != 0 || ((uintptr_t)scale & 3u) != 0)
    return EMK_ERR_ALIGN;
  return dtype == EMK_F32 ? launch<float>(h, x, residual, w, q, scale, hidden, rows, cols, eps, (cudaStream_t)stream)
                          : launch<__nv_bfloat16>(h, x, residual, w, q, scale, hidden, rows, cols, eps, (cudaStream_t)stream);
}
