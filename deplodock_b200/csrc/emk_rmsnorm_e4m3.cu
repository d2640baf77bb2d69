// RMSNorm with the residual's addition and an e4m3 output with one scale per row:
//   h = round(x + residual)  (stored: the new residual stream)        f = h (or x without a residual)
//   y = f * rsqrt(mean(f^2) + eps) * w  in fp32
//   s = max(max |y|, 2^-100) / 448,   q = e4m3(y / s)
// No rounding between the sum's and the output's: y stays in fp32 until it is divided by the scale (the bf16 kernel of
// emk_rmsnorm.cu rounds the normalised value as the eager module does; here the only consumer is the 8-bit rounding).
//
// Bound by HBM: x, residual in, h, q out, one pass, the row in registers. r = rsqrt(...) is a positive factor of the whole
// row, so max |y| = r * max |f * w| and one reduction carries both the sum of squares and the maximum: the row's serial
// chain (load, reduce, store) is what a warp waits on. All loads of a row are issued before the first store of its sum
// (they may alias), 8 to 256 threads share a row so that none holds more than four 16-byte packs, and rows of any length at
// any offset go through the same packs, taken at the aligned places of the whole array with the row's ends masked.
// Measured at 32768 x 1024 bf16 with a residual (235 MB): two reductions and loads behind stores 55.8 us, loads first 45.1,
// this form 39.4 (0.91 of the copy bandwidth); 32768 x 1001 (their weights still go element by element): 83.7 us element by
// element, 50.2 in packs; the same in fp32 without a residual: 50.6 us, 40.1 with four CTAs per SM and the odd elements'
// weights loaded with them.
// Launched under the tail of the kernel before it, as all kernels of the serving step: a layer of two norms, three linears
// and one token's append and attention takes 30.4 us so, 35.0 one after the other (512-token prompts gain nothing).
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
__device__ __forceinline__ Pack<T, V> load_raw(const T* p) {
  Pack<T, V> a;
  if constexpr (sizeof(a) == 16) {
    *reinterpret_cast<uint4*>(&a) = __ldcs(reinterpret_cast<const uint4*>(p));
  } else {
    a = *reinterpret_cast<const Pack<T, V>*>(p);
  }
  return a;
}
// the weight row: read by every row, so with the default caching
template <typename T, int V>
__device__ __forceinline__ void load_weight(const T* p, float* f) {
  const Pack<T, V> a = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f<T>(a.e[i]);
}
// The codes' factor r / s, as a product (row_codes).
struct Factor {
  float first, k;
};
// V codes of y * r / s
template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* y, Factor c) {
  if constexpr (V == 1) {
    *p = __nv_cvt_float_to_fp8(y[0] * c.first * c.k, __NV_SATFINITE, __NV_E4M3);
  } else {
    Pack<uint16_t, V / 2> o;
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      o.e[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * c.first * c.k, y[2 * i + 1] * c.first * c.k), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<Pack<uint16_t, V / 2>*>(p) = o;
  }
}

constexpr float FLT_LARGEST = 3.402823466e38f;
// (NaN where the largest value passes fp32's range: an infinite scale would leave zero codes)
__device__ __forceinline__ float row_scale(float amax) {
  return amax <= FLT_LARGEST ? fmaxf(amax, AMAX_FLOOR) / E4M3_MAX : __uint_as_float(0x7fc00000u);
}

constexpr float UP = 1.8446744073709552e19f;  // 2^64
constexpr float MEAN_MIN = 1.262177448e-29f;  // 2^-96: below it the squares of a row's values may have vanished

// Whether fp32 holds the mean square + eps of a row (NaN: no).
__device__ __forceinline__ bool mean_holds(float mean) { return mean >= MEAN_MIN && mean <= FLT_LARGEST; }

// Scale and codes' factor of a row from r = rsqrt(mean square + eps) and the largest |f * w|. Where the scale is at its floor and r
// is large (a row of zeros with eps = 1e-12: 1e6 / 1.8e-33) r / s passes fp32's range, and 0 * inf would be NaN. The values lie
// below 2^-119 there, so they take 2^64 of it first. One more product for all rows: a second store loop for those rows, or a
// call, cost the others registers (8 x 1024 1.60 -> 1.72 us).
__device__ __forceinline__ float row_codes(float r, float amax, Factor& c) {
  const float s = row_scale(amax * r);
  const float k = r / s;
  const bool large = k > FLT_LARGEST;  // (not where k is NaN: those codes are)
  c = {large ? UP : 1.f, large ? r * (1.f / UP) / s : k};
  return s;
}

// The same for a row whose squares fp32 does not hold: elements from about 2^64 on, or eps and all elements so small that the squares
// vanish. The squares are summed again of the row times a power of two (2^-80 or 2^96, `half` twice), by every LANES threads
// for themselves: `row` is x or the stored sum, `lane` this thread's place among them and `mask` they. (The test for such rows costs
// 8 x 1024 1.50 -> 1.58 us, 32768 x 1024 with a residual nothing.)
template <typename T, int LANES>
__device__ __forceinline__ float row_codes_far(const T* row, int64_t cols, float eps, float mean, float amax, int lane, unsigned mask,
                                               Factor& c) {
  const bool small = mean < 1.f;
  const float half = small ? 281474976710656.f : 9.094947017729282e-13f;  // 2^48, 2^-40
  __syncwarp(mask);  // what the others have stored of the sum is read here
  float ss = 0.f;
#pragma unroll 1
  for (int64_t i = lane; i < cols; i += LANES) {
    const float v = to_f<T>(row[i]) * half * half;
    ss = fmaf(v, v, ss);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
  const float r = 1.0f / sqrtf(ss / (float)cols + eps * half * half * half * half);  // times half^2: the row's
  const float s = row_scale((amax * half) * (r * half));
  c = {small ? UP : 1.f, r * half * (small ? 1.f / UP : 1.f) / s * half};
  return s;
}

// 16 bytes of a row, kept as they are loaded (a bf16 pack that the compiler takes apart costs a register an element).
template <typename T>
struct Raw;
template <>
struct Raw<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ void unpack(uint4 u, float* f) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Raw<__nv_bfloat16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void unpack(uint4 u, float* f) {
    f[0] = bf16_lo(u.x); f[1] = bf16_hi(u.x); f[2] = bf16_lo(u.y); f[3] = bf16_hi(u.y);
    f[4] = bf16_lo(u.z); f[5] = bf16_hi(u.z); f[6] = bf16_lo(u.w); f[7] = bf16_hi(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};

// CTAs per SM: as many as hold a row's packs in registers, but for a few words: the kernels of four packs in bf16 keep 8 to 32 bytes
// a thread in local memory (none or 8 where rows are aligned), those of eight packs 56 to 124 (fp32: 8 or none).
template <int NV, bool RAGGED, bool RES>
constexpr int NORM_CTAS = RAGGED ? (RES || NV == 8 ? 2 : 4) : NV == 8 ? (RES ? 2 : 3) : NV == 4 ? (RES ? 3 : 4) : 5;

// TPR threads hold a row (8, 32, 64, 128 or 256), NV packs of V elements each. RAGGED: the rows' length is no multiple of V;
// packs lie at the multiples of V of the whole array, and the elements of a row before its first and behind its last full
// pack (fewer than V each) go to one thread each. RES: with a residual (a kernel of its own: without one a row needs half
// the registers, and twice the rows fit an SM).
template <typename T, int NV, int TPR, bool RAGGED, bool RES>
__global__ void __launch_bounds__(256, NORM_CTAS<NV, RAGGED, RES>)
rmsnorm_e4m3_kernel(const T* x, const T* residual, const T* __restrict__ w, uint8_t* __restrict__ q, float* __restrict__ scale,
                    T* hidden, int64_t rows, int cols, float eps) {
  constexpr int V = Raw<T>::V;
  constexpr int RPC = 256 / TPR;                       // rows per CTA
  constexpr int LANES = TPR < 32 ? TPR : 32;           // lanes of a warp that share a row
  constexpr int WPR = TPR < 32 ? 1 : TPR / 32;         // warps that share a row
  static_assert(!RAGGED || TPR >= V, "a thread per odd element");
  __shared__ float red[2][2][8];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int tid = threadIdx.x % TPR;
  const float inv_cols = 1.0f / (float)cols;
  grid_dependency_wait();
  grid_launch_dependents();
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * RPC; first < rows; first += (int64_t)gridDim.x * RPC) {
    const int64_t row = first + threadIdx.x / TPR;
    const int64_t base = row * cols;
    // elements before the first full pack, full packs, elements behind them
    const int head = RAGGED ? min((int)((-base) & (V - 1)), cols) : 0;
    const int npack = row < rows ? (cols - head) / V : 0;
    const int tail = RAGGED ? cols - head - (cols - head) / V * V : 0;
    const int64_t at = base + head;
    // all loads of the row first: the stores of the sum may alias them, and would hold back every load behind them
    uint4 xr[NV], rr[RES ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * TPR + tid;
      xr[i] = make_uint4(0, 0, 0, 0);
      if (vi < npack) xr[i] = __ldcs(reinterpret_cast<const uint4*>(x + at + (int64_t)vi * V));
    }
    if (RES) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int vi = i * TPR + tid;
        rr[i] = make_uint4(0, 0, 0, 0);
        if (vi < npack) rr[i] = __ldcs(reinterpret_cast<const uint4*>(residual + at + (int64_t)vi * V));
      }
    }
    // this thread's odd elements: column tid of the head, column tid of the tail
    float odd[2] = {0.f, 0.f}, odd_w[2] = {0.f, 0.f};
    int odd_col[2] = {-1, -1};
    if (RAGGED && row < rows) {
      if (tid < head) odd_col[0] = tid;
      if (tid < tail) odd_col[1] = cols - tail + tid;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (odd_col[j] >= 0) {
          odd[j] = to_f<T>(x[base + odd_col[j]]);
          odd_w[j] = to_f<T>(__ldg(w + odd_col[j]));
          if (RES) odd[j] = to_f<T>(from_f<T>(odd[j] + to_f<T>(residual[base + odd_col[j]])));
        }
      }
    }
    float f[NV][V];  // f * w
    float ss = 0.f, amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * TPR + tid;
      if (vi < npack) {
        float v[V];
        Raw<T>::unpack(xr[i], v);
        if (RES) {  // the sum is rounded to T once: what is stored is what is normalised
          float r[V];
          Raw<T>::unpack(rr[i], r);
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] += r[e];
          const uint4 h = Raw<T>::pack(v);
          Raw<T>::unpack(h, v);
          *reinterpret_cast<uint4*>(hidden + at + (int64_t)vi * V) = h;
        }
        float wv[V];
        if constexpr (RAGGED) {
#pragma unroll
          for (int e = 0; e < V; ++e) wv[e] = to_f<T>(__ldg(w + head + vi * V + e));
        } else {
          Raw<T>::unpack(__ldg(reinterpret_cast<const uint4*>(w + (int64_t)vi * V)), wv);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ss = fmaf(v[e], v[e], ss);
          f[i][e] = v[e] * wv[e];
          amax = max_nan(amax, fabsf(f[i][e]));
        }
      }
    }
    if (RAGGED) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (odd_col[j] >= 0) {
          if (RES) hidden[base + odd_col[j]] = from_f<T>(odd[j]);
          ss = fmaf(odd[j], odd[j], ss);
          odd[j] *= odd_w[j];
          amax = max_nan(amax, fabsf(odd[j]));
        }
      }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (WPR > 1) {  // (two sets of places in turn: the next row's are written while this row's may still be read)
      if (lane == 0) {
        red[turn][0][wid] = ss;
        red[turn][1][wid] = amax;
      }
      __syncthreads();
      const int w0 = wid / WPR * WPR;
      ss = red[turn][0][w0];
      amax = red[turn][1][w0];
#pragma unroll
      for (int i = 1; i < WPR; ++i) {
        ss += red[turn][0][w0 + i];
        amax = max_nan(amax, red[turn][1][w0 + i]);
      }
      turn ^= 1;
    }
    const float mean = ss * inv_cols + eps;
    Factor k;
    float s = row_codes(1.0f / sqrtf(mean), amax, k);
    if (!mean_holds(mean) && row < rows)
      s = row_codes_far<T, LANES>((RES ? hidden : x) + base, cols, eps, mean, amax, lane % LANES,
                                  (0xffffffffu >> (32 - LANES)) << (lane / LANES * LANES), k);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * TPR + tid;
      if (vi < npack) store_codes<V>(q + at + (int64_t)vi * V, f[i], k);
    }
    if (RAGGED) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (odd_col[j] >= 0) store_codes<1>(q + base + odd_col[j], &odd[j], k);
    }
    if (tid == 0 && row < rows) scale[row] = s;
  }
}

// One pack of the normalised input: the residual is added in fp32 and rounded once to T, and that rounded sum is both what
// is stored and what is normalised.
template <typename T, int V>
__device__ __forceinline__ void sum_pack(const Pack<T, V>& x, const Pack<T, V>& r, bool add, T* hidden, float* f) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f<T>(x.e[i]);
  if (add) {
    Pack<T, V> h;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      h.e[i] = from_f<T>(f[i] + to_f<T>(r.e[i]));
      f[i] = to_f<T>(h.e[i]);
    }
    *reinterpret_cast<Pack<T, V>*>(hidden) = h;
  }
}

// Rows too long for the registers of a CTA, and pointers that are not aligned: one CTA per row, the row re-read (from L2)
// for the codes. With a residual the second sweep reads the stored sum, each element by the thread that wrote it.
template <typename T, int V>
__global__ void __launch_bounds__(256) rmsnorm_e4m3_long_kernel(const T* x, const T* residual,
                                                                const T* __restrict__ w, uint8_t* __restrict__ q,
                                                                float* __restrict__ scale, T* hidden, int64_t rows,
                                                                int64_t cols, float eps) {
  __shared__ float red_sum[8], red_max[8];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  grid_dependency_wait();
  grid_launch_dependents();
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * cols;
    const T* src = residual != nullptr ? hidden : x;
    float f[V], wv[V];
    float ss = 0.f, amax = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += 256 * V) {
      const Pack<T, V> xr = load_raw<T, V>(x + base + c);
      Pack<T, V> rr = {};
      if (residual != nullptr) rr = load_raw<T, V>(residual + base + c);
      sum_pack<T, V>(xr, rr, residual != nullptr, hidden + base + c, f);
      load_weight<T, V>(w + c, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        ss = fmaf(f[e], f[e], ss);
        amax = max_nan(amax, fabsf(f[e] * wv[e]));
      }
    }
    ss = warp_sum(ss);
    amax = warp_max_nan(amax);
    if (lane == 0) {
      red_sum[wid] = ss;
      red_max[wid] = amax;
    }
    __syncthreads();
    ss = red_sum[0];
    amax = red_max[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      ss += red_sum[i];
      amax = max_nan(amax, red_max[i]);
    }
    __syncthreads();
    const float mean = ss / (float)cols + eps;
    Factor k;
    float s = row_codes(1.0f / sqrtf(mean), amax, k);
    if (!mean_holds(mean)) s = row_codes_far<T, 32>(src + base, cols, eps, mean, amax, lane, 0xffffffffu, k);
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += 256 * V) {
      load_weight<T, V>(src + base + c, f);
      load_weight<T, V>(w + c, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= wv[e];
      store_codes<V>(q + base + c, f, k);
    }
    if (threadIdx.x == 0) scale[row] = s;
  }
}

template <typename T, int NV, int TPR, bool RAGGED>
int launch_rows(emk_handle_t h, const T* x, const T* residual, const T* w, uint8_t* q, float* scale, T* hidden, int64_t rows,
                int cols, float eps, cudaStream_t s) {
  const int64_t ctas = (rows + 256 / TPR - 1) / (256 / TPR), cap = (int64_t)h->sm_count * 16;
  const unsigned grid = (unsigned)(ctas < cap ? ctas : cap);
  const auto kernel =
      residual != nullptr ? rmsnorm_e4m3_kernel<T, NV, TPR, RAGGED, true> : rmsnorm_e4m3_kernel<T, NV, TPR, RAGGED, false>;
  EMK_CUDA_TRY(h, launch_after_prologue(kernel, grid, 256, 0, s, h->overlap_launch != 0, x, residual, w, q, scale, hidden,
                                        rows, cols, eps));
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}

// Threads per row: as few as hold it in four packs each where there are rows for all SMs (short chains of reductions, many
// rows in flight), a whole CTA of more than 128 packs where there are not (the row's latency counts: 64 x 4096 bf16 with a
// residual 2.2 us, with half a CTA a row 3.3; 1024 x 4096 7.7 and 9.0).
template <typename T, bool RAGGED>
int launch_packs(emk_handle_t h, const T* x, const T* residual, const T* w, uint8_t* q, float* scale, T* hidden, int64_t rows,
                 int cols, float eps, cudaStream_t s) {
  const int n = cols / Raw<T>::V > 0 ? cols / Raw<T>::V : 1;  // full packs a row has at most
#define EMK_NORM(NV, TPR) launch_rows<T, NV, TPR, RAGGED>(h, x, residual, w, q, scale, hidden, rows, cols, eps, s)
  if (rows >= (int64_t)h->sm_count * 8) {
    if (n <= 8) return EMK_NORM(1, 8);
    if (n <= 16) return EMK_NORM(2, 8);
    if (n <= 32) return EMK_NORM(4, 8);
    if (n <= 64) return EMK_NORM(2, 32);
    if (n <= 128) return EMK_NORM(4, 32);
    if (n <= 256) return EMK_NORM(4, 64);
  }
  if (n <= 128) return EMK_NORM(1, 128);
  if (n <= 256) return EMK_NORM(1, 256);
  if (n <= 512) return EMK_NORM(2, 256);
  if (n <= 1024) return EMK_NORM(4, 256);
  return EMK_NORM(8, 256);
#undef EMK_NORM
}

template <typename T>
int launch(emk_handle_t h, const void* x, const void* residual, const void* w, void* q, float* scale, void* hidden,
           int64_t rows, int64_t cols, float eps, cudaStream_t s) {
  constexpr int V = Raw<T>::V;
  const T *xt = (const T*)x, *rt = (const T*)residual, *wt = (const T*)w;
  const bool packs = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)hidden) & 15u) == 0 && ((uintptr_t)q & (V - 1)) == 0;
  if (packs && cols / V <= 2048) {
    if (cols % V == 0 && ((uintptr_t)w & 15u) == 0)
      return launch_packs<T, false>(h, xt, rt, wt, (uint8_t*)q, scale, (T*)hidden, rows, (int)cols, eps, s);
    return launch_packs<T, true>(h, xt, rt, wt, (uint8_t*)q, scale, (T*)hidden, rows, (int)cols, eps, s);
  }
  const unsigned grid = (unsigned)(rows < (int64_t)h->sm_count * 16 ? rows : (int64_t)h->sm_count * 16);
  const bool vectors = packs && cols % V == 0 && ((uintptr_t)w & 15u) == 0;
  const auto kernel = vectors ? rmsnorm_e4m3_long_kernel<T, V> : rmsnorm_e4m3_long_kernel<T, 1>;
  EMK_CUDA_TRY(h, launch_after_prologue(kernel, grid, 256, 0, s, h->overlap_launch != 0, xt, rt, wt, (uint8_t*)q, scale,
                                        (T*)hidden, rows, cols, eps));
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
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
