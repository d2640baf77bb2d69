// Appending keys and values to the paged e4m3 cache (emk_kv8.cuh).
//   scale of a page and head = 2^e, e the smallest integer in [-64, 120] with max |finite value| <= 448 * 2^e
// over the tokens the page holds. A page that keeps earlier tokens never shrinks its scale: new = max(old, scale of the
// appended tokens), and where it grows the codes already there are rounded again, e4m3(code * old / new).
//
// Why powers of two: the codes are floating point, so a finer scale buys no relative precision, x / 2^e is exact (one
// rounding per value, the same bits from any correct program), and a growing scale only moves the exponents of the codes
// already there: they lose bits only where they fall below e4m3's normal range (2^-6), and such a code may be rounded once
// more each time its page's scale grows. Non-finite values become NaN codes and do not enter the scale: one bad token
// must not wipe out its page.
//
// Bound by HBM for prompts (2 bytes read, 1 written per value), by launch latency for single tokens. One CTA owns one
// (touched page, KV head, K or V): the page's maximum, its scale and the rewrite of its earlier codes need no other CTA, so
// there are no atomics and no second pass over the cache. The appended rows are read twice (maximum, then codes); the
// second read of at most 64 KB comes from L1 / L2.
#include "emk_kv8.cuh"

#include <cuda_fp8.h>

namespace {

using namespace emk;

constexpr int AP_THREADS = 128;

struct AppendArgs {
  const __nv_bfloat16* x[2];  // keys, values: [T] rows of pitch ld, head h at h * D
  int64_t ld[2];
  uint8_t* codes[2];
  float* scales[2];
  const int32_t* table;
  const int32_t* ctx_lens;
  const int32_t* cu;
  int B, max_pages, num_pages, Hkv, page_shift;
  int64_t T;
  int* status;
};

// the smallest 2^e with amax <= 448 * 2^e (448 = 1.75 * 2^8), e in [-64, 120]; amax finite and not negative
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, -64), 120);  // zeros and subnormals have the lowest exponent field and end at -64
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;  // false for infinities and NaN
}
// values past the finite range become NaN before the saturating conversion
__device__ __forceinline__ float nan_if_infinite(float v) { return fabsf(v) <= 3.402823466e38f ? v : __uint_as_float(0x7fc00000u); }

__device__ __forceinline__ void rescale_codes4(uint32_t& c, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((c >> (16 * p)) & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
    out |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3) << (16 * p);
  }
  c = out;
}

template <int D>
__global__ void __launch_bounds__(AP_THREADS) kv8_append_kernel(const AppendArgs a) {
  constexpr int LPT = D / 8;  // lanes (16-byte pieces) per token
  constexpr int TPP = AP_THREADS / LPT;  // tokens per pass of the CTA
  __shared__ float red[AP_THREADS / 32];
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.y, which = blockIdx.z;
  const int page = 1 << a.page_shift;

  // ---- which sequence and which of its touched pages is item blockIdx.x (every warp finds it for itself) ----
  int64_t item = blockIdx.x;
  int seq = -1;
  int64_t ctx = 0, t0 = 0, n = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    int64_t c_ctx = 0, c_t0 = 0, c_n = 0, count = 0;
    if (b < a.B) {
      const int64_t lo = a.cu[b], hi = a.cu[b + 1], held = a.ctx_lens[b];
      c_t0 = min(max(lo, (int64_t)0), a.T);
      c_n = max(min(hi, a.T) - c_t0, (int64_t)0);
      if (lo < 0 || hi > a.T || hi < lo) emk_record_bounds(a.status, EMK_DEV_BOUNDS_CU_SEQLENS);
      c_ctx = max(held, (int64_t)0);
      const int64_t room = ((int64_t)a.max_pages << a.page_shift) - c_ctx;
      if (held < 0 || c_n > max(room, (int64_t)0)) emk_record_bounds(a.status, EMK_DEV_BOUNDS_CACHE_LEN);
      c_n = min(c_n, max(room, (int64_t)0));  // tokens that the table's row cannot hold are dropped
      count = c_n > 0 ? ((c_ctx & (page - 1)) + c_n + page - 1) >> a.page_shift : 0;
    }
    int64_t upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, item < upto);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      item -= __shfl_sync(0xffffffffu, upto - count, src);
      seq = b0 + src;
      ctx = __shfl_sync(0xffffffffu, c_ctx, src);
      t0 = __shfl_sync(0xffffffffu, c_t0, src);
      n = __shfl_sync(0xffffffffu, c_n, src);
      break;
    }
    item -= __shfl_sync(0xffffffffu, upto, 31);
  }
  if (seq < 0) return;  // uniform: the grid is an upper bound of the touched pages

  const int64_t slot = (ctx >> a.page_shift) + item;             // which page of the sequence
  const int64_t first = max(ctx, slot << a.page_shift);          // first and one past the last new token position in it
  const int64_t last = min(ctx + n, (slot + 1) << a.page_shift);
  const int at = (int)(first & (page - 1));                      // tokens that stay in front of them
  const int m = (int)(last - first);
  const int pid = a.table[(int64_t)seq * a.max_pages + slot];
  if (pid < 0 || pid >= a.num_pages) {  // nothing is written through a bad id
    emk_record_bounds(a.status, EMK_DEV_BOUNDS_PAGE);
    return;
  }
  const int64_t ld = which == 0 ? a.ld[0] : a.ld[1];
  const __nv_bfloat16* x = (which == 0 ? a.x[0] : a.x[1]) + (t0 + (first - ctx)) * ld + (int64_t)head * D;
  uint8_t* codes = (which == 0 ? a.codes[0] : a.codes[1]) + (((int64_t)pid * a.Hkv + head) << a.page_shift) * D;
  float* scale_at = (which == 0 ? a.scales[0] : a.scales[1]) + (int64_t)pid * a.Hkv + head;
  const int tok = threadIdx.x / LPT, piece = threadIdx.x % LPT;

  // ---- the appended tokens' maximum ----
  float amax = 0.f;
  for (int t = tok; t < m; t += TPP) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + (int64_t)t * ld + piece * 8);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(finite_abs(bf16_lo(u[i])), finite_abs(bf16_hi(u[i]))));
  }
  amax = warp_max(amax);
  if (lane == 0) red[threadIdx.x >> 5] = amax;
  const float old = at > 0 ? *scale_at : 0.f;  // read by all before the barrier, written by one after it
  __syncthreads();
  amax = red[0];
#pragma unroll
  for (int i = 1; i < AP_THREADS / 32; ++i) amax = fmaxf(amax, red[i]);
  const float mine = pow2_scale(amax);
  const float s = at > 0 && !(old < mine) ? old : mine;

  // ---- earlier codes of the page, where its scale grew ----
  if (at > 0 && s != old) {
    const float ratio = old / s;
    for (int i = threadIdx.x; i < at * (D / 16); i += AP_THREADS) {
      uint4 v = reinterpret_cast<uint4*>(codes)[i];
      rescale_codes4(v.x, ratio);
      rescale_codes4(v.y, ratio);
      rescale_codes4(v.z, ratio);
      rescale_codes4(v.w, ratio);
      reinterpret_cast<uint4*>(codes)[i] = v;
    }
  }
  // ---- the new codes ----
  const float inv = 1.0f / s;  // exact: a power of two within 2^-120 .. 2^64
  for (int t = tok; t < m; t += TPP) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + (int64_t)t * ld + piece * 8);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(
                       make_float2(nan_if_infinite(bf16_lo(u[i])) * inv, nan_if_infinite(bf16_hi(u[i])) * inv),
                       __NV_SATFINITE, __NV_E4M3)
                   << (16 * (i & 1));
    *reinterpret_cast<uint2*>(codes + (int64_t)(at + t) * D + piece * 8) = make_uint2(o[0], o[1]);
  }
  if (threadIdx.x == 0 && s != old) *scale_at = s;
}

}  // namespace

extern "C" int emk_kv8_append(emk_handle_t h, const void* k, const void* v, int64_t ld_k, int64_t ld_v, void* k_codes,
                              void* v_codes, float* k_scale, float* v_scale, const int32_t* page_table,
                              const int32_t* ctx_lens, const int32_t* cu_seqlens, int64_t B, int64_t T, int64_t max_pages,
                              int64_t num_pages, int64_t Hkv, int64_t page, int64_t D, emk_stream_t stream) {
  if (!h || !k || !v || !k_codes || !v_codes || !k_scale || !v_scale || !page_table || !ctx_lens || !cu_seqlens)
    return EMK_ERR_ARG;
  if (B <= 0 || T <= 0 || max_pages <= 0 || num_pages <= 0 || Hkv <= 0 || Hkv > 65535 || B > 0x3fffffff ||
      T > 0x7fffffff || max_pages > 0x7fffffff || num_pages > 0x7fffffff)
    return EMK_ERR_SHAPE;
  if ((D != 64 && D != 128) || !kv8_page_ok(page)) {
    EMK_SET_ERR(h, "emk_kv8_append: head dimension 64 or 128 and a page of 16, 32, 64, 128 or 256 tokens; got D=%lld page=%lld",
                (long long)D, (long long)page);
    return EMK_ERR_SHAPE;
  }
  if (ld_k / D < Hkv || ld_v / D < Hkv) return EMK_ERR_SHAPE;
  if (((ld_k | ld_v) & 7) != 0 || (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_codes | (uintptr_t)v_codes) & 15u) != 0 ||
      (((uintptr_t)k_scale | (uintptr_t)v_scale | (uintptr_t)page_table | (uintptr_t)ctx_lens | (uintptr_t)cu_seqlens) & 3u) != 0)
    return EMK_ERR_ALIGN;
  AppendArgs a = {};
  a.x[0] = (const __nv_bfloat16*)k;
  a.x[1] = (const __nv_bfloat16*)v;
  a.ld[0] = ld_k;
  a.ld[1] = ld_v;
  a.codes[0] = (uint8_t*)k_codes;
  a.codes[1] = (uint8_t*)v_codes;
  a.scales[0] = k_scale;
  a.scales[1] = v_scale;
  a.table = page_table;
  a.ctx_lens = ctx_lens;
  a.cu = cu_seqlens;
  a.B = (int)B;
  a.T = T;
  a.max_pages = (int)max_pages;
  a.num_pages = (int)num_pages;
  a.Hkv = (int)Hkv;
  a.page_shift = __builtin_ctzll((unsigned long long)page);
  a.status = h->status_dev;
  // touched pages: every one holds a new token (<= T), and n tokens touch at most n / page + 2
  const int64_t items = T < T / page + 2 * B ? T : T / page + 2 * B;
  const dim3 grid((unsigned)items, (unsigned)Hkv, 2);
  if (D == 128) kv8_append_kernel<128><<<grid, AP_THREADS, 0, (cudaStream_t)stream>>>(a);
  else kv8_append_kernel<64><<<grid, AP_THREADS, 0, (cudaStream_t)stream>>>(a);
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}
