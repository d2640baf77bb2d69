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
// Bound by HBM for prompts (2 bytes read, 1 written per value), by launch latency for single tokens. One group of threads
// owns one (touched page, KV head, K or V): the page's maximum, its scale and the rewrite of its earlier codes need no one
// else, so there are no atomics and no second pass; the appended rows stay in registers (at most eight 16-byte pieces a
// thread) between the maximum and the codes. A CTA finds its page once and walks its heads. Which page that is needs no sum
// over the sequences: sequence b gets the places cu[b] / page + 2 b up to the next one's, never fewer than the pages it
// can touch, and a warp finds b among 32 places at a time.
// Measured, 64 sequences of 512 tokens behind up to 2000, 8 heads of 128 (201 MB): rows read twice, a CTA per head 49.0 us;
// rows in registers, values taken apart into floats 47.3; on pairs of bf16, which leaves the issue slots to eight CTAs an SM
// 38.4 (0.80 of the copy bandwidth). Pages of 16 tokens 86.9 and 37.5; 256 single tokens 16.1 and 5.2.
#include "emk_kv8.cuh"

#include <cuda_fp8.h>

namespace {

using namespace emk;

constexpr int AP_PIECES = 8;  // 16-byte pieces of a page's new rows that a thread holds

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
  int64_t items;  // places
  int groups;     // CTAs per place
  int* status;
};

// the smallest 2^e with amax <= 448 * 2^e (448 = 1.75 * 2^8), e in [-64, 120]; amax finite and not negative
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, -64), 120);  // zeros and subnormals have the lowest exponent field and end at -64
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Pairs of bf16 as they are loaded: taken apart into floats, a value cost eleven instructions and their issue was the bound.
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {  // the other one where one is NaN
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// NaN in the place of infinities: x * 0 + x
__device__ __forceinline__ uint4 finite_or_nan(uint4 v) {
  return make_uint4(fma_bf16x2(v.x, 0u, v.x), fma_bf16x2(v.y, 0u, v.y), fma_bf16x2(v.z, 0u, v.z), fma_bf16x2(v.w, 0u, v.w));
}
// running maximum of the magnitudes, a pair; v from finite_or_nan, whose NaN it passes over
__device__ __forceinline__ uint32_t max_abs(uint32_t m, uint4 v) {
  m = max_bf16x2(m, v.x & 0x7fff7fffu);
  m = max_bf16x2(m, v.y & 0x7fff7fffu);
  m = max_bf16x2(m, v.z & 0x7fff7fffu);
  return max_bf16x2(m, v.w & 0x7fff7fffu);
}
__device__ __forceinline__ float pair_max(uint32_t m) { return fmaxf(bf16_lo(m), bf16_hi(m)); }
// Codes of v / s for inv = 1 / s. The product is exact in bf16: s is a power of two (where it is not, because the caller's
// scale was none, this rounds once more), and what falls below bf16's range is a zero code anyway.
__device__ __forceinline__ uint2 piece_codes(uint4 v, float inv) {
  const uint32_t k = pack_bf16x2(inv, inv);
  const uint32_t w[4] = {mul_bf16x2(v.x, k), mul_bf16x2(v.y, k), mul_bf16x2(v.z, k), mul_bf16x2(v.w, k)};
  uint32_t o[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    o[j >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(bf16_lo(w[j]), bf16_hi(w[j])), __NV_SATFINITE, __NV_E4M3) << (16 * (j & 1));
  return make_uint2(o[0], o[1]);
}

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

// First place of sequence b (see the top): between 0 and items, not falling in b for lengths that do not fall.
__device__ __forceinline__ int64_t first_place(const AppendArgs& a, int b) {
  const int64_t t = min(max((int64_t)a.cu[b], (int64_t)0), a.T);
  return (t >> a.page_shift) + 2 * (int64_t)b;
}

// What a place stands for; false where nothing does.
struct Touched {
  int at, m;      // tokens that stay in the page, tokens that are appended to it
  int pid;
  int64_t row0;   // first appended row
};

__device__ __forceinline__ bool find_page(const AppendArgs& a, int64_t place, Touched& p) {
  const int lane = threadIdx.x & 31;
  const int page = 1 << a.page_shift;
  // the last sequence b with first_place(b) <= place, 32 candidates at a time (every warp finds it for itself)
  int lo = 0, n_left = a.B;  // b lies in [lo, lo + n_left)
  while (n_left > 1) {
    const int step = (n_left + 31) / 32;
    const bool before = lane * step < n_left && first_place(a, lo + lane * step) <= place;
    const unsigned m = __ballot_sync(0xffffffffu, before);
    const int i = m == 0 ? 0 : 31 - __clz(m);
    lo += i * step;
    n_left = min(step, n_left - i * step);
  }
  const int seq = lo;
  const int64_t t0 = min(max((int64_t)a.cu[seq], (int64_t)0), a.T);
  const int64_t t1 = a.cu[seq + 1], held = a.ctx_lens[seq];
  const int64_t ctx = max(held, (int64_t)0);
  const int64_t room = max(((int64_t)a.max_pages << a.page_shift) - ctx, (int64_t)0);
  int64_t n = max(min(t1, a.T) - t0, (int64_t)0);
  if (t1 > a.T || t1 < a.cu[seq] || a.cu[seq] < 0) emk_record_bounds(a.status, EMK_DEV_BOUNDS_CU_SEQLENS);
  if (held < 0 || n > room) emk_record_bounds(a.status, EMK_DEV_BOUNDS_CACHE_LEN);
  n = min(n, room);  // tokens that the table's row cannot hold are dropped
  const int64_t slot = (ctx >> a.page_shift) + place - first_place(a, seq);  // which page of the sequence
  const int64_t first = max(ctx, slot << a.page_shift);                      // new token positions in it: [first, last)
  const int64_t last = min(ctx + n, (slot + 1) << a.page_shift);
  if (last <= first) return false;  // a place beyond the sequence's pages
  p.at = (int)(first & (page - 1));
  p.m = (int)(last - first);
  p.row0 = t0 + (first - ctx);
  p.pid = a.table[(int64_t)seq * a.max_pages + slot];
  if (p.pid < 0 || p.pid >= a.num_pages) {  // nothing is written through a bad id
    emk_record_bounds(a.status, EMK_DEV_BOUNDS_PAGE);
    return false;
  }
  return true;
}

// One (head, K or V) of the page: where its rows come from and go to.
struct Unit {
  const __nv_bfloat16* x;
  int64_t ld;
  uint8_t* codes;
  float* scale;
};
template <int D>
__device__ __forceinline__ Unit unit_of(const AppendArgs& a, const Touched& p, int u) {
  const bool v = u >= a.Hkv;
  const int head = v ? u - a.Hkv : u;
  const int64_t slab = (int64_t)p.pid * a.Hkv + head;
  Unit r;
  r.ld = v ? a.ld[1] : a.ld[0];
  r.x = (v ? a.x[1] : a.x[0]) + p.row0 * r.ld + (int64_t)head * D;
  r.codes = (v ? a.codes[1] : a.codes[0]) + (slab << a.page_shift) * D;
  r.scale = (v ? a.scales[1] : a.scales[0]) + slab;
  return r;
}

// codes of the first `at` tokens, whose page's scale grew from old to s
template <int D>
__device__ __forceinline__ void rescale_page(uint8_t* codes, int at, float ratio, int tid, int threads) {
#pragma unroll 4
  for (int i = tid; i < at * (D / 16); i += threads) {
    uint4 c = reinterpret_cast<uint4*>(codes)[i];
    rescale_codes4(c.x, ratio);
    rescale_codes4(c.y, ratio);
    rescale_codes4(c.z, ratio);
    rescale_codes4(c.w, ratio);
    reinterpret_cast<uint4*>(codes)[i] = c;
  }
}

// Few tokens a sequence (few_tokens): a warp per (page, head, K or V), nothing held between the two readings of a row (the second one
// hits L1), so that all warps of a step are resident at once.
template <int D>
__global__ void __launch_bounds__(128) kv8_append_few_kernel(const AppendArgs a) {
  constexpr int LPT = D / 8, TPP = 32 / LPT;
  const int lane = threadIdx.x & 31;
  const int u = (int)(blockIdx.x % a.groups) * 4 + (threadIdx.x >> 5);
  Touched p;
  grid_dependency_wait();
  grid_launch_dependents();
  if (u >= 2 * a.Hkv || !find_page(a, blockIdx.x / a.groups, p)) return;  // (a warp at a time)
  const Unit r = unit_of<D>(a, p, u);
  const int tok = lane / LPT, piece = lane % LPT;
  const float old = p.at > 0 ? *r.scale : 0.f;
  uint32_t top = 0;
  for (int i = tok; i < p.m; i += TPP) top = max_abs(top, finite_or_nan(*reinterpret_cast<const uint4*>(r.x + (int64_t)i * r.ld + piece * 8)));
  const float amax = warp_max(pair_max(top));
  const float fresh = pow2_scale(amax);
  const float s = p.at > 0 && !(old < fresh) ? old : fresh;
  if (p.at > 0 && s != old) rescale_page<D>(r.codes, p.at, old / s, lane, 32);
  const float inv = 1.0f / s;  // exact: a power of two within 2^-120 .. 2^64
  for (int i = tok; i < p.m; i += TPP)
    *reinterpret_cast<uint2*>(r.codes + (int64_t)(p.at + i) * D + piece * 8) =
        piece_codes(finite_or_nan(*reinterpret_cast<const uint4*>(r.x + (int64_t)i * r.ld + piece * 8)), inv);
  __syncwarp();  // all lanes have read the old scale
  if (lane == 0 && s != old) *r.scale = s;
}

// TPU threads (a power of two from 32 to 512) per page and head; THREADS >= 128 per CTA. The heads of a page are neighbours
// in the grid: a token's keys of all heads lie side by side, and are read at about the same time.
template <int D, int TPU>
__global__ void __launch_bounds__(TPU < 128 ? 128 : TPU, TPU <= 128 ? 8 : TPU == 256 ? 4 : 2) kv8_append_kernel(const AppendArgs a) {
  constexpr int THREADS = TPU < 128 ? 128 : TPU;
  constexpr int GROUPS = THREADS / TPU, WPU = TPU / 32;
  constexpr int LPT = D / 8;       // pieces per token
  constexpr int TPP = TPU / LPT;   // tokens per round of the group
  __shared__ float red[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Touched p;
  grid_dependency_wait();
  grid_launch_dependents();
  if (!find_page(a, blockIdx.x / a.groups, p)) return;  // uniform
  const int group = threadIdx.x / TPU, tid = threadIdx.x % TPU;
  const int tok = tid / LPT, piece = tid % LPT;
  const int u = (int)(blockIdx.x % a.groups) * GROUPS + group;
  const bool mine = u < 2 * a.Hkv;
  const Unit r = unit_of<D>(a, p, mine ? u : 0);
  // ---- the appended tokens and their maximum ----
  uint4 v[AP_PIECES];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < AP_PIECES; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (mine && i * TPP + tok < p.m) v[i] = __ldcs(reinterpret_cast<const uint4*>(r.x + (int64_t)(i * TPP + tok) * r.ld + piece * 8));
  }
  const float old = mine && p.at > 0 ? *r.scale : 0.f;  // read by all before the barrier, written by one after it
#pragma unroll
  for (int i = 0; i < AP_PIECES; ++i) {
    v[i] = finite_or_nan(v[i]);
    top = max_abs(top, v[i]);
  }
  float amax = warp_max(pair_max(top));
  if (WPU > 1) {
    if (lane == 0) red[warp] = amax;
    __syncthreads();
    amax = red[warp / WPU * WPU];
#pragma unroll
    for (int i = 1; i < WPU; ++i) amax = fmaxf(amax, red[warp / WPU * WPU + i]);
  } else {
    __syncwarp();
  }
  if (!mine) return;
  const float fresh = pow2_scale(amax);
  const float s = p.at > 0 && !(old < fresh) ? old : fresh;
  if (p.at > 0 && s != old) rescale_page<D>(r.codes, p.at, old / s, tid, TPU);
  const float inv = 1.0f / s;
#pragma unroll
  for (int i = 0; i < AP_PIECES; ++i)
    if (i * TPP + tok < p.m)
      *reinterpret_cast<uint2*>(r.codes + (int64_t)(p.at + i * TPP + tok) * D + piece * 8) = piece_codes(v[i], inv);
  if (tid == 0 && s != old) *r.scale = s;
}

// A CTA per place and `per` of its heads (K and V apart)
template <typename K>
int launch_units(emk_handle_t h, K kernel, AppendArgs a, int per, int threads, cudaStream_t s) {
  a.groups = (2 * a.Hkv + per - 1) / per;
  if (a.items > 0x7fffffff / a.groups) {
    EMK_SET_ERR(h, "emk_kv8_append: more than 2^31 - 1 blocks");
    return EMK_ERR_LIMIT;
  }
  EMK_CUDA_TRY(h, launch_after_prologue(kernel, (unsigned)(a.items * a.groups), (unsigned)threads, 0, s, h->overlap_launch != 0, a));
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}
template <int D, int TPU>
int launch_append(emk_handle_t h, const AppendArgs& a, cudaStream_t s) {
  constexpr int THREADS = TPU < 128 ? 128 : TPU;
  return launch_units(h, kv8_append_kernel<D, TPU>, a, THREADS / TPU, THREADS, s);
}

// Few tokens a sequence: the warps of the few-kernel go through a page's new rows in turn, but the places that stand for nothing
// (half of them at a token a sequence) cost it a warp instead of a CTA of registers. Up to four tokens a sequence on average in any case;
// up to 16 where the other kernel's CTAs would fill the machine one and a half times, or more often for pages longer than 64
// tokens, whose rows a warp takes longer to go through. 64 sequences of 8 tokens: 3.9 us against 6.5, of 16: 5.0 / 7.1; 256 of 8:
// 6.7 / 17.9; 255 single tokens and a prompt of 2048: 12.2 / 17.9; but 8 of 16: 3.9 / 3.0, and 31 single tokens and a prompt of 256:
// 7.3 / 4.2. (Where one sequence of 64 has nearly all of the tokens: 7.4 / 6.8, in pages of 256 39 / 20.)
bool few_tokens(const AppendArgs& a, int64_t sm_count, int64_t D) {
  if (a.T <= 4 * (int64_t)a.B) return true;
  const int64_t page = (int64_t)1 << a.page_shift;
  const double fills = (double)a.items * 2. * a.Hkv * (double)(page * D / (8 * AP_PIECES)) / (1024. * (double)sm_count);
  return a.T <= 16 * (int64_t)a.B && fills >= 1.5 * (double)(page > 64 ? page : 64) / 64.;
}

template <int D>
int launch_append_page(emk_handle_t h, const AppendArgs& a, cudaStream_t s) {
  switch (((1 << a.page_shift) * D) / (8 * AP_PIECES)) {  // threads that hold a page's rows
    case 16:
    case 32: return launch_append<D, 32>(h, a, s);
    case 64: return launch_append<D, 64>(h, a, s);
    case 128: return launch_append<D, 128>(h, a, s);
    case 256: return launch_append<D, 256>(h, a, s);
    default: return launch_append<D, 512>(h, a, s);
  }
}

}  // namespace

extern "C" int emk_kv8_append(emk_handle_t h, const void* k, const void* v, int64_t ld_k, int64_t ld_v, void* k_codes,
                              void* v_codes, float* k_scale, float* v_scale, const int32_t* page_table,
                              const int32_t* ctx_lens, const int32_t* cu_seqlens, int64_t B, int64_t T, int64_t max_pages,
                              int64_t num_pages, int64_t Hkv, int64_t page, int64_t D, emk_stream_t stream) {
  if (!h || !k || !v || !k_codes || !v_codes || !k_scale || !v_scale || !page_table || !ctx_lens || !cu_seqlens)
    return EMK_ERR_ARG;
  if (B <= 0 || T <= 0 || max_pages <= 0 || num_pages <= 0 || Hkv <= 0 || Hkv > 0x1fffffff || B > 0x1fffffff ||
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
  a.items = T / page + 2 * B;  // places: first_place(B)
  cudaStream_t s = (cudaStream_t)stream;
  if (few_tokens(a, h->sm_count, D))
    return D == 128 ? launch_units(h, kv8_append_few_kernel<128>, a, 4, 128, s) : launch_units(h, kv8_append_few_kernel<64>, a, 4, 128, s);
  return D == 128 ? launch_append_page<128>(h, a, s) : launch_append_page<64>(h, a, s);
}
