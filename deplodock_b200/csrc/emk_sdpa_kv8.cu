// Attention of one or a few query tokens per sequence over the paged e4m3 cache (emk_kv8.cuh), grouped KV heads:
//   o = softmax(scale * q K^T) V,  K = k_codes * k_scale[page, head],  V = v_codes * v_scale[page, head]
// query i of Sq sits at position len - Sq + i and sees the tokens up to itself; a row that sees nothing gives zeros.
//
// Bound by HBM: every cached byte is read once and meets 4 * (Hq/Hkv) * Sq flops. The rows that share a KV head (Hq/Hkv
// heads x Sq queries) form tiles of 16 and go through mma.sync m16n8k16 in f16 with fp32 sums: at a few rows per cache
// byte the tensor-memory path would be fed 1/16 full tiles, and what counts is the flow of bytes. Each lane of a warp copies
// with cp.async exactly the bytes that its own mma fragments need (four stages of 16 tokens in flight per warp), so the
// loop has no barrier: the token and channel order inside a fragment is permuted alike for both operands, which a sum does
// not notice.
//   K fragment: lane (g, t) holds token g and 8 + g, channels 16t.. and 64 + 16t..   (4 bytes = one k16 step)
//   V fragment: lane (g, t) holds tokens 2t, 2t+1, 2t+8, 2t+9, channels 16g..         (pairs of tokens interleaved by prmt)
//
// e4m3 -> f16 is exact. q is scaled per row by a power of two into f16's range (exact; elements 2^-38 below the row's
// largest may lose bits, far below the fp32 sum's own rounding). The scales of keys go into the logits; the scale of
// values cannot multiply the probabilities directly (f16's range), so the running maximum is kept over logit +
// log2(v_scale) and p * v_scale / max is what is rounded to f16 (2^-12 relative: p in [0, 2^15], so 2^-29 of the largest
// contribution is still normal), while the sum of the probabilities divides that scale out again in fp32.
//
// Work split: the tiles of 16 tokens of all (sequence, KV head, row tile) form one list, cut into equal ranges, one per
// warp: sequences of any mix of lengths load all SMs alike without the host knowing the lengths, and a warp needs nothing of
// its neighbours. Beginning a row costs a warp about as much as a tile (the queries, a pipeline to fill, an output), so a
// row counts ROW_COST tiles more than it has. A row that falls into one range is finished there; the others leave
// (maximum, sum, o) per range in the workspace, at most two per warp, and a second kernel joins them.
#include "emk_kv8.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace {

using namespace emk;

constexpr int SK_WARPS = 4;
constexpr int SK_THREADS = SK_WARPS * 32;
constexpr int SK_STAGES = 4;
constexpr int SK_TILE = 16;  // tokens
constexpr int ROW_COST = 1;
constexpr int SK_ROWS = 16;
constexpr int SK_CTAS_PER_SM = 3;
constexpr int SK_JOIN_WARPS = 16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float P_SHIFT = 8.f;  // p is rounded as 2^8 p: with the lazy maximum (below) at most 2^15
constexpr float LAZY = 7.f;     // the running maximum moves when the new one is more than 2^7 above it
constexpr float V_SCALE_MIN = 7.888609052210118e-31f;  // 2^-100: a zero scale (a page of zeros) has a logarithm

struct SdpaArgs {
  const __nv_bfloat16* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  const int32_t* lens;
  __nv_bfloat16* o;
  int64_t ld_q;
  int B, Sq, Hq, Hkv, G, row_tiles, row_cap, page_shift, max_pages, num_pages;
  float scale_log2;
  int2* info;    // [B * Hkv * row_tiles]: first and last range of the row
  float2* ml;    // [ranges][2][row_cap]: maximum, sum
  float* part;   // [ranges][2][row_cap][D]
  int* status;
};

__device__ __forceinline__ int seq_len(const SdpaArgs& a, int b) {
  const int64_t room = (int64_t)a.max_pages << a.page_shift;
  const int n = __ldg(a.lens + b);
  if (n < 0 || n > room) emk_record_bounds(a.status, EMK_DEV_BOUNDS_CACHE_LEN);
  return (int)min((int64_t)max(n, 0), room);
}
__device__ __forceinline__ int seq_tiles(int len) { return (int)(((int64_t)len + SK_TILE - 1) / SK_TILE); }
// what a row of `tiles` tiles counts in the list
__device__ __forceinline__ int64_t row_units(int tiles) { return tiles > 0 ? (int64_t)tiles + ROW_COST : 0; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// two e4m3 codes in the low half of w -> f16 pair
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w) {
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Unit `u` of `total` lies in range range_owner(u); range c is [c * total / ranges, (c+1) * total / ranges).
__device__ __forceinline__ int64_t range_start(int64_t c, int64_t total, int64_t ranges) { return c * total / ranges; }
__device__ __forceinline__ int64_t range_owner(int64_t u, int64_t total, int64_t ranges) { return ((u + 1) * ranges - 1) / total; }

template <int D>
struct SkLayout {
  static constexpr int K_CHUNKS = D / 64 * 2;            // 16-byte pieces of K per lane and 16-token tile
  static constexpr int V_BYTES = D / 8;                  // bytes of V per lane and token (16 or 8)
  static constexpr int STAGE = 16 * D * 2;               // K and V of 16 tokens
  static constexpr int WARP_RING = SK_STAGES * STAGE;
  static constexpr int RING = SK_WARPS * WARP_RING;
  static constexpr int SCALES = SK_WARPS * SK_STAGES * 8;
  static constexpr int SMEM = RING + SCALES;
};

template <int D>
__global__ void __launch_bounds__(SK_THREADS, SK_CTAS_PER_SM) sdpa_kv8_kernel(const SdpaArgs a) {
  using L = SkLayout<D>;
  constexpr int STEPS = D / 16;  // k16 steps of q K^T
  constexpr int NT = D / 8;      // n8 tiles of P V
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int heads = a.Hkv * a.row_tiles;  // rows (of tiles) per sequence
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- this warp's range of the list ----
  int64_t total = 0;
  for (int i = lane; i < a.B; i += 32) total += row_units(seq_tiles(seq_len(a, i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= heads;
  const int64_t ranges = min((int64_t)gridDim.x * SK_WARPS, total);  // no more ranges than units: none is empty
  const int64_t range = (int64_t)blockIdx.x + (int64_t)warp * gridDim.x;  // neighbours in the list run on different SMs
  if (range >= ranges) return;
  int64_t pos = range_start(range, total, ranges);
  const int64_t end = range_start(range + 1, total, ranges);
  int b = 0;
  int64_t prefix = 0;  // index of sequence b's first unit
  for (int b0 = 0;; b0 += 32) {
    const int64_t mine = b0 + lane < a.B ? row_units(seq_tiles(seq_len(a, b0 + lane))) * heads : 0;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, pos < prefix + upto);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      b = b0 + src;
      prefix += __shfl_sync(0xffffffffu, upto - mine, src);
      break;
    }
    prefix += __shfl_sync(0xffffffffu, upto, 31);
    if (b0 + 32 >= a.B) return;  // not reached: pos lies before total
  }

  uint8_t* ring = smem + warp * L::WARP_RING;
  const uint32_t ring_u32 = smem_u32(ring);
  float* scale_ring = reinterpret_cast<float*>(smem + L::RING) + warp * SK_STAGES * 2;
  const uint32_t scale_u32 = smem_u32(scale_ring);
  const uint8_t* const no_bytes = a.k;  // a readable address for zero-filled pieces

  while (pos < end) {
    // ---- the next row and the part of it that is ours ----
    int len = seq_len(a, b);
    int tiles = seq_tiles(len);
    int64_t units = row_units(tiles);
    while (pos >= prefix + units * heads) {
      prefix += units * heads;
      ++b;
      len = seq_len(a, b);
      tiles = seq_tiles(len);
      units = row_units(tiles);
    }
    const int hr = (int)((pos - prefix) / units);
    const int64_t tile0 = prefix + hr * units + ROW_COST;  // the unit of the row's first tile
    const int ta = (int)max(pos - tile0, (int64_t)0);
    const int tb = (int)min(end - tile0, (int64_t)tiles);
    pos = min(end, tile0 + tiles);
    if (tb <= ta) continue;  // only what a row counts beside its tiles
    const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
    const int rows = min(SK_ROWS, a.G * a.Sq - rt * SK_ROWS);
    const int32_t* table = a.table + (int64_t)b * a.max_pages;
    const int nsub = tb - ta;

    // lane j holds the page of tile i0 + j of this warp's list, for the 32 tiles that are issued now and the next 32
    auto page_of = [&](int i) {
      const int s = ta + i;
      return i < nsub ? kv8_page_id(table, ((int64_t)s * 16) >> a.page_shift, a.num_pages, a.status) : 0;
    };
    int pid_now = page_of(lane), pid_next = page_of(32 + lane);
    auto issue = [&](int i) {
      if (i < nsub) {
        if ((i & 31) == 0 && i > 0) {
          pid_now = pid_next;
          pid_next = page_of(i + 32 + lane);
        }
        const int pid = __shfl_sync(0xffffffffu, pid_now, i & 31);
        const int s = ta + i;
        const int64_t unit = (int64_t)pid * a.Hkv + hkv;
        const int64_t at = ((unit << a.page_shift) + ((s * 16) & ((1 << a.page_shift) - 1))) * D;
        const int left = len - s * 16;  // tokens of this tile that exist: the others are zeros, whatever the page holds
        const uint32_t st = ring_u32 + (i % SK_STAGES) * L::STAGE;
        const uint8_t* kp = a.k + at;
        const uint8_t* vp = a.v + at;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int tok = u * 8 + g;
#pragma unroll
          for (int c = 0; c < L::K_CHUNKS / 2; ++c)
            cp_async16(st + (u * (L::K_CHUNKS / 2) + c) * 512 + lane * 16,
                       tok < left ? kp + tok * D + c * 64 + t * 16 : no_bytes, tok < left ? 16 : 0);
        }
        const uint32_t sv = st + 16 * D;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int tok = 2 * t + (u & 1) + (u >> 1) * 8;
          if (D == 128)
            cp_async16(sv + u * 512 + lane * 16, tok < left ? vp + tok * D + g * 16 : no_bytes, tok < left ? 16 : 0);
          else
            cp_async8(sv + u * 256 + lane * 8, tok < left ? vp + tok * D + g * 8 : no_bytes, tok < left ? 8 : 0);
        }
        if (lane < 2) cp_async4(scale_u32 + ((i % SK_STAGES) * 2 + lane) * 4, (lane == 0 ? a.ks : a.vs) + unit);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < SK_STAGES - 1; ++i) issue(i);

    // ---- q: rows g and g + 8 of the tile, channels as the K fragment has them ----
    uint32_t qf[STEPS][4];
    float qs[2];
    int limit[2];  // tokens that the row sees
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + r * 8;
      const int rr = rt * SK_ROWS + row;
      const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
      const bool valid = row < rows;
      const __nv_bfloat16* qp = a.q + ((int64_t)b * a.Sq + (valid ? qi : 0)) * a.ld_q + (int64_t)(valid ? head : 0) * D + t * 16;
      uint32_t raw[D / 8];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint4 v = valid ? *reinterpret_cast<const uint4*>(qp + c * 64 + p * 8) : make_uint4(0, 0, 0, 0);
          raw[c * 8 + p * 4] = v.x;
          raw[c * 8 + p * 4 + 1] = v.y;
          raw[c * 8 + p * 4 + 2] = v.z;
          raw[c * 8 + p * 4 + 3] = v.w;
        }
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) amax = max_nan(amax, max_nan(fabsf(bf16_lo(raw[i])), fabsf(bf16_hi(raw[i]))));
      amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // 2^(14 - exponent of the largest), within the normal floats
      const int e = min(max(127 + 14 - ((int)(__float_as_uint(amax) >> 23) - 127), 1), 253);
      const float up = __uint_as_float((uint32_t)e << 23);
      qs[r] = amax <= 3.402823466e38f ? a.scale_log2 / up : __uint_as_float(0x7fc00000u);  // a row with no finite scores
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {  // step j: channels 64 (j / 4) + 16 t + 4 (j % 4) + {0, 1}, {2, 3}
        const uint32_t lo = raw[(j >> 2) * 8 + (j & 3) * 2], hi = raw[(j >> 2) * 8 + (j & 3) * 2 + 1];
        qf[j][r] = pack_f16x2(bf16_lo(lo) * up, bf16_hi(lo) * up);
        qf[j][2 + r] = pack_f16x2(bf16_lo(hi) * up, bf16_hi(hi) * up);
      }
      limit[r] = valid ? max(len - a.Sq + qi + 1, 0) : len;  // rows past the last are computed and dropped
    }
    const int limit_min = __reduce_min_sync(0xffffffffu, min(limit[0], limit[1]));

    float o[NT][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    for (int i = 0; i < nsub; ++i) {
      __syncwarp();  // all lanes have read the scales of the stage that is overwritten next
      issue(i + SK_STAGES - 1);
      cp_async_wait<SK_STAGES - 1>();
      __syncwarp();
      const uint8_t* st = ring + (i % SK_STAGES) * L::STAGE;
      const float ks = scale_ring[(i % SK_STAGES) * 2];
      const float vs_raw = scale_ring[(i % SK_STAGES) * 2 + 1];
      const float vs = max_nan(vs_raw, V_SCALE_MIN);

      // ---- logits: 16 rows x 16 tokens ----
      float s[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
        for (int c = 0; c < L::K_CHUNKS / 2; ++c) {
          const uint4 kv = *reinterpret_cast<const uint4*>(st + (u * (L::K_CHUNKS / 2) + c) * 512 + lane * 16);
          const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_f16(s[u], qf[c * 4 + j], e4m3x2_f16x2(w[j]), e4m3x2_f16x2(w[j] >> 16));
        }
      }
      const float c0 = qs[0] * ks, c1 = qs[1] * ks;
      const float lvs = lg2(vs), inv_vs = 1.0f / vs;
      const int tok0 = (ta + i) * 16 + 2 * t;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u][0] = fmaf(s[u][0], c0, lvs);
        s[u][1] = fmaf(s[u][1], c0, lvs);
        s[u][2] = fmaf(s[u][2], c1, lvs);
        s[u][3] = fmaf(s[u][3], c1, lvs);
      }
      if (tok0 - 2 * t + 16 > limit_min) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tok0 + u * 8 + (e & 1) >= limit[e >> 1]) s[u][e] = -INFINITY;
        }
      }
      // ---- running maximum (of logit + log2 v_scale), moved only when it would be passed by more than 2^LAZY ----
      float mx[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      if (__any_sync(0xffffffffu, mx[0] - m[0] > LAZY || mx[1] - m[1] > LAZY)) {  // (a difference: m + 7 may round up)
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float to = fmaxf(m[r], mx[r]);
          f[r] = m[r] == -INFINITY ? 0.f : ex2(m[r] - to);
          m[r] = to;
          l[r] *= f[r];
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          o[j][0] *= f[0];
          o[j][1] *= f[0];
          o[j][2] *= f[1];
          o[j][3] *= f[1];
        }
      }
      const float sub[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
      float p[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[u][e] = ex2((s[u][e] - sub[e >> 1]) + P_SHIFT);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
        l[r] = fmaf((p[0][2 * r] + p[0][2 * r + 1]) + (p[1][2 * r] + p[1][2 * r + 1]), inv_vs, l[r]);
      const uint32_t pa[4] = {pack_f16x2(p[0][0], p[0][1]), pack_f16x2(p[0][2], p[0][3]), pack_f16x2(p[1][0], p[1][1]),
                              pack_f16x2(p[1][2], p[1][3])};
      if (vs_raw == 0.f) continue;  // a page of zeros: it counts in the sum and adds nothing (uniform over the warp)
      // ---- o += P V: n8 tile j has the channels j, NT + j, 2 NT + j, ... ----
      uint32_t w[4][L::V_BYTES / 4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if constexpr (D == 128) {
          const uint4 v = *reinterpret_cast<const uint4*>(st + 16 * D + u * 512 + lane * 16);
          w[u][0] = v.x;
          w[u][1] = v.y;
          w[u][2] = v.z;
          w[u][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(st + 16 * D + u * 256 + lane * 8);
          w[u][0] = v.x;
          w[u][1] = v.y;
        }
      }
#pragma unroll
      for (int j = 0; j < L::V_BYTES / 4; ++j) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t a01 = __byte_perm(w[0][j], w[1][j], half == 0 ? 0x5140 : 0x7362);
          const uint32_t a89 = __byte_perm(w[2][j], w[3][j], half == 0 ? 0x5140 : 0x7362);
          mma_f16(o[j * 4 + half * 2], pa, e4m3x2_f16x2(a01), e4m3x2_f16x2(a89));
          mma_f16(o[j * 4 + half * 2 + 1], pa, e4m3x2_f16x2(a01 >> 16), e4m3x2_f16x2(a89 >> 16));
        }
      }
    }

    // ---- this range's part of the row: channels [2 t NT, (2 t + 2) NT) of rows g and g + 8 per lane ----
    cp_async_wait<0>();
    const bool whole = ta == 0 && tb == tiles;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int row = g + 8 * r;
      if (row < rows) {
        if (whole) {
          const int rr = rt * SK_ROWS + row;
          const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
          const float inv = l[r] == 0.f ? 0.f : 1.0f / l[r];
          __nv_bfloat16* out = a.o + (((int64_t)b * a.Sq + qi) * a.Hq + head) * D + 2 * t * NT;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int j = 0; j < NT; j += 8)
              *reinterpret_cast<uint4*>(out + c * NT + j) =
                  make_uint4(pack_bf16x2(o[j][2 * r + c] * inv, o[j + 1][2 * r + c] * inv),
                             pack_bf16x2(o[j + 2][2 * r + c] * inv, o[j + 3][2 * r + c] * inv),
                             pack_bf16x2(o[j + 4][2 * r + c] * inv, o[j + 5][2 * r + c] * inv),
                             pack_bf16x2(o[j + 6][2 * r + c] * inv, o[j + 7][2 * r + c] * inv));
          }
        } else {
          // the first part of a row ends its range (slot 1), any other begins it (slot 0)
          const int64_t at = (range * 2 + (ta == 0 ? 1 : 0)) * a.row_cap + row;
          if (t == 0) a.ml[at] = make_float2(m[r], l[r]);
          float* out = a.part + at * D + 2 * t * NT;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int j = 0; j < NT; j += 4)
              *reinterpret_cast<float4*>(out + c * NT + j) =
                  make_float4(o[j][2 * r + c], o[j + 1][2 * r + c], o[j + 2][2 * r + c], o[j + 3][2 * r + c]);
          }
        }
      }
    }
    if (ta == 0 && lane == 0)
      a.info[(int64_t)b * heads + hr] = make_int2((int)range, (int)range_owner(tile0 + tiles - 1, total, ranges));
    __syncwarp();
  }
}

// Joins the ranges of every row that was cut: block (row of tiles, row of the tile), the partial results dealt to warps.
template <int D>
__global__ void __launch_bounds__(SK_JOIN_WARPS * 32) sdpa_kv8_join_kernel(const SdpaArgs a) {
  constexpr int E = D / 32;  // channels per lane
  __shared__ float s_m[SK_JOIN_WARPS], s_l[SK_JOIN_WARPS];
  __shared__ float s_o[SK_JOIN_WARPS][D];
  grid_dependency_wait();
  grid_launch_dependents();
  const int heads = a.Hkv * a.row_tiles;
  const int b = blockIdx.x / heads, hr = blockIdx.x - b * heads;
  const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
  const int rr = rt * SK_ROWS + blockIdx.y;
  if (rr >= a.G * a.Sq) return;
  const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __nv_bfloat16* out = a.o + (((int64_t)b * a.Sq + qi) * a.Hq + head) * D;
  if (seq_len(a, b) == 0) {  // no tile, so no warp wrote this row
    if (threadIdx.x < D / 8) reinterpret_cast<uint4*>(out)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int2 span = a.info[blockIdx.x];
  if (span.x == span.y) return;
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int c = span.x + warp; c <= span.y; c += SK_JOIN_WARPS) {
    const int64_t at = ((int64_t)c * 2 + (c == span.x ? 1 : 0)) * a.row_cap + blockIdx.y;
    const float2 ml = a.ml[at];
    const float* p = a.part + at * D + lane * E;
    float v[E];
    if constexpr (E == 4) {
      const float4 u = *reinterpret_cast<const float4*>(p);
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
      const float2 u = *reinterpret_cast<const float2*>(p);
      v[0] = u.x; v[1] = u.y;
    }
    const float top = fmaxf(m, ml.x);
    const float f0 = m == -INFINITY ? 1.f : ex2(m - top), f1 = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);
    m = top;
    l = fmaf(l, f0, ml.y * f1);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], f0, v[e] * f1);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < SK_JOIN_WARPS; ++w) top = fmaxf(top, s_m[w]);
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < SK_JOIN_WARPS; ++w) {
      const float f = s_m[w] == -INFINITY ? 1.f : ex2(s_m[w] - top);
      sum = fmaf(s_l[w], f, sum);
      x = fmaf(s_o[w][threadIdx.x * 2], f, x);
      y = fmaf(s_o[w][threadIdx.x * 2 + 1], f, y);
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    reinterpret_cast<uint32_t*>(out)[threadIdx.x] = pack_bf16x2(x * inv, y * inv);
  }
}

int64_t align16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// Every product of the sizes that the kernels form in 32 bits fits.
bool sizes_ok(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv) {
  const int64_t limit = 0x7fffffff;
  if (B <= 0 || Sq <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return false;
  if (B > limit || Sq > limit || Hq > limit || Sq > limit / (Hq / Hkv)) return false;
  const int64_t row_tiles = (Hq / Hkv * Sq + SK_ROWS - 1) / SK_ROWS;
  return Hkv <= limit / row_tiles && B <= limit / (Hkv * row_tiles);
}

struct SkPlan {
  int row_tiles, row_cap;
  int64_t ctas, info_bytes, ml_bytes, part_bytes;
};

// The grid never has more warps than the longest possible list has units.
SkPlan plan_of(int sm_count, int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t max_tokens, int64_t D) {
  SkPlan p;
  p.row_tiles = (int)((Hq / Hkv * Sq + SK_ROWS - 1) / SK_ROWS);
  p.row_cap = Hq / Hkv * Sq < SK_ROWS ? (int)(Hq / Hkv * Sq) : SK_ROWS;
  const int64_t units = (max_tokens + SK_TILE - 1) / SK_TILE + ROW_COST;  // below 2^28
  const int64_t rows = B * Hkv * p.row_tiles;                              // below 2^31
  p.ctas = (int64_t)sm_count * SK_CTAS_PER_SM;
  if ((rows * units + SK_WARPS - 1) / SK_WARPS < p.ctas) p.ctas = (rows * units + SK_WARPS - 1) / SK_WARPS;
  p.info_bytes = align16(rows * (int64_t)sizeof(int2));
  p.ml_bytes = align16(p.ctas * SK_WARPS * 2 * p.row_cap * (int64_t)sizeof(float2));
  p.part_bytes = p.ctas * SK_WARPS * 2 * p.row_cap * D * (int64_t)sizeof(float);
  return p;
}

template <int D>
int launch_sdpa(emk_handle_t h, const SdpaArgs& a, const SkPlan& p, cudaStream_t s) {
  static emk_device_once once;
  {
    std::lock_guard<std::mutex> lk(once.mu);
    if (!once.done[h->device]) {
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(sdpa_kv8_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SkLayout<D>::SMEM));
      once.done[h->device] = true;
    }
  }
  EMK_CUDA_TRY(h, launch_after_prologue(sdpa_kv8_kernel<D>, (unsigned)p.ctas, SK_THREADS, SkLayout<D>::SMEM, s,
                                        h->overlap_launch != 0, a));
  EMK_LAUNCH_CHECK(h);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.row_tiles), (unsigned)a.row_cap, 1);
  cfg.blockDim = dim3(SK_JOIN_WARPS * 32, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = h->overlap_launch != 0 ? 1 : 0;
  EMK_CUDA_TRY(h, cudaLaunchKernelEx(&cfg, sdpa_kv8_join_kernel<D>, a));
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}

}  // namespace

extern "C" int64_t emk_sdpa_kv8_workspace_bytes(emk_handle_t h, int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv,
                                                int64_t max_tokens, int64_t D) {
  if (!h || !sizes_ok(B, Sq, Hq, Hkv) || max_tokens <= 0 || max_tokens > 0x7fffffff || (D != 64 && D != 128)) return 0;
  const SkPlan p = plan_of(h->sm_count, B, Sq, Hq, Hkv, max_tokens, D);
  return p.info_bytes + p.ml_bytes + p.part_bytes;
}

extern "C" int emk_sdpa_kv8(emk_handle_t h, const void* q, int64_t ld_q, const void* k_codes, const void* v_codes,
                            const float* k_scale, const float* v_scale, const int32_t* page_table, const int32_t* seq_lens,
                            void* o, int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D, int64_t page,
                            int64_t max_pages, int64_t num_pages, float scale, void* workspace, int64_t workspace_bytes,
                            emk_stream_t stream) {
  if (!h || !q || !k_codes || !v_codes || !k_scale || !v_scale || !page_table || !seq_lens || !o || !workspace)
    return EMK_ERR_ARG;
  if ((D != 64 && D != 128) || !kv8_page_ok(page)) {
    EMK_SET_ERR(h, "emk_sdpa_kv8: head dimension 64 or 128 and a page of 16, 32, 64, 128 or 256 tokens; got D=%lld page=%lld",
                (long long)D, (long long)page);
    return EMK_ERR_SHAPE;
  }
  if (B <= 0 || Sq <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_pages <= 0 || num_pages <= 0 ||
      num_pages > 0x7fffffff || max_pages > 0x7fffffff / page || ld_q / D < Hq)
    return EMK_ERR_SHAPE;
  if (!sizes_ok(B, Sq, Hq, Hkv)) {
    EMK_SET_ERR(h, "emk_sdpa_kv8: more than 2^31 - 1 tiles of 16 query rows");
    return EMK_ERR_LIMIT;
  }
  if (((uintptr_t)q & 15u) != 0 || (ld_q & 7) != 0 || (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)o) & 15u) != 0 ||
      (((uintptr_t)k_scale | (uintptr_t)v_scale | (uintptr_t)page_table | (uintptr_t)seq_lens) & 3u) != 0 ||
      ((uintptr_t)workspace & 15u) != 0)
    return EMK_ERR_ALIGN;
  const SkPlan p = plan_of(h->sm_count, B, Sq, Hq, Hkv, max_pages * page, D);
  if (workspace_bytes < p.info_bytes + p.ml_bytes + p.part_bytes) {
    EMK_SET_ERR(h, "emk_sdpa_kv8: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)(p.info_bytes + p.ml_bytes + p.part_bytes));
    return EMK_ERR_WORKSPACE;
  }
  SdpaArgs a = {};
  a.q = (const __nv_bfloat16*)q;
  a.k = (const uint8_t*)k_codes;
  a.v = (const uint8_t*)v_codes;
  a.ks = k_scale;
  a.vs = v_scale;
  a.table = page_table;
  a.lens = seq_lens;
  a.o = (__nv_bfloat16*)o;
  a.ld_q = ld_q;
  a.B = (int)B;
  a.Sq = (int)Sq;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.row_tiles = p.row_tiles;
  a.row_cap = p.row_cap;
  a.page_shift = __builtin_ctzll((unsigned long long)page);
  a.max_pages = (int)max_pages;
  a.num_pages = (int)num_pages;
  a.scale_log2 = scale * LOG2E;
  uint8_t* ws = (uint8_t*)workspace;
  a.info = (int2*)ws;
  a.ml = (float2*)(ws + p.info_bytes);
  a.part = (float*)(ws + p.info_bytes + p.ml_bytes);
  a.status = h->status_dev;
  return D == 128 ? launch_sdpa<128>(h, a, p, (cudaStream_t)stream) : launch_sdpa<64>(h, a, p, (cudaStream_t)stream);
}
