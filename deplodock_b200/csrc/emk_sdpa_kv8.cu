// Attention of one or a few query tokens per sequence over the paged e4m3 cache (emk_kv8.cuh), grouped KV heads:
//   o = softmax(scale * q K^T) V,  K = k_codes * k_scale[page, head],  V = v_codes * v_scale[page, head]
// query i of Sq sits at position len - Sq + i and sees the tokens up to itself; a row that sees nothing gives zeros.
//
// Bound by HBM: every cached byte is read once and meets 4 * (Hq/Hkv) * Sq flops. The rows that share a KV head (Hq/Hkv
// heads x Sq queries) form tiles of 8 or 16 and go through mma.sync m16n8k16 in f16 with fp32 sums, the cache as the
// instruction's 16 rows and the queries as its 8 columns:
//   S^T [tokens x rows] = K q^T,   o^T [channels x rows] = V^T P^T
// so that a group of up to eight rows wastes nothing. (At a few rows per cache byte the tensor-memory path would be fed 1/16
// full tiles; what counts is the flow of bytes and the instructions per byte.) A TMA load brings a tile of 16
// tokens, 16 rows of one page, into the warp's own ring, a few tiles ahead; nothing in the loop waits for another warp. (With
// cp.async in the order of the fragments, 16 bytes of four rows side by side, every sector crossed twice and every lane took
// a shared-memory cycle of its own: 26 cycles an instruction, and that was the bound; in address order the copies still took
// the cycles that the fragment loads need.) The token and channel order inside a fragment is permuted alike for both
// operands, which a sum does not notice; the permutation of the tokens is the one that TMA's swizzle makes free of bank
// conflicts.
//   K fragment: lane (g, t) holds tokens p(g) and 8 + p(g), channels 16t.. and 64 + 16t..   (4 bytes = one k16 step)
//   V fragment: lane (g, t) holds tokens p(2t), p(2t+1), 8 + both, channels (D/8) g..       (pairs interleaved by prmt)
// P^T comes out of S^T by movmatrix.
//
// e4m3 -> f16 is exact. q is scaled per row by a power of two into f16's range: exact for elements down to 2^-31 of the row's
// largest; smaller ones are off by 2^-39 of that largest at most, far below the fp32 sum's own rounding. The
// scales of keys go into the logits; the scale of values cannot multiply the probabilities directly (f16's range), so the running
// maximum is kept over logit + log2(v_scale). A term of the sum is 2^(logit - maximum) in fp32; the term times its page's value
// scale, 2^8 at the maximum (up to 2^15 before that moves), is rounded to f16: off by 2^-11 relative at most down to 2^-22 of the
// row's largest, by 2^-33 of that largest below. That rounding is what lets the matrix instruction run in f16;
// the sum does not see it. The sum keeps a page however far its value scale lies below another's: its terms do not pass through
// the scaled probability, and where the maximum moves it is multiplied in two steps (decay).
//
// Four kernels share the loop. Many rows of few tiles (short_rows): a warp each. Where no sequence can be long (split_of): a
// cluster of CTAs takes a row tile, deals its tiles to its warps and joins their pieces in distributed shared memory, the
// CTAs of the longest sequences first; with few rows (wide_split_of) CTAs as large as an SM. One launch each. Otherwise:
// Work split: the tiles of 16 tokens of all (sequence, KV head, row tile) form one list, cut into equal ranges, one per
// warp: sequences of any mix of lengths load all SMs alike without the host knowing the lengths. Beginning a row costs a
// warp about as much as a tile (the queries, a pipeline to fill, an output), so a row counts ROW_COST tiles more than it
// has. A row that falls into one range, or into the ranges of one CTA, is finished there; the others leave
// (maximum, sum, o) per piece in the workspace and a second kernel joins them.
#include "emk_kv8.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace {

using namespace emk;

constexpr int SK_WARPS = 4;
constexpr int SK_THREADS = SK_WARPS * 32;
constexpr int SK_TILE = 16;  // tokens: inside one page
constexpr int ROW_COST = 1;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float P_SHIFT = 8.f;   // p is rounded as 2^8 p relative to the running maximum ...
constexpr float P_LIMIT = 15.f;  // ... which moves when a logit is more than 7 above it: the rounded p is at most 2^15
constexpr float BIG = 65536.f;   // from here on fp32 logits are so coarse that their differences need a clamp
constexpr float V_SCALE_MIN = 7.888609052210118e-31f;  // 2^-100: smaller value scales, zero among them, count as zero
// The sum's terms are 2^SUM_SHIFT times larger than the probabilities relative to the maximum, and no page's value scale is taken
// as less than 2^V_LOG_MIN in that maximum: so neither a term, at most 2^(15 + 20 + 68) and 2^24 of them a lane, nor a probability
// under the largest scale that appending makes (2^120) leaves fp32's normal range. (Appending makes none below 2^-64.)
constexpr float SUM_SHIFT = 20.f, SUM_UNIT = 9.5367431640625e-07f;  // 2^-20
constexpr float V_LOG_MIN = -68.f;

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
  int B, Sq, Hq, Hkv, G, row_tiles, tile_rows, row_cap, page_shift, max_pages, num_pages;
  float scale_log2;
  int2* info;    // [B * Hkv * row_tiles]: first and last range of the row
  float2* ml;    // [ranges][2][row_cap]: maximum, sum
  float* part;   // [ranges][2][row_cap][D]
  int max_ranges;
  int ranked;  // rows kernel: the longest sequences first
  int* status;
  unsigned long long limit_ns;
};

__device__ __forceinline__ int seq_len(const SdpaArgs& a, int b) {
  const int64_t room = (int64_t)a.max_pages << a.page_shift;
  const int n = a.lens[b];
  if (n < 0 || n > room) emk_record_bounds(a.status, EMK_DEV_BOUNDS_CACHE_LEN);
  return (int)min((int64_t)max(n, 0), room);
}
__device__ __forceinline__ int seq_tiles(int len) { return (int)(((int64_t)len + SK_TILE - 1) / SK_TILE); }
// what a row of `tiles` tiles counts in the list
__device__ __forceinline__ int row_units(int tiles) { return tiles > 0 ? tiles + ROW_COST : 0; }

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
// l * 2^d for d <= 0, in two steps: a sum of small value scales next to a maximum of a large one (2^184 apart by appending, so is l)
__device__ __forceinline__ float decay(float l, float d) {
  const float half = ex2(0.5f * d);
  return l * half * half;
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
// four e4m3 codes -> two f16 pairs (exact)
__device__ __forceinline__ void e4m3x4_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// the transpose of an 8 x 8 tile of 16-bit values, a pair of a row per lane
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Unit `u` of `total` lies in range range_owner(u); range c is [c * total / ranges, (c+1) * total / ranges).
__device__ __forceinline__ int64_t range_start(int64_t c, int64_t total, int64_t ranges) { return c * total / ranges; }
__device__ __forceinline__ int64_t range_owner(int64_t u, int64_t total, int64_t ranges) { return ((u + 1) * ranges - 1) / total; }

// Token of row r of an 8-row fragment half. K is read two rows (r even, r odd) to a quarter warp, V one half of every
// pair: with TMA's 128-byte swizzle (16-byte unit ^ row % 8) the tokens of a pair have to differ in bit 2 and the even rows'
// tokens in bits 1 and 2; with the 64-byte swizzle of D = 64 (unit ^ row / 2 % 4, two rows a line) the tokens of a pair in
// bit 0, and four even rows' tokens have to cover both halves of two lines.
template <int D>
__device__ __forceinline__ constexpr int token_of(int r) {
  if (D == 128) return r ^ ((r & 1) << 2);
  const int e = ((r >> 1) & 1) | (((r >> 1) & 2) << 1);
  return (r & 1) ? e ^ 3 : e;
}

// RT: tiles of 8 rows per row tile. One: 16 warps per SM with a 12 KB ring each; two (twice the accumulators and query
// fragments): as many warps as hold them in registers, 8 at D = 128 and 12 at D = 64. (A spill inside the loop costs more
// than a third of the warps: local memory has to pass an L1 that the rings leave a few KB.)
template <int D, int RT>
struct SkLayout {
  static constexpr int ROWS = 8 * RT;
  static constexpr int CTAS_PER_SM = RT == 1 ? 4 : D == 128 ? 2 : 3;
  static constexpr int K_CHUNKS = D / 64;                // 16-byte pieces of K per lane and token
  static constexpr int V_BYTES = D / 8;                  // bytes of V per lane and token (16 or 8)
  static constexpr int HALF = SK_TILE * D;               // K or V of a tile
  static constexpr int STAGE = 2 * HALF;
  static constexpr int STAGES = (RT == 1 ? 12 : D == 128 ? 24 : 16) * 1024 / STAGE;
  static constexpr int WARP_RING = STAGES * STAGE;
  static constexpr int RING = SK_WARPS * WARP_RING;
  static constexpr int SMEM = RING + 1024;                // the swizzle wants 1024-byte aligned slots
  static constexpr int PIECE_PITCH = D + 4;              // floats; spreads the rows over the banks
  static_assert(ROWS * PIECE_PITCH * 4 <= WARP_RING, "a warp's last piece lies over its ring");
};

// The wide kernel: one CTA per SM, of as many warps as its registers hold.
template <int D, int RT>
struct WideLayout {
  static constexpr int WARPS = RT == 1 ? 16 : 8;  // (of either head dimension)
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SMEM = WARPS * SkLayout<D, RT>::WARP_RING + 1024;
};

// Ring position of a warp: slots that are filled and used next (equal between two parts), phase of the latter's barrier.
struct RingAt {
  int slot, use;
  uint32_t phase;
};

// What a warp has of a row tile: o[n][j][2 x + e] is row n * 8 + 2 t + e, channel D / 8 * g + 2 j + x; m the running maximum of
// logit + log2 v_scale, l this lane's part of the sum of 2^(logit - m), both of the rows n * 8 + 2 t + e.
template <int D, int RT>
struct Part {
  float o[RT][D / 16][4];
  float m[RT][2], l[RT][2];
};

// A tile that not all rows see to its end: a NaN value must not reach the rows whose probability of its token is a masked zero
// (0 * NaN). NaN codes leave the fragment, and the rows that see their tokens get NaN in those channels here.
template <int D, int RT>
__device__ __forceinline__ void spoil_seen(uint32_t (&w)[4][D / 32], int tok0, const int (&limit)[RT][2], Part<D, RT>& part) {
  const auto nan_bytes = [](uint32_t codes) { return __vcmpeq4(codes & 0x7f7f7f7fu, 0x7f7f7f7fu); };
  uint32_t any = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) any |= nan_bytes(w[u][j]);
  }
  if (!__any_sync(0xffffffffu, any != 0)) return;
  const int lane = threadIdx.x & 31;
  uint32_t seen[RT][2] = {};  // bit c: channel D / 8 * g + c has a NaN among the tokens that the row sees
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t mine = 0;  // of this lane's token u
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t v = nan_bytes(w[u][j]);
      w[u][j] &= ~v;
      mine |= (((v & 0x08040201u) * 0x01010101u) >> 24) << (4 * j);  // a bit per byte
    }
#pragma unroll
    for (int src = 0; src < 4; ++src) {  // the four lanes that hold these channels
      const uint32_t theirs = __shfl_sync(0xffffffffu, mine, (lane & 28) | src);
      const int tok = tok0 + token_of<D>(2 * src + (u & 1)) + (u >> 1) * 8;
#pragma unroll
      for (int n = 0; n < RT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) seen[n][e] |= tok < limit[n][e] ? theirs : 0u;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < RT; ++n) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if ((seen[n][x & 1] >> (2 * j + (x >> 1))) & 1u) part.o[n][j][x] = __uint_as_float(0x7fc00000u);
    }
  }
}

// Tiles [ta, tb) of the row tile rt of KV head hkv of sequence b, by one warp. False: a wait ran out (recorded). EVEN: a query
// token per sequence, so that all rows see the same tokens (a kernel of its own: the limits per row and what follows from them cost
// 16 warps an SM registers that they do not have, 3 % of 64 sequences of 4096 tokens).
template <int D, int RT, bool EVEN>
__device__ __forceinline__ bool row_part(const SdpaArgs& a, const CUtensorMap& tma_k, const CUtensorMap& tma_v, uint8_t* ring,
                                         uint64_t* full, const WaitCtx& wc, RingAt& at, int b, int hkv, int rt, int len, int ta,
                                         int tb, Part<D, RT>& part) {
  using L = SkLayout<D, RT>;
  constexpr int STEPS = D / 16;  // k16 steps of K q^T, and m16 tiles of V^T P^T
  constexpr int ROWS = L::ROWS;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int page_mask = (1 << a.page_shift) - 1;
  // Where this lane's fragments are in a tile: K chunk c at ^ 64 c, V's second token of the pair at v_odd; + 8 rows: + 8 D
  const int tk = token_of<D>(g), tv0 = token_of<D>(2 * t), tv1 = token_of<D>(2 * t + 1);
  const int k_from = D == 128 ? tk * 128 + ((t ^ tk) << 4) : tk * 64 + ((t ^ ((tk >> 1) & 3)) << 4);
  const int v_even = D == 128 ? tv0 * 128 + ((g ^ tv0) << 4) : tv0 * 64 + (((g >> 1) ^ ((tv0 >> 1) & 3)) << 4) + (g & 1) * 8;
  const int v_odd = D == 128 ? tv1 * 128 + ((g ^ tv1) << 4) : tv1 * 64 + (((g >> 1) ^ ((tv1 >> 1) & 3)) << 4) + (g & 1) * 8;
  const int rows = min(ROWS, a.G * a.Sq - rt * ROWS);
  const int32_t* table = a.table + (int64_t)b * a.max_pages;
  const int nsub = tb - ta;

  // lane j holds the (page, head) of tile i0 + j of this part, for the 32 tiles that are issued now and the next 32
  auto unit_of = [&](int i) {
    return i < nsub ? kv8_page_id(table, ((int64_t)(ta + i) * SK_TILE) >> a.page_shift, a.num_pages, a.status) * a.Hkv + hkv : 0;
  };
  int unit_now = unit_of(lane), unit_next = unit_of(32 + lane);
  // and the scales of those 32 tiles, for the tiles that are issued and those that are used
  float ks_issue = a.ks[unit_now], vs_issue = a.vs[unit_now], ks_use = 0.f, vs_use = 0.f;
  auto issue = [&](int i) {
    if (i < nsub) {
      if ((i & 31) == 0 && i > 0) {
        unit_now = unit_next;
        unit_next = unit_of(i + 32 + lane);
        ks_issue = a.ks[unit_now];
        vs_issue = a.vs[unit_now];
      }
      const int unit = __shfl_sync(0xffffffffu, unit_now, i & 31);
      if (lane == 0) {
        const int row = (unit << a.page_shift) + (((ta + i) * SK_TILE) & page_mask);
        uint64_t* bar = &full[at.slot];
        mbar_arrive_expect_tx(bar, L::STAGE);
        tma_load_2d(ring + at.slot * L::STAGE, &tma_k, bar, 0, row);
        tma_load_2d(ring + at.slot * L::STAGE + L::HALF, &tma_v, bar, 0, row);
      }
      at.slot = at.slot + 1 == L::STAGES ? 0 : at.slot + 1;
    }
  };
#pragma unroll
  for (int i = 0; i < L::STAGES - 1; ++i) issue(i);

  // ---- q: row g of each 8-row tile, channels as the K fragment has them ----
  uint32_t qf[RT][STEPS][2];
  // of the rows whose logits this lane gets, 2 t and 2 t + 1 of each tile: factor of the logits, tokens that the row sees
  float qs[RT][2];
  int limit[RT][2];
  int limit_min = len;  // (EVEN: of all rows)
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    const int row = n * 8 + g;
    const int rr = rt * ROWS + row;
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
    const float factor = amax <= 3.402823466e38f ? a.scale_log2 / up : __uint_as_float(0x7fc00000u);  // a row with no finite scores
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {  // step j: channels 64 (j / 4) + 16 t + 4 (j % 4) + {0, 1}, {2, 3}
      const uint32_t lo = raw[(j >> 2) * 8 + (j & 3) * 2], hi = raw[(j >> 2) * 8 + (j & 3) * 2 + 1];
      qf[n][j][0] = pack_f16x2(bf16_lo(lo) * up, bf16_hi(lo) * up);
      qf[n][j][1] = pack_f16x2(bf16_lo(hi) * up, bf16_hi(hi) * up);
    }
    const int sees = valid ? max(len - a.Sq + qi + 1, 0) : len;  // rows past the last are computed and dropped
    if (!EVEN) limit_min = min(limit_min, __reduce_min_sync(0xffffffffu, sees));
#pragma unroll
    for (int e2 = 0; e2 < 2; ++e2) {
      qs[n][e2] = __shfl_sync(0xffffffffu, factor, (2 * t + e2) * 4);
      limit[n][e2] = EVEN ? len : __shfl_sync(0xffffffffu, sees, (2 * t + e2) * 4);
    }
  }

  // what is added to a logit: P_SHIFT - the running maximum
  float shift[RT][2];
  bool big = false;
#pragma unroll
  for (int n = 0; n < RT; ++n) {
#pragma unroll
    for (int j = 0; j < STEPS; ++j) part.o[n][j][0] = part.o[n][j][1] = part.o[n][j][2] = part.o[n][j][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      part.m[n][e] = -INFINITY;
      shift[n][e] = INFINITY;
      part.l[n][e] = 0.f;
    }
  }

  for (int i = 0; i < nsub; ++i) {
    __syncwarp();  // all lanes have read the slot that is filled next
    issue(i + L::STAGES - 1);
    if ((i & 31) == 0) {  // (fewer stages than 32: the tiles that are issued are of the same 32)
      ks_use = ks_issue;
      vs_use = vs_issue;
    }
    const float ks = __shfl_sync(0xffffffffu, ks_use, i & 31), vs_raw = __shfl_sync(0xffffffffu, vs_use, i & 31);
    if (!mbar_wait_warp(&full[at.use], at.phase, wc, EMK_DEV_TIMEOUT_SOFTMAX)) return false;
    const uint8_t* st = ring + at.use * L::STAGE;
    const uint8_t* sv = st + L::HALF;
    at.use = at.use + 1 == L::STAGES ? 0 : at.use + 1;
    at.phase ^= at.use == 0 ? 1u : 0u;

    // ---- logits: 16 tokens x 8 RT rows, two partial sums each ----
    float s[RT][4];
    {
      float s2[RT][2][4];
#pragma unroll
      for (int n = 0; n < RT; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s2[n][0][x] = s2[n][1][x] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < L::K_CHUNKS; ++c) {
        const uint4 ka = *reinterpret_cast<const uint4*>(st + (k_from ^ (c * 64)));            // token p(g)
        const uint4 kb = *reinterpret_cast<const uint4*>(st + (k_from ^ (c * 64)) + 8 * D);  // token 8 + p(g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_f16x4(j == 0 ? ka.x : j == 1 ? ka.y : j == 2 ? ka.z : ka.w, a0, a2);
          e4m3x4_f16x4(j == 0 ? kb.x : j == 1 ? kb.y : j == 2 ? kb.z : kb.w, a1, a3);
#pragma unroll
          for (int n = 0; n < RT; ++n) mma_f16(s2[n][j & 1], a0, a1, a2, a3, qf[n][c * 4 + j][0], qf[n][c * 4 + j][1]);
        }
      }
#pragma unroll
      for (int n = 0; n < RT; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[n][x] = s2[n][0][x] + s2[n][1][x];
      }
    }
    const float lvs = fmaxf(lg2(vs_raw), V_LOG_MIN);
    const float x_limit = P_LIMIT + SUM_SHIFT - lvs;
    const int tok = (ta + i) * SK_TILE + tk;
    const bool edge = (ta + i) * SK_TILE + SK_TILE > limit_min;  // some row does not see all of the tile
    // p[n][2 u + e]: row n * 8 + 2 t + e, token tok + 8 u: logit - maximum + SUM_SHIFT + P_SHIFT, the sum's term, the
    // probability. A row that has seen nothing yet has an infinite shift: its first visible logit makes the maximum move.
    float p[RT][4];
    auto exponents = [&]() {
#pragma unroll
      for (int n = 0; n < RT; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) p[n][x] = fmaf(s[n][x], qs[n][x & 1] * ks, shift[n][x & 1]);
        if (edge) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (tok + (x >> 1) * 8 >= limit[n][x & 1]) p[n][x] = -INFINITY;
        }
      }
    };
    exponents();
    float most = -INFINITY;
#pragma unroll
    for (int n = 0; n < RT; ++n) most = fmaxf(most, fmaxf(fmaxf(p[n][0], p[n][1]), fmaxf(p[n][2], p[n][3])));
    if (__any_sync(0xffffffffu, most > x_limit)) {  // rare after a row's first tiles: no shuffles otherwise
      big = false;
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (!edge || tok + u * 8 < limit[n][e]) mx = fmaxf(mx, fmaf(s[n][2 * u + e], qs[n][e] * ks, lvs));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float to = fmaxf(part.m[n][e], mx);
          f[e] = part.m[n][e] == -INFINITY ? 0.f : ex2(part.m[n][e] - to);
          part.l[n][e] = part.m[n][e] == -INFINITY ? part.l[n][e] * 0.f : decay(part.l[n][e], part.m[n][e] - to);
          part.m[n][e] = to;
          shift[n][e] = P_SHIFT + SUM_SHIFT - to;
          big = big || (to != -INFINITY && fabsf(to) > BIG);
        }
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          part.o[n][j][0] *= f[0];
          part.o[n][j][1] *= f[1];
          part.o[n][j][2] *= f[0];
          part.o[n][j][3] *= f[1];
        }
      }
      big = __any_sync(0xffffffffu, big);
      exponents();
    }
    if (big) {  // logits that differ by a rounding may differ by more than fp16 holds
#pragma unroll
      for (int n = 0; n < RT; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) p[n][x] = p[n][x] > x_limit ? x_limit : p[n][x];
      }
    }
    const float weight = vs_raw * SUM_UNIT;
    uint32_t pb[RT][2];  // P^T: row g, tokens 2 t, 2 t + 1 (+ 8)
#pragma unroll
    for (int n = 0; n < RT; ++n) {
#pragma unroll
      for (int x = 0; x < 4; ++x) p[n][x] = ex2(p[n][x]);
#pragma unroll
      for (int e = 0; e < 2; ++e) part.l[n][e] += p[n][e] + p[n][2 + e];
#pragma unroll
      for (int x = 0; x < 4; ++x) p[n][x] *= weight;
#pragma unroll
      for (int u = 0; u < 2; ++u) pb[n][u] = transpose8x8(pack_f16x2(p[n][2 * u], p[n][2 * u + 1]));
    }
    // ---- o^T += V^T P^T ----
    uint32_t w[4][L::V_BYTES / 4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint8_t* from = sv + ((u & 1) == 0 ? v_even : v_odd) + (u >> 1) * 8 * D;
      if constexpr (D == 128) {
        const uint4 v = *reinterpret_cast<const uint4*>(from);
        w[u][0] = v.x;
        w[u][1] = v.y;
        w[u][2] = v.z;
        w[u][3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(from);
        w[u][0] = v.x;
        w[u][1] = v.y;
      }
    }
    // What lies behind the sequence's end counts as zeros, and so does a page whose scale is zero or below the smallest that the
    // shift holds: its tokens count in the sum and add nothing.
    if ((ta + i) * SK_TILE + SK_TILE > len || vs_raw < V_SCALE_MIN) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool in = (ta + i) * SK_TILE + ((u & 1) == 0 ? tv0 : tv1) + (u >> 1) * 8 < len && !(vs_raw < V_SCALE_MIN);
#pragma unroll
        for (int j = 0; j < L::V_BYTES / 4; ++j) w[u][j] = in ? w[u][j] : 0u;
      }
    }
    if (!EVEN && edge && limit_min < len) spoil_seen<D, RT>(w, (ta + i) * SK_TILE, limit, part);
#pragma unroll
    for (int j = 0; j < L::V_BYTES / 4; ++j) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // channels 4 j + 2 half (rows g of the tile) and the next (rows 8 + g)
        uint32_t a0, a1, a2, a3;
        e4m3x4_f16x4(__byte_perm(w[0][j], w[1][j], half == 0 ? 0x5140 : 0x7362), a0, a1);
        e4m3x4_f16x4(__byte_perm(w[2][j], w[3][j], half == 0 ? 0x5140 : 0x7362), a2, a3);
#pragma unroll
        for (int n = 0; n < RT; ++n) mma_f16(part.o[n][j * 2 + half], a0, a1, a2, a3, pb[n][0], pb[n][1]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < RT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) part.l[n][e] *= SUM_UNIT;
  }
  return true;
}

// Row rr of the queries of KV head hkv that a warp has seen to its end: channels [D / 8 * g, ...) of it, by its lanes t = const.
template <int D, int RT>
__device__ __forceinline__ void store_row(const SdpaArgs& a, const Part<D, RT>& part, int n, int e, float sum, int b, int hkv,
                                          int rr, int g) {
  const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing visible: zeros
  __nv_bfloat16* out = a.o + (((int64_t)b * a.Sq + qi) * a.Hq + head) * D + g * (D / 8);
#pragma unroll
  for (int j = 0; j < D / 16; j += 4)
    *reinterpret_cast<uint4*>(out + 2 * j) =
        make_uint4(pack_bf16x2(part.o[n][j][e] * inv, part.o[n][j][2 + e] * inv), pack_bf16x2(part.o[n][j + 1][e] * inv, part.o[n][j + 1][2 + e] * inv),
                   pack_bf16x2(part.o[n][j + 2][e] * inv, part.o[n][j + 2][2 + e] * inv),
                   pack_bf16x2(part.o[n][j + 3][e] * inv, part.o[n][j + 3][2 + e] * inv));
}

template <int D, int RT, bool EVEN>
__global__ void __launch_bounds__(SK_THREADS, SkLayout<D, RT>::CTAS_PER_SM) sdpa_kv8_kernel(const __grid_constant__ CUtensorMap tma_k,
                                                                                          const __grid_constant__ CUtensorMap tma_v,
                                                                                          const SdpaArgs a) {
  using L = SkLayout<D, RT>;
  constexpr int STEPS = D / 16;
  constexpr int CH = D / 8;      // channels of o per lane and row
  constexpr int ROWS = L::ROWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t s_full[SK_WARPS][L::STAGES];
  __shared__ int s_abort;
  // the last piece of a warp's range, where it is not a whole row: its row (or -1), whether it begins / ends the row, the
  // row's last range
  __shared__ int s_row[SK_WARPS], s_edge[SK_WARPS], s_owner[SK_WARPS];
  __shared__ float s_m[SK_WARPS][ROWS], s_l[SK_WARPS][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int heads = a.Hkv * a.row_tiles;  // rows (of tiles) per sequence
  if (threadIdx.x == 0) {
    for (int i = 0; i < SK_WARPS * L::STAGES; ++i) mbar_init(&s_full[0][0] + i, 1);
    s_abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
  }
  __syncthreads();
  grid_dependency_wait();
  const WaitCtx wc{&s_abort, a.status, a.limit_ns};

  // ---- this warp's range of the list ----
  int64_t total = 0;
  for (int i = lane; i < a.B; i += 32) total += row_units(seq_tiles(seq_len(a, i)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= heads;
  const int64_t ranges = min((int64_t)gridDim.x * SK_WARPS, total);  // no more ranges than units: none is empty
  if ((int64_t)blockIdx.x * SK_WARPS >= ranges) return;
  const int64_t range = (int64_t)blockIdx.x * SK_WARPS + warp;  // neighbours in the list join in shared memory
  if (lane == 0) s_row[warp] = -1;
  // the position in the list: unit `off` of sequence b, `left` units to go (the host admits sizes for which these fit)
  int b = 0, off = 0, left = 0;
  if (range < ranges) {
    int64_t pos = range_start(range, total, ranges);
    left = (int)(range_start(range + 1, total, ranges) - pos);
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int64_t mine = b0 + lane < a.B ? (int64_t)row_units(seq_tiles(seq_len(a, b0 + lane))) * heads : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const unsigned past = __ballot_sync(0xffffffffu, pos < upto);
      if (past != 0) {
        const int src = __ffs(past) - 1;
        b = b0 + src;
        off = (int)(pos - __shfl_sync(0xffffffffu, upto - mine, src));
        break;
      }
      pos -= __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  uint8_t* ring = smem + warp * L::WARP_RING;
  RingAt at{0, 0, 0};
  bool alive = true;        // no wait has run out

  while (left > 0 && alive) {
    // ---- the next row and the part of it that is ours ----
    int len = seq_len(a, b);
    int tiles = seq_tiles(len);
    int units = row_units(tiles);
    while (off >= units * heads) {
      off -= units * heads;
      ++b;
      len = seq_len(a, b);
      tiles = seq_tiles(len);
      units = row_units(tiles);
    }
    const int hr = off / units, within = off - hr * units;  // the row's tiles begin ROW_COST units into it
    const int ta = max(within - ROW_COST, 0), tb = min(within + left - ROW_COST, tiles);
    const int step = min(left, units - within);
    off += step;
    left -= step;
    if (tb <= ta) continue;  // only what a row counts beside its tiles
    const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
    const int rows = min(ROWS, a.G * a.Sq - rt * ROWS);
    Part<D, RT> part;
    alive = row_part<D, RT, EVEN>(a, tma_k, tma_v, ring, s_full[warp], wc, at, b, hkv, rt, len, ta, tb, part);
    if (!alive) break;
    // ---- this range's part of the row: channels [CH g, CH (g + 1)) of rows 2 t and 2 t + 1 of each tile per lane ----
    const bool whole = ta == 0 && tb == tiles;
    const bool last = !whole && left == 0;  // may go on in the next warp's range: left in shared memory
    if (last) __syncwarp();                   // every lane is done with the ring
#pragma unroll
    for (int n = 0; n < RT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = part.l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int row = n * 8 + 2 * t + e;
        if (row >= rows) continue;
        if (whole) {
          store_row<D, RT>(a, part, n, e, sum, b, hkv, rt * ROWS + row, g);
        } else {
          // (the first part of a row ends its range and takes slot 1, any other begins it and takes slot 0)
          const int64_t place = range * 2 * a.row_cap + row;
          if (g == 0) (last ? s_m[warp][row] : a.ml[place].x) = part.m[n][e];
          if (g == 0) (last ? s_l[warp][row] : a.ml[place].y) = sum;
          float* out = (last ? reinterpret_cast<float*>(ring) + row * L::PIECE_PITCH : a.part + place * D) + g * CH;
#pragma unroll
          for (int j = 0; j < STEPS; j += 2)
            *reinterpret_cast<float4*>(out + 2 * j) = make_float4(part.o[n][j][e], part.o[n][j][2 + e], part.o[n][j + 1][e], part.o[n][j + 1][2 + e]);
        }
      }
    }
    if (lane == 0) {
      const int row = b * heads + hr;
      if (whole) a.info[row] = make_int2((int)range, (int)range);
      if (last) {
        s_row[warp] = row;
        s_edge[warp] = (ta == 0 ? 1 : 0) | (tb == tiles ? 2 : 0);
        // (a row that begins here and is not whole goes on behind this range's end: its last tile is tiles - tb further)
        if (ta == 0) s_owner[warp] = (int)range_owner(range_start(range + 1, total, ranges) - 1 + tiles - tb, total, ranges);
      }
    }
    __syncwarp();
  }

  // Not earlier: blocks of the next kernel that wait beside this one's long-lived warps cost 19 us of 121 (64 sequences of up
  // to 8192 tokens); and not at all in the join, whose dependents are such a kernel.
  grid_launch_dependents();
  // ---- the last pieces of the CTA's warps: neighbours that belong to one row become one piece ----
  __syncthreads();
  if (s_abort) {  // a wait ran out (recorded): copies may be in flight, and pieces are missing
    abort_drain();
    return;
  }
  for (int w0 = 0; w0 < SK_WARPS; ++w0) {
    const int row_id = s_row[w0];
    if (row_id < 0 || (w0 > 0 && s_row[w0 - 1] == row_id)) continue;
    int w1 = w0 + 1;
    while (w1 < SK_WARPS && s_row[w1] == row_id) ++w1;
    const int seq = row_id / heads, hr = row_id - seq * heads;
    const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
    const int rows = min(ROWS, a.G * a.Sq - rt * ROWS);
    const bool begins = (s_edge[w0] & 1) != 0, whole = begins && (s_edge[w1 - 1] & 2) != 0;
    const int64_t first = (int64_t)blockIdx.x * SK_WARPS + w0;  // range of the run's first piece
    constexpr int TPR = SK_THREADS / ROWS, N = D / TPR;         // threads per row, channels per thread
    const int row = threadIdx.x / TPR, col = (threadIdx.x % TPR) * N;
    if (row < rows) {
      float top = -INFINITY;
      for (int w = w0; w < w1; ++w) top = fmaxf(top, s_m[w][row]);
      float sum = 0.f, acc[N];
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = 0.f;
      for (int w = w0; w < w1; ++w) {
        // a piece without a visible token has -inf here, zeros (or, through a NaN, NaN) in its sums
        const float f = s_m[w][row] == -INFINITY ? 1.f : ex2(s_m[w][row] - top);
        sum += s_m[w][row] == -INFINITY ? s_l[w][row] : decay(s_l[w][row], s_m[w][row] - top);
        const float* from = reinterpret_cast<const float*>(smem + w * L::WARP_RING) + row * L::PIECE_PITCH + col;
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(from + j);
          acc[j] = fmaf(v.x, f, acc[j]);
          acc[j + 1] = fmaf(v.y, f, acc[j + 1]);
          acc[j + 2] = fmaf(v.z, f, acc[j + 2]);
          acc[j + 3] = fmaf(v.w, f, acc[j + 3]);
        }
      }
      if (whole) {
        const int rr = rt * ROWS + row;
        const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        __nv_bfloat16* out = a.o + (((int64_t)seq * a.Sq + qi) * a.Hq + head) * D + col;
#pragma unroll
        for (int j = 0; j < N; j += 4)
          *reinterpret_cast<uint2*>(out + j) =
              make_uint2(pack_bf16x2(acc[j] * inv, acc[j + 1] * inv), pack_bf16x2(acc[j + 2] * inv, acc[j + 3] * inv));
      } else {
        const int64_t at = (first * 2 + (begins ? 1 : 0)) * a.row_cap + row;
        if (col == 0) {
          a.ml[at] = make_float2(top, sum);
          // the others' places in the row's list stay empty
          for (int w = w0 + 1; w < w1; ++w) a.ml[(first + w - w0) * 2 * a.row_cap + row] = make_float2(-INFINITY, 0.f);
        }
        float* out = a.part + at * D + col;
#pragma unroll
        for (int j = 0; j < N; j += 4)
          *reinterpret_cast<float4*>(out + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
    }
    if (begins && threadIdx.x == 0) a.info[row_id] = make_int2((int)first, whole ? (int)first : s_owner[w0]);
  }
}

// A warp's piece of a row tile: the outputs over its ring, the maxima and sums to m and l.
template <int D, int RT>
__device__ __forceinline__ void leave_piece(const Part<D, RT>& part, uint8_t* ring, float* m, float* l) {
  using L = SkLayout<D, RT>;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  __syncwarp();  // every lane is done with the ring
#pragma unroll
  for (int n = 0; n < RT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = part.l[n][e];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int row = n * 8 + 2 * t + e;
      if (g == 0) {
        m[row] = part.m[n][e];
        l[row] = sum;
      }
      float* out = reinterpret_cast<float*>(ring) + row * L::PIECE_PITCH + g * (D / 8);
#pragma unroll
      for (int j = 0; j < D / 16; j += 2)
        *reinterpret_cast<float4*>(out + 2 * j) =
            make_float4(part.o[n][j][e], part.o[n][j][2 + e], part.o[n][j + 1][e], part.o[n][j + 1][2 + e]);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_size_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
template <int E>
__device__ __forceinline__ void ld_cluster_vec(uint32_t addr, float* v) {
  if constexpr (E == 4)
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
}

// The sequence that comes at place `rank` when the longest come first: by buckets of a quarter octave of their tiles, those of
// a bucket in their own order. All threads of the block, B <= RANKED; the length comes back too.
constexpr int RANKED = 256;
__device__ __forceinline__ int sequence_of_rank(const SdpaArgs& a, int rank, int& len) {
  __shared__ int s_count[SK_THREADS], s_warp[SK_WARPS], s_pick[2];
  __shared__ int s_len[RANKED];
  __shared__ uint8_t s_bucket[RANKED];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  s_count[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int b = tid; b < RANKED; b += SK_THREADS) {
    int bucket = 0xff;  // none's
    if (b < a.B) {
      const int n = seq_len(a, b);
      const uint32_t x = (uint32_t)seq_tiles(n) << 2;  // tiles are below 2^28
      const int e = 31 - __clz(x | 4u);                // their exponent + 2
      bucket = x == 0 ? SK_THREADS - 1 : SK_THREADS - 2 - (((e - 2) << 2) + (int)((x >> (e - 2)) & 3u));  // 0: the longest
      s_len[b] = n;
      atomicAdd(&s_count[bucket], 1);
    }
    s_bucket[b] = (uint8_t)bucket;
  }
  __syncthreads();
  const int mine = s_count[tid];
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) s_warp[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SK_WARPS - 1; ++w) upto += w < warp ? s_warp[w] : 0;
  if (rank < upto && rank >= upto - mine) {
    s_pick[0] = tid;
    s_pick[1] = rank - (upto - mine);
  }
  __syncthreads();
  const int bucket = s_pick[0];
  int left = s_pick[1];
#pragma unroll
  for (int b0 = 0; b0 < RANKED; b0 += 32) {
    const bool hit = s_bucket[b0 + lane] == bucket;
    const unsigned in = __ballot_sync(0xffffffffu, hit);
    const int n = __popc(in);
    if (left < n) {
      const unsigned here = __ballot_sync(0xffffffffu, hit && __popc(in & ((1u << lane) - 1)) == left);
      const int b = b0 + __ffs(here) - 1;
      len = s_len[b];
      return b;
    }
    left -= n;
  }
  return 0;  // not reached: rank < B
}

// Many rows, or short ones (split_of): a cluster of 1, 2, 4 or 8 CTAs per row tile deals its tiles to its warps, whose
// pieces meet in distributed shared memory. No list to cut, no workspace, no second kernel: what is left of a call is one
// launch and one row's latency.
template <int D, int RT, bool EVEN>
__global__ void __launch_bounds__(SK_THREADS, SkLayout<D, RT>::CTAS_PER_SM)
sdpa_kv8_rows_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const SdpaArgs a) {
  using L = SkLayout<D, RT>;
  constexpr int ROWS = L::ROWS, E = D / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t s_full[SK_WARPS][L::STAGES];
  __shared__ int s_abort;
  __shared__ float s_m[SK_WARPS][ROWS], s_l[SK_WARPS][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = (int)cluster_size_x(), rank = (int)cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < SK_WARPS * L::STAGES; ++i) mbar_init(&s_full[0][0] + i, 1);
    s_abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
  }
  __syncthreads();
  const int heads = a.Hkv * a.row_tiles;
  const int row_id = blockIdx.x / split;
  int b = row_id / heads;
  const int hr = row_id - b * heads;
  const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
  const int rows = min(ROWS, a.G * a.Sq - rt * ROWS);
  const int pieces = split * SK_WARPS, piece = rank * SK_WARPS + warp;
  grid_dependency_wait();
  const WaitCtx wc{&s_abort, a.status, a.limit_ns};
  int len;
  if (a.ranked)
    b = sequence_of_rank(a, b, len);
  else
    len = seq_len(a, b);
  const int tiles = seq_tiles(len);
  const int ta = (int)((int64_t)tiles * piece / pieces), tb = (int)((int64_t)tiles * (piece + 1) / pieces);
  if (lane < ROWS) {
    s_m[warp][lane] = -INFINITY;
    s_l[warp][lane] = 0.f;
  }
  __syncwarp();
  if (tb > ta) {
    uint8_t* ring = smem + warp * L::WARP_RING;
    RingAt at{0, 0, 0};
    Part<D, RT> part;
    if (row_part<D, RT, EVEN>(a, tma_k, tma_v, ring, s_full[warp], wc, at, b, hkv, rt, len, ta, tb, part))
      leave_piece<D, RT>(part, ring, s_m[warp], s_l[warp]);
  }
  grid_launch_dependents();
  __syncthreads();
  if (s_abort) abort_drain();
  if (split > 1) cluster_sync_all();  // (reached by every thread of every CTA, whatever happened above)
  // a warp joins a row: lane i looks after piece i, then the lanes share the channels
  for (int row = piece; row < rows; row += pieces) {
    float m = -INFINITY, l = 0.f;
    if (lane < pieces) {
      m = ld_cluster(mapa_u32(smem_u32(&s_m[lane & (SK_WARPS - 1)][row]), (uint32_t)(lane / SK_WARPS)));
      l = ld_cluster(mapa_u32(smem_u32(&s_l[lane & (SK_WARPS - 1)][row]), (uint32_t)(lane / SK_WARPS)));
    }
    const unsigned holds = __ballot_sync(0xffffffffu, m != -INFINITY || l != 0.f);  // (a NaN sum counts)
    const float top = warp_max(m);
    const float f = m == -INFINITY ? 1.f : ex2(m - top);
    const float sum = warp_sum(m == -INFINITY ? l : decay(l, m - top));
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 8
    for (int i = 0; i < pieces; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      if ((holds >> i) & 1u) {
        const uint32_t from = smem_u32(smem) + (uint32_t)((i & (SK_WARPS - 1)) * L::WARP_RING + (row * L::PIECE_PITCH + lane * E) * 4);
        float v[E];
        ld_cluster_vec<E>(mapa_u32(from, (uint32_t)(i / SK_WARPS)), v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(v[e], fi, acc[e]);
      }
    }
    const int rr = rt * ROWS + row;
    const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing visible: zeros
    __nv_bfloat16* out = a.o + (((int64_t)b * a.Sq + qi) * a.Hq + head) * D + lane * E;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(out) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  }
  if (split > 1) cluster_sync_relaxed();  // no CTA leaves while another reads its shared memory
}

// Many rows of few tiles (short_rows): a warp takes a whole row tile, and nothing is joined.
template <int D, int RT, bool EVEN>
__global__ void __launch_bounds__(SK_THREADS, SkLayout<D, RT>::CTAS_PER_SM)
sdpa_kv8_short_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const SdpaArgs a) {
  using L = SkLayout<D, RT>;
  constexpr int ROWS = L::ROWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t s_full[SK_WARPS][L::STAGES];
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int i = 0; i < L::STAGES; ++i) mbar_init(&s_full[warp][i], 1);
    if (warp == 0) {
      s_abort = 0;
      tma_prefetch_desc(&tma_k);
      tma_prefetch_desc(&tma_v);
    }
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_wait();
  const WaitCtx wc{&s_abort, a.status, a.limit_ns};
  const int heads = a.Hkv * a.row_tiles;
  const int row_id = blockIdx.x * SK_WARPS + warp;
  if (row_id < a.B * heads) {
    const int b = row_id / heads, hr = row_id - b * heads;
    const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
    const int rows = min(ROWS, a.G * a.Sq - rt * ROWS);
    const int len = seq_len(a, b), tiles = seq_tiles(len);
    RingAt at{0, 0, 0};
    Part<D, RT> part;
    if (row_part<D, RT, EVEN>(a, tma_k, tma_v, smem + warp * L::WARP_RING, s_full[warp], wc, at, b, hkv, rt, len, 0, tiles, part)) {
#pragma unroll
      for (int n = 0; n < RT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = part.l[n][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int row = n * 8 + 2 * t + e;
          if (row >= rows) continue;
          store_row<D, RT>(a, part, n, e, sum, b, hkv, rt * ROWS + row, g);
        }
      }
    }
  }
  grid_launch_dependents();
  __syncthreads();
  if (s_abort) abort_drain();
}

// Few rows of a certain length (wide_split_of): the same with one CTA of as many warps as an SM holds, so that a row gets
// four times (16 rows: twice) the warps out of a cluster. A CTA's pieces meet in its own shared memory before the cluster's
// do.
template <int D, int RT, bool EVEN>
__global__ void __launch_bounds__(WideLayout<D, RT>::THREADS, 1)
sdpa_kv8_wide_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const SdpaArgs a) {
  using L = SkLayout<D, RT>;
  constexpr int ROWS = L::ROWS, E = D / 32, WARPS = WideLayout<D, RT>::WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t s_full[WARPS][L::STAGES];
  __shared__ int s_abort;
  __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS];
  __shared__ float s_cm[ROWS], s_cl[ROWS];                 // the CTA's piece
  __shared__ __align__(16) float s_o[ROWS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = (int)cluster_size_x(), rank = (int)cluster_ctarank();
  if (lane == 0) {
    for (int i = 0; i < L::STAGES; ++i) mbar_init(&s_full[warp][i], 1);
    if (warp == 0) {
      s_abort = 0;
      tma_prefetch_desc(&tma_k);
      tma_prefetch_desc(&tma_v);
    }
    fence_barrier_init();
  }
  __syncthreads();
  const int heads = a.Hkv * a.row_tiles;
  const int row_id = blockIdx.x / split;
  const int b = row_id / heads, hr = row_id - b * heads;
  const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
  const int rows = min(ROWS, a.G * a.Sq - rt * ROWS);
  const int pieces = split * WARPS, piece = rank * WARPS + warp;
  grid_dependency_wait();
  const WaitCtx wc{&s_abort, a.status, a.limit_ns};
  const int len = seq_len(a, b), tiles = seq_tiles(len);
  const int ta = (int)((int64_t)tiles * piece / pieces), tb = (int)((int64_t)tiles * (piece + 1) / pieces);
  if (lane < ROWS) {
    s_m[warp][lane] = -INFINITY;
    s_l[warp][lane] = 0.f;
  }
  __syncwarp();
  if (tb > ta) {
    uint8_t* ring = smem + warp * L::WARP_RING;
    RingAt at{0, 0, 0};
    Part<D, RT> part;
    if (row_part<D, RT, EVEN>(a, tma_k, tma_v, ring, s_full[warp], wc, at, b, hkv, rt, len, ta, tb, part))
      leave_piece<D, RT>(part, ring, s_m[warp], s_l[warp]);
  }
  grid_launch_dependents();
  __syncthreads();
  if (s_abort) abort_drain();
  const auto store = [&](int row, const float* acc, float sum) {
    const int rr = rt * ROWS + row;
    const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing visible: zeros
    __nv_bfloat16* out = a.o + (((int64_t)b * a.Sq + qi) * a.Hq + head) * D + lane * E;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(out) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  };
  // a warp joins a row: lane i looks after piece i, then the lanes share the channels
  for (int row = warp; row < rows; row += WARPS) {
    const float m = lane < WARPS ? s_m[lane][row] : -INFINITY, l = lane < WARPS ? s_l[lane][row] : 0.f;
    const unsigned holds = __ballot_sync(0xffffffffu, m != -INFINITY || l != 0.f);  // (a NaN sum counts)
    const float top = warp_max(m);
    const float f = m == -INFINITY ? 1.f : ex2(m - top);
    const float sum = warp_sum(m == -INFINITY ? l : decay(l, m - top));
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      if ((holds >> i) & 1u) {
        const float* from = reinterpret_cast<const float*>(smem + i * L::WARP_RING) + row * L::PIECE_PITCH + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(from[e], fi, acc[e]);
      }
    }
    if (split == 1) {
      store(row, acc, sum);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) s_o[row][lane * E + e] = acc[e];
      if (lane == 0) {
        s_cm[row] = top;
        s_cl[row] = sum;
      }
    }
  }
  if (split == 1) return;  // (uniform over the grid)
  cluster_sync_all();      // (reached by every thread of every CTA, whatever happened above)
  for (int row = rank + split * warp; row < rows; row += split * WARPS) {
    float m = -INFINITY, l = 0.f;
    if (lane < split) {
      m = ld_cluster(mapa_u32(smem_u32(&s_cm[row]), (uint32_t)lane));
      l = ld_cluster(mapa_u32(smem_u32(&s_cl[row]), (uint32_t)lane));
    }
    const float top = warp_max(m);
    const float f = m == -INFINITY ? (l != 0.f ? 1.f : 0.f) : ex2(m - top);
    const float sum = warp_sum(m == -INFINITY ? l : decay(l, m - top));
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      if (i < split) {
        float v[E];
        ld_cluster_vec<E>(mapa_u32(smem_u32(&s_o[row][lane * E]), (uint32_t)i), v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(v[e], fi, acc[e]);
      }
    }
    store(row, acc, sum);
  }
  cluster_sync_relaxed();  // no CTA leaves while another reads its shared memory
}

// Joins the pieces of every row that was cut: block (row of tiles, row of the tile). The places of a row's pieces are
// consecutive ranges; those that were joined within a CTA are empty (maximum -inf, sum 0) but for the first.
template <int D, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) sdpa_kv8_join_kernel(const SdpaArgs a) {
  constexpr int E = D / 32;  // channels per lane
  __shared__ int s_at[WARPS * 32];    // places that hold something, and their factors
  __shared__ float s_f[WARPS * 32];
  __shared__ int s_n[WARPS];
  __shared__ float s_m[WARPS], s_l[WARPS];
  __shared__ float s_o[WARPS][D];
  grid_dependency_wait();
  const int heads = a.Hkv * a.row_tiles;
  const int b = blockIdx.x / heads, hr = blockIdx.x - b * heads;
  const int hkv = hr / a.row_tiles, rt = hr - hkv * a.row_tiles;
  const int rr = rt * a.tile_rows + blockIdx.y;
  const int2 span = a.info[blockIdx.x];  // (of an empty sequence: not written, not used)
  const int len = seq_len(a, b);
  if (rr >= a.G * a.Sq) return;
  const int qi = rr / a.G, head = hkv * a.G + rr - qi * a.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __nv_bfloat16* out = a.o + (((int64_t)b * a.Sq + qi) * a.Hq + head) * D;
  if (len == 0) {  // no tile, so no warp wrote this row
    if (threadIdx.x < D / 8) reinterpret_cast<uint4*>(out)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    return;
  }
  // (the bounds hold unless the first kernel gave up on a wait and left places unwritten)
  if (span.x == span.y || span.x < 0 || span.y < span.x || span.y >= a.max_ranges) return;
  float m = -INFINITY, l = 0.f, o[E];  // m is the same in all threads, l and o are this warp's part
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int c0 = span.x; c0 <= span.y; c0 += WARPS * 32) {
    // ---- a place per thread: the block's maximum, and a list of those that hold something ----
    const int c = c0 + (int)threadIdx.x;
    int at = 0;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (c <= span.y) {
      at = c * 2 + (c == span.x ? 1 : 0);
      ml = a.ml[(int64_t)at * a.row_cap + blockIdx.y];
    }
    const bool holds = ml.x != -INFINITY || ml.y != 0.f;  // (a NaN sum counts)
    const unsigned mask = __ballot_sync(0xffffffffu, holds);
    const float wm = warp_max(ml.x);
    if (lane == 0) {
      s_n[warp] = __popc(mask);
      s_m[warp] = wm;
    }
    __syncthreads();
    float top = m;
    int before = 0, n = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      top = fmaxf(top, s_m[w]);
      before += w < warp ? s_n[w] : 0;
      n += s_n[w];
    }
    if (holds) {
      const int i = before + __popc(mask & ((1u << lane) - 1));
      s_at[i] = at;
      s_f[i] = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);
    }
    const float keep = m == -INFINITY ? 1.f : ex2(m - top);
    // each thread adds its own place's sum; the warps share the outputs out
    l = (m == -INFINITY ? l : decay(l, m - top)) + (holds ? (ml.x == -INFINITY ? ml.y : decay(ml.y, ml.x - top)) : 0.f);
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= keep;
    __syncthreads();
#pragma unroll 8
    for (int i = warp; i < n; i += WARPS) {
      const float f = s_f[i];
      const float* p = a.part + ((int64_t)s_at[i] * a.row_cap + blockIdx.y) * D + lane * E;
      float v[E];
      if constexpr (E == 4) {
        const float4 u = *reinterpret_cast<const float4*>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
      } else {
        const float2 u = *reinterpret_cast<const float2*>(p);
        v[0] = u.x; v[1] = u.y;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], f, o[e]);
    }
    __syncthreads();
  }
  l = warp_sum(l);
  if (lane == 0) s_l[warp] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      sum += s_l[w];
      x += s_o[w][threadIdx.x * 2];
      y += s_o[w][threadIdx.x * 2 + 1];
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    reinterpret_cast<uint32_t*>(out)[threadIdx.x] = pack_bf16x2(x * inv, y * inv);
  }
}

int64_t align16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// Up to eight rows that share a KV head go as one tile of 8; more as tiles of 16, each reading the cache once.
int tile_rows_of(int64_t rows) { return rows <= 8 ? 8 : 16; }

// Every product of the sizes that the kernels form in 32 bits fits.
bool sizes_ok(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv) {
  const int64_t limit = 0x7fffffff;
  if (B <= 0 || Sq <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return false;
  if (B > limit || Sq > limit || Hq > limit || Sq > limit / (Hq / Hkv)) return false;
  const int64_t rows = Hq / Hkv * Sq, row_tiles = (rows + tile_rows_of(rows) - 1) / tile_rows_of(rows);
  return Hkv <= limit / row_tiles && B <= limit / (Hkv * row_tiles);
}

enum class Way { LIST, ROWS, WIDE, SHORT };

struct SkPlan {
  int row_tiles, tile_rows, row_cap;
  Way way;
  int split;   // CTAs per row tile of the wide or the rows kernel
  int ranked;  // rows kernel: the longest sequences first
  int64_t ctas, info_bytes, ml_bytes, part_bytes;
};

// CTAs per row tile for the rows kernel, or 0 where the list kernel is to run. The host knows the longest a sequence can be
// (max_tokens), not the lengths. The rows kernel has no list to cut and nothing to join, and wins wherever its CTAs finish
// about together (8 KV heads, 64 sequences of 128 tokens: 6.9 us against 12.9; of 1024: 26.2 / 35.4; of 4096: 88.2 / 98.3; of
// 0..8192: 91.6 / 102.5; 128 of 0..4096: 87.0 / 108.9); a sequence much longer than the others it drags through a few
// warps, 0.7 us a tile at least. So: as many CTAs per row as fill the machine, or twice
// that, such that a row's warps take `limit` tiles each at most of the longest possible sequence:
//   32 (16 rows to a tile, where a tile takes longer: 24 if twice as many CTAs allow it; 17 x 4 tokens of up to 4097: 23.7 us
//   against 28.8), or as many as the machine reads in 0.75 us of the time that half of all the tables could hold takes, to 64;
//   10 where even 8 CTAs per row leave half of the machine idle (one sequence of 8192: 15.1 us against 12.8, of 16384: 24.6 /
//   15.9; what is shorter, but not short, goes to the wide kernel).
// More CTAs than that cost their start (about 6 us of a slot each) and are taken where that is small beside the reading (64 of
// 0..16384: 163 us in fours, 180 as a list).
int split_of(int64_t rows, int64_t max_tokens, int64_t D, int64_t slots, bool small_tile) {
  int fill = 1;
  while (fill < 8 && rows * fill * 2 <= slots) fill *= 2;
  const double all = (double)rows * (double)max_tokens * (double)D / 6.2e6;  // us: half of 2 D bytes a token and row
  const int64_t tiles = (max_tokens + SK_TILE - 1) / SK_TILE;
  const bool idle = rows * 16 <= slots;
  const double lo = idle ? 10. : small_tile ? 32. : 24.;
  const double limit = idle || all * 0.75 < lo ? lo : all * 0.75 < 64. ? all * 0.75 : 64.;
  int split = 0;
  for (int n = fill; n <= 8; n *= 2) {
    if (n > 2 * fill && (double)(rows * n) * 24. > all * (double)slots) break;
    const double each = (double)tiles / (n * SK_WARPS);
    if (each <= limit || (!idle && each <= 32.)) split = n;
    if (each <= limit) break;
  }
  while (split > 1 && tiles < split * 8) split /= 2;  // no CTA with less than two tiles a warp
  return rows * split <= 0x7fffffff ? split : 0;
}

// Whether a warp takes a whole row tile: where rows are so many and so short that the CTAs' starts and joins are most of a call,
// and a warp's serial tiles (0.6 us each) are not (8 KV heads; 64 sequences of 64 tokens: 5.2 us against 5.6, but of 128: 7.7 / 7.0;
// 128 of 128: 10.0 / 14.1; 256 of 32: 6.4 / 16.3, of 256: 26.2 / 32.6; 1024 of 128: 48.3 / 82.8). Not where the lengths may
// differ by more tiles than that (128 of 1..512: 25.7 / 19.9).
bool short_rows(int64_t rows, int64_t max_tokens, int64_t slots) {
  const int64_t tiles = (max_tokens + SK_TILE - 1) / SK_TILE;
  return tiles <= 32 && tiles * slots <= rows * 8;
}

// CTAs per row tile for the wide kernel, or 0: as many of 8, 4, 2 and 1 as fit an SM each (clusters of 8 fill no more than
// about half of the SMs) and have 8 tiles. It wins where a row gets more warps out of it than out of the rows kernel and
// sequences may be long enough to use them (8 KV heads; one sequence of 1500 tokens: 6.4 us against 7.5, of 4096: 7.6 / 10.5, of
// 8192: 9.5 / 12.8 in a list; four of 4096: 11.0 / 13.4; 16 of 512: 7.0 / 8.4, of 4096: 25.0 / 27.5; but one of 128: 5.0 / 4.5), up
// to 16 tiles a warp: beyond that, lengths that differ cost more than the warps gain (16 of 0..8192: 37.6 / 34.7). Where it
// leaves half of the machine idle, up to 10 (one of 16384: 14.1 / 16.0 in a list, of 32768: 22.6 / 21.1).
int wide_split_of(int64_t rows, int64_t max_tokens, int64_t sm_count, int64_t warps) {
  const int64_t tiles = (max_tokens + SK_TILE - 1) / SK_TILE, fit = sm_count - sm_count / 8;
  if (tiles < 32 || rows > fit) return 0;
  int split = rows * 16 <= sm_count ? 8 : rows * 4 <= fit ? 4 : rows * 2 <= fit ? 2 : 1;
  while (split > 1 && tiles < split * 8) split /= 2;
  return tiles <= (rows * split * 2 > sm_count ? 16 : 10) * split * warps ? split : 0;
}

// The grid never has more warps than the longest possible list has units.
SkPlan plan_of(int sm_count, int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t max_tokens, int64_t D) {
  SkPlan p;
  p.tile_rows = tile_rows_of(Hq / Hkv * Sq);
  p.row_tiles = (int)((Hq / Hkv * Sq + p.tile_rows - 1) / p.tile_rows);
  p.row_cap = Hq / Hkv * Sq < p.tile_rows ? (int)(Hq / Hkv * Sq) : p.tile_rows;
  const int64_t units = (max_tokens + SK_TILE - 1) / SK_TILE + ROW_COST;  // below 2^28
  const int64_t rows = B * Hkv * p.row_tiles;                              // below 2^31
  const int64_t slots = (int64_t)sm_count * (p.tile_rows == 8 ? 4 : D == 128 ? SkLayout<128, 2>::CTAS_PER_SM : SkLayout<64, 2>::CTAS_PER_SM);
  p.split = 0;
  p.way = Way::LIST;
  if (short_rows(rows, max_tokens, slots)) {
    p.way = Way::SHORT;
  } else if ((p.split = wide_split_of(rows, max_tokens, sm_count, p.tile_rows == 8 ? WideLayout<128, 1>::WARPS : WideLayout<128, 2>::WARPS)) > 0) {
    p.way = Way::WIDE;
  } else if ((p.split = split_of(rows, max_tokens, D, slots, p.tile_rows == 8)) > 0) {
    p.way = Way::ROWS;
  }
  // Longest first pays where a CTA may have more than a few tiles a warp and several CTAs share an SM or wait for one (64
  // sequences of 0..8192 tokens in pairs: 91.6 us against 109.9; 128 of 0..4096: 87.0 / 108.4) and costs 0.8 us a CTA (256
  // sequences of 128: 28.5 us against 25.6).
  p.ranked = p.way == Way::ROWS && B > 1 && B <= RANKED && rows * p.split > sm_count && units > (int64_t)p.split * SK_WARPS * 8 ? 1 : 0;
  p.ctas = slots;
  if ((rows * units + SK_WARPS - 1) / SK_WARPS < p.ctas) p.ctas = (rows * units + SK_WARPS - 1) / SK_WARPS;
  if (p.ctas < 1) p.ctas = 1;
  p.info_bytes = align16(rows * (int64_t)sizeof(int2));
  p.ml_bytes = align16(p.ctas * SK_WARPS * 2 * p.row_cap * (int64_t)sizeof(float2));
  p.part_bytes = p.ctas * SK_WARPS * 2 * p.row_cap * D * (int64_t)sizeof(float);
  if (p.way != Way::LIST) p.info_bytes = p.ml_bytes = p.part_bytes = 0;  // no workspace
  return p;
}

template <int D, int RT, bool EVEN>
int launch_sdpa(emk_handle_t h, const SdpaArgs& a, const SkPlan& p, cudaStream_t s) {
  CUtensorMap tk, tv;
  const uint64_t rows = (uint64_t)a.num_pages * a.Hkv << a.page_shift;
  constexpr CUtensorMapSwizzle SWIZZLE = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  int rc = emk_make_tmap_2d(h, &tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k, D, rows, D, D, SK_TILE, SWIZZLE);
  if (rc != EMK_OK) return rc;
  rc = emk_make_tmap_2d(h, &tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.v, D, rows, D, D, SK_TILE, SWIZZLE);
  if (rc != EMK_OK) return rc;
  static emk_device_once once;
  {
    std::lock_guard<std::mutex> lk(once.mu);
    if (!once.done[h->device]) {
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(sdpa_kv8_kernel<D, RT, EVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SkLayout<D, RT>::SMEM));
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(sdpa_kv8_rows_kernel<D, RT, EVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SkLayout<D, RT>::SMEM));
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(sdpa_kv8_short_kernel<D, RT, EVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SkLayout<D, RT>::SMEM));
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(sdpa_kv8_wide_kernel<D, RT, EVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize, WideLayout<D, RT>::SMEM));
      once.done[h->device] = true;
    }
  }
  if (p.way == Way::SHORT) {
    const unsigned ctas = (unsigned)(((int64_t)a.B * a.Hkv * a.row_tiles + SK_WARPS - 1) / SK_WARPS);
    EMK_CUDA_TRY(h, launch_after_prologue(sdpa_kv8_short_kernel<D, RT, EVEN>, ctas, SK_THREADS, SkLayout<D, RT>::SMEM, s,
                                          h->overlap_launch != 0, tk, tv, a));
    EMK_LAUNCH_CHECK(h);
    return EMK_OK;
  }
  if (p.way != Way::LIST) {
    const bool wide = p.way == Way::WIDE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.row_tiles * p.split), 1, 1);
    cfg.blockDim = dim3(wide ? WideLayout<D, RT>::THREADS : SK_THREADS, 1, 1);
    cfg.dynamicSmemBytes = wide ? WideLayout<D, RT>::SMEM : SkLayout<D, RT>::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = h->overlap_launch != 0 ? 2 : 1;
    EMK_CUDA_TRY(h, cudaLaunchKernelEx(&cfg, wide ? sdpa_kv8_wide_kernel<D, RT, EVEN> : sdpa_kv8_rows_kernel<D, RT, EVEN>, tk, tv, a));
    EMK_LAUNCH_CHECK(h);
    return EMK_OK;
  }
  EMK_CUDA_TRY(h, launch_after_prologue(sdpa_kv8_kernel<D, RT, EVEN>, (unsigned)p.ctas, SK_THREADS, SkLayout<D, RT>::SMEM, s,
                                        h->overlap_launch != 0, tk, tv, a));
  EMK_LAUNCH_CHECK(h);
  // Few rows: a row may be cut into hundreds of pieces, and sixteen warps share them; many rows: a few pieces each.
  const int64_t blocks = (int64_t)a.B * a.Hkv * a.row_tiles * a.row_cap;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.row_tiles), (unsigned)a.row_cap, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = h->overlap_launch != 0 ? 1 : 0;
  if (blocks <= (int64_t)h->sm_count * 4) {
    cfg.blockDim = dim3(16 * 32, 1, 1);
    EMK_CUDA_TRY(h, cudaLaunchKernelEx(&cfg, sdpa_kv8_join_kernel<D, 16>, a));
  } else {
    cfg.blockDim = dim3(4 * 32, 1, 1);
    EMK_CUDA_TRY(h, cudaLaunchKernelEx(&cfg, sdpa_kv8_join_kernel<D, 4>, a));
  }
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
  if (!h || !q || !k_codes || !v_codes || !k_scale || !v_scale || !page_table || !seq_lens || !o) return EMK_ERR_ARG;
  if ((D != 64 && D != 128) || !kv8_page_ok(page)) {
    EMK_SET_ERR(h, "emk_sdpa_kv8: head dimension 64 or 128 and a page of 16, 32, 64, 128 or 256 tokens; got D=%lld page=%lld",
                (long long)D, (long long)page);
    return EMK_ERR_SHAPE;
  }
  if (B <= 0 || Sq <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_pages <= 0 || num_pages <= 0 ||
      num_pages > 0x7fffffff || max_pages > 0x7fffffff / page || ld_q / D < Hq)
    return EMK_ERR_SHAPE;
  if (num_pages > 0x7fffffff / page / Hkv || !sizes_ok(B, Sq, Hq, Hkv)) {
    EMK_SET_ERR(h, "emk_sdpa_kv8: more than 2^31 - 1 rows in the cache or tiles of query rows");
    return EMK_ERR_LIMIT;
  }
  if (((uintptr_t)q & 15u) != 0 || (ld_q & 7) != 0 || (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)o) & 15u) != 0 ||
      (((uintptr_t)k_scale | (uintptr_t)v_scale | (uintptr_t)page_table | (uintptr_t)seq_lens) & 3u) != 0 ||
      ((uintptr_t)workspace & 15u) != 0)
    return EMK_ERR_ALIGN;
  const SkPlan p = plan_of(h->sm_count, B, Sq, Hq, Hkv, max_pages * page, D);
  const int64_t units = max_pages * page / SK_TILE + 1 + ROW_COST;
  if (Hkv * p.row_tiles > 0x7fffffff / units || B * Hkv * p.row_tiles * units / (p.ctas * SK_WARPS) > 0x7ffffffe) {
    EMK_SET_ERR(h, "emk_sdpa_kv8: %lld tokens a sequence are too many for the number of sequences and heads",
                (long long)(max_pages * page));
    return EMK_ERR_LIMIT;
  }
  if (workspace == nullptr && p.way == Way::LIST) return EMK_ERR_ARG;
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
  a.tile_rows = p.tile_rows;
  a.row_cap = p.row_cap;
  a.page_shift = __builtin_ctzll((unsigned long long)page);
  a.max_pages = (int)max_pages;
  a.num_pages = (int)num_pages;
  a.scale_log2 = scale * LOG2E;
  uint8_t* ws = (uint8_t*)workspace;
  a.info = (int2*)ws;
  a.ml = (float2*)(ws + p.info_bytes);
  a.part = (float*)(ws + p.info_bytes + p.ml_bytes);
  a.max_ranges = (int)(p.ctas * SK_WARPS);
  a.ranked = p.ranked;
  a.status = h->status_dev;
  a.limit_ns = h->wait_limit_ns;
  cudaStream_t s = (cudaStream_t)stream;
  if (p.tile_rows == 16) return D == 128 ? launch_sdpa<128, 2, false>(h, a, p, s) : launch_sdpa<64, 2, false>(h, a, p, s);
  if (Sq == 1) return D == 128 ? launch_sdpa<128, 1, true>(h, a, p, s) : launch_sdpa<64, 1, true>(h, a, p, s);
  return D == 128 ? launch_sdpa<128, 1, false>(h, a, p, s) : launch_sdpa<64, 1, false>(h, a, p, s);
}
