// e4m3 x e4m3 GEMM on the 5th-generation tensor cores: y[m,n] = bf16(x_scale[m] * w_scale[n] * sum_k x[m,k] * W[n,k]),
// x [M,K] and W [N,K] e4m3 codes, one fp32 scale per row of each, products exact, sums in fp32 in tensor memory.
// tcgen05.mma kind::f8f6f4 takes 32 codes (32 bytes) along K per instruction: the shared-memory tiles are the bf16
// kernels' byte for byte (128-byte rows, 128-byte swizzle), with twice the K in them.
//
// Two kernels:
//   gemm2_e4m3_kernel   many rows: CTA pairs on 256 x 256 tiles, persistent, two accumulators in tensor memory (the
//                       structure of emk_gemm2_sm100.cu: producer / MMA / sixteen epilogue warps per CTA). Bound by the
//                       tensor cores at K = 2048, by them and the output's drain together at K = 1024.
//   gemm_e4m3_rows_kernel   few rows: the operands change places, 128 rows of W are the instruction's M and 16 to 128
//                       tokens its N, so that no tensor-core row is padding and the grid is cut along W. The K axis is
//                       split over a cluster's CTAs, whose partial tiles meet in distributed shared memory (a fixed
//                       order of additions: the same bits on every run, no workspace, no atomics). Bound by reading W.
#include "emk_gemm_common.cuh"

namespace {

using namespace emk;

constexpr int BKB = 128;  // bytes (= codes) of K per slice: one swizzle row

// Instruction descriptor for kind::f8f6f4, e4m3 operands (format 0), both K-major, fp32 accumulation.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma8_pair_lohi(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(hi), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma8_lohi(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(hi), "r"(accumulate)
      : "memory");
}

struct Gemm8Args {
  __nv_bfloat16* y;
  const float* x_scale;
  const float* w_scale;
  int M, N;
  int tiles_m, tiles_n, kblocks;  // kblocks: 128-byte slices of K
  int stages;                     // few-rows kernel: ring depth
  int* status;
  unsigned long long limit_ns;
};

// ---------------------------------------------------------------------------------------------------------------
// Many rows: CTA pairs
// ---------------------------------------------------------------------------------------------------------------
constexpr int P8_THREADS = 576;  // warps 0-15: epilogue (four per quarter of the columns), 16: TMA, 17: MMA
constexpr int P8_TMA_WARP = 16, P8_MMA_WARP = 17;
constexpr int P8_GROUP_M = 8;
constexpr int P8_STAGES = 3;
constexpr int P8_KSUB = 2;
constexpr int P8_A_SUB = BM * BKB;  // one slice of this CTA's 128 rows of x

struct __align__(8) P8Barriers {
  uint64_t full[P8_STAGES];
  uint64_t empty[P8_STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int P8_OUT = 32 * 64;  // bytes of a warp's staging buffer: 32 rows of 32 columns
constexpr int p8_smem(int bn) {
  return P8_STAGES * P8_KSUB * (P8_A_SUB + bn / 2 * BKB) + 16 * P8_OUT + 1024 + (int)sizeof(P8Barriers);
}
static_assert(p8_smem(256) <= 227 * 1024, "shared memory of a CTA");

// 16 accumulator columns of a row -> bf16, scaled; lane first + i of wl holds column i's scale
__device__ __forceinline__ void scale16_e4m3(float wl, int first, const uint32_t* r, float xs, uint32_t* o) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float s0 = __shfl_sync(~0u, wl, first + 2 * q), s1 = __shfl_sync(~0u, wl, first + 2 * q + 1);
    o[q] = pack_bf16x2(__uint_as_float(r[2 * q]) * xs * s0, __uint_as_float(r[2 * q + 1]) * xs * s1);
  }
}

// keeps uses of these registers behind the tcgen05.wait::ld before it
__device__ __forceinline__ void tie_regs16(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(r[i]));
}

template <int BN>  // columns of a tile; each CTA loads half of them
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P8_THREADS, 1)
gemm2_e4m3_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const Gemm8Args g) {
  constexpr int B_SUB = BN / 2 * BKB;  // one slice of this CTA's half of the W tile
  constexpr int A_STAGE = P8_KSUB * P8_A_SUB, B_STAGE = P8_KSUB * B_SUB;
  constexpr uint32_t STAGE_TX = 2u * (A_STAGE + B_STAGE);  // both CTAs' bytes land on the leader's barrier
  constexpr int ACC = 256;             // tensor-memory columns from one accumulator to the next
  constexpr uint32_t IDESC = make_idesc_e4m3(2 * BM, BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + P8_STAGES * A_STAGE;
  uint8_t* sOut = sB + P8_STAGES * B_STAGE;
  P8Barriers* bars = reinterpret_cast<P8Barriers*>(sOut + 16 * P8_OUT);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;
  const int ntiles = g.tiles_m * g.tiles_n;

  if (threadIdx.x == 0) {
    for (int i = 0; i < P8_STAGES; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->tmem_full[i], 1);
      mbar_init(&bars->tmem_empty[i], 32);  // 16 epilogue warps of each CTA
    }
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == P8_TMA_WARP && lane == 0) {
    tma_prefetch_desc(&tma_a);
    tma_prefetch_desc(&tma_b);
  }
  if (warp == 0) {
    tmem_alloc_pair(&bars->tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
  const WaitCtx wc{&bars->abort_flag, g.status, g.limit_ns};

  if (warp == P8_TMA_WARP) {
    if (lane == 0) {  // TMA producer (both CTAs)
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < ntiles && ok; tile += npairs) {
        int tm, tn;
        tile_coords(tile, g.tiles_m, g.tiles_n, P8_GROUP_M, tm, tn);
        const int m0 = tm * 2 * BM + (int)rank * BM;
        const int n0 = tn * BN + (int)rank * (BN / 2);
        for (int kb = 0; kb < g.kblocks; kb += P8_KSUB) {
          if (!mbar_wait(&bars->empty[stage], phase ^ 1u, wc, EMK_DEV_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          const uint32_t full_leader = mapa_u32(smem_u32(&bars->full[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&bars->full[stage], STAGE_TX);
#pragma unroll
          for (int u = 0; u < P8_KSUB; ++u) {  // slices past K are zero-filled by TMA and add nothing
            const int k0 = (kb + u) * BKB;
            tma_load_2d_pair(sA + stage * A_STAGE + u * P8_A_SUB, &tma_a, full_leader, k0, m0);
            tma_load_2d_pair(sB + stage * B_STAGE + u * B_SUB, &tma_b, full_leader, k0, n0);
          }
          if (++stage == P8_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // the leader's last releases of this CTA's stages have arrived before it leaves (a stage that was never filled waits for none)
      for (int i = 0; i < P8_STAGES && ok; ++i) {
        ok = mbar_wait(&bars->empty[stage], phase ^ 1u, wc, EMK_DEV_TIMEOUT_PRODUCER);
        if (++stage == P8_STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == P8_MMA_WARP) {
    if (leader && lane == 0) {  // MMA issuer
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      const uint32_t desc_hi = smem_desc_hi(1024);
      const uint32_t a_lo0 = smem_desc_lo(smem_u32(sA), 0);
      const uint32_t b_lo0 = smem_desc_lo(smem_u32(sB), 0);
      for (int tile = pair; tile < ntiles && ok; tile += npairs, ++local) {
        const int acc = local & 1;
        const uint32_t acc_phase = (uint32_t)(local >> 1) & 1u;
        if (!mbar_wait(&bars->tmem_empty[acc], acc_phase ^ 1u, wc, EMK_DEV_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * ACC);
        for (int kb = 0; kb < g.kblocks; kb += P8_KSUB) {
          if (!mbar_wait(&bars->full[stage], phase, wc, EMK_DEV_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          const uint32_t a_st = a_lo0 + (uint32_t)(stage * (A_STAGE >> 4));
          const uint32_t b_st = b_lo0 + (uint32_t)(stage * (B_STAGE >> 4));
#pragma unroll
          for (int u = 0; u < P8_KSUB; ++u) {
#pragma unroll
            for (int k = 0; k < BKB / 32; ++k) {
              umma8_pair_lohi(d_tmem, a_st + (uint32_t)((u * P8_A_SUB + k * 32) >> 4), b_st + (uint32_t)((u * B_SUB + k * 32) >> 4), desc_hi, IDESC, (u | k) != 0 ? 1u : (uint32_t)(kb != 0));
            }
          }
          const uint32_t e_local = smem_u32(&bars->empty[stage]);
          tc_commit_pair(e_local);
          tc_commit_pair(mapa_u32(e_local, 1));
          if (++stage == P8_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) {
          const uint32_t f_local = smem_u32(&bars->tmem_full[acc]);
          tc_commit_pair(f_local);
          tc_commit_pair(mapa_u32(f_local, 1));
        }
      }
    }
  } else {
    // epilogue: a warp may only touch the tensor-memory lanes of its quarter (warp_id % 4); four warps share a quarter's
    // rows and take a fourth of the columns each. The drain of a K = 1024 tile lasts longer than its multiplication, and a
    // warp spends it waiting (tensor-memory loads, the turn through shared memory, stores).
    const int quarter = warp & 3, part = warp >> 2;
    int local = 0;
    for (int tile = pair; tile < ntiles; tile += npairs, ++local) {
      const int acc = local & 1;
      const uint32_t acc_phase = (uint32_t)(local >> 1) & 1u;
      int tm, tn;
      tile_coords(tile, g.tiles_m, g.tiles_n, P8_GROUP_M, tm, tn);
      const int row = tm * 2 * BM + (int)rank * BM + quarter * 32 + lane;
      const int n0 = tn * BN + part * (BN / 4);
      const float xs = row < g.M ? g.x_scale[row] : 0.f;
      float wl[(BN + 127) / 128];  // the columns' scales, one a lane
#pragma unroll
      for (int c = 0; c < (BN + 127) / 128; ++c) wl[c] = n0 + c * 32 + lane < g.N ? __ldg(g.w_scale + n0 + c * 32 + lane) : 0.f;
      if (!mbar_wait_warp(&bars->tmem_full[acc], acc_phase, wc, EMK_DEV_TIMEOUT_EPILOGUE)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * ACC + part * (BN / 4));
      // Lanes hold rows; what leaves is turned through shared memory, 32 columns at a time (16 last where a warp has 48), so
      // that four lanes write 64 bytes of a row side by side. Stored as they are held (a sector per lane and row) and with
      // each column's scale loaded by every lane, a 32768 x 4096 output of K = 1024 took 124 us instead of 116.
      uint8_t* const buf = sOut + warp * P8_OUT;
      constexpr int NC = BN / 64;
#pragma unroll
      for (int c = 0; c < NC; c += 2) {
        const int n = c + 1 < NC ? 2 : 1;  // 16-column chunks of this turn
        uint32_t r[2][16];
        tmem_ld_x16(taddr + (uint32_t)(c * 16), r[0]);
        if (n == 2) tmem_ld_x16(taddr + (uint32_t)(c * 16 + 16), r[1]);
        tmem_ld_wait();
        tie_regs16(r[0]);
        if (n == 2) tie_regs16(r[1]);
        if (c + 2 >= NC) {
          tc_fence_before();
          __syncwarp();
          // Only where the accumulator is used again, so that the leader's MMA warp waits for every arrive before it leaves: one that
          // nobody waits for could reach the leader's shared memory after the leader has gone (the last barrier orders nothing).
          if (lane == 0 && tile + 2 * npairs < ntiles) mbar_arrive_cluster_relaxed(mapa_u32(smem_u32(&bars->tmem_empty[acc]), 0));
        }
        __syncwarp();  // the buffer's last contents have been read
#pragma unroll
        for (int u = 0; u < n; ++u) {
          uint32_t o[8];
          scale16_e4m3(wl[c / 2], u * 16, r[u], xs, o);
#pragma unroll
          for (int v = 0; v < 2; ++v)  // 16-byte piece 2 u + v of row `lane`, swizzled by the row pair
            *reinterpret_cast<uint4*>(buf + lane * 64 + (((2 * u + v) ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        }
        __syncwarp();
        const int piece = lane & 3;
        const int col = n0 + c * 16 + piece * 8;
        const bool in = piece < 2 * n && col < g.N;  // N is a multiple of 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = i * 8 + (lane >> 2);
          const int64_t m = (int64_t)row - lane + rr;
          if (in && m < g.M)
            *reinterpret_cast<uint4*>(g.y + m * g.N + col) = *reinterpret_cast<const uint4*>(buf + rr * 64 + ((piece ^ ((rr >> 1) & 3)) << 4));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (bars->abort_flag) abort_drain();
  // The peer's shared and tensor memory stay alive until the leader's MMAs are done. Nothing is on its way to another CTA's shared
  // memory here: arrives and releases have been waited for above.
  cluster_sync_relaxed();
  if (warp == 0) tmem_dealloc_pair(tmem_base, 512);
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows: W rows along the instruction's M, tokens along its N, K split over the cluster
// ---------------------------------------------------------------------------------------------------------------
constexpr int R8_THREADS = 192;  // warps 0-3: epilogue, 4: TMA, 5: MMA
constexpr int R8_MAX_STAGES = 12;
constexpr int R8_MAX_SPLIT = 8;  // portable cluster size
constexpr int R8_W_STAGE = BM * BKB;

struct __align__(8) R8Barriers {
  uint64_t full[R8_MAX_STAGES];
  uint64_t empty[R8_MAX_STAGES];
  uint64_t tmem_full;
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ uint32_t cluster_size_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int NT>  // tokens per tile
__global__ void __launch_bounds__(R8_THREADS)
gemm_e4m3_rows_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x, const Gemm8Args g) {
  constexpr int X_STAGE = NT * BKB;
  constexpr int STAGE = R8_W_STAGE + X_STAGE;
  constexpr uint32_t TMEM_COLS = NT < 32 ? 32 : NT;
  constexpr uint32_t IDESC = make_idesc_e4m3(BM, NT);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t split = cluster_size_x();
  const uint32_t rank = cluster_ctarank();
  float* part = reinterpret_cast<float*>(ring);  // [NT][128] partial sums, once the ring is done with
  R8Barriers* bars = reinterpret_cast<R8Barriers*>(ring + max(g.stages * STAGE, NT * BM * 4));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tile = blockIdx.x / split;
  const int tn = tile % g.tiles_n, tm = tile / g.tiles_n;
  const int kb0 = (int)((int64_t)g.kblocks * rank / split), kb1 = (int)((int64_t)g.kblocks * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->tmem_full, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tma_w);
    tma_prefetch_desc(&tma_x);
  }
  // W may come to L2 while the kernel before this one still runs: a prefetch reads nothing, so it need not wait (a layer of a
  // single-token step with 400 MB of weights 29.8 -> 29.0 us).
  if (warp == 5 && lane == 0) {
    for (int kb = kb0; kb < kb1 && kb < kb0 + g.stages; ++kb) tma_prefetch_2d(&tma_w, kb * BKB, tn * BM);
  }
  if (warp == 0) {
    tmem_alloc(&bars->tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
  const WaitCtx wc{&bars->abort_flag, g.status, g.limit_ns};
  if (warp == 4) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&bars->empty[stage], phase ^ 1u, wc, EMK_DEV_TIMEOUT_PRODUCER)) break;
        mbar_arrive_expect_tx(&bars->full[stage], STAGE);
        tma_load_2d(ring + stage * STAGE, &tma_w, &bars->full[stage], kb * BKB, tn * BM);
        tma_load_2d(ring + stage * STAGE + R8_W_STAGE, &tma_x, &bars->full[stage], kb * BKB, tm * NT);
        if (++stage == g.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t desc_hi = smem_desc_hi(1024);
      const uint32_t lo0 = smem_desc_lo(smem_u32(ring), 0);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&bars->full[stage], phase, wc, EMK_DEV_TIMEOUT_MMA)) {
          ok = false;
          break;
        }
        const uint32_t w_lo = lo0 + (uint32_t)(stage * (STAGE >> 4));
        const uint32_t x_lo = w_lo + (uint32_t)(R8_W_STAGE >> 4);
#pragma unroll
        for (int k = 0; k < BKB / 32; ++k)
          umma8_lohi(tmem_base, w_lo + (uint32_t)(k * 2), x_lo + (uint32_t)(k * 2), desc_hi, IDESC,
                     k != 0 ? 1u : (uint32_t)(kb != kb0));
        tc_commit(&bars->empty[stage]);
        if (++stage == g.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) tc_commit(&bars->tmem_full);
    }
    __syncwarp();
  } else {
    // the partial tile goes to shared memory, token-major, over the ring: every MMA that read it has finished
    if (mbar_wait_warp(&bars->tmem_full, 0, wc, EMK_DEV_TIMEOUT_EPILOGUE)) {
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(warp * 32) << 16);
#pragma unroll
      for (int c = 0; c < NT / 16; ++c) {
        uint32_t r[16];
        tmem_ld_x16(taddr + (uint32_t)(c * 16), r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c * 16 + i) * BM + warp * 32 + lane] = __uint_as_float(r[i]);
      }
      tc_fence_before();
    }
  }

  __syncthreads();
  if (bars->abort_flag) abort_drain();
  if (warp == 0) tmem_dealloc(tmem_base, TMEM_COLS);
  if (split > 1) cluster_sync_all();  // (reached by every thread of every CTA, whatever happened above)
  // CTA `rank` finishes the tokens rank, rank + split, ...: a warp takes a token's 128 columns, four per lane, and adds
  // the cluster's partial sums in the order of the ranks
  const int n = tn * BM + lane * 4;
  if (n < g.N && bars->abort_flag == 0) {
    const float4 ws = __ldg(reinterpret_cast<const float4*>(g.w_scale + n));
    const uint32_t at = smem_u32(part) + (uint32_t)lane * 16u;
    const int tokens = min(NT, g.M - tm * NT);
    for (int tok = (int)rank + (int)split * warp; tok < tokens; tok += (int)split * (R8_THREADS / 32)) {
      const float xs = g.x_scale[tm * NT + tok];
      float4 v[R8_MAX_SPLIT];
#pragma unroll
      for (uint32_t s = 0; s < R8_MAX_SPLIT; ++s)
        if (s < split) v[s] = ld_cluster_f32x4(mapa_u32(at + (uint32_t)tok * (BM * 4), s));
#pragma unroll
      for (uint32_t s = 1; s < R8_MAX_SPLIT; ++s)
        if (s < split) {
          v[0].x += v[s].x;
          v[0].y += v[s].y;
          v[0].z += v[s].z;
          v[0].w += v[s].w;
        }
      *reinterpret_cast<uint2*>(g.y + (int64_t)(tm * NT + tok) * g.N + n) =
          make_uint2(pack_bf16x2(v[0].x * xs * ws.x, v[0].y * xs * ws.y), pack_bf16x2(v[0].z * xs * ws.z, v[0].w * xs * ws.w));
    }
  }
  __syncwarp();
  if (split > 1) cluster_sync_relaxed();  // no CTA leaves while another reads its shared memory
}

constexpr int rows_smem(int nt, int stages) {
  const int ring = stages * (R8_W_STAGE + nt * BKB), part = nt * BM * 4;
  return (ring > part ? ring : part) + 1024 + (int)sizeof(R8Barriers);
}

template <int NT>
int launch_rows(emk_handle_t h, const CUtensorMap& tw, const CUtensorMap& tx, Gemm8Args g, int split, cudaStream_t s) {
  constexpr int BUDGET = 110 * 1024;  // two CTAs per SM
  constexpr int ROOM = (BUDGET - 1024 - (int)sizeof(R8Barriers)) / (R8_W_STAGE + NT * BKB);
  static_assert(ROOM >= 3 && rows_smem(NT, 1) <= BUDGET, "a ring of three stages");
  const int want = (g.kblocks + split - 1) / split;
  g.stages = want < ROOM ? want : ROOM;
  if (g.stages > R8_MAX_STAGES) g.stages = R8_MAX_STAGES;
  const int smem = rows_smem(NT, g.stages);
  static emk_device_once once;
  {
    std::lock_guard<std::mutex> lk(once.mu);
    if (!once.done[h->device]) {
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(gemm_e4m3_rows_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, BUDGET));
      once.done[h->device] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.tiles_m * g.tiles_n * split), 1, 1);
  cfg.blockDim = dim3(R8_THREADS, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = h->overlap_launch != 0 ? 2 : 1;
  EMK_CUDA_TRY(h, cudaLaunchKernelEx(&cfg, gemm_e4m3_rows_kernel<NT>, tw, tx, g));
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}

int linear_rows(emk_handle_t h, const void* x, const void* w, Gemm8Args g, int64_t K, cudaStream_t s) {
  const int nt = g.M <= 16 ? 16 : g.M <= 32 ? 32 : g.M <= 64 ? 64 : 128;
  g.tiles_m = (g.M + nt - 1) / nt;
  g.tiles_n = (g.N + BM - 1) / BM;
  // Split K until every SM has a CTA, each with two slices at least. A third more CTAs than SMs still pays while the
  // partial tiles are small (1 x 6144 x 2048: 192 CTAs 4.7 us, 96 CTAs 5.3; 128 rows: 9.5 and 9.0), two per SM where each
  // keeps a long K (128 x 8192 x 8192: 19.7 us against 22.0), and eight parts only for small tiles or few of them
  // (128 x 2048 x 4096: 8.9 us in eight, 7.9 in four; one row 4.4 and 5.2; 1024 x 128 x 4096: 7.0 and 8.0).
  const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n, sms = h->sm_count;
  const int most = nt <= 32 || tiles <= 8 ? R8_MAX_SPLIT : 4;
  int split = 1;
  while (split < most && g.kblocks >= split * 4) {
    const int64_t cap = g.kblocks >= split * 2 * 16 ? 2 * sms : nt <= 32 ? sms + sms / 3 : sms;
    if (tiles * split * 2 > cap) break;
    split *= 2;
  }
  CUtensorMap tw, tx;
  int rc = emk_make_tmap_2d(h, &tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, (uint64_t)K, (uint64_t)g.N, (uint64_t)K, BKB, BM,
                            CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != EMK_OK) return rc;
  rc = emk_make_tmap_2d(h, &tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, (uint64_t)K, (uint64_t)g.M, (uint64_t)K, BKB,
                        (uint32_t)nt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != EMK_OK) return rc;
  switch (nt) {
    case 16: return launch_rows<16>(h, tw, tx, g, split, s);
    case 32: return launch_rows<32>(h, tw, tx, g, split, s);
    case 64: return launch_rows<64>(h, tw, tx, g, split, s);
    default: return launch_rows<128>(h, tw, tx, g, split, s);
  }
}

template <int BN>
int launch_pairs(emk_handle_t h, const CUtensorMap& ta, const void* w, Gemm8Args g, int64_t K, cudaStream_t s) {
  g.tiles_m = (g.M + 2 * BM - 1) / (2 * BM);
  g.tiles_n = (g.N + BN - 1) / BN;
  CUtensorMap tb;
  const int rc = emk_make_tmap_2d(h, &tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, (uint64_t)K, (uint64_t)g.N, (uint64_t)K, BKB,
                                  BN / 2, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != EMK_OK) return rc;
  static emk_device_once once;
  {
    std::lock_guard<std::mutex> lk(once.mu);
    if (!once.done[h->device]) {
      EMK_CUDA_TRY(h, cudaFuncSetAttribute(gemm2_e4m3_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, p8_smem(BN)));
      once.done[h->device] = true;
    }
  }
  const int ntiles = g.tiles_m * g.tiles_n;
  const int pairs = ntiles < h->sm_count / 2 ? ntiles : h->sm_count / 2;
  EMK_CUDA_TRY(h, launch_after_prologue(gemm2_e4m3_kernel<BN>, 2u * (unsigned)pairs, P8_THREADS, p8_smem(BN), s,
                                        h->overlap_launch != 0, ta, tb, g));
  EMK_LAUNCH_CHECK(h);
  return EMK_OK;
}

int linear_pairs(emk_handle_t h, const void* x, const void* w, const Gemm8Args& g, int64_t K, cudaStream_t s) {
  CUtensorMap ta;
  const int rc = emk_make_tmap_2d(h, &ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, (uint64_t)K, (uint64_t)g.M, (uint64_t)K, BKB,
                                  BM, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != EMK_OK) return rc;
  // Rounds of tiles over the machine's pairs, times what a round costs at the tile's width: with every pair busy a round of
  // 256-, 192- or 128-column tiles takes 7.3 / 6.0 / 4.8 us at K = 2048 and 3.8 / 3.2 / 2.5 at K = 1024 (operand traffic
  // per multiplication grows as the tile narrows), so narrow tiles pay only where they save rounds; the weights stand a
  // little above those ratios because near a tie the wide tile is the faster. Measured at 1024 x 6144 x 2048:
  // 16.9 / 15.3 / 17.8 us; 256 x 4096 x 1024: 7.4 / 6.3 / 5.5; 4096 x 6144 x 2048: 42.1 / 43.8 / 53.1.
  const int64_t pairs = h->sm_count / 2, tiles_m = (g.M + 2 * BM - 1) / (2 * BM);
  const auto cost = [&](int64_t bn, int64_t weight) { return (tiles_m * ((g.N + bn - 1) / bn) + pairs - 1) / pairs * weight; };
  const int64_t c256 = cost(256, 100), c192 = cost(192, 88), c128 = cost(128, 69);
  if (c128 < c192 && c128 < c256) return launch_pairs<128>(h, ta, w, g, K, s);
  return c192 < c256 ? launch_pairs<192>(h, ta, w, g, K, s) : launch_pairs<256>(h, ta, w, g, K, s);
}

// Which kernel: up to 64 rows the pairs would multiply padding (64 rows by 4096 x 1024 5.1 us here, 5.3 in pairs, by 28672 x 4096 24.5
// and 28.7, by 8192 x 8192 15.8 and 20.9; one row 3.8 / 5.8, 21.6 / 36.9, 13.7 / 31.8); beyond that the rows kernel wins where only its split of K
// fills the machine: few tiles and a K worth splitting (1024 x 128 x 4096: 6.9 us against 10.6; 512 x 512 x 2048: 6.4
// against 7.0), or a long K under one row of tiles (128 x 8192 x 8192: 18.2 against 21.4). It loses otherwise
// (128 x 2048 x 512: 6.5 against 4.5; 128 x 4096 x 1024: 6.2 against 5.4; 256 x 4096 x 1024: 7.5 against 5.5).
bool few_rows(int64_t M, int64_t N, int64_t K) {
  if (M <= 64) return true;
  return ((M + BM - 1) / BM * ((N + BM - 1) / BM) <= 16 && K >= 2048) || (M <= BM && K >= 4096);
}

}  // namespace

extern "C" int emk_linear_e4m3(emk_handle_t h, const void* x, const float* x_scale, const void* w, const float* w_scale,
                               void* y, int64_t M, int64_t N, int64_t K, emk_stream_t stream) {
  if (!h || !x || !x_scale || !w || !w_scale || !y) return EMK_ERR_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return EMK_ERR_SHAPE;
  if ((K % 16) != 0 || (N % 8) != 0) {
    EMK_SET_ERR(h, "emk_linear_e4m3: K must be a multiple of 16 and N of 8; got K=%lld N=%lld", (long long)K, (long long)N);
    return EMK_ERR_ALIGN;
  }
  if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)w_scale) & 15u) != 0 || ((uintptr_t)x_scale & 3u) != 0)
    return EMK_ERR_ALIGN;
  if ((M + 15) / 16 * ((N + 127) / 128) > (1 << 28)) {
    EMK_SET_ERR(h, "emk_linear_e4m3: output of %lld x %lld is too large for one launch", (long long)M, (long long)N);
    return EMK_ERR_LIMIT;
  }
  Gemm8Args g = {};
  g.y = (__nv_bfloat16*)y;
  g.x_scale = x_scale;
  g.w_scale = w_scale;
  g.M = (int)M;
  g.N = (int)N;
  g.kblocks = (int)((K + BKB - 1) / BKB);
  g.status = h->status_dev;
  g.limit_ns = h->wait_limit_ns;
  return few_rows(M, N, K) ? linear_rows(h, x, w, g, K, (cudaStream_t)stream) : linear_pairs(h, x, w, g, K, (cudaStream_t)stream);
}
