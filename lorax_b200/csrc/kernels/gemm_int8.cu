// Products of 8-bit integers with a scale for each token and each output channel, on the 5th-generation tensor cores:
//   out[t, n] = (sum_k xq[t, k] * wq[n, k]) * ws[n] * xs[t] + bias[n]
// The sums are whole numbers in 32 bits (tcgen05.mma.kind::i8, exact for K below 2^17: 128 * 128 * (2^17 - 1) < 2^31), so that no order in which parts of
// K are added changes a result; scales and bias are applied in 32-bit floating point, the
// weights' first (rows of any size then overflow only where their results do), and the result is rounded to bf16 once.
//
// Weights take the UMMA M side, 128 output features a tile; tokens the N side in steps of 16.  A stage of the ring is 128 bytes of K of both.
// Where there are fewer tiles than SMs the CTAs of a cluster share a tile's K and add their sums up through each other's shared memory: nothing is
// kept in global memory between CTAs, calls or graphs.
#include <math.h>
#include <string.h>

#include "pair.cuh"

namespace lx {

constexpr int kI8BM = 128;                        // output features of a tile
constexpr int kI8BK = 128;                        // bytes of K in a stage: one row of the 128-byte swizzle
constexpr int kI8Threads = 256;                   // 128 for tiles of 16 tokens, whose results are few: a row of 28672 x 4096 20.1 us, with 256 20.7
constexpr int kI8MaxStages = 16;
constexpr int kI8MaxParts = 8;                    // CTAs that share a tile's K: a portable cluster
constexpr int kI8ABytes = kI8BM * kI8BK;
constexpr int kI8Most = 0x7fff0000;               // rows, features: with a tile more they stay below 2^31

struct Int8GemmParams {
  int N, T, K;
  int bn, stages, parts, tmem_cols;               // token tile (a multiple of 16), stages of the ring, CTAs of a tile
  int reuse;                                      // more than one token tile: weights stay in L2
  const float* xs;                                // [T]
  const float* ws;                                // [N]
  const __nv_bfloat16* bias;                      // [N] or null
  __nv_bfloat16* out;
  long long ldo;
  int wide;                                       // rows of out begin at 8 bytes
  int* status;
  int w_const;                                    // no kernel that may still run writes the weights: their first tiles are loaded before pdl_wait
};

// kind::i8: both operands signed, sums in 32-bit integers.
LX_DEVICE void umma_i8_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__host__ __device__ constexpr uint32_t make_idesc_i8(uint32_t M, uint32_t N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);      // D in s32, A and B in s8, both K-major
}

LX_DEVICE int4 cluster_load_int4(uint32_t smem_addr, uint32_t rank) {
  int4 v;
  asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [ra];\n\t}"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_addr), "r"(rank) : "memory");
  return v;
}

// A tile's scales and biases in shared memory, fetched while its products are formed: behind them every load would wait for L2.
struct __align__(16) Int8Scales {
  float ws[kI8BM], bias[kI8BM], xs[256];
};
LX_DEVICE void int8_scales(const Int8GemmParams& p, Int8Scales& sc, int n0, int t0, int thread, int threads) {
  for (int i = thread; i < kI8BM; i += threads) {
    const int at = min(n0 + i, p.N - 1);
    sc.ws[i] = p.ws[at];
    sc.bias[i] = p.bias != nullptr ? __bfloat162float(p.bias[at]) : 0.f;
  }
  for (int i = thread; i < p.bn; i += threads) sc.xs[i] = p.xs[min(t0 + i, p.T - 1)];
}

// A tile's results from its parts' sums ([token][128 features] in the shared memory of the CTAs first, first + stride ... of the cluster; of this one, if there are
// no others).  A warp takes a token's features, four a lane; the tokens go round the warps of all parts, and the sums of several are on their way at a time: a
// trip to another CTA's shared memory takes the better part of a microsecond.
template <int PARTS, int ROWS>
LX_DEVICE void int8_join(const Int8GemmParams& p, const int* sums, const Int8Scales& sc, int part, uint32_t first, uint32_t stride, int n0, int t0, int live) {
  const int lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5, step = warps * p.parts, n = n0 + lane * 4;
  const float4 w4 = *reinterpret_cast<const float4*>(sc.ws + lane * 4), b4 = *reinterpret_cast<const float4*>(sc.bias + lane * 4);
  const float ws[4] = {w4.x, w4.y, w4.z, w4.w}, bias[4] = {b4.x, b4.y, b4.z, b4.w};
  const uint32_t at = smem_u32(sums) + (uint32_t)lane * 16;
  for (int t = (int)(threadIdx.x >> 5) * p.parts + part; t < live; t += ROWS * step) {
    int4 v[ROWS][PARTS];
    float xs[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int tu = min(t + u * step, live - 1);
      xs[u] = sc.xs[tu];
#pragma unroll
      for (int r = 0; r < PARTS; ++r) {
        const uint32_t src = at + (uint32_t)tu * (kI8BM * 4);
        if (PARTS == 1) v[u][r] = *reinterpret_cast<const int4*>(sums + tu * kI8BM + lane * 4);
        else if (r < p.parts) v[u][r] = cluster_load_int4(src, first + (uint32_t)r * stride);
      }
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if (t + u * step >= live) break;
      int4 s = v[u][0];
#pragma unroll
      for (int r = 1; r < PARTS; ++r)
        if (r < p.parts) { s.x += v[u][r].x; s.y += v[u][r].y; s.z += v[u][r].z; s.w += v[u][r].w; }
      const float f[4] = {(float)s.x * ws[0] * xs[u] + bias[0], (float)s.y * ws[1] * xs[u] + bias[1], (float)s.z * ws[2] * xs[u] + bias[2],
                          (float)s.w * ws[3] * xs[u] + bias[3]};
      __nv_bfloat16* row = p.out + (long long)(t0 + t + u * step) * p.ldo + n0;
      if (p.wide) {
        if (n + 4 <= p.N) *reinterpret_cast<uint2*>(row + lane * 4) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        else
          for (int q = 0; q < 4; ++q)
            if (n + q < p.N) row[lane * 4 + q] = __float2bfloat16(f[q]);
      } else {
        // a row that begins anywhere: 32 neighbours a store, fetched from the lanes that hold them
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float g = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float h = __shfl_sync(0xffffffffu, f[q], 8 * e + (lane >> 2));
            if ((lane & 3) == q) g = h;
          }
          if (n0 + 32 * e + lane < p.N) row[32 * e + lane] = __float2bfloat16(g);
        }
      }
    }
  }
}

// One tile a cluster, one part of its K a CTA.  Warp 0 loads, warp 1 multiplies, all (four or eight) write results.  Short steps: the weights' way from HBM is the bound, and
// two CTAs an SM with six stages of 16 KB each keep enough of them on their way whatever the number of tiles (a persistent CTA an SM would leave the last wave
// short): one row of 28672 x 4096 20.1 to 21.1 us (5.7 TB/s), 48 rows 22.3.  Narrow layers have fewer tiles than SMs: one row of 4096 x 14336 by eight CTAs a tile 12.9 us, alone 34.5.
// Middle steps take large tiles, whose operands come from L2 at 100 bytes a nanosecond and SM: 256 rows of 4096 x 14336 20.7 us by four CTAs a tile of 256 tokens.
__global__ void __launch_bounds__(kI8Threads, 3)
gemm_int8_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = kI8ABytes + p.bn * kI8BK;
  Int8Scales& scales = *reinterpret_cast<Int8Scales*>(smem + p.stages * stage_bytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(&scales + 1);
  uint64_t* empty_bar = full_bar + kI8MaxStages;
  uint64_t* done_bar = empty_bar + kI8MaxStages;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
  int* sums = reinterpret_cast<int*>(smem);                  // [token][128 features], over the ring when its last stage has been read

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = (int)blockIdx.x % p.parts, item = (int)blockIdx.x / p.parts;
  const int tiles_b = (p.T + p.bn - 1) / p.bn;
  const int ta = item / tiles_b, tb = item % tiles_b;        // the token tiles of a weight tile run side by side
  const int kblocks = (p.K + kI8BK - 1) / kI8BK;
  const int kb0 = (int)((long long)kblocks * part / p.parts), kb1 = (int)((long long)kblocks * (part + 1) / p.parts);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) { tmem_alloc(tmem_base_slot, (uint32_t)p.tmem_cols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_d = *tmem_base_slot;

  if (!p.w_const) pdl_wait();
  const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
  const uint32_t bytes = (uint32_t)stage_bytes;
  const int ahead = min(p.stages, kb1 - kb0);
  const auto load_w = [&](int kb, int stage) {
    if (p.reuse) tma_load_2d(smem + stage * stage_bytes, &tmap_w, &full_bar[stage], kb * kI8BK, ta * kI8BM);
    else tma_load_2d_hint(smem + stage * stage_bytes, &tmap_w, &full_bar[stage], kb * kI8BK, ta * kI8BM, pol_w);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < ahead; ++s) {
      mbar_expect_tx(&full_bar[s], bytes);
      load_w(kb0 + s, s);
    }
  }
  pdl_wait();
  pdl_trigger();

  int loaded = 0;                                            // (of thread 0) stages filled so far
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++loaded) {
        if (loaded >= ahead) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
            report_status(p.status, kTimeoutEmptyBarrier, item);
            *abort_flag = 1;
            break;
          }
          mbar_expect_tx(&full_bar[stage], bytes);
          load_w(kb, stage);
        }
        tma_load_2d_hint(smem + stage * stage_bytes + kI8ABytes, &tmap_x, &full_bar[stage], kb * kI8BK, tb * p.bn, pol_x);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_i8(kI8BM, (uint32_t)p.bn);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag)) {
          report_status(p.status, kTimeoutFullBarrier, item);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * stage_bytes);
        const uint64_t da = make_desc_k_sw128(sa), db = make_desc_k_sw128(sa + kI8ABytes);
#pragma unroll
        for (int k = 0; k < kI8BK / 32; ++k) umma_i8_ss(tmem_d, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
        tc_commit(&empty_bar[stage]);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      tc_commit(done_bar);
    }
    __syncwarp();
  } else {
    int8_scales(p, scales, ta * kI8BM, tb * p.bn, (int)threadIdx.x - 64, (int)blockDim.x - 64);
  }

  // (done: every load of this CTA has arrived and been read, so the ring is free)
  const bool ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag));
  if (!ok) {
    report_status(p.status, kTimeoutTmemFull, item);
    *abort_flag = 1;
  }
  const int t0 = tb * p.bn, live = min(p.bn, p.T - t0);
  if (ok) {
    tc_fence_after();
    const int quad = warp & 3;                               // (the lanes that a warp may read; two warps take turns at their columns)
    const uint32_t taddr = tmem_d + ((uint32_t)(quad * 32) << 16);
    int* mine = sums + quad * 32 + lane;
    for (int c = (warp >> 2) * 16; c < live; c += (int)blockDim.x / 8) {
      uint32_t r[16];
      tmem_ld_32x32b_x16(taddr + c, r);
      tc_wait_ld();
#pragma unroll
      for (int q = 0; q < 16; ++q) mine[(c + q) * kI8BM] = (int)r[q];      // (rows of the tile behind the last token too: there is room for bn of them)
    }
    tc_fence_before();
  }
  if (p.parts > 1) cluster_sync();
  else __syncthreads();
  if (__syncthreads_or(*abort_flag) == 0) {
    if (p.parts == 1) int8_join<1, 4>(p, sums, scales, 0, 0, 0, ta * kI8BM, t0, live);
    else if (p.parts <= 4) int8_join<4, 2>(p, sums, scales, part, 0, 1, ta * kI8BM, t0, live);
    else int8_join<kI8MaxParts, 1>(p, sums, scales, part, 0, 1, ta * kI8BM, t0, live);
  }
  if (*abort_flag && threadIdx.x == 0)  // copies still on their way arrive before this CTA leaves
    for (int s = 0; s < min(p.stages, loaded); ++s) mbar_wait(&full_bar[s], (uint32_t)((loaded - 1 - s) / p.stages) & 1u, nullptr);
  __syncwarp();
  if (p.parts > 1) cluster_sync();      // nobody leaves while its sums are read
  else __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_d, (uint32_t)p.tmem_cols); }
}

// ------------------------------------------------------------------------------------------------
// Long steps, by pairs of CTAs (cta_group::2): a tile is 256 features x up to 256 tokens, of which each CTA loads 128 rows of the weights and half of
// the tokens, 32 KB a stage for 4 x 256 x 256 x 32 products, where one CTA on 128 x 256 takes 48 KB for half as many.  What comes in from L2 is what bounds a
// single CTA at these sizes (some 95 bytes a nanosecond).  One part: persistent pairs, whose accumulators take turns, so that a tile's results are written while
// the next one is multiplied.  Several: a cluster of pairs shares one tile's K, as above.  4001 rows of 28672 x 4096: 318 to 332 us (2.9 POP/s; cuBLAS's integer
// product 293 to 296), the tensor pipe 77 % active at the 1.64 GHz that the power limit leaves, its stages waiting for 32 KB each at 80 bytes a nanosecond.
// ------------------------------------------------------------------------------------------------
constexpr int kI8PairStages = 6;
constexpr int kI8PairEpiWarps = 8;                // two for each quarter of the features, half of the tokens each
constexpr int kI8PairThreads = 64 + 32 * kI8PairEpiWarps;
constexpr int kI8PairStageBytes = 2 * kI8ABytes;
constexpr int kI8PairMaxParts = 4;
constexpr int kI8TurnBytes = kI8PairEpiWarps * 16 * 32 * 4;      // a warp's 32 features x 32 tokens in bf16, two tokens a word
constexpr int kI8PairSmem = kI8PairStages * kI8PairStageBytes + kI8TurnBytes + (int)sizeof(Int8Scales) + 256 + 1024;
static_assert(kI8PairSmem <= 227 * 1024 && 256 * kI8BM * 4 <= kI8PairStages * kI8PairStageBytes, "the ring holds a tile's sums");

LX_DEVICE void pair_mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// pair_commit of a pair that is not the cluster's first.
LX_DEVICE void pair_commit_of(uint64_t* bar, uint32_t even) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"((uint16_t)(3u << even)) : "memory");
}

__global__ void __launch_bounds__(kI8PairThreads, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint32_t* turn_all = reinterpret_cast<uint32_t*>(smem + kI8PairStages * kI8PairStageBytes);
  Int8Scales& scales = *reinterpret_cast<Int8Scales*>(smem + kI8PairStages * kI8PairStageBytes + kI8TurnBytes);    // (of a shared tile)
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(&scales + 1);                                                   // (the even CTA's are used)
  uint64_t* empty_bar = full_bar + kI8PairStages;
  uint64_t* tmem_full = empty_bar + kI8PairStages;
  uint64_t* tmem_empty = tmem_full + 2;                                                                            // (the even CTA's are used)
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_rank(), even = cta & ~1u;
  const int rank = (int)(cta & 1), part = (int)(cta >> 1);
  const int tiles_b = (p.T + p.bn - 1) / p.bn;
  const int num_tiles = (p.N + 2 * kI8BM - 1) / (2 * kI8BM) * tiles_b;
  const int first = (int)blockIdx.x / (2 * p.parts), step = p.parts > 1 ? num_tiles : (int)gridDim.x / 2;      // (parts: one tile a cluster)
  const int kblocks = (p.K + kI8BK - 1) / kI8BK;
  const int kb0 = (int)((long long)kblocks * part / p.parts), kb1 = (int)((long long)kblocks * (part + 1) / p.parts);
  const int half = p.bn >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kI8PairStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&tmem_full[s], 1); mbar_init(&tmem_empty[s], 2 * kI8PairEpiWarps); }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) pair_tmem_alloc(tmem_base_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                      // both CTAs' barriers and columns are there
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;

  if (!p.w_const) pdl_wait();
  const uint32_t bytes = 2u * (uint32_t)(kI8ABytes + half * kI8BK);      // of a stage, in both CTAs
  int ahead = 0;
  if (threadIdx.x == 0 && first < num_tiles) {
    ahead = min(kI8PairStages, kb1 - kb0);
    for (int s = 0; s < ahead; ++s) {
      if (rank == 0) mbar_expect_tx(&full_bar[s], bytes);
      pair_load_2d(smem + s * kI8PairStageBytes, &tmap_w, pair_map(&full_bar[s], even), (kb0 + s) * kI8BK, (2 * (first / tiles_b) + rank) * kI8BM);
    }
  }
  pdl_wait();
  pdl_trigger();

  int loaded = 0;                                      // (of thread 0) stages filled so far
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        const int i0 = (2 * (tile / tiles_b) + rank) * kI8BM, j0 = tile % tiles_b * p.bn + rank * half;
        for (int kb = kb0; kb < kb1; ++kb, ++loaded) {
          const uint32_t bar = pair_map(&full_bar[stage], even);
          uint8_t* sa = smem + stage * kI8PairStageBytes;
          if (loaded >= ahead) {
            if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
              report_status(p.status, kTimeoutEmptyBarrier, tile);
              *abort_flag = 1;
              ok = false;
              break;
            }
            if (rank == 0) mbar_expect_tx(&full_bar[stage], bytes);
            pair_load_2d(sa, &tmap_w, bar, kb * kI8BK, i0);
          }
          pair_load_2d(sa + kI8ABytes, &tmap_x, bar, kb * kI8BK, j0);
          if (++stage == kI8PairStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      const uint32_t idesc = make_idesc_i8(2 * kI8BM, (uint32_t)p.bn);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase[2] = {0, 0};
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        if (!pair_wait(&tmem_empty[acc], acc_phase[acc] ^ 1, abort_flag)) {
          report_status(p.status, kTimeoutTmemEmpty, tile);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t tmem_d = tmem_base + (uint32_t)(acc * 256);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) {
            report_status(p.status, kTimeoutFullBarrier, tile);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kI8PairStageBytes);
          const uint64_t da = make_desc_k_sw128(sa), db = make_desc_k_sw128(sa + kI8ABytes);
#pragma unroll
          for (int k = 0; k < kI8BK / 32; ++k) pair_mma_i8(tmem_d, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          pair_commit_of(&empty_bar[stage], even);
          if (++stage == kI8PairStages) { stage = 0; phase ^= 1; }
        }
        if (ok) pair_commit_of(&tmem_full[acc], even);
        acc_phase[acc] ^= 1;
        acc ^= 1;
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, late = (warp - 2) >> 2;      // (late: the warp that takes every other 32 tokens from the second on)
    uint32_t* turn = turn_all + (warp - 2) * (16 * 32);
    int* sums = reinterpret_cast<int*>(smem);          // [token][128 features], of a shared tile: over the ring, which has been read by then
    int acc = 0;
    uint32_t acc_phase[2] = {0, 0};
    for (int tile = first; tile < num_tiles; tile += step) {
      const int j0 = tile % tiles_b * p.bn, jend = min(p.T, j0 + p.bn);
      const int f0 = (2 * (tile / tiles_b) + rank) * kI8BM + quad * 32, fi = min(f0 + lane, p.N - 1);
      float ws = 0.f, bias = 0.f, xl[4];                // (fetched while the tile's products are formed; xl[i]: the scale of token 32 (2 i + late) + lane)
      if (p.parts > 1) {
        int8_scales(p, scales, f0 - quad * 32, j0, (int)threadIdx.x - 64, kI8PairThreads - 64);
      } else {
        ws = p.ws[fi];
        if (p.bias != nullptr) bias = __bfloat162float(p.bias[fi]);
#pragma unroll
        for (int i = 0; i < 4; ++i) xl[i] = p.xs[min(j0 + 32 * (2 * i + late) + lane, p.T - 1)];
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase[acc], abort_flag))) {
        report_status(p.status, kTimeoutTmemFull, tile);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      acc_phase[acc] ^= 1;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * 256);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 32 * (2 * i + late);
        if (c >= p.bn || j0 + c >= jend) break;
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + c, r);
        tc_wait_ld();
        if (p.parts > 1) {
#pragma unroll
          for (int q = 0; q < 32; ++q) sums[(c + q) * kI8BM + quad * 32 + lane] = (int)r[q];
          continue;
        }
        if (!p.wide) {
          // rows that begin anywhere: 32 neighbours a store, as they are
#pragma unroll
          for (int q = 0; q < 32; ++q) {
            const float v = (float)(int)r[q] * ws * __shfl_sync(0xffffffffu, xl[i], q) + bias;
            if (j0 + c + q < jend && f0 + lane < p.N) p.out[(long long)(j0 + c + q) * p.ldo + f0 + lane] = __float2bfloat16(v);
          }
          continue;
        }
        // a thread holds one feature of 32 tokens; the warp turns its block around, two tokens a word, and a lane stores eight features of two tokens
#pragma unroll
        for (int q = 0; q < 32; q += 2) {
          const float a = (float)(int)r[q] * ws * __shfl_sync(0xffffffffu, xl[i], q) + bias;
          const float b = (float)(int)r[q + 1] * ws * __shfl_sync(0xffffffffu, xl[i], q + 1) + bias;
          turn[(q >> 1) * 32 + lane] = pack_bf16x2(a, b);
        }
        __syncwarp();
        const int n = f0 + (lane & 3) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pr = h * 8 + (lane >> 2), t = j0 + c + 2 * pr;
          const uint4 u = *reinterpret_cast<const uint4*>(turn + pr * 32 + (lane & 3) * 8), v = *reinterpret_cast<const uint4*>(turn + pr * 32 + (lane & 3) * 8 + 4);
          const uint4 lo = make_uint4(__byte_perm(u.x, u.y, 0x5410), __byte_perm(u.z, u.w, 0x5410), __byte_perm(v.x, v.y, 0x5410), __byte_perm(v.z, v.w, 0x5410));
          const uint4 hi = make_uint4(__byte_perm(u.x, u.y, 0x7632), __byte_perm(u.z, u.w, 0x7632), __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x7632));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint4 o = k ? hi : lo;
            if (t + k >= jend || n >= p.N) continue;
            __nv_bfloat16* dst = p.out + (long long)(t + k) * p.ldo + n;
            if (n + 8 <= p.N) {
              *reinterpret_cast<uint4*>(dst) = o;
            } else {
              const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (n + e < p.N) reinterpret_cast<unsigned short*>(dst)[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair_arrive(pair_map(&tmem_empty[acc], even));
      acc ^= 1;
    }
    __syncwarp();
  }

  if (*abort_flag && rank == 0 && threadIdx.x == 0)    // copies still on their way to either CTA arrive before the pair leaves
    for (int s = 0; s < min(kI8PairStages, loaded); ++s) mbar_wait(&full_bar[s], (uint32_t)((loaded - 1 - s) / kI8PairStages) & 1u, nullptr);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                      // nothing of this pair is on its way to a CTA that has left; the parts' sums are there
  if (p.parts > 1) {
    const int j0 = first % tiles_b * p.bn;
    if (__syncthreads_or(*abort_flag) == 0)
      int8_join<kI8PairMaxParts, 2>(p, reinterpret_cast<const int*>(smem), scales, part, (uint32_t)rank, 2, (2 * (first / tiles_b) + rank) * kI8BM, j0, min(p.bn, p.T - j0));
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    pair_tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFnI8)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                    const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFnI8 encode_fn_i8() {
  static EncodeTiledFnI8 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
    return reinterpret_cast<EncodeTiledFnI8>(f);
  }();
  return fn;
}

// Rows of K bytes, `box_rows` of them by one stage's K a copy; zeros behind the last byte of a row and the last row.
static int make_tmap_i8(CUtensorMap* out, const void* base, uint64_t rows, uint64_t K, uint64_t row_bytes, uint32_t box_rows) {
  EncodeTiledFnI8 fn = encode_fn_i8();
  if (fn == nullptr) return -1;
  cuuint64_t dims[2] = {K, rows};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {(cuuint32_t)kI8BK, box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -(int)r - 100;
}

struct Int8Plan {
  int pairs, bn, stages, parts, tmem_cols, smem;      // pairs: of CTAs that stay, 0: single ones
};
static int int8_up(int a, int b) { return (a - 1) / b + 1; }      // of a >= 1, where a + b may pass 31 bits

// By single CTAs: where there are more of them than SMs, or clusters, which leave SMs empty, the ring of small tiles takes half of an SM's shared memory, so
// that two share an SM; else all of it.
static Int8Plan int8_single_plan(int T, int N, int K, int bn, int parts, int num_sms) {
  Int8Plan w{};
  w.bn = bn;
  w.parts = parts;
  const int stage = kI8ABytes + w.bn * kI8BK;
  const bool share = w.bn <= 64 && (parts > 1 || (long long)int8_up(N, kI8BM) * int8_up(T, bn) > num_sms);
  const int room = share ? 108 * 1024 : 216 * 1024, most = int8_up(int8_up(K, kI8BK), w.parts);
  w.stages = room / stage < kI8MaxStages ? room / stage : kI8MaxStages;
  if (w.stages > most) w.stages = most > 4 ? most : 4;
  w.tmem_cols = 32;
  while (w.tmem_cols < w.bn) w.tmem_cols *= 2;
  w.smem = w.stages * stage + (int)sizeof(Int8Scales) + (2 * kI8MaxStages + 1) * 8 + 16 + 1024;
  return w;
}

// What a plan costs, in ns.  A CTA's time is that of its operands' way in from L2 (112 bytes a nanosecond, 83 where all SMs work in pairs; a second CTA on an SM
// adds three eighths) and of its tokens' results; waves of CTAs add a start, parts a join; and the weights come from HBM meanwhile, and all operands through L2: the fourth powers of both
// times add up, so that the smaller one counts where they are near.  The constants are fitted to 7000 plans of 209 shapes (1 to 3900 rows, 144 to 28672 features,
// K 159 to 14336): the plan of least cost is 2 % slower than the quickest one on average, over 10 % in five shapes, at worst 30 % (7.7 us where 5.9 are possible).  On 1892 plans
// of 100 shapes, 64 of them drawn anew: 1.7 % on average, over 10 % in five, at worst 18 % (27 rows of 1034 x 6921).
static double int8_beside(double t, double hbm) {
  const double a = t * t, b = hbm * hbm;
  return sqrt(sqrt(a * a + b * b));
}
static double int8_single_cost(int T, int N, int K, const Int8Plan& w, int num_sms) {
  const int blocks = int8_up(int8_up(K, kI8BK), w.parts), live = w.bn < T ? w.bn : T;
  int fit = 233472 / (w.smem + 1024);                                     // CTAs an SM
  if (fit > 4) fit = 4;
  const long long ctas = (long long)int8_up(N, kI8BM) * int8_up(T, w.bn) * w.parts;
  long long slots = (long long)(num_sms - (w.parts == 1 ? 0 : w.parts == 2 ? 2 : w.parts == 8 ? 18 : 16)) * fit;      // (clusters leave some SMs empty)
  if (slots < 1) slots = 1;
  const long long waves = (ctas + slots - 1) / slots;
  long long together = (ctas + num_sms - 1) / num_sms;
  if (together > fit) together = fit;
  const double fill = blocks * (double)(kI8ABytes + kI8BK * w.bn) * (1 + 0.38 * (double)(together - 1)) / 111.7;
  const double t = 1230.0 + (double)waves * (fill + 1639.0 + 15.7 * live * (double)together) + (w.parts > 1 ? 685.0 + 2.5 * live : 0.0);
  const double hbm = ((double)N * K + (double)T * K) / 4853.0, l2 = (double)ctas * blocks * (kI8ABytes + kI8BK * w.bn) / 18590.0;
  return int8_beside(t, 2869.0 + (hbm > l2 ? hbm : l2));
}
static double int8_pair_cost(int T, int N, int K, int bn, int parts, int clusters) {
  const int blocks = int8_up(int8_up(K, kI8BK), parts), live = bn < T ? bn : T;
  const long long tiles = (long long)int8_up(N, 2 * kI8BM) * int8_up(T, bn), waves = (tiles + clusters - 1) / clusters;
  const double in = (kI8ABytes + kI8BK / 2 * bn) / 83.0, mma = 1.29 * bn;
  const double t = 2007.0 + (double)waves * (blocks * (in > mma ? in : mma) + 1008.0) + 20.1 * live + (parts > 1 ? 633.0 + 0.8 * live : 0.0);
  return int8_beside(t, 3015.0 + ((double)N * K + (double)T * K) / 4853.0);
}

// clusters[parts]: clusters of `parts` pairs that run at the same time.
static Int8Plan int8_plan(int T, int N, int K, int num_sms, const int* clusters) {
  Int8Plan best{};
  double least = 1e30;
  const int kblocks = int8_up(K, kI8BK);
  for (int most = 256; most >= 16; most -= most > 64 ? 32 : 16) {
    const int tiles = int8_up(T, most);
    if (most < 256 && tiles == int8_up(T, most + (most >= 64 ? 32 : 16))) continue;      // (the same tiles, evened out)
    if (most < 256 && tiles > 64) break;
    const int bn = int8_up(int8_up(T, tiles), 16) * 16, bn2 = int8_up(bn, 32) * 32;
    for (int parts : {1, 2, 3, 4, 8}) {
      if (parts > kblocks) break;
      // (three, whose CTAs would have an SM and half its shared memory each: 64 rows of 6144 features 10.9 us, by four 9.1; two an SM, one row of 11008: 9.7, by two 11.4)
      if (parts == 3 && (long long)int8_up(N, kI8BM) * int8_up(T, bn) * parts <= num_sms) continue;
      const Int8Plan w = int8_single_plan(T, N, K, bn, parts, num_sms);
      const double c = int8_single_cost(T, N, K, w, num_sms);
      if (c < least) { least = c; best = w; }
    }
    for (int parts = 1; T > 32 && bn2 <= 256 && parts <= kI8PairMaxParts && parts <= kblocks; ++parts) {
      if (clusters[parts] < 1 || (parts > 1 && (long long)int8_up(N, 2 * kI8BM) * int8_up(T, bn2) > clusters[parts])) break;
      const double c = int8_pair_cost(T, N, K, bn2, parts, clusters[parts]);
      if (c < least) {
        least = c;
        best = Int8Plan{clusters[1], bn2, 0, parts, 0, kI8PairSmem};
      }
    }
  }
  return best;
}

// Tiles of a product; the kernels count them in 32 bits, with a grid's more.
static long long int8_tiles(int T, int N, const Int8Plan& w) { return (long long)int8_up(N, w.pairs ? 2 * kI8BM : kI8BM) * int8_up(T, w.bn); }

// Clusters of `parts` pairs that run at the same time on `dev`, the current device (none of a size that no part of it holds), or a query's negative error, which the
// next call makes again.
static int int8_clusters(int parts, int dev) {
  static int known[64][kI8PairMaxParts + 1] = {{0}};
  int n = 0;
  if (known[dev][parts] != 0) return known[dev][parts] - 1;
  cudaError_t e = cudaFuncSetAttribute(gemm_int8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kI8PairSmem);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2u * (unsigned)parts);
    cfg.blockDim = dim3(kI8PairThreads);
    cfg.dynamicSmemBytes = kI8PairSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2u * (unsigned)parts; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&n, gemm_int8_pair_kernel, &cfg);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return -(int)e;
  }
  known[dev][parts] = n + 1;
  return n;
}

}  // namespace lx

extern "C" {

int lx_gemm_int8_max_k() { return (1 << 17) - 1; }

// The plan that a product takes where `clusters` (of 1, 2, 3, 4 pairs) run at the same time: out[0] pairs of CTAs (0: single ones), out[1] tokens a tile,
// out[2] CTAs or pairs that share a tile's K, out[3] stages of a single CTA's ring.
int lx_gemm_int8_plan(int T, int N, int K, int num_sms, const int* clusters, int* out) {
  using namespace lx;
  if (T <= 0 || N <= 0 || K <= 0 || K > lx_gemm_int8_max_k() || T > kI8Most || N > kI8Most) return -1000;
  const int fit[kI8PairMaxParts + 1] = {0, clusters[0], clusters[1], clusters[2], clusters[3]};
  const Int8Plan w = int8_plan(T, N, K, num_sms, fit);
  if (int8_tiles(T, N, w) > kI8Most) return -1001;
  out[0] = w.pairs; out[1] = w.bn; out[2] = w.parts; out[3] = w.stages;
  return 0;
}

int lx_gemm_int8_clusters(int parts) {
  int dev = 0;
  if (parts < 1 || parts > lx::kI8PairMaxParts || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  return lx::int8_clusters(parts, dev);
}

// Arguments in one block of 8-byte fields: a call by ctypes pays for each argument of its own (17 of them 2.4 us, a packed block 0.6).
struct LxGemmInt8Args {
  const void* xq;             // [T, K] int8, rows ldq bytes apart (multiples of 16)
  long long ldq;
  const float* xs;            // [T]
  const void* wq;             // [N, K] int8, rows ldw bytes apart
  long long ldw;
  const float* ws;            // [N]
  const void* bias;           // [N] bf16 or null
  void* out;                  // [T, N] bf16
  long long ldo, T, N, K;
  long long w_const;          // the kernel in front on the stream does not write wq
  int* status;
  long long num_sms;
  long long force;            // 0, or 1 + pairs + 2 * (parts | bn << 8): a plan to measure
  void* stream;
};
int lx_gemm_int8_bytes() { return (int)sizeof(LxGemmInt8Args); }

// out = xq wq^T * ws[n] * xs[t] + bias[n].
int lx_gemm_int8(const char* args) {
  using namespace lx;
  LxGemmInt8Args a;
  memcpy(&a, args, sizeof(a));
  if (a.T <= 0 || a.N <= 0) return 0;
  if (a.K <= 0 || a.K > lx_gemm_int8_max_k() || a.ldq % 16 != 0 || a.ldw % 16 != 0 || a.T > kI8Most || a.N > kI8Most) return -1000;
  const int T = (int)a.T, N = (int)a.N, K = (int)a.K, num_sms = (int)a.num_sms;
  const long long force = a.force;
  int dev = 0, clusters[kI8PairMaxParts + 1] = {0};
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  for (int parts = 1; parts <= kI8PairMaxParts; ++parts) {
    const int n = int8_clusters(parts, dev);
    if (n < 0) return n;
    clusters[parts] = pairs_on(num_sms / parts, n);
  }
  Int8Plan w;
  if (force) {
    const int pairs = (int)((force - 1) & 1), parts = (int)(((force - 1) >> 1) & 255), bn = (int)((force - 1) >> 9);
    if (bn < 16 || bn > 256 || bn % (pairs ? 32 : 16) != 0 || parts < 1 || parts > (pairs ? kI8PairMaxParts : kI8MaxParts) || parts > int8_up(K, kI8BK) ||
        (pairs && clusters[parts] < 1))
      return -1004;
    w = pairs ? Int8Plan{clusters[1], bn, 0, parts, 0, kI8PairSmem} : int8_single_plan(T, N, K, bn, parts, num_sms);
  } else {
    // a plan takes some microseconds to choose and goes by sizes alone: the last ones of a thread are kept
    struct Known { int T, N, K, sms, dev; Int8Plan w; };
    static thread_local Known known[64] = {};
    Known& k = known[((unsigned)T * 31u + (unsigned)N * 7u + (unsigned)K) % 64u];
    if (k.T != T || k.N != N || k.K != K || k.sms != num_sms || k.dev != dev) k = Known{T, N, K, num_sms, dev, int8_plan(T, N, K, num_sms, clusters)};
    w = k.w;
  }
  const long long tiles = int8_tiles(T, N, w);
  const long long ctas = !w.pairs ? tiles * w.parts : 2 * (w.parts > 1 ? tiles * w.parts : tiles < w.pairs ? tiles : w.pairs);
  if (tiles > kI8Most || ctas > 0x7fffffffll) return -1001;
  Int8GemmParams p{};
  p.N = N; p.T = T; p.K = K;
  p.bn = w.bn; p.stages = w.stages; p.parts = w.parts; p.tmem_cols = w.tmem_cols;
  p.reuse = T > w.bn;
  p.xs = a.xs; p.ws = a.ws;
  p.bias = reinterpret_cast<const __nv_bfloat16*>(a.bias);
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out); p.ldo = a.ldo;
  const int wide = w.pairs && w.parts == 1 ? 8 : 4;      // values that a thread stores at once
  p.wide = reinterpret_cast<uintptr_t>(a.out) % (2 * wide) == 0 && a.ldo % wide == 0;
  p.status = a.status;
  p.w_const = (int)a.w_const;
  CUtensorMap tw, tx;
  if (make_tmap_i8(&tw, a.wq, N, K, a.ldw, kI8BM)) return -1002;
  if (make_tmap_i8(&tx, a.xq, T, K, a.ldq, w.pairs ? w.bn / 2 : w.bn)) return -1003;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a.stream);
  if (w.pairs) {
    launch_pdl_cluster(gemm_int8_pair_kernel, dim3((unsigned)ctas), dim3(kI8PairThreads), dim3(2u * (unsigned)w.parts), (size_t)w.smem, stream, tw, tx, p);
    return -(int)cudaGetLastError();
  }
  static bool set[64] = {false};
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 222 * 1024);
    if (e != cudaSuccess) return -(int)e;
    set[dev] = true;
  }
  launch_pdl_cluster(gemm_int8_kernel, dim3((unsigned)ctas), dim3(w.bn <= 16 ? kI8Threads / 2 : kI8Threads), dim3((unsigned)w.parts), (size_t)w.smem, stream, tw, tx, p);
  return -(int)cudaGetLastError();
}

}  // extern "C"
