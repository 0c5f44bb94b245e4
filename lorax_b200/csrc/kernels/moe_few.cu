// A whole mixture-of-experts layer for a few tokens (T <= 16): every byte of the experts that the tokens reach is read once, by all SMs at
// the HBM's rate, and nothing else of size is moved.
//
//   z[t, e] = x_t . Wr_e; the k largest z of a token (the lower expert on ties); w[t, j] = exp(z_j - z_max) over their sum (or over the sum of
//   all experts), times a constant
//   up      h[t, j, i] = w[t, j] act(G_e[i] . x_t) (U_e[i] . x_t)    for the experts e = e(t, j) that this rank owns
//   down    out[t, n] = sum_j D_e[n] . h[t, j]
//
// Both products are streams of weights against at most 16 columns.  A thread of a CTA keeps a ring of shared memory filled by TMA, some 100 KB of it
// on their way.  A box is 64 of K x some rows x up to 16 times 64 of K further on: the tensor map takes a row's blocks of 64 as a dimension of
// their own, so that one copy brings 16 to 32 KB (bulk copies of one row's 1 to 2 KB each took 50 ns apiece: 5.0 and 3.2 TB/s; 16-byte loads
// into registers, 96 KB in flight, 5.4 and 4.1).  The tokens' side of a stage travels in it, a copy a token: loaded by the math warps it came through
// the same queues as the weights, 2 to 4 us behind its request.  Eight warps multiply what has arrived by mma.sync: the weights are the A operand
// (16 rows x 16 of K), read 16 bytes a lane in the order of K in which they lie (the other operand is read in the same order, so the sum is
// the same); tokens stand in the columns, those that an expert does not serve as zeros.  What is left of K behind its last 64 is loaded directly.
//   up:   the rows of all reached experts, eight features of gate and up to a tile, are dealt evenly to the CTAs; the warps split K and sum
//         their parts through shared memory
//   down: the rows of the output are dealt to the CTAs; K runs over the reached experts' features one expert behind the other, so the sum
//         over a token's experts forms in the accumulators (their weights are in h), in the order of the experts' numbers
// h is held as two bf16 terms, value and remainder, which take two MMAs: it is as exact as the fp32 sums, and the tensor cores have room.  Its
// rows lie in the order of the experts, the tokens of one behind the other.
// Every CTA chooses the experts for itself from the logits; no CTA waits for another.
#include <type_traits>

#include "common.cuh"

namespace lx {

constexpr int kFewTokens = 16;
constexpr int kFewExperts = 256;
constexpr int kFewTop = 32;
constexpr int kFewMath = 8;                // warps that multiply; one more fills the ring
constexpr int kFewWarps = kFewMath + 1;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kFewRowTiles = 4;            // tiles of 16 rows of a CTA (down)
constexpr int kFewUpSteps = 4;             // steps of 32 of K of a stage and a math warp, at most (up)
constexpr int kFewMaxStages = 16;
constexpr int kFewInFlight = 104 * 1024;   // bytes of weights on their way: more of them only wait longer (96 and 192 KB: 6.4 TB/s both)
constexpr int kFewSums = 2;                // tiles whose sums over the math warps may wait (up)
constexpr int kFewSmem = 232448 - 14 * 1024;      // (the rest: what is static)

enum FewAct : int { kFewSilu = 0, kFewGelu = 1, kFewGeluTanh = 2, kFewRelu = 3, kFewRelu2 = 4 };

struct MoeFewParams {
  const __nv_bfloat16* x;      // [T, H]
  long long ldx;
  const __nv_bfloat16* wr;     // [E, H]
  long long ldr;
  const float* logits;         // [T, E], or null: the up kernel forms them itself
  const __nv_bfloat16* w13;    // [e_local, 2 I, H]: gate rows, then up rows
  const __nv_bfloat16* w2;     // [e_local, H, I]
  int* ids;                    // [T, k]: the chosen experts, for the second kernel
  __nv_bfloat16* h;            // two planes of [T k, I], in the order of the experts
  __nv_bfloat16* out;          // [T, H]
  long long ldo;
  int* status;
  int T, E, k, e0, e_local, H, I, act, renorm;
  float scale;
  // blocks of 64 of K of a stage of the up and the down kernel; rows of a stage of the latter
  int up_blocks, down_blocks, down_rows;
};

LX_DEVICE void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 of K: rows p and q of A (eight elements a lane), column b of B.
LX_DEVICE void few_mma32(float (&d)[4], const uint4& p, const uint4& q, const uint4& b) {
  few_mma(d, p.x, q.x, p.y, q.y, b.x, b.y);
  few_mma(d, p.z, q.z, p.w, q.w, b.z, b.w);
}
// Eight elements of K behind the last block, or zeros.
LX_DEVICE uint4 few_load(const __nv_bfloat16* p, bool valid) {
  uint4 v;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t"
      "}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)valid));
  return v;
}

LX_DEVICE float few_act(float x, int act) {
  switch (act) {
    case kFewSilu: return x / (1.f + expf(-x));
    case kFewGelu: return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    case kFewGeluTanh: return 0.5f * x * (1.f + tanhf(0.79788456080286536f * (x + 0.044715f * x * x * x)));
    case kFewRelu: return fmaxf(x, 0.f);
    default: { const float r = fmaxf(x, 0.f); return r * r; }
  }
}

// ------------------------------------------------------------------------------------------------ choice of experts, and who is reached
struct FewPlan {
  float w[kFewTokens * kFewTop];
  int ids[kFewTokens * kFewTop];
  uint32_t mask[kFewExperts];                   // tokens of a local expert
  uint8_t place[kFewTokens][kFewExperts];       // which of its choices a local expert is for a token
  short list[kFewExperts];                      // local experts that have a token, ascending
  short base[kFewExperts];                      // the first row of h of each of those
  int warps[kFewWarps];
  int reached, most;                            // number of those, and the most tokens of one
};

// z[t, e] for all experts, by every CTA for itself: the router's rows stand where the up kernel has its tiles.
template <int NT>
LX_DEVICE void few_route(float* z, float4* red, const MoeFewParams& p) {
  constexpr int kBatch = 8 / NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  const int steps = (p.H + 31) / 32, tiles = (p.E + 15) / 16;
  for (int i = 0; i < tiles; ++i) {
    float acc[NT][4];
#pragma unroll
    for (int m = 0; m < NT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
    for (int s0 = warp; s0 < steps; s0 += kFewWarps * kBatch) {
      uint4 a[kBatch][2], b[kBatch][NT];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = (s0 + j * kFewWarps) * 32 + c8, e = i * 16 + g;
        const bool ok = k < p.H;
        a[j][0] = few_load(p.wr + e * p.ldr + k, ok && e < p.E);
        a[j][1] = few_load(p.wr + (e + 8) * p.ldr + k, ok && e + 8 < p.E);
#pragma unroll
        for (int m = 0; m < NT; ++m) b[j][m] = few_load(p.x + (m * 8 + g) * p.ldx + k, ok && m * 8 + g < p.T);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int m = 0; m < NT; ++m) few_mma32(acc[m], a[j][0], a[j][1], b[j][m]);
    }
#pragma unroll
    for (int m = 0; m < NT; ++m) red[((warp * tiles + i) * NT + m) * 32 + lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
  }
  __syncthreads();
  for (int q = tid; q < tiles * NT * 32; q += kFewThreads) {
    const int i = q / (NT * 32), m = q / 32 % NT, l = q & 31;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float4 part = red[((w * tiles + i) * NT + m) * 32 + l];
      v.x += part.x; v.y += part.y; v.z += part.z; v.w += part.w;
    }
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const int t = m * 8 + (l & 3) * 2 + (o & 1), e = i * 16 + (l >> 2) + (o >> 1) * 8;
      if (t < p.T && e < p.E) z[t * p.E + e] = o == 0 ? v.x : o == 1 ? v.y : o == 2 ? v.z : v.w;
    }
  }
  __syncthreads();
}

// One warp per token.  A NaN orders as -inf (its weight is NaN all the same); no expert is chosen twice.
LX_DEVICE void few_select(FewPlan& plan, const float* logits, const MoeFewParams& p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kPer = kFewExperts / 32;
  for (int t = warp; t < p.T; t += kFewWarps) {
    const float* row = logits + t * p.E;
    float z[kPer];
    uint32_t taken = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      z[i] = e < p.E ? row[e] : 0.f;
      if (e >= p.E) taken |= 1u << i;
    }
    float all = 0.f, top = 0.f, own = 0.f;
    int id = 0;
    for (int j = 0; j < p.k; ++j) {
      float bv = -INFINITY;
      int bi = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float v = z[i] == z[i] ? z[i] : -INFINITY;
        if (!((taken >> i) & 1) && (bi == 0x7fffffff || v > bv)) { bv = v; bi = lane + 32 * i; }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        if (oi != 0x7fffffff && (bi == 0x7fffffff || ov > bv || (ov == bv && oi < bi))) { bv = ov; bi = oi; }
      }
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == (bi >> 5)) {
          v = z[i];
          if (lane == (bi & 31)) taken |= 1u << i;
        }
      v = __shfl_sync(0xffffffffu, v, bi & 31);
      if (j == 0) top = v;
      if (lane == j) { id = bi; own = expf(v - top); }
    }
    if (p.renorm) {
      all = warp_sum(lane < p.k ? own : 0.f);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < p.E) all += expf(z[i] - top);
      all = warp_sum(all);
    }
    if (lane < p.k) {
      plan.ids[t * p.k + lane] = id;
      plan.w[t * p.k + lane] = own / all * p.scale;
    }
  }
}

// From plan.ids: which tokens every local expert serves, and the experts that serve any.
LX_DEVICE void few_reached(FewPlan& plan, const MoeFewParams& p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  static_assert(kFewThreads >= kFewExperts, "a thread for every expert");
  if (threadIdx.x < kFewExperts) plan.mask[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.k; i += kFewThreads) {
    const int e = plan.ids[i] - p.e0, t = i / p.k;
    if (e >= 0 && e < p.e_local) {
      atomicOr(&plan.mask[e], 1u << t);
      plan.place[t][e] = (uint8_t)(i - t * p.k);
    }
  }
  __syncthreads();
  const bool has = threadIdx.x < kFewExperts && plan.mask[threadIdx.x] != 0;
  const uint32_t votes = __ballot_sync(0xffffffffu, has);
  if (lane == 0) plan.warps[warp] = __popc(votes);
  __syncthreads();
  int at = __popc(votes & ((1u << lane) - 1)), all = 0;
#pragma unroll
  for (int i = 0; i < kFewWarps; ++i) {
    if (i < warp) at += plan.warps[i];
    all += plan.warps[i];
  }
  if (has) plan.list[at] = (short)threadIdx.x;
  if (threadIdx.x == 0) plan.reached = all;
  __syncthreads();
  if (warp == 0) {
    int sum = 0, most = 0;
    for (int d0 = 0; d0 < all; d0 += 32) {
      const int n = d0 + lane < all ? __popc(plan.mask[plan.list[d0 + lane]]) : 0;
      most = max(most, n);
      int v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (d0 + lane < all) plan.base[d0 + lane] = (short)(sum + v - n);
      sum += __shfl_sync(0xffffffffu, v, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) plan.most = most;
  }
  __syncthreads();
}

// Row of h of token t (one of `mask`) within its expert's.
LX_DEVICE int few_slot(uint32_t mask, int t) { return __popc(mask & ((1u << t) - 1)); }
// The i-th token of `mask`.
LX_DEVICE int few_token(uint32_t mask, int i) { return __fns(mask, 0, i + 1); }

// ------------------------------------------------------------------------------------------------ the ring
// Stages of shared memory, filled by one warp and read by the math warps.  Waits are bounded: one that runs out is reported, the filling warp stops (and
// waits for its copies), and the math warps go on without waiting (they meet at barriers), so that the launch ends.
struct FewRing {
  uint64_t full[kFewMaxStages], empty[kFewMaxStages];
  uint64_t sums[kFewSums], read[kFewSums];      // the math warps' sums of a tile: written, read
  int stop;
};

LX_DEVICE void few_ring_init(FewRing& r) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewMaxStages; ++s) { mbar_init(&r.full[s], 1); mbar_init(&r.empty[s], kFewMath); }
    for (int s = 0; s < kFewSums; ++s) { mbar_init(&r.sums[s], kFewMath); mbar_init(&r.read[s], 1); }
    r.stop = 0;
    mbar_fence_init();
  }
}

// Stages of `bytes` each, `weights` of them weights: as many as are worth having on their way.
LX_DEVICE int few_stages(int ring, int bytes, int weights) { return min(min(max(3, kFewInFlight / weights), ring / bytes), kFewMaxStages); }

struct FewCursor {
  int stage = 0;
  uint32_t phase = 0;
  LX_DEVICE void next(int stages) {
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
};

// Filling thread: waits for the stage that comes next, then copy(stage's barrier) brings its `bytes`.
template <typename Copy>
LX_DEVICE bool few_fill(FewRing& r, FewCursor& at, int stages, uint32_t bytes, int* status, Copy&& copy) {
  if (!mbar_wait(&r.empty[at.stage], at.phase ^ 1, &r.stop)) {
    report_status(status, kTimeoutEmptyBarrier, (int)blockIdx.x);
    r.stop = 1;
    return false;
  }
  mbar_expect_tx(&r.full[at.stage], bytes);
  copy(&r.full[at.stage]);
  at.next(stages);
  return true;
}

// Filling warp, after the last of its `filled` stages: the copies on their way are waited for.
LX_DEVICE void few_drain(FewRing& r, FewCursor at, int stages, long long filled) {
  for (int i = 0; i < stages && i < filled; ++i) {
    if (--at.stage < 0) { at.stage = stages - 1; at.phase ^= 1; }
    mbar_wait(&r.full[at.stage], at.phase, nullptr);
  }
}

LX_DEVICE void few_await(FewRing& r, uint64_t* bar, uint32_t phase, bool& ok, int* status) {
  if (ok && !mbar_wait(bar, phase, &r.stop)) {
    if ((threadIdx.x & 31) == 0) report_status(status, kTimeoutFullBarrier, (int)blockIdx.x);
    r.stop = 1;
    ok = false;
  }
}

LX_DEVICE void few_release(FewRing& r, FewCursor& at, int stages) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&r.empty[at.stage]);
  at.next(stages);
}

LX_DEVICE void few_math_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kFewMath) : "memory"); }

// Where a lane's eight elements of the weights of a stage lie: row `r` of `rows` (an even number), step `s` of 32 of K, elements c8 .. c8 + 7 of it.
// Blocks of 64 of K lie one behind the other, rows of 128 bytes in each, their 16-byte chunks permuted by the low bits of the row's place
// (128-byte swizzle).  The next step of the same warp, eight further on, lies 512 rows bytes further: four blocks are a multiple of eight rows.
LX_DEVICE int few_place(int rows, int r, int s, int c8) {
  const int line = (s >> 1) * rows + r;
  return line * 128 + ((((s & 1) * 4 + (c8 >> 3)) ^ (line & 7)) << 4);
}
// The row of a tile that lane group g takes: neighbouring groups take rows four apart, whose chunks the permutation sends to other banks.
LX_DEVICE int few_lane_row(int g) { return (g >> 1) | ((g & 1) << 2); }
LX_DEVICE uint4 few_row(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
constexpr int kFewZeros = kFewUpSteps * 512;      // what the lanes of a column without a token read instead of one

// ------------------------------------------------------------------------------------------------ up
// NT: columns of eight tokens.
template <int NT>
__global__ void __launch_bounds__(kFewThreads, 1) moe_few_up_kernel(const __grid_constant__ CUtensorMap weights, const __grid_constant__ CUtensorMap tokens,
                                                                    const __grid_constant__ MoeFewParams p) {
  __shared__ FewPlan plan;
  __shared__ FewRing ring;
  __shared__ __align__(16) uint8_t zeros[kFewZeros];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  few_ring_init(ring);
  for (int i = tid; i < kFewZeros / 4; i += kFewThreads) reinterpret_cast<uint32_t*>(zeros)[i] = 0;
  pdl_wait();
  pdl_trigger();
  const float* logits = p.logits;
  if (logits == nullptr) {
    float4* sums = reinterpret_cast<float4*>(smem);
    float* z = reinterpret_cast<float*>(sums + kFewWarps * ((p.E + 15) / 16) * NT * 32);
    few_route<NT>(z, sums, p);
    logits = z;
  }
  few_select(plan, logits, p);
  fence_proxy_async_smem();                    // (the ring lies where the sums and logits did)
  __syncthreads();
  few_reached(plan, p);
  if (blockIdx.x == 0)
    for (int i = tid; i < p.T * p.k; i += kFewThreads) p.ids[i] = plan.ids[i];
  // a stage: gate rows, up rows, then the expert's tokens
  const int units = p.I / 8, blocks = p.H / 64, chunks = (blocks + p.up_blocks - 1) / p.up_blocks, half = p.up_blocks * 1024;
  const int token = p.up_blocks * 128, stage_bytes = (2 * half + plan.most * token + 1023) & ~1023;
  const int stages = few_stages(kFewSmem - 1024 - kFewSums * kFewMath * NT * 32 * (int)sizeof(float4), stage_bytes, 2 * half);
  const long long all = (long long)plan.reached * units;
  const int u0 = (int)(all * blockIdx.x / gridDim.x), u1 = (int)(all * (blockIdx.x + 1) / gridDim.x);
  FewCursor at;
  if (warp == kFewMath) {
    if (lane == 0) {
      const uint64_t policy = policy_evict_first();
      long long filled = 0;
      bool ok = true;
      for (int u = u0; ok && u < u1; ++u) {
        const int d = u / units, c = (u - d * units) * 8, e = plan.list[d];
        const uint32_t mask = plan.mask[e], bytes = 2 * half + __popc(mask) * token;
        for (int ch = 0; ok && ch < chunks; ++ch, ++filled) {
          uint8_t* stage = smem + at.stage * stage_bytes;
          ok = few_fill(ring, at, stages, bytes, p.status, [&](uint64_t* bar) {
            tma_load_4d_hint(stage, &weights, bar, 0, c, ch * p.up_blocks, e, policy);
            tma_load_4d_hint(stage + half, &weights, bar, 0, p.I + c, ch * p.up_blocks, e, policy);
            uint8_t* to = stage + 2 * half;
            for (uint32_t m = mask; m != 0; m &= m - 1, to += token) tma_load_4d(to, &tokens, bar, 0, __ffs(m) - 1, ch * p.up_blocks, 0);
          });
        }
      }
      few_drain(ring, at, stages, filled);
    }
    return;
  }
  float4* red = reinterpret_cast<float4*>(smem + stages * stage_bytes);      // [kFewSums][math warps][NT][32 lanes]
  const int steps = 2 * blocks, per = 2 * p.up_blocks, place = few_place(8, few_lane_row(g), warp, c8), column = 2 * half + (warp * 32 + c8) * 2;
  const int rest = blocks * 64 + warp * 32 + c8;      // K of this lane behind the blocks
  bool ok = true;
  uint32_t sums_phase = 0;
  // A tile for an expert of up to 8 N tokens: they stand in the columns in their order.
  auto tile = [&](auto n, int u) {
    constexpr int N = decltype(n)::value;
    const int d = u / units, e = plan.list[d], col = (u - d * units) * 8 + few_lane_row(g), buf = (u - u0) % kFewSums;
    const uint32_t mask = plan.mask[e];
    const int served = __popc(mask);
    float acc[2][N][4];                        // (two chains of MMAs)
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int m = 0; m < N; ++m) acc[o][m][0] = acc[o][m][1] = acc[o][m][2] = acc[o][m][3] = 0.f;
    if (blocks * 64 + warp * 32 < p.H) {
      const __nv_bfloat16* w = p.w13 + ((long long)e * 2 * p.I + col) * p.H + rest;
      const uint4 gate = few_load(w, rest < p.H), up = few_load(w + (long long)p.I * p.H, rest < p.H);
#pragma unroll
      for (int m = 0; m < N; ++m) {
        const bool on = m * 8 + g < served;
        few_mma32(acc[0][m], gate, up, few_load(p.x + (on ? few_token(mask, m * 8 + g) * p.ldx : 0) + rest, on && rest < p.H));
      }
    }
    for (int ch = 0; ch < chunks; ++ch) {
      const uint32_t stage = smem_u32(smem) + at.stage * stage_bytes;
      uint32_t xt[N];
#pragma unroll
      for (int m = 0; m < N; ++m) xt[m] = m * 8 + g < served ? stage + column + (m * 8 + g) * token : smem_u32(zeros);
      few_await(ring, &ring.full[at.stage], at.phase, ok, p.status);
#pragma unroll
      for (int j = 0; j < kFewUpSteps; ++j) {
        const int s = j * kFewMath + warp;
        if (s < per && ch * per + s < steps) {
          const uint4 gate = few_row(stage + place + j * 4096), up = few_row(stage + half + place + j * 4096);
#pragma unroll
          for (int m = 0; m < N; ++m) few_mma32(acc[j & 1][m], gate, up, few_row(xt[m] + j * 512));
        }
      }
      few_release(ring, at, stages);
    }
    few_await(ring, &ring.read[buf], sums_phase ^ 1, ok, p.status);
    float4* part = red + buf * kFewMath * NT * 32;
#pragma unroll
    for (int m = 0; m < N; ++m)
      part[(warp * N + m) * 32 + lane] = make_float4(acc[0][m][0] + acc[1][m][0], acc[0][m][1] + acc[1][m][1], acc[0][m][2] + acc[1][m][2], acc[0][m][3] + acc[1][m][3]);
    __syncwarp();
    if (lane == 0) mbar_arrive(&ring.sums[buf]);
    if ((u - u0) % kFewMath == warp) {         // one warp a tile, in turn, sums up the warps' parts
      few_await(ring, &ring.sums[buf], sums_phase, ok, p.status);
#pragma unroll
      for (int m = 0; m < N; ++m) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFewMath; ++w) {
          const float4 a = part[(w * N + m) * 32 + lane];
          v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
        }
#pragma unroll
        for (int o = 0; o < 2; ++o) {          // (gate and up of the lane's column, tokens 2 (lane % 4) and the next)
          const int i = m * 8 + (lane & 3) * 2 + o;
          if (i >= served) continue;
          const int t = few_token(mask, i);
          const float h = few_act(o ? v.y : v.x, p.act) * (o ? v.w : v.z) * plan.w[t * p.k + plan.place[t][e]];
          const __nv_bfloat16 hi = __float2bfloat16(h);
          const float back = __bfloat162float(hi);
          const long long row = plan.base[d] + i;
          p.h[row * p.I + col] = hi;
          p.h[(row + p.T * p.k) * p.I + col] = __float2bfloat16(fabsf(back) < INFINITY ? h - back : 0.f);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring.read[buf]);
    }
    if (buf == kFewSums - 1) sums_phase ^= 1;
  };
  for (int u = u0; u < u1; ++u) {
    if (NT == 1 || __popc(plan.mask[plan.list[u / units]]) <= 8) tile(std::integral_constant<int, 1>{}, u);
    else tile(std::integral_constant<int, NT>{}, u);
  }
}

// ------------------------------------------------------------------------------------------------ down
// MT: tiles of 16 rows; steps of 32 of K of a stage and a math warp: as many as make stages of up to 32 KB.
template <int MT>
constexpr int few_down_steps() { return MT == 1 ? 4 : MT == 2 ? 2 : 1; }

template <int MT, int NT>
__global__ void __launch_bounds__(kFewThreads, 1) moe_few_down_kernel(const __grid_constant__ CUtensorMap weights, const __grid_constant__ CUtensorMap tokens,
                                                                      const __grid_constant__ MoeFewParams p) {
  __shared__ FewPlan plan;
  __shared__ FewRing ring;
  __shared__ __align__(16) uint8_t zeros[kFewZeros];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  few_ring_init(ring);
  for (int i = tid; i < kFewZeros / 4; i += kFewThreads) reinterpret_cast<uint32_t*>(zeros)[i] = 0;
  pdl_wait();
  pdl_trigger();
  for (int i = tid; i < p.T * p.k; i += kFewThreads) plan.ids[i] = p.ids[i];
  __syncthreads();
  few_reached(plan, p);
  // a stage: rows of the weights, then value and remainder of the expert's tokens
  const int blocks = p.I / 64, chunks = (blocks + p.down_blocks - 1) / p.down_blocks, reached = plan.reached;
  const int rows = p.down_rows, bytes = p.down_blocks * rows * 128, wide = (bytes + 1023) & ~1023, plane = p.down_blocks * 128;
  const int stage_bytes = (wide + plan.most * 2 * plane + 1023) & ~1023;
  const int stages = few_stages(kFewSmem - 1024 - kFewMath * MT * NT * 32 * (int)sizeof(float4), stage_bytes, wide);
  FewCursor at;
  if (warp == kFewMath) {
    if (lane == 0) {
      const uint64_t policy = policy_evict_first();
      long long filled = 0;
      bool ok = true;
      for (int r0 = blockIdx.x * rows; ok && r0 < p.H; r0 += gridDim.x * rows)
        for (int d = 0; ok && d < reached; ++d) {
          const int n = __popc(plan.mask[plan.list[d]]);
          for (int ch = 0; ok && ch < chunks; ++ch, ++filled) {
            uint8_t* stage = smem + at.stage * stage_bytes;
            ok = few_fill(ring, at, stages, bytes + n * 2 * plane, p.status, [&](uint64_t* bar) {
              tma_load_4d_hint(stage, &weights, bar, 0, r0, ch * p.down_blocks, plan.list[d], policy);
              for (int i = 0; i < n; ++i) tma_load_4d(stage + wide + i * 2 * plane, &tokens, bar, 0, plan.base[d] + i, ch * p.down_blocks, 0);
            });
          }
        }
      few_drain(ring, at, stages, filled);
    }
    return;
  }
  float4* red = reinterpret_cast<float4*>(smem + stages * stage_bytes);      // [math warps][MT][NT][32 lanes]
  constexpr int kSteps = few_down_steps<MT>();
  const int steps = 2 * blocks, per = 2 * p.down_blocks, column = wide + (warp * 32 + c8) * 2;
  int row[MT][2], place[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      row[m][o] = min(m * 16 + o * 8 + few_lane_row(g), rows - 1);      // rows past the last one are taken from it: nobody stores their sums
      place[m][o] = few_place(rows, row[m][o], warp, c8);
    }
  const int rest = blocks * 64 + warp * 32 + c8;      // K of this lane behind the blocks
  bool ok = true;
  for (int r0 = blockIdx.x * rows; r0 < p.H; r0 += gridDim.x * rows) {
    const int last = min(r0 + rows, p.H);
    float acc[2][MT][NT][4];                   // (of values and of remainders)
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[o][m][n][0] = acc[o][m][n][1] = acc[o][m][n][2] = acc[o][m][n][3] = 0.f;
    auto multiply = [&](const uint4& a0, const uint4& a1, const uint4 (&h)[NT][2], int m) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        few_mma32(acc[0][m][n], a0, a1, h[n][0]);
        few_mma32(acc[1][m][n], a0, a1, h[n][1]);
      }
    };
    for (int d = 0; d < reached; ++d) {
      const int e = plan.list[d];
      const uint32_t mask = plan.mask[e];
      int slot[NT];                            // where the lane's tokens lie in a stage
#pragma unroll
      for (int n = 0; n < NT; ++n) slot[n] = ((mask >> (n * 8 + g)) & 1) ? column + few_slot(mask, n * 8 + g) * 2 * plane : -1;
      for (int ch = 0; ch < chunks; ++ch) {
        const uint32_t stage = smem_u32(smem) + at.stage * stage_bytes;
        uint32_t ht[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          ht[n][0] = slot[n] >= 0 ? stage + slot[n] : smem_u32(zeros);
          ht[n][1] = slot[n] >= 0 ? ht[n][0] + plane : ht[n][0];
        }
        few_await(ring, &ring.full[at.stage], at.phase, ok, p.status);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const int s = j * kFewMath + warp;
          if (s < per && ch * per + s < steps) {
            uint4 h[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              h[n][0] = few_row(ht[n][0] + j * 512);
              h[n][1] = few_row(ht[n][1] + j * 512);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) multiply(few_row(stage + place[m][0] + j * 512 * rows), few_row(stage + place[m][1] + j * 512 * rows), h, m);
          }
        }
        few_release(ring, at, stages);
      }
      if (blocks * 64 + warp * 32 < p.I) {
        const bool in = rest < p.I;
        uint4 h[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int t = n * 8 + g;
          const bool on = in && ((mask >> t) & 1);
          const __nv_bfloat16* from = p.h + (long long)(on ? plan.base[d] + few_slot(mask, t) : 0) * p.I + rest;
          h[n][0] = few_load(from, on);
          h[n][1] = few_load(from + (long long)p.T * p.k * p.I, on);
        }
        const __nv_bfloat16* w = p.w2 + ((long long)e * p.H + r0) * p.I + rest;
#pragma unroll
        for (int m = 0; m < MT; ++m)
          multiply(few_load(w + (long long)row[m][0] * p.I, in && r0 + row[m][0] < p.H), few_load(w + (long long)row[m][1] * p.I, in && r0 + row[m][1] < p.H), h, m);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float(&hi)[4] = acc[0][m][n], (&lo)[4] = acc[1][m][n];
        red[((warp * MT + m) * NT + n) * 32 + lane] = make_float4(hi[0] + lo[0], hi[1] + lo[1], hi[2] + lo[2], hi[3] + lo[3]);
      }
    few_math_sync();
    for (int q = tid; q < MT * NT * 32; q += 32 * kFewMath) {
      const int m = q / (NT * 32), n = q / 32 % NT, l = q & 31;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewMath; ++w) {
        const float4 part = red[((w * MT + m) * NT + n) * 32 + l];
        v.x += part.x; v.y += part.y; v.z += part.z; v.w += part.w;
      }
#pragma unroll
      for (int o = 0; o < 4; ++o) {              // (the row of lane group l / 4 and 8 behind it, tokens 2 (l % 4) and the next)
        const int t = n * 8 + (l & 3) * 2 + (o & 1), r = m * 16 + (o >> 1) * 8 + few_lane_row(l >> 2);
        if (t < p.T && r < rows && r0 + r < last) p.out[(long long)t * p.ldo + r0 + r] = __float2bfloat16(o == 0 ? v.x : o == 1 ? v.y : o == 2 ? v.z : v.w);
      }
    }
    few_math_sync();
  }
}

// Matrices [outer, rows, K], rows `ld` and matrices `ldo` elements apart, as {64 of K, rows, blocks of 64, outer}; boxes of `box_rows` rows x
// `box_blocks` blocks x `box_outer`.  K behind the last whole block is left out; what a box has past the rows or blocks reads as zero.
static int few_tmap(CUtensorMap* out, const void* base, long long outer, long long rows, long long K, long long ld, long long ldo, int box_rows, int box_blocks,
                    int box_outer, bool swizzle) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return -4;
    encode = reinterpret_cast<Encode>(fn);
  }
  if (outer == 0 || K < 64) return 0;          // (no copy is made)
  const cuuint64_t dims[4] = {64, (cuuint64_t)rows, (cuuint64_t)(K / 64), (cuuint64_t)outer};
  const cuuint64_t strides[3] = {(cuuint64_t)ld * 2, 128, (cuuint64_t)ldo * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_blocks, (cuuint32_t)box_outer}, each[4] = {1, 1, 1, 1};
  return encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0 : -5;
}

// Blocks of a stage, of `all`: at most `most`, in equal parts.
static int few_blocks(int all, int most) {
  if (all <= 0) return 1;
  const int parts = (all + most - 1) / most;
  return (all + parts - 1) / parts;
}

template <typename K>
static int few_opt_in(K* kernel, bool (&set)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
    if (e != cudaSuccess) return -(int)e;
    set[dev] = true;
  }
  return 0;
}

template <int MT, int NT>
static int moe_few_down(MoeFewParams& p, int num_sms, cudaStream_t s) {
  static bool set[64] = {};
  if (const int rc = few_opt_in(moe_few_down_kernel<MT, NT>, set)) return rc;
  p.down_blocks = few_blocks(p.I / 64, few_down_steps<MT>() * kFewMath / 2);
  CUtensorMap map{}, tokens{};
  if (const int rc = few_tmap(&map, p.w2, p.e_local, p.H, p.I, p.I, (long long)p.H * p.I, p.down_rows, p.down_blocks, 1, true)) return rc;
  if (const int rc = few_tmap(&tokens, p.h, 2, (long long)p.T * p.k, p.I, p.I, (long long)p.T * p.k * p.I, 1, p.down_blocks, 2, false)) return rc;
  launch_pdl(moe_few_down_kernel<MT, NT>, dim3(num_sms), dim3(kFewThreads), kFewSmem, s, map, tokens, p);
  return -(int)cudaGetLastError();
}

template <int NT>
static int moe_few_launch(MoeFewParams& p, int num_sms, cudaStream_t s) {
  static bool set[64] = {};
  if (const int rc = few_opt_in(moe_few_up_kernel<NT>, set)) return rc;
  p.up_blocks = few_blocks(p.H / 64, kFewUpSteps * kFewMath / 2);
  CUtensorMap map{}, tokens{};
  if (const int rc = few_tmap(&map, p.w13, p.e_local, 2LL * p.I, p.H, p.H, 2LL * p.I * p.H, 8, p.up_blocks, 1, true)) return rc;
  if (const int rc = few_tmap(&tokens, p.x, 1, p.T, p.H, p.ldx, p.T * p.ldx, 1, p.up_blocks, 1, false)) return rc;
  launch_pdl(moe_few_up_kernel<NT>, dim3(num_sms), dim3(kFewThreads), kFewSmem, s, map, tokens, p);
  const int rows = ((p.H + num_sms - 1) / num_sms + 1) & ~1;
  p.down_rows = rows < 16 * kFewRowTiles ? rows : 16 * kFewRowTiles;
  if (rows <= 16) return moe_few_down<1, NT>(p, num_sms, s);
  if (rows <= 32) return moe_few_down<2, NT>(p, num_sms, s);
  if (rows <= 48) return moe_few_down<3, NT>(p, num_sms, s);
  return moe_few_down<kFewRowTiles, NT>(p, num_sms, s);
}

}  // namespace lx

extern "C" {

int lx_moe_few_max_tokens() { return lx::kFewTokens; }

int lx_moe_router_logits(const void* x, long long ldx, const void* wr, long long ldw, float* logits, int T, int E, int H, int* counts, int ncounts,
                         void* stream);

// `logits` [T, E], `ids` [T, k] and `h` [2, T k, I] are scratch of the call.
int lx_moe_few(const void* x, long long ldx, const void* wr, long long ldw, const void* w13, const void* w2, float* logits, int* ids, void* h, void* out, long long ldo, int T,
               int E, int k, int e0, int e_local, int H, int I, int act, int renorm, float scale, int* status, int num_sms, void* stream) {
  using namespace lx;
  if (T < 0 || T > kFewTokens || E <= 0 || E > kFewExperts || k <= 0 || k > kFewTop || k > E || e_local < 0 || e_local > kFewExperts || H <= 0 || H % 8 != 0 ||
      I <= 0 || I % 8 != 0 || act < 0 || act > kFewRelu2 || num_sms <= 0)
    return -1;
  for (const void* q : {x, wr, w13, w2, (const void*)h})
    if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return -2;
  if (ldx % 8 != 0 || ldw % 8 != 0) return -2;
  if (T == 0) return 0;
  const bool by_itself = getenv("FEW_ROUTE") ? atoi(getenv("FEW_ROUTE")) : E * (long long)H <= 65536;
  if (!by_itself)
    if (const int rc = lx_moe_router_logits(x, ldx, wr, ldw, logits, T, E, H, nullptr, 0, stream)) return rc;
  MoeFewParams p{};
  p.x = reinterpret_cast<const __nv_bfloat16*>(x); p.ldx = ldx; p.logits = by_itself ? nullptr : logits;
  p.wr = reinterpret_cast<const __nv_bfloat16*>(wr); p.ldr = ldw;
  p.w13 = reinterpret_cast<const __nv_bfloat16*>(w13); p.w2 = reinterpret_cast<const __nv_bfloat16*>(w2);
  p.ids = ids; p.h = reinterpret_cast<__nv_bfloat16*>(h); p.out = reinterpret_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.T = T; p.E = E; p.k = k; p.e0 = e0; p.e_local = e_local; p.H = H; p.I = I; p.act = act; p.renorm = renorm; p.scale = scale; p.status = status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return T <= 8 ? moe_few_launch<1>(p, num_sms, s) : moe_few_launch<2>(p, num_sms, s);
}

}  // extern "C"
