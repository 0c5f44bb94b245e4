// A whole mixture-of-experts layer for a few tokens (T <= 16): every byte of the experts that the tokens reach is read once, by all SMs at
// the HBM's rate, and nothing else of size is moved.
//
//   z[t, e] = x_t . Wr_e; the k largest z of a token (the lower expert on ties); w[t, j] = exp(z_j - z_max) over their sum (or over the sum of
//   all experts), times a constant
//   up      h[t, j, i] = w[t, j] act(G_e[i] . x_t) (U_e[i] . x_t)    for the experts e = e(t, j) that this rank owns
//   down    out[t, n] = sum_j D_e[n] . h[t, j]
//
// Both products are streams of weights against at most 16 columns.  A thread of a CTA keeps a ring of shared memory filled by TMA, 200 KB of it.
// A box is 64 of K x some rows x up to 32 times 64 of K further on: the tensor map takes a row's blocks of 64 as a dimension of their own, so
// that one copy brings up to 32 KB (bulk copies of one row's 1 to 2 KB each took 50 ns apiece: 5.0 and 3.2 TB/s; 16-byte loads into registers,
// 96 KB in flight, 5.4 and 4.1).  What a row has behind its last block comes through a second map, which ends with the row.  The tokens' side of
// a stage travels in it, a copy a token: loaded by the math warps it came through the same queues as the weights, 2 to 4 us behind its request.
// Eight warps multiply what has arrived by mma.sync: the weights are the A operand (16 rows x 16 of K), read 16 bytes a lane in the order of
// K in which they lie (the other operand is read in the same order, so the sum is the same); tokens stand in the columns, those that an expert
// does not serve as zeros.
//   up:   the rows of all reached experts, eight features of gate and up to a tile, are dealt evenly to the CTAs; the warps split K and
//         leave their parts in shared memory, where two warps of their own sum them up, so that nobody waits for activations and stores
//   down: the rows of the output are dealt to the CTAs; K runs over the reached experts' features one expert behind the other, so the sum
//         over a token's experts forms in the accumulators (their weights are in h), in the order of the experts' numbers
// h is held as two bf16 terms, value and remainder, which take two MMAs: it is as exact as the fp32 sums, and the tensor cores have room.  Its
// rows lie in the order of the experts, the tokens of one behind the other.
// Every CTA chooses the experts for itself from the logits; no CTA waits for another.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace lx {

constexpr int kFewTokens = 16;
constexpr int kFewExperts = 256;
constexpr int kFewTop = 32;
constexpr int kFewMath = 8;                // warps that multiply; one more fills the ring
constexpr int kFewSumWarps = 2;            // and two sum up the others' parts of a tile (up; by the math warps in turn, nine experts of 512 x 10752 took 145 us, now 111)
constexpr int kFewWarps = kFewMath + 1 + kFewSumWarps;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kFewRowTiles = 4;            // tiles of 16 rows of a CTA (down)
constexpr int kFewUpSteps = 8;             // steps of 32 of K of a stage and a math warp, at most (up): stages of 64 KB (of 32 KB: 110 -> 114 us for one token)
constexpr int kFewMaxStages = 16;
constexpr int kFewSums = 4;                // tiles of eight columns whose sums over the math warps may wait (up)
constexpr int kFewSmem = 232448 - 17 * 1024;      // (the rest: what is static)

enum FewAct : int { kFewSilu = 0, kFewGelu = 1, kFewGeluTanh = 2, kFewRelu = 3, kFewRelu2 = 4 };

struct MoeFewParams {
  const __nv_bfloat16* x;      // [T, H]
  long long ldx;
  const __nv_bfloat16* wr;     // [E, H]
  long long ldr;
  const float* logits;         // [T, E], or null: the up kernel forms them itself
  const __nv_bfloat16* w13;    // [e_local, 2 I, H]: gate rows, then up rows
  const __nv_bfloat16* w2;     // [e_local, H, I]
  __nv_bfloat16* h;            // two planes of [T k, I], in the order of the experts
  __nv_bfloat16* out;          // [T, H]
  long long ldo;
  int* status;
  int T, E, k, e0, e_local, H, I, act, renorm;
  float scale;
  // blocks of 64 of K of a copy of the up and of a stage of the down kernel; rows of a stage of the latter, and the logarithm of the rows of h that a copy brings
  int up_blocks, down_blocks, down_rows, h_shift;
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
// Eight elements, or zeros.  From L2: the down kernel chooses in front of its own wait, so nothing has made its SM's L1 forget what stood there before.
LX_DEVICE uint4 few_load(const __nv_bfloat16* p, bool valid) {
  uint4 v;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.relaxed.gpu.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t"
      "}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)valid));
  return v;
}

LX_DEVICE float few_act(float x, int act) {
  switch (act) {
    case kFewSilu: return x / (1.f + expf(-x));
    case kFewGelu: return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    case kFewGeluTanh: return 0.5f * x * (1.f + tanhf(0.79788456080286536f * (x + 0.044715f * x * x * x)));
    case kFewRelu: return x < 0.f ? 0.f : x;      // (a NaN stays)
    default: { const float r = x < 0.f ? 0.f : x; return r * r; }
  }
}

LX_DEVICE float few_logit(const float* p) {      // (the same, of the logits that a kernel in front of the up kernel left, or of shared memory)
  float v;
  asm volatile("ld.relaxed.gpu.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

// ------------------------------------------------------------------------------------------------ choice of experts, and who is reached
struct FewPlan {
  float w[kFewTokens * kFewTop];                // of a token's choices
  uint32_t mask[kFewExperts];                   // tokens of a local expert
  uint8_t place[kFewTokens][kFewExperts];       // which of its choices a local expert is for a token
  short list[kFewExperts];                      // local experts that have a token, ascending
  short base[kFewExperts];                      // the first row of h of each of those
  int4 warps[kFewWarps];
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

// One warp per token, PER experts a lane: its experts, their weights, and its mark with those that this rank owns (plan.mask is zero).  A NaN
// orders as -inf, and a token with one among its logits has weights that are NaN, whichever experts it goes to; no expert is chosen twice.
template <int PER>
LX_DEVICE void few_select(FewPlan& plan, const float* logits, const MoeFewParams& p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = warp; t < p.T; t += kFewWarps) {
    const float* row = logits + t * p.E;
    float z[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) z[i] = lane + 32 * i < p.E ? few_logit(row + lane + 32 * i) : 0.f;
    // logits as numbers whose order is theirs; 0: taken, or no expert
    uint32_t key[PER];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      odd |= z[i] != z[i];
      const float v = z[i] == z[i] ? z[i] + 0.f : -INFINITY;
      const uint32_t b = __float_as_uint(v);
      key[i] = lane + 32 * i < p.E ? ((b >> 31) ? ~b : b | 0x80000000u) : 0;
    }
    float top = 0.f, mine = 0.f;
    int id = 0;
    for (int j = 0; j < p.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      int lowest = kFewExperts;
#pragma unroll
      for (int i = PER - 1; i >= 0; --i)
        if (key[i] == best) lowest = lane + 32 * i;
      const int e = __reduce_min_sync(0xffffffffu, lowest);
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i == e) { v = z[i]; key[i] = 0; }
      v = __shfl_sync(0xffffffffu, v, e & 31);
      if (j == 0) top = v;
      if (lane == j) { id = e; mine = v; }
    }
    const float own = lane < p.k ? expf(mine - top) : 0.f;
    float all = own;
    if (!p.renorm) {
      all = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < p.E) all += expf(z[i] - top);
    }
    all = __any_sync(0xffffffffu, odd) ? NAN : warp_sum(all);
    const int e = id - p.e0;
    if (lane < p.k && e >= 0 && e < p.e_local) {
      plan.w[t * p.k + lane] = own / all * p.scale;
      plan.place[t][e] = (uint8_t)lane;
      atomicOr(&plan.mask[e], 1u << t);
    }
  }
}

// The experts that serve any token, and where their rows of h begin: one thread an expert.
LX_DEVICE void few_reached(FewPlan& plan) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  static_assert(kFewThreads >= kFewExperts, "a thread for every expert");
  const int n = threadIdx.x < kFewExperts ? __popc(plan.mask[threadIdx.x]) : 0;
  const uint32_t votes = __ballot_sync(0xffffffffu, n > 0);
  int v = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  const int most = __reduce_max_sync(0xffffffffu, n);
  if (lane == 31) plan.warps[warp] = make_int4(__popc(votes), v, most, 0);
  __syncthreads();
  int at = __popc(votes & ((1u << lane) - 1)), row = v - n, all = 0, top = 0;
#pragma unroll
  for (int i = 0; i < kFewWarps; ++i) {
    const int4 w = plan.warps[i];
    if (i < warp) { at += w.x; row += w.y; }
    all += w.x;
    top = max(top, w.z);
  }
  if (n > 0) {
    plan.list[at] = (short)threadIdx.x;
    plan.base[at] = (short)row;
  }
  if (threadIdx.x == 0) {
    plan.reached = all;
    plan.most = top;
  }
  __syncthreads();
}

// The plan of the launch, by every CTA for itself: from the logits that a kernel in front of the up kernel left, or from logits of its own.
template <int NT>
LX_DEVICE void few_choose(FewPlan& plan, uint8_t* smem, const MoeFewParams& p) {
  const float* logits = p.logits;
  if (threadIdx.x < kFewExperts) plan.mask[threadIdx.x] = 0;
  __syncthreads();
  if (logits == nullptr) {
    float4* sums = reinterpret_cast<float4*>(smem);
    float* z = reinterpret_cast<float*>(sums + kFewWarps * ((p.E + 15) / 16) * NT * 32);
    few_route<NT>(z, sums, p);
    logits = z;
  }
  if (p.E <= 64) few_select<2>(plan, logits, p);
  else few_select<kFewExperts / 32>(plan, logits, p);
  fence_proxy_async_smem();                    // (the ring lies where the sums and logits did)
  __syncthreads();
  few_reached(plan);
}

// Row of h of token t (one of `mask`) within its expert's.
LX_DEVICE int few_slot(uint32_t mask, int t) { return __popc(mask & ((1u << t) - 1)); }
// Copies of 2^shift rows of h that bring n of them.
__host__ __device__ inline int few_copies(int n, int shift) { return (n + (1 << shift) - 1) >> shift; }
// The i-th token of `mask`.
LX_DEVICE int few_token(uint32_t mask, int i) {
  for (; i > 0; --i) mask &= mask - 1;
  return __ffs(mask) - 1;
}

// Feature `row` of token t from the experts that serve it alone, by one warp.  A column of the down product has zeros where an expert does not serve its token, and
// an h that one bf16 term holds has a remainder of zero: times a weight that is infinite or no number, both are NaN.  Sums that are not finite are formed again by
// this, unless the token's own weights are NaN.
LX_DEVICE float few_alone(const FewPlan& plan, const MoeFewParams& p, int t, int row) {
  const int lane = threadIdx.x & 31;
  float sum = 0.f;
  for (int d = 0; d < plan.reached; ++d) {
    const int e = plan.list[d];
    const uint32_t mask = plan.mask[e];
    if (((mask >> t) & 1) == 0) continue;
    const float w = plan.w[t * p.k + plan.place[t][e]];
    if (w != w) return NAN;
    const __nv_bfloat16* weights = p.w2 + ((long long)e * p.H + row) * p.I;
    const __nv_bfloat16* value = p.h + (long long)(plan.base[d] + few_slot(mask, t)) * p.I;
    const __nv_bfloat16* remainder = value + (long long)p.T * p.k * p.I;
    for (int i = lane * 8; i < p.I; i += 256) {
      const uint4 a = few_load(weights + i, true), b = few_load(value + i, true), c = few_load(remainder + i, true);
      const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
      float part = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        part += __uint_as_float(av[q] << 16) * (__uint_as_float(bv[q] << 16) + __uint_as_float(cv[q] << 16));
        part += __uint_as_float(av[q] & 0xffff0000u) * (__uint_as_float(bv[q] & 0xffff0000u) + __uint_as_float(cv[q] & 0xffff0000u));
      }
      sum += part;
    }
  }
  return warp_sum(sum);
}

// ------------------------------------------------------------------------------------------------ the ring
// Stages of shared memory, filled by one warp and read by the math warps.  Waits are bounded: one that runs out is reported, the filling warp stops (and
// waits for its copies), and the math warps go on without waiting (they meet at barriers), so that the launch ends.
struct FewRing {
  uint64_t full[kFewMaxStages], empty[kFewMaxStages];
  uint64_t sums[kFewSums], read[kFewSums];      // the math warps' sums of a tile: written, read
  int stop;
  int odd;                                      // a result is not finite (down)
};

LX_DEVICE void few_ring_init(FewRing& r) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewMaxStages; ++s) { mbar_init(&r.full[s], 1); mbar_init(&r.empty[s], kFewMath); }
    for (int s = 0; s < kFewSums; ++s) { mbar_init(&r.sums[s], kFewMath); mbar_init(&r.read[s], 1); }
    r.stop = r.odd = 0;
    mbar_fence_init();
  }
}

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

// Tensor maps of a product's operands: whole blocks of 64 of K, and what is behind them.  [1]: boxes of twice the blocks (up), of half of them (down).
struct FewMaps {
  CUtensorMap weights[2], tokens[2], weights_rest, tokens_rest;
};

LX_DEVICE void few_prefetch(const FewMaps& maps) {
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&maps.weights[0]);
    tma_prefetch_desc(&maps.tokens[0]);
  }
}

// ------------------------------------------------------------------------------------------------ up
// NT: columns of eight tokens.
template <int NT>
__global__ void __launch_bounds__(kFewThreads, 1) moe_few_up_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ MoeFewParams p) {
  __shared__ FewPlan plan;
  __shared__ FewRing ring;
  __shared__ __align__(16) uint8_t zeros[kFewZeros];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  few_ring_init(ring);
  for (int i = tid; i < kFewZeros / 4; i += kFewThreads) reinterpret_cast<uint32_t*>(zeros)[i] = 0;
  few_prefetch(maps);
  pdl_wait();
  pdl_trigger();
  few_choose<NT>(plan, smem, p);
  // A stage: gate rows, up rows, the expert's tokens (in large boxes where two such stages fit); the same of what is behind the last block, for a
  // tile's last stage.
  const int units = p.I / 8, blocks = p.H / 64, most = plan.most;
  const bool rest = p.H % 64 != 0;
  constexpr int kSums = kFewSums / NT, kRoom = kFewSmem - 1024 - kSums * kFewMath * NT * 32 * (int)sizeof(float4);
  const auto stage_of = [&](int b) { return ((b * (2048 + most * 128) + 1023) & ~1023) + (rest ? (2048 + most * 128 + 1023) & ~1023 : 0); };
  const bool large = blocks > p.up_blocks && 2 * stage_of(2 * p.up_blocks) <= kRoom;
  const int wide = p.up_blocks << large;
  const int chunks = max(1, (blocks + wide - 1) / wide), half = wide * 1024, token = wide * 128;
  const int rest_at = (2 * half + most * token + 1023) & ~1023, stage_bytes = stage_of(wide), stages = min(kRoom / stage_bytes, kFewMaxStages);
  const long long all = (long long)plan.reached * units;
  const int u0 = (int)(all * blockIdx.x / gridDim.x), u1 = (int)(all * (blockIdx.x + 1) / gridDim.x);
  FewCursor at;
  if (warp == kFewMath) {
    if (lane == 0) {
      const uint64_t policy = policy_evict_first();
      long long filled = 0;
      bool ok = true;
      int d = u0 / units, c = (u0 - d * units) * 8 - 8, e = 0, n = 0;
      uint32_t mask = 0;
      for (int u = u0; ok && u < u1; ++u) {
        if ((c += 8) == p.I) { c = 0; ++d; }
        if (u == u0 || c == 0) {
          e = plan.list[d];
          mask = plan.mask[e];
          n = __popc(mask);
        }
        for (int ch = 0; ok && ch < chunks; ++ch, ++filled) {
          uint8_t* stage = smem + at.stage * stage_bytes;
          const bool ends = rest && ch == chunks - 1;
          ok = few_fill(ring, at, stages, (blocks > 0 ? 2 * half + n * token : 0) + (ends ? 2048 + n * 128 : 0), p.status, [&](uint64_t* bar) {
            if (blocks > 0) {
              tma_load_4d_hint(stage, &maps.weights[large], bar, 0, c, ch * wide, e, policy);
              tma_load_4d_hint(stage + half, &maps.weights[large], bar, 0, p.I + c, ch * wide, e, policy);
              uint8_t* to = stage + 2 * half;
              for (uint32_t m = mask; m != 0; m &= m - 1, to += token) tma_load_4d(to, &maps.tokens[large], bar, 0, __ffs(m) - 1, ch * wide, 0);
            }
            if (ends) {
              tma_load_4d_hint(stage + rest_at, &maps.weights_rest, bar, blocks * 64, c, 0, e, policy);
              tma_load_4d_hint(stage + rest_at + 1024, &maps.weights_rest, bar, blocks * 64, p.I + c, 0, e, policy);
              uint8_t* to = stage + rest_at + 2048;
              for (uint32_t m = mask; m != 0; m &= m - 1, to += 128) tma_load_4d(to, &maps.tokens_rest, bar, blocks * 64, __ffs(m) - 1, 0, 0);
            }
          });
        }
      }
      few_drain(ring, at, stages, filled);
    }
    return;
  }
  float4* red = reinterpret_cast<float4*>(smem + stages * stage_bytes);      // [kSums][math warps][NT][32 lanes]
  if (warp > kFewMath) {
    // (a buffer is always the same warp's: one that waited for another's phase could take the last but one of the same parity for it)
    static_assert(kSums % kFewSumWarps == 0, "whole turns");
    bool ok = true;
    int d = u0 / units, c = (u0 - d * units) * 8 - 8, e = 0, served = 0, row = 0;
    uint32_t mask = 0;
    for (int u = u0; u < u1; ++u) {
      if ((c += 8) == p.I) { c = 0; ++d; }
      if (u == u0 || c == 0) {
        e = plan.list[d];
        mask = plan.mask[e];
        served = __popc(mask);
        row = plan.base[d];
      }
      const int turn = u - u0, buf = turn % kSums, n = NT == 1 || served <= 8 ? 1 : NT;
      if (turn % kFewSumWarps != warp - kFewMath - 1) continue;
      const int col = c + few_lane_row(g);
      const float4* part = red + buf * kFewMath * NT * 32;
      few_await(ring, &ring.sums[buf], (turn / kSums) & 1, ok, p.status);
      for (int m = 0; m < n; ++m) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFewMath; ++w) {
          const float4 a = part[(w * n + m) * 32 + lane];
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
          const long long at = (long long)(row + i) * p.I + col;
          p.h[at] = hi;
          p.h[at + (long long)p.T * p.k * p.I] = __float2bfloat16(fabsf(back) < INFINITY ? h - back : 0.f);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring.read[buf]);
    }
    return;
  }
  const int steps = 2 * blocks, per = 2 * wide, place = few_place(8, few_lane_row(g), warp, c8), column = (warp * 32 + c8) * 2;
  bool ok = true;
  uint32_t sums_phase = 0;
  // A tile for an expert of up to 8 N tokens: they stand in the columns in their order.
  int d = u0 / units, c = (u0 - d * units) * 8 - 8, e = 0, served = 0;
  uint32_t mask = 0;
  auto tile = [&](auto n, int u) {
    constexpr int N = decltype(n)::value;
    const int buf = (u - u0) % kSums;
    float acc[2][N][4];                        // (two chains of MMAs)
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int m = 0; m < N; ++m) acc[o][m][0] = acc[o][m][1] = acc[o][m][2] = acc[o][m][3] = 0.f;
    for (int ch = 0; ch < chunks; ++ch) {
      const uint32_t stage = smem_u32(smem) + at.stage * stage_bytes;
      uint32_t xt[N];
#pragma unroll
      for (int m = 0; m < N; ++m) {
        const int i = m * 8 + g;
        xt[m] = i < served ? stage + 2 * half + column + i * token : smem_u32(zeros);
      }
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
      if (rest && ch == chunks - 1 && warp < 2) {
        const uint4 gate = few_row(stage + rest_at + place), up = few_row(stage + rest_at + 1024 + place);
#pragma unroll
        for (int m = 0; m < N; ++m)
          few_mma32(acc[0][m], gate, up, few_row(m * 8 + g < served ? stage + rest_at + 2048 + (m * 8 + g) * 128 + column : smem_u32(zeros)));
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
    if (buf == kSums - 1) sums_phase ^= 1;
  };
  for (int u = u0; u < u1; ++u) {
    if ((c += 8) == p.I) { c = 0; ++d; }
    if (u == u0 || c == 0) {
      e = plan.list[d];
      mask = plan.mask[e];
      served = __popc(mask);
    }
    if (NT == 1 || served <= 8) tile(std::integral_constant<int, 1>{}, u);
    else tile(std::integral_constant<int, NT>{}, u);
  }
}

// ------------------------------------------------------------------------------------------------ down
// MT: tiles of 16 rows; steps of 32 of K of a stage and a math warp: as many as bring 32 to 64 KB of weights (of half of that, 470 -> 490 us for 16 tokens).
template <int MT, int NT>
constexpr int few_down_steps() { return MT == 1 || MT + NT == 3 ? 4 : 2; }
static int few_down_tiles(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 48 ? 3 : kFewRowTiles; }

// A stage: rows of the weights, values and remainders of the expert's tokens (at most `copies` copies); the same of what is behind the last block, for an expert's last
// stage.  Where only one such stage fits beside the sums, it has half the blocks: filling and multiplying would take turns (wide layers whose 13 to 16 tokens
// share an expert, and some with a rest of K and more than four or twelve: 16 tokens at two experts of 9472 x 8192 232 -> 207 us).
struct FewDownStage {
  int blocks, rest, wide, plane, plane_rest, rest_at, rest_h, bytes, stages;
  bool half;
  __host__ __device__ FewDownStage(int mt, int nt, int I, int rows, int all_blocks, int copies, int h_shift) : rest(I % 64 != 0), plane_rest(128 << h_shift) {
    const int room = kFewSmem - 1024 - kFewMath * mt * nt * 32 * (int)sizeof(float4);
    blocks = all_blocks;
    for (half = false;; half = true, blocks = (all_blocks + 1) / 2) {
      wide = (blocks * rows * 128 + 1023) & ~1023;
      plane = blocks * 128 << h_shift;
      rest_at = (wide + copies * 2 * plane + 1023) & ~1023;
      rest_h = (rest_at + rows * 128 + 127) & ~127;
      bytes = rest ? (rest_h + copies * 2 * plane_rest + 1023) & ~1023 : rest_at;
      stages = room / bytes < kFewMaxStages ? room / bytes : kFewMaxStages;
      if (stages > 1 || half) return;
    }
  }
};

template <int MT, int NT>
__global__ void __launch_bounds__(kFewThreads, 1) moe_few_down_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ MoeFewParams p) {
  __shared__ FewPlan plan;
  __shared__ FewRing ring;
  __shared__ __align__(16) uint8_t zeros[kFewZeros];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  few_ring_init(ring);
  for (int i = tid; i < kFewZeros / 4; i += kFewThreads) reinterpret_cast<uint32_t*>(zeros)[i] = 0;
  few_prefetch(maps);
  // In front of the wait for the up kernel: every CTA of it has waited itself for what wrote the tokens, the router and the logits, and triggers behind that, so
  // they are complete in L2, where few_load and few_logit read them.
  few_choose<NT>(plan, smem, p);
  const FewDownStage geo(MT, NT, p.I, p.down_rows, p.down_blocks, few_copies(plan.most, p.h_shift), p.h_shift);
  const int blocks = p.I / 64, deep = geo.blocks, chunks = max(1, (blocks + deep - 1) / deep), reached = plan.reached, rows = p.down_rows;
  const int bytes = deep * rows * 128, wide = geo.wide, plane = geo.plane, plane_rest = geo.plane_rest;
  const bool rest = geo.rest;
  const int rest_at = geo.rest_at, rest_h = geo.rest_h, stage_bytes = geo.bytes, stages = geo.stages;
  FewCursor at;
  if (warp == kFewMath) {
    if (lane == 0) {
      const uint64_t policy = policy_evict_first();
      long long filled = 0;
      bool ok = true;
      // the weights of the first round of stages go ahead of the wait; their tokens follow
      bool waited = false;
      auto copies_of = [&](int d) { return few_copies(__popc(plan.mask[plan.list[d]]), p.h_shift); };
      auto tokens_of = [&](uint8_t* stage, uint64_t* bar, int row, int n, int ch) {
        if (blocks > 0)
          for (int i = 0; i < n; ++i) tma_load_4d(stage + wide + i * 2 * plane, &maps.tokens[geo.half], bar, 0, row + (i << p.h_shift), ch * deep, 0);
        if (rest && ch == chunks - 1)
          for (int i = 0; i < n; ++i) tma_load_4d(stage + rest_h + i * 2 * plane_rest, &maps.tokens_rest, bar, blocks * 64, row + (i << p.h_shift), 0, 0);
      };
      auto catch_up = [&]() {
        pdl_wait();
        waited = true;
        int d = 0, ch = 0;
        for (int i = 0; i < filled; ++i) {
          tokens_of(smem + i * stage_bytes, &ring.full[i], plan.base[d], copies_of(d), ch);
          if (++ch == chunks) { ch = 0; d = d + 1 == reached ? 0 : d + 1; }
        }
      };
      for (int r0 = blockIdx.x * rows; ok && r0 < p.H; r0 += gridDim.x * rows)
        for (int d = 0; ok && d < reached; ++d) {
          const int e = plan.list[d], row = plan.base[d], n = copies_of(d), whole = blocks > 0 ? bytes + n * 2 * plane : 0;
          for (int ch = 0; ok && ch < chunks; ++ch, ++filled) {
            if (!waited && filled == stages) catch_up();
            uint8_t* stage = smem + at.stage * stage_bytes;
            const bool ends = rest && ch == chunks - 1;
            ok = few_fill(ring, at, stages, whole + (ends ? rows * 128 + n * 2 * plane_rest : 0), p.status, [&](uint64_t* bar) {
              if (blocks > 0) tma_load_4d_hint(stage, &maps.weights[geo.half], bar, 0, r0, ch * deep, e, policy);
              if (ends) tma_load_4d_hint(stage + rest_at, &maps.weights_rest, bar, blocks * 64, r0, 0, e, policy);
              if (waited) tokens_of(stage, bar, row, n, ch);
            });
          }
        }
      if (!waited) catch_up();
      few_drain(ring, at, stages, filled);
    }
    return;
  }
  if (warp > kFewMath) return;
  pdl_wait();
  pdl_trigger();
  float4* red = reinterpret_cast<float4*>(smem + stages * stage_bytes);      // [math warps][MT][NT][32 lanes]
  constexpr int kSteps = few_down_steps<MT, NT>();
  const int steps = 2 * blocks, per = 2 * deep;
  int place[MT][2];                            // (rows past the last one are taken from it: nobody stores their sums)
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int o = 0; o < 2; ++o) place[m][o] = few_place(rows, min(m * 16 + o * 8 + few_lane_row(g), rows - 1), warp, c8);
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
      // where the lane's tokens lie in a stage: copies of some rows, in each the rows of a block side by side, the blocks of the values, those of
      // the remainders
      int slot[NT], slot_rest[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int i = few_slot(mask, n * 8 + g);
        slot_rest[n] = rest_h + (i >> p.h_shift) * 2 * plane_rest + (i & ((1 << p.h_shift) - 1)) * 128 + (warp & 1) * 64 + c8 * 2;
        slot[n] = ((mask >> (n * 8 + g)) & 1) ? wide + (i >> p.h_shift) * 2 * plane + (((warp >> 1) << p.h_shift) + (i & ((1 << p.h_shift) - 1))) * 128 + (warp & 1) * 64 + c8 * 2 : -1;
      }
      for (int ch = 0; ch < chunks; ++ch) {
        const uint32_t stage = smem_u32(smem) + at.stage * stage_bytes;
        uint32_t ht[NT][2], step[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bool on = slot[n] >= 0;
          ht[n][0] = on ? stage + slot[n] : smem_u32(zeros);
          ht[n][1] = ht[n][0] + (on ? plane : 0);
          step[n] = on ? 512 << p.h_shift : 0;
        }
        few_await(ring, &ring.full[at.stage], at.phase, ok, p.status);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const int s = j * kFewMath + warp;
          if (s < per && ch * per + s < steps) {
            uint4 h[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              h[n][0] = few_row(ht[n][0] + j * step[n]);
              h[n][1] = few_row(ht[n][1] + j * step[n]);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) multiply(few_row(stage + place[m][0] + j * 512 * rows), few_row(stage + place[m][1] + j * 512 * rows), h, m);
          }
        }
        if (rest && ch == chunks - 1 && warp < 2) {
          uint4 h[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const bool on = slot[n] >= 0;
            h[n][0] = few_row(on ? stage + slot_rest[n] : smem_u32(zeros));
            h[n][1] = few_row(on ? stage + slot_rest[n] + plane_rest : smem_u32(zeros));
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) multiply(few_row(stage + rest_at + place[m][0]), few_row(stage + rest_at + place[m][1]), h, m);
        }
        few_release(ring, at, stages);
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
        const float y = o == 0 ? v.x : o == 1 ? v.y : o == 2 ? v.z : v.w;
        if (t < p.T && r < rows && r0 + r < last) {
          p.out[(long long)t * p.ldo + r0 + r] = __float2bfloat16(y);
          if (!(fabsf(y) < INFINITY)) ring.odd = 1;
        }
      }
    }
    few_math_sync();
  }
  // Results that are not finite, once more.  (Behind everything else: in the loop above, as a call, it cost the finite ones 2 % of narrow layers.)
  if (ring.odd == 0) return;
  for (int r0 = blockIdx.x * rows; r0 < p.H; r0 += gridDim.x * rows) {
    const int n = min(rows, p.H - r0);
    for (int i = warp; i < n * p.T; i += kFewMath) {
      const int t = i / n, r = r0 + i % n;
      __nv_bfloat16* out = p.out + (long long)t * p.ldo + r;
      if (fabsf(__bfloat162float(*out)) < INFINITY) continue;
      const float y = few_alone(plan, p, t, r);
      if (lane == 0) *out = __float2bfloat16(y);
    }
  }
}

// Matrices [outer, rows, K], rows `ld` and matrices `ldo` elements apart.  `out`: {64 of K, rows, blocks of 64, outer}, boxes of `box_rows` rows x
// `box_blocks` blocks x `box_outer`; `rest`: {K, rows, 1, outer}, boxes of 64 of K x `box_rows` rows x `box_outer`, for what a row has behind its last
// whole block.  What a box has past the rows, the blocks or K reads as zero.
static int few_tmap(CUtensorMap* out, CUtensorMap* rest, const void* base, long long outer, long long rows, long long K, long long ld, long long ldo, int box_rows,
                    int box_blocks, int box_outer, bool swizzle) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return -4;
    encode = reinterpret_cast<Encode>(fn);
  }
  if (outer == 0) return 0;                    // (no copy is made)
  const cuuint64_t strides[3] = {(cuuint64_t)ld * 2, 128, (cuuint64_t)ldo * 2};
  const cuuint32_t each[4] = {1, 1, 1, 1};
  for (int r = 0; r < 2; ++r) {
    if (r == 0 ? K < 64 : K % 64 == 0 || rest == nullptr) continue;
    const cuuint64_t dims[4] = {r == 0 ? 64 : (cuuint64_t)K, (cuuint64_t)rows, r == 0 ? (cuuint64_t)(K / 64) : 1, (cuuint64_t)outer};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, r == 0 ? (cuuint32_t)box_blocks : 1, (cuuint32_t)box_outer};
    if (encode(r == 0 ? out : rest, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
               swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return -5;
  }
  return 0;
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

// Rows of a CTA's stages of the down kernel, and the logarithm of the rows of h of a copy (what a copy brings beyond the expert's tokens is not read).
static int few_down_rows(int H, int num_sms) { return std::min(((H + num_sms - 1) / num_sms + 1) & ~1, 16 * kFewRowTiles); }
static int few_h_shift(int T) { return T <= 2 ? T - 1 : 2; }

template <int MT, int NT>
static int moe_few_down(MoeFewParams& p, int num_sms, cudaStream_t s) {
  static bool set[64] = {};
  if (const int rc = few_opt_in(moe_few_down_kernel<MT, NT>, set)) return rc;
  p.down_blocks = few_blocks(p.I / 64, few_down_steps<MT, NT>() * kFewMath / 2);
  FewMaps maps{};
  // (the half ones are made where the most tokens an expert can have need them; the kernel goes by those that it has)
  const int n = FewDownStage(MT, NT, p.I, p.down_rows, p.down_blocks, few_copies(p.T, p.h_shift), p.h_shift).half ? 2 : 1;
  for (int i = 0; i < n; ++i) {
    const int blocks = (p.down_blocks + i) >> i;
    if (const int rc = few_tmap(&maps.weights[i], i == 0 ? &maps.weights_rest : nullptr, p.w2, p.e_local, p.H, p.I, p.I, (long long)p.H * p.I, p.down_rows, blocks, 1, true)) return rc;
    if (const int rc = few_tmap(&maps.tokens[i], i == 0 ? &maps.tokens_rest : nullptr, p.h, 2, (long long)p.T * p.k, p.I, p.I, (long long)p.T * p.k * p.I, 1 << p.h_shift, blocks, 2,
                                false)) return rc;
  }
  launch_pdl(moe_few_down_kernel<MT, NT>, dim3(num_sms), dim3(kFewThreads), kFewSmem, s, maps, p);
  return -(int)cudaGetLastError();
}

template <int NT>
static int moe_few_launch(MoeFewParams& p, int num_sms, cudaStream_t s) {
  static bool set[64] = {};
  if (const int rc = few_opt_in(moe_few_up_kernel<NT>, set)) return rc;
  p.up_blocks = few_blocks(p.H / 64, kFewUpSteps * kFewMath / 4);
  FewMaps maps{};
  for (int i = 0; i < 2; ++i) {
    if (const int rc = few_tmap(&maps.weights[i], i == 0 ? &maps.weights_rest : nullptr, p.w13, p.e_local, 2LL * p.I, p.H, p.H, 2LL * p.I * p.H, 8, p.up_blocks << i, 1, true)) return rc;
    if (const int rc = few_tmap(&maps.tokens[i], i == 0 ? &maps.tokens_rest : nullptr, p.x, 1, p.T, p.H, p.ldx, p.T * p.ldx, 1, p.up_blocks << i, 1, false)) return rc;
  }
  launch_pdl(moe_few_up_kernel<NT>, dim3(num_sms), dim3(kFewThreads), kFewSmem, s, maps, p);
  p.h_shift = few_h_shift(p.T);
  p.down_rows = few_down_rows(p.H, num_sms);
  switch (few_down_tiles(p.down_rows)) {
    case 1: return moe_few_down<1, NT>(p, num_sms, s);
    case 2: return moe_few_down<2, NT>(p, num_sms, s);
    case 3: return moe_few_down<3, NT>(p, num_sms, s);
    default: return moe_few_down<kFewRowTiles, NT>(p, num_sms, s);
  }
}

}  // namespace lx

extern "C" {

int lx_moe_few_max_tokens() { return lx::kFewTokens; }

int lx_moe_router_logits(const void* x, long long ldx, const void* wr, long long ldw, float* logits, int T, int E, int H, int* counts, int ncounts,
                         void* stream);

// Stages of the down kernel's ring for T tokens, `most` of which one expert serves.
int lx_moe_few_down_stages(int T, int H, int I, int most, int num_sms) {
  using namespace lx;
  if (T <= 0 || T > kFewTokens || most <= 0 || most > T || H <= 0 || I <= 0 || num_sms <= 0) return -1;
  const int rows = few_down_rows(H, num_sms), mt = few_down_tiles(rows), nt = T <= 8 ? 1 : 2, shift = few_h_shift(T);
  const int steps = mt == 1 ? few_down_steps<1, 1>() : mt == 2 ? (nt == 1 ? few_down_steps<2, 1>() : few_down_steps<2, 2>()) : mt == 3 ? few_down_steps<3, 1>() : few_down_steps<4, 1>();
  return FewDownStage(mt, nt, I, rows, few_blocks(I / 64, steps * kFewMath / 2), few_copies(most, shift), shift).stages;
}

// -> kernels launched, or an error below zero.  `logits` [T, E] and `h` [2, T k, I] are scratch of the call.
int lx_moe_few(const void* x, long long ldx, const void* wr, long long ldw, const void* w13, const void* w2, float* logits, void* h, void* out, long long ldo, int T,
               int E, int k, int e0, int e_local, int H, int I, int act, int renorm, float scale, int* status, int num_sms, void* stream) {
  using namespace lx;
  if (T < 0 || T > kFewTokens || E <= 0 || E > kFewExperts || k <= 0 || k > kFewTop || k > E || e_local < 0 || e_local > kFewExperts || H <= 0 || H % 8 != 0 ||
      I <= 0 || I % 8 != 0 || act < 0 || act > kFewRelu2 || num_sms <= 0)
    return -1;
  for (const void* q : {x, wr, w13, w2, (const void*)h})
    if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return -2;
  if (ldx % 8 != 0 || ldw % 8 != 0) return -2;
  if (T == 0) return 0;
  // Up to 128 KB of router and tokens, every CTA of both kernels forms the logits itself; beyond, they are a launch of their own in front (one token of 4096
  // and 8 experts 116 -> 115 us, of 2048 and 64 experts 30 -> 37).
  const bool by_itself = (E + T) * (long long)H <= 65536;
  if (!by_itself)
    if (const int rc = lx_moe_router_logits(x, ldx, wr, ldw, logits, T, E, H, nullptr, 0, stream)) return rc;
  MoeFewParams p{};
  p.x = reinterpret_cast<const __nv_bfloat16*>(x); p.ldx = ldx; p.logits = by_itself ? nullptr : logits;
  p.wr = reinterpret_cast<const __nv_bfloat16*>(wr); p.ldr = ldw;
  p.w13 = reinterpret_cast<const __nv_bfloat16*>(w13); p.w2 = reinterpret_cast<const __nv_bfloat16*>(w2);
  p.h = reinterpret_cast<__nv_bfloat16*>(h); p.out = reinterpret_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.T = T; p.E = E; p.k = k; p.e0 = e0; p.e_local = e_local; p.H = H; p.I = I; p.act = act; p.renorm = renorm; p.scale = scale; p.status = status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = T <= 8 ? moe_few_launch<1>(p, num_sms, s) : moe_few_launch<2>(p, num_sms, s);
  return rc != 0 ? rc : by_itself ? 2 : 3;
}

}  // extern "C"
