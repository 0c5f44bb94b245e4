// A whole mixture-of-experts layer for a few tokens (T <= 16): every byte of the experts that the tokens reach is read once, by all SMs at
// the HBM's rate, and nothing else of size is moved.
//
//   z[t, e] = x_t . Wr_e; the k largest z of a token (the lower expert on ties); w[t, j] = exp(z_j - z_max) over their sum (or over the sum of
//   all experts), times a constant
//   up      h[t, j, i] = w[t, j] act(G_e[i] . x_t) (U_e[i] . x_t)    for the experts e = e(t, j) that this rank owns
//   down    out[t, n] = sum_j D_e[n] . h[t, j]
//
// Both products are streams of weights against at most 16 columns: the weights are the A operand of mma.sync (16 rows x 16 of K), loaded
// straight from global memory into registers, 16 bytes a lane, in the order of K in which a lane finds them (the other operand is read in
// the same order, so the sum is the same); tokens stand in the columns, those that an expert does not serve as zeros.
//   up:   the rows of all reached experts, eight features of gate and up to a tile, are dealt evenly to the CTAs; the warps of a CTA split
//         K and sum their parts through shared memory
//   down: the rows of the output are dealt to the CTAs; K runs over the reached experts' features one expert behind the other, so the sum
//         over a token's experts forms in the accumulators (their weights are in h), in the order of the experts' numbers
// h is held as two bf16 terms, value and remainder, which take two MMAs: it is as exact as the fp32 sums, and the tensor cores have room.
// Every CTA chooses the experts for itself from the logits; no CTA waits for another.
#include "common.cuh"

namespace lx {

constexpr int kFewTokens = 16;
constexpr int kFewExperts = 256;
constexpr int kFewTop = 32;
constexpr int kFewWarps = 8;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kFewTiles = 32;              // tiles whose sums over K wait in shared memory at once (up), for eight columns
constexpr int kFewRowTiles = 4;            // tiles of 16 rows of a CTA (down)

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
  __nv_bfloat16* h;            // two planes of [T k, I]
  __nv_bfloat16* out;          // [T, H]
  long long ldo;
  int T, E, k, e0, e_local, H, I, act, renorm;
  float scale;
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
// Loads of a batch are issued in the order written here, in front of the batch's MMAs (left to itself the compiler moves each load to its use, and
// few bytes are in flight).  Weights are read once and kept out of L1; what is not valid reads as zero.
LX_DEVICE uint4 few_weights(const __nv_bfloat16* p, bool valid) {
  uint4 v;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n\t"
      "}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((int)valid));
  return v;
}
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
  int warps[kFewWarps];
  int reached;
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
  static_assert(kFewThreads == kFewExperts, "a thread for every expert");
  plan.mask[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.T * p.k; i += kFewThreads) {
    const int e = plan.ids[i] - p.e0, t = i / p.k;
    if (e >= 0 && e < p.e_local) {
      atomicOr(&plan.mask[e], 1u << t);
      plan.place[t][e] = (uint8_t)(i - t * p.k);
    }
  }
  __syncthreads();
  const bool has = plan.mask[threadIdx.x] != 0;
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
}

// ------------------------------------------------------------------------------------------------ up
// NT: columns of eight tokens.
template <int NT>
__global__ void __launch_bounds__(kFewThreads) moe_few_up_kernel(const __grid_constant__ MoeFewParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kTiles = kFewTiles / NT, kBatch = 8 / NT;
  __shared__ FewPlan plan;
  extern __shared__ float4 red[];              // [warps][kTiles][NT][32 lanes]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  const float* logits = p.logits;
  if (logits == nullptr) {
    __shared__ float z[kFewTokens * kFewExperts];
    few_route<NT>(z, red, p);
    logits = z;
  }
  few_select(plan, logits, p);
  __syncthreads();
  few_reached(plan, p);
  if (blockIdx.x == 0)
    for (int i = tid; i < p.T * p.k; i += kFewThreads) p.ids[i] = plan.ids[i];
  const int units = p.I / 8, steps = (p.H + 31) / 32;
  const long long all = (long long)plan.reached * units;
  const int u0 = (int)(all * blockIdx.x / gridDim.x), u1 = (int)(all * (blockIdx.x + 1) / gridDim.x);
  const int batches = (steps + kFewWarps * kBatch - 1) / (kFewWarps * kBatch);      // of a tile
  struct Buffer { uint4 a[kBatch][2], b[kBatch][NT]; };
  for (int r0 = u0; r0 < u1; r0 += kTiles) {
    const int n = min(kTiles, u1 - r0), total = n * batches;
    // batch q of this round: K steps of tile q / batches.  The next batch is on its way while one is multiplied.
    int tile = 0, part = 0;                    // of the batch that is loaded next
    const __nv_bfloat16 *gate = nullptr, *xt[NT];
    bool on[NT];
    auto load = [&](Buffer& v) {
      if (part == 0) {
        const int d = (r0 + tile) / units, e = plan.list[d];
        gate = p.w13 + ((long long)e * 2 * p.I + (r0 + tile - d * units) * 8 + g) * p.H + c8;
        const uint32_t mask = plan.mask[e];
#pragma unroll
        for (int m = 0; m < NT; ++m) {
          on[m] = (mask >> (m * 8 + g)) & 1;
          xt[m] = p.x + (long long)(m * 8 + g) * p.ldx + c8;
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k0 = ((part * kBatch + j) * kFewWarps + warp) * 32;
        const bool ok = k0 + c8 < p.H;
        v.a[j][0] = few_weights(gate + k0, ok);
        v.a[j][1] = few_weights(gate + (long long)p.I * p.H + k0, ok);
#pragma unroll
        for (int m = 0; m < NT; ++m) v.b[j][m] = few_load(xt[m] + k0, ok && on[m]);
      }
      if (++part == batches) { part = 0; ++tile; }
    };
    float acc[NT][4];
#pragma unroll
    for (int m = 0; m < NT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
    int done = 0, in_tile = 0;                 // tiles summed up, batches of the one at hand
    auto take = [&](const Buffer& v) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int m = 0; m < NT; ++m) few_mma32(acc[m], v.a[j][0], v.a[j][1], v.b[j][m]);
      if (++in_tile < batches) return;
#pragma unroll
      for (int m = 0; m < NT; ++m) {
        red[((warp * kTiles + done) * NT + m) * 32 + lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
        acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
      }
      in_tile = 0;
      ++done;
    };
    Buffer v0, v1;
    load(v0);
    for (int q = 0; q < total; q += 2) {
      if (q + 1 < total) load(v1);
      take(v0);
      if (q + 1 >= total) break;
      if (q + 2 < total) load(v0);
      take(v1);
    }
    __syncthreads();
    for (int q = tid; q < n * NT * 32; q += kFewThreads) {
      const int i = q / (NT * 32), m = q / 32 % NT, l = q & 31;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float4 part = red[((w * kTiles + i) * NT + m) * 32 + l];
        v.x += part.x; v.y += part.y; v.z += part.z; v.w += part.w;
      }
      const int d = (r0 + i) / units, col = (r0 + i - d * units) * 8 + (l >> 2), e = plan.list[d];
#pragma unroll
      for (int o = 0; o < 2; ++o) {              // (gate and up of the tile's column l / 4, tokens 2 (l % 4) and the next)
        const int t = m * 8 + (l & 3) * 2 + o;
        if (!((plan.mask[e] >> t) & 1)) continue;
        const int pair = t * p.k + plan.place[t][e];
        const float h = few_act(o ? v.y : v.x, p.act) * (o ? v.w : v.z) * plan.w[pair];
        const __nv_bfloat16 hi = __float2bfloat16(h);
        const float back = __bfloat162float(hi);
        p.h[(long long)pair * p.I + col] = hi;
        p.h[((long long)p.T * p.k + pair) * p.I + col] = __float2bfloat16(fabsf(back) < INFINITY ? h - back : 0.f);
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ down
// MT: tiles of 16 rows.
template <int MT, int NT>
__global__ void __launch_bounds__(kFewThreads) moe_few_down_kernel(const __grid_constant__ MoeFewParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kBatch = MT + NT <= 2 ? 4 : MT + NT <= 4 ? 3 : 2;
  __shared__ FewPlan plan;
  __shared__ float4 red[kFewWarps][MT][NT][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c8 = (lane & 3) * 8;
  for (int i = tid; i < p.T * p.k; i += kFewThreads) plan.ids[i] = p.ids[i];
  __syncthreads();
  few_reached(plan, p);
  const int steps = (p.I + 31) / 32, items = plan.reached * steps;
  const int first = (int)((long long)p.H * blockIdx.x / gridDim.x), last = (int)((long long)p.H * (blockIdx.x + 1) / gridDim.x);
  const long long plane = (long long)p.T * p.k * p.I;
  for (int r0 = first; r0 < last; r0 += MT * 16) {
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
    struct Buffer { uint4 a[kBatch][MT][2], b[kBatch][NT][2]; };
    int next = warp;                           // the item that is loaded next
    auto load = [&](Buffer& v) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j, next += kFewWarps) {
        const int d = min(next / steps, plan.reached - 1), k0 = (next - d * steps) * 32 + c8, e = plan.list[d];
        const bool ok = next < items && k0 < p.I;
        const __nv_bfloat16* w = p.w2 + ((long long)e * p.H + r0 + g) * p.I + k0;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          v.a[j][m][0] = few_weights(w + (long long)(m * 16) * p.I, ok && r0 + m * 16 + g < last);
          v.a[j][m][1] = few_weights(w + (long long)(m * 16 + 8) * p.I, ok && r0 + m * 16 + 8 + g < last);
        }
        const uint32_t mask = plan.mask[e];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int t = n * 8 + g;
          const bool on = ok && ((mask >> t) & 1);
          const __nv_bfloat16* ht = p.h + (long long)(t * p.k + (on ? plan.place[t][e] : 0)) * p.I + k0;
          v.b[j][n][0] = few_load(ht, on);
          v.b[j][n][1] = few_load(ht + plane, on);
        }
      }
    };
    auto take = [&](const Buffer& v) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            few_mma32(acc[m][n], v.a[j][m][0], v.a[j][m][1], v.b[j][n][0]);
            few_mma32(acc[m][n], v.a[j][m][0], v.a[j][m][1], v.b[j][n][1]);
          }
    };
    const int total = (items + kFewWarps * kBatch - 1) / (kFewWarps * kBatch);
    Buffer v0, v1;
    if (total > 0) load(v0);
    for (int q = 0; q < total; q += 2) {
      if (q + 1 < total) load(v1);
      take(v0);
      if (q + 1 >= total) break;
      if (q + 2 < total) load(v0);
      take(v1);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) red[warp][m][n][lane] = make_float4(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
    __syncthreads();
    for (int q = tid; q < MT * NT * 32; q += kFewThreads) {
      const int m = q / (NT * 32), n = q / 32 % NT, l = q & 31;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float4 part = red[w][m][n][l];
        v.x += part.x; v.y += part.y; v.z += part.z; v.w += part.w;
      }
#pragma unroll
      for (int o = 0; o < 4; ++o) {              // (rows l / 4 and 8 behind it, tokens 2 (l % 4) and the next)
        const int t = n * 8 + (l & 3) * 2 + (o & 1), r = r0 + m * 16 + (l >> 2) + (o >> 1) * 8;
        if (t < p.T && r < last) p.out[(long long)t * p.ldo + r] = __float2bfloat16(o == 0 ? v.x : o == 1 ? v.y : o == 2 ? v.z : v.w);
      }
    }
    __syncthreads();
  }
}

template <int NT>
static int moe_few_launch(const MoeFewParams& p, int num_sms, cudaStream_t s) {
  constexpr size_t smem = sizeof(float4) * kFewWarps * kFewTiles * 32;
  static bool set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(moe_few_up_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
    set[dev] = true;
  }
  launch_pdl(moe_few_up_kernel<NT>, dim3(num_sms), dim3(kFewThreads), smem, s, p);
  const int rows = (p.H + num_sms - 1) / num_sms;
  const dim3 grid(num_sms), block(kFewThreads);
  if (rows <= 16) launch_pdl(moe_few_down_kernel<1, NT>, grid, block, 0, s, p);
  else if (rows <= 32) launch_pdl(moe_few_down_kernel<2, NT>, grid, block, 0, s, p);
  else if (rows <= 48) launch_pdl(moe_few_down_kernel<3, NT>, grid, block, 0, s, p);
  else launch_pdl(moe_few_down_kernel<kFewRowTiles, NT>, grid, block, 0, s, p);
  return -(int)cudaGetLastError();
}

}  // namespace lx

extern "C" {

int lx_moe_few_max_tokens() { return lx::kFewTokens; }

int lx_moe_router_logits(const void* x, long long ldx, const void* wr, long long ldw, float* logits, int T, int E, int H, int* counts, int ncounts,
                         void* stream);

// `logits` [T, E], `ids` [T, k] and `h` [2, T k, I] are scratch of the call.
int lx_moe_few(const void* x, long long ldx, const void* wr, long long ldw, const void* w13, const void* w2, float* logits, int* ids, void* h, void* out, long long ldo, int T,
               int E, int k, int e0, int e_local, int H, int I, int act, int renorm, float scale, int num_sms, void* stream) {
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
  p.T = T; p.E = E; p.k = k; p.e0 = e0; p.e_local = e_local; p.H = H; p.I = I; p.act = act; p.renorm = renorm; p.scale = scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return T <= 8 ? moe_few_launch<1>(p, num_sms, s) : moe_few_launch<2>(p, num_sms, s);
}

}  // extern "C"
