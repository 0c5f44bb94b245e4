// Scores of tokens from a row of logits x[0 .. V): log-probabilities of a given token and of the k best, and the entropy of the distribution.
//
//   c_i = x_i, or cap * tanh(x_i / cap);  m = max c;  s = sum exp(c_i - m);  u = sum (c_i - m) exp(c_i - m)
//   log p_i = (c_i - m) - log s;  entropy = -sum p_i log p_i = log s - u / s
//   best: by x descending, then by index ascending (the cap is monotone: it changes no order); a NaN orders as -inf
//
// One pass over the row with running m, s, u (a thread rescales its sums when its maximum grows), merged over lanes, warps and, where the rows
// alone do not fill the GPU, the CTAs of a cluster that share a row.  The sums are fp32: a thread adds some hundred terms of at most one, the
// rest is a tree.  A logit of -inf adds nothing; a row of nothing else, one with a NaN and one with +inf have no distribution and score NaN.
//
// The k best come from the threads' own best elements: the k-th best of those, by (value, index), is a lower bound of the row's k-th best, so
// only the elements of the k threads at or above it can take part.  Those threads' elements are read again (one in 512 / k of the row, from
// L2), what is at or above the bound is listed, and the list is ranked by counting.  The order of (value, index) pairs is total, so the outcome
// depends on no order of execution.
#include "common.cuh"

namespace lx {

constexpr int kScoreThreads = 512;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxParts = 8;         // CTAs of a row (the portable cluster)
constexpr int kScoreMaxTop = 32;
constexpr int kScoreList = 2048;          // candidates that are ranked at once
constexpr int kScoreUnroll = 4;           // 16-byte loads of a thread in flight

struct TokenScoresParams {
  const void* logits;
  long long ld;            // elements
  int V;
  const void* targets;     // [T] int32 or int64, or null
  int wide_targets;
  int k;
  float softcap;
  float* logprobs;         // [T] or null
  float* entropy;          // [T]
  int* top_ids;            // [T, k]
  float* top_logprobs;     // [T, k]
};

struct ScoreSums { float m, s, u; };

// exp(-200) is zero in fp32.  Differences are held above it: a lower one, times a sum or times its own exponential, could be infinite or no number
// (masks of -inf or of the type's lowest value).
constexpr float kScoreFloor = -200.f;

LX_DEVICE void score_merge(ScoreSums& a, const ScoreSums& b) {
  const float nm = fmaxf(a.m, b.m);
  // (a side without a logit above -inf has s = u = 0, or NaN, which stays)
  const float da = a.m == -INFINITY ? 0.f : fmaxf(a.m - nm, kScoreFloor), db = b.m == -INFINITY ? 0.f : fmaxf(b.m - nm, kScoreFloor);
  const float fa = __expf(da), fb = __expf(db);
  a.u = (a.u + da * a.s) * fa + (b.u + db * b.s) * fb;
  a.s = a.s * fa + b.s * fb;
  a.m = nm;
}

// Order of logits as an unsigned number; -0 is 0, NaN is -inf.
LX_DEVICE uint32_t score_key(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
LX_DEVICE float score_value(uint32_t key) { return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key); }
// (value, index) pairs as one number, larger is better.
LX_DEVICE unsigned long long score_pair(uint32_t key, int i) { return ((unsigned long long)key << 32) | (0xffffffffu - (uint32_t)i); }

LX_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename L>
struct ScoreLoad;
template <>
struct ScoreLoad<__nv_bfloat16> {
  static constexpr int kVec = 8;
  LX_DEVICE static void vec(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 f = unpack_bf16x2(w[q]);
      x[2 * q] = f.x;
      x[2 * q + 1] = f.y;
    }
  }
  LX_DEVICE static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};
template <>
struct ScoreLoad<float> {
  static constexpr int kVec = 4;
  LX_DEVICE static void vec(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
  LX_DEVICE static float one(const float* p) { return *p; }
};

struct ScoreThread {
  ScoreSums sums;
  float best;              // of the raw logits, with the lowest index that has it
  int index;
};

// N logits from index i on (indices only grow).
template <int N, bool TOP, bool CAP>
LX_DEVICE void score_take(ScoreThread& t, float (&x)[N], int i, float cap) {
  float top = x[0];
#pragma unroll
  for (int q = 1; q < N; ++q) top = fmaxf(top, x[q]);      // (passes over NaN)
  if (TOP && top > t.best) {
    t.best = top;
#pragma unroll
    for (int q = N - 1; q >= 0; --q)
      if (x[q] == top) t.index = i + q;
  }
  if constexpr (CAP) {
#pragma unroll
    for (int q = 0; q < N; ++q) x[q] = cap * tanhf(x[q] / cap);
    top = cap * tanhf(top / cap);
  }
  ScoreSums& a = t.sums;
  if (top > a.m) {
    if (a.m != -INFINITY) {
      const float d = fmaxf(a.m - top, kScoreFloor), f = __expf(d);
      a.u = (a.u + d * a.s) * f;
      a.s *= f;
    }
    a.m = top;
  }
  const float m = a.m == -INFINITY ? 0.f : a.m;      // (logits of -inf only, so far: they add zeros)
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float d = max_nan(x[q] - m, kScoreFloor);
    const float e = __expf(d);
    a.s += e;
    a.u = fmaf(d, e, a.u);
  }
}

struct ScoreShared {
  ScoreSums warps[kScoreWarps];
  ScoreSums parts[kScoreMaxParts];                             // (of the cluster's first CTA)
  unsigned long long best[kScoreMaxParts * kScoreMaxTop];      // the parts' best pairs, 0: none (of the cluster's first CTA)
  unsigned long long list[kScoreList];
  unsigned long long own[kScoreMaxTop];
  int cand[kScoreThreads];
  int ncand, n;
};

// The pairs list[0 .. n), ranked: own[r] = the r-th best, r < k; 0 where there are fewer.
LX_DEVICE void score_rank(const unsigned long long* list, int n, int k, unsigned long long* own) {
  if (threadIdx.x < k && (int)threadIdx.x >= n) own[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < n; i += kScoreThreads) {
    const unsigned long long a = list[i];
    int r = 0;
    for (int j = 0; j < n && r < k; ++j) r += list[j] > a;
    if (r < k) own[r] = a;
  }
}

template <typename L, bool VEC, bool TOP, bool CAP>
__global__ void __launch_bounds__(kScoreThreads) token_scores_kernel(const __grid_constant__ TokenScoresParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kVec = VEC ? ScoreLoad<L>::kVec : 1;
  __shared__ ScoreShared sh;
  const int t = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  const L* row = reinterpret_cast<const L*>(p.logits) + (long long)t * p.ld;
  const int chunk = ((p.V + parts - 1) / parts + 7) & ~7;
  const int lo = min(part * chunk, p.V), hi = min(lo + chunk, p.V);
  const int whole = lo + (hi - lo) / kVec * kVec;      // a thread's elements: kVec from lo + (it * threads + tid) * kVec on, and one from `whole` on
  ScoreThread me{{-INFINITY, 0.f, 0.f}, -INFINITY, -1};
  if (lo + tid * kVec < whole) me.index = lo + tid * kVec;
  else if (whole + tid < hi) me.index = whole + tid;
  constexpr int kStep = kScoreThreads * kVec;
  int i = lo + tid * kVec;
  for (; i + (kScoreUnroll - 1) * kStep < whole; i += kScoreUnroll * kStep) {
    float x[kScoreUnroll][kVec];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) {
      if constexpr (VEC) ScoreLoad<L>::vec(row + i + r * kStep, x[r]);
      else x[r][0] = ScoreLoad<L>::one(row + i + r * kStep);
    }
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) score_take<kVec, TOP, CAP>(me, x[r], i + r * kStep, p.softcap);
  }
  for (; i < whole; i += kStep) {
    float x[kVec];
    if constexpr (VEC) ScoreLoad<L>::vec(row + i, x);
    else x[0] = ScoreLoad<L>::one(row + i);
    score_take<kVec, TOP, CAP>(me, x, i, p.softcap);
  }
  if (whole + tid < hi) {
    float x[1] = {ScoreLoad<L>::one(row + whole + tid)};
    score_take<1, TOP, CAP>(me, x, whole + tid, p.softcap);
  }

  // sums of the CTA
  auto from_lane = [](const ScoreSums& a, int o) {
    return ScoreSums{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)};
  };
  ScoreSums a = me.sums;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) score_merge(a, from_lane(a, o));
  if ((tid & 31) == 0) sh.warps[tid >> 5] = a;
  if (tid == 0) sh.ncand = sh.n = 0;
  __syncthreads();
  if (parts > 1) cluster_sync();      // every CTA of the cluster has started: its shared memory may be written
  if (tid < 32) {
    a = sh.warps[tid & (kScoreWarps - 1)];
#pragma unroll
    for (int o = kScoreWarps / 2; o > 0; o >>= 1) score_merge(a, from_lane(a, o));
    if (tid == 0) {
      if (parts > 1) {
        const uint32_t to = smem_u32(&sh.parts[part]);
        cluster_store_f32(to, 0, a.m);
        cluster_store_f32(to + 4, 0, a.s);
        cluster_store_f32(to + 8, 0, a.u);
      } else {
        sh.parts[0] = a;
      }
    }
  }

  if constexpr (TOP) {
    // the bound: the k-th best (value, index) of the threads' own best
    const int k = p.k;
    const bool live = me.index >= 0;
    const uint32_t key = score_key(me.best);
    constexpr int kLow = sizeof(L) == 2 ? 16 : 0;      // a bf16's order is in the upper half
    uint32_t bound = 0;
    for (int b = 31; b >= kLow; --b) {
      const uint32_t at = bound | (1u << b);
      if (__syncthreads_count(live && key >= at) >= k) bound = at;
    }
    const int above = __syncthreads_count(live && (key >> kLow) > (bound >> kLow));
    const bool tie = live && (key >> kLow) == (bound >> kLow);
    const int ties = __syncthreads_count(tie);
    int limit = 0x7fffffff;                            // of the elements that equal the bound, those up to this index take part
    if (above + ties > k) {
      limit = 0;
      for (int b = 30; b >= 0; --b) {                  // the largest index with fewer than k - above ties below it is the last one
        const int at = limit | (1 << b);
        if (__syncthreads_count(tie && me.index < at) < k - above) limit = at;
      }
    }
    auto takes = [&](uint32_t x, int idx) { return (x >> kLow) > (bound >> kLow) || ((x >> kLow) == (bound >> kLow) && idx <= limit); };
    if (live && takes(key, me.index)) sh.cand[atomicAdd(&sh.ncand, 1)] = tid;
    __syncthreads();
    const int ncand = sh.ncand, warp = tid >> 5, lane = tid & 31;
    const int its = (whole - lo + kStep - 1) / kStep;
    auto push = [&](float x, int idx) {
      const uint32_t kx = score_key(x);
      if (takes(kx, idx)) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kScoreList) sh.list[at] = score_pair(kx, idx);
      }
    };
    // elements of thread c in its rounds [it0, it1), one round a lane; its last element with round `its`
    auto collect = [&](int c, int it0, int it1) {
      for (int it = it0 + lane; it < it1; it += 32) {
        if (it == its) {
          if (whole + c < hi) push(ScoreLoad<L>::one(row + whole + c), whole + c);
          continue;
        }
        const int from = lo + (it * kScoreThreads + c) * kVec;
        if (from >= whole) continue;
        float x[kVec];
        if constexpr (VEC) ScoreLoad<L>::vec(row + from, x);
        else x[0] = ScoreLoad<L>::one(row + from);
#pragma unroll
        for (int q = 0; q < kVec; ++q) push(x[q], from + q);
      }
    };
    for (int c = warp; c < ncand; c += kScoreWarps) collect(sh.cand[c], 0, its + 1);
    __syncthreads();
    if (sh.n <= kScoreList) {
      score_rank(sh.list, sh.n, k, sh.own);
    } else {
      // more than the list holds (large logits side by side in the threads' strides): portions that fit, with the best so far among them
      constexpr int kPortion = (kScoreList - kScoreMaxTop) / kVec / 32 * 32;
      int have = 0;
      for (int c = 0; c < ncand; ++c) {
        for (int it = 0; it <= its; it += kPortion) {
          __syncthreads();
          if (tid < have) sh.list[tid] = sh.own[tid];
          if (tid == 0) sh.n = have;
          __syncthreads();
          if (warp == 0) collect(sh.cand[c], it, min(it + kPortion, its + 1));
          __syncthreads();
          score_rank(sh.list, sh.n, k, sh.own);
          have = min(k, sh.n);
        }
      }
    }
    __syncthreads();
    if (parts > 1) {
      if (tid < k) {
        const uint32_t to = smem_u32(&sh.best[part * kScoreMaxTop + tid]);
        cluster_store_f32(to, 0, __uint_as_float((uint32_t)sh.own[tid]));
        cluster_store_f32(to + 4, 0, __uint_as_float((uint32_t)(sh.own[tid] >> 32)));
      }
      cluster_sync();      // (the parts have arrived)
      if (part != 0) return;
      // empty places are zeros and rank behind every pair
      for (int j = tid; j < parts * kScoreMaxTop; j += kScoreThreads) sh.list[j] = (j & (kScoreMaxTop - 1)) < k ? sh.best[j] : 0;
      __syncthreads();
      score_rank(sh.list, parts * kScoreMaxTop, k, sh.own);
      __syncthreads();
    }
  } else if (parts > 1) {
    cluster_sync();
    if (part != 0) return;
  } else {
    __syncthreads();
  }

  if (tid >= 32) return;
  ScoreSums all = sh.parts[0];
  for (int c = 1; c < parts; ++c) score_merge(all, sh.parts[c]);
  const float logs = logf(all.s);
  auto capped = [&](float x) { return CAP ? p.softcap * tanhf(x / p.softcap) : x; };
  if (tid == 0) {
    p.entropy[t] = logs - all.u / all.s;
    if (p.logprobs != nullptr) {
      const long long target = p.targets == nullptr ? -1
                               : p.wide_targets     ? reinterpret_cast<const long long*>(p.targets)[t]
                                                    : reinterpret_cast<const int*>(p.targets)[t];
      float lp = NAN;
      if (target >= 0 && target < p.V) lp = (capped(ScoreLoad<L>::one(row + target)) - all.m) - logs;
      p.logprobs[t] = lp;
    }
  }
  if constexpr (TOP) {
    for (int j = tid; j < p.k; j += 32) {
      const unsigned long long pair = sh.own[j];
      p.top_ids[(long long)t * p.k + j] = (int)(0xffffffffu - (uint32_t)pair);
      p.top_logprobs[(long long)t * p.k + j] = (capped(score_value((uint32_t)(pair >> 32))) - all.m) - logs;
    }
  }
}

template <typename L, bool VEC>
static int token_scores_launch(const TokenScoresParams& p, int T, int parts, cudaStream_t s) {
  void (*kernel)(TokenScoresParams);
  if (p.softcap > 0.f) kernel = p.k > 0 ? token_scores_kernel<L, VEC, true, true> : token_scores_kernel<L, VEC, false, true>;
  else kernel = p.k > 0 ? token_scores_kernel<L, VEC, true, false> : token_scores_kernel<L, VEC, false, false>;
  const cudaError_t e = launch_pdl_cluster(kernel, dim3(T, parts), dim3(kScoreThreads), dim3(1, parts), 0, s, p);
  return e != cudaSuccess ? -(int)e : -(int)cudaGetLastError();
}

}  // namespace lx

extern "C" {

int lx_token_scores_max_top() { return lx::kScoreMaxTop; }

// fp32: the logits are fp32 instead of bf16.  `targets` may be null (then `logprobs` is too); one outside [0, V) scores NaN.
int lx_token_scores(const void* logits, long long ld, int fp32, int T, int V, const void* targets, int wide_targets, int k, float softcap,
                    float* logprobs, float* entropy, int* top_ids, float* top_logprobs, void* stream) {
  using namespace lx;
  if (T < 0 || V <= 0 || k < 0 || k > kScoreMaxTop || k > V || softcap < 0.f || (T > 1 && ld < V)) return -1;
  if (T == 0) return 0;
  TokenScoresParams p{logits, ld, V, targets, wide_targets, k, softcap, logprobs, entropy, top_ids, top_logprobs};
  // CTAs of a row: enough of them for two per SM, and at least one load per thread
  const int vec = fp32 ? 4 : 8;
  int parts = 1;
  while (parts < kScoreMaxParts && (long long)T * parts * 2 <= 2 * 148 && V >= parts * kScoreThreads * vec) parts *= 2;
  const bool aligned = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (T == 1 || ld % vec == 0);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (fp32) return aligned ? token_scores_launch<float, true>(p, T, parts, s) : token_scores_launch<float, false>(p, T, parts, s);
  return aligned ? token_scores_launch<__nv_bfloat16, true>(p, T, parts, s) : token_scores_launch<__nv_bfloat16, false>(p, T, parts, s);
}

}  // extern "C"
