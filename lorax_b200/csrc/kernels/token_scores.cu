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
// The k best: of 64 groups of threads, each has a best element; the k-th best of those, by (value, index), is a lower bound of the row's k-th
// best, so only threads whose own best is at or above it can hold any (k 64 / (64 - k) or so of 512).  Their elements are read again (from L2),
// what is at or above the bound is listed, and the list is ranked by counting.  The order of (value, index) pairs is total, so the outcome
// depends on no order of execution.
//
// Without alternatives a kernel of its own has more rows on an SM (lean, below).  With them the pass over the row is bound by its instructions, not
// by the HBM: 2048 rows of 128256 bf16 take 145 us with 20 alternatives (3.6 TB/s), 96 rows 12 us, one row of 32000 in eight CTAs 6.6 us, most of it
// launch, cluster and merges.
#include "common.cuh"

namespace lx {

constexpr int kScoreThreads = 512;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxParts = 8;         // CTAs of a row (the portable cluster)
constexpr int kScoreMaxTop = 32;
constexpr int kScoreGroups = 64;          // of threads whose best elements set the bound: twice the most alternatives
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

LX_DEVICE ScoreSums score_from_lane(const ScoreSums& a, int o) {
  return ScoreSums{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)};
}

template <bool CAP>
LX_DEVICE float score_cap(float x, float cap) { return CAP ? cap * tanhf(x / cap) : x; }

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

LX_DEVICE uint64_t pack_f32x2(float lo, float hi) { return ((uint64_t)__float_as_uint(hi) << 32) | __float_as_uint(lo); }
LX_DEVICE float2 unpack_f32x2(uint64_t v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }
LX_DEVICE uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
LX_DEVICE uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
LX_DEVICE uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
LX_DEVICE float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 16 bytes of logits (VEC), or one.  What lies past the end reads as -inf: it adds nothing.
template <typename L, bool VEC>
struct ScoreLoad;
template <>
struct ScoreLoad<__nv_bfloat16, true> {
  static constexpr int kN = 8;
  using Raw = uint4;
  LX_DEVICE static Raw load(const __nv_bfloat16* p, bool ok) { return ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  LX_DEVICE static void values(const Raw& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = __uint_as_float(w[q] << 16);
      x[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
    }
  }
  LX_DEVICE static float top(const Raw& v) {      // passes over NaN
    auto two = [](uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(two(v.x), two(v.y)), __hmax2(two(v.z), two(v.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct ScoreLoad<float, true> {
  static constexpr int kN = 4;
  using Raw = float4;
  LX_DEVICE static Raw load(const float* p, bool ok) { return ok ? *reinterpret_cast<const float4*>(p) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
  LX_DEVICE static void values(const Raw& v, float (&x)[4]) { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
  LX_DEVICE static float top(const Raw& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
};
template <>
struct ScoreLoad<__nv_bfloat16, false> {
  static constexpr int kN = 1;
  using Raw = float;
  LX_DEVICE static Raw load(const __nv_bfloat16* p, bool ok) { return ok ? __bfloat162float(*p) : -INFINITY; }
  LX_DEVICE static void values(const Raw& v, float (&x)[1]) { x[0] = v; }
  LX_DEVICE static float top(const Raw& v) { return v; }
};
template <>
struct ScoreLoad<float, false> {
  static constexpr int kN = 1;
  using Raw = float;
  LX_DEVICE static Raw load(const float* p, bool ok) { return ok ? *p : -INFINITY; }
  LX_DEVICE static void values(const Raw& v, float (&x)[1]) { x[0] = v; }
  LX_DEVICE static float top(const Raw& v) { return v; }
};

// Entropy of row t and the log-probability of its target, from the sums of the whole row.
template <typename L, bool CAP>
LX_DEVICE void score_row(const TokenScoresParams& p, int t, const L* row, const ScoreSums& all, float logs) {
  p.entropy[t] = logs - all.u / all.s;
  if (p.logprobs == nullptr) return;
  const long long target = p.wide_targets ? reinterpret_cast<const long long*>(p.targets)[t] : reinterpret_cast<const int*>(p.targets)[t];
  float lp = NAN;
  if (target >= 0 && target < p.V) lp = (score_cap<CAP>(ScoreLoad<L, false>::load(row + target, true), p.softcap) - all.m) - logs;
  p.logprobs[t] = lp;
}

struct ScoreThread {
  float m;                 // running maximum of the (capped) logits
  uint64_t s, u;           // running sums, of even and odd elements
  float best;              // of the raw logits, with the lowest index that has it
  int index;
};

// R loads of a thread, the first from index i on, the others `step` further each (indices only grow); from `end` on they are not of the row.
template <typename Load, int R, bool CAP>
LX_DEVICE void score_take(ScoreThread& t, const typename Load::Raw (&raw)[R], int i, int step, int end, float cap) {
  constexpr int N = Load::kN;
  float top = Load::top(raw[0]);
#pragma unroll
  for (int r = 1; r < R; ++r) top = fmaxf(top, Load::top(raw[r]));
  if (top > t.best) {
    t.best = top;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float x[N];
      Load::values(raw[r], x);
#pragma unroll
      for (int q = N - 1; q >= 0; --q)
        if (x[q] == top) t.index = i + r * step + q;
    }
  }
  top = score_cap<CAP>(top, cap);
  if (top > t.m) {
    if (t.m != -INFINITY) {
      const float d = fmaxf(t.m - top, kScoreFloor), f = __expf(d);
      const uint64_t d2 = pack_f32x2(d, d), f2 = pack_f32x2(f, f);
      t.u = mul_f32x2(fma_f32x2(d2, t.s, t.u), f2);
      t.s = mul_f32x2(t.s, f2);
    }
    t.m = top;
  }
  const float m = t.m == -INFINITY ? 0.f : t.m;      // (logits of -inf only, so far: they add zeros)
  const uint64_t m2 = pack_f32x2(-m, -m), log2e = pack_f32x2(1.4426950408889634f, 1.4426950408889634f);
  auto add = [&](float a, float b) {
    float2 d = unpack_f32x2(add_f32x2(pack_f32x2(a, b), m2));
    d.x = max_nan(d.x, kScoreFloor);
    d.y = max_nan(d.y, kScoreFloor);
    const uint64_t d2 = pack_f32x2(d.x, d.y);
    const float2 l = unpack_f32x2(mul_f32x2(d2, log2e));
    const uint64_t e = pack_f32x2(exp2_fast(l.x), exp2_fast(l.y));
    t.s = add_f32x2(t.s, e);
    t.u = fma_f32x2(d2, e, t.u);
  };
  auto capped = [&](float x, int r) { return r == 0 || i + r * step < end ? score_cap<CAP>(x, cap) : -INFINITY; };
  // (all values of the batch are formed before the chains of adds: N R is even but for the last element of a row)
  float x[R][N];
#pragma unroll
  for (int r = 0; r < R; ++r) Load::values(raw[r], x[r]);
  if constexpr (N > 1) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < N; q += 2) add(capped(x[r][q], r), capped(x[r][q + 1], r));
  } else {
#pragma unroll
    for (int r = 0; r < R; r += 2) add(capped(x[r][0], r), r + 1 < R ? capped(x[r + 1][0], r + 1) : -INFINITY);
  }
}

struct ScoreShared {
  ScoreSums warps[kScoreWarps];
  ScoreSums parts[kScoreMaxParts];                             // (of the cluster's first CTA)
  unsigned long long best[kScoreMaxParts * kScoreMaxTop];      // the parts' best pairs (of the cluster's first CTA)
  unsigned long long group[kScoreGroups];
  unsigned long long list[kScoreList];
  unsigned long long own[kScoreMaxTop];
  unsigned long long bound;
  int cand[kScoreThreads];
  int ncand, n;
};

// The pairs list[0 .. n), ranked by counting: own[r] = the r-th best, r < k; 0 where there are fewer.  Several neighbouring lanes share a pair's
// comparisons where there are threads for it.
LX_DEVICE void score_rank(const unsigned long long* list, int n, int k, unsigned long long* own) {
  if ((int)threadIdx.x < k && (int)threadIdx.x >= n) own[threadIdx.x] = 0;
  int share = 32;
  while (share > 1 && share * n > kScoreThreads) share >>= 1;
  const int at = threadIdx.x & (share - 1), rounds = (n * share + kScoreThreads - 1) / kScoreThreads;
  for (int r = 0; r < rounds; ++r) {
    const int i = (threadIdx.x + r * kScoreThreads) / share;
    const unsigned long long a = i < n ? list[i] : 0;
    int above = 0;
    for (int j = at; j < n; j += share) above += list[j] > a;
    for (int o = share >> 1; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (i < n && at == 0 && above < k) own[above] = a;
  }
}

template <typename L, bool VEC, bool CAP>
__global__ void __launch_bounds__(kScoreThreads, 2) token_scores_kernel(const __grid_constant__ TokenScoresParams p) {
  using Load = ScoreLoad<L, VEC>;
  constexpr int kVec = Load::kN, kStep = kScoreThreads * kVec;
  __shared__ ScoreShared sh;
  const int t = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  if (parts > 1) cluster_arrive();      // (waited for in front of the first write to another CTA: it has started by then)
  pdl_wait();
  pdl_trigger();
  const L* row = reinterpret_cast<const L*>(p.logits) + (long long)t * p.ld;
  const int chunk = ((p.V + parts - 1) / parts + 7) & ~7;
  const int lo = min(part * chunk, p.V), hi = min(lo + chunk, p.V);
  const int whole = lo + (hi - lo) / kVec * kVec;      // a thread's elements: kVec from lo + (it * threads + tid) * kVec on, and one from `whole` on
  ScoreThread me{-INFINITY, 0, 0, -INFINITY, -1};
  if (lo + tid * kVec < whole) me.index = lo + tid * kVec;
  else if (whole + tid < hi) me.index = whole + tid;
  for (int i = lo + tid * kVec; i < whole; i += kScoreUnroll * kStep) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, i + r * kStep < whole);
    score_take<Load, kScoreUnroll, CAP>(me, raw, i, kStep, whole, p.softcap);
  }
  if (VEC && whole + tid < hi) {
    using One = ScoreLoad<L, false>;
    const float raw[1] = {One::load(row + whole + tid, true)};
    score_take<One, 1, CAP>(me, raw, whole + tid, 0, hi, p.softcap);
  }

  // sums of the CTA
  const float2 s2 = unpack_f32x2(me.s), u2 = unpack_f32x2(me.u);
  ScoreSums a{me.m, s2.x + s2.y, u2.x + u2.y};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) score_merge(a, score_from_lane(a, o));
  if ((tid & 31) == 0) sh.warps[tid >> 5] = a;
  const bool live = me.index >= 0;
  const unsigned long long mine = live ? score_pair(score_key(me.best), me.index) : 0;
  unsigned long long g = mine;
#pragma unroll
  for (int o = 1; o < kScoreThreads / kScoreGroups; o <<= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, g, o);
    g = other > g ? other : g;
  }
  if ((tid & (kScoreThreads / kScoreGroups - 1)) == 0) sh.group[tid / (kScoreThreads / kScoreGroups)] = g;
  if (tid == 0) {
    sh.ncand = sh.n = 0;
    sh.bound = 0;
  }
  __syncthreads();
  if (tid < 32) {
    a = sh.warps[tid & (kScoreWarps - 1)];
#pragma unroll
    for (int o = kScoreWarps / 2; o > 0; o >>= 1) score_merge(a, score_from_lane(a, o));
  }

  // the bound: the k-th best of the groups' best, or none where there are fewer
  const int k = p.k;
  {
    constexpr int kShare = kScoreThreads / kScoreGroups;
    const unsigned long long g = sh.group[tid / kShare];
    int above = 0;
#pragma unroll
    for (int j = 0; j < kScoreGroups / kShare; ++j) above += sh.group[(tid & (kShare - 1)) + j * kShare] > g;
#pragma unroll
    for (int o = kShare / 2; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (g != 0 && above == k - 1 && (tid & (kShare - 1)) == 0) sh.bound = g;
  }
  __syncthreads();
  const unsigned long long bound = sh.bound;
  if (live && mine >= bound) sh.cand[atomicAdd(&sh.ncand, 1)] = tid;
  __syncthreads();
  const int ncand = sh.ncand;
  const int its = (whole - lo + kStep - 1) / kStep;      // loads of a thread; its single element counts as one more
  auto push = [&](float x, int idx) {
    const unsigned long long pair = score_pair(score_key(x), idx);
    if (pair >= bound) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < kScoreList) sh.list[at] = pair;
    }
  };
  auto collect = [&](int c, int it) {
    if (it == its) {
      if (VEC && whole + c < hi) push(ScoreLoad<L, false>::load(row + whole + c, true), whole + c);
      return;
    }
    const int from = lo + (it * kScoreThreads + c) * kVec;
    if (from >= whole) return;
    float x[kVec];
    Load::values(Load::load(row + from, true), x);
#pragma unroll
    for (int q = 0; q < kVec; ++q) push(x[q], from + q);
  };
  for (int q = tid; q < ncand * (its + 1); q += kScoreThreads) {
    const int c = q / (its + 1);
    collect(sh.cand[c], q - c * (its + 1));
  }
  __syncthreads();
  if (sh.n <= kScoreList) {
    score_rank(sh.list, sh.n, k, sh.own);
  } else {
    // more than the list holds (large logits side by side in the threads' strides): portions that fit, with the best so far among them
    constexpr int kPortion = (kScoreList - kScoreMaxTop) / kVec;
    int have = 0;
    for (int c = 0; c < ncand; ++c) {
      for (int it = 0; it <= its; it += kPortion) {
        __syncthreads();
        if (tid < have) sh.list[tid] = sh.own[tid];
        if (tid == 0) sh.n = have;
        __syncthreads();
        for (int q = it + tid; q < min(it + kPortion, its + 1); q += kScoreThreads) collect(sh.cand[c], q);
        __syncthreads();
        score_rank(sh.list, sh.n, k, sh.own);
        have = min(k, sh.n);
      }
    }
  }
  __syncthreads();

  if (parts > 1) {
    cluster_wait();
    if (tid == 0) {
      const uint32_t to = smem_u32(&sh.parts[part]);
      cluster_store_f32(to, 0, a.m);
      cluster_store_f32(to + 4, 0, a.s);
      cluster_store_f32(to + 8, 0, a.u);
    }
    if (tid < p.k) {
      const uint32_t to = smem_u32(&sh.best[part * p.k + tid]);
      cluster_store_f32(to, 0, __uint_as_float((uint32_t)sh.own[tid]));
      cluster_store_f32(to + 4, 0, __uint_as_float((uint32_t)(sh.own[tid] >> 32)));
    }
    cluster_sync();      // (the parts have arrived)
    if (part != 0) return;
    score_rank(sh.best, parts * p.k, p.k, sh.own);      // (empty places are zeros and rank behind every pair)
    __syncthreads();
  } else {
    if (tid == 0) sh.parts[0] = a;
    __syncthreads();
  }

  if (tid >= 32) return;
  ScoreSums all = sh.parts[0];
  for (int c = 1; c < parts; ++c) score_merge(all, sh.parts[c]);
  const float logs = logf(all.s);
  if (tid == 0) score_row<L, CAP>(p, t, row, all, logs);
  for (int j = tid; j < p.k; j += 32) {
    const unsigned long long pair = sh.own[j];
    p.top_ids[(long long)t * p.k + j] = (int)(0xffffffffu - (uint32_t)pair);
    p.top_logprobs[(long long)t * p.k + j] = (score_cap<CAP>(score_value((uint32_t)(pair >> 32)), p.softcap) - all.m) - logs;
  }
}

// ------------------------------------------------------------------------------------------------ without alternatives
// Bound by the HBM, and by the instructions of a logit: 2048 rows of 128256 bf16 in 86 us (6.1 TB/s), 4001 of 32000 in 51 (5.0 TB/s; with 512 threads a
// CTA, which reach the ends of their rows together, 63 to 72).  With a cap 1000 rows of 32000 take 50 us: tanhf.
// exp(c - m) is formed as 2^(log2e c + shift) with shift = -log2e m rounded: one FMA a logit, whose product is not rounded.  What the rounding of the
// shift leaves out is the same for all terms and put right where the sums change hands.  Where the maximum is too far out for that (masks of the
// type's lowest value, infinities) the difference comes first.
constexpr int kLeanThreads = 256;
constexpr int kLeanWarps = kLeanThreads / 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Below 2048 the shift is rounded by at most 2^-13, and what the linear term of lean_sums leaves of that is under 2^-27.
constexpr float kLeanFar = 2048.f;

LX_DEVICE bool lean_far(float m) { return !(fabsf(m) < kLeanFar); }

struct LeanThread {
  float m, shift;          // running maximum of the (capped) logits
  float s, u;              // running sums of e = 2^a and of a e, a = log2e c + shift
};

// The sums as they are for a shift that is not rounded, in natural logarithms.
LX_DEVICE ScoreSums lean_sums(const LeanThread& t) {
  const float off = lean_far(t.m) ? 0.f : fmaf(kLog2e, t.m, t.shift);      // (at most half a step of the shift)
  const float f = 1.f - off * kLn2;                                        // 2^-off
  return ScoreSums{t.m, t.s * f, (t.u - off * t.s) * f * kLn2};
}

// R loads of a thread, the first from index i on, the others `step` further each; from `end` on they are not of the row (GUARD: there may be such).
template <typename Load, int R, bool CAP, bool GUARD>
LX_DEVICE void lean_take(LeanThread& t, const typename Load::Raw (&raw)[R], int i, int step, int end, float cap) {
  float top = Load::top(raw[0]);
#pragma unroll
  for (int r = 1; r < R; ++r) top = fmaxf(top, Load::top(raw[r]));
  top = score_cap<CAP>(top, cap);
  if (top > t.m) {
    const float shift = lean_far(top) ? 0.f : -kLog2e * top;
    if (t.m != -INFINITY) {
      const float d = fmaxf(lean_far(top) || lean_far(t.m) ? (t.m - top) * kLog2e : shift - t.shift, kScoreFloor), f = exp2_fast(d);
      t.u = fmaf(d, t.s, t.u) * f;
      t.s *= f;
    }
    t.m = top;
    t.shift = shift;
  }
  auto add = [&](float a) {
    a = max_nan(a, kScoreFloor);
    const float e = exp2_fast(a);
    t.s += e;
    t.u = fmaf(a, e, t.u);
  };
  const bool far = lean_far(t.m);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (GUARD && r > 0 && i + r * step >= end) continue;
    float x[Load::kN];
    Load::values(raw[r], x);
    if (!far) {
#pragma unroll
      for (int q = 0; q < Load::kN; ++q) add(fmaf(score_cap<CAP>(x[q], cap), kLog2e, t.shift));
    } else {                             // (logits of -inf only, so far: they add zeros)
#pragma unroll 1
      for (int q = 0; q < Load::kN; ++q) add((score_cap<CAP>(x[q], cap) - (t.m == -INFINITY ? 0.f : t.m)) * kLog2e);
    }
  }
}

template <typename L, bool VEC, bool CAP>
__global__ void __launch_bounds__(kLeanThreads, 6) token_logprobs_kernel(const __grid_constant__ TokenScoresParams p) {
  using Load = ScoreLoad<L, VEC>;
  constexpr int kVec = Load::kN, kStep = kLeanThreads * kVec;
  __shared__ ScoreSums warps[kLeanWarps], ends[kScoreMaxParts];      // (the latter of the cluster's first CTA)
  const int t = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  if (parts > 1) cluster_arrive();      // (waited for in front of the first write to another CTA: it has started by then)
  pdl_wait();
  pdl_trigger();
  const L* row = reinterpret_cast<const L*>(p.logits) + (long long)t * p.ld;
  const int chunk = ((p.V + parts - 1) / parts + 7) & ~7;
  const int lo = min(part * chunk, p.V), hi = min(lo + chunk, p.V), whole = lo + (hi - lo) / kVec * kVec;
  LeanThread me{-INFINITY, 0.f, 0.f, 0.f};
  int i = lo + tid * kVec;
  for (; i + (kScoreUnroll - 1) * kStep < whole; i += kScoreUnroll * kStep) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, true);
    lean_take<Load, kScoreUnroll, CAP, false>(me, raw, i, kStep, whole, p.softcap);
  }
  if (i < whole) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, i + r * kStep < whole);
    lean_take<Load, kScoreUnroll, CAP, true>(me, raw, i, kStep, whole, p.softcap);
  }
  if (VEC && whole + tid < hi) {
    using One = ScoreLoad<L, false>;
    const float raw[1] = {One::load(row + whole + tid, true)};
    lean_take<One, 1, CAP, false>(me, raw, whole + tid, 0, hi, p.softcap);
  }
  ScoreSums a = lean_sums(me);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) score_merge(a, score_from_lane(a, o));
  if ((tid & 31) == 0) warps[tid >> 5] = a;
  __syncthreads();
  if (tid < 32) {
    a = warps[tid & (kLeanWarps - 1)];
#pragma unroll
    for (int o = kLeanWarps / 2; o > 0; o >>= 1) score_merge(a, score_from_lane(a, o));
  }
  if (parts > 1) {
    cluster_wait();
    if (tid == 0) {
      const uint32_t to = smem_u32(&ends[part]);
      cluster_store_f32(to, 0, a.m);
      cluster_store_f32(to + 4, 0, a.s);
      cluster_store_f32(to + 8, 0, a.u);
    }
    cluster_sync();      // (the parts have arrived)
    if (part != 0 || tid != 0) return;
    a = ends[0];
    for (int c = 1; c < parts; ++c) score_merge(a, ends[c]);
  }
  if (tid == 0) score_row<L, CAP>(p, t, row, a, logf(a.s));
}

template <typename L, bool VEC>
static int token_scores_launch(const TokenScoresParams& p, int T, int parts, cudaStream_t s) {
  void (*kernel)(TokenScoresParams);
  if (p.k > 0) kernel = p.softcap > 0.f ? token_scores_kernel<L, VEC, true> : token_scores_kernel<L, VEC, false>;
  else kernel = p.softcap > 0.f ? token_logprobs_kernel<L, VEC, true> : token_logprobs_kernel<L, VEC, false>;
  const cudaError_t e = launch_pdl_cluster(kernel, dim3(T, parts), dim3(p.k > 0 ? kScoreThreads : kLeanThreads), dim3(1, parts), 0, s, p);
  return e != cudaSuccess ? -(int)e : -(int)cudaGetLastError();
}

}  // namespace lx

extern "C" {

int lx_token_scores_max_top() { return lx::kScoreMaxTop; }

// fp32: the logits are fp32 instead of bf16.  `targets` may be null (then `logprobs` is too); one outside [0, V) scores NaN.
int lx_token_scores(const void* logits, long long ld, int fp32, int T, int V, const void* targets, int wide_targets, int k, float softcap,
                    float* logprobs, float* entropy, int* top_ids, float* top_logprobs, void* stream) {
  using namespace lx;
  if (T < 0 || V <= 0 || V >= 1 << 30 || k < 0 || k > kScoreMaxTop || k > V || !(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f)) || (T > 1 && ld < V) || (logprobs != nullptr && targets == nullptr)) return -1;
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
