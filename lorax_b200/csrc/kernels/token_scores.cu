// Scores of tokens from a row of logits x[0 .. V): log-probabilities of a given token and of the k best, and the entropy of the distribution.
//
//   c_i = x_i, or cap * tanh(x_i / cap);  m = max c;  s = sum exp(c_i - m);  u = sum (c_i - m) exp(c_i - m)
//   log p_i = (c_i - m) - log s;  entropy = -sum p_i log p_i = log s - u / s
//   best: by x descending, then by index ascending (the cap is monotone: it changes no order); a NaN orders as -inf
//
// One pass over the row with running m, s, u (a thread rescales its sums when its maximum grows), joined over lanes, warps and, where the rows
// alone do not fill the GPU, the CTAs of a cluster that share a row.  The sums are fp32: a thread adds some hundred terms of at most one, the
// rest is a tree.  Exponentials are the approximate ones (ex2.approx, __expf: within about 2^-22), logarithms and the cap's tanh are full.  A logit of -inf adds nothing; a row of nothing else, one with a NaN and one with +inf have no distribution and score NaN.
//
// The k best: of 64 groups of threads, each has a best element; the k-th best of those, by (value, index), is a lower bound of the row's k-th
// best, so only threads whose own best is at or above it can hold any (k 64 / (64 - k) or so of 512).  Their elements are read again (from L2),
// what is at or above the bound is listed, and the list is ranked by counting.  The order of (value, index) pairs is total, so the outcome
// depends on no order of execution.
//
// Without alternatives a kernel of its own has more rows on an SM (below).  With them a CTA is through with its row by some 4 us of joining, listing
// and ranking, beside one other CTA on its SM, and the pass itself is bound by its instructions (ten a logit), not by the HBM: 2048 rows of 128256 bf16
// take 124 us with 20 alternatives (4.3 TB/s; 115 with one), 4001 rows of 32000 101 us, 48 rows of 128256 fp32 12.4 us, one row of 32000 in eight CTAs
// 6.0 us, most of it launch, cluster and joins.
#include <algorithm>

#include "common.cuh"

namespace lx {

constexpr int kScoreThreads = 512;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxParts = 8;         // CTAs of a row (the portable cluster)
constexpr int kScoreMaxTop = 32;
constexpr int kScoreGroups = 64;          // of threads whose best elements set the bound: twice the most alternatives
constexpr int kScoreList = 2048;          // candidates that are ranked at once
constexpr int kScoreUnroll = 4;           // 16-byte loads of a thread in flight

// What the kernel with alternatives takes for granted of these numbers.  A row's single logits are read by the first threads of two warps, up to seven each
// (ScorePart::single); the warps' sums, and the parts', are joined by one warp.
static_assert(kScoreThreads % 32 == 0 && kScoreThreads >= 64 && kScoreWarps <= 32 && kScoreMaxParts <= 32, "whole warps, two of them, and no more sums than lanes");
// The threads of a group are neighbours within a warp, and so many threads share the comparisons of its best element, each with as many others.
constexpr int kScoreShare = kScoreThreads / kScoreGroups;
static_assert(kScoreShare * kScoreGroups == kScoreThreads && (kScoreShare & (kScoreShare - 1)) == 0 && kScoreShare <= 32 && kScoreGroups % kScoreShare == 0,
              "groups are a power of two of lanes");
// A bound exists only with as many groups as alternatives, an alternative has a thread of its own to write its place, and the list takes the best so far beside a
// portion of at least one wide load (eight elements).
static_assert(kScoreMaxTop <= kScoreGroups && kScoreMaxTop <= kScoreThreads && kScoreMaxTop + 8 <= kScoreList, "places for the alternatives");
// A pair's comparisons are shared by up to 32 neighbouring lanes of the same warp in rounds of all threads (score_rank).
static_assert(kScoreMaxParts * kScoreMaxTop <= kScoreList, "the parts' best are ranked like a list");

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

// The lanes' sums joined, in every lane.  (A side without a logit above -inf has s = u = 0, or NaN, which stays.)
LX_DEVICE ScoreSums score_join(ScoreSums a) {
  const float m = score_value(__reduce_max_sync(0xffffffffu, score_key(a.m)));
  const float d = a.m == -INFINITY ? 0.f : fmaxf(a.m - m, kScoreFloor), f = __expf(d);
  a.u = (a.u + d * a.s) * f;
  a.s *= f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  return ScoreSums{m, a.s, a.u};
}
// The first n of a list of at most 32.
LX_DEVICE ScoreSums score_join(const ScoreSums* list, int n) {
  const int lane = threadIdx.x & 31;
  return score_join(lane < n ? list[lane] : ScoreSums{-INFINITY, 0.f, 0.f});
}

LX_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

LX_DEVICE uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
LX_DEVICE float2 unpack_f32x2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
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

// 16 bytes of logits, or one (WIDE).  What lies past the end reads as -inf: it adds nothing.  values: those below `floor` are raised to it.  Tops pass over NaN.
template <typename L, bool WIDE>
struct ScoreLoad;
template <>
struct ScoreLoad<__nv_bfloat16, true> {
  static constexpr int kN = 8;
  using Raw = uint4;
  using Top = __nv_bfloat162;      // of even and odd elements
  LX_DEVICE static __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  LX_DEVICE static Raw load(const __nv_bfloat16* p, bool ok) { return ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  LX_DEVICE static void values(const Raw& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = __uint_as_float(w[q] << 16);
      x[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
    }
  }
  // (two elements an instruction; the floor is rounded: what is raised to it adds nothing all the same)
  LX_DEVICE static void values(const Raw& v, float (&x)[8], float floor) {
    const __nv_bfloat162 low = __float2bfloat162_rn(floor);
    auto up = [&](uint32_t w) {
      const __nv_bfloat162 r = __hmax2_nan(two(w), low);
      return *reinterpret_cast<const uint32_t*>(&r);
    };
    values(make_uint4(up(v.x), up(v.y), up(v.z), up(v.w)), x);
  }
  LX_DEVICE static Top top(const Raw& v) { return __hmax2(__hmax2(two(v.x), two(v.y)), __hmax2(two(v.z), two(v.w))); }
  LX_DEVICE static Top top(const Top& a, const Top& b) { return __hmax2(a, b); }
  LX_DEVICE static float value(const Top& a) { return fmaxf(__low2float(a), __high2float(a)); }
};
template <>
struct ScoreLoad<float, true> {
  static constexpr int kN = 4;
  using Raw = float4;
  using Top = float;
  LX_DEVICE static Raw load(const float* p, bool ok) { return ok ? *reinterpret_cast<const float4*>(p) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
  LX_DEVICE static void values(const Raw& v, float (&x)[4]) { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
  LX_DEVICE static void values(const Raw& v, float (&x)[4], float floor) {
    x[0] = max_nan(v.x, floor); x[1] = max_nan(v.y, floor); x[2] = max_nan(v.z, floor); x[3] = max_nan(v.w, floor);
  }
  LX_DEVICE static Top top(const Raw& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
  LX_DEVICE static Top top(Top a, Top b) { return fmaxf(a, b); }
  LX_DEVICE static float value(Top a) { return a; }
};
template <typename L>
struct ScoreLoad<L, false> {
  static constexpr int kN = 1;
  using Raw = float;
  using Top = float;
  LX_DEVICE static Raw load(const L* p, bool ok) { return ok ? (float)*p : -INFINITY; }
  LX_DEVICE static void values(const Raw& v, float (&x)[1]) { x[0] = v; }
  LX_DEVICE static void values(const Raw& v, float (&x)[1], float floor) { x[0] = max_nan(v, floor); }
  LX_DEVICE static Top top(const Raw& v) { return v; }
  LX_DEVICE static Top top(Top a, Top b) { return fmaxf(a, b); }
  LX_DEVICE static float value(Top a) { return a; }
};

// The target of row t, -1 where there is none.
LX_DEVICE int score_target(const TokenScoresParams& p, int t) {
  if (p.logprobs == nullptr) return -1;
  const long long target = p.wide_targets ? reinterpret_cast<const long long*>(p.targets)[t] : reinterpret_cast<const int*>(p.targets)[t];
  return target >= 0 && target < p.V ? (int)target : -1;
}
// Entropy of row t and the log-probability of its target, a logit (NaN: none), from the sums of the whole row.
template <bool CAP>
LX_DEVICE void score_row(const TokenScoresParams& p, int t, float given, const ScoreSums& all, float logs) {
  p.entropy[t] = logs - all.u / all.s;
  if (p.logprobs != nullptr) p.logprobs[t] = (score_cap<CAP>(given, p.softcap) - all.m) - logs;
}

// exp(c - m) is formed as 2^(log2e c + shift) with shift = -log2e m rounded: one FMA for two logits, whose products are not rounded.  What the rounding of
// the shift leaves out is the same for all terms and put right where the sums change hands.  Where the maximum is too far out for that (masks of the
// type's lowest value, infinities) the difference comes first.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Below 2048 the shift is rounded by at most 2^-13, and what the linear term of score_sums leaves of that is under 2^-27.
constexpr float kScoreFar = 2048.f;

LX_DEVICE bool score_far(float m) { return !(fabsf(m) < kScoreFar); }

struct ScoreThread {
  float m, shift;          // running maximum of the (capped) logits
  uint64_t s, u;           // running sums of e = 2^a and of a e, a = log2e c + shift, of even and odd elements
  float best;              // of the raw logits (TOP), and the first element of the first load that has it
  int place;
};

// The sums as they are for a shift that is not rounded, in natural logarithms.
LX_DEVICE ScoreSums score_sums(const ScoreThread& t) {
  const float2 s2 = unpack_f32x2(t.s), u2 = unpack_f32x2(t.u);
  const float s = s2.x + s2.y, u = u2.x + u2.y, off = score_far(t.m) ? 0.f : fmaf(kLog2e, t.m, t.shift);      // (at most half a step of the shift)
  const float f = 1.f - off * kLn2;                                                                           // 2^-off
  return ScoreSums{t.m, s * f, (u - off * s) * f * kLn2};
}

// R loads of a thread, the first from index i on, the others `step` further each; from `end` on they are not of the row (GUARD: there may be such).  Wide
// loads come in the order of the row; a single one may be in front of them.
template <typename Load, int R, bool TOP, bool CAP, bool GUARD>
LX_DEVICE void score_take(ScoreThread& t, const typename Load::Raw (&raw)[R], int i, int step, int end, float cap) {
  constexpr int N = Load::kN;
  typename Load::Top tops[R], all = tops[0] = Load::top(raw[0]);
#pragma unroll
  for (int r = 1; r < R; ++r) all = Load::top(all, tops[r] = Load::top(raw[r]));
  float top = Load::value(all);
  if (TOP && (top > t.best || (N == 1 && i < t.place && (top == top ? top : -INFINITY) == t.best))) {      // (NaN orders as -inf)
    t.best = fmaxf(t.best, top);
#pragma unroll
    for (int r = R - 1; r >= 0; --r)
      if (N == 1 || Load::value(tops[r]) == top) t.place = i + r * step;
  }
  top = score_cap<CAP>(top, cap);
  if (top > t.m) {
    const float shift = score_far(top) ? 0.f : -kLog2e * top;
    if (t.m != -INFINITY) {
      const float by = score_far(top) ? (score_far(t.m) ? (t.m - top) * kLog2e : -fmaf(kLog2e, top, t.shift))
                                      : (score_far(t.m) ? fmaf(kLog2e, t.m, shift) : shift - t.shift);
      const float d = fmaxf(by, kScoreFloor), f = exp2_fast(d);
      const uint64_t d2 = pack_f32x2(d, d), f2 = pack_f32x2(f, f);
      t.u = mul_f32x2(fma_f32x2(d2, t.s, t.u), f2);
      t.s = mul_f32x2(t.s, f2);
    }
    t.m = top;
    t.shift = shift;
  }
  auto add = [&](uint64_t a2, bool low) {
    float2 a = unpack_f32x2(a2);
    if (low) {
      a.x = max_nan(a.x, kScoreFloor);
      a.y = max_nan(a.y, kScoreFloor);
    }
    const uint64_t e = pack_f32x2(exp2_fast(a.x), exp2_fast(a.y));
    t.s = add_f32x2(t.s, e);
    t.u = fma_f32x2(pack_f32x2(a.x, a.y), e, t.u);
  };
  // two logits of a load; a single one has one of -inf beside it, which is raised to the floor
  auto pair = [&](const float (&x)[N], int q) {
    return pack_f32x2(score_cap<CAP>(x[q], cap), N > 1 ? score_cap<CAP>(x[(q + 1) % N], cap) : -INFINITY);
  };
  const uint64_t log2e = pack_f32x2(kLog2e, kLog2e);
  if (!score_far(t.m)) {
    const uint64_t shift = pack_f32x2(t.shift, t.shift);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (GUARD && CAP && r > 0 && i + r * step >= end) continue;      // (without a cap they are -inf and add nothing)
      float x[N];
      if (CAP) Load::values(raw[r], x);
      else Load::values(raw[r], x, t.m + kScoreFloor);
#pragma unroll
      for (int q = 0; q < N; q += 2) add(fma_f32x2(pair(x, q), log2e, shift), CAP || N == 1);
    }
  } else {
    const float m = t.m == -INFINITY ? 0.f : -t.m;      // (logits of -inf only, so far: they add zeros)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (GUARD && CAP && r > 0 && i + r * step >= end) continue;
      float x[N];
      Load::values(raw[r], x);
#pragma unroll
      for (int q = 0; q < N; q += 2) add(mul_f32x2(add_f32x2(pair(x, q), pack_f32x2(m, m)), log2e), true);
    }
  }
}

// A part [lo, hi) of a row: 16-byte loads from `body` to `whole`, where the row's alignment allows them; single logits in front and behind, one each for the
// first threads of two warps.
struct ScorePart {
  int lo, hi, body, whole;
  template <int N, typename L>
  LX_DEVICE static ScorePart of(const L* row, int V) {
    const int chunk = ((V + gridDim.y - 1) / gridDim.y + 7) & ~7;
    ScorePart s;
    s.lo = min((int)blockIdx.y * chunk, V);
    s.hi = min(s.lo + chunk, V);
    s.body = min(s.lo + (int)((0 - reinterpret_cast<uintptr_t>(row + s.lo) / sizeof(L)) & (N - 1)), s.hi);
    s.whole = s.body + (s.hi - s.body) / N * N;
    return s;
  }
  LX_DEVICE int single(int thread) const {
    if (thread < body - lo) return lo + thread;
    return thread >= 32 && thread - 32 < hi - whole ? whole + thread - 32 : -1;
  }
};

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
  int shift = 5;
  while (shift > 0 && n << shift > kScoreThreads) --shift;
  const int share = 1 << shift, at = threadIdx.x & (share - 1), rounds = ((n << shift) + kScoreThreads - 1) / kScoreThreads;
  for (int r = 0; r < rounds; ++r) {
    const int i = (threadIdx.x + r * kScoreThreads) >> shift;
    const unsigned long long a = i < n ? list[i] : 0;
    int above = 0;
    for (int j = at; j < n; j += share) above += list[j] > a;
    for (int o = share >> 1; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (i < n && at == 0 && above < k) own[above] = a;
  }
}

template <typename L, bool CAP>
__global__ void __launch_bounds__(kScoreThreads, 2) token_scores_kernel(const __grid_constant__ TokenScoresParams p) {
  using Load = ScoreLoad<L, true>;
  using One = ScoreLoad<L, false>;
  constexpr int kVec = Load::kN, kStep = kScoreThreads * kVec;
  __shared__ ScoreShared sh;
  const int t = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  if (parts > 1) cluster_arrive();      // (waited for in front of the first write to another CTA: it has started by then)
  pdl_wait();
  pdl_trigger();
  const L* row = reinterpret_cast<const L*>(p.logits) + (long long)t * p.ld;
  const ScorePart row_part = ScorePart::of<kVec>(row, p.V);
  const int whole = row_part.whole, single = row_part.single(tid);
  ScoreThread me{-INFINITY, 0.f, 0, 0, -INFINITY, -1};
  int i = row_part.body + tid * kVec;
  if (i < whole) me.place = i;
  else if (single >= 0) me.place = single;
  for (; i + (kScoreUnroll - 1) * kStep < whole; i += kScoreUnroll * kStep) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, true);
    score_take<Load, kScoreUnroll, true, CAP, false>(me, raw, i, kStep, whole, p.softcap);
  }
  if (i < whole) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, i + r * kStep < whole);
    score_take<Load, kScoreUnroll, true, CAP, true>(me, raw, i, kStep, whole, p.softcap);
  }
  if (single >= 0) {
    const float raw[1] = {One::load(row + single, true)};
    score_take<One, 1, true, CAP, false>(me, raw, single, 0, p.V, p.softcap);
  }

  // sums of the CTA
  const int target = tid == 0 ? score_target(p, t) : -1;      // (its loads are on their way while the sums are joined)
  ScoreSums a = score_join(score_sums(me));
  if ((tid & 31) == 0) sh.warps[tid >> 5] = a;
  const float given = target >= 0 ? One::value(One::load(row + target, true)) : NAN;
  // A thread's best element is one of those from `place` on that came in one load: it ranks between these two pairs.
  const bool live = me.place >= 0;
  const unsigned long long mine = live ? score_pair(score_key(me.best), me.place) : 0;
  unsigned long long g = live ? score_pair(score_key(me.best), me.place + (me.place == single ? 0 : kVec - 1)) : 0;
#pragma unroll
  for (int o = 1; o < kScoreShare; o <<= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, g, o);
    g = other > g ? other : g;
  }
  if ((tid & (kScoreShare - 1)) == 0) sh.group[tid / kScoreShare] = g;
  if (tid == 0) {
    sh.ncand = sh.n = 0;
    sh.bound = 0;
  }
  __syncthreads();
  if (tid < 32) a = score_join(sh.warps, kScoreWarps);

  // the bound: the k-th best of the groups' best, or none where there are fewer
  const int k = p.k;
  {
    const unsigned long long g = sh.group[tid / kScoreShare];
    int above = 0;
#pragma unroll
    for (int j = 0; j < kScoreGroups / kScoreShare; ++j) above += sh.group[(tid & (kScoreShare - 1)) + j * kScoreShare] > g;
#pragma unroll
    for (int o = kScoreShare / 2; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (g != 0 && above == k - 1 && (tid & (kScoreShare - 1)) == 0) sh.bound = g;
  }
  __syncthreads();
  const unsigned long long bound = sh.bound;
  if (live && mine >= bound) sh.cand[atomicAdd(&sh.ncand, 1)] = tid;
  __syncthreads();
  const int ncand = sh.ncand;
  const int its = (whole - row_part.body + kStep - 1) / kStep;      // wide loads of a thread; its single element counts as one more
  auto push = [&](float x, int idx) {
    const unsigned long long pair = score_pair(score_key(x), idx);
    if (pair >= bound) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < kScoreList) sh.list[at] = pair;
    }
  };
  const float low = score_value((uint32_t)(bound >> 32));      // (no number where there is no bound: nothing is below it)
  auto collect = [&](int c, int it) {
    if (it == its) {
      const int one = row_part.single(c);
      if (one >= 0) push(One::value(One::load(row + one, true)), one);
      return;
    }
    const int from = row_part.body + (it * kScoreThreads + c) * kVec;
    if (from >= whole) return;
    const typename Load::Raw raw = Load::load(row + from, true);
    if (Load::value(Load::top(raw)) < low) return;
    float x[kVec];
    Load::values(raw, x);
#pragma unroll
    for (int q = 0; q < kVec; ++q) push(x[q], from + q);
  };
  const int lanes = its > 1 ? min(32 - __clz(its - 1), 5) : 0;      // (a power of two of neighbours for a candidate)
  for (int c = tid >> lanes; c < ncand; c += kScoreThreads >> lanes)
    for (int it = tid & ((1 << lanes) - 1); it < its; it += 1 << lanes) collect(sh.cand[c], it);
  if (tid < ncand) collect(sh.cand[tid], its);
  __syncthreads();
  if (sh.n <= kScoreList) {
    score_rank(sh.list, sh.n, k, sh.own);
  } else {
    // more than the list holds (large logits side by side in the threads' strides): portions that fit, with the best so far among them
    constexpr int kPortion = (kScoreList - kScoreMaxTop) / kVec;
    static_assert(kPortion >= 1 && kPortion * kVec + kScoreMaxTop <= kScoreList, "a portion and the best so far fit the list");
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
  const ScoreSums all = score_join(sh.parts, parts);
  const float logs = logf(all.s);
  if (tid == 0) score_row<CAP>(p, t, given, all, logs);
  for (int j = tid; j < p.k; j += 32) {
    const unsigned long long pair = sh.own[j];
    p.top_ids[(long long)t * p.k + j] = (int)(0xffffffffu - (uint32_t)pair);
    p.top_logprobs[(long long)t * p.k + j] = (score_cap<CAP>(score_value((uint32_t)(pair >> 32)), p.softcap) - all.m) - logs;
  }
}

// ------------------------------------------------------------------------------------------------ without alternatives
// Bound by the HBM, and by the instructions of a logit (six, one of them the exponential, whose unit is busy for three quarters of the time): 2048 rows of
// 128256 bf16 in 87 us (6.1 TB/s), 4001 of 32000 in 45 (5.7 TB/s; with 512 threads a CTA, which reach the ends of their rows together, half as long
// again).  With a cap 1000 rows of 32000 take 49 us: tanhf.
constexpr int kLeanThreads = 256;
constexpr int kLeanWarps = kLeanThreads / 32;
template <typename L, bool CAP>
__global__ void __launch_bounds__(kLeanThreads, 6) token_logprobs_kernel(const __grid_constant__ TokenScoresParams p) {
  using Load = ScoreLoad<L, true>;
  using One = ScoreLoad<L, false>;
  constexpr int kVec = Load::kN, kStep = kLeanThreads * kVec;
  __shared__ ScoreSums warps[kLeanWarps], ends[kScoreMaxParts];      // (the latter of the cluster's first CTA)
  const int t = blockIdx.x, part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  if (parts > 1) cluster_arrive();      // (waited for in front of the first write to another CTA: it has started by then)
  pdl_wait();
  pdl_trigger();
  const L* row = reinterpret_cast<const L*>(p.logits) + (long long)t * p.ld;
  const ScorePart row_part = ScorePart::of<kVec>(row, p.V);
  const int whole = row_part.whole, single = row_part.single(tid);
  ScoreThread me{-INFINITY, 0.f, 0, 0, -INFINITY, -1};
  int i = row_part.body + tid * kVec;
  for (; i + (kScoreUnroll - 1) * kStep < whole; i += kScoreUnroll * kStep) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, true);
    score_take<Load, kScoreUnroll, false, CAP, false>(me, raw, i, kStep, whole, p.softcap);
  }
  if (i < whole) {
    typename Load::Raw raw[kScoreUnroll];
#pragma unroll
    for (int r = 0; r < kScoreUnroll; ++r) raw[r] = Load::load(row + i + r * kStep, i + r * kStep < whole);
    score_take<Load, kScoreUnroll, false, CAP, true>(me, raw, i, kStep, whole, p.softcap);
  }
  if (single >= 0) {
    const float raw[1] = {One::load(row + single, true)};
    score_take<One, 1, false, CAP, false>(me, raw, single, 0, p.V, p.softcap);
  }
  const int target = tid == 0 ? score_target(p, t) : -1;      // (its loads are on their way while the sums are joined)
  ScoreSums a = score_join(score_sums(me));
  if ((tid & 31) == 0) warps[tid >> 5] = a;
  const float given = target >= 0 ? One::value(One::load(row + target, true)) : NAN;
  __syncthreads();
  if (tid < 32) a = score_join(warps, kLeanWarps);
  if (parts > 1) {
    cluster_wait();
    if (tid == 0) {
      const uint32_t to = smem_u32(&ends[part]);
      cluster_store_f32(to, 0, a.m);
      cluster_store_f32(to + 4, 0, a.s);
      cluster_store_f32(to + 8, 0, a.u);
    }
    cluster_sync();      // (the parts have arrived)
    if (part != 0 || tid >= 32) return;
    a = score_join(ends, parts);
  }
  if (tid == 0) score_row<CAP>(p, t, given, a, logf(a.s));
}

// SMs of the current device.
static int score_sms() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) {
    int n = 0;
    sms[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
  }
  return sms[dev];
}

template <typename L>
static int token_scores_launch(const TokenScoresParams& p, int T, int parts, cudaStream_t s) {
  void (*kernel)(TokenScoresParams);
  if (p.k > 0) kernel = p.softcap > 0.f ? token_scores_kernel<L, true> : token_scores_kernel<L, false>;
  else kernel = p.softcap > 0.f ? token_logprobs_kernel<L, true> : token_logprobs_kernel<L, false>;
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
  // CTAs of a row: enough of them for two per SM, and at least one load per thread.  Without alternatives up to the six that an SM holds, of 16384 logits and
  // more (rows of 128256 bf16: 96 of them 12.4 -> 10.7 us, 200 19.7 -> 13.9, 440 24.4 -> 22.9; halves of 32000: 300 rows 7.6 -> 9.0).
  const int vec = fp32 ? 4 : 8;
  const int sms = score_sms();
  int parts = 1;
  while (parts < kScoreMaxParts && (long long)T * parts * 2 <= 2 * sms && V >= parts * kScoreThreads * vec) parts *= 2;
  if (k == 0) parts = std::max(parts, std::min({kScoreMaxParts, 6 * sms / T, V / 16384}));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return fp32 ? token_scores_launch<float>(p, T, parts, s) : token_scores_launch<__nv_bfloat16>(p, T, parts, s);
}

}  // extern "C"
