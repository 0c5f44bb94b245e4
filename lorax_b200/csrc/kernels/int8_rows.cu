// Quantisers of rows for products in 8-bit integers (int8_rows.cuh states the numbers): rows as they are, or the activations of a feed-forward's
// gate and up halves, which then pass through memory once, as bytes, instead of being written in bf16 and read again.
#include <string.h>

#include "int8_rows.cuh"

namespace lx {

constexpr int kRowStages = 3;
constexpr int kRowRing = 108 * 1024;      // bytes of a block's stages, so that two blocks share an SM
// Rows an SM from which blocks that stay take them.  A compromise (us, a block per row and blocks that stay).  Activations of 14336: 200 rows 8.3 and 7.3, 400 12.6 and 11.8, 592
// 16.7 and 12.3, 4001 98 and 64; of 8192: 400 6.2 and 7.8, 592 8.1 and 8.3, 1000 11.5 and 12.6, 4001 36.3 and 36.2.  Rows as they are, of 14336: 400 6.8 and 8.5, 592 8.3 and 9.2, 1000
// 12.5 and 14.0, 4001 42.9 and 40.8; of 4096: 592 3.3 and 3.7, 1000 5.0 and 5.6, 4001 14.4 and 13.7.
constexpr int kRowRingRows = 4;

enum RowsAct : int { kRowsPlain = -1, kRowsSilu = 0, kRowsGelu = 1, kRowsGeluTanh = 2, kRowsRelu = 3, kRowsRelu2 = 4 };

// x / (1 + exp(-x)) = x * s for x >= 0, x * a * s below, with a = exp(-|x|), s = 1 / (1 + a): nothing overflows, small results keep their digits, and
// the reciprocal's argument lies in [1, 2], where the approximate one is within one last place.  A NaN stays one.
LX_DEVICE float times_sigmoid(float x, float z) {
  const float a = __expf(-fabsf(z));
  float s;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + a));
  return x * (z < 0.f ? a : 1.f) * s;
}

template <int ACT>
LX_DEVICE float rows_act(float x) {
  if (ACT == kRowsSilu) return times_sigmoid(x, x);
  if (ACT == kRowsGelu) return 0.5f * x * erfcf(-0.70710678118654752f * x);      // (1 + erf loses the digits of rows whose gates are all shut)
  if (ACT == kRowsGeluTanh) return times_sigmoid(x, 1.5957691216057308f * (x + 0.044715f * x * x * x));      // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
  if (ACT == kRowsRelu || ACT == kRowsRelu2) {
    const float r = x <= 0.f ? 0.f : x;      // (a NaN stays one)
    return ACT == kRowsRelu2 ? r * r : r;
  }
  return x;
}

struct RowsInt8Params {
  const __nv_bfloat16* x;      // [T, n], or [T, 2 n] gate and up
  long long ldx;
  int8_t* q;                   // [T, n]
  long long ldq;
  float* scale;                // [T]
  __nv_bfloat16* out;          // [T, n] the values themselves, or null
  long long ldo;
  int n, gated, T, stages;
  int* status;
};

// (M of rows that begin anywhere is kRowsShifted with a shift of 0: their bytes begin at 16, and that is where groups do)
template <int ACT, int M>
LX_DEVICE void rows_values(const RowsInt8Params& p, const VectorRaw& gate, const VectorRaw& up, int it, float (&f)[8], int in, int in_up) {
  vector_take<M>(gate, it, p.n, f, 0, in);
  if (ACT == kRowsPlain) return;
  float u[8];
  if (p.gated) vector_take<M>(up, it, p.n, u, 0, in_up);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    f[q] = rows_act<ACT>(f[q]);
    if (p.gated) f[q] *= u[q];
  }
}

template <int ACT, int M>
LX_DEVICE void rows_values(const RowsInt8Params& p, const __nv_bfloat16* row, int it, float (&f)[8], int in = 0, int in_up = 0) {
  const VectorRaw g = vector_fetch<M>(row, it, p.n, 0, in);
  rows_values<ACT, M>(p, g, ACT != kRowsPlain && p.gated ? vector_fetch<M>(row + p.n, it, p.n, 0, in_up) : g, it, f, in, in_up);
}

// One block per row: for few rows, whose own chain of loads, maximum and stores is the bound (one row of 14336 3.0 us, 256 of them 4.9, their activations 8.8).  NV: groups of eight that a thread keeps in registers between the pass for the maximum and the quotients; 0: any number, read and
// computed again (from L2: a row was read a moment ago).
template <int ACT, int NV, int M>
__global__ void __launch_bounds__(NV == 4 ? kRowThreads4 : 1024) rows_int8_kernel(const RowsInt8Params p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[32];
  const long long t = blockIdx.x;
  const __nv_bfloat16* row = p.x + t * p.ldx;
  float m = 0.f;
  const int in = M == kRowsShifted ? vector_in(row, 0) : 0, in_up = M == kRowsShifted ? vector_in(row + p.n, 0) : 0;
  constexpr int KEEP = NV > 0 ? NV : 1;
  float f[KEEP][8];
  const int passes = NV > 0 ? NV : (p.n + (int)blockDim.x * 8 - 1) / ((int)blockDim.x * 8);
  if (NV > 0) {
    VectorRaw g[KEEP], u[KEEP];
#pragma unroll
    for (int it = 0; it < KEEP; ++it) {
      g[it] = vector_fetch<M>(row, it, p.n, 0, in);
      if (ACT != kRowsPlain && p.gated) u[it] = vector_fetch<M>(row + p.n, it, p.n, 0, in_up);
    }
#pragma unroll
    for (int it = 0; it < KEEP; ++it) {
      rows_values<ACT, M>(p, g[it], u[it], it, f[it], in, in_up);
      m = largest_magnitude(m, f[it]);
    }
  } else {
    for (int it = 0; it < passes; ++it) {
      rows_values<ACT, M>(p, row, it, f[0], in, in_up);
      m = largest_magnitude(m, f[0]);
    }
  }
  const RowScale s = row_scale(block_max(m, red));
  if (threadIdx.x == 0) p.scale[t] = s.scale;
#pragma unroll
  for (int it = 0; it < (NV > 0 ? NV : passes); ++it) {
    if (NV == 0) rows_values<ACT, M>(p, row, it, f[0], in, in_up);
    row_store_int8<M>(p.q + t * p.ldq, it, p.n, f[NV > 0 ? it : 0], s);
    if (p.out != nullptr) {
      if (M == kRowsWide) {
        row_store<kRowsWide>(p.out + t * p.ldo, it, p.n, f[NV > 0 ? it : 0]);
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (row_has<M>(it, q, p.n, 0)) p.out[t * p.ldo + row_at<M>(it, q)] = __float2bfloat16(f[NV > 0 ? it : 0][q]);
      }
    }
  }
}

// Many rows: blocks that stay, whose next rows come by bulk copies while one is quantised; a row's values stand in registers from its maximum to its quotients,
// so that its stage is free between the two.  Bound by instructions (issue slots 70 to 74 %, two special functions a value of silu): 4001 rows of 14336 41 us (4.2 TB/s;
// a block per row 43), their activations 63 (4.6 TB/s; 98), 2048 of them 35.5.
template <int ACT, int NV>
__global__ void __launch_bounds__(kRowThreads4, 2) rows_int8_ring_kernel(const RowsInt8Params p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kRowStages];
  __shared__ uint32_t red[2][32];
  __shared__ int abort_word, fetched;
  volatile int* abort_flag = &abort_word;
  const int step = (int)gridDim.x;
  const uint32_t stage_bytes = (uint32_t)p.n * (p.gated ? 4 : 2);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    abort_word = fetched = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const auto fetch = [&](int t, int s) {
    ++fetched;
    mbar_expect_tx(&full[s], stage_bytes);
    bulk_load_1d(ring + s * stage_bytes, p.x + t * p.ldx, stage_bytes, &full[s]);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < p.stages && (int)blockIdx.x + s * step < p.T; ++s) fetch((int)blockIdx.x + s * step, s);
  int s = 0;
  uint32_t phase = 0;
  for (int row = (int)blockIdx.x, i = 0; row < p.T; row += step, ++i) {
    const long long t = row;
    if (!mbar_wait(&full[s], phase, abort_flag)) {      // (every thread goes on to the block's barriers all the same)
      report_status(p.status, kTimeoutFullBarrier, row);
      *abort_flag = 1;
    }
    float f[NV][8], m = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      rows_values<ACT, kRowsWide>(p, reinterpret_cast<const __nv_bfloat16*>(ring + s * stage_bytes), it, f[it]);
      m = largest_magnitude(m, f[it]);
    }
    const RowScale sc = row_scale(block_max(m, red[i & 1]));
    if (threadIdx.x == 0) {
      p.scale[t] = sc.scale;
      if (row + p.stages * step < p.T && !*abort_flag) fetch(row + p.stages * step, s);
    }
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      row_store_int8<kRowsWide>(p.q + t * p.ldq, it, p.n, f[it], sc);
      if (p.out != nullptr) row_store<kRowsWide>(p.out + t * p.ldo, it, p.n, f[it]);
    }
    if (++s == p.stages) { s = 0; phase ^= 1; }
  }
  if (threadIdx.x == 0 && *abort_flag)      // copies still on their way arrive before the block leaves
    for (int j = max(0, fetched - p.stages); j < fetched; ++j) mbar_wait(&full[j % p.stages], (uint32_t)(j / p.stages) & 1u, nullptr);
}

// Two blocks an SM by their registers; as many stages as fit then, up to three.
template <int ACT, int NV>
static int launch_rows_ring(RowsInt8Params p, int num_sms, cudaStream_t s) {
  const int threads = ((p.n / 8 + NV - 1) / NV + 31) / 32 * 32, stage = p.n * (p.gated ? 4 : 2);
  static bool set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(rows_int8_ring_kernel<ACT, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowRing);
    if (e != cudaSuccess) return -(int)e;
    set[dev] = true;
  }
  int blocks = 1024 / threads;
  if (blocks > 16) blocks = 16;
  p.stages = kRowRing / ((blocks + 1) / 2 * stage);
  p.stages = p.stages > kRowStages ? kRowStages : p.stages < 1 ? 1 : p.stages;
  const int grid = p.T < num_sms * blocks ? p.T : num_sms * blocks;
  launch_pdl(rows_int8_ring_kernel<ACT, NV>, dim3((unsigned)grid), dim3((unsigned)threads), (size_t)p.stages * stage, s, p);
  return -(int)cudaGetLastError();
}

template <int ACT, int M>
static int launch_rows(const RowsInt8Params& p, int num_sms, int ring, cudaStream_t s) {
  if (M == kRowsWide && p.n <= kRowThreads4 * 4 * 8 && (ring < 0 ? p.T >= kRowRingRows * num_sms : ring))
    return p.n <= kRowThreads4 * 2 * 8 ? launch_rows_ring<ACT, 2>(p, num_sms, s) : launch_rows_ring<ACT, 4>(p, num_sms, s);
  const RowShape r = row_shape(p.T, p.n, num_sms, 1024);
  const dim3 grid((unsigned)p.T), block((unsigned)r.threads);
  if (r.groups == 1) launch_pdl(rows_int8_kernel<ACT, 1, M>, grid, block, 0, s, p);
  else if (r.groups == 2) launch_pdl(rows_int8_kernel<ACT, 2, M>, grid, block, 0, s, p);
  else if (r.groups == 4) launch_pdl(rows_int8_kernel<ACT, 4, M>, grid, block, 0, s, p);
  else launch_pdl(rows_int8_kernel<ACT, 0, M>, grid, block, 0, s, p);
  return -(int)cudaGetLastError();
}

}  // namespace lx

extern "C" {

// In one block, as for lx_gemm_int8.
struct LxRowsInt8Args {
  const void* x;              // act < 0: [T, n] as it is; else act(x[:, :n]), times x[:, n : 2 n] where gated
  long long ldx;
  void* q;
  long long ldq;
  float* scale;
  void* out;                  // [T, n] bf16 or null
  long long ldo, T, n, act, gated;
  int* status;
  long long num_sms;
  long long ring;             // as of lx_norm_block
  void* stream;
};
int lx_rows_int8_bytes() { return (int)sizeof(LxRowsInt8Args); }

int lx_rows_int8(const char* args) {
  using namespace lx;
  LxRowsInt8Args a;
  memcpy(&a, args, sizeof(a));
  if (a.T <= 0) return 0;
  if (a.n <= 0 || a.n > (1 << 30) || a.T > kRowsMost) return -1;
  const void *x = a.x, *q = a.q, *out = a.out;
  const long long ldx = a.ldx, ldq = a.ldq, ldo = a.ldo;
  const int n = (int)a.n, num_sms = (int)a.num_sms, ring = (int)a.ring;
  RowsInt8Params p{reinterpret_cast<const __nv_bfloat16*>(x), ldx, reinterpret_cast<int8_t*>(a.q), ldq, a.scale, reinterpret_cast<__nv_bfloat16*>(a.out), ldo, n,
                   (int)a.gated, (int)a.T, 0, a.status};
  const auto at = [](const void* v) { return reinterpret_cast<uintptr_t>(v); };
  const bool wide = n % 8 == 0 && at(x) % 16 == 0 && ldx % 8 == 0 && at(q) % 8 == 0 && ldq % 8 == 0 && at(out) % 16 == 0 && ldo % 8 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(a.stream);
#define LX_ROWS(A) return wide ? launch_rows<A, kRowsWide>(p, num_sms, ring, s) : launch_rows<A, kRowsShifted>(p, num_sms, ring, s)
  switch (a.act) {
    case kRowsSilu: LX_ROWS(kRowsSilu);
    case kRowsGelu: LX_ROWS(kRowsGelu);
    case kRowsGeluTanh: LX_ROWS(kRowsGeluTanh);
    case kRowsRelu: LX_ROWS(kRowsRelu);
    case kRowsRelu2: LX_ROWS(kRowsRelu2);
    default: LX_ROWS(kRowsPlain);
  }
#undef LX_ROWS
}

}  // extern "C"
