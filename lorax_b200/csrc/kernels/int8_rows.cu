// Quantisers of rows for products in 8-bit integers (int8_rows.cuh states the numbers): rows as they are, or the activations of a feed-forward's
// gate and up halves, which then pass through memory once, as bytes, instead of being written in bf16 and read again.
//
// The reference has no such layers (its 8-bit integer weights meet bf16 activations, server/lorax_server/layers/eetq.py:1-26).
#include "int8_rows.cuh"

namespace lx {

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
  if (ACT == kRowsGelu) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
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
  int n, gated;
};

template <int ACT, bool WIDE>
LX_DEVICE void rows_values(const RowsInt8Params& p, const __nv_bfloat16* row, int it, float (&f)[8]) {
  row_load<WIDE>(row, it, p.n, f);
  if (ACT == kRowsPlain) return;
  float u[8];
  if (p.gated) row_load<WIDE>(row + p.n, it, p.n, u);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    f[q] = rows_act<ACT>(f[q]);
    if (p.gated) f[q] *= u[q];
  }
}

// One block per row.  NV: groups of eight that a thread keeps in registers between the pass for the maximum and the quotients; 0: any number, read and
// computed again (from L2: a row was read a moment ago).
template <int ACT, int NV, bool WIDE>
__global__ void __launch_bounds__(NV == 4 ? kRowThreads4 : 1024) rows_int8_kernel(const RowsInt8Params p) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[32];
  const long long t = blockIdx.x;
  const __nv_bfloat16* row = p.x + t * p.ldx;
  float m = 0.f;
  constexpr int KEEP = NV > 0 ? NV : 1;
  float f[KEEP][8];
  const int passes = NV > 0 ? NV : (p.n + (int)blockDim.x * 8 - 1) / ((int)blockDim.x * 8);
#pragma unroll
  for (int it = 0; it < (NV > 0 ? NV : passes); ++it) {
    rows_values<ACT, WIDE>(p, row, it, f[NV > 0 ? it : 0]);
    m = largest_magnitude(m, f[NV > 0 ? it : 0]);
  }
  const RowScale s = row_scale(block_max(m, red));
  if (threadIdx.x == 0) p.scale[t] = s.scale;
#pragma unroll
  for (int it = 0; it < (NV > 0 ? NV : passes); ++it) {
    if (NV == 0) rows_values<ACT, WIDE>(p, row, it, f[0]);
    row_store_int8<WIDE>(p.q + t * p.ldq, it, p.n, f[NV > 0 ? it : 0], s);
    if (p.out != nullptr) row_store<WIDE>(p.out + t * p.ldo, it, p.n, f[NV > 0 ? it : 0]);
  }
}

template <int ACT, bool WIDE>
static void launch_rows(const RowsInt8Params& p, int T, const RowShape& r, cudaStream_t s) {
  const dim3 grid((unsigned)T), block((unsigned)r.threads);
  if (r.groups == 1) launch_pdl(rows_int8_kernel<ACT, 1, WIDE>, grid, block, 0, s, p);
  else if (r.groups == 2) launch_pdl(rows_int8_kernel<ACT, 2, WIDE>, grid, block, 0, s, p);
  else if (r.groups == 4) launch_pdl(rows_int8_kernel<ACT, 4, WIDE>, grid, block, 0, s, p);
  else launch_pdl(rows_int8_kernel<ACT, 0, WIDE>, grid, block, 0, s, p);
}

}  // namespace lx

extern "C" {

// act < 0: x [T, n] as it is; else act(x[:, :n]), times x[:, n : 2 n] where gated.  out (bf16) may be null.
int lx_rows_int8(const void* x, long long ldx, void* q, long long ldq, void* scale, void* out, long long ldo, int T, int n, int act, int gated, int num_sms,
                 void* stream) {
  using namespace lx;
  if (T <= 0) return 0;
  if (n <= 0) return -1;
  RowsInt8Params p{reinterpret_cast<const __nv_bfloat16*>(x), ldx, reinterpret_cast<int8_t*>(q), ldq, reinterpret_cast<float*>(scale),
                   reinterpret_cast<__nv_bfloat16*>(out), ldo, n, gated};
  const auto at = [](const void* a) { return reinterpret_cast<uintptr_t>(a); };
  const bool wide = n % 8 == 0 && at(x) % 16 == 0 && ldx % 8 == 0 && at(q) % 8 == 0 && ldq % 8 == 0 && at(out) % 16 == 0 && ldo % 8 == 0;
  const RowShape r = row_shape(T, n, num_sms, 1024);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define LX_ROWS(A)                          \
  if (wide) launch_rows<A, true>(p, T, r, s); \
  else launch_rows<A, false>(p, T, r, s)
  switch (act) {
    case kRowsSilu: LX_ROWS(kRowsSilu); break;
    case kRowsGelu: LX_ROWS(kRowsGelu); break;
    case kRowsGeluTanh: LX_ROWS(kRowsGeluTanh); break;
    case kRowsRelu: LX_ROWS(kRowsRelu); break;
    case kRowsRelu2: LX_ROWS(kRowsRelu2); break;
    default: LX_ROWS(kRowsPlain); break;
  }
#undef LX_ROWS
  return -(int)cudaGetLastError();
}

}  // extern "C"
