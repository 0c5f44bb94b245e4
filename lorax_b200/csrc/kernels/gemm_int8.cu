// Products of 8-bit integers with a scale for each token and each output channel, on the 5th-generation tensor cores:
//   out[t, n] = (sum_k xq[t, k] * wq[n, k]) * ws[n] * xs[t] + bias[n]
// The sums are whole numbers in 32 bits (tcgen05.mma.kind::i8, exact for K up to 2^17: 2^17 * 127 * 128 < 2^31), so that no order in which parts of
// K are added changes a result; scales and bias are applied in 32-bit floating point, the
// weights' first (rows of any size then overflow only where their results do), and the result is rounded to bf16 once.
//
// Weights take the UMMA M side, 128 output features a tile; tokens the N side in steps of 16.  A stage of the ring is 128 bytes of K of both.
// Where there are fewer tiles than SMs the CTAs of a cluster share a tile's K and add their sums up through each other's shared memory: nothing is
// kept in global memory between CTAs, calls or graphs.
//
// The reference has no such product (it expands 8-bit integer weights beside bf16 activations, server/lorax_server/layers/eetq.py:1-26).
#include "common.cuh"

namespace lx {

constexpr int kI8BM = 128;                        // output features of a tile
constexpr int kI8BK = 128;                        // bytes of K in a stage: one row of the 128-byte swizzle
constexpr int kI8Threads = 128;
constexpr int kI8MaxStages = 16;
constexpr int kI8MaxParts = 8;                    // CTAs that share a tile's K: a portable cluster
constexpr int kI8ABytes = kI8BM * kI8BK;

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

// Results of four features of one token.
LX_DEVICE void int8_store4(const Int8GemmParams& p, int t, int n, int4 s) {
  const float xs = p.xs[t];
  const int v[4] = {s.x, s.y, s.z, s.w};
  float f[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int at = min(n + q, p.N - 1);
    f[q] = (float)v[q] * p.ws[at] * xs + (p.bias != nullptr ? __bfloat162float(p.bias[at]) : 0.f);
  }
  __nv_bfloat16* o = p.out + (long long)t * p.ldo + n;
  if (p.wide && n + 4 <= p.N) {
    *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n + q < p.N) o[q] = __float2bfloat16(f[q]);
  }
}

// One tile a cluster, one part of its K a CTA.  Warp 0 loads, warp 1 multiplies, all four write results.
__global__ void __launch_bounds__(kI8Threads)
gemm_int8_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = kI8ABytes + p.bn * kI8BK;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + p.stages * stage_bytes);
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
  }

  // (done: every load of this CTA has arrived and been read, so the ring is free)
  bool ok = mbar_wait(done_bar, 0, abort_flag);
  if (!ok) {
    report_status(p.status, kTimeoutTmemFull, item);
    *abort_flag = 1;
    // copies still on their way arrive before this CTA leaves
    if (threadIdx.x == 0)
      for (int s = 0; s < min(p.stages, loaded); ++s) mbar_wait(&full_bar[s], (uint32_t)((loaded - 1 - s) / p.stages) & 1u, nullptr);
  }
  const int t0 = tb * p.bn, live = min(p.bn, p.T - t0);
  if (ok) {
    tc_fence_after();
    const uint32_t taddr = tmem_d + ((uint32_t)(warp * 32) << 16);
    for (int c = 0; c < live; c += 16) {
      uint32_t r[16];
      tmem_ld_32x32b_x16(taddr + c, r);
      tc_wait_ld();
#pragma unroll
      for (int q = 0; q < 16; ++q)
        if (c + q < live) sums[(c + q) * kI8BM + warp * 32 + lane] = (int)r[q];
    }
    tc_fence_before();
  }
  if (p.parts > 1) cluster_sync();
  else __syncthreads();
  // four features of a token at a time, in turn over the cluster's threads
  const int4* mine = reinterpret_cast<const int4*>(sums);
  for (int u = part * kI8Threads + (int)threadIdx.x; u < live * (kI8BM / 4); u += p.parts * kI8Threads) {
    const int n = ta * kI8BM + u % (kI8BM / 4) * 4;
    if (n >= p.N) continue;
    int4 s = make_int4(0, 0, 0, 0);
    if (p.parts > 1) {
      int4 v[kI8MaxParts];
#pragma unroll
      for (int r = 0; r < kI8MaxParts; ++r)
        if (r < p.parts) v[r] = cluster_load_int4(smem_u32(mine + u), (uint32_t)r);
#pragma unroll
      for (int r = 0; r < kI8MaxParts; ++r)
        if (r < p.parts) { s.x += v[r].x; s.y += v[r].y; s.z += v[r].z; s.w += v[r].w; }
    } else {
      s = mine[u];
    }
    if (ok) int8_store4(p, t0 + u / (kI8BM / 4), n, s);
  }
  if (p.parts > 1) cluster_sync();      // nobody leaves while its sums are read
  else __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_d, (uint32_t)p.tmem_cols); }
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
  int bn, stages, parts, tmem_cols, smem;
};
static Int8Plan int8_plan(int T, int N, int K, int num_sms) {
  Int8Plan w{};
  const int t16 = (T + 15) / 16 * 16, token_tiles = (t16 + 255) / 256;
  w.bn = ((t16 + token_tiles - 1) / token_tiles + 15) / 16 * 16;
  const int kblocks = (K + kI8BK - 1) / kI8BK;
  const long long tiles = (long long)((N + kI8BM - 1) / kI8BM) * ((T + w.bn - 1) / w.bn);
  w.parts = 1;
  while (w.parts < kI8MaxParts && tiles * w.parts < num_sms && kblocks >= 4 * (w.parts + 1)) ++w.parts;
  const int stage = kI8ABytes + w.bn * kI8BK;
  const int room = w.bn <= 64 ? 108 * 1024 : 216 * 1024;      // two CTAs an SM of small tiles, or one
  w.stages = room / stage < kI8MaxStages ? room / stage : kI8MaxStages;
  const int most = (kblocks + w.parts - 1) / w.parts;
  if (w.stages > most) w.stages = most > 4 ? most : 4;
  w.tmem_cols = 32;
  while (w.tmem_cols < w.bn) w.tmem_cols *= 2;
  w.smem = w.stages * stage + (2 * kI8MaxStages + 1) * 8 + 16 + 1024;
  return w;
}

}  // namespace lx

extern "C" {

int lx_gemm_int8_max_k() { return 1 << 17; }

// out[T, N] (bf16) = xq[T, K] wq[N, K]^T * xs[T] * ws[N] + bias[N].  Rows of xq and wq are ldq and ldw bytes apart (multiples of 16).
// w_const: the kernel in front on the stream does not write wq.
int lx_gemm_int8(const void* xq, long long ldq, const void* xs, const void* wq, long long ldw, const void* ws, const void* bias, void* out, long long ldo,
                 int T, int N, int K, int w_const, int* status, int num_sms, void* stream) {
  using namespace lx;
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K > lx_gemm_int8_max_k() || ldq % 16 != 0 || ldw % 16 != 0) return -1000;
  const Int8Plan w = int8_plan(T, N, K, num_sms);
  const long long ctas = (long long)((N + kI8BM - 1) / kI8BM) * ((T + w.bn - 1) / w.bn) * w.parts;
  if (ctas > 0x7fffffffll) return -1001;
  Int8GemmParams p{};
  p.N = N; p.T = T; p.K = K;
  p.bn = w.bn; p.stages = w.stages; p.parts = w.parts; p.tmem_cols = w.tmem_cols;
  p.reuse = T > w.bn;
  p.xs = reinterpret_cast<const float*>(xs); p.ws = reinterpret_cast<const float*>(ws);
  p.bias = reinterpret_cast<const __nv_bfloat16*>(bias);
  p.out = reinterpret_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.wide = reinterpret_cast<uintptr_t>(out) % 8 == 0 && ldo % 4 == 0;
  p.status = status;
  p.w_const = w_const;
  CUtensorMap tw, tx;
  if (make_tmap_i8(&tw, wq, N, K, ldw, kI8BM)) return -1002;
  if (make_tmap_i8(&tx, xq, T, K, ldq, w.bn)) return -1003;
  static bool set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    if (e != cudaSuccess) return -(int)e;
    set[dev] = true;
  }
  launch_pdl_cluster(gemm_int8_kernel, dim3((unsigned)ctas), dim3(kI8Threads), dim3((unsigned)w.parts), (size_t)w.smem,
                     reinterpret_cast<cudaStream_t>(stream), tw, tx, p);
  return -(int)cudaGetLastError();
}

}  // extern "C"
