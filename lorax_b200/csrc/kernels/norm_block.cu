// Norms on both sides of a block in one pass over its rows:
//   h = residual + scale * gate * N_post(y)         (N_post: left out without a weight of its own; gate: any of one, [T, 1], [H], [T, H])
//   x = N(h),  N(v) = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * (w + offset) + b      (RMS norm: without the means)
// h replaces the residual (or is written elsewhere) in bf16, and N reads the rounded h, as whoever reads the stream later does.  x leaves in bf16, in 8 bits
// with a scale for each row (int8_rows.cuh), from the same 32-bit values, or both.
#include <string.h>

#include "int8_rows.cuh"

namespace lx {

struct NormBlockParams {
  const __nv_bfloat16* y;              // [T, H], or null: h is the residual
  const __nv_bfloat16* residual;       // [T, H]
  __nv_bfloat16* residual_out;         // [T, H], may be the residual; null: not written
  const __nv_bfloat16* post_w;         // [H] or null
  const __nv_bfloat16* post_b;
  const __nv_bfloat16* w;              // [H]
  const __nv_bfloat16* b;              // [H] or null
  const __nv_bfloat16* gate;           // or null
  long long gate_t;                    // elements between two rows' gates (0: the same)
  int gate_h, gate_wide;               // 1: every channel has its own, 0: a row has one; rows of gates begin at 16 bytes
  __nv_bfloat16* out;                  // [T, H] or null
  int8_t* q;                           // [T, H] or null
  float* q_scale;
  long long ldy, ldr, ldro, ldo, ldq;
  int H, T;
  float eps, w_offset, scale;
  int* status;
};

// Sums over the block of up to three norms' passes, each with words of its own.
template <bool LAYERNORM, int NV, int M>
LX_DEVICE void norm_rows(float (&f)[NV][8], int H, float eps, float (*red)[32], int shift = 0) {
  float mean = 0.f;
  if (LAYERNORM) {
    float s = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it)
#pragma unroll
      for (int q = 0; q < 8; ++q) s += f[it][q];
    mean = block_sum(s, red[0]) / H;
  }
  float s = 0.f;
#pragma unroll
  for (int it = 0; it < NV; ++it)
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (LAYERNORM) f[it][q] = row_has<M>(it, q, H, shift) ? f[it][q] - mean : 0.f;
      s = fmaf(f[it][q], f[it][q], s);
    }
  const float r = rsqrtf(block_sum(s, red[1]) / H + eps);
#pragma unroll
  for (int it = 0; it < NV; ++it)
#pragma unroll
    for (int q = 0; q < 8; ++q) f[it][q] *= r;
}

template <int NV, int M>
LX_DEVICE void scale_rows(float (&f)[NV][8], int H, const VectorRaw (&raw)[NV], const __nv_bfloat16* b, float offset, int shift, int in) {
#pragma unroll
  for (int it = 0; it < NV; ++it) {
    float g[8];
    vector_take<M>(raw[it], it, H, g, shift, in);
#pragma unroll
    for (int q = 0; q < 8; ++q) f[it][q] *= g[q] + offset;
    if (b != nullptr) {
      vector_load<M>(b, it, H, g, shift, in);
#pragma unroll
      for (int q = 0; q < 8; ++q) f[it][q] += g[q];
    }
  }
}

template <int M>
LX_DEVICE void gates(const NormBlockParams& p, long long t, int it, float (&g)[8], int shift = 0) {
  const __nv_bfloat16* gate = p.gate + t * p.gate_t;
  if (p.gate_h == 0) {
    const float one = __bfloat162float(*gate);
#pragma unroll
    for (int q = 0; q < 8; ++q) g[q] = one;
  } else if (M != kRowsWide || p.gate_wide) {
    vector_load<M>(gate, it, p.H, g, shift, M == kRowsShifted ? vector_in(gate, shift) : 0);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) g[q] = row_has<M>(it, q, p.H, shift) ? __bfloat162float(gate[row_at<M>(it, q, shift)]) : 0.f;
  }
}

// One block per row; NV groups of eight a thread, all in registers, with the loads of rows and weights ahead of the first sum.  The chain of loads, sums over the block and
// stores is the bound: one row of 4096 2.1 us, in 8 bits 2.4; 259 rows 4.1.  Shifted rows are bound by instructions: 600 of 2049 6.4 us, as layer norms with gate and biases 9.6.
template <bool LAYERNORM, int NV, int M>
__global__ void __launch_bounds__(M != kRowsShifted ? kRowThreads4 : NV == 1 ? kRowShifted1 : kRowShifted2, M == kRowsShifted && NV == 1 ? 2 : 1) norm_block_kernel(const NormBlockParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[4][32];
  __shared__ uint32_t red_max[32];
  const long long t = blockIdx.x;
  const int H = p.H, shift = M == kRowsShifted ? (int)((reinterpret_cast<uintptr_t>(p.residual + t * p.ldr) & 15) >> 1) : 0;
  const int in = (8 - shift) & 7;                // (the vectors begin at 16 bytes)
  const __nv_bfloat16 *res = p.residual + t * p.ldr, *block = p.y + t * p.ldy;
  const Extent res_at = extent(p.residual, p.ldr, p.T, H), block_at = extent(p.y, p.ldy, p.T, H);
  uint4 hr[NV], yr[NV];
  VectorRaw wr[NV], pr[NV];
#pragma unroll
  for (int it = 0; it < NV; ++it) {
    hr[it] = row_fetch<M>(res, it, H, shift, res_at);
    if (p.y != nullptr) yr[it] = row_fetch<M>(block, it, H, shift, block_at);
  }
#pragma unroll
  for (int it = 0; it < NV; ++it) {
    if (p.post_w != nullptr) pr[it] = vector_fetch<M>(p.post_w, it, H, shift, in);
    wr[it] = vector_fetch<M>(p.w, it, H, shift, in);
  }
  float h[NV][8];
#pragma unroll
  for (int it = 0; it < NV; ++it) row_take<M>(hr[it], it, H, h[it], shift);
  if (p.y != nullptr) {
    float y[NV][8];
#pragma unroll
    for (int it = 0; it < NV; ++it) row_take<M>(yr[it], it, H, y[it], shift);
    if (p.post_w != nullptr) {
      norm_rows<LAYERNORM, NV, M>(y, H, p.eps, red, shift);
      scale_rows<NV, M>(y, H, pr, p.post_b, p.w_offset, shift, in);
    }
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      if (p.gate != nullptr) {
        float g[8];
        gates<M>(p, t, it, g, shift);
#pragma unroll
        for (int q = 0; q < 8; ++q) y[it][q] *= g[q];
      }
#pragma unroll
      for (int q = 0; q < 8; q += 2) {
        const float2 r = unpack_bf16x2(pack_bf16x2(fmaf(p.scale, y[it][q], h[it][q]), fmaf(p.scale, y[it][q + 1], h[it][q + 1])));
        h[it][q] = r.x;
        h[it][q + 1] = r.y;
      }
    }
  }
  if (p.residual_out != nullptr) {
#pragma unroll
    for (int it = 0; it < NV; ++it) row_store<M>(p.residual_out + t * p.ldro, it, H, h[it], shift);
  }
  norm_rows<LAYERNORM, NV, M>(h, H, p.eps, red + 2, shift);
  scale_rows<NV, M>(h, H, wr, p.b, p.w_offset, shift, in);
  if (p.out != nullptr) {
#pragma unroll
    for (int it = 0; it < NV; ++it) row_store<M>(p.out + t * p.ldo, it, H, h[it], shift);
  }
  if (p.q != nullptr) {
    float m = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      if (!row_whole<M>(it, H, shift)) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (!row_has<M>(it, q, H, shift)) h[it][q] = 0.f;      // (0 times a row's infinite or NaN factors)
      }
      m = largest_magnitude(m, h[it]);
    }
    const RowScale s = row_scale(block_max(m, red_max));
    if (threadIdx.x == 0) p.q_scale[t] = s.scale;
#pragma unroll
    for (int it = 0; it < NV; ++it) row_store_int8<M>(p.q + t * p.ldq, it, H, h[it], s, shift);
  }
}

// ------------------------------------------------------------------------------------------------
// Many rows: blocks that stay, with the next row of y and of the residual on its way by bulk copies (no registers, no waiting warps) while one is normed.
// Rows are read from shared memory as often as a pass needs them, so that a thread holds the values of one row only, and the norms' weights for all rows.  4001 rows of
// 8192: 44 us (6.0 TB/s: HBM), a block per row 83; in 8 bits 55 (issue slots), a block per row 90; as layer norms with biases 71 (four sums over the block), a block per row 113.
// ------------------------------------------------------------------------------------------------
constexpr int kNormStages = 2;
// Values of the stream an SM has to norm from which they are worth it (us, norms on both sides, a block per row and blocks that stay).  In bf16: 1200 rows of 1024 4.3 and 4.7, 1500
// 6.0 and 5.1; 200 of 4096 4.1 and 3.9, 300 6.0 and 5.2, 400 6.8 and 5.6; 200 of 8192 7.3 and 5.8.  In 8 bits: 4.8 and 5.1, 6.5 and 5.4; 4.4 and 4.7, 6.5 and 5.8, 7.3 and 6.2; 7.8 and
// 6.5.  Layer norms: 5.4 and 6.3, 7.7 and 6.7; 5.1 and 5.6, 8.1 and 7.3, 9.0 and 7.6; 10.3 and 7.7; in 8 bits 6.0 and 6.5, 8.1 and 6.9; 5.5 and 6.2, 8.7 and 7.5, 9.4 and 7.8; 10.9 and 8.3.
constexpr int kNormRingValues = 9600;

template <bool LAYERNORM, int NV, bool INT8>
__global__ void __launch_bounds__(kRowThreads4, NV == 4 ? 1 : 2) norm_block_ring_kernel(const NormBlockParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kNormStages];
  __shared__ float red[2][4][32];
  __shared__ uint32_t red_max[2][32];
  __shared__ int abort_word, fetched;
  volatile int* abort_flag = &abort_word;
  const int H = p.H, nvec = H / 8, step = (int)gridDim.x;
  const uint32_t row_bytes = (uint32_t)H * 2, stage_bytes = row_bytes * (p.y != nullptr ? 2 : 1);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kNormStages; ++s) mbar_init(&full[s], 1);
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
    bulk_load_1d(ring + s * stage_bytes, p.residual + t * p.ldr, row_bytes, &full[s]);
    if (p.y != nullptr) bulk_load_1d(ring + s * stage_bytes + row_bytes, p.y + t * p.ldy, row_bytes, &full[s]);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < kNormStages && (int)blockIdx.x + s * step < p.T; ++s) fetch((int)blockIdx.x + s * step, s);
  // The norms' weights stay in registers, or in L1 where the quotients need the registers.
  uint4 wv[NV], pv[NV];
  const auto weight = [&](const __nv_bfloat16* w, int it) {
    const int v = it * (int)blockDim.x + (int)threadIdx.x;
    return v < nvec ? reinterpret_cast<const uint4*>(w)[v] : make_uint4(0, 0, 0, 0);
  };
  if (!INT8) {
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      wv[it] = weight(p.w, it);
      if (p.post_w != nullptr) pv[it] = weight(p.post_w, it);
    }
  }
  int i = 0;
  for (int row = (int)blockIdx.x; row < p.T; row += step, ++i) {
    const long long t = row;
    const int s = i % kNormStages;
    float(*sums)[32] = red[i & 1];
    if (!mbar_wait(&full[s], (uint32_t)(i / kNormStages) & 1u, abort_flag)) {      // (every thread goes on to the block's barriers all the same)
      report_status(p.status, kTimeoutFullBarrier, row);
      *abort_flag = 1;
    }
    const uint4* rs = reinterpret_cast<const uint4*>(ring + s * stage_bytes);
    const uint4* ys = reinterpret_cast<const uint4*>(ring + s * stage_bytes + row_bytes);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float h[NV][8];
    if (p.y == nullptr) {
#pragma unroll
      for (int it = 0; it < NV; ++it) {
        const int v = it * (int)blockDim.x + (int)threadIdx.x;
        unpack8(v < nvec ? rs[v] : zero, h[it]);
      }
    } else {
#pragma unroll
      for (int it = 0; it < NV; ++it) {
        const int v = it * (int)blockDim.x + (int)threadIdx.x;
        unpack8(v < nvec ? ys[v] : zero, h[it]);
      }
      if (p.post_w != nullptr) {
        norm_rows<LAYERNORM, NV, kRowsWide>(h, H, p.eps, sums);
#pragma unroll
        for (int it = 0; it < NV; ++it) {
          float g[8];
          unpack8(INT8 ? weight(p.post_w, it) : pv[it], g);
#pragma unroll
          for (int q = 0; q < 8; ++q) h[it][q] *= g[q] + p.w_offset;
          if (p.post_b != nullptr) {
            float b[8];
            vector_load<kRowsWide>(p.post_b, it, H, b);
#pragma unroll
            for (int q = 0; q < 8; ++q) h[it][q] += b[q];
          }
        }
      }
#pragma unroll
      for (int it = 0; it < NV; ++it) {
        const int v = it * (int)blockDim.x + (int)threadIdx.x;
        if (p.gate != nullptr) {
          float g[8];
          gates<kRowsWide>(p, t, it, g);
#pragma unroll
          for (int q = 0; q < 8; ++q) h[it][q] *= g[q];
        }
        float r[8];
        unpack8(v < nvec ? rs[v] : zero, r);
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          w[q] = pack_bf16x2(fmaf(p.scale, h[it][2 * q], r[2 * q]), fmaf(p.scale, h[it][2 * q + 1], r[2 * q + 1]));
          const float2 u = unpack_bf16x2(w[q]);
          h[it][2 * q] = u.x;
          h[it][2 * q + 1] = u.y;
        }
        if (v < nvec) reinterpret_cast<uint4*>(p.residual_out + t * p.ldro)[v] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    norm_rows<LAYERNORM, NV, kRowsWide>(h, H, p.eps, sums + 2);
    // (a barrier has passed since the row was read last: its stage takes the one after the next)
    if (threadIdx.x == 0 && row + kNormStages * step < p.T && !*abort_flag) fetch(row + kNormStages * step, s);
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      float g[8];
      unpack8(INT8 ? weight(p.w, it) : wv[it], g);
#pragma unroll
      for (int q = 0; q < 8; ++q) h[it][q] *= g[q] + p.w_offset;
      if (p.b != nullptr) {
        float b[8];
        vector_load<kRowsWide>(p.b, it, H, b);
#pragma unroll
        for (int q = 0; q < 8; ++q) h[it][q] += b[q];
      }
      if (p.out != nullptr) row_store<kRowsWide>(p.out + t * p.ldo, it, H, h[it]);
    }
    if (INT8) {
      float m = 0.f;
#pragma unroll
      for (int it = 0; it < NV; ++it)
        if (row_whole<kRowsWide>(it, H, 0)) m = largest_magnitude(m, h[it]);
      const RowScale sc = row_scale(block_max(m, red_max[i & 1]));
      if (threadIdx.x == 0) p.q_scale[t] = sc.scale;
#pragma unroll
      for (int it = 0; it < NV; ++it) row_store_int8<kRowsWide>(p.q + t * p.ldq, it, H, h[it], sc);
    }
  }
  if (threadIdx.x == 0 && *abort_flag)      // copies still on their way arrive before the block leaves
    for (int j = max(0, fetched - kNormStages); j < fetched; ++j) mbar_wait(&full[j % kNormStages], (uint32_t)(j / kNormStages) & 1u, nullptr);
}

// Blocks that an SM holds at a time go by their registers (64 a thread, 128 with four groups) and their stages.
template <bool LAYERNORM, int NV, bool INT8>
static int launch_norm_ring(const NormBlockParams& p, int num_sms, cudaStream_t s) {
  const int need = p.H / 8, threads = ((need + NV - 1) / NV + 31) / 32 * 32;
  const int smem = kNormStages * p.H * 2 * (p.y != nullptr ? 2 : 1);
  static bool set[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(norm_block_ring_kernel<LAYERNORM, NV, INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormStages * 2 * 2 * kRowThreads4 * 8 * NV);
    if (e != cudaSuccess) return -(int)e;
    set[dev] = true;
  }
  int blocks = 65536 / (threads * (NV == 4 ? 128 : 64));
  if (blocks > 220 * 1024 / (smem + 4096)) blocks = 220 * 1024 / (smem + 4096);
  if (blocks > 32) blocks = 32;
  if (blocks < 1) blocks = 1;
  const int grid = p.T < num_sms * blocks ? p.T : num_sms * blocks;
  launch_pdl(norm_block_ring_kernel<LAYERNORM, NV, INT8>, dim3((unsigned)grid), dim3((unsigned)threads), (size_t)smem, s, p);
  return -(int)cudaGetLastError();
}

// Many shifted rows: blocks that stay, each on rows a multiple of eight apart, which all begin at the same distance from 16 bytes.  The norms' vectors are brought into
// that place once, to be read from shared memory, and the next row's values are on their way while one is normed.  Bound by instructions and by the chain of a layer norm's sums: 1500
// layer norms of 2049 with gate and biases 16.4 us, 6000 of 4097 88 (a block per row 18.1 and 124); RMS norms on both sides, 6000 of 4097, 67 (77).
constexpr int kNormVectors = 5;      // post_w, post_b, w, b, a channel's gate
template <bool LAYERNORM>
__global__ void __launch_bounds__(kRowShifted1, 2) norm_block_shifted_kernel(const NormBlockParams p) {
  constexpr int M = kRowsShifted;
  extern __shared__ uint4 vectors[];
  __shared__ float red[2][4][32];
  __shared__ uint32_t red_max[2][32];
  pdl_wait();
  pdl_trigger();
  const int H = p.H, shift = (int)((reinterpret_cast<uintptr_t>(p.residual + blockIdx.x * p.ldr) & 15) >> 1);
  uint4* mine = vectors + threadIdx.x;               // (nobody else reads a thread's part)
  const auto keep = [&](const __nv_bfloat16* v, int k) {
    if (v == nullptr) return;
    const int in = vector_in(v, shift);
    mine[k * (int)blockDim.x] = vector_shift<M>(vector_fetch<M>(v, 0, H, shift, in), 0, H, shift, in);
  };
  const bool channels = p.gate != nullptr && p.gate_h != 0 && p.gate_t == 0;
  keep(p.post_w, 0);
  keep(p.post_b, 1);
  keep(p.w, 2);
  keep(p.b, 3);
  if (channels) keep(p.gate, 4);
  const auto scale_by = [&](float (&f)[1][8], int k, const __nv_bfloat16* b) {
    float g[8];
    unpack8(mine[k * (int)blockDim.x], g);
#pragma unroll
    for (int q = 0; q < 8; ++q) f[0][q] *= g[q] + p.w_offset;
    if (b == nullptr) return;
    unpack8(mine[(k + 1) * (int)blockDim.x], g);
#pragma unroll
    for (int q = 0; q < 8; ++q) f[0][q] += g[q];
  };
  const Extent res_at = extent(p.residual, p.ldr, p.T, H), block_at = extent(p.y, p.ldy, p.T, H);
  uint4 hr = make_uint4(0, 0, 0, 0), yr = hr;          // of the next row
  const auto fetch = [&](long long t) {
    hr = row_fetch<M>(p.residual + t * p.ldr, 0, H, shift, res_at);
    if (p.y != nullptr) yr = row_fetch<M>(p.y + t * p.ldy, 0, H, shift, block_at);
  };
  if ((int)blockIdx.x < p.T) fetch(blockIdx.x);
  int i = 0;
  for (int row = (int)blockIdx.x; row < p.T; row += (int)gridDim.x, i ^= 1) {
    const long long t = row;
    float h[1][8];
    if (p.y != nullptr) {
      float r[8];
      row_take<M>(yr, 0, H, h[0], shift);
      if (p.post_w != nullptr) {
        norm_rows<LAYERNORM, 1, M>(h, H, p.eps, red[i], shift);
        scale_by(h, 0, p.post_b);
      }
      if (p.gate != nullptr) {
        float g[8];
        if (channels) unpack8(mine[4 * (int)blockDim.x], g);
        else gates<M>(p, t, 0, g, shift);
#pragma unroll
        for (int q = 0; q < 8; ++q) h[0][q] *= g[q];
      }
      row_take<M>(hr, 0, H, r, shift);
#pragma unroll
      for (int q = 0; q < 8; q += 2) {
        const float2 u = unpack_bf16x2(pack_bf16x2(fmaf(p.scale, h[0][q], r[q]), fmaf(p.scale, h[0][q + 1], r[q + 1])));
        h[0][q] = u.x;
        h[0][q + 1] = u.y;
      }
      row_store<M>(p.residual_out + t * p.ldro, 0, H, h[0], shift);
    } else {
      row_take<M>(hr, 0, H, h[0], shift);
    }
    if (row + (int)gridDim.x < p.T) fetch(row + (int)gridDim.x);
    norm_rows<LAYERNORM, 1, M>(h, H, p.eps, red[i] + 2, shift);
    scale_by(h, 2, p.b);
    if (p.out != nullptr) row_store<M>(p.out + t * p.ldo, 0, H, h[0], shift);
    if (p.q != nullptr) {
      if (!row_whole<M>(0, H, shift)) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (!row_has<M>(0, q, H, shift)) h[0][q] = 0.f;      // (0 times a row's infinite or NaN factors)
      }
      const RowScale s = row_scale(block_max(largest_magnitude(0.f, h[0]), red_max[i]));
      if (threadIdx.x == 0) p.q_scale[t] = s.scale;
      row_store_int8<M>(p.q + t * p.ldq, 0, H, h[0], s, shift);
    }
  }
}

// Blocks that run at the same time, by their registers (56 a thread): a multiple of eight.
static int norm_shifted_grid(const RowShape& r, int num_sms) {
  const int fit = 65536 / (r.threads * 56), grid = num_sms * (fit < 32 ? fit : 32) / 8 * 8;
  return grid < 8 ? 8 : grid;
}
// Where each has two rows or more and they are wide, or the norms have several vectors (us, a block per row and blocks that stay).  RMS norms, one vector: 6000 of 1021 19.4 and
// 20.9, of 1535 25.8 and 26.4, of 1791 30.4 and 28.7 (1500 9.7 and 9.9), of 2049 31.7 and 29.5 (1500 10.2 and 10.5), 1500 of 4097 17.8 and 16.1; norms on both sides, two vectors: 6000 of
// 1021 23.5 and 25.3, of 1791 37.0 and 34.7, of 2049 38.6 and 36.3.  Layer norms on both sides, a gate: 1500 of 1021 (one or two rows each) 11.8 and 12.8, 6000 37.3 and 31.4.
static bool norm_shifted_stays(const NormBlockParams& p, const RowShape& r, int num_sms) {
  const int kept = 1 + (p.post_w != nullptr) + (p.post_b != nullptr) + (p.b != nullptr) + (p.gate != nullptr && p.gate_h != 0 && p.gate_t == 0);
  return p.T >= 2ll * norm_shifted_grid(r, num_sms) && (p.H > 2000 || kept >= 3);
}
template <bool LAYERNORM>
static int launch_norm_shifted(const NormBlockParams& p, const RowShape& r, int num_sms, cudaStream_t s) {
  int grid = norm_shifted_grid(r, num_sms);
  if (grid > p.T) grid = (p.T + 7) / 8 * 8;      // (of the last eight blocks some have no row)
  launch_pdl(norm_block_shifted_kernel<LAYERNORM>, dim3((unsigned)grid), dim3((unsigned)r.threads), (size_t)kNormVectors * r.threads * 16, s, p);
  return -(int)cudaGetLastError();
}

template <bool LAYERNORM, int M>
static void launch_norm_block(const NormBlockParams& p, int T, const RowShape& r, cudaStream_t s) {
  const dim3 grid((unsigned)T), block((unsigned)r.threads);
  if (r.groups == 1) launch_pdl(norm_block_kernel<LAYERNORM, 1, M>, grid, block, 0, s, p);
  else if (r.groups == 2) launch_pdl(norm_block_kernel<LAYERNORM, 2, M>, grid, block, 0, s, p);
  else if (M != kRowsShifted) launch_pdl(norm_block_kernel<LAYERNORM, M == kRowsShifted ? 2 : 4, M>, grid, block, 0, s, p);
}

}  // namespace lx

extern "C" {

int lx_norm_block_max_width() { return lx::kRowThreads4 * 4 * 8; }

// In one block, as for lx_gemm_int8.
struct LxNormBlockArgs {
  const void* y;              // [T, H] or null
  long long ldy;
  const void* residual;
  long long ldr;
  void* residual_out;         // or null
  long long ldro;
  const void *post_w, *post_b, *w, *b, *gate;
  long long gate_t, gate_h;   // elements between two rows' gates, two channels' (0 or 1)
  void* out;                  // [T, H] bf16 or null
  long long ldo;
  void* q;                    // [T, H] int8 or null
  long long ldq;
  void* q_scale;
  long long T, H, layernorm;
  int* status;
  long long num_sms;
  long long ring;             // -1: the library's choice; 0 or 1 (where such a kernel takes the rows): a block per row or blocks that stay, to measure each
  void* stream;
  double eps, w_offset, scale;
};
int lx_norm_block_bytes() { return (int)sizeof(LxNormBlockArgs); }

int lx_norm_block(const char* args) {
  using namespace lx;
  LxNormBlockArgs a;
  memcpy(&a, args, sizeof(a));
  if (a.T <= 0) return 0;
  if (a.H <= 0 || a.H > lx_norm_block_max_width() || a.T > kRowsMost || (a.y != nullptr && a.residual_out == nullptr)) return -1;
  const void *y = a.y, *residual = a.residual, *residual_out = a.residual_out, *out = a.out, *q = a.q, *gate = a.gate;
  const long long ldy = a.ldy, ldr = a.ldr, ldro = a.ldro, ldo = a.ldo, ldq = a.ldq, gate_t = a.gate_t;
  const int T = (int)a.T, H = (int)a.H, num_sms = (int)a.num_sms, ring = (int)a.ring, layernorm = (int)a.layernorm;
  const auto bf = [](const void* v) { return reinterpret_cast<const __nv_bfloat16*>(v); };
  NormBlockParams p{bf(y), bf(residual), reinterpret_cast<__nv_bfloat16*>(a.residual_out), bf(a.post_w), bf(a.post_b), bf(a.w), bf(a.b), bf(gate), gate_t,
                    (int)a.gate_h, reinterpret_cast<uintptr_t>(gate) % 16 == 0 && gate_t % 8 == 0, reinterpret_cast<__nv_bfloat16*>(a.out),
                    reinterpret_cast<int8_t*>(a.q), reinterpret_cast<float*>(a.q_scale), ldy, ldr, ldro, ldo, ldq, H, T, (float)a.eps, (float)a.w_offset,
                    (float)a.scale, a.status};
  uintptr_t bits = 0;
  for (const void* v : {y, residual, residual_out, a.post_w, a.post_b, a.w, a.b, out}) bits |= reinterpret_cast<uintptr_t>(v);
  const bool wide = H % 8 == 0 && bits % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && (ldy | ldr | ldro | ldo | ldq) % 8 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(a.stream);
  if (wide && (ring < 0 ? T > num_sms && (long long)T * H >= (long long)kNormRingValues * num_sms : ring)) {
#define LX_RING(LN, Q) return H <= 2 * 8 * kRowThreads4 ? launch_norm_ring<LN, 2, Q>(p, num_sms, s) : launch_norm_ring<LN, 4, Q>(p, num_sms, s)
    if (layernorm && q != nullptr) LX_RING(true, true);
    if (layernorm) LX_RING(true, false);
    if (q != nullptr) LX_RING(false, true);
    LX_RING(false, false);
#undef LX_RING
  }
  // every row of every tensor as far from 16 bytes as the residual's, and the vectors at 16 bytes?
  bool alike = H + 7 <= kRowShifted2 * 2 * 8;
  const auto as_residual = [&](const void* v, long long ld) {
    return v == nullptr || ((reinterpret_cast<uintptr_t>(v) ^ reinterpret_cast<uintptr_t>(residual)) % 16 == 0 && (T == 1 || (ld - ldr) % 8 == 0));
  };
  for (const void* v : {a.post_w, a.post_b, a.w, a.b}) alike = alike && reinterpret_cast<uintptr_t>(v) % 16 == 0;
  alike = alike && as_residual(y, ldy) && as_residual(residual_out, ldro) && as_residual(out, ldo) && reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
  const RowShape r = wide || !alike ? row_shape(0, H, num_sms, kRowThreads4) : row_shape_shifted(H + 7);
  if (!wide && alike && r.groups == 1 && (ring < 0 ? norm_shifted_stays(p, r, num_sms) : ring))
    return layernorm ? launch_norm_shifted<true>(p, r, num_sms, s) : launch_norm_shifted<false>(p, r, num_sms, s);
  if (layernorm) {
    if (wide) launch_norm_block<true, kRowsWide>(p, T, r, s);
    else if (alike) launch_norm_block<true, kRowsShifted>(p, T, r, s);
    else launch_norm_block<true, kRowsApart>(p, T, r, s);
  } else {
    if (wide) launch_norm_block<false, kRowsWide>(p, T, r, s);
    else if (alike) launch_norm_block<false, kRowsShifted>(p, T, r, s);
    else launch_norm_block<false, kRowsApart>(p, T, r, s);
  }
  return -(int)cudaGetLastError();
}

}  // extern "C"
