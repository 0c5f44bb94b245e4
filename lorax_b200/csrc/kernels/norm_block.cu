// Norms on both sides of a block in one pass over its rows:
//   h = residual + scale * gate * N_post(y)         (N_post: left out without a weight of its own; gate: any of one, [T, 1], [H], [T, H])
//   x = N(h),  N(v) = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * (w + offset) + b      (RMS norm: without the means)
// h replaces the residual (or is written elsewhere) in bf16, and N reads the rounded h, as whoever reads the stream later does.  x leaves in bf16, in 8 bits
// with a scale for each row (int8_rows.cuh), from the same 32-bit values, or both.
//
// The reference norms and adds in separate kernels (server/lorax_server/models/custom_modeling/flash_gemma2_modeling.py:355-396).
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
  long long gate_t, gate_h;            // elements between two rows' and two channels' gates (0: the same)
  __nv_bfloat16* out;                  // [T, H] or null
  int8_t* q;                           // [T, H] or null
  float* q_scale;
  long long ldy, ldr, ldro, ldo, ldq;
  int H;
  float eps, w_offset, scale;
};

// Sums over the block of up to three norms' passes, each with words of its own.
template <bool LAYERNORM, int NV, bool WIDE>
LX_DEVICE void norm_rows(float (&f)[NV][8], int H, float eps, float (*red)[32]) {
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
      f[it][q] = row_at<WIDE>(it, q) < H ? f[it][q] - mean : 0.f;
      s = fmaf(f[it][q], f[it][q], s);
    }
  const float r = rsqrtf(block_sum(s, red[1]) / H + eps);
#pragma unroll
  for (int it = 0; it < NV; ++it)
#pragma unroll
    for (int q = 0; q < 8; ++q) f[it][q] *= r;
}

template <int NV, bool WIDE>
LX_DEVICE void scale_rows(float (&f)[NV][8], int H, const __nv_bfloat16* w, const __nv_bfloat16* b, float offset) {
#pragma unroll
  for (int it = 0; it < NV; ++it) {
    float g[8];
    row_load<WIDE>(w, it, H, g);
#pragma unroll
    for (int q = 0; q < 8; ++q) f[it][q] *= g[q] + offset;
    if (b != nullptr) {
      row_load<WIDE>(b, it, H, g);
#pragma unroll
      for (int q = 0; q < 8; ++q) f[it][q] += g[q];
    }
  }
}

// One block per row; NV groups of eight a thread, all in registers.
template <bool LAYERNORM, int NV, bool WIDE>
__global__ void __launch_bounds__(kRowThreads4) norm_block_kernel(const NormBlockParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[4][32];
  __shared__ uint32_t red_max[32];
  const long long t = blockIdx.x;
  float h[NV][8];
#pragma unroll
  for (int it = 0; it < NV; ++it) row_load<WIDE>(p.residual + t * p.ldr, it, p.H, h[it]);
  if (p.y != nullptr) {
    float y[NV][8];
#pragma unroll
    for (int it = 0; it < NV; ++it) row_load<WIDE>(p.y + t * p.ldy, it, p.H, y[it]);
    if (p.post_w != nullptr) {
      norm_rows<LAYERNORM, NV, WIDE>(y, p.H, p.eps, red);
      scale_rows<NV, WIDE>(y, p.H, p.post_w, p.post_b, p.w_offset);
    }
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      if (p.gate != nullptr) {
        const __nv_bfloat16* gate = p.gate + t * p.gate_t;
        float g[8];
        if (p.gate_h == 0) {
          const float one = __bfloat162float(*gate);
#pragma unroll
          for (int q = 0; q < 8; ++q) g[q] = one;
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int c = row_at<WIDE>(it, q);
            g[q] = c < p.H ? __bfloat162float(gate[c * p.gate_h]) : 0.f;
          }
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) y[it][q] *= g[q];
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) h[it][q] = __bfloat162float(__float2bfloat16(fmaf(p.scale, y[it][q], h[it][q])));
    }
  }
  if (p.residual_out != nullptr) {
#pragma unroll
    for (int it = 0; it < NV; ++it) row_store<WIDE>(p.residual_out + t * p.ldro, it, p.H, h[it]);
  }
  norm_rows<LAYERNORM, NV, WIDE>(h, p.H, p.eps, red + 2);
  scale_rows<NV, WIDE>(h, p.H, p.w, p.b, p.w_offset);
  if (p.out != nullptr) {
#pragma unroll
    for (int it = 0; it < NV; ++it) row_store<WIDE>(p.out + t * p.ldo, it, p.H, h[it]);
  }
  if (p.q != nullptr) {
    uint32_t m = 0;
#pragma unroll
    for (int it = 0; it < NV; ++it)
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (row_at<WIDE>(it, q) < p.H) m = larger_magnitude(m, h[it][q]);
    const RowScale s = row_scale(block_max(m, red_max));
    if (threadIdx.x == 0) p.q_scale[t] = s.scale;
#pragma unroll
    for (int it = 0; it < NV; ++it) row_store_int8<WIDE>(p.q + t * p.ldq, it, p.H, h[it], s);
  }
}

template <bool LAYERNORM, bool WIDE>
static void launch_norm_block(const NormBlockParams& p, int T, const RowShape& r, cudaStream_t s) {
  const dim3 grid((unsigned)T), block((unsigned)r.threads);
  if (r.groups == 1) launch_pdl(norm_block_kernel<LAYERNORM, 1, WIDE>, grid, block, 0, s, p);
  else if (r.groups == 2) launch_pdl(norm_block_kernel<LAYERNORM, 2, WIDE>, grid, block, 0, s, p);
  else launch_pdl(norm_block_kernel<LAYERNORM, 4, WIDE>, grid, block, 0, s, p);
}

}  // namespace lx

extern "C" {

int lx_norm_block_max_width() { return lx::kRowThreads4 * 4 * 8; }

int lx_norm_block(const void* y, long long ldy, const void* residual, long long ldr, void* residual_out, long long ldro, const void* post_w,
                  const void* post_b, const void* w, const void* b, const void* gate, long long gate_t, long long gate_h, void* out, long long ldo, void* q,
                  long long ldq, void* q_scale, int T, int H, float eps, float w_offset, float scale, int layernorm, int num_sms, void* stream) {
  using namespace lx;
  if (T <= 0) return 0;
  if (H <= 0 || H > lx_norm_block_max_width()) return -1;
  const auto bf = [](const void* a) { return reinterpret_cast<const __nv_bfloat16*>(a); };
  NormBlockParams p{bf(y), bf(residual), reinterpret_cast<__nv_bfloat16*>(residual_out), bf(post_w), bf(post_b), bf(w), bf(b), bf(gate), gate_t, gate_h,
                    reinterpret_cast<__nv_bfloat16*>(out), reinterpret_cast<int8_t*>(q), reinterpret_cast<float*>(q_scale), ldy, ldr, ldro, ldo, ldq, H, eps,
                    w_offset, scale};
  uintptr_t bits = 0;
  for (const void* a : {y, residual, static_cast<const void*>(residual_out), post_w, post_b, w, b, static_cast<const void*>(out)}) bits |= reinterpret_cast<uintptr_t>(a);
  const bool wide = H % 8 == 0 && bits % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && (ldy | ldr | ldro | ldo | ldq) % 8 == 0;
  const RowShape r = row_shape(T, H, num_sms, kRowThreads4);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (layernorm) {
    if (wide) launch_norm_block<true, true>(p, T, r, s);
    else launch_norm_block<true, false>(p, T, r, s);
  } else {
    if (wide) launch_norm_block<false, true>(p, T, r, s);
    else launch_norm_block<false, false>(p, T, r, s);
  }
  return -(int)cudaGetLastError();
}

}  // extern "C"
