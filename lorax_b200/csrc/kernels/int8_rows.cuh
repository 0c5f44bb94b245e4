// Rows in 8-bit integers with a scale for each row:  scale = max |v| / 127,  q = v / scale rounded to the nearest integer (ties to the even one).
// What the kernels that write such rows share: the largest magnitude of a row, the quotients, and sums over a block.
//
// A row's scale is the 32-bit quotient; q is exact for that scale.  A row whose largest magnitude is not finite has a NaN for its scale, so that its
// products are NaN; where the scale is zero, as for a row of zeros, so are all q.
#pragma once

#include "common.cuh"

namespace lx {

// Position of a thread's value q of its `it`-th group of eight: eight neighbours (16-byte loads), or values a block's width apart where rows do not
// begin at 16 bytes or their length is no multiple of eight (a warp's loads are then still of neighbours).
template <bool WIDE>
LX_DEVICE int row_at(int it, int q) {
  return WIDE ? (it * (int)blockDim.x + (int)threadIdx.x) * 8 + q : (it * 8 + q) * (int)blockDim.x + (int)threadIdx.x;
}

// A thread's eight values of a row (0 behind its end), in 32 bits.
template <bool WIDE>
LX_DEVICE void row_load(const __nv_bfloat16* row, int it, int n, float (&f)[8]) {
  if (WIDE) {
    const int c = row_at<true>(it, 0);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c < n) v = *reinterpret_cast<const uint4*>(row + c);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 t = unpack_bf16x2(w[q]);
      f[2 * q] = t.x;
      f[2 * q + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int c = row_at<false>(it, q);
      f[q] = c < n ? __bfloat162float(row[c]) : 0.f;
    }
  }
}

template <bool WIDE>
LX_DEVICE void row_store(__nv_bfloat16* row, int it, int n, const float (&f)[8]) {
  if (WIDE) {
    const int c = row_at<true>(it, 0);
    if (c < n)
      *reinterpret_cast<uint4*>(row + c) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int c = row_at<false>(it, q);
      if (c < n) row[c] = __float2bfloat16(f[q]);
    }
  }
}

// The largest magnitude of eight values and one that stands already; a NaN among them stays one.
LX_DEVICE float larger_of(float m, float a, float b) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b));
  return d;
}
LX_DEVICE float largest_magnitude(float m, const float (&f)[8]) {
#pragma unroll
  for (int q = 0; q < 8; q += 2) m = larger_of(m, f[q], f[q + 1]);
  return m;
}

// Over a block of up to 1024 threads, for all of them.  `red` holds 32 words; a barrier stands between two uses of the same ones.  (Every warp joins the warps'
// parts by itself, a lane each: a loop over them was a quarter of the norms' instructions.)
LX_DEVICE float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31;
  v = warp_sum(v);
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < ((int)blockDim.x >> 5) ? red[lane] : 0.f);
}
// Of magnitudes.  Their bits order as they do, infinity above all numbers and NaN above infinity.
LX_DEVICE uint32_t block_max(float magnitude, uint32_t* red) {
  const int lane = threadIdx.x & 31;
  const uint32_t v = __reduce_max_sync(0xffffffffu, __float_as_uint(magnitude) & 0x7fffffffu);
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < ((int)blockDim.x >> 5) ? red[lane] : 0u);
}

struct RowScale {
  float scale, inv;      // inv: 1 / scale, rounded; 0 where all of the row's q are 0
};
LX_DEVICE RowScale row_scale(uint32_t magnitude) {
  RowScale s;
  if (magnitude >= 0x7f800000u) {
    s.scale = __uint_as_float(0x7fffffffu);
    s.inv = 0.f;
  } else {
    s.scale = __fdiv_rn(__uint_as_float(magnitude), 127.f);
    s.inv = s.scale > 0.f ? __fdiv_rn(1.f, s.scale) : 0.f;
  }
  return s;
}

// Quotients of rows whose scale is below 2^-128, where 1 / scale passes what 32 bits hold.
static __device__ __noinline__ int tiny_quotient(float v, float scale) { return (int)rint((double)v / (double)scale); }

// Eight quotients as bytes.  v * inv, unrounded, is off from v / scale by 127 * 2^-24 = 7.6e-6 at most (inv's rounding; |v| <= 127 scales), and its distance from the
// integer by 2^-26 more, so that only a quotient within 1e-5 of a border may have gone to the wrong side.  Groups with such a one compare what is left with half the
// scale: r = v - q * scale is exact there, a multiple of the smaller last place of v and scale and no larger than the scale.  Rows of bf16 numbers hold ties by the
// hundred (their quotients are 127 times ratios of 8-bit numbers), so that the comparison has to be short.
LX_DEVICE uint2 row_quotients(const float (&f)[8], const RowScale& s) {
  constexpr float kWhole = 12582912.f;                       // 1.5 * 2^23: a sum's last place is 1, and its low byte the integer's
  float u[8], far = 0.f;
#pragma unroll
  for (int q = 0; q < 8; q += 2) {
    u[q] = fmaf(f[q], s.inv, kWhole);
    u[q + 1] = fmaf(f[q + 1], s.inv, kWhole);
    far = larger_of(far, fmaf(f[q], s.inv, -__fsub_rn(u[q], kWhole)), fmaf(f[q + 1], s.inv, -__fsub_rn(u[q + 1], kWhole)));
  }
  if (!(far < 0.49999f)) {
    if (s.inv == 0.f) return make_uint2(0, 0);
    if (s.inv > 3e38f) {
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] = __int_as_float(tiny_quotient(f[q], s.scale));
    } else {
      const float half = 0.5f * s.scale;                     // (exact: the scale is 2^-128 at least)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float r = fmaf(-__fsub_rn(u[q], kWhole), s.scale, f[q]);
        // over half, or a tie at an odd integer: the neighbour on r's side
        if (fabsf(r) > half || (fabsf(r) == half && (__float_as_int(u[q]) & 1))) u[q] += r > 0.f ? 1.f : -1.f;
      }
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = __byte_perm(__byte_perm(__float_as_uint(u[4 * h]), __float_as_uint(u[4 * h + 1]), 0x0040),
                       __byte_perm(__float_as_uint(u[4 * h + 2]), __float_as_uint(u[4 * h + 3]), 0x0040), 0x5410);
  return make_uint2(w[0], w[1]);
}

// A thread's eight quotients to its row's bytes.
template <bool WIDE>
LX_DEVICE void row_store_int8(int8_t* row, int it, int n, const float (&f)[8], const RowScale& s) {
  if (WIDE && row_at<true>(it, 0) >= n) return;
  const uint2 w = row_quotients(f, s);
  if (WIDE) {
    *reinterpret_cast<uint2*>(row + row_at<true>(it, 0)) = w;
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int c = row_at<false>(it, q);
      if (c < n) row[c] = (int8_t)((q < 4 ? w.x : w.y) >> (8 * (q & 3)));
    }
  }
}

// Threads of a block and groups of eight that each holds, for rows of n values.  Few rows: as many threads as there are groups (`most`), since the row's own
// chain of loads, sums and stores is what takes time.  Many: 256 threads and more groups, whose loads are in flight together.
constexpr int kRowThreads4 = 512;      // of a block whose threads hold four groups
struct RowShape {
  int threads, groups;                 // groups: 1, 2, 4; 0: the row is longer than a block's registers hold
};
inline RowShape row_shape(int rows, int n, int num_sms, int most) {
  const int need = (n + 7) / 8;
  if (rows > num_sms) most = 256;
  for (int g = 1; g <= 4; g *= 2) {
    const int threads = ((need + g - 1) / g + 31) / 32 * 32;
    if (threads <= (g == 4 ? kRowThreads4 : most)) return RowShape{threads, g};
  }
  return RowShape{1024, 0};
}

}  // namespace lx
