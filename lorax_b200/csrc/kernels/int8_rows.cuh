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

// The larger magnitude, as the bits of a 32-bit number: those order as the magnitudes do, infinity above all numbers and NaN above infinity.
LX_DEVICE uint32_t larger_magnitude(uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7fffffffu); }

// Over a block of up to 1024 threads, for all of them.  `red` holds 32 words; a barrier stands between two uses of the same ones.
LX_DEVICE float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = (int)blockDim.x >> 5;
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s += red[i];
  return s;
}
LX_DEVICE uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = (int)blockDim.x >> 5;
  uint32_t m = 0;
  for (int i = 0; i < warps; ++i) m = max(m, red[i]);
  return m;
}

struct RowScale {
  float scale, inv;      // inv: about 1 / scale, 0 where all of the row's q are 0
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

// v / scale to the nearest integer.  v * inv is off by 2^-16 at most (|q| <= 127, two roundings of 2^-24 each, one of the scale), so only quotients that near
// to a border need more: there v - q * scale is exact (a multiple of the smaller last place of v and scale, no larger than the scale), and is
// compared with half the scale.  inv is infinite for scales below 2^-128: quotients of those rows all go through the division.
LX_DEVICE int row_quotient(float v, const RowScale& s) {
  constexpr float kWhole = 12582912.f;                       // 1.5 * 2^23: the sum's last place is 1
  const float t = v * s.inv;
  float q = __fsub_rn(__fadd_rn(t, kWhole), kWhole);
  if (!(fabsf(t - q) < 0.4998f)) {
    if (s.inv == 0.f) return 0;
    if (!(fabsf(t) < 256.f)) q = rintf(__fdiv_rn(v, s.scale));
    const float r = fmaf(-q, s.scale, v), a = fabsf(r), rest = s.scale - a;      // (a > rest: over half; exact, both are within a factor of two)
    const float step = r > 0.f ? 1.f : -1.f;
    if (a > rest || (a == rest && (((int)q) & 1))) q += step;
  }
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// A thread's eight quotients to its row's bytes.
template <bool WIDE>
LX_DEVICE void row_store_int8(int8_t* row, int it, int n, const float (&f)[8], const RowScale& s) {
  if (WIDE) {
    const int c = row_at<true>(it, 0);
    if (c >= n) return;
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int a = row_quotient(f[4 * h], s), b = row_quotient(f[4 * h + 1], s), d = row_quotient(f[4 * h + 2], s), e = row_quotient(f[4 * h + 3], s);
      w[h] = __byte_perm(__byte_perm((uint32_t)a, (uint32_t)b, 0x0040), __byte_perm((uint32_t)d, (uint32_t)e, 0x0040), 0x5410);
    }
    *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int c = row_at<false>(it, q);
      if (c < n) row[c] = (int8_t)row_quotient(f[q], s);
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
