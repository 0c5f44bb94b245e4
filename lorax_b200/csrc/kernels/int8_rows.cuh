// Rows in 8-bit integers with a scale for each row:  scale = max |v| / 127,  q = v / scale rounded to the nearest integer (ties to the even one).
// What the kernels that write such rows share: the largest magnitude of a row, the quotients, and sums over a block.
//
// A row's scale is the 32-bit quotient; q is exact for that scale.  A row whose largest magnitude is not finite has a NaN for its scale, so that its
// products are NaN; where the scale is zero, as for a row of zeros, so are all q.
#pragma once

#include "common.cuh"

namespace lx {

// How a thread's groups of eight lie in a row.  kRowsWide: eight neighbours, rows of a multiple of eight that begin at 16 bytes.  kRowsShifted: eight
// neighbours that begin at 16 bytes, wherever the row does: `shift` values in front of it, so that all groups but a row's first and last are loaded and stored at
// once.  kRowsApart: values a block's width apart, for rows of which every tensor begins elsewhere (a warp's loads are still of neighbours).
enum RowsMode : int { kRowsApart = 0, kRowsWide = 1, kRowsShifted = 2 };

template <int M>
LX_DEVICE int row_at(int it, int q, int shift = 0) {
  return M == kRowsApart ? (it * 8 + q) * (int)blockDim.x + (int)threadIdx.x : (it * (int)blockDim.x + (int)threadIdx.x) * 8 + q - (M == kRowsShifted ? shift : 0);
}
template <int M>
LX_DEVICE bool row_has(int it, int q, int n, int shift) {
  const int c = row_at<M>(it, M == kRowsWide ? 0 : q, shift);
  return c < n && (M != kRowsShifted || c >= 0);
}
// Whether the group lies in the row as a whole.
template <int M>
LX_DEVICE bool row_whole(int it, int n, int shift) {
  const int c = row_at<M>(it, 0, shift);
  return M == kRowsWide ? c < n : M == kRowsShifted && c >= 0 && c + 8 <= n;
}

LX_DEVICE void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 t = unpack_bf16x2(w[q]);
    f[2 * q] = t.x;
    f[2 * q + 1] = t.y;
  }
}

// The values of a group that lie in the row, one by one, and zeros.
template <int M>
LX_DEVICE uint4 row_pieces(const __nv_bfloat16* row, int it, int n, int shift) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const unsigned short* v = reinterpret_cast<const unsigned short*>(row);
    const uint32_t a = row_has<M>(it, 2 * q, n, shift) ? v[row_at<M>(it, 2 * q, shift)] : 0u, b = row_has<M>(it, 2 * q + 1, n, shift) ? v[row_at<M>(it, 2 * q + 1, shift)] : 0u;
    w[q] = a | b << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Where the elements of a tensor of rows lie: from `lo` up to `hi`.
struct Extent {
  const __nv_bfloat16 *lo, *hi;
};
LX_DEVICE Extent extent(const __nv_bfloat16* base, long long ld, int rows, int n) { return Extent{base, base + (rows - 1) * ld + n}; }

// A thread's eight values of a row (0 outside it), in two steps: loads, all of them on their way before the first is waited for, and what becomes of them.  A shifted
// row's first and last 16 bytes are loaded as a whole where they lie in the tensor, and what belongs to its neighbours is cut off.
template <int M>
LX_DEVICE uint4 row_fetch(const __nv_bfloat16* row, int it, int n, int shift, const Extent& e) {
  if (M == kRowsApart) return row_pieces<M>(row, it, n, shift);
  const int c = row_at<M>(it, 0, shift);
  const __nv_bfloat16* a = row + c;
  uint4 v = make_uint4(0, 0, 0, 0);
  const bool some = c < n && c + 8 > 0, inside = M == kRowsWide || (a >= e.lo && a + 8 <= e.hi);
  if (some && inside) v = *reinterpret_cast<const uint4*>(a);
  if (M == kRowsShifted && some && !inside) v = row_pieces<M>(row, it, n, shift);
  return v;
}
template <int M>
LX_DEVICE void row_take(const uint4& v, int it, int n, float (&f)[8], int shift) {
  unpack8(v, f);
  if (M == kRowsShifted && !row_whole<M>(it, n, shift)) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (!row_has<M>(it, q, n, shift)) f[q] = 0.f;
  }
}

// The same of a vector whose first 16 bytes lie elsewhere in its groups: two 16-byte loads and a shift where both lie inside the vector, else its pieces.  `in`: values
// of the first load in front of a group, the same for all groups.
struct VectorRaw {
  uint4 lo, hi;
};
LX_DEVICE int vector_in(const __nv_bfloat16* v, int shift) { return (int)((reinterpret_cast<uintptr_t>(v - shift) & 15) >> 1); }
template <int M>
LX_DEVICE bool vector_whole(int it, int n, int shift, int in) {
  const int a = row_at<M>(it, 0, shift) - in;
  return M != kRowsShifted ? row_whole<M>(it, n, shift) : a >= 0 && a + 16 <= n;
}
template <int M>
LX_DEVICE VectorRaw vector_fetch(const __nv_bfloat16* v, int it, int n, int shift, int in) {
  VectorRaw r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (vector_whole<M>(it, n, shift, in)) {
    const uint4* a = reinterpret_cast<const uint4*>(v + (row_at<M>(it, 0, shift) - (M == kRowsShifted ? in : 0)));
    r.lo = a[0];
    if (M == kRowsShifted) r.hi = a[1];
  } else if (M != kRowsWide) {
    r.lo = row_pieces<M>(v, it, n, shift);
  }
  return r;
}
template <int M>
LX_DEVICE uint4 vector_shift(const VectorRaw& r, int it, int n, int shift, int in) {
  uint32_t w[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
  if (M == kRowsShifted) {
    if (!vector_whole<M>(it, n, shift, in)) in = 0;      // (pieces stand where they belong)
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = in & 4 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = in & 2 ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (in & 1) * 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int M>
LX_DEVICE void vector_take(const VectorRaw& r, int it, int n, float (&f)[8], int shift, int in) {
  unpack8(vector_shift<M>(r, it, n, shift, in), f);
}
template <int M>
LX_DEVICE void vector_load(const __nv_bfloat16* v, int it, int n, float (&f)[8], int shift = 0, int in = 0) {
  vector_take<M>(vector_fetch<M>(v, it, n, shift, in), it, n, f, shift, in);
}

template <int M>
LX_DEVICE void row_store(__nv_bfloat16* row, int it, int n, const float (&f)[8], int shift = 0) {
  if (row_whole<M>(it, n, shift)) {
    *reinterpret_cast<uint4*>(row + row_at<M>(it, 0, shift)) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else if (M != kRowsWide) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (row_has<M>(it, q, n, shift)) row[row_at<M>(it, q, shift)] = __float2bfloat16(f[q]);
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

// Quotients of rows whose scale is below 2^-123: 1 / scale may pass what 32 bits hold, and half the scale fall between two numbers.  A scale of k units of 2^-149 is off
// from max / 127 by up to half a unit, so that quotients reach 127 (k + 1/2) / k, and end at 127 as those of all other rows do.
constexpr float kTinyInv = 1e37f;
static __device__ __noinline__ int tiny_quotient(float v, float scale) { return max(-127, min(127, (int)rint((double)v / (double)scale))); }

// Eight quotients as bytes.  v * inv, unrounded, is off from v / scale by 127 * 2^-24 = 7.6e-6 at most (inv's rounding; |v| is at most 127 scales and a rounding), and its
// distance from the integer by 2^-26 more, so that only a quotient within 1e-5 of a border may have gone to the wrong side.  Groups with such a one compare what is left with half the
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
    if (s.inv > kTinyInv) {
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] = __int_as_float(tiny_quotient(f[q], s.scale));
    } else {
      const float half = 0.5f * s.scale;                     // (exact: the scale is 1e-37 at least)
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

// A thread's eight quotients to its row's bytes, which begin at 16 bytes.
template <int M>
LX_DEVICE void row_store_int8(int8_t* row, int it, int n, const float (&f)[8], const RowScale& s, int shift = 0) {
  if (M == kRowsWide && !row_whole<M>(it, n, 0)) return;
  const uint2 w = row_quotients(f, s);
  if (M != kRowsApart && (row_at<M>(it, 0, shift) & 7) == 0 && row_whole<M>(it, n, shift)) {
    *reinterpret_cast<uint2*>(row + row_at<M>(it, 0, shift)) = w;
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (row_has<M>(it, q, n, shift)) row[row_at<M>(it, q, shift)] = (int8_t)((q < 4 ? w.x : w.y) >> (8 * (q & 3)));
  }
}

// Threads of a block and groups of eight that each holds, for rows of n values.  Few rows: as many threads as there are groups (`most`), since the row's own
// chain of loads, sums and stores is what takes time.  Many: 256 threads and more groups, whose loads are in flight together.
constexpr int kRowsMost = 0x7fff0000;  // of a call: a row's number and the rows ahead of it stay below 2^31
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
// For kRowsShifted, whose groups take more registers: one a thread in blocks of up to 576 (56 registers, so that four blocks of 288 share an SM), or two in blocks of up to 768.
constexpr int kRowShifted1 = 576, kRowShifted2 = 768;
inline RowShape row_shape_shifted(int n) {
  const int need = (n + 7) / 8, g = need <= kRowShifted1 ? 1 : 2;
  return RowShape{((need + g - 1) / g + 31) / 32 * 32, g};
}

}  // namespace lx
