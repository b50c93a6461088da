// One int8 scale per row (token): shared by quantize_rows and residual_norm.
//
//   peak  = max |x| over the row          scale = peak / 127 (fp32, IEEE division)
//   q     = rint(x * 127 / peak)          |q| <= 127 by construction
//
// with the quotient rounded as if computed exactly, half to even: the same int8
// row whichever of the two writes it.
//
// A row of zeros has scale 0 and q 0. A row that holds an infinity or a NaN
// has scale NaN and q 0: whatever is multiplied by it comes out NaN instead
// of silently finite.
#pragma once

#include "nd_common.cuh"

namespace nd {

constexpr uint32_t kInfBits = 0x7f800000u;

// |x| as bits: ordered like |x|, with NaN above infinity, so an unsigned
// maximum finds the peak and keeps any NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The row's peak and stored scale.
struct RowScale {
  float peak, scale;
  bool zero;  // every q is 0: a row of zeros, or one that is not finite
};
__device__ __forceinline__ RowScale row_scale(uint32_t peak_bits) {
  RowScale r;
  r.peak = __uint_as_float(peak_bits);
  r.zero = peak_bits == 0 || peak_bits >= kInfBits;
  r.scale = peak_bits >= kInfBits ? __uint_as_float(0x7fffffffu) : __fdiv_rn(r.peak, 127.0f);
  return r;
}

// t + kRintMagic (1.5 * 2^23) leaves no fraction bits: for |t| < 2^22 its low
// bits are rint(t), round to nearest even.
constexpr float kRintMagic = 12582912.0f;

// Where 127 / peak or 127 x would leave fp32's range, a row is worked on times
// this power of two (which changes no quotient).
__device__ __forceinline__ float range_shift(float peak) { return peak < 1e-30f ? 0x1p96f : peak > 1e30f ? 0x1p-64f : 1.f; }

// 127 / peak as hi + lo.
struct Inverse {
  float hi, lo;
};
__device__ __forceinline__ Inverse inverse_of(float peak) {
  Inverse v;
  v.hi = __fdiv_rn(127.0f, peak);
  v.lo = __fdiv_rn(fmaf(-v.hi, peak, 127.0f), peak);  // the remainder is exact
  return v;
}

// The exact rounding of x * 127 / peak, given r, its integer by the fast
// product, where the quotient lies near r +- 1/2. 127 x = hi + lo and
// r peak = hi2 + lo2 exactly (fma remainders); hi - hi2, 2 |d| - peak and
// lo - lo2 are differences of near neighbours or of few bits and exact, so the
// sign of their sum says on which side of the half the quotient lies.
__device__ __forceinline__ float near_half(float x, float r, float peak) {
  const float hi = x * 127.0f, lo = fmaf(x, 127.0f, -hi);
  const float hi2 = r * peak, lo2 = fmaf(r, peak, -hi2);
  const float d = hi - hi2;
  const float way = d < 0.f ? -1.f : 1.f;
  const float past = (2.f * fabsf(d) - peak) + 2.f * way * (lo - lo2);
  const bool odd = (__float2int_rn(r) & 1) != 0;
  return past > 0.f || (past == 0.f && odd) ? r + way : r;
}

// N values (already multiplied by range_shift) as rint(x * 127 / peak) + kRintMagic.
// EXACT: fp32 values, whose quotient may lie closer to a half than t resolves.
template <bool EXACT, int N>
__device__ __forceinline__ void quantize_values(const float (&f)[N], Inverse inv, float peak, float (&m)[N]) {
  float most = 0.f;
  if constexpr (N > 1) {
    const float2 hi2 = make_float2(inv.hi, inv.hi), lo2 = make_float2(inv.lo, inv.lo);
    const float2 magic2 = make_float2(kRintMagic, kRintMagic);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 x2 = make_float2(f[j], f[j + 1]);
      const float2 t2 = ffma2(x2, hi2, fmul2(x2, lo2));
      const float2 m2 = fadd2(t2, magic2);
      if constexpr (EXACT) {
        const float2 r2 = fadd2(magic2, make_float2(-m2.x, -m2.y));
        const float2 off = fadd2(t2, r2);
        most = fmax3(most, fabsf(off.x), fabsf(off.y));
      }
      m[j] = m2.x;
      m[j + 1] = m2.y;
    }
  } else {
    const float t = fmaf(f[0], inv.hi, f[0] * inv.lo);
    m[0] = t + kRintMagic;
    most = fabsf(t - (m[0] - kRintMagic));
  }
  if (EXACT && most == 0.5f) {
#pragma unroll
    for (int j = 0; j < N; ++j) m[j] = near_half(f[j], m[j] - kRintMagic, peak) + kRintMagic;
  }
}

// Four values' low bytes as one word.
__device__ __forceinline__ uint32_t pack_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace nd
