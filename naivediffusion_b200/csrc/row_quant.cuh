// One int8 scale per row (token): shared by quantize_rows and residual_norm.
//
//   peak  = max |x| over the row          scale = peak / 127 (fp32, IEEE division)
//   q     = rint(x * 127 / peak)          |q| <= 127 by construction
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

// The row's stored scale and the factor x is multiplied by.
struct RowScale {
  float peak, scale, inverse;
};
__device__ __forceinline__ RowScale row_scale(uint32_t peak_bits) {
  RowScale r;
  r.peak = __uint_as_float(peak_bits);
  if (peak_bits >= kInfBits) {
    r.scale = __uint_as_float(0x7fffffffu);
    r.inverse = 0.f;
  } else {
    r.scale = __fdiv_rn(r.peak, 127.0f);
    r.inverse = peak_bits == 0 ? 0.f : __fdiv_rn(127.0f, r.peak);
  }
  return r;
}

// t + kRintMagic (1.5 * 2^23) leaves no fraction bits: for |t| < 2^22 its low
// bits are rint(t), round to nearest even.
constexpr float kRintMagic = 12582912.0f;

// Four values' low bytes as one word.
__device__ __forceinline__ uint32_t pack_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace nd
