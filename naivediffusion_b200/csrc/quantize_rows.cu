// Activations as int8 with one scale per row (token), the operand of the
// int8 x int8 product (linear_w8a8):
//
//   scale[r] = max |x[r]| / 127,   q[r, c] = rint(x[r, c] * 127 / max |x[r]|)
//
// The quotient is rounded as if computed exactly, half to even. The fast
// product t = x * (127 / peak) is off by at most 2^-23 * 127; only where t lies
// that near a half is its integer r checked against x * 127 - r * peak, which
// two products and their fma remainders give exactly (near_half below). A
// second pass over the thread's values with double division instead took 99 us
// at 4352 x 12288: values of exactly half the peak make one in most rows.
//
// Bound by HBM: the row is read once, stays in registers while its peak is
// found, and one byte per value is written.
#include <algorithm>
#include <climits>

#include "nd_common.cuh"
#include "nd_internal.h"
#include "nd_runtime.h"
#include "row_quant.cuh"

namespace nd {

namespace {

// The fast product x * (127 / peak) is off by at most 2^-23 * 127 = 1.5e-5.
constexpr float kNearHalf = 0.49997f;

// VEC values of type ND_F32 / ND_F16 / ND_BF16 as fp32: VEC 8 or 1.
template <int VEC>
__device__ __forceinline__ void load_vals(const void* p, long long i, int type, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    uint32_t w[4];
    if (type == ND_F32) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(f[4 * h]), "=f"(f[4 * h + 1]), "=f"(f[4 * h + 2]), "=f"(f[4 * h + 3])
                     : "l"(static_cast<const float*>(p) + i + 4 * h));
      return;
    }
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(static_cast<const uint16_t*>(p) + i));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = type == ND_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[j]))
                                      : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  } else {
    f[0] = type == ND_F32   ? __ldg(static_cast<const float*>(p) + i)
           : type == ND_F16 ? __half2float(static_cast<const __half*>(p)[i])
                            : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
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

// VEC values (already multiplied by `shift`'s power of two) to int8.
template <int VEC>
__device__ __forceinline__ void quantize_store(int8_t* q, const float (&f)[VEC], float inverse, float peak) {
  float m[VEC];  // rint(t) + 1.5 * 2^23
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float t = f[j] * inverse;
    m[j] = t + kRintMagic;
    most = fmaxf(most, fabsf(t - (m[j] - kRintMagic)));
  }
  if (most > kNearHalf) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) m[j] = near_half(f[j], m[j] - kRintMagic, peak) + kRintMagic;
  }
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint2*>(q) =
        make_uint2(pack_low_bytes(__float_as_uint(m[0]), __float_as_uint(m[1]), __float_as_uint(m[2]), __float_as_uint(m[3])),
                   pack_low_bytes(__float_as_uint(m[4]), __float_as_uint(m[5]), __float_as_uint(m[6]), __float_as_uint(m[7])));
  } else {
    *q = static_cast<int8_t>(__float_as_uint(m[0]) & 0xffu);
  }
}

template <int T>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < T / 32; ++i) v = max(v, red[i]);
  return v;
}

// One block per row; V x VEC values per thread in registers, the rest of a
// longer row read twice.
template <int VEC, int V, int T>
__global__ void __launch_bounds__(T) quantize_rows_kernel(const void* x, long long ldx, int type, int width,
                                                            int8_t* q, long long ldq, float* scale) {
  griddep_launch();
  griddep_wait();
  __shared__ uint32_t red[T / 32];
  const long long r = blockIdx.x;
  const long long x0 = r * ldx;
  float v[V][VEC];
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (threadIdx.x + T * i) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    if (c < width) load_vals<VEC>(x, x0 + c, type, v[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) peak = max(peak, abs_bits(v[i][j]));
  for (int c = (threadIdx.x + T * V) * VEC; c < width; c += T * VEC) {
    float w[VEC];
    load_vals<VEC>(x, x0 + c, type, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) peak = max(peak, abs_bits(w[j]));
  }
  const RowScale s = row_scale(block_max<T>(peak, red));
  if (threadIdx.x == 0) scale[r] = s.scale;
  int8_t* out = q + r * ldq;
  if (s.inverse == 0.f) {  // zeros, or infinities and NaN: every q is 0
    const float zero[VEC] = {};
#pragma unroll 1
    for (int c = threadIdx.x * VEC; c < width; c += T * VEC) quantize_store<VEC>(out + c, zero, 0.f, 1.f);
    return;
  }
  // Where 127 / peak or 127 x would leave fp32's range, the row is worked on
  // times a power of two (which changes no quotient).
  const float shift = s.peak < 1e-30f ? 0x1p96f : s.peak > 1e30f ? 0x1p-64f : 1.f;
  const float row_peak = s.peak * shift;
  const float inverse = shift == 1.f ? s.inverse : __fdiv_rn(127.0f, row_peak);
  auto finish = [&](int c, float(&w)[VEC]) {
    if (shift != 1.f) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] *= shift;
    }
    quantize_store<VEC>(out + c, w, inverse, row_peak);
  };
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (threadIdx.x + T * i) * VEC;
    if (c < width) finish(c, v[i]);
  }
  for (int c = (threadIdx.x + T * V) * VEC; c < width; c += T * VEC) {
    float w[VEC];
    load_vals<VEC>(x, x0 + c, type, w);
    finish(c, w);
  }
}

}  // namespace

int quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                  float* scale, cudaStream_t stream) {
  if (dtype != ND_F32 && dtype != ND_F16 && dtype != ND_BF16)
    return fail(ND_ERR_INVALID, "quantize_rows: x must be f32, f16 or bf16");
  if (rows <= 0 || cols <= 0) return fail(ND_ERR_INVALID, "quantize_rows: empty shape");
  if (rows > INT_MAX || cols > INT_MAX / 2) return fail(ND_ERR_INVALID, "quantize_rows: shape too large");
  if (!x || !q || !scale) return fail(ND_ERR_INVALID, "quantize_rows: null operand");
  if (ldx < cols || ldq < cols) return fail(ND_ERR_INVALID, "quantize_rows: a row stride is smaller than cols");
  const bool by8 = cols % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const dim3 grid(static_cast<unsigned>(rows));
  const int w = static_cast<int>(cols);
#define ND_QR(VEC, V, T) \
  ND_CUDA(launch_pdl(quantize_rows_kernel<VEC, V, T>, grid, dim3(T), 0, stream, x, ldx, dtype, w, q, ldq, scale))
  if (by8) {
    const int64_t w8 = cols / 8;
    if (w8 <= 128) ND_QR(8, 1, 128);
    else if (w8 <= 256) ND_QR(8, 2, 128);
    else if (w8 <= 512) ND_QR(8, 2, 256);
    else if (w8 <= 1024) ND_QR(8, 2, 512);
    else ND_QR(8, 3, 512);
  } else {
    if (cols <= 1024) ND_QR(1, 4, 256);
    else if (cols <= 4096) ND_QR(1, 16, 256);
    else ND_QR(1, 16, 512);
  }
#undef ND_QR
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

}  // namespace nd
