// Activations as int8 with one scale per row (token), the operand of the
// int8 x int8 product (linear_w8a8):
//
//   scale[r] = max |x[r]| / 127,   q[r, c] = rint(x[r, c] * 127 / max |x[r]|)
//
// The quotient is rounded as if computed exactly, half to even: the fast
// product x * (127 / peak) is at most 2^-23 * 127 off, so only values whose
// product lies within that of a half are divided again, in double, where
// x * 127 is exact and no quotient of two fp32 values lies closer to a half
// than a double resolves without being one.
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

// VEC values of type ND_F32 / ND_F16 / ND_BF16 as fp32.
template <int VEC>
__device__ __forceinline__ void load_vals(const void* p, long long i, int type, float (&f)[VEC]) {
  if constexpr (VEC == 4) {
    if (type == ND_F32) {
      asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                   : "l"(static_cast<const float*>(p) + i));
    } else {
      uint32_t a, b;
      asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
                   : "=r"(a), "=r"(b)
                   : "l"(static_cast<const uint16_t*>(p) + i));
      float2 lo, hi;
      if (type == ND_F16) {
        lo = __half22float2(*reinterpret_cast<const __half2*>(&a));
        hi = __half22float2(*reinterpret_cast<const __half2*>(&b));
      } else {
        lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&a));
        hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&b));
      }
      f[0] = lo.x; f[1] = lo.y; f[2] = hi.x; f[3] = hi.y;
    }
  } else {
    f[0] = type == ND_F32   ? __ldg(static_cast<const float*>(p) + i)
           : type == ND_F16 ? __half2float(static_cast<const __half*>(p)[i])
                            : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
}

// The exact quotient's nearest integer, as bits whose low byte is q.
__device__ __forceinline__ uint32_t rint_exact(float x, float peak) {
  return static_cast<uint32_t>(__double2int_rn(__ddiv_rn(static_cast<double>(x) * 127.0, static_cast<double>(peak))));
}

// VEC values by the fast product; returns their largest distance from the
// integer taken.
template <int VEC>
__device__ __forceinline__ float quantize_store(int8_t* q, const float (&f)[VEC], float inverse) {
  uint32_t u[4] = {0u, 0u, 0u, 0u};
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float off;
    u[j] = rint_bits(f[j] * inverse, off);
    most = fmaxf(most, off);
  }
  if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(q) = pack_low_bytes(u[0], u[1], u[2], u[3]);
  else *q = static_cast<int8_t>(u[0] & 0xffu);
  return most;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < static_cast<int>(blockDim.x >> 5); ++i) v = max(v, red[i]);
  return v;
}

// One block per row; V x VEC values per thread in registers, the rest of a
// longer row read twice.
template <int VEC, int V>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* x, long long ldx, int type, int width,
                                                            int8_t* q, long long ldq, float* scale) {
  griddep_launch();
  griddep_wait();
  __shared__ uint32_t red[8];
  const long long r = blockIdx.x;
  const long long x0 = r * ldx;
  float v[V][VEC];
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (threadIdx.x + blockDim.x * i) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    if (c < width) load_vals<VEC>(x, x0 + c, type, v[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) peak = max(peak, abs_bits(v[i][j]));
  for (int c = (threadIdx.x + blockDim.x * V) * VEC; c < width; c += blockDim.x * VEC) {
    float w[VEC];
    load_vals<VEC>(x, x0 + c, type, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) peak = max(peak, abs_bits(w[j]));
  }
  const RowScale s = row_scale(block_max(peak, red));
  if (threadIdx.x == 0) scale[r] = s.scale;
  int8_t* out = q + r * ldq;
  if (s.inverse == 0.f) {  // zeros, or infinities and NaN: every q is 0
    const float zero[VEC] = {};
#pragma unroll 1
    for (int c = threadIdx.x * VEC; c < width; c += blockDim.x * VEC) quantize_store<VEC>(out + c, zero, 0.f);
    return;
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (threadIdx.x + blockDim.x * i) * VEC;
    if (c < width) most = fmaxf(most, quantize_store<VEC>(out + c, v[i], s.inverse));
  }
  for (int c = (threadIdx.x + blockDim.x * V) * VEC; c < width; c += blockDim.x * VEC) {
    float w[VEC];
    load_vals<VEC>(x, x0 + c, type, w);
    most = fmaxf(most, quantize_store<VEC>(out + c, w, s.inverse));
  }
  // Rare (one thread in a few hundred): a value whose quotient may lie on the
  // other side of a half, or a row whose 127 / peak leaves fp32's range. The
  // thread's values are read again, out of the cache, and those divided.
  const bool tiny = s.peak < 1e-30f;
  if (tiny || most > kNearHalf) {
#pragma unroll 1
    for (int c = threadIdx.x * VEC; c < width; c += blockDim.x * VEC) {
      float w[VEC];
      load_vals<VEC>(x, x0 + c, type, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float off;
        rint_bits(w[j] * s.inverse, off);
        if (tiny || off > kNearHalf) out[c + j] = static_cast<int8_t>(rint_exact(w[j], s.peak) & 0xffu);
      }
    }
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
  const int elem = dtype == ND_F32 ? 4 : 2;
  const bool by4 = cols % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * elem) == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 4 == 0;
  const dim3 grid(static_cast<unsigned>(rows));
  const int w = static_cast<int>(cols);
#define ND_QR(VEC, V, T) \
  ND_CUDA(launch_pdl(quantize_rows_kernel<VEC, V>, grid, dim3(T), 0, stream, x, ldx, dtype, w, q, ldq, scale))
  if (by4) {
    const int64_t w4 = cols / 4;
    if (w4 <= 128) ND_QR(4, 1, 128);
    else if (w4 <= 512) ND_QR(4, 4, 128);
    else if (w4 <= 1024) ND_QR(4, 4, 256);
    else ND_QR(4, 12, 256);
  } else {
    if (cols <= 512) ND_QR(1, 4, 128);
    else ND_QR(1, 24, 256);
  }
#undef ND_QR
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

}  // namespace nd
