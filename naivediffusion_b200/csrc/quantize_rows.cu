// Activations as int8 with one scale per row (token), the operand of the
// int8 x int8 product (linear_w8a8):
//
//   scale[r] = max |x[r]| / 127,   q[r, c] = rint(x[r, c] * 127 / max |x[r]|)
//
// The quotient is rounded as if computed exactly, half to even. 127 / peak is
// held as a sum hi + lo of two fp32 values (2^-47 of it is missing), and
// t = fma(x, hi, x * lo) is then the exact quotient rounded to fp32: a quotient
// that is a half comes out as that half, and for 16-bit x any other differs
// from a half by more than 1.9e-6 of itself, where t is off by 2^-24. Two fp32
// values may have a quotient closer to a half than fp32 resolves; where t is a
// half, x * 127 - r * peak decides, which two products and their fma remainders
// give exactly (near_half). With 127 / peak in one fp32 value the near-half
// check was needed for 16-bit x too (half the peak is common): 30 us at
// 4352 x 12288 where this takes 26.
//
// Bound by HBM: the row is read once, stays in registers while its peak is
// found, and one byte per value is written. 4352 x 12288 bf16 26 us (6.1 TB/s,
// 93 % of the copy rate), 8192 x 8192 bf16 30 us, 4352 x 4096 fp32 14 us (98 %); rows that are no
// multiple of 8 values are read a value at a time, four neighbours per thread
// (1001 x 5121 fp32 8.1 us, 48 %; 4000 x 9001 bf16 46 us where one value per
// thread and store took 54).
#include <algorithm>
#include <climits>

#include "nd_common.cuh"
#include "nd_internal.h"
#include "nd_runtime.h"
#include "row_quant.cuh"

namespace nd {

namespace {

// A thread's share of a row as it lies in memory: VEC values of one type. The
// 16-bit types stay packed until they are quantized (half the registers, so
// twice the rows in flight), and |x| is compared as integers: bit patterns of
// one sign order like the values, with NaN above infinity. VEC = 8: vector loads
// (aligned rows); 4: single loads of four neighbours (rows of any width and
// alignment, whose int8 rows still take 4-byte stores), of which `n` exist; 1.
template <int TYPE, int VEC>
struct Raw;
template <>
struct Raw<ND_F32, 8> {
  float4 w[2];
  __device__ __forceinline__ void clear() { w[0] = w[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const void* p, long long i, int) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(w[h].x), "=f"(w[h].y), "=f"(w[h].z), "=f"(w[h].w)
                   : "l"(static_cast<const float*>(p) + i + 4 * h));
  }
  __device__ __forceinline__ void peak(uint32_t& m) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      m = max(max(m, max(abs_bits(w[h].x), abs_bits(w[h].y))), max(abs_bits(w[h].z), abs_bits(w[h].w)));
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f[4 * h] = w[h].x; f[4 * h + 1] = w[h].y; f[4 * h + 2] = w[h].z; f[4 * h + 3] = w[h].w;
    }
  }
};
template <>
struct Raw<ND_F32, 1> {
  float w;
  __device__ __forceinline__ void clear() { w = 0.f; }
  __device__ __forceinline__ void load(const void* p, long long i, int) { w = __ldg(static_cast<const float*>(p) + i); }
  __device__ __forceinline__ void peak(uint32_t& m) const { m = max(m, abs_bits(w)); }
  __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = w; }
};
template <>
struct Raw<ND_F32, 4> {
  float w[4];
  __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0.f; }
  __device__ __forceinline__ void load(const void* p, long long i, int n) {
    const float* f = static_cast<const float*>(p) + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = j < n ? __ldg(f + j) : 0.f;
  }
  __device__ __forceinline__ void peak(uint32_t& m) const {
    m = max(max(m, max(abs_bits(w[0]), abs_bits(w[1]))), max(abs_bits(w[2]), abs_bits(w[3])));
  }
  __device__ __forceinline__ void values(float (&f)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = w[j];
  }
};
template <int TYPE>
__device__ __forceinline__ float2 halves(uint32_t w) {
  if constexpr (TYPE == ND_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int TYPE>
struct Raw<TYPE, 8> {
  uint4 w;
  __device__ __forceinline__ void clear() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const void* p, long long i, int) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "l"(static_cast<const uint16_t*>(p) + i));
  }
  __device__ __forceinline__ void peak(uint32_t& m) const {  // two 16-bit maxima
    constexpr uint32_t k = 0x7fff7fffu;
    m = __vmaxu2(__vmaxu2(m, __vmaxu2(w.x & k, w.y & k)), __vmaxu2(w.z & k, w.w & k));
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = halves<TYPE>(v[j]);
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  }
};
template <int TYPE>
struct Raw<TYPE, 4> {
  uint32_t w[2];
  __device__ __forceinline__ void clear() { w[0] = w[1] = 0u; }
  __device__ __forceinline__ void load(const void* p, long long i, int n) {
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
    uint32_t t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = j < n ? __ldg(h + j) : 0u;
    w[0] = __byte_perm(t[0], t[1], 0x5410);
    w[1] = __byte_perm(t[2], t[3], 0x5410);
  }
  __device__ __forceinline__ void peak(uint32_t& m) const {  // two 16-bit maxima
    m = __vmaxu2(m, __vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu));
  }
  __device__ __forceinline__ void values(float (&f)[4]) const {
    const float2 a = halves<TYPE>(w[0]), b = halves<TYPE>(w[1]);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  }
};
template <int TYPE>
struct Raw<TYPE, 1> {
  uint16_t w;
  __device__ __forceinline__ void clear() { w = 0; }
  __device__ __forceinline__ void load(const void* p, long long i, int) { w = __ldg(static_cast<const uint16_t*>(p) + i); }
  __device__ __forceinline__ void peak(uint32_t& m) const { m = max(m, static_cast<uint32_t>(w & 0x7fff)); }
  __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = halves<TYPE>(w).x; }
};
// The peak's bits as fp32's.
template <int TYPE>
__device__ __forceinline__ uint32_t peak_bits(uint32_t m) {
  if constexpr (TYPE == ND_F32) return m;
  else return __float_as_uint(halves<TYPE>(max(m & 0xffffu, m >> 16)).x);
}

// VEC values (already multiplied by range_shift) to int8, of which n exist.
template <int TYPE, int VEC>
__device__ __forceinline__ void quantize_store(int8_t* q, const float (&f)[VEC], Inverse inv, float peak, int n) {
  float m[VEC];
  quantize_values<TYPE == ND_F32>(f, inv, peak, m);
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint2*>(q) =
        make_uint2(pack_low_bytes(__float_as_uint(m[0]), __float_as_uint(m[1]), __float_as_uint(m[2]), __float_as_uint(m[3])),
                   pack_low_bytes(__float_as_uint(m[4]), __float_as_uint(m[5]), __float_as_uint(m[6]), __float_as_uint(m[7])));
  } else if constexpr (VEC == 4) {
    const uint32_t w = pack_low_bytes(__float_as_uint(m[0]), __float_as_uint(m[1]), __float_as_uint(m[2]), __float_as_uint(m[3]));
    if (n >= 4) {
      *reinterpret_cast<uint32_t*>(q) = w;
    } else {
      for (int j = 0; j < n; ++j) q[j] = static_cast<int8_t>((w >> (8 * j)) & 0xffu);
    }
  } else {
    *q = static_cast<int8_t>(__float_as_uint(m[0]) & 0xffu);
  }
}

template <int T>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < T / 32; ++i) v = max(v, red[i]);
  }
  return v;
}

// T threads per row (a warp for narrow rows, four rows to a block), V x VEC
// values per thread in registers, the rest of a longer row read twice.
// 1536 threads per SM (40 registers; fp32 vectors take 64) keep enough rows in
// flight: with fp32 values in registers and 1024 threads 4352 x 12288 bf16 took
// 52 us, and 32768 x 640 with a block per row 35 us where four warps take 14.
template <int TYPE, int VEC, int V, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T, (TYPE == ND_F32 && VEC == 8 ? 1024 : 1536) / (T < 128 ? 128 : T))
    quantize_rows_kernel(const void* x, long long ldx, int rows, int width, int8_t* q, long long ldq, float* scale) {
  griddep_launch();
  griddep_wait();
  __shared__ uint32_t red[T / 32];
  constexpr int kRows = T < 128 ? 128 / T : 1;
  const int t = threadIdx.x % T;
  const long long r = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / T;
  if (r >= rows) return;  // whole warps: only T = 32 has several rows per block
  const long long x0 = r * ldx;
  Raw<TYPE, VEC> v[V];
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + T * i) * VEC;
    v[i].clear();
    if (c < width) v[i].load(x, x0 + c, width - c);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i].peak(peak);
  for (int c = (t + T * V) * VEC; c < width; c += T * VEC) {
    Raw<TYPE, VEC> w;
    w.load(x, x0 + c, width - c);
    w.peak(peak);
  }
  const RowScale s = row_scale(block_max<T>(peak_bits<TYPE>(peak), red));
  if (t == 0) scale[r] = s.scale;
  int8_t* out = q + r * ldq;
  if (s.zero) {
    const float zero[VEC] = {};
#pragma unroll 1
    for (int c = t * VEC; c < width; c += T * VEC) quantize_store<TYPE, VEC>(out + c, zero, Inverse{0.f, 0.f}, 1.f, width - c);
    return;
  }
  const float shift = range_shift(s.peak);
  const float row_peak = s.peak * shift;
  const Inverse inverse = inverse_of(row_peak);
  auto finish = [&](int c, const Raw<TYPE, VEC>& raw) {
    float w[VEC];
    raw.values(w);
    if (shift != 1.f) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] *= shift;
    }
    quantize_store<TYPE, VEC>(out + c, w, inverse, row_peak, width - c);
  };
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + T * i) * VEC;
    if (c < width) finish(c, v[i]);
  }
  for (int c = (t + T * V) * VEC; c < width; c += T * VEC) {
    Raw<TYPE, VEC> w;
    w.load(x, x0 + c, width - c);
    finish(c, w);
  }
}

template <int TYPE>
int launch(const void* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
           cudaStream_t stream) {
  const bool by8 = cols % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const int w = static_cast<int>(cols), n = static_cast<int>(rows);
#define ND_QR(VEC, V, T)                                                                                            \
  ND_CUDA(launch_pdl(quantize_rows_kernel<TYPE, VEC, V, T>, dim3((n + (T < 128 ? 128 / T : 1) - 1) /                  \
                     (T < 128 ? 128 / T : 1)), dim3(T < 128 ? 128 : T), 0, stream, x, ldx, n, w, q, ldq, scale))
  if (by8) {
    const int64_t w8 = cols / 8;
    if (w8 <= 64) ND_QR(8, 2, 32);
    else if (w8 <= 128) ND_QR(8, 4, 32);
    else if (w8 <= 256) ND_QR(8, 2, 128);
    else if (w8 <= 512) ND_QR(8, 4, 128);
    else if (w8 <= 1024) ND_QR(8, 4, 256);
    else if (w8 <= 1536) ND_QR(8, 3, 512);
    else ND_QR(8, 4, 512);
  } else if (ldq % 4 == 0 && reinterpret_cast<uintptr_t>(q) % 4 == 0) {
    if (cols <= 512) ND_QR(4, 4, 32);
    else if (cols <= 2048) ND_QR(4, 4, 128);
    else if (cols <= 4096) ND_QR(4, 4, 256);
    else ND_QR(4, 4, 512);
  } else {
    if (cols <= 2048) ND_QR(1, 8, 256);
    else ND_QR(1, 12, 512);
  }
#undef ND_QR
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

}  // namespace

int quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                  float* scale, cudaStream_t stream) {
  if (dtype != ND_F32 && dtype != ND_F16 && dtype != ND_BF16)
    return fail(ND_ERR_INVALID, "quantize_rows: x must be f32, f16 or bf16");
  if (rows <= 0 || cols <= 0) return fail(ND_ERR_INVALID, "quantize_rows: empty shape");
  if (rows > INT_MAX - 128 || cols > INT_MAX / 2) return fail(ND_ERR_INVALID, "quantize_rows: shape too large");
  if (!x || !q || !scale) return fail(ND_ERR_INVALID, "quantize_rows: null operand");
  if (ldx < cols || ldq < cols) return fail(ND_ERR_INVALID, "quantize_rows: a row stride is smaller than cols");
  if (dtype == ND_F32) return launch<ND_F32>(x, rows, cols, ldx, q, ldq, scale, stream);
  if (dtype == ND_F16) return launch<ND_F16>(x, rows, cols, ldx, q, ldq, scale, stream);
  return launch<ND_BF16>(x, rows, cols, ldx, q, ldq, scale, stream);
}

}  // namespace nd
