// int8 x int8 product for a few rows (single tokens, modulation vectors):
// bound by reading the weights once, at most kGemvI8Rows rows of x against
// every weight row on the CUDA cores' dp4a.
//
// A warp takes two weight rows (the two factors' rows of one output for the
// gated epilogues): lane l reads 16-byte groups l, l + 32, .. of both rows,
// kGroups of each in flight, against the same groups of x, which stay in L1.
// One warp per pair of rows and about one wave of blocks, so every load of the
// weights is in flight early: 1 x 4096 x 12288 9.5 us (5.3 TB/s) over three
// layers' weights in turn (150 MB, which L2 partly holds), 10.8 us (4.7 TB/s) over
// twelve layers' (600 MB). Two rows of x
// take two groups and 48 warps per SM (10.2 us against 12.4 with four groups);
// one, three and four rows lose by that (4 x 4096 x 12288 12.9 against 18.4).
#pragma once

#include "gemm_i8_sm100.cuh"

namespace nd {

// At four rows against gemm_i8_few_kernel, us: 1024 x 1024 2.5 / 5.4, 4096 x 12288
// 12.9 / 12.9; a fifth row of x would double the loads from L1 per weight.
constexpr int kGemvI8Rows = 4;
constexpr int kGemvI8Threads = 128;

// 16 bytes that are read once.
__device__ __forceinline__ uint4 load16_once(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// The first `n` of 16 bytes, the others 0: a row's end need not be followed
// by readable memory.
__device__ __forceinline__ uint4 load16_part(const int8_t* p, int n) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < n) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int c) {
  c = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), c);
  c = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), c);
  c = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), c);
  return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), c);
}

struct I8GemvArgs {
  I8GemmArgs g;
  const int8_t* x;
  const int8_t* w;
  long long ldx, ldw;
};

__device__ __forceinline__ float load_16bit(const void* p, long long i, int f16) {
  return f16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

template <int MR>
__global__ void __launch_bounds__(kGemvI8Threads, MR == 1 ? 9 : MR == 2 ? 12 : 7) gemv_i8_kernel(const I8GemvArgs args) {
  constexpr int kGroups = MR == 2 ? 2 : 4;
  griddep_launch();
  griddep_wait();
  const I8GemmArgs& a = args.g;
  // Blocks times warps: the threads' own numbers pass 32 bits at 2^27 gated outputs.
  const int warp = static_cast<int>(blockIdx.x) * (kGemvI8Threads / 32) + static_cast<int>(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const bool gated = a.half > 0;
  const int n0 = gated ? warp : 2 * warp;
  const int n1 = gated ? warp + a.half : 2 * warp + 1;
  if (n0 >= (gated ? a.half : a.N)) return;
  const bool have1 = n1 < a.N;
  const int8_t* w0 = args.w + n0 * args.ldw;
  const int8_t* w1 = args.w + (have1 ? n1 : n0) * args.ldw;
  const int groups = a.K >> 4;
  int acc[MR][2];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m][0] = acc[m][1] = 0;

  for (int c0 = lane; c0 < groups; c0 += 32 * kGroups) {
    uint4 p[kGroups], q[kGroups];
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int c = c0 + 32 * u;
      p[u] = q[u] = make_uint4(0u, 0u, 0u, 0u);
      if (c < groups) {
        p[u] = load16_once(w0 + 16 * c);
        q[u] = load16_once(w1 + 16 * c);
      }
    }
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int c = c0 + 32 * u;
      if (c < groups) {
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(args.x + m * args.ldx) + c);
          acc[m][0] = dot16(x, p[u], acc[m][0]);
          acc[m][1] = dot16(x, q[u], acc[m][1]);
        }
      }
    }
  }
  const int rest = a.K & 15;
  if (rest && lane == 0) {
    const int k = groups * 16;
    const uint4 p = load16_part(w0 + k, rest), q = load16_part(w1 + k, rest);
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const uint4 x = load16_part(args.x + m * args.ldx + k, rest);
      acc[m][0] = dot16(x, p, acc[m][0]);
      acc[m][1] = dot16(x, q, acc[m][1]);
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[m][j] = __reduce_add_sync(0xffffffffu, acc[m][j]);

  // Lane 2 m + j finishes row m's column n_j (gated: lane 2 m, both factors).
  if (lane >= 2 * MR) return;
  const int m = lane >> 1, j = lane & 1;
  int s0 = 0, s1 = 0;
#pragma unroll
  for (int i = 0; i < MR; ++i)
    if (i == m) {
      s0 = acc[i][0];
      s1 = acc[i][1];
    }
  if (gated ? j == 1 : (j == 1 && !have1)) return;
  const int col = j ? n1 : n0;
  const bool second = a.shared_weights && m >= a.group_split;
  const float sx = __ldg(a.x_scale + m);
  const float* bias = a.bias ? a.bias + (second ? a.bias_stride : 0) : nullptr;
  auto scaled = [&](int sum, int n) {
    return fmaf(static_cast<float>(sum) * __ldg(a.w_scale + n), sx, bias ? __ldg(bias + n) : 0.f);
  };
  float v = scaled(j ? s1 : s0, col);
  switch (a.epi) {
    case kEpiGeluTanh: v = i8_gelu_tanh(splat(v)).x; break;
    case kEpiGeluErf: v = i8_gelu_erf(splat(v)).x; break;
    case kEpiSilu: v = i8_silu(splat(v)).x; break;
    case kEpiSwiGlu: v = i8_silu(splat(v)).x * scaled(s1, n1); break;
    case kEpiGeGlu: v *= i8_gelu_erf(splat(scaled(s1, n1))).x; break;
    case kEpiResidualGate: v *= __ldg(a.gate + (second ? a.gate_stride : 0) + col); break;
    case kEpiAddStore: v += load_16bit(a.addend, m * a.ld_add + col, a.out_f16); break;
    default: break;
  }
  const long long at = m * a.ld + col;
  if (a.epi == kEpiStoreF32) a.residual[at] = v;
  else if (a.epi == kEpiResidualGate || a.epi == kEpiResidualAdd) a.residual[at] += v;
  else a.y[at] = static_cast<uint16_t>(a.out_f16 ? pack_f16(v, 0.f) : pack_bf16(v, 0.f));
}

}  // namespace nd
