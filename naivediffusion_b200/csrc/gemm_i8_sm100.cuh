// int8 x int8 GEMM for sm_100a with a scale per row of A and per row of W:
//   C[m, n] = epilogue(sx[m] * sw[n] * sum_k A[m, k] W[n, k] + bias[n])
// on tcgen05.mma kind::i8: signed 8-bit operands, exact 32-bit integer sums in
// tensor memory. Both operands are K-major, 128 values (128 bytes) per k
// block, so tiles have the byte geometry of the 16-bit kernels' 64-deep
// blocks (128-byte swizzle, 32 bytes of K per instruction); a k block does
// twice the multiplications for the same bytes.
//
// The scales are applied to the finished sum in fp32: fma(float(sum) * sw, sx,
// bias), three roundings (the conversion of a sum above 2^24 is one), then the
// activation, then one rounding to the output type.
#pragma once

#include "gemm2_sm100.cuh"

namespace nd {

struct I8GemmArgs {
  int M, N, K;        // N: rows of W per group (2 F for the gated epilogues)
  int group_split;    // first row of group 1 (INT_MAX: one group)
  int shared_weights; // groups differ in bias / gate only, chosen per row
  int epi;            // GemmEpilogue
  int out_f16;
  int half;           // F for the gated epilogues, else 0
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  int bias_stride;
  const float* gate;
  long long gate_stride;
  const void* addend;
  long long ld_add;
  uint16_t* y;        // 16-bit output, or
  float* residual;    // the fp32 epilogues'
  long long ld;       // its row stride
  uint32_t idesc;
  unsigned* status;
};

// Instruction descriptor for kind::i8: signed 8-bit A and B, 32-bit integer D.
__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void umma_ss_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// A whole warp's wait: true only where every lane's is, so that after a timeout
// no part of the warp goes on alone into tcgen05 instructions that all of it
// has to run.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort, unsigned* status,
                                               unsigned where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, where));
}

// ------------------------------------------------------------ epilogue
// A warp's columns of the per-column vectors, staged in its own shared memory
// while the tile's MMAs run. With that, the paired fp32 arithmetic and the ex2 /
// rcp activations below the pair kernel's 8192 x 2048 x 8192 GELU went from
// 132 to 100 us on one box (25 to 13 instructions per output). It depends on the
// clock: 100-115 us in bursts, 127-134 us back to back at 1.49 GHz (erf 111 and
// 133, SILU 106 and 127, STORE 91 and 110):
//   words [0, 128)    w_scale     (gated: the first factor's 64, then the second's)
//   words [128, 256)  bias        (likewise)
//   words [256, 384)  gate
constexpr int kI8VecWords = 384;

// Lane l's four of the warp's columns: columns col + 4 l .. of a plain tile;
// gated, lanes 0..15 the first factor's columns, lanes 16..31 the second's.
// Columns at and past n are 0. Any alignment: a second weight group's vectors
// start wherever n puts them.
__device__ __forceinline__ void i8_stage_cols(uint32_t dst, const float* src, int col, int n, int half, int lane) {
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  if (src) {
    int c = col + 4 * lane;
    if (half > 0 && lane >= 16) {
      src += half;
      c -= 64;
    }
    if (c + 4 <= n && (reinterpret_cast<uintptr_t>(src + c) & 15u) == 0) {
      t = __ldg(reinterpret_cast<const float4*>(src + c));
    } else {
      if (c < n) t.x = __ldg(src + c);
      if (c + 1 < n) t.y = __ldg(src + c + 1);
      if (c + 2 < n) t.z = __ldg(src + c + 2);
      if (c + 3 < n) t.w = __ldg(src + c + 3);
    }
  }
  st_shared_v4(dst + lane * 16, __float_as_uint(t.x), __float_as_uint(t.y), __float_as_uint(t.z), __float_as_uint(t.w));
}

// A warp's place in the two bias / gate groups of shared weights: the group
// of its rows, and whether the split falls between them (then each lane reads
// its own group's bias and gate from global memory, and the staged ones are 0).
struct I8Rows {
  int bgroup;
  bool mixed;
};
__device__ __forceinline__ I8Rows i8_rows(const I8GemmArgs& a, int wgroup, int row0) {
  I8Rows r;
  r.bgroup = a.shared_weights ? (row0 >= a.group_split ? 1 : 0) : wgroup;
  r.mixed = a.shared_weights && row0 < a.group_split && row0 + 31 >= a.group_split;
  return r;
}

// Stage the warp's vectors for output columns [col, col + 128) (gated: + 64).
__device__ __forceinline__ void i8_stage_vectors(const I8GemmArgs& a, uint32_t vecs, int wgroup, const I8Rows& rows,
                                                 int col, int lane) {
  const int n = a.half > 0 ? a.half : a.N;
  const float* bias = a.bias && !rows.mixed ? a.bias + static_cast<long long>(rows.bgroup) * a.bias_stride : nullptr;
  __syncwarp();  // the previous tile's reads are done
  i8_stage_cols(vecs, a.w_scale + static_cast<long long>(wgroup) * a.N, col, n, a.half, lane);
  i8_stage_cols(vecs + 512, bias, col, n, a.half, lane);
  if (a.epi == kEpiResidualGate)
    i8_stage_cols(vecs + 1024, rows.mixed ? nullptr : a.gate + rows.bgroup * a.gate_stride, col, n, 0, lane);
  __syncwarp();
}

__device__ __forceinline__ float2 as_float2(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}

// Sums -> fma(float(sum) * sw, sx, bias) for 32 columns of this lane's row;
// `vecs` points at the first column's w_scale.
__device__ __forceinline__ void i8_scaled(const uint32_t (&r)[32], float sx, uint32_t vecs, float2 (&v)[16]) {
  const float2 sx2 = make_float2(sx, sx);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t w[4], b[4];
    ld_shared_v4(vecs + 16 * i, w[0], w[1], w[2], w[3]);
    ld_shared_v4(vecs + 512 + 16 * i, b[0], b[1], b[2], b[3]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 sum = make_float2(static_cast<float>(static_cast<int>(r[4 * i + 2 * j])),
                                     static_cast<float>(static_cast<int>(r[4 * i + 2 * j + 1])));
      v[2 * i + j] = ffma2(fmul2(sum, as_float2(w[2 * j], w[2 * j + 1])), sx2, as_float2(b[2 * j], b[2 * j + 1]));
    }
  }
}

// This lane's own 32 values in global memory, of which n exist, for a warp that
// straddles the split: its bias, v * sx + bias (v: sums times w_scale, not yet
// times sx, so that a row is rounded as often as in any other warp), or its gate,
// v * gate.
template <bool GATE>
__device__ __forceinline__ void i8_own(float2 (&v)[16], float sx, const float* own, int n) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float f = i < n ? __ldg(own + i) : 0.f;
    float& t = (i & 1) ? v[i >> 1].y : v[i >> 1].x;
    t = GATE ? t * f : fmaf(t, sx, f);
  }
}

// Activations to fp32 accuracy: exponentials and reciprocals on the SFU, a few
// ulp (tanh.approx, which the 16-bit kernels use, is off by 2^-11 of a tanh
// that 1 + tanh cancels for negative arguments). The .ftz forms: a result or
// operand below 2^-126 counts as 0, where a sigmoid is 0 or 1 to fp32. Where
// exp(-u) overflows the sigmoid is 0.
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// sigmoid(u) given -u * log2(e).
__device__ __forceinline__ float2 i8_sigmoid2(float2 t) {
  const float2 d = fadd2(make_float2(fast_exp2(t.x), fast_exp2(t.y)), make_float2(1.f, 1.f));
  return make_float2(fast_rcp(d.x), fast_rcp(d.y));
}
__device__ __forceinline__ float2 splat(float f) { return make_float2(f, f); }
__device__ __forceinline__ float2 i8_silu(float2 x) { return fmul2(x, i8_sigmoid2(fmul2(x, splat(-kLog2e)))); }
// x sigmoid(2 sqrt(2 / pi) (x + 0.044715 x^3))
__device__ __forceinline__ float2 i8_gelu_tanh(float2 x) {
  constexpr float c = -1.5957691216057308f * kLog2e;
  return fmul2(x, i8_sigmoid2(fmul2(x, ffma2(fmul2(x, x), splat(0.044715f * c), splat(c)))));
}
// Exact GELU, x (1 + erf(x / sqrt 2)) / 2 = max(x, 0) - |x| erfc(|x| / sqrt 2) / 2,
// with erfc(z) = (a1 t + .. + a5 t^5) exp(-z^2), t = 1 / (1 + p z): Abramowitz
// and Stegun 7.1.26, off by at most 1.5e-7, the form the reference's
// CpuMath.Gelu has. Half the instructions of erff. +inf counts as the largest
// finite |x|, whose erfc is 0 too: the last product would be inf * 0.
__device__ __forceinline__ float2 i8_gelu_erf(float2 x) {
  constexpr float kMost = 3.402823466e38f;
  const float2 ax = make_float2(fabsf(fminf(x.x, kMost)), fabsf(fminf(x.y, kMost)));
  const float2 d = ffma2(ax, splat(0.3275911f * 0.70710678118654752f), splat(1.f));
  const float2 t = make_float2(fast_rcp(d.x), fast_rcp(d.y));
  float2 p = ffma2(t, splat(1.061405429f), splat(-1.453152027f));
  p = ffma2(t, p, splat(1.421413741f));
  p = ffma2(t, p, splat(-0.284496736f));
  p = ffma2(t, p, splat(0.254829592f));
  const float2 z = fmul2(fmul2(x, x), splat(-0.5f * kLog2e));
  const float2 e = fmul2(fmul2(p, t), make_float2(fast_exp2(z.x), fast_exp2(z.y)));
  return ffma2(fmul2(ax, splat(-0.5f)), e, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
}

// One warp's [32 rows x 32 columns] chunk (lane = row) through its 4 KB of
// staging to TMA, in the tensor map's swizzle: 16-bit chunks alternate
// between two halves, fp32 ones take all of it. (Two 16-bit chunks as one store
// of 128-byte rows from a single buffer: 4096 x 640 x 5120 GEGLU 35 -> 44 us;
// three halves: no faster.)
//
// TMA clips a store's columns at 16 bytes, not at the tensor's width: where the
// width ends inside 16 bytes, the output's last chunk is stored from the
// registers instead, so that what lies beside it stays.
__device__ __forceinline__ void i8_emit(const I8GemmArgs& a, const CUtensorMap* tm, int kind, int width, uint32_t buf, int& sb,
                                        int lane, int row0, int col, const float2 (&v)[16]) {
  if (col + 32 > width && (width & (kind == kEmitBf16 || kind == kEmitF16 ? 7 : 3)) != 0) {
    if (row0 + lane < a.M) {
      const long long o = (row0 + lane) * a.ld + col;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (col + i < width) {
          const float f = (i & 1) ? v[i >> 1].y : v[i >> 1].x;
          if (kind == kEmitF32) a.residual[o + i] = f;
          else if (kind == kEmitAddF32) a.residual[o + i] += f;
          else a.y[o + i] = static_cast<uint16_t>(kind == kEmitF16 ? pack_f16(f, 0.f) : pack_bf16(f, 0.f));
        }
      }
    }
    __syncwarp();
    return;
  }
  if (kind == kEmitBf16 || kind == kEmitF16) {
    buf += static_cast<uint32_t>(sb) * 2048u;
    sb ^= 1;
    if (lane == 0) bulk_wait_read<1>();
    __syncwarp();
    uint32_t p[16];
    if (kind == kEmitF16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = pack_f16(v[i].x, v[i].y);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = pack_bf16(v[i].x, v[i].y);
    }
    // 64-byte rows, 64B swizzle: 16-byte chunk c of row r at c ^ ((r >> 1) & 3).
#pragma unroll
    for (int c = 0; c < 4; ++c)
      st_shared_v4(buf + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4), p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
  } else {
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
    // 128-byte rows, 128B swizzle: 16-byte chunk c of row r at c ^ (r & 7).
#pragma unroll
    for (int c = 0; c < 8; ++c)
      st_shared_v4(buf + lane * 128 + ((c ^ (lane & 7)) << 4), __float_as_uint(v[2 * c].x), __float_as_uint(v[2 * c].y),
                   __float_as_uint(v[2 * c + 1].x), __float_as_uint(v[2 * c + 1].y));
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (kind == kEmitAddF32) tma_reduce_add_2d(tm, buf, col, row0);
    else tma_store_2d(tm, buf, col, row0);
    bulk_commit();
  }
}

// One chunk of 32 output columns from `ocol`, rows row0 + lane: the sums `r`
// (and, for the gated epilogues, the second factor's sums `r2`) through the
// epilogue to the output's tensor map. `vecs`: the warp's staged vectors, `lc`
// the chunk's first column among them.
__device__ __forceinline__ void i8_chunk(const I8GemmArgs& a, const CUtensorMap* tmC, const I8Rows& rows, int row0,
                                         int ocol, int lc, float sx, const uint32_t (&r)[32], const uint32_t (&r2)[32],
                                         uint32_t vecs, uint32_t buf, int& sb, int lane) {
  const int row = row0 + lane;
  const bool second = row >= a.group_split;  // read by straddling warps only
  int kind = a.out_f16 ? kEmitF16 : kEmitBf16;
  const bool own_bias = rows.mixed && a.bias;
  const float sx1 = own_bias ? 1.f : sx;  // the staged bias is 0 then: sum * w_scale comes out as it is
  float2 v[16];
  i8_scaled(r, sx1, vecs + 4 * lc, v);
  if (a.half > 0) {
    float2 g[16];
    i8_scaled(r2, sx1, vecs + 4 * (64 + lc), g);
    if (own_bias) {
      const float* own = a.bias + (second ? a.bias_stride : 0) + ocol;
      i8_own<false>(v, sx, own, a.half - ocol);
      i8_own<false>(g, sx, own + a.half, a.half - ocol);
    }
    if (a.epi == kEpiGeGlu) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = fmul2(v[i], i8_gelu_erf(g[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = fmul2(i8_silu(v[i]), g[i]);
    }
    i8_emit(a, tmC, kind, a.half, buf, sb, lane, row0, ocol, v);
    return;
  }
  if (own_bias) i8_own<false>(v, sx, a.bias + (second ? a.bias_stride : 0) + ocol, a.N - ocol);
  switch (a.epi) {
    case kEpiGeluTanh:
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i8_gelu_tanh(v[i]);
      break;
    case kEpiGeluErf:
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i8_gelu_erf(v[i]);
      break;
    case kEpiSilu:
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i8_silu(v[i]);
      break;
    case kEpiResidualGate:
      if (rows.mixed) {
        i8_own<true>(v, 1.f, a.gate + (second ? a.gate_stride : 0) + ocol, a.N - ocol);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t g[4];
          ld_shared_v4(vecs + 1024 + 4 * lc + 16 * i, g[0], g[1], g[2], g[3]);
          v[2 * i] = fmul2(v[2 * i], as_float2(g[0], g[1]));
          v[2 * i + 1] = fmul2(v[2 * i + 1], as_float2(g[2], g[3]));
        }
      }
      kind = kEmitAddF32;
      break;
    case kEpiResidualAdd:
      kind = kEmitAddF32;
      break;
    case kEpiStoreF32:
      kind = kEmitF32;
      break;
    case kEpiAddStore:
      if (row < a.M) {
        const uint16_t* ad = static_cast<const uint16_t*>(a.addend) + static_cast<long long>(row) * a.ld_add + ocol;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (ocol + i < a.N) {
            const uint16_t h = ad[i];
            float& t = (i & 1) ? v[i >> 1].y : v[i >> 1].x;
            t += a.out_f16 ? __half2float(*reinterpret_cast<const __half*>(&h))
                           : __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(&h));
          }
        }
      }
      break;
    default:
      break;
  }
  i8_emit(a, tmC, kind, a.N, buf, sb, lane, row0, ocol, v);
}

template <int BN, int STAGES>
struct I8Smem {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kTiles = STAGES * kStageBytes;
  static constexpr int kEpiOffset = kTiles;  // 4 warps x 4 KB
  static constexpr int kVecOffset = kEpiOffset + 4 * 4096;
  static constexpr int kBarOffset = kVecOffset + 4 * kI8VecWords * 4;
  static constexpr int kNumBars = 2 * STAGES + 2;  // full[S], empty[S], acc_full, drain
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotal = kMiscOffset + 16;
  static constexpr int kLaunchBytes = kTotal + 1024;
};

__device__ __forceinline__ uint32_t cluster_nctas() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ int ld_shared_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// One 128 x BN tile per cluster of S CTAs, S = 1 where the tiles fill the GPU.
// With few tiles the k blocks are split over the cluster: each CTA sums its
// share, leaves its integer sums in its own shared memory (columns of 128
// rows, where the operand tiles were), and after a cluster barrier the tile's
// [32 x 32] chunks are divided over the CTAs, each chunk added up from all S
// shared memories. Integer sums: the split changes no bit, and nothing goes
// through global memory. 192 threads: warp 0 loads, warp 1 issues the MMAs,
// warps 2..5 are the epilogue (warp w reads TMEM lanes 32 (w % 4) on).
template <int BN, int STAGES>
__global__ void __launch_bounds__(192, 1)
    gemm_i8_sm100_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmC, const I8GemmArgs args) {
  using L = I8Smem<BN, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bars = sbase + L::kBarOffset;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  const uint32_t accf_bar = bars + 8u * (2 * STAGES);
  const uint32_t drain_bar = bars + 8u * (2 * STAGES + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_m = (args.M + 127) / 128;
  const int num_n = (args.N + BN - 1) / BN;
  const int splits = static_cast<int>(cluster_nctas());
  const int rank = static_cast<int>(cluster_ctarank());
  const int all_kb = (args.K + 127) / 128;
  const int kb0 = all_kb * rank / splits;  // this CTA's k blocks: at least one, the host sees to it
  const int num_kb = all_kb * (rank + 1) / splits - kb0;
  int mt, nt;
  tile_coords(blockIdx.x / splits, num_m, num_n, mt, nt);
  const int m0 = mt * 128;
  const int wgroup = !args.shared_weights && m0 >= args.group_split ? 1 : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(accf_bar, 1);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmC);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch();
  griddep_wait();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, issued_parity = 0;
      bool ok = true;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, args.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        const uint32_t a_dst = sbase + stage * L::kStageBytes;
        const uint32_t b_dst = a_dst + L::kABytes;
        mbar_arrive_expect_tx(full_bar(stage), L::kStageBytes);
        const int k0 = (kb0 + kb) * 128;
        tma_load_2d(a_dst, &tmA, full_bar(stage), k0, m0);
        if (args.half > 0) {
          tma_load_2d(b_dst, &tmB, full_bar(stage), k0, wgroup * args.N + nt * (BN / 2));
          tma_load_2d(b_dst + (BN / 2) * 128, &tmB, full_bar(stage), k0,
                      wgroup * args.N + args.half + nt * (BN / 2));
        } else {
          tma_load_2d(b_dst, &tmB, full_bar(stage), k0, wgroup * args.N + nt * BN);
        }
        issued |= 1u << stage;
        issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        // Aborted: let the loads in flight land before shared memory goes away.
        volatile int never = 0;
        for (int s = 0; s < STAGES; ++s)
          if (issued & (1u << s)) mbar_wait(full_bar(s), (issued_parity >> s) & 1u, &never, nullptr, 0);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(full_bar(stage), phase, abort_flag, args.status, kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = sbase + stage * L::kStageBytes;
        const uint32_t b_addr = a_addr + L::kABytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ss_i8(tmem_base, make_sdesc_sw128(a_addr + k * 32, 16, 1024), make_sdesc_sw128(b_addr + k * 32, 16, 1024),
                     args.idesc, (kb | k) != 0 ? 1u : 0u);
        umma_commit(empty_bar(stage));
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) umma_commit(accf_bar);
      umma_commit(drain_bar);
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never, args.status, kStatusTimeoutDrain);
    }
  } else {
    const int ew = warp & 3;
    const int row0 = m0 + ew * 32;
    const uint32_t buf = sbase + L::kEpiOffset + ew * 4096;
    const uint32_t vecs = sbase + L::kVecOffset + ew * kI8VecWords * 4;
    const I8Rows rows = i8_rows(args, wgroup, row0);
    const float sx = row0 + lane < args.M ? __ldg(args.x_scale + row0 + lane) : 0.f;
    int sb = 0;
    const int width = args.half > 0 ? args.half : args.N;
    const int per_tile = args.half > 0 ? BN / 2 : BN;
    const int col0 = nt * per_tile;
    if (row0 < args.M && splits == 1) i8_stage_vectors(args, vecs, wgroup, rows, col0, lane);
    if (row0 < args.M && mbar_wait_warp(accf_bar, 0, abort_flag, args.status, kStatusTimeoutEpilogue)) {
      __syncwarp();
      tc_fence_after();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(ew * 32) << 16);
      if (splits == 1) {
#pragma unroll 1
        for (int c = 0; c < per_tile / 32 && col0 + c * 32 < width; ++c) {
          uint32_t r[32], r2[32];
          tmem_ld32(tbase + c * 32, r);
          if (args.half > 0) tmem_ld32(tbase + BN / 2 + c * 32, r2);
          tmem_ld_wait();
          i8_chunk(args, &tmC, rows, row0, col0 + c * 32, c * 32, sx, r, r2, vecs, buf, sb, lane);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(tbase + c * 32, r);
          tmem_ld_wait();
          const uint32_t dst = sbase + (c * 32 * 128 + ew * 32 + lane) * 4;
#pragma unroll
          for (int i = 0; i < 32; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + i * 512), "r"(r[i]) : "memory");
        }
      }
      tc_fence_before();
    }
    if (splits == 1 && lane == 0) bulk_wait_read<0>();
  }
  __syncwarp();
  tc_fence_before();
  if (splits == 1) {
    __syncthreads();
  } else {
    // Every CTA of the cluster gets here, timed out or not.
    cluster_sync_all();
    if (warp >= 2) {
      const int ew = warp - 2;
      const uint32_t buf = sbase + L::kEpiOffset + ew * 4096;
      const uint32_t vecs = sbase + L::kVecOffset + ew * kI8VecWords * 4;
      const int width = args.half > 0 ? args.half : args.N;
      const int per_tile = args.half > 0 ? BN / 2 : BN;
      const int col0 = nt * per_tile;
      const int quarters = min(4, (args.M - m0 + 31) / 32);  // of rows that exist
      const int chunks = min(per_tile / 32, (width - col0 + 31) / 32);
      int sb = 0;
      // Chunk u of the tile: its columns are u / quarters, its rows u % quarters.
#pragma unroll 1
      for (int u = rank + splits * ew; u < quarters * chunks; u += 4 * splits) {
        const int c = u / quarters, q = u % quarters;
        const int row0 = m0 + q * 32;
        const I8Rows rows = i8_rows(args, wgroup, row0);
        i8_stage_vectors(args, vecs, wgroup, rows, col0, lane);
        const float sx = row0 + lane < args.M ? __ldg(args.x_scale + row0 + lane) : 0.f;
        const uint32_t at = sbase + (c * 32 * 128 + q * 32 + lane) * 4;
        uint32_t r[32], r2[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = r2[i] = 0u;
#pragma unroll 1
        for (int s = 0; s < splits; ++s) {
          const uint32_t src = mapa_shared(at, static_cast<uint32_t>(s));
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] += ld_shared_cluster(src + i * 512);
          if (args.half > 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) r2[i] += ld_shared_cluster(src + BN / 2 * 512 + i * 512);
          }
        }
        i8_chunk(args, &tmC, rows, row0, col0 + c * 32, c * 32, sx, r, r2, vecs, buf, sb, lane);
      }
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
    }
    cluster_sync_all();  // no shared memory goes away while a peer reads it
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, BN);
}

}  // namespace nd
