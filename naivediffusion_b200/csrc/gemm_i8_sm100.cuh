// int8 x int8 GEMM for sm_100a with a scale per row of A and per row of W:
//   C[m, n] = epilogue(sx[m] * sw[n] * sum_k A[m, k] W[n, k] + bias[n])
// on tcgen05.mma kind::i8: signed 8-bit operands, exact 32-bit integer sums in
// tensor memory. Both operands are K-major, 128 values (128 bytes) per k
// block, so tiles have the byte geometry of the 16-bit kernels' 64-deep
// blocks (128-byte swizzle, 32 bytes of K per instruction); a k block does
// twice the multiplications for the same bytes.
//
// The scales are applied to the finished sum in fp32: (float(sum) * sx) * sw,
// three roundings (the conversion of a sum above 2^24 is one), then the bias
// and the activation, then one rounding to the output type.
#pragma once

#include "gemm_sm100.cuh"

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

// 32 values of a per-column vector from `col` on; columns at and past n read
// as 0. Any alignment: a second weight group's vectors start wherever n puts
// them.
__device__ __forceinline__ void load_cols32(const float* src, int col, int n, float (&v)[32]) {
  if (col + 32 <= n && (reinterpret_cast<uintptr_t>(src + col) & 15u) == 0) {
    const float4* s = reinterpret_cast<const float4*>(src + col);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 t = __ldg(s + i);
      v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = (col + i < n) ? __ldg(src + col + i) : 0.f;
  }
}

// Sums -> (float(sum) * sx) * sw + bias for 32 columns of this lane's row.
__device__ __forceinline__ void i8_scaled(const I8GemmArgs& a, const uint32_t (&r)[32], float sx, const float* sw,
                                          const float* bias, int col, int n, float (&v)[32]) {
  float w[32];
  load_cols32(sw, col, n, w);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = static_cast<float>(static_cast<int>(r[i])) * sx * w[i];
  if (bias) {
    load_cols32(bias, col, n, w);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += w[i];
  }
}

// Activations to fp32 accuracy: exponentials and reciprocals on the SFU,
// a few ulp (the 16-bit kernels' tanh.approx is 2^-11 of tanh, which a large
// negative argument multiplies).
__device__ __forceinline__ float i8_sigmoid(float u) { return __fdividef(1.0f, 1.0f + __expf(-u)); }
__device__ __forceinline__ float i8_silu(float x) {
  // exp(-x) overflows below -88: x * 0 is the limit (-0), not -inf * 0.
  return x * i8_sigmoid(x);
}
__device__ __forceinline__ float i8_gelu_tanh(float x) {
  return x * i8_sigmoid(1.5957691216f * fmaf(0.044715f * x, x * x, x));
}

// One chunk of 32 output columns from `ocol`, rows row0 + lane: the sums `r`
// (and, for the gated epilogues, the second factor's sums `r2`) through the
// epilogue to the output's tensor map.
__device__ __forceinline__ void i8_chunk(const I8GemmArgs& a, const CUtensorMap* tmC, int wgroup, int row0, int ocol,
                                         float sx, const uint32_t (&r)[32], const uint32_t (&r2)[32], uint32_t buf0,
                                         int& sb, int lane) {
  const int row = row0 + lane;
  const int bgroup = a.shared_weights ? (row >= a.group_split ? 1 : 0) : wgroup;
  const float* sw = a.w_scale + static_cast<long long>(wgroup) * a.N;
  const float* bias = a.bias ? a.bias + static_cast<long long>(bgroup) * a.bias_stride : nullptr;
  int kind = a.out_f16 ? kEmitF16 : kEmitBf16;
  float v[32];
  if (a.half > 0) {
    float g[32];
    i8_scaled(a, r, sx, sw, bias, ocol, a.half, v);
    i8_scaled(a, r2, sx, sw + a.half, bias ? bias + a.half : nullptr, ocol, a.half, g);
    if (a.epi == kEpiGeGlu) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= gelu_erf(g[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i8_silu(v[i]) * g[i];
    }
    emit_chunk(tmC, kind, buf0, sb, lane, row0, a.M, ocol, v);
    return;
  }
  i8_scaled(a, r, sx, sw, bias, ocol, a.N, v);
  switch (a.epi) {
    case kEpiGeluTanh:
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i8_gelu_tanh(v[i]);
      break;
    case kEpiGeluErf:
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = gelu_erf(v[i]);
      break;
    case kEpiSilu:
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i8_silu(v[i]);
      break;
    case kEpiResidualGate: {
      float g[32];
      load_cols32(a.gate + bgroup * a.gate_stride, ocol, a.N, g);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= g[i];
      kind = kEmitAddF32;
      break;
    }
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
            v[i] += a.out_f16 ? __half2float(*reinterpret_cast<const __half*>(&h))
                              : __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(&h));
          }
        }
      }
      break;
    default:
      break;
  }
  emit_chunk(tmC, kind, buf0, sb, lane, row0, a.M, ocol, v);
}

template <int BN, int STAGES>
struct I8Smem {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kTiles = STAGES * kStageBytes;
  static constexpr int kEpiOffset = kTiles;  // 4 warps x 2 buffers x 4 KB
  static constexpr int kBarOffset = kEpiOffset + 4 * 2 * 4096;
  static constexpr int kNumBars = 2 * STAGES + 2;  // full[S], empty[S], acc_full, drain
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotal = kMiscOffset + 16;
  static constexpr int kLaunchBytes = kTotal + 1024;
};

// One 128 x BN tile per CTA. 192 threads: warp 0 loads, warp 1 issues the
// MMAs, warps 2..5 are the epilogue (warp w reads TMEM lanes 32 (w % 4) on).
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
  const int num_kb = (args.K + 127) / 128;
  int mt, nt;
  tile_coords(blockIdx.x, num_m, num_n, mt, nt);
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
        tma_load_2d(a_dst, &tmA, full_bar(stage), kb * 128, m0);
        if (args.half > 0) {
          tma_load_2d(b_dst, &tmB, full_bar(stage), kb * 128, wgroup * args.N + nt * (BN / 2));
          tma_load_2d(b_dst + (BN / 2) * 128, &tmB, full_bar(stage), kb * 128,
                      wgroup * args.N + args.half + nt * (BN / 2));
        } else {
          tma_load_2d(b_dst, &tmB, full_bar(stage), kb * 128, wgroup * args.N + nt * BN);
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
    const uint32_t buf0 = sbase + L::kEpiOffset + ew * 2 * 4096;
    int sb = 0;
    if (row0 < args.M && mbar_wait(accf_bar, 0, abort_flag, args.status, kStatusTimeoutEpilogue)) {
      __syncwarp();
      tc_fence_after();
      const float sx = row0 + lane < args.M ? __ldg(args.x_scale + row0 + lane) : 0.f;
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(ew * 32) << 16);
      const int width = args.half > 0 ? args.half : args.N;
      const int per_tile = args.half > 0 ? BN / 2 : BN;
#pragma unroll 1
      for (int c = 0; c < per_tile / 32; ++c) {
        const int ocol = nt * per_tile + c * 32;
        if (ocol >= width) break;
        uint32_t r[32], r2[32];
        tmem_ld32(tbase + c * 32, r);
        if (args.half > 0) tmem_ld32(tbase + BN / 2 + c * 32, r2);
        tmem_ld_wait();
        i8_chunk(args, &tmC, wgroup, row0, ocol, sx, r, r2, buf0, sb, lane);
      }
      tc_fence_before();
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, BN);
}

}  // namespace nd
