// int8 x int8 product for few rows (5 to 64 tokens): bound by streaming the
// weights, so the operands change places. 128 weight rows are the MMA's M side
// and NT tokens its N side: a k block is 16 KB of weights and NT x 128 B of
// tokens instead of a 128-row token tile that is mostly padding, and as many k
// blocks as shared memory holds are in flight (the loop runs at a load's
// latency divided by their number).
//
// One tile of 128 weight rows per cluster of S CTAs. Gated, the tile's rows
// are 16 of the first factor, the 16 matching ones of the second, and so on,
// so that each warp's 32 TMEM lanes hold both factors of 16 outputs.
//  S = 1: a lane owns one weight row and finishes its tokens straight out of
//         TMEM (gated: lane l and l + 16 exchange factors and take every
//         other token).
//  S > 1: the k blocks are split over the cluster. Every CTA leaves its
//         integer sums in shared memory, [token][weight row]; after a cluster
//         barrier the tokens are divided over the CTAs and each sum is added
//         up from all S shared memories.
#pragma once

#include "gemv_i8.cuh"

namespace nd {

template <int NT, int STAGES>
struct I8FewSmem {
  static constexpr int kWBytes = 128 * 128;
  static constexpr int kXBytes = NT * 128;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kBarOffset = STAGES * kStageBytes;  // the sums take the stages' place
  static constexpr int kNumBars = 2 * STAGES + 2;          // full[S], empty[S], acc_full, drain
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotal = kMiscOffset + 16;
  static constexpr int kLaunchBytes = kTotal + 1024;
  static constexpr int kTmemCols = NT < 32 ? 32 : NT;
};

__device__ __forceinline__ int2 ld_shared_cluster2(uint32_t addr) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// One finished value v (the epilogue's activations are applied) at (m, col).
__device__ __forceinline__ void few_store(const I8GemmArgs& a, int m, int col, float v) {
  const long long o = m * a.ld + col;
  if (a.epi == kEpiStoreF32) a.residual[o] = v;
  else if (a.epi == kEpiResidualGate || a.epi == kEpiResidualAdd) a.residual[o] += v;
  else a.y[o] = static_cast<uint16_t>(a.out_f16 ? pack_f16(v, 0.f) : pack_bf16(v, 0.f));
}

// S = 1: this lane's weight row of tile `tile` against every token.
template <int NT>
__device__ __forceinline__ void few_direct(const I8GemmArgs& a, uint32_t tbase, int tile, int ew, int lane) {
  const bool gated = a.half > 0;
  const int col = gated ? tile * 64 + ew * 16 + (lane & 15) : tile * 128 + ew * 32 + lane;
  const int wrow = gated && lane >= 16 ? a.half + col : col;
  const bool live = col < (gated ? a.half : a.N);
  auto load = [&](const float* p, long long i) { return live && p ? __ldg(p + i) : 0.f; };
  const float sw = load(a.w_scale, wrow);
  const bool groups2 = a.shared_weights && a.group_split < a.M;
  const float bias_a = load(a.bias, wrow), bias_b = groups2 ? load(a.bias, a.bias_stride + wrow) : bias_a;
  const bool gate = a.epi == kEpiResidualGate;
  const float gate_a = gate ? load(a.gate, col) : 0.f, gate_b = gate && groups2 ? load(a.gate, a.gate_stride + col) : gate_a;
#pragma unroll 1
  for (int c = 0; c < NT && c < a.M; c += 16) {
    uint32_t r[16];
    tmem_ld16(tbase + c, r);
    float v[16];
    const float my_sx = c + (lane & 15) < a.M ? __ldg(a.x_scale + c + (lane & 15)) : 0.f;
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool second = groups2 && c + i >= a.group_split;
      v[i] = fmaf(static_cast<float>(static_cast<int>(r[i])) * sw, __shfl_sync(0xffffffffu, my_sx, i),
                  second ? bias_b : bias_a);
    }
    if (gated) {
      // Lanes 0..15 hold first factors, 16..31 second ones: exchanged, the lower half finishes even tokens, the
      // upper half odd ones.
      const bool upper = lane >= 16;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float got = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + 1], 16);
        const float first = upper ? got : v[i], second = upper ? v[i + 1] : got;
        const int m = c + i + (upper ? 1 : 0);
        const float f = a.epi == kEpiGeGlu ? first * i8_gelu_erf(splat(second)).x : i8_silu(splat(first)).x * second;
        if (live && m < a.M) few_store(a, m, col, f);
      }
      __syncwarp();
      continue;
    }
    switch (a.epi) {
      case kEpiGeluTanh:
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i8_gelu_tanh(splat(v[i])).x;
        break;
      case kEpiGeluErf:
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i8_gelu_erf(splat(v[i])).x;
        break;
      case kEpiSilu:
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i8_silu(splat(v[i])).x;
        break;
      case kEpiResidualGate:
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= groups2 && c + i >= a.group_split ? gate_b : gate_a;
        break;
      case kEpiAddStore:
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (live && c + i < a.M) v[i] += load_16bit(a.addend, (c + i) * a.ld_add + col, a.out_f16);
        break;
      default:
        break;
    }
    const int n = a.M - c;  // of these 16 tokens, the first n exist
    if (!live) {
      // This lane's column is past the output's.
    } else if (a.epi == kEpiResidualGate || a.epi == kEpiResidualAdd || a.epi == kEpiStoreF32) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < n) few_store(a, c + i, col, v[i]);
    } else {
      uint16_t* y = a.y + c * a.ld + col;
      if (a.out_f16) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < n) y[i * a.ld] = static_cast<uint16_t>(pack_f16(v[i], 0.f));
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < n) y[i * a.ld] = static_cast<uint16_t>(pack_bf16(v[i], 0.f));
      }
    }
    __syncwarp();  // the next columns are loaded by the whole warp
  }
}

template <int NT, int STAGES>
__global__ void __launch_bounds__(192, 1)
    gemm_i8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                       const I8GemmArgs a) {
  using L = I8FewSmem<NT, STAGES>;
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
  const int splits = static_cast<int>(cluster_nctas());
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / splits;
  const int all_kb = (a.K + 127) / 128;
  const int kb0 = all_kb * rank / splits;  // this CTA's k blocks: at least one, the host sees to it
  const int num_kb = all_kb * (rank + 1) / splits - kb0;
  const bool gated = a.half > 0;

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
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), L::kTmemCols);
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
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, a.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        const uint32_t w_dst = sbase + stage * L::kStageBytes;
        const int k0 = (kb0 + kb) * 128;
        mbar_arrive_expect_tx(full_bar(stage), L::kStageBytes);
        if (gated) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            tma_load_2d(w_dst + i * 32 * 128, &tmW, full_bar(stage), k0, tile * 64 + i * 16);
            tma_load_2d(w_dst + (i * 32 + 16) * 128, &tmW, full_bar(stage), k0, a.half + tile * 64 + i * 16);
          }
        } else {
          tma_load_2d(w_dst, &tmW, full_bar(stage), k0, tile * 128);
        }
        tma_load_2d(w_dst + L::kWBytes, &tmX, full_bar(stage), k0, 0);
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
        if (!mbar_wait(full_bar(stage), phase, abort_flag, a.status, kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w_addr = sbase + stage * L::kStageBytes;
        const uint32_t x_addr = w_addr + L::kWBytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ss_i8(tmem_base, make_sdesc_sw128(w_addr + k * 32, 16, 1024), make_sdesc_sw128(x_addr + k * 32, 16, 1024),
                     a.idesc, (kb | k) != 0 ? 1u : 0u);
        umma_commit(empty_bar(stage));
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) umma_commit(accf_bar);
      umma_commit(drain_bar);
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never, a.status, kStatusTimeoutDrain);
    }
  } else if (mbar_wait_warp(accf_bar, 0, abort_flag, a.status, kStatusTimeoutEpilogue)) {
    __syncwarp();
    tc_fence_after();
    const int ew = warp & 3;  // TMEM lanes 32 ew on: weight rows
    const uint32_t tbase = tmem_base + (static_cast<uint32_t>(ew * 32) << 16);
    if (splits == 1) {
      few_direct<NT>(a, tbase, tile, ew, lane);
    } else {
      const uint32_t dst = sbase + (ew * 32 + lane) * 4;
#pragma unroll 1
      for (int c = 0; c < NT && c < a.M; c += 16) {
        uint32_t r[16];
        tmem_ld16(tbase + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + (c + i) * 512), "r"(r[i]) : "memory");
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  if (splits == 1) {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, L::kTmemCols);
    return;
  }
  // Every CTA of the cluster gets here, timed out or not.
  cluster_sync_all();

  const int width = gated ? a.half : a.N;
  const int per_tile = gated ? 64 : 128;
  const int pairs = per_tile / 2;
  const int c0 = 2 * (static_cast<int>(threadIdx.x) % pairs);  // this thread's two outputs in the tile
  const int col = tile * per_tile + c0;
  if (col < width) {
    const bool two = col + 1 < width;
    auto vec2 = [&](const float* p) { return p ? make_float2(__ldg(p + col), two ? __ldg(p + col + 1) : 0.f) : splat(0.f); };
    auto moved = [](const float* p, long long by) { return p ? p + by : nullptr; };
    const float2 sw = vec2(a.w_scale);
    const float2 sw2 = gated ? vec2(a.w_scale + a.half) : splat(0.f);
    // The two row groups' bias and gate (or second factor's bias): one group unless weights are shared.
    const bool groups2 = a.shared_weights && a.group_split < a.M;
    const float* third = gated ? moved(a.bias, a.half) : a.epi == kEpiResidualGate ? a.gate : nullptr;
    const float2 bias_a = vec2(a.bias), third_a = vec2(third);
    const float2 bias_b = groups2 ? vec2(moved(a.bias, a.bias_stride)) : bias_a;
    const float2 third_b = groups2 ? vec2(moved(third, gated ? a.bias_stride : a.gate_stride)) : third_a;
    // This thread's tokens are `step` apart; kBatch of them are summed at once, so their loads overlap.
    constexpr int kBatch = 4;
    const int step = splits * (192 / pairs);
    const bool add = a.epi == kEpiResidualGate || a.epi == kEpiResidualAdd;
#pragma unroll 1
    for (int m0 = rank + splits * (static_cast<int>(threadIdx.x) / pairs); m0 < a.M; m0 += kBatch * step) {
      int2 s1[kBatch], s2[kBatch];
      float sx[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        s1[j] = s2[j] = make_int2(0, 0);
        sx[j] = m0 + j * step < a.M ? __ldg(a.x_scale + m0 + j * step) : 0.f;
      }
#pragma unroll 1
      for (int s = 0; s < splits; ++s) {
        // Weight row of output c0 in the tile, and 16 further its second factor's.
        const int w0 = gated ? (c0 / 16) * 32 + c0 % 16 : c0;
        const uint32_t src = mapa_shared(sbase + w0 * 4, static_cast<uint32_t>(s));
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int m = min(m0 + j * step, a.M - 1);
          const int2 p = ld_shared_cluster2(src + m * 512);
          s1[j].x += p.x;
          s1[j].y += p.y;
          if (gated) {
            const int2 q = ld_shared_cluster2(src + m * 512 + 16 * 4);
            s2[j].x += q.x;
            s2[j].y += q.y;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int m = m0 + j * step;
        if (m >= a.M) break;
        const bool second = groups2 && m >= a.group_split;
        auto scaled = [&](int2 s, float2 w, float2 b) {
          return ffma2(fmul2(make_float2(static_cast<float>(s.x), static_cast<float>(s.y)), w), splat(sx[j]), b);
        };
        const float2 third_m = second ? third_b : third_a;
        float2 v = scaled(s1[j], sw, second ? bias_b : bias_a);
        switch (a.epi) {
          case kEpiGeluTanh: v = i8_gelu_tanh(v); break;
          case kEpiGeluErf: v = i8_gelu_erf(v); break;
          case kEpiSilu: v = i8_silu(v); break;
          case kEpiSwiGlu: v = fmul2(i8_silu(v), scaled(s2[j], sw2, third_m)); break;
          case kEpiGeGlu: v = fmul2(v, i8_gelu_erf(scaled(s2[j], sw2, third_m))); break;
          case kEpiResidualGate: v = fmul2(v, third_m); break;
          case kEpiAddStore:
            v.x += load_16bit(a.addend, m * a.ld_add + col, a.out_f16);
            if (two) v.y += load_16bit(a.addend, m * a.ld_add + col + 1, a.out_f16);
            break;
          default: break;
        }
        const long long o = m * a.ld + col;
        if (add || a.epi == kEpiStoreF32) {
          float* p = a.residual + o;
          if (two) {
            float2* p2 = reinterpret_cast<float2*>(p);
            *p2 = add ? fadd2(*p2, v) : v;
          } else {
            *p = add ? *p + v.x : v.x;
          }
        } else if (two) {
          *reinterpret_cast<uint32_t*>(a.y + o) = a.out_f16 ? pack_f16(v.x, v.y) : pack_bf16(v.x, v.y);
        } else {
          a.y[o] = static_cast<uint16_t>(a.out_f16 ? pack_f16(v.x, 0.f) : pack_bf16(v.x, 0.f));
        }
      }
    }
  }
  __syncwarp();
  cluster_sync_all();  // no shared memory goes away while a peer reads it
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, L::kTmemCols);
}

}  // namespace nd
