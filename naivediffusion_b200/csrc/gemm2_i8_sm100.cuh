// Two-SM (cta_group::2) int8 x int8 GEMM: 256 x BN tiles, one per CTA pair,
// for products with enough rows and columns to give most pairs a tile. The
// pair's division of a tile, its barriers and its TMEM accumulators are those
// of the 16-bit pair kernel (gemm2_sm100.cuh): CTA r loads A rows
// [m0 + 128 r, +128) and its half of the W tile, the leader issues M = 256
// MMAs that read both CTAs' shared memory, each CTA's tensor memory holds its
// own 128 rows of two accumulators. Per SM and 128-deep k block 16 KB of A and
// BN / 2 x 128 B of W feed 128 x BN x 128 multiplications, half the operand
// bytes per multiplication of the one-SM kernel's 128 x 128 tiles.
//
// At twice the 16-bit rate a tile's MMAs last half as long per k, so the
// epilogue has eight warps per CTA (two per TMEM lane quarter, each half of
// the tile's columns) instead of four; sixteen warps of sixteen columns
// measured even (4096 x 640 x 5120 GEGLU 34-40 us both).
//
// 4352 x 4096 x 24576 SwiGLU: 266-278 us in bursts, 3.15-3.29 POP/s, the tensor
// pipe 95 % active (ncu), 318 us back to back at 1.28 GHz; 4352 x 12288 x 4096: 139
// us, 3.15 POP/s (3.68 rounds of pairs), and 168 at 1.35 GHz; its RESIDUAL
// epilogues 147 and 176, ADD_STORE, whose lanes read the addend two bytes at a
// time, 211 and 241.
// Below about K = 2048 the epilogue bounds it (4096 x 640 x 5120 GEGLU: 1.5
// POP/s, tensor pipe 37 %).
#pragma once

#include "gemm2_sm100.cuh"
#include "gemm_i8_sm100.cuh"

namespace nd {

__device__ __forceinline__ void umma_ss_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int BN, int STAGES>
struct I8PairSmem {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = (BN / 2) * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kTiles = STAGES * kStageBytes;
  static constexpr int kEpiOffset = kTiles;  // 8 warps x 4 KB
  static constexpr int kVecOffset = kEpiOffset + 8 * 4096;
  static constexpr int kBarOffset = kVecOffset + 8 * kI8VecWords * 4;
  static constexpr int kNumBars = 2 * STAGES + 5;  // full[S], empty[S], acc_full[2], acc_empty[2], drain
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotal = kMiscOffset + 16;
  static constexpr int kLaunchBytes = kTotal + 1024;
  static constexpr int kTmemCols = 2 * BN <= 256 ? 256 : 512;
};

constexpr int kI8PairThreads = 320;  // producer, MMA issuer, eight epilogue warps

template <int BN, int STAGES>
__global__ void __launch_bounds__(kI8PairThreads, 1)
    gemm2_i8_sm100_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmC, const I8GemmArgs args) {
  using L = I8PairSmem<BN, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bars = sbase + L::kBarOffset;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto accf_bar = [&](int s) { return bars + 8u * (2 * STAGES + s); };
  auto acce_bar = [&](int s) { return bars + 8u * (2 * STAGES + 2 + s); };
  const uint32_t drain_bar = bars + 8u * (2 * STAGES + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0: leader, 1: peer
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;
  const int num_m2 = (args.M + 255) / 256;
  const int num_n = (args.N + BN - 1) / BN;
  const int total = num_m2 * num_n;
  const int num_kb = (args.K + 127) / 128;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(accf_bar(s), 1);
      mbar_init(acce_bar(s), 16);  // eight epilogue warps in each CTA of the pair
    }
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
    tmem_alloc_pair(smem_u32(tmem_slot), L::kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch();
  griddep_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, issued_parity = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs) {
        int mt2, nt;
        pair_tile_coords(t, num_m2, num_n, mt2, nt);
        const int m0 = mt2 * 256 + static_cast<int>(rank) * 128;
        // The host keeps a pair inside one weight group.
        const int wrow = !args.shared_weights && mt2 * 256 >= args.group_split ? args.N : 0;
        // This CTA's W rows: its half of the tile, or (gated) the first
        // factor's rows in the leader and the second's in the peer.
        const int brow = wrow + (args.half > 0 ? (rank ? args.half : 0) + nt * (BN / 2)
                                               : nt * BN + static_cast<int>(rank) * (BN / 2));
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, args.status, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t a_dst = sbase + stage * L::kStageBytes;
          const uint32_t fbar = mapa_shared(full_bar(stage), 0);
          if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * L::kStageBytes);
          tma_load_2d_pair(a_dst, &tmA, fbar, kb * 128, m0);
          tma_load_2d_pair(a_dst + L::kABytes, &tmB, fbar, kb * 128, brow);
          issued |= 1u << stage;
          issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && rank == 0) {
        // Aborted: let the loads this pair started land before shared memory goes away.
        volatile int never = 0;
        for (int s = 0; s < STAGES; ++s)
          if (issued & (1u << s)) mbar_wait(full_bar(s), (issued_parity >> s) & 1u, &never, nullptr, 0);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (rank == 0 && elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(acce_bar(acc), ((local >> 1) & 1) ^ 1u, abort_flag, args.status, kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
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
            umma_ss_i8_pair(d_tmem, make_sdesc_sw128(a_addr + k * 32, 16, 1024),
                            make_sdesc_sw128(b_addr + k * 32, 16, 1024), args.idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit_pair(empty_bar(stage), 0x3);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(accf_bar(acc), 0x3);
      }
      umma_commit_pair(drain_bar, 0x1);
      volatile int never = 0;
      mbar_wait(drain_bar, 0, &never, args.status, kStatusTimeoutDrain);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int ew = warp & 3;          // TMEM lane quarter
    const int side = (warp - 2) >> 2; // half of the tile's columns
    const uint32_t buf = sbase + L::kEpiOffset + (warp - 2) * 4096;
    const uint32_t vecs = sbase + L::kVecOffset + (warp - 2) * kI8VecWords * 4;
    const uint32_t acce_leader0 = mapa_shared(acce_bar(0), 0);
    const uint32_t acce_leader1 = mapa_shared(acce_bar(1), 0);
    const int width = args.half > 0 ? args.half : args.N;
    const int per_tile = args.half > 0 ? BN / 2 : BN;
    int sb = 0;
    int local = 0;
    for (int t = pair; t < total; t += pairs, ++local) {
      const int acc = local & 1;
      int mt2, nt;
      pair_tile_coords(t, num_m2, num_n, mt2, nt);
      const int row0 = mt2 * 256 + static_cast<int>(rank) * 128 + ew * 32;
      const int wgroup = !args.shared_weights && mt2 * 256 >= args.group_split ? 1 : 0;
      const I8Rows rows = i8_rows(args, wgroup, row0);
      const int col0 = nt * per_tile + side * (per_tile / 2);
      const float sx = row0 + lane < args.M ? __ldg(args.x_scale + row0 + lane) : 0.f;
      if (row0 < args.M) i8_stage_vectors(args, vecs, wgroup, rows, col0, lane);
      if (!mbar_wait_warp(accf_bar(acc), (local >> 1) & 1, abort_flag, args.status, kStatusTimeoutEpilogue)) break;
      __syncwarp();
      tc_fence_after();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + acc * BN;
      if (row0 < args.M) {
        const uint32_t at = tbase + side * (per_tile / 2);
        const int chunks = min(per_tile / 64, (width - col0 + 31) / 32);  // may be <= 0
        if (args.half > 0) {
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            uint32_t r[32], r2[32];
            tmem_ld32(at + c * 32, r);
            tmem_ld32(at + BN / 2 + c * 32, r2);
            tmem_ld_wait();
            i8_chunk(args, &tmC, rows, row0, col0 + c * 32, c * 32, sx, r, r2, vecs, buf, sb, lane);
          }
        } else if (chunks > 0) {
          // The next chunk's sums are on their way while this one is worked on.
          uint32_t r[32], next[32];
          tmem_ld32(at, r);
          tmem_ld_wait();
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            if (c + 1 < chunks) tmem_ld32(at + (c + 1) * 32, next);
            i8_chunk(args, &tmC, rows, row0, col0 + c * 32, c * 32, sx, r, r, vecs, buf, sb, lane);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = next[i];
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc ? acce_leader1 : acce_leader0);
    }
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
  }

  // Every MMA into this pair's TMEM has retired (the leader waited on its
  // drain barrier) and every read of it is done before it is freed.
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, L::kTmemCols);
}

}  // namespace nd
