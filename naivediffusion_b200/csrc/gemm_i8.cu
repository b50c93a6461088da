// Host side of the int8 x int8 GEMM: argument checks, tensor maps, choice of
// kernel and launch. The kernels are in gemm_i8_sm100.cuh.
#include <algorithm>
#include <climits>

#include "gemm2_i8_sm100.cuh"
#include "gemm_i8_few_sm100.cuh"
#include "gemm_i8_sm100.cuh"
#include "gemv_i8.cuh"
#include "nd_internal.h"
#include "nd_runtime.h"

namespace nd {

namespace {

constexpr int kMaxSplits = 8;  // the portable cluster size
// Rows of gemm_i8_few_kernel. Against the 128 x 128 tiles, us: 16 x 4096 x 12288
// 12.4 / 19.8, 32 x 4096 x 4096 7.4 / 8.4, 48 x 4096 x 12288 14.5 / 14.5,
// 64 x 4096 x 12288 15.3 / 14.4.
constexpr int kFewRows = 32;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch a kernel whose clusters of S CTAs share a tile's k blocks. The rule
// counts block_us for a k block on one SM, and fixed_us + S * each_us for a
// split: the cluster barriers and the sums' way through the cluster's shared
// memory: estimates, one set per kernel. S is the cheapest count whose clusters
// all run at once (`most`, looked up once per kernel and device).
//
// What a k block takes without a split, from the times' slope over K: the
// 128 x 128 kernel's 32 KB 0.19-0.23 us with 144 tiles at once (140-170 GB/s per
// SM); the few-rows kernel's 18 KB 0.155 us with 96 tiles and the weights in L2
// (119 GB/s per SM), 0.23-0.28 us once they come from HBM.
struct SplitCost {
  float block_us, fixed_us, each_us;
};
template <typename Kernel, typename... Args>
int launch_split(Kernel kernel, int* most, int smem, int tiles, int num_kb, SplitCost c, cudaStream_t stream,
                 const Args&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (!most[1]) {
    ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cfg.numAttrs = 1;
    for (int s = kMaxSplits; s >= 1; --s) {
      attr[0].val.clusterDim.x = s;
      cfg.gridDim = dim3(s * sm_count());
      int n = 0;
      ND_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
      most[s] = std::max(n, 1);
    }
  }
  int splits = 1;
  float best = c.block_us * num_kb;
  for (int s = 2; s <= std::min(kMaxSplits, num_kb); ++s) {
    const float cost = c.block_us * ((num_kb + s - 1) / s) + c.fixed_us + c.each_us * s;
    if (tiles <= most[s] && cost < best) {
      best = cost;
      splits = s;
    }
  }
  attr[0].val.clusterDim.x = splits;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * splits);
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  ND_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

int current_device(int* dev) {
  ND_CUDA(cudaGetDevice(dev));
  return ND_OK;
}

// The one-SM kernel: 128 x BN tiles.
template <int BN, int STAGES>
int launch_i8(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const I8GemmArgs& g,
              cudaStream_t stream) {
  using L = I8Smem<BN, STAGES>;
  static int most[64][kMaxSplits + 1] = {};
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const int tiles = ((g.M + 127) / 128) * ((g.N + BN - 1) / BN);
  const float quarters = static_cast<float>(std::min(4, (g.M + 31) / 32));  // of a tile's rows that exist: what is summed
  return launch_split(gemm_i8_sm100_kernel<BN, STAGES>, most[dev & 63], L::kLaunchBytes, tiles, (g.K + 127) / 128,
                      SplitCost{0.165f, 0.1f * quarters, 0.3f * quarters}, stream, ta, tb, tc, g);
}

// The kernel for few rows: 128 weight rows x NT tokens.
template <int NT, int STAGES>
int launch_i8_few(const CUtensorMap& tw, const CUtensorMap& tx, const I8GemmArgs& g, cudaStream_t stream) {
  using L = I8FewSmem<NT, STAGES>;
  static int most[64][kMaxSplits + 1] = {};
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const int tiles = g.half > 0 ? g.half / 64 : (g.N + 127) / 128;
  return launch_split(gemm_i8_few_kernel<NT, STAGES>, most[dev & 63], L::kLaunchBytes, tiles, (g.K + 127) / 128,
                      SplitCost{0.17f, 0.f, 0.25f}, stream, tw, tx, g);
}

// The pair kernel: clusters of two CTAs, as many pairs as fit on the GPU at
// once (looked up once per device), each looping over 256-row tiles.
template <int BN, int STAGES>
int launch_i8_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const I8GemmArgs& g,
                   cudaStream_t stream) {
  using L = I8PairSmem<BN, STAGES>;
  auto kernel = gemm2_i8_sm100_kernel<BN, STAGES>;
  static int max_pairs[64] = {};
  int dev = 0;
  ND_CUDA(cudaGetDevice(&dev));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kI8PairThreads);
  cfg.dynamicSmemBytes = L::kLaunchBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (!max_pairs[dev & 63]) {
    ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kLaunchBytes));
    cfg.gridDim = dim3(2 * sm_count());
    cfg.numAttrs = 1;
    int n = 0;
    ND_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    if (n <= 0) return fail(ND_ERR_UNSUPPORTED, "linear_w8a8: no CTA pair fits on this GPU");
    max_pairs[dev & 63] = n;
  }
  const int tiles = ((g.M + 255) / 256) * ((g.N + BN - 1) / BN);
  cfg.gridDim = dim3(2 * std::min(tiles, max_pairs[dev & 63]));
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  ND_CUDA(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tc, g));
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

// Pair or one-SM kernel. Either loads 32 KB per k block and SM, the pair kernel
// for a 128 x 256 share of its tile (0.32-0.35 us with one round of pairs), the
// one-SM kernel for 128 x 128 (0.19-0.23 us; missing rows cost nothing); the rule
// compares the rounds that both need, and its crossings were measured. Pair /
// one-SM, us: 256 x 4096 x 12288 18.3 / 23.8,
// 512 x 4096 x 4096 16.1 / 12.2, 1024 x 4096 x 4096 17.2 / 22.7,
// 1024 x 640 x 2048 7.9 / 6.4.
bool pair_is_faster(int64_t rows, int64_t n) {
  const int sms = sm_count();
  const int64_t pair_tiles = ((rows + 255) / 256) * ((n + 255) / 256), tiles = ((rows + 127) / 128) * ((n + 127) / 128);
  const int64_t pair_rounds = (pair_tiles + sms / 2 - 1) / (sms / 2), rounds = (tiles + sms - 1) / sms;
  const float real = rows < 128 ? rows / 128.f : 1.f;
  return pair_rounds < rounds * (0.5f + 0.5f * real);
}

int launch_i8_gemv(const nd_linear_w8a8_args& a, const I8GemmArgs& g, int64_t ldw, cudaStream_t stream) {
  I8GemvArgs v{};
  v.g = g;
  v.x = a.x;
  v.w = a.weight;
  v.ldx = a.ldx;
  v.ldw = ldw;
  const int warps = g.half > 0 ? g.half : (g.N + 1) / 2;
  const dim3 grid((warps + kGemvI8Threads / 32 - 1) / (kGemvI8Threads / 32));
  switch (g.M) {
    case 1: ND_CUDA(launch_pdl(gemv_i8_kernel<1>, grid, dim3(kGemvI8Threads), 0, stream, v)); break;
    case 2: ND_CUDA(launch_pdl(gemv_i8_kernel<2>, grid, dim3(kGemvI8Threads), 0, stream, v)); break;
    case 3: ND_CUDA(launch_pdl(gemv_i8_kernel<3>, grid, dim3(kGemvI8Threads), 0, stream, v)); break;
    default: ND_CUDA(launch_pdl(gemv_i8_kernel<4>, grid, dim3(kGemvI8Threads), 0, stream, v)); break;
  }
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

}  // namespace

int linear_w8a8(const nd_linear_w8a8_args& a, cudaStream_t stream) {
  if (a.dtype != ND_BF16 && a.dtype != ND_F16) return fail(ND_ERR_INVALID, "linear_w8a8: dtype must be bf16 or f16");
  if (a.rows <= 0 || a.in_features <= 0 || a.out_features <= 0)
    return fail(ND_ERR_INVALID, "linear_w8a8: empty shape");
  if (a.rows > INT_MAX / 2 || a.out_features > INT_MAX / 8) return fail(ND_ERR_INVALID, "linear_w8a8: shape too large");
  if (a.in_features >= 131072)  // 128 * 128 * 131072 = 2^31
    return fail(ND_ERR_INVALID, "linear_w8a8: in_features above 131071 could overflow the 32-bit sums");
  if (!a.x || !a.weight || !a.x_scale || !a.w_scale) return fail(ND_ERR_INVALID, "linear_w8a8: null operand");
  const int64_t ldw = a.ldw > 0 ? a.ldw : a.in_features;
  if (a.ldx < a.in_features || a.ldx % 16 || !aligned16(a.x))
    return fail(ND_ERR_INVALID, "linear_w8a8: x must be 16-byte aligned with ldx >= in_features, ldx % 16 == 0");
  if (ldw < a.in_features || ldw % 16 || !aligned16(a.weight))
    return fail(ND_ERR_INVALID, "linear_w8a8: weight must be 16-byte aligned with ldw >= in_features, ldw % 16 == 0");
  const bool split = a.group_split < a.rows;
  const bool shared = a.shared_weights != 0;
  if (split && a.group_split <= 0) return fail(ND_ERR_INVALID, "linear_w8a8: group_split must be positive");
  if (split && !shared && a.group_split % 128 != 0)
    return fail(ND_ERR_INVALID, "linear_w8a8: group_split must be a multiple of 128 (or give shared_weights)");
  const int epi = a.epilogue;
  if (epi < 0 || epi > ND_EPI_GEGLU || epi == ND_EPI_QK_NORM_ROPE)
    return fail(ND_ERR_INVALID, "linear_w8a8: unknown epilogue (QK_NORM_ROPE is not offered)");
  const bool gated = epi == ND_EPI_SWIGLU || epi == ND_EPI_GEGLU;
  if (gated && a.out_features % 128)
    return fail(ND_ERR_INVALID, "linear_w8a8: SWIGLU / GEGLU need out_features % 128 == 0");
  const bool resid = epi == ND_EPI_RESIDUAL_GATE || epi == ND_EPI_RESIDUAL_ADD || epi == ND_EPI_STORE_F32;
  if (resid && (!a.residual || a.ldr < a.out_features || a.ldr % 4 || !aligned16(a.residual)))
    return fail(ND_ERR_INVALID,
                "linear_w8a8: this epilogue needs a 16-byte aligned residual with ldr >= out_features, ldr % 4 == 0");
  if (!resid && (!a.y || a.ldy < a.out_features || a.ldy % 8 || !aligned16(a.y)))
    return fail(ND_ERR_INVALID, "linear_w8a8: y must be 16-byte aligned with ldy >= out_features, ldy % 8 == 0");
  if (epi == ND_EPI_RESIDUAL_GATE && !a.gate) return fail(ND_ERR_INVALID, "linear_w8a8: gate missing");
  if (a.gate && a.gate_stride != 0 && a.gate_stride < a.out_features)
    return fail(ND_ERR_INVALID, "linear_w8a8: gate_stride is smaller than out_features");
  if (epi == ND_EPI_ADD_STORE && (!a.addend || a.ld_add < a.out_features))
    return fail(ND_ERR_INVALID, "linear_w8a8: ADD_STORE needs addend with ld_add >= out_features");

  const int64_t n_all = gated ? 2 * a.out_features : a.out_features;
  const int groups = split && !shared ? 2 : 1;
  I8GemmArgs g{};
  g.M = static_cast<int>(a.rows);
  g.N = static_cast<int>(n_all);
  g.K = static_cast<int>(a.in_features);
  g.group_split = split ? static_cast<int>(a.group_split) : INT_MAX;
  g.shared_weights = shared ? 1 : 0;
  g.epi = epi;
  g.out_f16 = a.dtype == ND_F16;
  g.half = gated ? static_cast<int>(a.out_features) : 0;
  g.x_scale = a.x_scale;
  g.w_scale = a.w_scale;
  g.bias = a.bias;
  g.bias_stride = static_cast<int>(n_all);
  g.gate = a.gate;
  g.gate_stride = a.gate_stride > 0 ? a.gate_stride : a.out_features;
  g.addend = a.addend;
  g.ld_add = a.ld_add;
  g.y = static_cast<uint16_t*>(a.y);
  g.residual = a.residual;
  g.ld = resid ? a.ldr : a.ldy;
  g.status = device_status();
  if (!g.status) return fail(ND_ERR_CUDA, "linear_w8a8: no device status word");

  if (a.rows <= kGemvI8Rows) return launch_i8_gemv(a, g, ldw, stream);

  CUtensorMap ta, tb, tc;
  // More tiles of 128 weight rows than SMs: half the stages, so that two CTAs
  // share an SM and one's loads run under the other's start and end
  // (16 x 4096 x 24576 SwiGLU 26.5 -> 20.1 us). That also takes 33 to 64 rows
  // (48 x 1280 x 24576 10.2 us against 15.6 in 128 x 128 tiles).
  const bool two = (gated ? a.out_features / 64 : (n_all + 127) / 128) > sm_count();
  if (a.rows <= kFewRows || (two && a.rows <= 2 * kFewRows)) {
    const int nt = a.rows <= 16 ? 16 : a.rows <= 32 ? 32 : 64;
    int rc = make_tmap_2d(&ta, a.weight, 1, n_all, a.in_features, ldw, gated ? 16 : 128, 128, true);
    if (rc) return rc;
    rc = make_tmap_2d(&tb, a.x, 1, a.rows, a.in_features, a.ldx, nt, 128, true);
    if (rc) return rc;
    g.idesc = make_idesc_i8(128, nt);
    if (nt == 16) return two ? launch_i8_few<16, 6>(ta, tb, g, stream) : launch_i8_few<16, 12>(ta, tb, g, stream);
    if (nt == 32) return two ? launch_i8_few<32, 5>(ta, tb, g, stream) : launch_i8_few<32, 11>(ta, tb, g, stream);
    return launch_i8_few<64, 4>(ta, tb, g, stream);
  }
  int rc = make_tmap_2d(&ta, a.x, 1, a.rows, a.in_features, a.ldx, 128, 128, true);
  if (rc) return rc;
  if (resid) rc = make_tmap_2d_typed(&tc, a.residual, ND_F32, a.rows, a.out_features, a.ldr, 32, 32, 128);
  else rc = make_tmap_2d_typed(&tc, a.y, a.dtype, a.rows, a.out_features, a.ldy, 32, 32, 64);
  if (rc) return rc;
  const bool pair_groups = !split || shared || a.group_split % 256 == 0;
  if (pair_groups && pair_is_faster(a.rows, n_all)) {
    g.idesc = make_idesc_i8(256, 256);
    rc = make_tmap_2d(&tb, a.weight, 1, groups * n_all, a.in_features, ldw, 128, 128, true);
    if (rc) return rc;
    return launch_i8_pair<256, 5>(ta, tb, tc, g, stream);
  }
  constexpr int bn = 128;
  g.idesc = make_idesc_i8(128, bn);
  rc = make_tmap_2d(&tb, a.weight, 1, groups * n_all, a.in_features, ldw, gated ? bn / 2 : bn, 128, true);
  if (rc) return rc;
  return launch_i8<bn, 6>(ta, tb, tc, g, stream);
}

}  // namespace nd
