// Host side of the int8 x int8 GEMM: argument checks, tensor maps, choice of
// kernel and launch. The kernels are in gemm_i8_sm100.cuh.
#include <algorithm>
#include <climits>

#include "gemm2_i8_sm100.cuh"
#include "gemm_i8_sm100.cuh"
#include "nd_internal.h"
#include "nd_runtime.h"

namespace nd {

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int BN, int STAGES>
int launch_i8(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const I8GemmArgs& g,
              cudaStream_t stream) {
  using L = I8Smem<BN, STAGES>;
  auto kernel = gemm_i8_sm100_kernel<BN, STAGES>;
  static bool configured[64] = {};
  int dev = 0;
  ND_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kLaunchBytes));
    configured[dev & 63] = true;
  }
  const int tiles = ((g.M + 127) / 128) * ((g.N + BN - 1) / BN);
  ND_CUDA(launch_pdl(kernel, dim3(tiles), dim3(192), L::kLaunchBytes, stream, ta, tb, tc, g));
  ND_CUDA(cudaGetLastError());
  return ND_OK;
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
  g.status = device_status();
  if (!g.status) return fail(ND_ERR_CUDA, "linear_w8a8: no device status word");

  CUtensorMap ta, tb, tc;
  int rc = make_tmap_2d(&ta, a.x, 1, a.rows, a.in_features, a.ldx, 128, 128, true);
  if (rc) return rc;
  if (resid) rc = make_tmap_2d_typed(&tc, a.residual, ND_F32, a.rows, a.out_features, a.ldr, 32, 32, 128);
  else rc = make_tmap_2d_typed(&tc, a.y, a.dtype, a.rows, a.out_features, a.ldy, 32, 32, 64);
  if (rc) return rc;
  const int64_t pair_tiles = ((a.rows + 255) / 256) * ((n_all + 255) / 256);
  const bool pair_groups = !split || shared || a.group_split % 256 == 0;
  if (a.rows >= 512 && pair_groups && 2 * pair_tiles >= sm_count() / 2) {
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
