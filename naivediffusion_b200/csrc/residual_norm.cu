// The norms around a block's branch, with its gate and residual in one pass:
//
//   x' = residual_scale * x + gate[v] * post(branch)
//   y  = pre(x') * (1 + scale[v]) + shift[v]
//
// post / pre: nothing, RMSNorm or LayerNorm (each with an optional weight),
// v = min(row / rows_per_vec, vecs - 1): the row's vectors (one set per batch
// item, or image and text rows). y is fp32, bf16, fp16 or int8 with one scale
// per row. The parts are Transformer.Modulate and the gated residual
// (src/NaiveDiffusion/Graph/Transformer.cs:72-80) and Layers.RmsNorm
// (src/NaiveDiffusion/Graph/Layers.cs:209-221), which the reference runs as
// separate graph nodes.
//
// Bound by HBM: every element of x and branch is read once, x' and y are
// written once; the row stays in registers between its (up to five) row-wide
// reductions. Variances are centred second moments over the registers, in
// fp32. The vectors are read from L1 / L2.
#include <algorithm>
#include <climits>

#include "nd_common.cuh"
#include "nd_internal.h"
#include "nd_runtime.h"
#include "row_quant.cuh"

namespace nd {

namespace {

struct ResidualNorm {
  const float* x;
  float* x_out;
  const void* branch;
  void* y;
  float* y_scale;
  const float* post_weight;
  const float* pre_weight;
  const float* gate;
  const float* scale;
  const float* shift;
  long long ldx, ldxo, ldb, ldy, vec_stride, rows_per_vec;
  int rows, width, vecs;
  int branch_type, out_type, post, pre;
  float residual_scale, plus_one, eps;
};

template <int VEC>
struct Vals {
  float f[VEC];
};

// VEC consecutive fp32 values that are read once (they stay out of L1).
template <int VEC>
__device__ __forceinline__ Vals<VEC> load_once(const float* p) {
  Vals<VEC> r;
  if constexpr (VEC == 4) {
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(r.f[0]), "=f"(r.f[1]), "=f"(r.f[2]), "=f"(r.f[3])
                 : "l"(p));
  } else {
    r.f[0] = *p;
  }
  return r;
}

template <int VEC>
__device__ __forceinline__ Vals<VEC> load_branch(const void* p, long long i, int type) {
  if (type == ND_F32) return load_once<VEC>(static_cast<const float*>(p) + i);
  Vals<VEC> r;
  if constexpr (VEC == 4) {
    uint32_t a, b;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
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
    r.f[0] = lo.x; r.f[1] = lo.y; r.f[2] = hi.x; r.f[3] = hi.y;
  } else {
    r.f[0] = type == ND_F16 ? __half2float(static_cast<const __half*>(p)[i])
                            : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
  return r;
}

template <int VEC>
__device__ __forceinline__ Vals<VEC> load_vec(const float* p) {
  Vals<VEC> r;
  if constexpr (VEC == 4) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(p));
    r.f[0] = t.x; r.f[1] = t.y; r.f[2] = t.z; r.f[3] = t.w;
  } else {
    r.f[0] = __ldg(p);
  }
  return r;
}

// VEC values as out_type (ND_F32, ND_F16 or ND_BF16) at element i.
template <int VEC>
__device__ __forceinline__ void store_vals(void* p, long long i, const Vals<VEC>& v, int type) {
  if constexpr (VEC == 4) {
    if (type == ND_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v.f[0], v.f[1], v.f[2], v.f[3]);
    } else {
      const uint2 w = type == ND_F16 ? make_uint2(pack_f16(v.f[0], v.f[1]), pack_f16(v.f[2], v.f[3]))
                                     : make_uint2(pack_bf16(v.f[0], v.f[1]), pack_bf16(v.f[2], v.f[3]));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = w;
    }
  } else {
    if (type == ND_F32) static_cast<float*>(p)[i] = v.f[0];
    else if (type == ND_F16) static_cast<__half*>(p)[i] = __float2half_rn(v.f[0]);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v.f[0]);
  }
}

// Sum / maximum over the T threads of a row, in a fixed order. `slot`: this
// reduction's own T / 32 words of shared memory, so one barrier is enough.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) v += slot[i];
  }
  return v;
}
template <int T>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* slot) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0u;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) v = max(v, slot[i]);
  }
  return v;
}

// T threads per row, V x VEC values per thread (width <= T * V * VEC). Blocks
// of max(T, 128) threads: four rows each where a warp holds a row.
template <int VEC, int V, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T) residual_norm_kernel(const ResidualNorm a) {
  griddep_launch();
  griddep_wait();
  __shared__ float red[5][T / 32];
  constexpr int kRows = T < 128 ? 128 / T : 1;
  const int t = threadIdx.x % T;
  const int row = blockIdx.x * kRows + threadIdx.x / T;
  if (row >= a.rows) return;  // whole warps: only T = 32 has several rows per block
  const long long r = row;
  const long long vec = min(r / a.rows_per_vec, static_cast<long long>(a.vecs - 1)) * a.vec_stride;
  const float count = static_cast<float>(a.width);
  auto col = [&](int i) { return (t + T * i) * VEC; };

  Vals<VEC> v[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col(i);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i].f[j] = b[i].f[j] = 0.f;
    if (c < a.width) {
      v[i] = load_once<VEC>(a.x + r * a.ldx + c);
      if (a.branch) b[i] = load_branch<VEC>(a.branch, r * a.ldb + c, a.branch_type);
    }
  }
  // Subtract the mean (LayerNorm), then return rsqrt(mean square + eps).
  auto normalize = [&](Vals<VEC> (&w)[V], int kind, int slot) {
    if (kind == ND_NORM_LAYER) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col(i) < a.width)
#pragma unroll
          for (int j = 0; j < VEC; ++j) s += w[i].f[j];
      const float mean = row_sum<T>(s, red[slot]) / count;
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[i].f[j] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (col(i) < a.width)
#pragma unroll
        for (int j = 0; j < VEC; ++j) q = fmaf(w[i].f[j], w[i].f[j], q);
    return rsqrtf(row_sum<T>(q, red[slot + 1]) / count + a.eps);
  };

  if (a.branch) {
    const float rstd = a.post != ND_NORM_NONE ? normalize(b, a.post, 0) : 1.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = col(i);
      if (c < a.width) {
        Vals<VEC> k;
#pragma unroll
        for (int j = 0; j < VEC; ++j) k.f[j] = rstd;
        if (a.post_weight) {
          const Vals<VEC> w = load_vec<VEC>(a.post_weight + c);
#pragma unroll
          for (int j = 0; j < VEC; ++j) k.f[j] *= w.f[j] + a.plus_one;
        }
        if (a.gate) {
          const Vals<VEC> g = load_vec<VEC>(a.gate + vec + c);
#pragma unroll
          for (int j = 0; j < VEC; ++j) k.f[j] *= g.f[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i].f[j] = fmaf(b[i].f[j], k.f[j], a.residual_scale * v[i].f[j]);
      }
    }
  } else if (a.residual_scale != 1.f) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i].f[j] *= a.residual_scale;
  }
  if (a.x_out) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = col(i);
      if (c < a.width) store_vals<VEC>(a.x_out, r * a.ldxo + c, v[i], ND_F32);
    }
  }
  if (!a.y) return;

  const float rstd = a.pre != ND_NORM_NONE ? normalize(v, a.pre, 2) : 1.f;
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col(i);
    if (c < a.width) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i].f[j] *= rstd;
      if (a.pre_weight) {
        const Vals<VEC> w = load_vec<VEC>(a.pre_weight + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i].f[j] *= w.f[j] + a.plus_one;
      }
      if (a.scale) {
        const Vals<VEC> s = load_vec<VEC>(a.scale + vec + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i].f[j] = fmaf(v[i].f[j], s.f[j], v[i].f[j]);
      }
      if (a.shift) {
        const Vals<VEC> s = load_vec<VEC>(a.shift + vec + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i].f[j] += s.f[j];
      }
      if (a.out_type != ND_I8) store_vals<VEC>(a.y, r * a.ldy + c, v[i], a.out_type);
#pragma unroll
      for (int j = 0; j < VEC; ++j) peak = max(peak, abs_bits(v[i].f[j]));
    }
  }
  if (a.out_type != ND_I8) return;
  // y is an fp32 result already, so the quotient's last bit decides nothing
  // that fp32 had not rounded before: multiply by 127 / peak.
  const RowScale s = row_scale(row_max<T>(peak, reinterpret_cast<uint32_t*>(red[4])));
  if (t == 0) a.y_scale[r] = s.scale;
  int8_t* y = static_cast<int8_t*>(a.y) + r * a.ldy;
  const bool tiny = s.peak < 1e-30f;  // 127 / peak leaves fp32's range: divide instead
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col(i);
    if (c < a.width) {
      float q[4] = {0.f, 0.f, 0.f, 0.f};
      if (s.inverse != 0.f) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          q[j] = tiny ? static_cast<float>(v[i].f[j] * 127.0 / s.peak) : v[i].f[j] * s.inverse;
      }
      const uint32_t p = pack_rint(q[0], q[1], q[2], q[3]);
      if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(y + c) = p;
      else y[c] = static_cast<int8_t>(p & 0xffu);
    }
  }
}

template <int VEC, int V, int T>
int launch(const ResidualNorm& a, cudaStream_t stream) {
  constexpr int kRows = T < 128 ? 128 / T : 1;
  const unsigned grid = static_cast<unsigned>((static_cast<long long>(a.rows) + kRows - 1) / kRows);
  ND_CUDA(launch_pdl(residual_norm_kernel<VEC, V, T>, dim3(grid), dim3(T < 128 ? 128 : T), 0, stream, a));
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

bool aligned(const void* p, int64_t ld, int elem) {  // rows of 4 elements at once
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) % (4 * elem)) == 0 && ld % 4 == 0);
}

int elem_bytes(int dtype) { return dtype == ND_F32 ? 4 : dtype == ND_I8 ? 1 : 2; }

}  // namespace

int residual_norm(const nd_residual_norm_args& a, cudaStream_t stream) {
  if (a.rows <= 0 || a.width <= 0) return fail(ND_ERR_INVALID, "residual_norm: empty shape");
  if (a.rows > INT_MAX) return fail(ND_ERR_INVALID, "residual_norm: too many rows");
  if (a.width > 16384) return fail(ND_ERR_UNSUPPORTED, "residual_norm: width above 16384");
  if (!a.x) return fail(ND_ERR_INVALID, "residual_norm: null x");
  if (!a.x_out && !a.y) return fail(ND_ERR_INVALID, "residual_norm: neither x_out nor y given");
  if (a.ldx < a.width || (a.x_out && a.ldxo < a.width) || (a.branch && a.ldb < a.width) || (a.y && a.ldy < a.width))
    return fail(ND_ERR_INVALID, "residual_norm: a row stride is smaller than the width");
  if (a.x_out == a.x && a.x_out && a.ldxo != a.ldx)
    return fail(ND_ERR_INVALID, "residual_norm: in place, x_out needs x's row stride");
  auto known = [](int kind) { return kind == ND_NORM_NONE || kind == ND_NORM_RMS || kind == ND_NORM_LAYER; };
  if (!known(a.post_norm) || !known(a.pre_norm)) return fail(ND_ERR_INVALID, "residual_norm: unknown norm");
  if (a.branch && a.branch_dtype != ND_F32 && a.branch_dtype != ND_F16 && a.branch_dtype != ND_BF16)
    return fail(ND_ERR_INVALID, "residual_norm: branch_dtype must be f32, f16 or bf16");
  if (!a.branch && (a.gate || a.post_weight || a.post_norm != ND_NORM_NONE))
    return fail(ND_ERR_INVALID, "residual_norm: a gate or post norm needs a branch");
  if (a.post_weight && a.post_norm == ND_NORM_NONE)
    return fail(ND_ERR_INVALID, "residual_norm: post_weight without a post norm");
  if (!a.y && (a.pre_norm != ND_NORM_NONE || a.pre_weight || a.scale || a.shift))
    return fail(ND_ERR_INVALID, "residual_norm: pre norm, scale or shift without y");
  if (a.pre_weight && a.pre_norm == ND_NORM_NONE)
    return fail(ND_ERR_INVALID, "residual_norm: pre_weight without a pre norm");
  if (a.y && a.out_dtype != ND_F32 && a.out_dtype != ND_F16 && a.out_dtype != ND_BF16 && a.out_dtype != ND_I8)
    return fail(ND_ERR_INVALID, "residual_norm: out_dtype must be f32, f16, bf16 or i8");
  if (a.y && a.out_dtype == ND_I8 && !a.y_scale) return fail(ND_ERR_INVALID, "residual_norm: an int8 y needs y_scale");
  if (a.vecs < 1 || a.vecs > INT_MAX) return fail(ND_ERR_INVALID, "residual_norm: vecs must be positive");
  if (a.vecs > 1 && a.rows_per_vec <= 0)
    return fail(ND_ERR_INVALID, "residual_norm: several vectors need rows_per_vec > 0");
  if (a.vecs > 1 && (a.gate || a.scale || a.shift) && a.vec_stride < a.width)
    return fail(ND_ERR_INVALID, "residual_norm: vec_stride is smaller than the width");

  ResidualNorm k{};
  k.x = a.x; k.ldx = a.ldx;
  k.x_out = a.x_out; k.ldxo = a.ldxo;
  k.branch = a.branch; k.ldb = a.ldb; k.branch_type = a.branch_dtype;
  k.y = a.y; k.ldy = a.ldy; k.out_type = a.out_dtype; k.y_scale = a.y_scale;
  k.post = a.post_norm; k.post_weight = a.post_weight;
  k.pre = a.pre_norm; k.pre_weight = a.pre_weight;
  k.gate = a.gate; k.scale = a.scale; k.shift = a.shift;
  k.vecs = static_cast<int>(a.vecs);
  k.vec_stride = a.vecs > 1 ? a.vec_stride : 0;
  k.rows_per_vec = a.vecs > 1 ? a.rows_per_vec : INT_MAX;
  k.rows = static_cast<int>(a.rows);
  k.width = static_cast<int>(a.width);
  k.residual_scale = a.residual_scale;
  k.plus_one = a.plus_one ? 1.f : 0.f;
  k.eps = a.eps;

  const int64_t vs = k.vec_stride;
  const bool by4 = a.width % 4 == 0 && aligned(a.x, a.ldx, 4) && aligned(a.x_out, a.ldxo, 4) &&
                   aligned(a.branch, a.ldb, elem_bytes(a.branch_dtype)) && aligned(a.y, a.ldy, elem_bytes(a.out_dtype)) &&
                   aligned(a.gate, vs, 4) && aligned(a.scale, vs, 4) && aligned(a.shift, vs, 4) &&
                   aligned(a.post_weight, 0, 4) && aligned(a.pre_weight, 0, 4);
  if (!by4) {
    if (a.width <= 1024) return launch<1, 4, 256>(k, stream);
    if (a.width <= 4096) return launch<1, 16, 256>(k, stream);
    return launch<1, 16, 1024>(k, stream);
  }
  const int64_t w4 = a.width / 4;
  if (w4 <= 128) return launch<4, 4, 32>(k, stream);
  if (w4 <= 256) return launch<4, 2, 128>(k, stream);
  if (w4 <= 512) return launch<4, 4, 128>(k, stream);
  if (w4 <= 1024) return launch<4, 4, 256>(k, stream);
  if (w4 <= 2048) return launch<4, 4, 512>(k, stream);
  return launch<4, 4, 1024>(k, stream);
}

}  // namespace nd
