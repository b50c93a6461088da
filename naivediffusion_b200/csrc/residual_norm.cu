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
// fp32.
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
  long long ldx, ldxo, ldb, ldy, vec_stride;
  int rows, width, vecs, rows_per_vec;
  int branch_type, out_type, post, pre;
  float residual_scale, plus_one, eps, inv_width;
};

template <int VEC>
struct Vals {
  float f[VEC];
};

// Element by element; four at a time as two paired operations.
template <int VEC>
__device__ __forceinline__ Vals<VEC> mul(const Vals<VEC>& a, const Vals<VEC>& b) {
  Vals<VEC> r;
  if constexpr (VEC == 4) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float2 t = fmul2(make_float2(a.f[j], a.f[j + 1]), make_float2(b.f[j], b.f[j + 1]));
      r.f[j] = t.x;
      r.f[j + 1] = t.y;
    }
  } else {
    r.f[0] = a.f[0] * b.f[0];
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ Vals<VEC> fma(const Vals<VEC>& a, const Vals<VEC>& b, const Vals<VEC>& c) {
  Vals<VEC> r;
  if constexpr (VEC == 4) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float2 t = ffma2(make_float2(a.f[j], a.f[j + 1]), make_float2(b.f[j], b.f[j + 1]), make_float2(c.f[j], c.f[j + 1]));
      r.f[j] = t.x;
      r.f[j + 1] = t.y;
    }
  } else {
    r.f[0] = fmaf(a.f[0], b.f[0], c.f[0]);
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ Vals<VEC> all(float f) {
  Vals<VEC> r;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r.f[j] = f;
  return r;
}

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

constexpr int kMaxSlots = 8;

// A bulk copy into this CTA's shared memory (16-byte aligned addresses, a
// multiple of 16 bytes), counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Four branch values from shared memory.
__device__ __forceinline__ Vals<4> shared_branch(const uint8_t* p, int c, int type) {
  Vals<4> r;
  if (type == ND_F32) {
    const float4 t = *reinterpret_cast<const float4*>(p + c * 4);
    r.f[0] = t.x; r.f[1] = t.y; r.f[2] = t.z; r.f[3] = t.w;
  } else {
    const uint2 t = *reinterpret_cast<const uint2*>(p + c * 2);
    float2 lo, hi;
    if (type == ND_F16) {
      lo = __half22float2(*reinterpret_cast<const __half2*>(&t.x));
      hi = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
    } else {
      lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.x));
      hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.y));
    }
    r.f[0] = lo.x; r.f[1] = lo.y; r.f[2] = hi.x; r.f[3] = hi.y;
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

// The per-column factors of the VEC columns from c: the branch's post weight
// times gate, y's pre weight times (1 + scale), and the shift.
template <int VEC>
__device__ __forceinline__ Vals<VEC> factor(const float* weight, float plus_one, const float* vec, float plus, int c) {
  Vals<VEC> k;
#pragma unroll
  for (int j = 0; j < VEC; ++j) k.f[j] = 1.f;
  if (weight) {
    const Vals<VEC> w = load_vec<VEC>(weight + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) k.f[j] = w.f[j] + plus_one;
  }
  if (vec) {
    const Vals<VEC> w = load_vec<VEC>(vec + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) k.f[j] *= w.f[j] + plus;
  }
  return k;
}
// Read where they are used, or held in registers from row to row.
template <int VEC, int V, int T>
struct LazyFactors {
  const ResidualNorm& a;
  long long vec;
  int t;
  __device__ __forceinline__ int col(int i) const { return (t + T * i) * VEC; }
  __device__ __forceinline__ Vals<VEC> branch(int i) const {
    return factor<VEC>(a.post_weight, a.plus_one, a.gate ? a.gate + vec : nullptr, 0.f, col(i));
  }
  __device__ __forceinline__ Vals<VEC> y(int i) const {
    return factor<VEC>(a.pre_weight, a.plus_one, a.scale ? a.scale + vec : nullptr, 1.f, col(i));
  }
  __device__ __forceinline__ Vals<VEC> shift(int i) const {
    Vals<VEC> k;
#pragma unroll
    for (int j = 0; j < VEC; ++j) k.f[j] = 0.f;
    return a.shift ? load_vec<VEC>(a.shift + vec + col(i)) : k;
  }
};
template <int VEC, int V, int T>
struct HeldFactors {
  Vals<VEC> b[V], s[V], h[V];
  __device__ __forceinline__ void load(const ResidualNorm& a, long long vec, int t) {
    const LazyFactors<VEC, V, T> lazy{a, vec, t};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (lazy.col(i) < a.width) {
        b[i] = lazy.branch(i);
        s[i] = lazy.y(i);
        h[i] = lazy.shift(i);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) b[i].f[j] = s[i].f[j] = h[i].f[j] = 0.f;
      }
    }
  }
  __device__ __forceinline__ Vals<VEC> branch(int i) const { return b[i]; }
  __device__ __forceinline__ Vals<VEC> y(int i) const { return s[i]; }
  __device__ __forceinline__ Vals<VEC> shift(int i) const { return h[i]; }
};

// The vector set of row r, as an offset, and the first row past its share.
__device__ __forceinline__ long long vec_of(const ResidualNorm& a, int r, int* end = nullptr) {
  const int i = min(r / a.rows_per_vec, a.vecs - 1);
  if (end) *end = i == a.vecs - 1 ? INT_MAX : static_cast<int>(min((i + 1LL) * a.rows_per_vec, static_cast<long long>(INT_MAX)));
  return i * a.vec_stride;
}

// sum over pairs of a thread's values: f32x2 where there are four at a time.
template <int VEC, int V, bool SQUARE>
__device__ __forceinline__ float thread_sum(const Vals<VEC> (&w)[V]) {
  if constexpr (VEC == 4) {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 p = make_float2(w[i].f[j], w[i].f[j + 1]);
        s = SQUARE ? ffma2(p, p, s) : fadd2(s, p);
      }
    return s.x + s.y;
  } else {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) s = SQUARE ? fmaf(w[i].f[0], w[i].f[0], s) : s + w[i].f[0];
    return s;
  }
}

// One row, held by T threads as V x VEC values each (columns at and past the
// width are 0 in v and b): x' and y. `red`: five reductions' words.
template <int VEC, int V, int T, typename Factors>
__device__ __forceinline__ void finish_row(const ResidualNorm& a, long long r, int t, Vals<VEC> (&v)[V],
                                           Vals<VEC> (&b)[V], const Factors& k, float (*red)[T / 32]) {
  auto col = [&](int i) { return (t + T * i) * VEC; };
  // Subtract the mean (LayerNorm), then return rsqrt(mean square + eps).
  auto normalize = [&](Vals<VEC> (&w)[V], int kind, int slot) {
    if (kind == ND_NORM_LAYER) {
      const float mean = row_sum<T>(thread_sum<VEC, V, false>(w), red[slot]) * a.inv_width;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col(i) < a.width) w[i] = fma(w[i], all<VEC>(1.f), all<VEC>(-mean));
    }
    return rsqrtf(fmaf(row_sum<T>(thread_sum<VEC, V, true>(w), red[slot + 1]), a.inv_width, a.eps));
  };

  if (a.branch) {
    const float rstd = a.post != ND_NORM_NONE ? normalize(b, a.post, 0) : 1.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (col(i) < a.width) v[i] = fma(mul(b[i], all<VEC>(rstd)), k.branch(i), mul(v[i], all<VEC>(a.residual_scale)));
  } else if (a.residual_scale != 1.f) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = mul(v[i], all<VEC>(a.residual_scale));
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
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col(i);
    if (c < a.width) {
      v[i] = fma(mul(v[i], all<VEC>(rstd)), k.y(i), k.shift(i));
      if (a.out_type != ND_I8) store_vals<VEC>(a.y, r * a.ldy + c, v[i], a.out_type);
    }
  }
  if (a.out_type != ND_I8) return;
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (col(i) < a.width)
#pragma unroll
      for (int j = 0; j < VEC; ++j) peak = max(peak, abs_bits(v[i].f[j]));
  // y is an fp32 result already, so the quotient's last bit decides nothing
  // that fp32 had not rounded before: multiply by 127 / peak.
  const RowScale s = row_scale(row_max<T>(peak, reinterpret_cast<uint32_t*>(red[4])));
  if (t == 0) a.y_scale[r] = s.scale;
  int8_t* y = static_cast<int8_t*>(a.y) + r * a.ldy;
  // Where 127 / peak leaves fp32's range, both are first multiplied up.
  const float shift = s.peak < 1e-30f ? 0x1p96f : 1.f;
  const float inverse = s.inverse == 0.f || shift == 1.f ? s.inverse : __fdiv_rn(127.0f, s.peak * shift);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = col(i);
    if (c < a.width) {
      Vals<VEC> q = v[i];
      if (shift != 1.f) q = mul(q, all<VEC>(shift));
      q = fma(inverse != 0.f ? q : all<VEC>(0.f), all<VEC>(inverse), all<VEC>(kRintMagic));
      if constexpr (VEC == 4)
        *reinterpret_cast<uint32_t*>(y + c) = pack_low_bytes(__float_as_uint(q.f[0]), __float_as_uint(q.f[1]),
                                                             __float_as_uint(q.f[2]), __float_as_uint(q.f[3]));
      else
        y[c] = static_cast<int8_t>(__float_as_uint(q.f[0]) & 0xffu);
    }
  }
}

// One row per T threads, loaded straight into registers: few rows, narrow
// rows (a warp each, four to a block) and rows of any width or alignment.
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
  Vals<VEC> v[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + T * i) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i].f[j] = b[i].f[j] = 0.f;
    if (c < a.width) {
      v[i] = load_once<VEC>(a.x + r * a.ldx + c);
      if (a.branch) b[i] = load_branch<VEC>(a.branch, r * a.ldb + c, a.branch_type);
    }
  }
  finish_row<VEC, V, T>(a, r, t, v, b, LazyFactors<VEC, V, T>{a, vec_of(a, row), t}, red);
}

// Many rows: persistent blocks of T threads, each working through rows
// blockIdx.x, + gridDim.x, .. that bulk copies bring into a ring of `slots`
// row buffers, so that loads stay in flight through the rows' reductions (one
// row per block straight into registers ran at 55 % of the copy rate at
// 4352 x 4096: the loads paused while the rows were reduced and written). The
// thread's columns are the same in every row, so the per-column factors stay
// in registers and are read again only where the vector set changes.
template <int V, int T, int CTAS>
__global__ void __launch_bounds__(T, CTAS) residual_norm_ring_kernel(const ResidualNorm a, int slots, unsigned* status) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float red[5][T / 32];
  __shared__ uint64_t full_bars[kMaxSlots];
  __shared__ volatile int abort_flag;
  const int t = threadIdx.x;
  const uint32_t x_bytes = a.width * 4u;
  const uint32_t b_bytes = a.branch ? a.width * (a.branch_type == ND_F32 ? 4u : 2u) : 0u;
  const uint32_t slot_bytes = x_bytes + b_bytes;
  const uint32_t base = smem_u32(ring);
  if (t == 0) {
    for (int s = 0; s < slots; ++s) mbar_init(smem_u32(&full_bars[s]), 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  griddep_launch();
  griddep_wait();
  auto fetch = [&](int row, int s) {
    const long long r = row;  // one thread
    const uint32_t bar = smem_u32(&full_bars[s]), dst = base + s * slot_bytes;
    mbar_arrive_expect_tx(bar, slot_bytes);
    bulk_load(dst, a.x + r * a.ldx, x_bytes, bar);
    if (b_bytes)
      bulk_load(dst + x_bytes, static_cast<const uint8_t*>(a.branch) + r * a.ldb * (a.branch_type == ND_F32 ? 4 : 2), b_bytes, bar);
  };
  const int step = gridDim.x;
  int next = blockIdx.x;  // thread 0: the next row to ask for
  if (t == 0)
    for (int i = 0; i < slots && next < a.rows; ++i, next += step) fetch(next, i);

  HeldFactors<4, V, T> k;
  int vec_end = 0;  // first row past the held set's share
  int it = 0, s = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (int r = blockIdx.x; r < a.rows; r += step, ++it) {
    if (t < 32) ok = mbar_wait(smem_u32(&full_bars[s]), parity, &abort_flag, status, kStatusTimeoutProducer);
    if (!__syncthreads_and(ok)) break;
    // Everyone is done with the row before this one: its slot is filled again.
    if (t == 0 && it > 0 && next < a.rows) {
      fetch(next, s > 0 ? s - 1 : slots - 1);
      next += step;
    }
    if (r >= vec_end) k.load(a, vec_of(a, r, &vec_end), t);
    Vals<4> v[V], b[V];
    const uint8_t* slot = ring + s * slot_bytes;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + T * i) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i].f[j] = b[i].f[j] = 0.f;
      if (c < a.width) {
        const float4 x = *reinterpret_cast<const float4*>(slot + c * 4);
        v[i].f[0] = x.x; v[i].f[1] = x.y; v[i].f[2] = x.z; v[i].f[3] = x.w;
        if (b_bytes) b[i] = shared_branch(slot + x_bytes, c, a.branch_type);
      }
    }
    finish_row<4, V, T>(a, r, t, v, b, k, red);
    if (++s == slots) {
      s = 0;
      parity ^= 1u;
    }
  }
  if (!ok && t == 0) {
    // Timed out: let the copies in flight (rows r to next) land before shared memory goes away.
    volatile int never = 0;
    for (int r = blockIdx.x + it * step; r < next; r += step) {
      mbar_wait(smem_u32(&full_bars[s]), parity, &never, nullptr, 0);
      if (++s == slots) {
        s = 0;
        parity ^= 1u;
      }
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

// The ring kernel: CTAS blocks of T threads per SM, their rings sharing its
// shared memory.
template <int V, int T, int CTAS>
int launch_ring(const ResidualNorm& a, cudaStream_t stream) {
  auto kernel = residual_norm_ring_kernel<V, T, CTAS>;
  constexpr int kRing = 220 * 1024 / CTAS - 1024;  // the SM's 227 KB, less the blocks' static share and reserve
  static bool configured[64] = {};
  int dev = 0;
  ND_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing));
    configured[dev & 63] = true;
  }
  const int row_bytes = a.width * (4 + (a.branch ? (a.branch_type == ND_F32 ? 4 : 2) : 0));
  const int slots = std::min(kMaxSlots, kRing / row_bytes);
  unsigned* status = device_status();
  if (!status) return fail(ND_ERR_CUDA, "residual_norm: no device status word");
  const unsigned grid = static_cast<unsigned>(std::min(a.rows, CTAS * sm_count()));
  ND_CUDA(launch_pdl(kernel, dim3(grid), dim3(T), slots * row_bytes, stream, a, slots, status));
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
  if (a.rows > INT_MAX - (1 << 20)) return fail(ND_ERR_INVALID, "residual_norm: too many rows");
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
  k.rows_per_vec = static_cast<int>(a.vecs > 1 ? std::min<int64_t>(a.rows_per_vec, INT_MAX) : INT_MAX);
  k.rows = static_cast<int>(a.rows);
  k.width = static_cast<int>(a.width);
  k.residual_scale = a.residual_scale;
  k.plus_one = a.plus_one ? 1.f : 0.f;
  k.eps = a.eps;
  k.inv_width = 1.f / static_cast<float>(a.width);

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
  // Bulk copies take rows whose starts and lengths are multiples of 16 bytes.
  const bool bulk = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                    (!a.branch || (reinterpret_cast<uintptr_t>(a.branch) % 16 == 0 &&
                                   (a.branch_dtype == ND_F32 || (a.width % 8 == 0 && a.ldb % 8 == 0))));
  if (bulk && w4 > 256 && a.rows >= 8 * sm_count()) {
    if (w4 <= 512) return launch_ring<4, 128, 4>(k, stream);
    if (w4 <= 1024) return launch_ring<4, 256, 2>(k, stream);
    if (w4 <= 2048) return launch_ring<4, 512, 1>(k, stream);
  }
  if (w4 <= 128) return launch<4, 4, 32>(k, stream);
  if (w4 <= 256) return launch<4, 2, 128>(k, stream);
  if (w4 <= 512) return launch<4, 4, 128>(k, stream);
  if (w4 <= 1024) return launch<4, 4, 256>(k, stream);
  if (w4 <= 2048) return launch<4, 4, 512>(k, stream);
  return launch<4, 4, 1024>(k, stream);
}

}  // namespace nd
