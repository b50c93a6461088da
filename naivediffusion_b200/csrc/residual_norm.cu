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
// fp32. 4352 x 4096 (bf16 branch and y) 39 us, 5.5 TB/s, 83 % of the copy rate;
// 8192 x 2048 to int8 36 us, 79 % (34 with one fp32 factor 127 / peak, whose
// int8 rows were one off quantize_rows' near halves); 4000 x 3001 41 us, 54 %.
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

// A thread's share of a row: V groups of VEC neighbouring columns, T * VEC
// apart, as pairs for the paired fp32 instructions (VEC = 1: two groups make a
// pair). Pointers are to the thread's first column, so every offset is a
// constant; `rem` is the width less that column. Columns at and past the width
// load as 0.
template <int VEC, int V, int T>
struct Share {
  static constexpr int H = VEC * V / 2;
  static constexpr int kStep = VEC * T;

  template <bool ONCE>  // read once from global memory: past L1
  static __device__ __forceinline__ void load(const float* p, int rem, float2 (&v)[H]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (VEC == 4) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (kStep * i < rem) {
          if constexpr (ONCE)
            asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                         : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                         : "l"(p + kStep * i));
          else
            x = *reinterpret_cast<const float4*>(p + kStep * i);
        }
        v[2 * i] = make_float2(x.x, x.y);
        v[2 * i + 1] = make_float2(x.z, x.w);
      } else {
        (i & 1 ? v[i / 2].y : v[i / 2].x) = kStep * i < rem ? p[kStep * i] : 0.f;
      }
    }
  }
  template <bool F16>
  static __device__ __forceinline__ void load(const uint16_t* p, int rem, float2 (&v)[H]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (VEC == 4) {
        uint2 w = make_uint2(0u, 0u);
        if (kStep * i < rem) w = *reinterpret_cast<const uint2*>(p + kStep * i);
        v[2 * i] = halves<F16>(w.x);
        v[2 * i + 1] = halves<F16>(w.y);
      } else {
        const uint32_t w = kStep * i < rem ? p[kStep * i] : 0u;
        (i & 1 ? v[i / 2].y : v[i / 2].x) = halves<F16>(w).x;
      }
    }
  }
  template <bool F16>
  static __device__ __forceinline__ float2 halves(uint32_t w) {
    if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  // From `p` + the thread's first column, element type `type`.
  template <bool ONCE>
  static __device__ __forceinline__ void load_typed(const void* p, int first, int type, int rem, float2 (&v)[H]) {
    if (type == ND_F32) load<ONCE>(static_cast<const float*>(p) + first, rem, v);
    else if (type == ND_F16) load<true>(static_cast<const uint16_t*>(p) + first, rem, v);
    else load<false>(static_cast<const uint16_t*>(p) + first, rem, v);
  }

  static __device__ __forceinline__ void store(float* p, int rem, const float2 (&v)[H]) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (kStep * i < rem) {
        if constexpr (VEC == 4)
          *reinterpret_cast<float4*>(p + kStep * i) = make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
        else p[kStep * i] = i & 1 ? v[i / 2].y : v[i / 2].x;
      }
  }
  template <bool F16>
  static __device__ __forceinline__ void store(uint16_t* p, int rem, const float2 (&v)[H]) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (kStep * i < rem) {
        if constexpr (VEC == 4) {
          const float2 a = v[2 * i], b = v[2 * i + 1];
          *reinterpret_cast<uint2*>(p + kStep * i) = F16 ? make_uint2(pack_f16(a.x, a.y), pack_f16(b.x, b.y))
                                                         : make_uint2(pack_bf16(a.x, a.y), pack_bf16(b.x, b.y));
        } else {
          const float f = i & 1 ? v[i / 2].y : v[i / 2].x;
          p[kStep * i] = static_cast<uint16_t>(F16 ? pack_f16(f, 0.f) : pack_bf16(f, 0.f));
        }
      }
  }
  // The low bytes of v's bit patterns.
  static __device__ __forceinline__ void store(int8_t* p, int rem, const float2 (&v)[H]) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (kStep * i < rem) {
        if constexpr (VEC == 4)
          *reinterpret_cast<uint32_t*>(p + kStep * i) =
              pack_low_bytes(__float_as_uint(v[2 * i].x), __float_as_uint(v[2 * i].y), __float_as_uint(v[2 * i + 1].x),
                             __float_as_uint(v[2 * i + 1].y));
        else p[kStep * i] = static_cast<int8_t>(__float_as_uint(i & 1 ? v[i / 2].y : v[i / 2].x) & 0xffu);
      }
  }
};

__device__ __forceinline__ float2 splat(float f) { return make_float2(f, f); }

constexpr int kMaxSlots = 8;

// A bulk copy into this CTA's shared memory (16-byte aligned addresses, a
// multiple of 16 bytes), counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
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

// A thread's per-column factors for vector set offset `vec`: the branch's post
// weight times gate, y's pre weight times (1 + scale), and the shift. Held from
// row to row, or (lazy) read where they are used.
template <int VEC, int V, int T>
struct Factors {
  using S = Share<VEC, V, T>;
  static __device__ __forceinline__ void product(const float* weight, float plus_one, const float* vec, float plus, int rem,
                                                 float2 (&k)[S::H]) {
    if (weight) {
      S::template load<false>(weight, rem, k);
#pragma unroll
      for (int h = 0; h < S::H; ++h) k[h] = fadd2(k[h], splat(plus_one));
    } else {
#pragma unroll
      for (int h = 0; h < S::H; ++h) k[h] = splat(1.f);
    }
    if (vec) {
      float2 g[S::H];
      S::template load<false>(vec, rem, g);
#pragma unroll
      for (int h = 0; h < S::H; ++h) k[h] = fmul2(k[h], fadd2(g[h], splat(plus)));
    }
  }
  static __device__ __forceinline__ const float* at(const float* p, long long i) { return p ? p + i : nullptr; }
  static __device__ __forceinline__ void branch(const ResidualNorm& a, long long vec, int first, float2 (&k)[S::H]) {
    product(at(a.post_weight, first), a.plus_one, at(a.gate, vec + first), 0.f, a.width - first, k);
  }
  static __device__ __forceinline__ void y(const ResidualNorm& a, long long vec, int first, float2 (&k)[S::H],
                                           float2 (&shift)[S::H]) {
    product(at(a.pre_weight, first), a.plus_one, at(a.scale, vec + first), 1.f, a.width - first, k);
    if (a.shift) {
      S::template load<false>(a.shift + vec + first, a.width - first, shift);
    } else {
#pragma unroll
      for (int h = 0; h < S::H; ++h) shift[h] = splat(0.f);
    }
  }
};

// The vector set of row r, as an offset, and the first row past its share.
__device__ __forceinline__ long long vec_of(const ResidualNorm& a, int r, int* end = nullptr) {
  const int i = min(r / a.rows_per_vec, a.vecs - 1);
  if (end) *end = i == a.vecs - 1 ? INT_MAX : static_cast<int>(min((i + 1LL) * a.rows_per_vec, static_cast<long long>(INT_MAX)));
  return i * a.vec_stride;
}

// One row in T threads' registers: x' and y. `red`: five reductions' words.
// held: this row's factors, or null to read them here.
template <int VEC, int V, int T>
struct HeldFactors {
  float2 branch[VEC * V / 2], y[VEC * V / 2], shift[VEC * V / 2];
};
template <int VEC, int V, int T>
__device__ __forceinline__ void finish_row(const ResidualNorm& a, long long r, int t, float2 (&v)[VEC * V / 2],
                                           float2 (&b)[VEC * V / 2], const HeldFactors<VEC, V, T>* held, long long vec,
                                           float (*red)[T / 32]) {
  using S = Share<VEC, V, T>;
  const int first = t * VEC, rem = a.width - first;
  // Subtract the mean (LayerNorm), then return rsqrt(mean square + eps).
  auto normalize = [&](float2 (&w)[S::H], int kind, int slot) {
    if (kind == ND_NORM_LAYER) {
      float2 s = splat(0.f);
#pragma unroll
      for (int h = 0; h < S::H; ++h) s = fadd2(s, w[h]);
      const float mean = row_sum<T>(s.x + s.y, red[slot]) * a.inv_width;
#pragma unroll
      for (int i = 0; i < V; ++i)  // columns past the width stay 0
        if (S::kStep * i < rem) {
          if constexpr (VEC == 4) {
            w[2 * i] = fadd2(w[2 * i], splat(-mean));
            w[2 * i + 1] = fadd2(w[2 * i + 1], splat(-mean));
          } else {
            (i & 1 ? w[i / 2].y : w[i / 2].x) -= mean;
          }
        }
    }
    float2 q = splat(0.f);
#pragma unroll
    for (int h = 0; h < S::H; ++h) q = ffma2(w[h], w[h], q);
    return rsqrtf(fmaf(row_sum<T>(q.x + q.y, red[slot + 1]), a.inv_width, a.eps));
  };

  const float2 alpha = splat(a.residual_scale);
  if (a.branch) {
    const float2 rstd = splat(a.post != ND_NORM_NONE ? normalize(b, a.post, 0) : 1.f);
    float2 own[S::H];
    if (!held) Factors<VEC, V, T>::branch(a, vec, first, own);
#pragma unroll
    for (int h = 0; h < S::H; ++h) v[h] = ffma2(fmul2(b[h], rstd), held ? held->branch[h] : own[h], fmul2(v[h], alpha));
  } else if (a.residual_scale != 1.f) {
#pragma unroll
    for (int h = 0; h < S::H; ++h) v[h] = fmul2(v[h], alpha);
  }
  if (a.x_out) S::store(a.x_out + r * a.ldxo + first, rem, v);
  if (!a.y) return;

  const float2 rstd = splat(a.pre != ND_NORM_NONE ? normalize(v, a.pre, 2) : 1.f);
  if (held) {
#pragma unroll
    for (int h = 0; h < S::H; ++h) v[h] = ffma2(fmul2(v[h], rstd), held->y[h], held->shift[h]);
  } else {
    float2 k[S::H], shift[S::H];
    Factors<VEC, V, T>::y(a, vec, first, k, shift);
#pragma unroll
    for (int h = 0; h < S::H; ++h) v[h] = ffma2(fmul2(v[h], rstd), k[h], shift[h]);
  }
  if (a.out_type == ND_BF16) {
    S::template store<false>(static_cast<uint16_t*>(a.y) + r * a.ldy + first, rem, v);
    return;
  }
  if (a.out_type == ND_F16) {
    S::template store<true>(static_cast<uint16_t*>(a.y) + r * a.ldy + first, rem, v);
    return;
  }
  if (a.out_type == ND_F32) {
    S::store(static_cast<float*>(a.y) + r * a.ldy + first, rem, v);
    return;
  }
  // int8. Columns past the width: their factors are anything, their bits not counted.
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (S::kStep * i < rem) {
      if constexpr (VEC == 4)
        peak = max(max(peak, max(abs_bits(v[2 * i].x), abs_bits(v[2 * i].y))),
                   max(abs_bits(v[2 * i + 1].x), abs_bits(v[2 * i + 1].y)));
      else peak = max(peak, abs_bits(i & 1 ? v[i / 2].y : v[i / 2].x));
    }
  const RowScale s = row_scale(row_max<T>(peak, reinterpret_cast<uint32_t*>(red[4])));
  if (t == 0) a.y_scale[r] = s.scale;
  if (s.zero) {
#pragma unroll
    for (int h = 0; h < S::H; ++h) v[h] = splat(kRintMagic);
  } else {
    const float shift = range_shift(s.peak);
    if (shift != 1.f) {
#pragma unroll
      for (int h = 0; h < S::H; ++h) v[h] = fmul2(v[h], splat(shift));
    }
    const float row_peak = s.peak * shift;
    const Inverse inverse = inverse_of(row_peak);
#pragma unroll
    for (int h = 0; h < S::H; h += 2) {
      const float f[4] = {v[h].x, v[h].y, v[h + 1].x, v[h + 1].y};
      float m[4];
      quantize_values<true>(f, inverse, row_peak, m);
      v[h] = make_float2(m[0], m[1]);
      v[h + 1] = make_float2(m[2], m[3]);
    }
  }
  S::store(static_cast<int8_t*>(a.y) + r * a.ldy + first, rem, v);
}

// One row per T threads, loaded straight into registers: few rows, narrow
// rows (a warp each, four to a block) and rows of any width or alignment.
template <int VEC, int V, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T) residual_norm_kernel(const ResidualNorm a) {
  griddep_launch();
  griddep_wait();
  __shared__ float red[5][T / 32];
  using S = Share<VEC, V, T>;
  constexpr int kRows = T < 128 ? 128 / T : 1;
  const int t = threadIdx.x % T;
  const int row = blockIdx.x * kRows + threadIdx.x / T;
  if (row >= a.rows) return;  // whole warps: only T = 32 has several rows per block
  const long long r = row;
  float2 v[S::H], b[S::H];
  S::template load<true>(a.x + r * a.ldx + t * VEC, a.width - t * VEC, v);
  if (a.branch) {
    const uint8_t* p = static_cast<const uint8_t*>(a.branch) + r * a.ldb * (a.branch_type == ND_F32 ? 4 : 2);
    S::template load_typed<true>(p, t * VEC, a.branch_type, a.width - t * VEC, b);
  }
  finish_row<VEC, V, T>(a, r, t, v, b, nullptr, vec_of(a, row), red);
}

// The part of one row that a bulk copy takes: from the 16-byte boundary at or
// before its first byte to the one at or after its last, except where that
// would leave the matrix (rows at its ends that start or end off a boundary);
// those few bytes are copied by hand.
struct RowSpan {
  const uint8_t* start;  // of the row
  uint32_t skip;         // bytes between the 16-byte boundary before it and the row: its place in its buffer
  uint32_t head, tail;   // bytes of the row to copy by hand at either end
};
__device__ __forceinline__ RowSpan row_span(const uint8_t* start, const uint8_t* first, const uint8_t* last, uint32_t bytes) {
  RowSpan s;  // first, last: the matrix
  s.start = start;
  s.skip = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(start) & 15u);
  const uint32_t end = (s.skip + bytes) & 15u;  // bytes past the last boundary inside the row's end
  s.head = s.skip && start - s.skip < first ? min(16u - s.skip, bytes) : 0u;
  s.tail = end && start + bytes + (16u - end) > last ? min(end, bytes - s.head) : 0u;
  return s;
}
// Ask for the row into `dst` (16-byte aligned, bytes + 30 long); returns the
// bytes that the bulk copy brings. Called by one thread, before it arrives.
__device__ __forceinline__ uint32_t span_bulk(const RowSpan& s, uint32_t bytes, uint32_t& from) {
  from = s.head ? 16u : 0u;  // the copy's first byte in the buffer
  const uint32_t all = (s.skip + bytes + 15u) & ~15u;
  const uint32_t to = s.tail ? (s.skip + bytes) & ~15u : all;
  return to > from ? to - from : 0u;
}

// Many rows: persistent blocks of T threads, each working through rows
// blockIdx.x, + gridDim.x, .. that bulk copies bring into a ring of `slots`
// row buffers, so that loads stay in flight through the rows' reductions (one
// row per block straight into registers ran at 55 % of the copy rate at
// 4352 x 4096: the loads paused while the rows were reduced and written). The
// thread's columns are the same in every row, so the per-column factors stay
// in registers and are read again only where the vector set changes. VEC = 1:
// rows of any width and alignment, shared memory and stores one value at a
// time.
template <int VEC, int V, int T, int CTAS>
__global__ void __launch_bounds__(T, CTAS) residual_norm_ring_kernel(const ResidualNorm a, int slots, uint32_t x_room,
                                                                     uint32_t b_room, unsigned* status) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float red[5][T / 32];
  __shared__ uint64_t full_bars[kMaxSlots];
  __shared__ volatile int abort_flag;
  const int t = threadIdx.x;
  const int b_elem = a.branch_type == ND_F32 ? 4 : 2;
  const uint32_t x_bytes = a.width * 4u;
  const uint32_t b_bytes = a.branch ? static_cast<uint32_t>(a.width * b_elem) : 0u;
  const uint32_t slot_bytes = x_room + b_room;
  const uint32_t base = smem_u32(ring);
  if (t == 0) {
    for (int s = 0; s < slots; ++s) mbar_init(smem_u32(&full_bars[s]), 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  griddep_launch();
  griddep_wait();
  // Thread 0 asks for rows: the next one, where it starts, and the slot it goes to.
  const int step = gridDim.x;
  int next = blockIdx.x;
  const uint8_t* next_x = reinterpret_cast<const uint8_t*>(a.x + next * a.ldx);
  const uint8_t* next_b = static_cast<const uint8_t*>(a.branch) + (b_bytes ? next * a.ldb * b_elem : 0);
  const long long x_step = step * a.ldx * 4, b_step = b_bytes ? step * a.ldb * b_elem : 0;
  bool dirty = false;
  auto fetch = [&](int s) {
    const uint32_t bar = smem_u32(&full_bars[s]), dst = base + s * slot_bytes;
    if constexpr (VEC == 4) {
      mbar_arrive_expect_tx(bar, x_bytes + b_bytes);
      bulk_load(dst, next_x, x_bytes, bar);
      if (b_bytes) bulk_load(dst + x_room, next_b, b_bytes, bar);
    } else {
      uint32_t from_x, from_b = 0, n_b = 0;
      const uint8_t* fx = reinterpret_cast<const uint8_t*>(a.x);
      const RowSpan x = row_span(next_x, fx, fx + (a.rows - 1) * a.ldx * 4 + x_bytes, x_bytes);
      const uint32_t n_x = span_bulk(x, x_bytes, from_x);
      RowSpan b{};
      if (b_bytes) {
        const uint8_t* fb = static_cast<const uint8_t*>(a.branch);
        b = row_span(next_b, fb, fb + (a.rows - 1) * a.ldb * b_elem + b_bytes, b_bytes);
        n_b = span_bulk(b, b_bytes, from_b);
      }
      auto by_hand = [&](const RowSpan& w, uint32_t at, uint32_t bytes) {
        uint8_t* to = ring + at + w.skip;
        for (uint32_t i = 0; i < w.head; i += 2)
          *reinterpret_cast<uint16_t*>(to + i) = *reinterpret_cast<const uint16_t*>(w.start + i);
        for (uint32_t i = bytes - w.tail; i < bytes; i += 2)
          *reinterpret_cast<uint16_t*>(to + i) = *reinterpret_cast<const uint16_t*>(w.start + i);
      };
      // Bytes once copied by hand may lie where a later bulk copy goes.
      if (dirty) fence_proxy_async_smem();
      if (x.head | x.tail | b.head | b.tail) {
        by_hand(x, s * slot_bytes, x_bytes);
        by_hand(b, s * slot_bytes + x_room, b_bytes);
        dirty = true;
      }
      mbar_arrive_expect_tx(bar, n_x + n_b);
      if (n_x) bulk_load(dst + from_x, x.start - x.skip + from_x, n_x, bar);
      if (n_b) bulk_load(dst + x_room + from_b, b.start - b.skip + from_b, n_b, bar);
    }
    next += step;
    next_x += x_step;
    next_b += b_step;
  };
  if (t == 0)
    for (int i = 0; i < slots && next < a.rows; ++i) fetch(i);

  using S = Share<VEC, V, T>;
  HeldFactors<VEC, V, T> k;
  int vec_end = 0;  // first row past the held set's share
  int it = 0, s = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (int r = blockIdx.x; r < a.rows; r += step, ++it) {
    if (t < 32) ok = mbar_wait(smem_u32(&full_bars[s]), parity, &abort_flag, status, kStatusTimeoutProducer);
    ok = __syncthreads_and(ok);  // the block's: thread 0 sees another lane's timeout too
    if (!ok) break;
    // Everyone is done with the row before this one: its slot is filled again.
    if (t == 0 && it > 0 && next < a.rows) fetch(s > 0 ? s - 1 : slots - 1);
    if (r >= vec_end) {
      const long long vec = vec_of(a, r, &vec_end);
      Factors<VEC, V, T>::branch(a, vec, t * VEC, k.branch);
      Factors<VEC, V, T>::y(a, vec, t * VEC, k.y, k.shift);
    }
    const uint8_t* x_row = ring + s * slot_bytes;
    const uint8_t* b_row = x_row + x_room;
    if constexpr (VEC == 1) {
      x_row += reinterpret_cast<uintptr_t>(a.x + r * a.ldx) & 15u;
      if (b_bytes) b_row += reinterpret_cast<uintptr_t>(static_cast<const uint8_t*>(a.branch) + r * a.ldb * b_elem) & 15u;
    }
    float2 v[S::H], b[S::H];
    S::template load<false>(reinterpret_cast<const float*>(x_row) + t * VEC, a.width - t * VEC, v);
    if (b_bytes) S::template load_typed<false>(b_row, t * VEC, a.branch_type, a.width - t * VEC, b);
    finish_row<VEC, V, T>(a, r, t, v, b, &k, 0, red);
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
template <int VEC, int V, int T, int CTAS>
int launch_ring(const ResidualNorm& a, cudaStream_t stream) {
  auto kernel = residual_norm_ring_kernel<VEC, V, T, CTAS>;
  // The SM's 228 KB, less a block's reserve of 1 KB and its static share.
  constexpr int kRing = (228 * 1024 / CTAS - 1024 - 512) & ~15;
  static_assert(kRing + 512 <= 227 * 1024, "a block's most");
  static bool configured[64] = {};
  int dev = 0;
  ND_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    ND_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing));
    configured[dev & 63] = true;
  }
  // A row of any alignment lies up to 15 bytes past its buffer's start.
  auto room = [](int bytes) { return VEC == 4 ? bytes : (bytes + 15 + 15) & ~15; };
  const int x_room = room(a.width * 4);
  const int b_room = a.branch ? room(a.width * (a.branch_type == ND_F32 ? 4 : 2)) : 0;
  const int slots = std::min(kMaxSlots, kRing / (x_room + b_room));
  unsigned* status = device_status();
  if (!status) return fail(ND_ERR_CUDA, "residual_norm: no device status word");
  const unsigned grid = static_cast<unsigned>(std::min(a.rows, CTAS * sm_count()));
  ND_CUDA(launch_pdl(kernel, dim3(grid), dim3(T), slots * (x_room + b_room), stream, a, slots,
                     static_cast<uint32_t>(x_room), static_cast<uint32_t>(b_room), status));
  ND_CUDA(cudaGetLastError());
  return ND_OK;
}

template <int VEC>
int launch_ring_for(const ResidualNorm& a, cudaStream_t stream) {  // width <= 8192
  constexpr int V = 16 / VEC;
  if (a.width <= 512) return launch_ring<VEC, V, 32, 14>(a, stream);
  if (a.width <= 1024) return launch_ring<VEC, V, 64, 8>(a, stream);
  if (a.width <= 2048) return launch_ring<VEC, V, 128, 4>(a, stream);
  if (a.width <= 4096) return launch_ring<VEC, V, 256, 2>(a, stream);
  return launch_ring<VEC, V, 512, 1>(a, stream);
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
  // Bulk copies of whole rows take starts and lengths that are multiples of 16 bytes.
  const bool bulk = by4 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                    (!a.branch || (reinterpret_cast<uintptr_t>(a.branch) % 16 == 0 &&
                                   (a.branch_dtype == ND_F32 || (a.width % 8 == 0 && a.ldb % 8 == 0))));
  // Ring or straight into registers, us (both measured): 1500 x 4096 17.9 / 17.3, 4352 x 4096 39 / 46, 2048 x 1280
  // 9.5 / 8.3, 16384 x 1024 37 / 38, 300 x 8192 10.7 / 12.2; unaligned 333 x 1155 5.7 / 4.7, 300 x 3001 8.5 / 12.3,
  // 4000 x 3001 41 / 115.
  const int64_t values = a.rows * a.width;
  if (a.width <= 8192) {
    if (bulk && (a.width > 4096 ? a.rows >= 2 * sm_count() : values >= (8 << 20))) return launch_ring_for<4>(k, stream);
    if (!by4 && values >= 600000) return launch_ring_for<1>(k, stream);
  }
  if (!by4) {
    if (a.width <= 1024) return launch<1, 4, 256>(k, stream);
    if (a.width <= 2048) return launch<1, 8, 256>(k, stream);
    if (a.width <= 8192) return launch<1, 8, 1024>(k, stream);
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
