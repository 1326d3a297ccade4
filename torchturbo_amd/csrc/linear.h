// What the kernels of the dense products share: the product's description and
// what becomes of its sums (bias, activation, gate, dropout, row scale, residual).
#pragma once

#include <math.h>

#include "gemm.h"
#include "philox.h"

// What becomes of the fp32 sums v = sum over r of A(i, r) B(r, j):
//   ACT    y = act(v + bias)
//   GATED  y = act(v + bias) * (u + bias'), u the sums of the second J columns
//   RES    y = residual + scale[i] * (v + bias)
//   DROP   y = residual + scale[i] * drop(v + bias)
//   DGRAD  y = scale[i] * alpha v; xs = scale[i] * x; dots[i] = sum over j of x * alpha v
//   PLAIN  y = alpha v
enum { LIN_ACT = 0, LIN_GATED = 1, LIN_RES = 2, LIN_DROP = 3, LIN_DGRAD = 4, LIN_PLAIN = 5 };
// Activations.
enum { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2 };
// Columns that one partial dot product of DGRAD covers: the least that a wave has.
constexpr int LIN_DOT = 32;

// C [I, J] of A and B, both of the type of `out` (GATED: B has 2 J columns, the
// gate's first). Which of A and B has the reduction contiguous in memory is the
// kernel's template; lda and ldb are the distance of their rows, in elements.
// Null pointers: that part is left out.
struct LinArgs {
  const void* a;
  const void* b;
  void* out;
  int64_t I, J, R, lda, ldb;
  const void* bias;
  int bias_dt;
  int act;
  float* pre;  // ACT / GATED: v + bias, [I, J] or [I, 2 J] fp32
  const void* res;
  const void* scale;
  int scale_dt;
  uint32_t threshold;  // DROP
  float alpha;         // DROP, DGRAD, PLAIN: 1 / (share kept)
  const int64_t* key;
  const void* x;  // DGRAD
  void* xs;
  float* dots;  // [I, ceil(J / LIN_DOT)]
  float* part;  // a split reduction's sums [splits, I, J or 2 J], instead of all of the above
  int splits;
  int64_t rsplit;  // reduction elements of a split
};

namespace {

// The activation and its derivative. 16-bit tensors take the hardware's exp2 and
// reciprocal (a few ulp of fp32, far below the rounding of what they end in).
template <class TT>
__device__ __forceinline__ float lin_sigmoid(float a) {
  if constexpr (sizeof(typename TT::storage) == 4) return 1.0f / (1.0f + expf(-a));
  else return __builtin_amdgcn_rcpf(1.0f + __expf(-a));
}
template <class TT>
__device__ __forceinline__ float lin_act(int act, float a) {
  if (act == ACT_SILU) return a * lin_sigmoid<TT>(a);
  if (act == ACT_GELU) return 0.5f * a * (1.0f + erff(a * 0.70710678118654752f));
  return a;
}
template <class TT>
__device__ __forceinline__ void lin_act_grad(int act, float a, float& value, float& slope) {
  if (act == ACT_SILU) {
    const float s = lin_sigmoid<TT>(a);
    value = a * s;
    slope = s * (1.0f + a * (1.0f - s));
  } else if (act == ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(a * 0.70710678118654752f));
    value = a * cdf;
    slope = cdf + a * 0.39894228040143268f * expf(-0.5f * a * a);
  } else {
    value = a;
    slope = 1.0f;
  }
}

// W consecutive elements at p[at], widened; n of them exist (VEC: all, aligned; the
// memory instructions take any address, and an aligned one is one line less).
template <class TT, int W, bool VEC>
__device__ __forceinline__ void lin_load(const void* p, int64_t at, int n, float (&o)[W]) {
  typedef typename TT::storage St;
  const St* q = static_cast<const St*>(p) + at;
  if constexpr (VEC) {
    St v[W];
    __builtin_memcpy(v, __builtin_assume_aligned(q, sizeof(St) * W < 16 ? sizeof(St) * W : 16), sizeof(v));
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = TT::to_f32(v[j]);
  } else if (n == W) {
    St v[W];
    __builtin_memcpy(v, q, sizeof(v));
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = TT::to_f32(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = j < n ? TT::to_f32(q[j]) : 0.f;
  }
}
template <class TT, int W, bool VEC>
__device__ __forceinline__ void lin_store(void* p, int64_t at, int n, const float (&v)[W]) {
  typedef typename TT::storage St;
  St* q = static_cast<St*>(p) + at;
  if (VEC || n == W) {
    constexpr int AT = VEC ? (sizeof(St) * W < 16 ? sizeof(St) * W : 16) : sizeof(St);
    if constexpr (sizeof(St) == 2) {
      uint2 o[W / 4];
#pragma unroll
      for (int e = 0; e < W / 4; ++e)
        o[e] = pack4<__is_same(TT, BF16T) ? TT_BF16 : TT_F16>(v[4 * e], v[4 * e + 1], v[4 * e + 2],
                                                              v[4 * e + 3]);
      __builtin_memcpy(__builtin_assume_aligned(q, AT), o, sizeof(o));
    } else {
      __builtin_memcpy(__builtin_assume_aligned(q, AT), v, sizeof(v));
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < n) q[j] = TT::from_f32(v[j]);
  }
}

// What a result needs besides its sums: of its columns (the same for every row),
// and of its row; fetched ahead of the sums' arrival where a kernel can.
template <int KIND, int W>
struct LinCols {
  float b[W], bu[KIND == LIN_GATED ? W : 1];
};
template <class TT, int W>
struct LinRow {
  typename TT::storage v[W];  // RES: the residual, DGRAD: x
  float s;                    // the row's scale
};

// Columns j .. j + W - 1, n of them exist.
template <int KIND, int W>
__device__ __forceinline__ LinCols<KIND, W> lin_cols(const LinArgs& p, int64_t j, int n) {
  LinCols<KIND, W> c;
#pragma unroll
  for (int e = 0; e < W; ++e) c.b[e] = 0.f;
  if constexpr (KIND == LIN_GATED) {
#pragma unroll
    for (int e = 0; e < W; ++e) c.bu[e] = 0.f;
  }
  if (KIND <= LIN_DROP && p.bias != nullptr) {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < n) c.b[e] = load_as_f32(p.bias, p.bias_dt, j + e);
    if constexpr (KIND == LIN_GATED) {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (e < n) c.bu[e] = load_as_f32(p.bias, p.bias_dt, p.J + j + e);
    }
  }
  return c;
}

template <int KIND, class TT, int W, bool VEC>
__device__ __forceinline__ LinRow<TT, W> lin_row(const LinArgs& p, int64_t i, int64_t j, int n) {
  typedef typename TT::storage St;
  LinRow<TT, W> r;
  r.s = 1.f;
#pragma unroll
  for (int e = 0; e < W; ++e) r.v[e] = St(0);
  if constexpr (KIND == LIN_RES || KIND == LIN_DROP || KIND == LIN_DGRAD) {
    const void* src = KIND == LIN_DGRAD ? (p.scale != nullptr ? p.x : nullptr) : p.res;
    if (p.scale != nullptr) r.s = load_as_f32(p.scale, p.scale_dt, i);
    if (src != nullptr) {
      const St* q = static_cast<const St*>(src) + i * p.J + j;
      if constexpr (VEC) {
        __builtin_memcpy(r.v, __builtin_assume_aligned(q, sizeof(St) * W < 16 ? sizeof(St) * W : 16),
                         sizeof(r.v));
      } else if (n == W) {
        __builtin_memcpy(r.v, q, sizeof(r.v));
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (e < n) r.v[e] = q[e];
      }
    }
  }
  return r;
}

// The sums v (GATED: gate v and up u) of row i, columns j .. j + W - 1 (n of
// them exist) to what KIND makes of them. j is a multiple of W, which is 8.
// Returns DGRAD's share of the row's dot product.
template <int KIND, class TT, int W, bool VEC>
__device__ __forceinline__ float lin_finish(const LinArgs& p, int64_t i, int64_t j, int n,
                                            float (&v)[W], float (&u)[W], const DropKey& dk,
                                            const LinCols<KIND, W>& col, const LinRow<TT, W>& row) {
  float dot = 0.f;
  if constexpr (KIND == LIN_ACT || KIND == LIN_GATED) {
    const int64_t width = KIND == LIN_GATED ? 2 * p.J : p.J;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      v[e] += col.b[e];
      if constexpr (KIND == LIN_GATED) u[e] += col.bu[e];
    }
    if (p.pre != nullptr) {
      lin_store<F32T, W, VEC>(p.pre, i * width + j, n, v);
      if constexpr (KIND == LIN_GATED) lin_store<F32T, W, VEC>(p.pre, i * width + p.J + j, n, u);
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      v[e] = lin_act<TT>(p.act, v[e]);
      if constexpr (KIND == LIN_GATED) v[e] *= u[e];
    }
  } else if constexpr (KIND == LIN_RES || KIND == LIN_DROP) {
    uint32_t w[4] = {};
    if constexpr (KIND == LIN_DROP) philox(dk, (uint32_t)(j >> 3), (uint32_t)i, w);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      float t = v[e] + col.b[e];
      if constexpr (KIND == LIN_DROP) {
        t = keeps(w, e, p.threshold) ? t * p.alpha : 0.f;
      }
      if (p.scale != nullptr) t *= row.s;
      v[e] = p.res != nullptr ? t + TT::to_f32(row.v[e]) : t;
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] *= p.alpha;
    if constexpr (KIND == LIN_DGRAD) {
      if (p.scale != nullptr) {
        float x[W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          x[e] = TT::to_f32(row.v[e]);
          dot += e < n ? x[e] * v[e] : 0.f;
          v[e] *= row.s;
          x[e] *= row.s;
        }
        if (p.xs != nullptr) lin_store<TT, W, VEC>(p.xs, i * p.J + j, n, x);
      }
      if (p.out == nullptr) return dot;
    }
  }
  lin_store<TT, W, VEC>(p.out, i * p.J + j, n, v);
  return dot;
}

// Sum over the four lanes of a quad.
__device__ __forceinline__ float sum4(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xf, 0xf, true));  // ^ 1
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xf, 0xf, true));  // ^ 2
  return v;
}

// The sums of a wave's (32 FM) x (32 FN) part of a tile to what KIND makes of them, from
// row iw and output column jw on, at any alignment: 32 rows at a time through the wave's LDS,
// so that a lane gets eight consecutive columns (GATED: the first half of the wave's columns
// are gates, the second half their ups). stage(mi, put): calls put(row, column, four sums)
// for the lane's part of the 32 rows mi.
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
template <int FN>
constexpr int LIN_WAVE_FLOATS = 32 * (32 * FN + 4);  // rows of the wave's sums and four more

template <int KIND, class TT, int FM, int FN, typename F>
__device__ __forceinline__ void lin_finish_wave(const LinArgs& p, const F& stage, float* region,
                                                int64_t iw, int64_t jw, int lane) {
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int W = 32 * FN, LD = W + 4, OUT = GATED ? W / 2 : W, NG = OUT / 8;
  const int64_t width = GATED ? 2 * p.J : p.J;
  DropKey dk{};
  if constexpr (KIND == LIN_DROP) dk = load_key(p.key);
#pragma unroll
  for (int mi = 0; mi < FM; ++mi) {
    stage(mi, [&](int row, int column, const f32x4_t& v) {
      *reinterpret_cast<f32x4_t*>(region + row * LD + column) = v;
    });
#pragma unroll 1
    for (int it = lane; it < 32 * NG; it += 64) {
      const int r = it / NG, gi = it % NG;
      const int64_t i = iw + 32 * mi + r, j = jw + 8 * gi;
      const bool live = i < p.I && j < p.J;
      const int n = !live ? 0 : p.J - j < 8 ? (int)(p.J - j) : 8;
      float v[8], u[8] = {}, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = region[r * LD + 8 * gi + e];
        if constexpr (GATED) u[e] = region[r * LD + OUT + 8 * gi + e];
      }
      if (live && p.part != nullptr) {
        const int64_t at = ((int64_t)blockIdx.y * p.I + i) * width + j;
        lin_store<F32T, 8, false>(p.part, at, n, v);
        if constexpr (GATED) lin_store<F32T, 8, false>(p.part, at + p.J, n, u);
      } else if (live) {
        dot = lin_finish<KIND, TT, 8, false>(p, i, j, n, v, u, dk, lin_cols<KIND, 8>(p, j, n),
                                             lin_row<KIND, TT, 8, false>(p, i, j, n));
      }
      if constexpr (KIND == LIN_DGRAD) {
        if (p.dots != nullptr && p.part == nullptr) {
          static_assert(NG % 4 == 0, "four lanes of a run in one row");
          dot = sum4(dot);
          if (live && (lane & 3) == 0)
            p.dots[i * ((p.J + LIN_DOT - 1) / LIN_DOT) + j / LIN_DOT] = dot;
        }
      }
    }
  }
}

}  // namespace

// Operand layouts of a product: NT: A [I, R], B [J, R]. NN: A [I, R], B [R, J].
// TN: A [R, I], B [R, J].
enum { LAY_NT = 0, LAY_NN = 1, LAY_TN = 2 };

// The kernels: fp32, few rows, tiles of the 16-bit matrix instructions, and tiles for any
// alignment.
enum { LIN_F32 = TT_LINEAR_KERNEL_F32, LIN_ROWS = TT_LINEAR_KERNEL_ROWS,
       LIN_T64 = TT_LINEAR_KERNEL_T64, LIN_T128 = TT_LINEAR_KERNEL_T128,
       LIN_T256x128 = TT_LINEAR_KERNEL_T256X128, LIN_T256 = TT_LINEAR_KERNEL_T256,
       LIN_ODD64 = TT_LINEAR_KERNEL_ODD64, LIN_ODD128 = TT_LINEAR_KERNEL_ODD128 };

// fp32 tensors of any size and alignment (linear_f32.hip).
int tt_linear_f32(int kind, const LinArgs& a, hipStream_t s);
// 16-bit matrix instructions on tiles (LIN_T64 ...), for aligned rows of whole 16-byte
// vectors, or (LIN_ODD64, LIN_ODD128) for any (linear_tile.hip).
int tt_linear_tile(int kind, int tile, int dtype, const LinArgs& a, hipStream_t s);
// The same for at most 64 rows of x, NT, aligned (linear_rows.hip).
int tt_linear_rows(int kind, int dtype, const LinArgs& a, hipStream_t s);
