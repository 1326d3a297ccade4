// Dense products with bias, activation, gate, dropout, row scale and residual in
// their epilogue, and their gradients: which kernel runs a product, the joining of
// split reductions, and the passes over rows that the gradients need (gfx950).
#include <algorithm>
#include <initializer_list>

#include "linear.h"

namespace {

inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int L_NT = 256;
constexpr int64_t MAX_BLOCKS = 1 << 20;  // of a pass whose blocks take rows in turn

// ---------------------------------------------------------------------------
// Joins the sums of a split reduction, in the order of the splits. A thread
// takes eight columns; a row's groups of eight are padded to whole LIN_DOT runs
// so that one run's lanes lie together.
// ---------------------------------------------------------------------------
template <int KIND, class TT, bool VEC>
__global__ __launch_bounds__(L_NT) void linear_join_kernel(LinArgs p, int64_t groups) {
  const int64_t idx = (int64_t)blockIdx.x * L_NT + threadIdx.x;
  const int64_t i = idx / groups, j = 8 * (idx % groups);
  const bool live = i < p.I && j < p.J;
  const int n = !live ? 0 : p.J - j < 8 ? (int)(p.J - j) : 8;
  const int64_t width = KIND == LIN_GATED ? 2 * p.J : p.J;
  const LinCols<KIND, 8> cols = lin_cols<KIND, 8>(p, j, n);
  LinRow<TT, 8> row{};
  float v[8] = {}, u[8] = {};
  if (live) {
    row = lin_row<KIND, TT, 8, VEC>(p, i, j, n);
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      const int64_t at = ((int64_t)s * p.I + i) * width + j;
      float t[8];
      lin_load<F32T, 8, VEC>(p.part, at, n, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[e];
      if constexpr (KIND == LIN_GATED) {
        lin_load<F32T, 8, VEC>(p.part, at + p.J, n, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] += t[e];
      }
    }
  }
  DropKey dk{};
  if constexpr (KIND == LIN_DROP) dk = load_key(p.key);
  float dot = 0.f;
  if (live) dot = lin_finish<KIND, TT, 8, VEC>(p, i, j, n, v, u, dk, cols, row);
  if constexpr (KIND == LIN_DGRAD) {
    if (p.dots != nullptr) {
#pragma unroll
      for (int off = 1; off < LIN_DOT / 8; off <<= 1) dot += __shfl_xor(dot, off, 64);
      if (live && j % LIN_DOT == 0)
        p.dots[i * ((p.J + LIN_DOT - 1) / LIN_DOT) + j / LIN_DOT] = dot;
    }
  }
}

bool vectors(const LinArgs& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) |
                       reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.res) |
                       reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.xs) |
                       reinterpret_cast<uintptr_t>(p.pre);
  return at % 16 == 0 && p.lda % 8 == 0 && p.ldb % 8 == 0 && p.J % 8 == 0;
}

template <int KIND, class TT>
int join(const LinArgs& p, hipStream_t s) {
  const int64_t run = LIN_DOT / 8, groups = ((p.J + 7) / 8 + run - 1) / run * run;
  const int64_t blocks = (p.I * groups + L_NT - 1) / L_NT;
  TT_REQUIRE(tt_grid_ok(blocks, L_NT), "linear: grid too large");
  if (vectors(p))
    hipLaunchKernelGGL((linear_join_kernel<KIND, TT, true>), dim3((unsigned)blocks), dim3(L_NT), 0,
                       s, p, groups);
  else
    hipLaunchKernelGGL((linear_join_kernel<KIND, TT, false>), dim3((unsigned)blocks), dim3(L_NT),
                       0, s, p, groups);
  return tt_check_launch("linear_join");
}

template <class TT>
int join_kind(int kind, const LinArgs& p, hipStream_t s) {
  switch (kind) {
    case LIN_ACT: return join<LIN_ACT, TT>(p, s);
    case LIN_GATED: return join<LIN_GATED, TT>(p, s);
    case LIN_RES: return join<LIN_RES, TT>(p, s);
    case LIN_DROP: return join<LIN_DROP, TT>(p, s);
    case LIN_DGRAD: return join<LIN_DGRAD, TT>(p, s);
    default: return join<LIN_PLAIN, TT>(p, s);
  }
}

// Splits of a reduction of R elements into whole runs of 64.
struct Split {
  int splits;
  int64_t run;
};
Split split_of(int64_t R, int64_t wanted) {
  const int64_t runs = (R + 63) / 64;
  if (wanted > runs) wanted = runs;
  if (wanted < 1) wanted = 1;
  if (runs <= 1) return Split{1, 64};
  const int64_t per = ((runs + wanted - 1) / wanted) * 64;
  return Split{(int)((R + per - 1) / per), per};
}

// The kernel that runs a product and how many parts its reduction is split into.
struct Plan {
  int kernel;
  Split split;
};

// The part of an MN-major operand that a block of the 16-bit tiles walks has to
// stay within 32-bit offsets.
int64_t least_splits(int layout, int64_t I, int64_t J, int64_t R) {
  const int64_t ld = layout == LAY_TN ? std::max(I, J) : layout == LAY_NN ? J : 0;
  return std::max<int64_t>((R * ld * 2 + (1ll << 31) - 1) >> 31, 1);
}

// Microseconds of a product of `tiles` tiles in `splits` parts of nkt 64-deep k-tiles. A
// k-tile of a 64-wide tile takes 0.30 us where a CU has one block and 0.5 with two,
// of a 128-wide one 0.62 and 1.0, of a 256-wide one (one block per CU) 0.85 on a few
// CUs and 1.2 on all (the part is then at its power limit); the rest are starts and
// epilogues. Measured (back to back in a graph) / this estimate: 1000 x 704 -> 1024 (256
// tiles of 64) 7.4 / 6.1, 1000 x 1024 -> 1408 (352) 10.5 / 10.8, 2048 x 768 -> 2048 (1024 of
// 64) 16.4 / 15.8, in 256 tiles of 128 13.8 / 11.6, 512 x 2048 -> 7168 (224 of 128) 26.1 /
// 24.0, 1000 rows (448 of 128) 35.0 / 36.2, 2048 rows (224 of 256) 52.2 / 57.0; 24 x 7168 ->
// 4096 in four parts (256 blocks of 64) 16.3 / 19.1, 24 x 2048 -> 7168 (112 of 64) 12.7 / 12.4
// and in four parts 10.6 / 13.1. Over 170 random sizes the choice took 1.03 (forward), 1.01
// (gradient of x) and 1.02 (of the weight) times the best kernel's time in the mean, at
// most 1.2, 1.3 and 1.3 times among the tiles.
// No plan is faster than its operands' bytes at 4.6 TB/s.
double tile_us(int tile, int64_t tiles, int64_t splits, int64_t nkt, int64_t sums, int64_t bytes) {
  const int64_t blocks = tiles * splits, full = blocks / 512, rest = blocks % 512;
  double us;
  if (tile >= LIN_T256x128) {
    const bool sq = tile == LIN_T256;
    const double fill = std::min(1.0, (double)blocks / 256);
    us = (sq ? 8 : 5) + (double)((blocks + 255) / 256) *
                            ((sq ? 12 : 6) + (double)nkt * (sq ? 0.85 + 0.35 * fill : 0.5 + 0.2 * fill));
  } else {
    const bool small = tile == LIN_T64;
    const double one = small ? 0.30 : 0.62, two = small ? 0.5 : 1.0;
    us = (small ? 2.8 : 4.2) + (double)full * (small ? 0.5 : 1.5) +
         (double)nkt * ((double)full * two + (rest == 0 ? 0 : rest <= 256 ? one : two));
  }
  us = std::max(us, 2.8 + (double)bytes / 4.6e6);
  // The parts are written and read again by a second launch.
  return splits == 1 ? us : us + 3 + (double)(splits * sums) * 8 / 6.5e6;
}

// The same of the kernel of few rows: the weight at 4.6 TB/s and, for each block of its
// columns, all of x at 9 TB/s, with fewer than 256 blocks accordingly slower. Measured /
// this estimate: 1 x 7168 -> 2 x 2048 12.5 / 14.7, 16 x 2048 -> 7168 10.5 / 11.1, 24 rows
// 12.8 / 12.8 (the 64-wide tiles, chosen there, 12.7), 24 x 2048 -> 2 x 768 8.5 / 7.9, 64 x
// 7168 -> 2 x 2048 35.5 / 40.4. Bytes alone are too little for a short reduction: 52 x 152 ->
// 2 x 4304 10.6 / 3.0, where the tiles take 4.7.
double rows_us(int64_t blocks, int64_t I, int64_t J, int64_t R) {
  const double work = (double)(J * R) * 2 / 4.6e6 + (double)(blocks * I * R) * 2 / 9e6;
  return 1.5 + work * std::max(1.0, 256.0 / (double)blocks);
}

// `how` of a product: 16-bit on the tiles (FAST) or on those for any alignment (ODD), or fp32.
enum { HOW_F32 = 0, HOW_ODD = 1, HOW_FAST = 2 };

Plan plan_of(int layout, int kind, int64_t I, int64_t J, int64_t R, int how) {
  const int64_t half = kind == LIN_GATED ? 2 : 1, width = half * J;
  auto tiles = [&](int64_t bm, int64_t bn) { return ((I + bm - 1) / bm) * ((width + bn - 1) / bn); };
  if (how == HOW_ODD) {
    // 128-wide tiles where they fill the CUs, else 64-wide ones with the reduction in as
    // many parts as that takes, each at least 512 long. 128 / 64 in us: 4099 x 2051 -> 4099
    // 189 / 226, 4001 x 1201 -> 1703 63 / 65, 2001 x 1201 -> 2001 45 / 46, and 2051 x 515 ->
    // 2051 32 / 29. 64-wide tiles take operands of fewer than eight elements, too.
    const bool big = R >= 8 && tiles(128, 128) >= 256;
    const int64_t want = std::min<int64_t>(256 / std::max<int64_t>(tiles(64, 64), 1), R / 512);
    return Plan{big ? LIN_ODD128 : LIN_ODD64, split_of(R, big ? 1 : std::min<int64_t>(want, 8))};
  }
  if (how == HOW_F32) {
    // Two blocks for each CU, each reduction at least 256 long: 1024 x 4096 -> 1024 in two
    // parts 93 us, whole 97.
    const int64_t want = std::min<int64_t>(512 / std::max<int64_t>(tiles(64, 64), 1), R / 256);
    return Plan{LIN_F32, split_of(R, std::min<int64_t>(want, 32))};
  }
  const int64_t least = least_splits(layout, I, J, R);
  Plan best{LIN_T256, split_of(R, least)};
  double best_us = 1e30;
  if (layout == LAY_NT && I <= 64) {
    best = Plan{LIN_ROWS, split_of(R, 1)};
    best_us = rows_us((width + 15) / 16, I, width, R);
  }
  for (int tile : {LIN_T64, LIN_T128, LIN_T256x128, LIN_T256}) {
    const int64_t bm = tile == LIN_T64 ? 64 : tile == LIN_T128 ? 128 : 256;
    const int64_t bn = tile == LIN_T64 ? 64 : tile == LIN_T256 ? 256 : 128;
    for (int64_t want = least; want <= std::max<int64_t>(least, 16); want *= 2) {
      const Split sp = split_of(R, want);
      if (sp.splits > least && sp.run < 256) break;
      const double us = tile_us(tile, tiles(bm, bn), sp.splits, sp.run / 64, I * width,
                                (I + width) * R * 2);
      if (us < best_us) {
        best_us = us;
        best = Plan{tile, sp};
      }
    }
  }
  return best;
}

size_t part_bytes(int kind, int64_t I, int64_t J, int64_t splits) {
  return splits <= 1 ? 0 : (size_t)splits * I * J * (kind == LIN_GATED ? 2 : 1) * 4;
}
size_t dots_bytes(int64_t I, int64_t J) {
  return (((size_t)I * ((J + LIN_DOT - 1) / LIN_DOT) * 4) + 255) / 256 * 256;
}

// How the sizes of a product may run: the 16-bit tiles want rows of whole 16-byte
// vectors and tiles within reach of a 32-bit offset (a gated tile's columns lie half
// the weight apart); those for any alignment have 64-bit addresses.
int how_sizes(int layout, int kind, int dtype, int64_t I, int64_t J, int64_t R) {
  if (dtype == TT_F32) return HOW_F32;
  if (R == 0) return HOW_ODD;
  const bool a_ok = layout == LAY_TN ? I % 8 == 0 : R % 8 == 0;
  const bool b_ok = layout == LAY_NT ? R % 8 == 0 : J % 8 == 0;
  if (!a_ok || !b_ok || J % 8 != 0) return HOW_ODD;
  const int64_t row = 2 * std::max(J, layout == LAY_TN ? I : R);  // of an operand or of C
  const bool near = row * 256 < (1ll << 31) &&
                    (kind != LIN_GATED || (J + 256) * R * 2 < (1ll << 31));
  return near ? HOW_FAST : HOW_ODD;
}

int run_product(int layout, int kind, int dtype, LinArgs p, void* ws, size_t ws_bytes,
                hipStream_t s) {
  int how = how_sizes(layout, kind, dtype, p.I, p.J, p.R);
  if (how == HOW_FAST && !vectors(p)) how = HOW_ODD;
  Plan pl = plan_of(layout, kind, p.I, p.J, p.R, how);
  if (part_bytes(kind, p.I, p.J, pl.split.splits) > ws_bytes) {
    // Without room for the parts: a whole reduction, on the kernel for any alignment
    // where the tiles cannot walk it.
    if (how == HOW_FAST && least_splits(layout, p.I, p.J, p.R) > 1)
      pl = plan_of(layout, kind, p.I, p.J, p.R, HOW_ODD);
    pl.split = split_of(p.R, 1);
  }
  const Split sp = pl.split;
  p.splits = sp.splits;
  p.rsplit = sp.run;
  p.part = sp.splits > 1 ? static_cast<float*>(ws) : nullptr;
  const int rc = pl.kernel == LIN_F32    ? tt_linear_f32(kind, p, s)
                 : pl.kernel == LIN_ROWS ? tt_linear_rows(kind, dtype, p, s)
                                         : tt_linear_tile(kind, pl.kernel, dtype, p, s);
  if (rc != TT_OK || p.part == nullptr) return rc;
  switch (dtype) {
    case TT_BF16: return join_kind<BF16T>(kind, p, s);
    case TT_F16: return join_kind<F16T>(kind, p, s);
    default: return join_kind<F32T>(kind, p, s);
  }
}

// ---------------------------------------------------------------------------
// Passes over rows, bound by memory: the gated activation's gradient of 8192 x 14336 in
// 350 us, 4.7 TB/s of dy, the fp32 `pre` and da. A block takes 256 columns (32 lanes of
// eight) of a chunk of rows, eight rows at a time; column sums are added in a fixed order: a thread's
// rows, the block's eight threads of a column, then the chunks.
// ---------------------------------------------------------------------------
constexpr int P_COLS = 256, P_ROWS = 8;

__device__ __forceinline__ void chunk_sums(const float (&sum)[8], float* part, int64_t width,
                                           int64_t j, int64_t J, float* lds) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) lds[ty * P_COLS + 8 * tx + e] = sum[e];
  __syncthreads();
  const int c = threadIdx.x;
  float t = 0.f;
#pragma unroll
  for (int y = 0; y < P_ROWS; ++y) t += lds[y * P_COLS + c];
  const int64_t col = j - 8 * tx + c;
  if (col < J) part[(int64_t)blockIdx.x * width + col] = t;
}

// da of y = act(a) (GATED: act(a_g) a_u) from dy and the fp32 a, rounded to the
// tensor's type, and the column sums of the unrounded da.
template <class TT, bool GATED, bool VEC>
__global__ __launch_bounds__(L_NT) void linear_act_bwd_kernel(
    const typename TT::storage* __restrict__ dy, const float* __restrict__ pre,
    typename TT::storage* __restrict__ da, float* __restrict__ part, int64_t rows, int64_t J,
    int64_t per, int act) {
  __shared__ float lds[P_ROWS * P_COLS];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.y * P_COLS + 8 * tx, width = GATED ? 2 * J : J;
  const int64_t r0 = (int64_t)blockIdx.x * per, r1 = r0 + per < rows ? r0 + per : rows;
  const int n = j >= J ? 0 : J - j < 8 ? (int)(J - j) : 8;
  float sum[8] = {}, sum_u[8] = {};
  if (n > 0) {
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += P_ROWS) {
      float d[8], a[8], o[8];
      lin_load<TT, 8, VEC>(dy, r * J + j, n, d);
      lin_load<F32T, 8, VEC>(pre, r * width + j, n, a);
      if constexpr (GATED) {
        float u[8], ou[8];
        lin_load<F32T, 8, VEC>(pre, r * width + J + j, n, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float value, slope;
          lin_act_grad<TT>(act, a[e], value, slope);
          o[e] = d[e] * u[e] * slope;
          ou[e] = d[e] * value;
          sum[e] += o[e];
          sum_u[e] += ou[e];
        }
        lin_store<TT, 8, VEC>(da, r * width + J + j, n, ou);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float value, slope;
          lin_act_grad<TT>(act, a[e], value, slope);
          o[e] = d[e] * slope;
          sum[e] += o[e];
        }
      }
      lin_store<TT, 8, VEC>(da, r * width + j, n, o);
    }
  }
  if (part == nullptr) return;
  chunk_sums(sum, part, width, j, J, lds);
  if constexpr (GATED) chunk_sums(sum_u, part + J, width, j, J, lds);
}

// g = dy with the dropped elements cleared (MASK), and the column sums of
// scale[i] * g (scale may be null) where part is given.
template <class TT, bool MASK, bool VEC>
__global__ __launch_bounds__(L_NT) void linear_res_bwd_kernel(
    const typename TT::storage* __restrict__ dy, const void* __restrict__ scale, int scale_dt,
    uint32_t threshold, const int64_t* __restrict__ key, typename TT::storage* __restrict__ g,
    float* __restrict__ part, int64_t rows, int64_t J, int64_t per) {
  __shared__ float lds[P_ROWS * P_COLS];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.y * P_COLS + 8 * tx;
  const int64_t r0 = (int64_t)blockIdx.x * per, r1 = r0 + per < rows ? r0 + per : rows;
  const int n = j >= J ? 0 : J - j < 8 ? (int)(J - j) : 8;
  DropKey dk{};
  if constexpr (MASK) dk = load_key(key);
  float sum[8] = {};
  if (n > 0) {
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += P_ROWS) {
      float d[8];
      lin_load<TT, 8, VEC>(dy, r * J + j, n, d);
      if constexpr (MASK) {
        uint32_t w[4];
        philox(dk, (uint32_t)(j >> 3), (uint32_t)r, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = keeps(w, e, threshold) ? d[e] : 0.f;
        lin_store<TT, 8, VEC>(g, r * J + j, n, d);
      }
      if (part != nullptr) {
        const float s = scale != nullptr ? load_as_f32(scale, scale_dt, r) : 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += s * d[e];
      }
    }
  }
  if (part != nullptr) chunk_sums(sum, part, J, j, J, lds);
}

// out[j] = alpha * the chunks' sums of column j: 32 columns per block, eight
// threads to each.
__global__ __launch_bounds__(L_NT) void linear_colsum_kernel(const float* __restrict__ part,
                                                             int64_t chunks, int64_t width,
                                                             float alpha, void* __restrict__ out,
                                                             int dt) {
  __shared__ float lds[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.x * 32 + tx;
  float t = 0.f;
  if (j < width) {
#pragma unroll 4
    for (int64_t c = ty; c < chunks; c += 8) t += part[c * width + j];
  }
  lds[ty][tx] = t;
  __syncthreads();
  if (ty != 0 || j >= width) return;
#pragma unroll
  for (int y = 1; y < 8; ++y) t += lds[y][tx];
  store_from_f32(out, dt, j, alpha * t);
}

// out[i] = sum over j of g[i, j] * bias[j], one wave per row at a time.
__global__ __launch_bounds__(L_NT) void linear_rowdot_kernel(const void* __restrict__ g, int dtype,
                                                             const void* __restrict__ bias,
                                                             int bias_dt, int64_t rows, int64_t J,
                                                             float* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows; i += 4ll * gridDim.x) {
    float t = 0.f;
    for (int64_t j = threadIdx.x & 63; j < J; j += 64)
      t += load_as_f32(g, dtype, i * J + j) * load_as_f32(bias, bias_dt, j);
    t = wave_sum(t);
    if ((threadIdx.x & 63) == 0) out[i] = t;
  }
}

// out[i] = the dots of row i, in order, + alpha * extra[i].
__global__ __launch_bounds__(L_NT) void linear_rowsum_kernel(const float* __restrict__ dots, int nd,
                                                             const float* __restrict__ extra,
                                                             float alpha, int64_t rows,
                                                             void* __restrict__ out, int dt) {
  const int64_t i = (int64_t)blockIdx.x * L_NT + threadIdx.x;
  if (i >= rows) return;
  float t = 0.f;
#pragma unroll 8
  for (int d = 0; d < nd; ++d) t += dots[i * nd + d];
  if (extra != nullptr) t += alpha * extra[i];
  store_from_f32(out, dt, i, t);
}

// Chunks of rows of a pass over rows x J: about 1024 blocks, whole runs of
// P_ROWS rows.
int64_t chunk_rows(int64_t rows, int64_t J) {
  const int64_t ct = (J + P_COLS - 1) / P_COLS;
  int64_t chunks = 1024 / (ct > 0 ? ct : 1);
  if (chunks < 1) chunks = 1;
  int64_t per = (rows + chunks - 1) / chunks;
  per = (per + P_ROWS - 1) / P_ROWS * P_ROWS;
  return per > 0 ? per : P_ROWS;
}

int sizes_ok(int dtype, int64_t m, int64_t k, int64_t n) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16,
             "linear: tensors must be f32, bf16 or f16");
  TT_REQUIRE(m >= 0 && k >= 0 && n >= 0 && m < (1ll << 31) && k < (1ll << 31) && n < (1ll << 30),
             "linear: bad sizes (%lld x %lld x %lld)", (long long)m, (long long)k, (long long)n);
  return TT_OK;
}
int vector_ok(const char* what, const void* p, int dtype) {
  TT_REQUIRE(p == nullptr || dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16,
             "linear: %s must be f32, bf16 or f16", what);
  return TT_OK;
}

#define TT_TRY(call)            \
  do {                          \
    const int rc_ = (call);     \
    if (rc_ != TT_OK) return rc_; \
  } while (0)

// A pointer that the call reads or writes (`used`) has to be there, a workspace that it
// takes anything of has to be there and aligned: the kernels get addresses and cannot tell.
int pointer_ok(const char* what, const void* p, bool used) {
  TT_REQUIRE(p != nullptr || !used, "linear: null pointer (%s)", what);
  return TT_OK;
}
int workspace_ok(const void* ws, size_t bytes) {
  TT_TRY(pointer_ok("the workspace", ws, bytes != 0));
  TT_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 256 == 0,
             "linear: the workspace must be aligned to 256 bytes");
  return TT_OK;
}

template <typename F>
int typed(int dtype, F f) {
  switch (dtype) {
    case TT_BF16: return f(BF16T{});
    case TT_F16: return f(F16T{});
    default: return f(F32T{});
  }
}

bool all_aligned(std::initializer_list<const void*> ps) {
  uintptr_t at = 0;
  for (const void* p : ps) at |= reinterpret_cast<uintptr_t>(p);
  return at % 16 == 0;
}

// Bytes of the parts of a product, for the larger of its two plans: which one runs also
// depends on the addresses.
size_t parts_of(int layout, int kind, int dtype, int64_t I, int64_t J, int64_t R) {
  const int how = how_sizes(layout, kind, dtype, I, J, R);
  int64_t splits = plan_of(layout, kind, I, J, R, how).split.splits;
  if (how == HOW_FAST) splits = std::max<int64_t>(splits, plan_of(layout, kind, I, J, R, HOW_ODD).split.splits);
  return part_bytes(kind, I, J, splits);
}
size_t round256(size_t bytes) { return (bytes + 255) / 256 * 256; }

// dx = row_scale (alpha g w) and what goes with it (linear.h's DGRAD).
int data_gradient(const void* g, const void* w, const void* x, const void* scale, int scale_dt,
                  int dtype, int64_t m, int64_t k, int64_t n, float alpha, void* dx, void* xs,
                  float* dots, void* ws, size_t ws_bytes, hipStream_t s) {
  LinArgs p{};
  p.a = g;
  p.b = w;
  p.out = dx;
  p.I = m;
  p.J = p.ldb = k;
  p.R = p.lda = n;
  p.scale = scale;
  p.scale_dt = scale_dt;
  p.alpha = alpha;
  p.x = x;
  p.xs = xs;
  p.dots = dots;
  return m == 0 || k == 0 ? TT_OK : run_product(LAY_NN, LIN_DGRAD, dtype, p, ws, ws_bytes, s);
}

// dw [n, k] = alpha g^T x.
int weight_gradient(const void* g, const void* x, int dtype, int64_t m, int64_t k, int64_t n,
                    float alpha, void* dw, void* ws, size_t ws_bytes, hipStream_t s) {
  LinArgs p{};
  p.a = g;
  p.b = x;
  p.out = dw;
  p.I = p.lda = n;
  p.J = p.ldb = k;
  p.R = m;
  p.alpha = alpha;
  return n == 0 || k == 0 ? TT_OK : run_product(LAY_TN, LIN_PLAIN, dtype, p, ws, ws_bytes, s);
}

// Passes over the rows of [m, n]: chunks of rows, tiles of columns.
struct RowPass {
  int64_t per, chunks, tiles;
  RowPass(int64_t m, int64_t n)
      : per(chunk_rows(m, n)), chunks((m + per - 1) / per), tiles((n + P_COLS - 1) / P_COLS) {}
  dim3 grid() const { return dim3((unsigned)chunks, (unsigned)tiles); }
};

int column_sums(const float* part, const RowPass& rp, int64_t width, float alpha, void* out, int dt,
                hipStream_t s) {
  hipLaunchKernelGGL(linear_colsum_kernel, dim3((unsigned)((width + 31) / 32)), dim3(L_NT), 0, s,
                     part, rp.chunks, width, alpha, out, dt);
  return tt_check_launch("linear_colsum");
}

// A workspace handed out in 256-byte aligned pieces.
struct Pieces {
  char* at;
  size_t left;
  void* take(size_t bytes) {
    const size_t n = round256(bytes);
    if (n > left) return nullptr;
    char* p = at;
    at += n;
    left -= n;
    return p;
  }
};


}  // namespace

extern "C" size_t tt_linear_workspace(int32_t op, int dtype, int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || k < 0 || n <= 0) return 0;
  switch (op) {
    case TT_LINEAR_ACT: return parts_of(LAY_NT, LIN_ACT, dtype, m, n, k);
    case TT_LINEAR_GATED: return parts_of(LAY_NT, LIN_GATED, dtype, m, n, k);
    case TT_LINEAR_RESIDUAL: return parts_of(LAY_NT, LIN_RES, dtype, m, n, k);
    default: return 0;
  }
}

extern "C" int tt_linear_plan(int32_t op, int32_t pass, int dtype, int64_t m, int64_t k, int64_t n,
                              int32_t aligned) {
  if (op < TT_LINEAR_ACT || op > TT_LINEAR_RESIDUAL || pass < 0 || pass > 2 || m < 0 || k < 0 ||
      n < 0 || (dtype != TT_F32 && dtype != TT_BF16 && dtype != TT_F16))
    return -1;
  const bool gated = op == TT_LINEAR_GATED;
  const int64_t width = gated ? 2 * n : n;
  const int layout = pass == 0 ? LAY_NT : pass == 1 ? LAY_NN : LAY_TN;
  const int kind = pass == 1   ? LIN_DGRAD
                   : pass == 2 ? LIN_PLAIN
                   : gated     ? LIN_GATED
                               : LIN_ACT;  // RES's and DROP's plan as well
  const int64_t I = pass == 2 ? width : m, J = pass == 0 ? n : k;
  const int64_t R = pass == 0 ? k : pass == 1 ? width : m;
  if (I == 0 || J == 0) return -1;
  int how = how_sizes(layout, kind, dtype, I, J, R);
  if (how == HOW_FAST && !aligned) how = HOW_ODD;
  const Plan pl = plan_of(layout, kind, I, J, R, how);
  return pl.kernel + 256 * pl.split.splits;
}

extern "C" int tt_linear_act_fwd(const void* x, const void* w, const void* bias, int bias_dtype,
                                 int dtype, int64_t m, int64_t k, int64_t n, int32_t act,
                                 int32_t gated, float* pre, void* y, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  TT_TRY(sizes_ok(dtype, m, k, n));
  TT_TRY(vector_ok("the bias", bias, bias_dtype));
  TT_REQUIRE(act >= ACT_NONE && act <= ACT_GELU, "linear: unknown activation %d", act);
  if (m == 0 || n == 0) return TT_OK;
  TT_TRY(pointer_ok("x", x, k > 0));
  TT_TRY(pointer_ok("w", w, k > 0));
  TT_TRY(pointer_ok("y", y, true));
  TT_TRY(workspace_ok(workspace, workspace_bytes));
  LinArgs p{};
  p.a = x;
  p.b = w;
  p.out = y;
  p.I = m;
  p.J = n;
  p.R = p.lda = p.ldb = k;
  p.bias = bias;
  p.bias_dt = bias_dtype;
  p.act = act;
  p.pre = pre;
  return run_product(LAY_NT, gated ? LIN_GATED : LIN_ACT, dtype, p, workspace, workspace_bytes,
                     S(stream));
}

// Workspace: da where there is an activation, then the parts of one step at a time.
extern "C" size_t tt_linear_act_bwd_workspace(int dtype, int64_t m, int64_t k, int64_t n,
                                              int32_t act, int32_t gated) {
  if (m < 0 || k < 0 || n < 0) return 0;
  const int64_t width = gated ? 2 * n : n;
  const size_t sums = (size_t)RowPass(m, n).chunks * width * 4;
  const size_t parts = std::max(parts_of(LAY_NN, LIN_DGRAD, dtype, m, k, width),
                                parts_of(LAY_TN, LIN_PLAIN, dtype, width, k, m));
  const bool own = act != ACT_NONE || gated;
  return (own ? round256((size_t)m * width * tt_elem_size(dtype)) : 0) +
         round256(std::max(sums, parts));
}

extern "C" int tt_linear_act_bwd(const void* dy, const void* x, const void* w, const float* pre,
                                 int dtype, int64_t m, int64_t k, int64_t n, int32_t act,
                                 int32_t gated, void* dx, void* dw, void* dbias, int bias_dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  TT_TRY(sizes_ok(dtype, m, k, n));
  TT_TRY(vector_ok("the bias", dbias, bias_dtype));
  TT_REQUIRE(act >= ACT_NONE && act <= ACT_GELU, "linear: unknown activation %d", act);
  const bool own = act != ACT_NONE || gated;
  const size_t needed = tt_linear_act_bwd_workspace(dtype, m, k, n, act, gated);
  TT_REQUIRE(workspace_bytes >= needed, "linear_act_bwd: the workspace is too small");
  if (dx == nullptr && dw == nullptr && dbias == nullptr) return TT_OK;
  const bool products = m > 0 && k > 0 && n > 0;
  TT_TRY(pointer_ok("dy", dy, m > 0 && n > 0));
  TT_TRY(pointer_ok("pre", pre, own && m > 0 && n > 0));
  TT_TRY(pointer_ok("w", w, dx != nullptr && products));
  TT_TRY(pointer_ok("x", x, dw != nullptr && products));
  TT_TRY(workspace_ok(workspace, needed));
  const int64_t width = gated ? 2 * n : n;
  Pieces ws{static_cast<char*>(workspace), workspace_bytes};
  void* const da = own ? ws.take((size_t)m * width * tt_elem_size(dtype)) : nullptr;
  const RowPass rp(m, n);
  TT_REQUIRE(rp.tiles <= 65535, "linear: too many columns");
  float* const part = dbias != nullptr ? reinterpret_cast<float*>(ws.at) : nullptr;
  if (m > 0 && n > 0 && (own || dbias != nullptr)) {
    const bool vec = n % 8 == 0 && all_aligned({dy, pre});
    TT_TRY(typed(dtype, [&](auto tt) {
      typedef decltype(tt) TT;
      typedef typename TT::storage St;
      if (!own) {  // the bias's sums alone
        auto go = [&](auto kernel) {
          hipLaunchKernelGGL(kernel, rp.grid(), dim3(L_NT), 0, S(stream), static_cast<const St*>(dy),
                             nullptr, 0, 0u, nullptr, nullptr, part, m, n, rp.per);
          return tt_check_launch("linear_res_bwd");
        };
        return vec ? go(&linear_res_bwd_kernel<TT, false, true>)
                   : go(&linear_res_bwd_kernel<TT, false, false>);
      }
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, rp.grid(), dim3(L_NT), 0, S(stream), static_cast<const St*>(dy),
                           pre, static_cast<St*>(da), part, m, n, rp.per, (int)act);
        return tt_check_launch("linear_act_bwd");
      };
      if (gated)
        return vec ? go(&linear_act_bwd_kernel<TT, true, true>)
                   : go(&linear_act_bwd_kernel<TT, true, false>);
      return vec ? go(&linear_act_bwd_kernel<TT, false, true>)
                 : go(&linear_act_bwd_kernel<TT, false, false>);
    }));
  }
  if (dbias != nullptr && n > 0)
    TT_TRY(column_sums(part, rp, width, 1.0f, dbias, bias_dtype, S(stream)));
  const void* const g = own ? da : dy;
  if (dx != nullptr)
    TT_TRY(data_gradient(g, w, nullptr, nullptr, 0, dtype, m, k, width, 1.0f, dx, nullptr, nullptr,
                         ws.at, ws.left, S(stream)));
  if (dw != nullptr)
    TT_TRY(weight_gradient(g, x, dtype, m, k, width, 1.0f, dw, ws.at, ws.left, S(stream)));
  return TT_OK;
}

extern "C" int tt_linear_residual_fwd(const void* x, const void* w, const void* bias,
                                      int bias_dtype, const void* residual, const void* row_scale,
                                      int scale_dtype, int dtype, int64_t m, int64_t k, int64_t n,
                                      int32_t threshold, const int64_t* key, void* y,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  TT_TRY(sizes_ok(dtype, m, k, n));
  TT_TRY(vector_ok("the bias", bias, bias_dtype));
  TT_TRY(vector_ok("the row scale", row_scale, scale_dtype));
  TT_REQUIRE(threshold >= 0 && threshold <= 65536, "linear: the threshold must be in [0, 65536]");
  TT_REQUIRE(threshold == 0 || key != nullptr, "linear: dropout without a key");
  if (m == 0 || n == 0) return TT_OK;
  TT_TRY(pointer_ok("x", x, k > 0));
  TT_TRY(pointer_ok("w", w, k > 0));
  TT_TRY(pointer_ok("y", y, true));
  TT_TRY(workspace_ok(workspace, workspace_bytes));
  LinArgs p{};
  p.a = x;
  p.b = w;
  p.out = y;
  p.I = m;
  p.J = n;
  p.R = p.lda = p.ldb = k;
  p.bias = bias;
  p.bias_dt = bias_dtype;
  p.res = residual;
  p.scale = row_scale;
  p.scale_dt = scale_dtype;
  p.threshold = (uint32_t)threshold;
  p.alpha = keep_inverse(threshold);
  p.key = key;
  return run_product(LAY_NT, threshold != 0 ? LIN_DROP : LIN_RES, dtype, p, workspace,
                     workspace_bytes, S(stream));
}

// Workspace: dy without its dropped elements; with a row scale the scaled rows, the dot
// products of its gradient and the bias's part of it; then the parts of one step at
// a time.
extern "C" size_t tt_linear_residual_bwd_workspace(int dtype, int64_t m, int64_t k, int64_t n,
                                                   int32_t scaled, int32_t dropped) {
  if (m < 0 || k < 0 || n < 0) return 0;
  const size_t es = tt_elem_size(dtype);
  const size_t sums = (size_t)RowPass(m, n).chunks * n * 4;
  const size_t parts = std::max(parts_of(LAY_NN, LIN_DGRAD, dtype, m, k, n),
                                parts_of(LAY_TN, LIN_PLAIN, dtype, n, k, m));
  return (dropped ? round256((size_t)m * n * es) : 0) +
         (scaled ? round256((size_t)m * k * es) + dots_bytes(m, k) + round256((size_t)m * 4) : 0) +
         round256(std::max(sums, parts));
}

extern "C" int tt_linear_residual_bwd(const void* dy, const void* x, const void* w,
                                      const void* bias, int bias_dtype, const void* row_scale,
                                      int scale_dtype, int dtype, int64_t m, int64_t k, int64_t n,
                                      int32_t threshold, const int64_t* key, void* dx, void* dw,
                                      void* dbias, void* dscale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  TT_TRY(sizes_ok(dtype, m, k, n));
  TT_TRY(vector_ok("the bias", bias != nullptr ? bias : dbias, bias_dtype));
  TT_TRY(vector_ok("the row scale", row_scale, scale_dtype));
  TT_REQUIRE(threshold >= 0 && threshold <= 65536, "linear: the threshold must be in [0, 65536]");
  TT_REQUIRE(threshold == 0 || key != nullptr, "linear: dropout without a key");
  TT_REQUIRE(row_scale != nullptr || dscale == nullptr,
             "linear_residual_bwd: the scale's gradient needs a row scale");
  const size_t needed =
      tt_linear_residual_bwd_workspace(dtype, m, k, n, row_scale != nullptr, threshold != 0);
  TT_REQUIRE(workspace_bytes >= needed, "linear_residual_bwd: the workspace is too small");
  if (dx == nullptr && dw == nullptr && dbias == nullptr && dscale == nullptr) return TT_OK;
  // With a row scale the weight's gradient takes the rows that the product for dx scales.
  const bool back = dx != nullptr || dscale != nullptr || (row_scale != nullptr && dw != nullptr);
  TT_TRY(pointer_ok("dy", dy, m > 0 && n > 0));
  TT_TRY(pointer_ok("w", w, back && m > 0 && k > 0 && n > 0));
  TT_TRY(pointer_ok("x", x, (dw != nullptr || dscale != nullptr) && m > 0 && k > 0));
  TT_TRY(workspace_ok(workspace, needed));
  const size_t es = tt_elem_size(dtype);
  const float alpha = keep_inverse(threshold);
  Pieces ws{static_cast<char*>(workspace), workspace_bytes};
  void* const kept = threshold != 0 ? ws.take((size_t)m * n * es) : nullptr;
  void* const rows = row_scale != nullptr ? ws.take((size_t)m * k * es) : nullptr;
  float* const dots = row_scale != nullptr ? static_cast<float*>(ws.take(dots_bytes(m, k))) : nullptr;
  float* const extra = row_scale != nullptr ? static_cast<float*>(ws.take((size_t)m * 4)) : nullptr;
  if (n > 0) {
    const RowPass rp(m, n);
    TT_REQUIRE(rp.tiles <= 65535, "linear: too many columns");
    float* const part = dbias != nullptr ? reinterpret_cast<float*>(ws.at) : nullptr;
    if (m > 0 && (threshold != 0 || dbias != nullptr)) {
      const bool vec = n % 8 == 0 && all_aligned({dy});
      TT_TRY(typed(dtype, [&](auto tt) {
        typedef decltype(tt) TT;
        typedef typename TT::storage St;
        auto go = [&](auto kernel) {
          hipLaunchKernelGGL(kernel, rp.grid(), dim3(L_NT), 0, S(stream), static_cast<const St*>(dy),
                             row_scale, scale_dtype, (uint32_t)threshold, key,
                             static_cast<St*>(kept), part, m, n, rp.per);
          return tt_check_launch("linear_res_bwd");
        };
        if (threshold != 0)
          return vec ? go(&linear_res_bwd_kernel<TT, true, true>)
                     : go(&linear_res_bwd_kernel<TT, true, false>);
        return vec ? go(&linear_res_bwd_kernel<TT, false, true>)
                   : go(&linear_res_bwd_kernel<TT, false, false>);
      }));
    }
    if (dbias != nullptr) TT_TRY(column_sums(part, rp, n, alpha, dbias, bias_dtype, S(stream)));
  }
  const void* const g = threshold != 0 ? kept : dy;
  // The weight's gradient takes the rows times their scale, which the pass for dx writes;
  // that pass runs for them, or for the scale's gradient, where dx is not wanted.
  const bool scaled_rows = row_scale != nullptr && dw != nullptr;
  if (back)
    TT_TRY(data_gradient(g, w, x, row_scale, scale_dtype, dtype, m, k, n, alpha, dx,
                         scaled_rows ? rows : nullptr, dscale != nullptr ? dots : nullptr, ws.at,
                         ws.left, S(stream)));
  if (dscale != nullptr && m > 0) {
    if (bias != nullptr) {
      const int64_t blocks = std::min<int64_t>((m + 3) / 4, MAX_BLOCKS);
      hipLaunchKernelGGL(linear_rowdot_kernel, dim3((unsigned)blocks), dim3(L_NT), 0, S(stream), g,
                         dtype, bias, bias_dtype, m, n, extra);
      TT_TRY(tt_check_launch("linear_rowdot"));
    }
    hipLaunchKernelGGL(linear_rowsum_kernel, dim3((unsigned)((m + L_NT - 1) / L_NT)), dim3(L_NT), 0,
                       S(stream), dots, (int)((k + LIN_DOT - 1) / LIN_DOT),
                       bias != nullptr ? extra : nullptr, alpha, m, dscale, scale_dtype);
    TT_TRY(tt_check_launch("linear_rowsum"));
  }
  if (dw != nullptr)
    TT_TRY(weight_gradient(g, scaled_rows ? rows : x, dtype, m, k, n, alpha, dw, ws.at, ws.left,
                           S(stream)));
  return TT_OK;
}
