// Dropout with a counter-based mask (gfx950): y = keep x / (share kept), the
// mask of element (row, col) as in philox.h, so nothing but the key is stored
// for the backward, which is the same call on the gradient. A dropped element is
// 0 whatever it held (infinities and NaN included).
//
// One read and one write, 131072 x 2048 bf16 in 207 us: 5.2 TB/s, the rate of a copy. The
// ten rounds of a group of eight are about 80 instructions, four rows of them in flight
// per thread: under the time of their memory accesses. Widths off eight elements and
// unaligned rows are loaded one element at a time: 131072 x 2047 in 291 us.
#include "linear.h"

namespace {

constexpr int DR_NT = 256;
constexpr int DR_ROWS = 4;  // rows in flight per thread
constexpr int64_t DR_BLOCKS = 1 << 20;  // along rows; with more rows they take them in turn

// Lanes along the groups of eight columns (L of a block's 256 threads, a power
// of two), the others along rows; a thread keeps its group and walks rows.
template <class TT, bool VEC>
__global__ __launch_bounds__(DR_NT) void dropout_kernel(const typename TT::storage* __restrict__ x,
                                                        typename TT::storage* __restrict__ y,
                                                        int64_t rows, int64_t cols, int L,
                                                        uint32_t threshold, float inv,
                                                        const int64_t* __restrict__ key) {
  typedef typename TT::storage St;
  const DropKey dk = load_key(key);
  const int64_t group = (int64_t)blockIdx.y * L + (threadIdx.x & (L - 1));
  const int64_t c0 = 8 * group;
  if (c0 >= cols) return;
  const int64_t step = (int64_t)gridDim.x * (DR_NT / L);
  const int64_t first = (int64_t)blockIdx.x * (DR_NT / L) + threadIdx.x / L;
  for (int64_t r0 = first; r0 < rows; r0 += step * DR_ROWS) {
    St v[DR_ROWS][8];
#pragma unroll
    for (int q = 0; q < DR_ROWS; ++q) {
      const int64_t r = r0 + q * step;
      if (r >= rows) break;
      if constexpr (VEC) {
        __builtin_memcpy(v[q], x + r * cols + c0, sizeof(v[q]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + j < cols) v[q][j] = x[r * cols + c0 + j];
      }
    }
#pragma unroll
    for (int q = 0; q < DR_ROWS; ++q) {
      const int64_t r = r0 + q * step;
      if (r >= rows) break;
      uint32_t w[4];
      philox(dk, (uint32_t)group, (uint32_t)r, w);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = keeps(w, j, threshold) ? TT::to_f32(v[q][j]) * inv : 0.f;
      const int n = cols - c0 < 8 ? (int)(cols - c0) : 8;
      lin_store<TT, 8, VEC>(y, r * cols + c0, n, o);
    }
  }
}

template <class TT>
int launch(const void* x, void* y, int64_t rows, int64_t cols, int32_t threshold,
           const int64_t* key, hipStream_t s) {
  typedef typename TT::storage St;
  const int64_t groups = (cols + 7) / 8;
  int L = 1;
  while (L < DR_NT && L < groups) L *= 2;
  const int64_t gy = (groups + L - 1) / L;
  int64_t gx = (rows + (DR_NT / L) * DR_ROWS - 1) / ((DR_NT / L) * DR_ROWS);
  TT_REQUIRE(gy <= 65535, "dropout: too many columns (%lld)", (long long)cols);
  if (gx > DR_BLOCKS) gx = DR_BLOCKS;
  const bool vec = cols % 8 == 0 && ((reinterpret_cast<uintptr_t>(x) |
                                      reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(DR_NT);
  const float inv = keep_inverse(threshold);
  if (vec)
    hipLaunchKernelGGL((dropout_kernel<TT, true>), grid, block, 0, s, static_cast<const St*>(x),
                       static_cast<St*>(y), rows, cols, L, (uint32_t)threshold, inv, key);
  else
    hipLaunchKernelGGL((dropout_kernel<TT, false>), grid, block, 0, s, static_cast<const St*>(x),
                       static_cast<St*>(y), rows, cols, L, (uint32_t)threshold, inv, key);
  return tt_check_launch("dropout");
}

}  // namespace

extern "C" int tt_dropout(const void* x, int dtype, int64_t rows, int64_t cols, int32_t threshold,
                          const int64_t* key, void* y, void* stream) {
  TT_REQUIRE(rows >= 0 && cols >= 0 && rows < (1ll << 32), "dropout: bad sizes");
  TT_REQUIRE(threshold >= 0 && threshold <= 65536, "dropout: the threshold must be in [0, 65536]");
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16,
             "dropout: x must be f32, bf16 or f16");
  if (rows == 0 || cols == 0) return TT_OK;
  TT_REQUIRE(x != nullptr && y != nullptr && key != nullptr, "dropout: null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case TT_BF16: return launch<BF16T>(x, y, rows, cols, threshold, key, s);
    case TT_F16: return launch<F16T>(x, y, rows, cols, threshold, key, s);
    default: return launch<F32T>(x, y, rows, cols, threshold, key, s);
  }
}
