// Dense product with an epilogue for few rows (gfx950): C [I, J] = x w^T, I at
// most 64, 16-bit x [I, R] and w [rows, R]: the decode of one or some sequences.
//
// Such a call reads the weight once and is bound by that stream. A block takes 16
// rows of the weight and all of x, and its eight waves split the reduction
// among them, so that every CU streams with a few blocks however few columns there
// are, with no second launch to join parts. Operands go from memory to registers
// in the layout of the 16x16x32 products (a lane's 16 bytes are eight consecutive
// reduction elements of row l % 16), U steps at a time, the next ones in flight while
// the ones before are multiplied. The waves' sums meet in LDS and are added in order.
// 1 x 7168 -> 2 x 2048 12.5 us (the 59 MB of weights at 4.7 TB/s); with more rows the
// blocks' reading of x is the bound, 16 x 2048 -> 7168 10.5 us (2.8 TB/s).
// GATED: a 16-row block of weights is eight gates and their eight ups.
#include "linear.h"

namespace {

constexpr int N_NT = 512, N_W = N_NT / 64;
constexpr int U = 4;  // 32-deep steps fetched together

template <int ET>
__device__ __forceinline__ f32x4_t mma16(const u32x4& a, const u32x4& b, const f32x4_t& c) {
  if constexpr (ET == TT_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int KIND, class TT, int MB>
__global__ __launch_bounds__(N_NT) void linear_rows_kernel(LinArgs p) {
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int ET = sizeof(typename TT::storage) == 2 && __is_same(TT, BF16T) ? TT_BF16 : TT_F16;
  constexpr int CB = GATED ? 8 : 16;  // output columns of a block
  constexpr int LD = 16 + 4;          // row stride of the sums: 16-byte chunks, spread
  __shared__ __align__(16) float sums[N_W][16 * MB][LD];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t j0 = (int64_t)blockIdx.x * CB;
  const int R = (int)p.R;
  // This wave's 32-deep steps of the reduction.
  const int steps = (R + 31) / 32;
  const int s0 = steps * wave / N_W, s1 = steps * (wave + 1) / N_W;
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<void*>(p.a), (short)0, (int)(uint32_t)(p.I * p.lda * 2), 0x00020000);
  uint32_t xo[MB];
  const char* const w0 = static_cast<const char*>(p.b) + j0 * p.ldb * 2;
  const int64_t wleft = ((GATED ? 2 : 1) * p.J - j0) * p.ldb * 2;
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(w0), (short)0,
      (int)(wleft < (int64_t)DM_OOB ? (uint32_t)wleft : DM_OOB), 0x00020000);
#pragma unroll
  for (int m = 0; m < MB; ++m)
    xo[m] = 16 * m + r < p.I ? (uint32_t)(((16 * m + r) * p.lda + 8 * g) * 2) : DM_OOB;
  const int64_t c = GATED ? r & 7 : r;  // column of the block
  const int64_t row = GATED && r >= 8 ? p.J + c : c;
  const uint32_t wo = j0 + c < p.J ? (uint32_t)((row * p.ldb + 8 * g) * 2) : DM_OOB;
  f32x4_t acc[MB] = {};
  u32x4 xv[2][U][MB], wv[2][U];
  auto fetch = [&](int s, int buf) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      // Steps past the wave's last and elements past the row's end read as zeros.
      const bool ok = s + q < s1 && 32 * (s + q) + 8 * g < R;
      const uint32_t at = (uint32_t)(s + q) * 64u;
      wv[buf][q] = __builtin_amdgcn_raw_buffer_load_b128(
          rw, (int)(ok && wo != DM_OOB ? wo + at : DM_OOB), 0, 0);
#pragma unroll
      for (int m = 0; m < MB; ++m)
        xv[buf][q][m] = __builtin_amdgcn_raw_buffer_load_b128(
            rx, (int)(ok && xo[m] != DM_OOB ? xo[m] + at : DM_OOB), 0, 0);
    }
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int m = 0; m < MB; ++m) acc[m] = mma16<ET>(wv[buf][q], xv[buf][q][m], acc[m]);
  };
  if (s0 < s1) fetch(s0, 0);
  for (int s = s0; s < s1; s += 2 * U) {
    if (s + U < s1) fetch(s + U, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(0);
    if (s + U >= s1) break;
    if (s + 2 * U < s1) fetch(s + 2 * U, 0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
  }
  // Lane l holds row 16 m + l % 16 of x, rows 4 (l / 16) + 0..3 of the weights.
#pragma unroll
  for (int m = 0; m < MB; ++m)
    *reinterpret_cast<f32x4_t*>(&sums[wave][16 * m + r][4 * g]) = acc[m];
  __syncthreads();
  constexpr int NG = CB / 8;  // groups of eight outputs
  DropKey dk{};
  if constexpr (KIND == LIN_DROP) dk = load_key(p.key);
  for (int it = threadIdx.x; it < (int)p.I * NG; it += N_NT) {
    const int i = it / NG, og = it % NG;
    const int64_t j = j0 + 8 * og;
    if (j >= p.J) continue;
    const int at = GATED ? 16 * og : 8 * og;
    float v[8] = {}, u[8] = {};
#pragma unroll
    for (int w = 0; w < N_W; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] += sums[w][i][at + e];
        if constexpr (GATED) u[e] += sums[w][i][at + 8 + e];
      }
    lin_finish<KIND, TT, 8, true>(p, i, j, 8, v, u, dk, lin_cols<KIND, 8>(p, j, 8),
                                  lin_row<KIND, TT, 8, true>(p, i, j, 8));
  }
}

template <int KIND, class TT, int MB>
int launch(const LinArgs& p, hipStream_t s) {
  constexpr int CB = KIND == LIN_GATED ? 8 : 16;
  const int64_t blocks = (p.J + CB - 1) / CB;
  TT_REQUIRE(tt_grid_ok(blocks, N_NT), "linear: grid too large");
  hipLaunchKernelGGL((linear_rows_kernel<KIND, TT, MB>), dim3((unsigned)blocks), dim3(N_NT),
                     0, s, p);
  return tt_check_launch("linear_rows");
}

template <int KIND, class TT>
int rows(const LinArgs& p, hipStream_t s) {
  if (p.I <= 16) return launch<KIND, TT, 1>(p, s);
  if (p.I <= 32) return launch<KIND, TT, 2>(p, s);
  return launch<KIND, TT, 4>(p, s);
}

template <int KIND>
int typed(int dtype, const LinArgs& p, hipStream_t s) {
  return dtype == TT_BF16 ? rows<KIND, BF16T>(p, s) : rows<KIND, F16T>(p, s);
}

}  // namespace

int tt_linear_rows(int kind, int dtype, const LinArgs& p, hipStream_t s) {
  switch (kind) {
    case LIN_ACT: return typed<LIN_ACT>(dtype, p, s);
    case LIN_GATED: return typed<LIN_GATED>(dtype, p, s);
    case LIN_RES: return typed<LIN_RES>(dtype, p, s);
    default: return typed<LIN_DROP>(dtype, p, s);
  }
}
