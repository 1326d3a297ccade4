// Product of few rows with 4-bit weights (gfx950): decoding, short prompts, experts of few rows.
//
// Such a call reads the weights once and is bound by that stream. A block takes 16 NB weight rows
// and 16 MB rows of x, and its W waves split the reduction among them; operands go from memory to
// registers in the layout of the matrix instructions, U steps of 128 reduction elements at a time,
// the next ones in flight while the ones before are multiplied. E4M3 rows are multiplied with the
// codes as they are (scaled 16x16x128 products); for bf16 rows the codes become bf16 with their
// scale, two to an instruction and exact, and take the 16x16x32 products. The waves' sums meet in
// LDS and are added in order. GATED: 16 weight rows are eight gates and their eight ups.
#include "mx_gemm.h"

namespace {

template <bool MX, bool GATED, bool OUT8, int MB, int NB, int W, int U>
__global__ __launch_bounds__(64 * W) void mx_rows_kernel(MxArgs p, int tiles_j) {
  constexpr int NT = 64 * W;
  constexpr int CB = (GATED ? 8 : 16) * NB;  // output columns of a block
  constexpr int LD = 16 * NB + 4;            // row stride of the sums
  constexpr int XV = MX ? 2 : 4;             // 16-byte pieces of a row per step
  __shared__ __align__(16) float sums[W][16 * MB][LD];
  RowTile t;
  if (p.counts != nullptr) {
    if (!row_tile<16 * MB, NT>(p.counts, p.E, tiles_j, reinterpret_cast<char*>(sums), t)) return;
    // Counts that sum to more than M end at its last row.
    if (t.seg0 + t.nrows > p.M) t.nrows = p.M - t.seg0;
    if ((int64_t)t.mt * 16 * MB >= t.nrows) return;
  } else {
    t.e = 0;
    t.nt = (int)(blockIdx.x % (unsigned)tiles_j);
    t.mt = (int)(blockIdx.x / (unsigned)tiles_j);
    t.seg0 = 0;
    t.nrows = p.M;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t K = p.K, j0 = (int64_t)t.nt * CB, i0 = (int64_t)t.mt * 16 * MB;
  const int64_t rows = t.nrows - i0;  // valid rows of the tile, at least one
  const int groups = (int)(K / MX_GROUP);
  // Steps of 128 elements; the last may be short.
  const int steps = (groups + 3) / 4;
  const int s0 = steps * wave / W, s1 = steps * (wave + 1) / W;
  // A lane's rows. Rows past the last one read it again: their results are not stored.
  const uint8_t *wp[NB], *wsp[NB];
  const char* xp[MB];
  const uint8_t* xsp[MB];
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    int64_t n = j0 + (GATED ? 8 * q + (r & 7) : 16 * q + r);
    n = n < p.N ? n : p.N - 1;
    if (GATED && r >= 8) n += p.N;
    n += (int64_t)t.e * (GATED ? 2 : 1) * p.N;
    wp[q] = p.w + n * (K / 2) + 16 * g;
    wsp[q] = p.ws + n * groups + g;
  }
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int64_t i = 16 * m + r;
    const int64_t v = mx_source_row(p, t.seg0 + i0 + (i < rows ? i : rows - 1));
    xp[m] = static_cast<const char*>(p.x) + v * K * (MX ? 1 : 2) + (MX ? 16 : 64) * g;
    xsp[m] = MX ? p.xs + v * groups + g : nullptr;
  }
  f32x4_t acc[MB][NB] = {};
  uint4 wv[2][U][NB], xv[2][U][MB][XV];
  uint32_t wsv[2][U][NB], xsv[2][U][MB];
  auto fetch = [&](int s, int buf) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= s1) break;
      const int64_t k = s + u;
      if (4 * (s + u) + 4 <= groups) {
#pragma unroll
        for (int q = 0; q < NB; ++q) {
          wv[buf][u][q] = *reinterpret_cast<const uint4*>(wp[q] + 64 * k);
          wsv[buf][u][q] = wsp[q][4 * k];
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) {
#pragma unroll
          for (int c = 0; c < XV; ++c)
            xv[buf][u][m][c] =
                *reinterpret_cast<const uint4*>(xp[m] + (MX ? 128 * k + 64 * c : 256 * k + 16 * c));
          if constexpr (MX) xsv[buf][u][m] = xsp[m][4 * k];
        }
      } else {
        // The short step: groups past the last read as zeros of scale 1. A lane's group of the
        // weights (and of bf16 rows) is g; its two pieces of E4M3 rows belong to g / 2 and 2 + g / 2.
        const int left = groups - 4 * (s + u);
        const uint4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < NB; ++q) {
          wv[buf][u][q] = g < left ? *reinterpret_cast<const uint4*>(wp[q] + 64 * k) : zero;
          wsv[buf][u][q] = g < left ? wsp[q][4 * k] : 127u;
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) {
#pragma unroll
          for (int c = 0; c < XV; ++c) {
            const int group = MX ? 2 * c + (g >> 1) : g;
            xv[buf][u][m][c] =
                group < left ? *reinterpret_cast<const uint4*>(
                                   xp[m] + (MX ? 128 * k + 64 * c : 256 * k + 16 * c))
                             : zero;
          }
          if constexpr (MX) xsv[buf][u][m] = g < left ? xsp[m][4 * k] : 127u;
        }
      }
    }
  };
  auto multiply = [&](int s, int buf) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= s1) break;
      if constexpr (MX) {
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
          for (int m = 0; m < MB; ++m)
            acc[m][q] = mx_mma16<0, 0>(wv[buf][u][q], xv[buf][u][m][0], xv[buf][u][m][1],
                                       wsv[buf][u][q], xsv[buf][u][m], acc[m][q]);
      } else {
#pragma unroll
        for (int q = 0; q < NB; ++q) {
          const uint32_t c[4] = {wv[buf][u][q].x, wv[buf][u][q].y, wv[buf][u][q].z,
                                 wv[buf][u][q].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bf16x8 a = __builtin_bit_cast(bf16x8, mx_bf16x8(c[i], wsv[buf][u][q]));
#pragma unroll
            for (int m = 0; m < MB; ++m)
              acc[m][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  a, __builtin_bit_cast(bf16x8, xv[buf][u][m][i]), acc[m][q], 0, 0, 0);
          }
        }
      }
    }
  };
  if (s0 < s1) fetch(s0, 0);
  for (int s = s0; s < s1; s += 2 * U) {
    if (s + U < s1) fetch(s + U, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(s, 0);
    if (s + U >= s1) break;
    if (s + 2 * U < s1) fetch(s + 2 * U, 0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(s + U, 1);
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int q = 0; q < NB; ++q)
      *reinterpret_cast<f32x4_t*>(&sums[wave][16 * m + r][16 * q + 4 * g]) = acc[m][q];
  __syncthreads();
  constexpr int NG = CB / 8;  // groups of eight outputs
  const int items = (int)(rows < 16 * MB ? rows : 16 * MB) * NG;
  for (int it = threadIdx.x; it < items; it += NT) {
    const int i = it / NG, og = it % NG;
    const int64_t j = j0 + 8 * og;
    if (j >= p.N) continue;  // OUT8: whole groups of four lanes
    const int at = GATED ? 16 * og : 8 * og;
    float v[8] = {}, up[8] = {};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] += sums[w][i][at + e];
        if constexpr (GATED) up[e] += sums[w][i][at + 8 + e];
      }
    const int64_t row = t.seg0 + i0 + i;
    const float f = p.probs != nullptr ? load_as_f32(p.probs, p.pdt, row) : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = mx_act(v[e], p.act);
      if constexpr (GATED) v[e] *= up[e];
      if (p.probs != nullptr) v[e] *= f;
    }
    if constexpr (OUT8) mx_store_rows(p, row, j, v);
    else mx_store_bf16(p, row, j, v);
  }
}

template <bool MX, bool GATED, bool OUT8, int MB, int NB, int W, int U>
int launch(const MxArgs& p, hipStream_t s) {
  constexpr int CB = (GATED ? 8 : 16) * NB;
  const int64_t tiles_j = (p.N + CB - 1) / CB;
  // Row tiles: those of a dense product, or the most that the experts' counts can make.
  int64_t tiles_i = (p.M + 16 * MB - 1) / (16 * MB);
  if (p.counts != nullptr) tiles_i = p.M / (16 * MB) + (p.E < p.M ? p.E : p.M);
  TT_REQUIRE(tiles_i < (1ll << 31) && tiles_j < (1ll << 31) && tiles_i * tiles_j < (1ll << 31) &&
                 tt_grid_ok(tiles_i * tiles_j, 64 * W),
             "mx product: grid too large");
  hipLaunchKernelGGL((mx_rows_kernel<MX, GATED, OUT8, MB, NB, W, U>), dim3((unsigned)(tiles_i * tiles_j)),
                     dim3(64 * W), 0, s, p, (int)tiles_j);
  return tt_check_launch("mx_rows");
}

// Weight tiles and waves of a block by how many 16-row tiles the launch has (those of the experts
// that can have rows): few tiles are spread over all CUs with the reduction split eight ways, many
// share their reads of x and their block's start. us, bf16 rows, <1, 8> / <4, 4> / <4, 2>:
// 1 x 7168 -> 2 x 2048 (256 tiles) 8.4 / 18.0 / 20.9, 4 x 4096 -> 2 x 14336 (1792) 34.6 / 24.5 /
// 25.7, 128 rows of 128 experts 2048 -> 2 x 768 (12288) 129 / 34.7 / 33.0, 768 -> 2048 91 / 22.8 / 18.5.
template <bool MX, bool GATED, bool OUT8>
int rows(const MxArgs& p, hipStream_t s) {
  constexpr int N8 = GATED ? 4 : 2;  // weight tiles of 32 outputs, a group's
  const int64_t per = p.counts != nullptr ? (p.M + p.E - 1) / p.E : p.M;
  const int64_t tiles = ((GATED ? 2 : 1) * p.N + 15) / 16 * (p.counts == nullptr || p.E < p.M ? p.E : p.M);
  if (per > 16) return launch<MX, GATED, OUT8, 2, OUT8 ? N8 : 2, 4, 2>(p, s);
  if (tiles < 1024) return launch<MX, GATED, OUT8, 1, OUT8 ? N8 : 1, 8, 1>(p, s);
  if (tiles < 4096) return launch<MX, GATED, OUT8, 1, OUT8 ? N8 : 4, 4, 1>(p, s);
  return launch<MX, GATED, OUT8, 1, OUT8 ? N8 : 4, 2, 1>(p, s);
}

template <bool MX, bool GATED>
int out(const MxArgs& p, hipStream_t s) {
  return p.ys != nullptr ? rows<MX, GATED, true>(p, s) : rows<MX, GATED, false>(p, s);
}

}  // namespace

int tt_mx_rows(const MxArgs& p, bool gated, hipStream_t s) {
  if (p.xs != nullptr) return gated ? out<true, true>(p, s) : out<true, false>(p, s);
  return gated ? out<false, true>(p, s) : out<false, false>(p, s);
}
