// Product of few rows with 4-bit weights (gfx950): decoding, short prompts, experts of few rows.
//
// Such a call reads the weights once and is bound by that stream. A block takes 16 NB weight rows
// and 16 MB rows of x, and its W waves split the reduction among them; operands go from memory to
// registers in the layout of the matrix instructions, 128 reduction elements a step, two steps in
// flight. E4M3 rows are multiplied with the codes as they are (scaled 16x16x128 products); for bf16
// rows the codes become bf16 with their scale, two to an instruction and exact, and take the
// 16x16x32 products. The waves' sums meet in LDS and are added in order. GATED: 16 weight rows are
// eight gates and their eight ups.
#include "mx_gemm.h"

namespace {

// Bytes of an operand that loads of nothing leave alone: a lane with no row (off < 0) or past the end
// (!ok) gets zeros. Near operands are buffers, whose loads need no branch for it.
template <bool NEAR>
struct Operand;

template <>
struct Operand<true> {
  using Off = int32_t;
  __amdgpu_buffer_rsrc_t buffer;
  __device__ Operand(const uint8_t* base, int64_t bytes)
      : buffer(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), (short)0, (int)bytes,
                                                 0x00020000)) {}
  __device__ u32x4 b128(Off off, Off by, bool ok) const {
    return __builtin_amdgcn_raw_buffer_load_b128(buffer, ok && off >= 0 ? off + by : (int)DM_OOB, 0, 0);
  }
  __device__ uint32_t b8(Off, Off, bool) const { return 0; }
};

template <>
struct Operand<false> {
  using Off = int64_t;
  const uint8_t* base;
  __device__ Operand(const uint8_t* base, int64_t) : base(base) {}
  __device__ u32x4 b128(Off off, Off by, bool ok) const {
    const u32x4 zero = {0, 0, 0, 0};
    return ok && off >= 0 ? *reinterpret_cast<const u32x4*>(base + off + by) : zero;
  }
  __device__ uint32_t b8(Off off, Off by, bool ok) const {
    return ok && off >= 0 ? base[off + by] : 0u;
  }
};

// NEAR: K is a multiple of 128, the scales are 4-byte aligned, an expert's weights and the rows lie
// within 2 GiB (32-bit offsets into buffers), and the scales of four steps come in one load of sixteen
// bytes a row: what a CU's memory path takes is lines, sixteen to a load of codes or of scales. Without
// it a load of a byte a step and 64-bit addresses: 1 x 7168 -> 2 x 2048 10.6 us for 7.2, 128 rows
// of 128 experts 2048 -> 2 x 768 39 for 27.
template <bool MX, bool GATED, bool OUT8, int MB, int NB, int W, bool NEAR>
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
  // A lane's rows as offsets into the operands, negative for rows past the last one: those read as
  // zeros and cost no traffic (with one row of x, fifteen sixteenths of it).
  using Off = typename Operand<NEAR>::Off;
  const int64_t width = (GATED ? 2 : 1) * p.N;
  const bool gather = p.arow != nullptr;
  const int64_t first = gather ? 0 : t.seg0 + i0;
  const int64_t held = gather ? p.src_rows : (rows < 16 * MB ? rows : 16 * MB);
  constexpr int ES = MX ? 1 : 2;
  const Operand<NEAR> w(p.w + (int64_t)t.e * width * (K / 2), width * (K / 2)),
      ws(p.ws + (int64_t)t.e * width * groups, width * groups),
      x(static_cast<const uint8_t*>(p.x) + first * K * ES, held * K * ES),
      xs(MX ? p.xs + first * groups : nullptr, MX ? held * groups : 0);
  Off wo[NB], wso[NB], xo[MB], xso[MB];
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    int64_t n = j0 + (GATED ? 8 * q + (r & 7) : 16 * q + r);
    const bool in = n < p.N;
    if (GATED && r >= 8) n += p.N;
    wo[q] = in ? (Off)(n * (K / 2) + 16 * g) : -1;
    wso[q] = in ? (Off)(n * groups + (NEAR ? 0 : g)) : -1;
  }
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int64_t i = 16 * m + r;
    xo[m] = xso[m] = -1;
    if (i < rows) {
      const int64_t v = gather ? mx_source_row(p, t.seg0 + i0 + i) : i;
      xo[m] = (Off)(v * K * ES + (MX ? 16 : 64) * g);
      xso[m] = (Off)(v * groups + (NEAR ? 0 : g));
    }
  }
  f32x4_t acc[MB][NB] = {};
  // No load and no product depends on a branch, so that a step waits for its own loads alone: groups
  // past the wave's last one read as zeros of scale zero, which add nothing.
  u32x4 wv[2][NB], xv[2][MB][XV], ws4[2][NB], xs4[2][MB];
  uint32_t ws1[2][NB], xs1[2][MB];
  const int limit = 4 * s1 < groups ? 4 * s1 : groups;
  // The scales of steps s to s + 3; words behind the operand's last one read as zeros.
  auto fetch_scales = [&](int s, int d) {
    if constexpr (NEAR) {
#pragma unroll
      for (int q = 0; q < NB; ++q) ws4[d][q] = ws.b128(wso[q], 4 * s, 4 * s < limit);
      if constexpr (MX)
#pragma unroll
        for (int m = 0; m < MB; ++m) xs4[d][m] = xs.b128(xso[m], 4 * s, 4 * s < limit);
    }
  };
  auto fetch = [&](int s, int d) {
    const bool ok = 4 * s + g < limit;
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      wv[d][q] = w.b128(wo[q], 64 * (Off)s, ok);
      if constexpr (!NEAR) ws1[d][q] = ws.b8(wso[q], 4 * s, ok);
    }
    // E4M3: a lane's two pieces are halves of groups g / 2 and 2 + g / 2 of the step.
    const bool ok0 = MX ? 4 * s + (g >> 1) < limit : ok, ok1 = MX ? 4 * s + 2 + (g >> 1) < limit : ok;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
#pragma unroll
      for (int c = 0; c < XV; ++c)
        xv[d][m][c] = x.b128(xo[m], MX ? 128 * (Off)s + 64 * c : 256 * (Off)s + 16 * c,
                             c == 0 ? ok0 : ok1);
      if constexpr (MX && !NEAR) xs1[d][m] = xs.b8(xso[m], 4 * s, ok);
    }
  };
  // Step s in slot d, the i-th of the four whose scales slot ds holds. A load of four steps' scales
  // may end in the next row: a group past the end takes none of them.
  auto multiply = [&](int s, int d, int i, int ds) {
    const bool ok = 4 * s + g < limit;
    uint32_t xscale[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m)
      xscale[m] = !MX ? 0u : NEAR ? (ok ? (xs4[ds][m][i] >> (8 * g)) & 255u : 0u) : xs1[d][m];
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const uint4 a4 = __builtin_bit_cast(uint4, wv[d][q]);
      const uint32_t scale = NEAR ? (ok ? (ws4[ds][q][i] >> (8 * g)) & 255u : 0u) : ws1[d][q];
      if constexpr (MX) {
#pragma unroll
        for (int m = 0; m < MB; ++m)
          acc[m][q] = mx_mma16<0, 0>(a4, __builtin_bit_cast(uint4, xv[d][m][0]),
                                     __builtin_bit_cast(uint4, xv[d][m][1]), scale, xscale[m],
                                     acc[m][q]);
      } else {
        const uint32_t c[4] = {a4.x, a4.y, a4.z, a4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8 a = __builtin_bit_cast(bf16x8, mx_bf16x8(c[j], scale));
#pragma unroll
          for (int m = 0; m < MB; ++m)
            acc[m][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                a, __builtin_bit_cast(bf16x8, xv[d][m][j]), acc[m][q], 0, 0, 0);
        }
      }
    }
  };
  if (s0 < s1) {
    fetch_scales(s0, 0);
    fetch(s0, 0);
    fetch(s0 + 1, 1);
    for (int s = s0; s < s1; s += 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i == 4 && s + 4 >= s1) break;
        if ((i & 3) == 0) fetch_scales(s + i + 4, (i >> 2) ^ 1);
        multiply(s + i, i & 1, i & 3, i >> 2);
        fetch(s + i + 2, i & 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int q = 0; q < NB; ++q)
      *reinterpret_cast<f32x4_t*>(&sums[wave][16 * m + r][16 * q + 4 * g]) = acc[m][q];
  __syncthreads();
  // The waves' sums, in order, four at a time by all threads.
  constexpr int Q4 = 4 * NB;
  const int valid = (int)(rows < 16 * MB ? rows : 16 * MB);
  for (int it = threadIdx.x; it < valid * Q4; it += NT) {
    const int i = it / Q4, c = 4 * (it % Q4);
    f32x4_t v = *reinterpret_cast<f32x4_t*>(&sums[0][i][c]);
#pragma unroll
    for (int w = 1; w < W; ++w) v += *reinterpret_cast<f32x4_t*>(&sums[w][i][c]);
    *reinterpret_cast<f32x4_t*>(&sums[0][i][c]) = v;
  }
  __syncthreads();
  constexpr int NG = CB / 8;  // groups of eight outputs
  const int items = valid * NG;
  for (int it = threadIdx.x; it < items; it += NT) {
    const int i = it / NG, og = it % NG;
    const int64_t j = j0 + 8 * og;
    if (j >= p.N) continue;  // OUT8: whole groups of four lanes
    const int at = GATED ? 16 * og : 8 * og;
    float v[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = sums[0][i][at + e];
      up[e] = GATED ? sums[0][i][at + 8 + e] : 0.f;
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

template <bool MX, bool GATED, bool OUT8, int MB, int NB, int W, bool NEAR>
int launch(const MxArgs& p, hipStream_t s) {
  constexpr int CB = (GATED ? 8 : 16) * NB;
  const int64_t tiles_j = (p.N + CB - 1) / CB;
  // Row tiles: those of a dense product, or the most that the experts' counts can make.
  int64_t tiles_i = (p.M + 16 * MB - 1) / (16 * MB);
  if (p.counts != nullptr) tiles_i = p.M / (16 * MB) + (p.E < p.M ? p.E : p.M);
  TT_REQUIRE(tiles_i < (1ll << 31) && tiles_j < (1ll << 31) && tiles_i * tiles_j < (1ll << 31) &&
                 tt_grid_ok(tiles_i * tiles_j, 64 * W),
             "mx product: grid too large");
  hipLaunchKernelGGL((mx_rows_kernel<MX, GATED, OUT8, MB, NB, W, NEAR>), dim3((unsigned)(tiles_i * tiles_j)),
                     dim3(64 * W), 0, s, p, (int)tiles_j);
  return tt_check_launch("mx_rows");
}

template <bool MX, bool GATED, bool OUT8, int MB, int NB, int W>
int block(const MxArgs& p, hipStream_t s) {
  const int64_t es = MX ? 1 : 2, limit = 1ll << 31;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.xs);
  const bool near = p.K % 128 == 0 && (at & 3) == 0 && (GATED ? 2 : 1) * p.N * (p.K / 2) < limit &&
                    (p.arow != nullptr ? p.src_rows : (int64_t)16 * MB) * p.K * es < limit;
  return near ? launch<MX, GATED, OUT8, MB, NB, W, true>(p, s)
              : launch<MX, GATED, OUT8, MB, NB, W, false>(p, s);
}

// Weight tiles and waves of a block by how many 16-row tiles the launch has (those of the experts
// that can have rows): few tiles are spread over all CUs with the reduction split four ways, many
// share their reads of x and their block's start. us, bf16 rows, <1, 4> / <2, 4> / <4, 4> / <4, 1>:
// 1 x 7168 -> 2 x 2048 (256 tiles) 7.3 / 8.9 / 12.8 / 21.5, 2048 -> 7168 (448) 5.5 / 4.9 / 6.2 / 8.5,
// 4 x 4096 -> 2 x 14336 (1792) 25.0 / 21.8 / 19.6 / 21.9, 8 rows of 256 experts 7168 -> 2 x 2048 (2048)
// 34.8 / 28.1 / 28.1 / 26.5, 128 of 128 experts 2048 -> 2 x 768 (12288) 52.3 / 38.2 / 33.5 / 26.5, 768 ->
// 2048 (16384) 61.2 / 42.3 / 34.4 / 17.2. More than 16 rows, blocks of 32 by
// <2, 2> / of 16 by <1, 4>: 24 x 2048 -> 7168 7.3 / 11.8, 64 x 7168 -> 2 x 2048 19.3 / 36.4.
template <bool MX, bool GATED, bool OUT8>
int rows(const MxArgs& p, hipStream_t s) {
  const int64_t per = p.counts != nullptr ? (p.M + p.E - 1) / p.E : p.M;
  const int64_t tiles = ((GATED ? 2 : 1) * p.N + 15) / 16 * (p.counts == nullptr || p.E < p.M ? p.E : p.M);
  if constexpr (OUT8) {
    constexpr int N8 = GATED ? 4 : 2;  // weight tiles of 32 outputs, a group's
    if (per > 16) return block<MX, GATED, true, 2, N8, 2>(p, s);
    if (tiles < 2048) return block<MX, GATED, true, 1, N8, 4>(p, s);
    return block<MX, GATED, true, 1, N8, 1>(p, s);
  } else {
    if (per > 16) return block<MX, GATED, false, 2, 2, 2>(p, s);
    if (tiles < 384) return block<MX, GATED, false, 1, 1, 4>(p, s);
    if (tiles < 1024) return block<MX, GATED, false, 1, 2, 4>(p, s);
    if (tiles < 2048) return block<MX, GATED, false, 1, 4, 4>(p, s);
    return block<MX, GATED, false, 1, 4, 1>(p, s);
  }
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
