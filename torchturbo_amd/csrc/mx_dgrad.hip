// Gradient of bf16 rows through frozen 4-bit weights (gfx950): dx [M, K] = dy [M, N] W[e], with
// W [N, K] in groups of 32 along K.
//
// The reduction runs across the rows of W, whose elements lie along K, so the matrix instructions
// need W transposed: a block turns a 64 x 128 piece of codes into bf16 (exact, two codes an
// instruction, each thread one group with its scale) and writes it to LDS as it lies; the transposing
// LDS reads then give each lane eight reduction elements of a column. dy goes straight from memory
// to LDS, two stages deep: the next k-tile's loads (W's in registers) are in flight while a tile is
// multiplied. One copy of W's piece leaves room for three blocks on a CU, which cover one another's
// barriers (1531 x 2048 -> 5632 66 -> 54 us, 8192 rows of 128 experts 1536 -> 2048 155 -> 127, against
// two copies and two blocks). Every product is exact in fp32; sums run in fp32 and dx is rounded once.
//
// Two limits: rows of dy off 16 bytes come by single elements through registers (1531 x 2047 -> 5632
// 168 us for 56 at 2048, 8192 x 4095 -> 4096, which loses the larger tile too, 1009 for 232), and the
// reduction is never split, so that few rows take the time of K / 128 blocks' loops (1 to 512 rows of 2048
// -> 5632 23 to 26 us, 16 rows of 14336 -> 4096 144, 1 to 64 rows for each of 128 experts 1536 -> 2048 103 to 115).
#include "mx_gemm.h"

namespace {

constexpr int D_NT = 256, D_BM = 128, D_BN = 128, D_BK = 64;
constexpr int D_A = D_BM * D_BK * 2, D_B = D_BN * D_BK * 2;  // two stages of dy, one of W

// The block's tile of a dense product: eight row tiles at a time, so that the blocks an XCD has at
// work read few panels of either operand.
__device__ __forceinline__ void dense_tile(RowTile& t, int64_t M, int tiles_i, int tiles_j) {
  const int at = xcd_remap(blockIdx.x, tiles_i * tiles_j), group = 8 * tiles_j;
  const int m0 = at / group * 8, gm = tiles_i - m0 < 8 ? tiles_i - m0 : 8;
  t.e = 0;
  t.mt = m0 + at % group % gm;
  t.nt = at % group / gm;
  t.seg0 = 0;
  t.nrows = M;
}

// ALIGNED: rows of dy are multiples of 16 bytes at 16-byte addresses.
template <bool ALIGNED>
__global__ __launch_bounds__(D_NT, 3) void mx_dgrad_kernel(
    const char* __restrict__ dy, const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
    char* __restrict__ dx, int64_t M, int64_t K, int64_t N, int E,
    const int64_t* __restrict__ counts, int tiles_j) {
  __shared__ __align__(16) char lds_raw[2 * D_A + D_B];
  RowTile t;
  if (counts != nullptr) {
    if (!row_tile<D_BM, D_NT>(counts, E, tiles_j, lds_raw, t)) return;
    // Counts that sum to more than M end at its last row.
    if (t.seg0 + t.nrows > M) t.nrows = M - t.seg0;
    if ((int64_t)t.mt * D_BM >= t.nrows) return;
  } else {
    dense_tile(t, M, (int)((M + D_BM - 1) / D_BM), tiles_j);
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t i0 = (int64_t)t.mt * D_BM, j0 = (int64_t)t.nt * D_BN;
  const int64_t rows = t.nrows - i0;
  const int nkt = (int)((N + D_BK - 1) / D_BK);
  lds_char* const lds = (lds_char*)lds_raw;

  // dy: wave w loads rows 32 w + 8 q + lane / 8, chunk slot lane % 8 holding chunk
  // slot ^ ((row >> 1) & 7); rows past the expert's and elements past a row's end read as zeros.
  const char* const a0 = dy + (t.seg0 + i0) * N * 2;
  const i32x4 ra = make_rsrc(a0, (rows < D_BM ? rows : D_BM) * N * 2);
  uint32_t aoff[4];
  int akof[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = 32 * wave + 8 * q + (lane >> 3);
    const int c = (lane & 7) ^ ((r >> 1) & 7);
    akof[q] = 8 * c;
    aoff[q] = (uint32_t)(r * N + 8 * c) * 2u;
  }
  // W: a thread takes one group of a row, four neighbours the tile's columns of it; 16 lanes take
  // rows four apart, which the swizzle below spreads over all banks. Groups past a row's end read the
  // last one again: their columns are not stored.
  const int wr = 16 * (tid >> 6) + 4 * ((tid >> 2) & 3) + ((tid >> 4) & 3);
  const int64_t groups = K / MX_GROUP;
  int64_t wg = j0 / MX_GROUP + (tid & 3);
  wg = wg < groups ? wg : groups - 1;
  const uint8_t* const wp = w + (int64_t)t.e * N * (K / 2) + wg * 16;
  const uint8_t* const wsp = ws + (int64_t)t.e * N * groups + wg;

  uint4 wv;
  uint32_t wsv;
  auto load = [&](int kt, int buf) {
    const int64_t n = (int64_t)kt * D_BK + wr;
    wv = uint4{0, 0, 0, 0};
    wsv = 127u;
    if (n < N) {
      wv = *reinterpret_cast<const uint4*>(wp + n * (K / 2));
      wsv = wsp[n * groups];
    }
    lds_char* const a = lds + buf * D_A;
    if constexpr (ALIGNED) {
      const uint32_t base = lds_addr_of(a) + (uint32_t)(4 * wave) * 1024u;
      const i32x4 rk = advance_rsrc(ra, (uint32_t)kt * (D_BK * 2));
#pragma unroll
      for (int q = 0; q < 4; ++q)
        dma16((int64_t)kt * D_BK + akof[q] < N ? aoff[q] : DM_OOB, rk, base + q * 1024u);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 32 * wave + 8 * q + (lane >> 3);
        const int64_t n0 = (int64_t)kt * D_BK + akof[q];
        const uint16_t* const p = reinterpret_cast<const uint16_t*>(a0) + r * N + n0;
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = r < rows && n0 + 2 * e < N ? p[2 * e] : 0u;
          const uint32_t hi = r < rows && n0 + 2 * e + 1 < N ? p[2 * e + 1] : 0u;
          v[e] = lo | hi << 16;
        }
        *reinterpret_cast<lds_u32x4*>(a + (4 * wave + q) * 1024 + 16 * lane) =
            u32x4{v[0], v[1], v[2], v[3]};
      }
    }
  };
  // The k-row's chunk c (eight columns) lies in slot c ^ (4 (row % 4)) ^ (row / 4 % 4).
  auto put = [&]() {
    lds_char* const b = lds + 2 * D_A + wr * 256;
    const uint32_t q[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = mx_bf16x8(q[i], wsv);
      const int c = 4 * (tid & 3) + i;
      *reinterpret_cast<lds_u32x4*>(b + ((c ^ (4 * (wr & 3)) ^ ((wr >> 2) & 3)) << 4)) =
          u32x4{v.x, v.y, v.z, v.w};
    }
  };
  // Wave w multiplies rows 64 (w / 2) .. + 63 and columns 64 (w % 2) .. + 63.
  const int m0 = 64 * (wave >> 1), n0 = 64 * (wave & 1);
  uint32_t fa[4], fb[4][2];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    fa[s] = fragk64(m0, s, lane);
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int col = n0 + 32 * b + 16 * (g & 1) + 4 * (i & 3);
      const int kr = 16 * s + 8 * (g >> 1) + (i >> 2);
      fb[s][b] = 2 * D_A + (uint32_t)(kr * 256 + (col & 7) * 2 +
                                  (((col >> 3) ^ (4 * (kr & 3)) ^ ((kr >> 2) & 3)) << 4));
    }
  }
  f32x16 acc[2][2] = {};
  if (nkt > 0) load(0, 0);
  for (int kt = 0; kt < nkt; ++kt) {
    put();  // the k-tile's codes, loaded during the one before
    TT_WAIT_VMCNT(0);
    TT_LDS_BARRIER();
    if (kt + 1 < nkt) load(kt + 1, (kt & 1) ^ 1);
    lds_char* const st = lds + (kt & 1) * D_A;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint4 b[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds + fb[s][j]));
        // Four k-rows on: 1024 bytes, and the other slot of a pair.
        const i16x4 v1 =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds + (fb[s][j] ^ 16) + 1024));
        const uint2 p0 = __builtin_bit_cast(uint2, v0), p1 = __builtin_bit_cast(uint2, v1);
        b[j] = uint4{p0.x, p0.y, p1.x, p1.y};
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 a = read_k(st, fa[s] + i * 4096);
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = Mma<TT_BF16>::run(b[j], a, acc[i][j]);
      }
    }
    TT_LDS_BARRIER();
  }
  // The tile through LDS, rows of 256 bytes, chunk c of row r in slot c ^ (r % 16). Register 4 q + e
  // of lane l: row l % 32, column 8 q + 4 (l / 32) + e.
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = m0 + 32 * i + (lane & 31), c = (n0 + 32 * j) / 8 + q;
        const uint2 v = pack4<TT_BF16>(acc[i][j][4 * q], acc[i][j][4 * q + 1],
                                       acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        *reinterpret_cast<lds_u32x2*>(lds + r * 256 + ((c ^ (r & 15)) << 4) + 8 * (lane >> 5)) =
            u32x2{v.x, v.y};
      }
  TT_LDS_BARRIER();
  const int c = tid & 15;
  if (j0 + 8 * c >= K) return;
#pragma unroll
  for (int p = 0; p < D_BM / 16; ++p) {
    const int r = 16 * p + (tid >> 4);
    if (r < rows)
      *reinterpret_cast<uint4*>(dx + ((t.seg0 + i0 + r) * K + j0 + 8 * c) * 2) =
          read_k(lds, (uint32_t)(r * 256 + ((c ^ (r & 15)) << 4)));
  }
}

// The same in tiles of 256 x 256, one block per CU, for launches with enough of them: a wave
// multiplies 128 x 128, so that an LDS byte serves twice the products of the smaller tile (whose
// fragment reads bound it). One wave per SIMD: the fragments of a step are read during the step
// before it, and the barrier stands before a k-tile's last step, whose fragments are in registers by
// then. The next k-tile's codes become bf16 during the third step; loads for the one after it
// go out after the barrier.
constexpr int G_BM = 256, G_BN = 256;
constexpr int G_A = G_BM * D_BK * 2, G_STAGE = G_A + G_BN * D_BK * 2;

__global__ __launch_bounds__(D_NT, 1) void mx_dgrad_big_kernel(
    const char* __restrict__ dy, const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
    char* __restrict__ dx, int64_t M, int64_t K, int64_t N, int E,
    const int64_t* __restrict__ counts, int tiles_j) {
  __shared__ __align__(16) char lds_raw[2 * G_STAGE];
  RowTile t;
  if (counts != nullptr) {
    if (!row_tile<G_BM, D_NT>(counts, E, tiles_j, lds_raw, t)) return;
    // Counts that sum to more than M end at its last row.
    if (t.seg0 + t.nrows > M) t.nrows = M - t.seg0;
    if ((int64_t)t.mt * G_BM >= t.nrows) return;
  } else {
    dense_tile(t, M, (int)((M + G_BM - 1) / G_BM), tiles_j);
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t i0 = (int64_t)t.mt * G_BM, j0 = (int64_t)t.nt * G_BN;
  const int64_t rows = t.nrows - i0;
  const int nkt = (int)((N + D_BK - 1) / D_BK);
  lds_char* const lds = (lds_char*)lds_raw;

  // dy: wave w loads rows 64 w + 8 q + lane / 8.
  const i32x4 ra = make_rsrc(dy + (t.seg0 + i0) * N * 2, (rows < G_BM ? rows : G_BM) * N * 2);
  const uint32_t aoff0 = (uint32_t)((64 * wave + (lane >> 3)) * N) * 2u;
  // W: thread t takes pieces t and t + 256 of a k-tile's 64 rows of eight groups.
  const int64_t groups = K / MX_GROUP;
  int64_t wg = j0 / MX_GROUP + (tid & 7);
  wg = wg < groups ? wg : groups - 1;
  const uint8_t* const wp = w + (int64_t)t.e * N * (K / 2) + wg * 16;
  const uint8_t* const wsp = ws + (int64_t)t.e * N * groups + wg;
  // 16 lanes take two rows four apart: with the swizzle below, all banks.
  const int a0 = tid >> 3;
  const int wr0 = ((a0 >> 1) & 3) + 4 * (a0 & 1) + 8 * (a0 >> 3);  // the second piece: row + 32

  uint4 wv[2];
  uint32_t wsv[2];
  // k-tiles past the last one read nothing of dy, and W's last row again.
  auto load_w = [&](int kt, int h) {
    const int n = kt * D_BK + wr0 + 32 * h;
    const uint32_t at = (uint32_t)(n < (int)N ? n : (int)N - 1);
    wv[h] = *reinterpret_cast<const uint4*>(wp + (uint64_t)at * (uint32_t)(K / 2));
    wsv[h] = wsp[(uint64_t)at * (uint32_t)groups];
  };
  auto load_dy = [&](int kt, int buf, int q, i32x4 rk) {
    const int r = 8 * q + (lane >> 3);  // row of the wave's 64
    const int c = (lane & 7) ^ ((r >> 1) & 7);
    const uint32_t off = aoff0 + (uint32_t)(8 * q * N) * 2u + 16u * (uint32_t)c;
    dma16(kt * D_BK + 8 * c < (int)N ? off : DM_OOB, rk,
          lds_addr_of(lds) + (uint32_t)(buf * G_STAGE) + (uint32_t)(8 * wave + q) * 1024u);
  };
  // Chunk c (eight columns) of k-row r lies in slot c ^ (4 (r % 4)) ^ (r / 4 % 2) ^ (2 (c / 16)).
  auto put = [&](int buf, int kt, int n) {
    const int h = n >> 2, i = n & 3;
    const int wr = wr0 + 32 * h, c = 4 * (tid & 7) + i;
    const uint32_t q = i == 0 ? wv[h].x : i == 1 ? wv[h].y : i == 2 ? wv[h].z : wv[h].w;
    // Scale 2^-127 where dy is zero: a NaN scale would not vanish.
    const uint4 v = mx_bf16x8(q, kt * D_BK + wr0 + 32 * h < (int)N ? wsv[h] : 0u);
    *reinterpret_cast<lds_u32x4*>(
        lds + buf * G_STAGE + G_A + wr * 512 +
        ((c ^ (4 * (wr & 3)) ^ ((wr >> 2) & 1) ^ (2 * (c >> 4))) << 4)) = u32x4{v.x, v.y, v.z, v.w};
  };
  const int m0 = 128 * (wave >> 1), n0 = 128 * (wave & 1);
  uint32_t fa[4], fb[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) fa[s] = fragk64(m0, s, lane);
  {
    const int g = lane >> 4, i = lane & 15;
    const int kr = 8 * (g >> 1) + (i >> 2);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = n0 + 32 * j + 16 * (g & 1) + 4 * (i & 3), c = col >> 3;
      fb[j] = G_A + (uint32_t)(kr * 512 + (col & 7) * 2 +
                               ((c ^ (4 * (kr & 3)) ^ ((kr >> 2) & 1) ^ (2 * (c >> 4))) << 4));
    }
  }
  f32x16 acc[4][4] = {};
  uint4 fra[2][4];
  uint2 frb[2][8];
  // Fragment reads of a step, twelve: in the order in which the products need them.
  auto read = [&](int buf, int s, int to, int n) {
    lds_char* const st = lds + buf * G_STAGE;
    if (n >= 2 && n < 6) {
      fra[to][n - 2] = read_k(st, fa[s] + (n - 2) * 4096);
      return;
    }
    const int v = n < 2 ? n : n - 4, j = v >> 1;
    // The second half: four k-rows on, 2048 bytes and the other slot of a pair.
    const uint32_t at = fb[j] + s * 8192;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_i16x4*)(st + (v & 1 ? (at ^ 16) + 2048 : at)));
    frb[to][v] = __builtin_bit_cast(uint2, x);
  };
  auto product = [&](int from, int n) {
    const int i = n & 3, j = n >> 2;
    const uint2 lo = frb[from][2 * j], hi = frb[from][2 * j + 1];
    acc[i][j] = Mma<TT_BF16>::run(uint4{lo.x, lo.y, hi.x, hi.y}, fra[from][i], acc[i][j]);
  };
  if (nkt > 0) {
    load_w(0, 0);
    load_w(0, 1);
#pragma unroll
    for (int q = 0; q < 8; ++q) load_dy(0, 0, q, ra);
#pragma unroll
    for (int n = 0; n < 8; ++n) put(0, 0, n);
    TT_WAIT_VMCNT(0);
    TT_LDS_BARRIER();
    load_w(1, 0);
    load_w(1, 1);
    const i32x4 r1 = advance_rsrc(ra, D_BK * 2);
#pragma unroll
    for (int q = 0; q < 8; ++q) load_dy(1, 1, q, r1);
#pragma unroll
    for (int n = 0; n < 12; ++n) read(0, 0, 0, n);
    for (int kt = 0; kt < nkt; ++kt) {
      const int buf = kt & 1;
      // Each product is followed by a share of the step's other work, in this order.
#pragma unroll
      for (int s = 0; s < 3; ++s) {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          product(s & 1, n);
          if (n < 12) read(buf, s + 1, (s & 1) ^ 1, n);
          if (s == 2 && (n & 1) == 1) put(buf ^ 1, kt + 1, n >> 1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      TT_WAIT_VMCNT(0);
      TT_LDS_BARRIER();
      const i32x4 rk = advance_rsrc(ra, (uint32_t)(kt + 2) * (D_BK * 2));
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        product(1, n);
        if (n < 12) read(buf ^ 1, 0, 0, n);
        if (n < 2) load_w(kt + 2, n);
        if (n >= 2 && (n & 1) == 0) load_dy(kt + 2, buf, n / 2 - 1, rk);
        if (n == 15) load_dy(kt + 2, buf, 7, rk);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    TT_WAIT_VMCNT(0);
  }
  // A wave's 128 x 128 outputs through 32 KiB of LDS of its own, rows of 256 bytes.
  TT_LDS_BARRIER();
  lds_char* const out = lds + wave * 32768;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 32 * i + (lane & 31), c = 4 * j + q;
        const uint2 v = pack4<TT_BF16>(acc[i][j][4 * q], acc[i][j][4 * q + 1],
                                       acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        *reinterpret_cast<lds_u32x2*>(out + r * 256 + ((c ^ (r & 15)) << 4) + 8 * (lane >> 5)) =
            u32x2{v.x, v.y};
      }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const int64_t col = j0 + n0 + 8 * (lane & 15);
  if (col >= K) return;
#pragma unroll 8
  for (int p = 0; p < 32; ++p) {
    const int r = 4 * p + (lane >> 4);
    if (m0 + r < rows)
      *reinterpret_cast<uint4*>(dx + ((t.seg0 + i0 + m0 + r) * K + col) * 2) =
          read_k(out, (uint32_t)(r * 256 + (((lane & 15) ^ (r & 15)) << 4)));
  }
}

}  // namespace

extern "C" int tt_mx_dgrad(const void* dy, const uint8_t* codes, const uint8_t* scales, int64_t M,
                           int64_t K, int64_t N, int32_t num_experts,
                           const int64_t* tokens_per_expert, void* dx, void* stream) {
  TT_REQUIRE(M >= 0 && K >= 0 && N >= 0 && num_experts > 0, "mx dgrad: bad sizes");
  TT_REQUIRE(K % MX_GROUP == 0, "mx dgrad: the weights' rows are whole groups of 32 elements");
  TT_REQUIRE(K < (1ll << 31) && N < (1ll << 24) && M < (1ll << 31) && num_experts <= 65536,
             "mx dgrad: sizes past 2^31 (2^24 columns)");
  TT_REQUIRE(tokens_per_expert != nullptr || num_experts == 1,
             "mx dgrad: several experts need their counts");
  if (M == 0 || K == 0) return TT_OK;
  TT_REQUIRE(dx != nullptr && (N == 0 || (dy != nullptr && codes != nullptr && scales != nullptr)),
             "mx dgrad: NULL tensor");
  TT_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(dx)) & 15) == 0,
             "mx dgrad: codes and dx must be 16-byte aligned");
  const bool aligned = N % 8 == 0 && (reinterpret_cast<uintptr_t>(dy) & 15) == 0;
  // Tiles of 256 x 256 where the launch has at least one for each of 256 CUs and experts fill them.
  const bool big = aligned && N < (1ll << 22) && M / num_experts >= 256 &&
                   (M / G_BM) * (K / G_BN) >= 256;
  const int64_t bm = big ? G_BM : D_BM, bn = big ? G_BN : D_BN;
  const int64_t tiles_j = (K + bn - 1) / bn;
  int64_t tiles_i = (M + bm - 1) / bm;
  if (tokens_per_expert != nullptr) tiles_i = M / bm + (num_experts < M ? num_experts : M);
  TT_REQUIRE(tiles_i * tiles_j < (1ll << 31) && tt_grid_ok(tiles_i * tiles_j, D_NT),
             "mx dgrad: grid too large");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(tiles_i * tiles_j));
  if (big)
    hipLaunchKernelGGL(mx_dgrad_big_kernel, grid, dim3(D_NT), 0, s, static_cast<const char*>(dy),
                       codes, scales, static_cast<char*>(dx), M, K, N, num_experts,
                       tokens_per_expert, (int)tiles_j);
  else if (aligned)
    hipLaunchKernelGGL((mx_dgrad_kernel<true>), grid, dim3(D_NT), 0, s, static_cast<const char*>(dy),
                       codes, scales, static_cast<char*>(dx), M, K, N, num_experts,
                       tokens_per_expert, (int)tiles_j);
  else
    hipLaunchKernelGGL((mx_dgrad_kernel<false>), grid, dim3(D_NT), 0, s,
                       static_cast<const char*>(dy), codes, scales, static_cast<char*>(dx), M, K, N,
                       num_experts, tokens_per_expert, (int)tiles_j);
  return tt_check_launch("mx_dgrad");
}
