// Product of many rows with 4-bit weights (gfx950): prompts, training, experts of many rows.
//
// A block computes 128 rows by 256 weight rows (gated: 128 columns, a wave's blocks of 32 weight
// rows alternating between gates and their ups), four waves of 64 x 128 each on 32-wide matrix
// instructions. k-tiles go from memory straight to LDS, swizzled so that fragment reads are
// free of bank conflicts; two blocks share a CU, so that one's matrix instructions cover the
// other's waits, prologue and epilogue. Rows of 4-bit weights are a quarter of bf16 rows' bytes
// (half of E4M3 rows'), which is why the tile is twice as wide in them.
//
// E4M3 rows: k-tiles of 128, two stages; codes are multiplied as they are, with the groups' bytes as
// the instruction's scales (a row's four bytes of a k-tile are one word in LDS).
// bf16 rows: k-tiles of 64, three stages; a lane's 16 bytes of codes are one group of a weight row,
// which it turns into four bf16 fragments with the group's scale. The order of the reduction
// within a k-tile is free as long as both operands agree: lane half g of step s takes elements
// 32 g + 8 s .. + 7.
#include <type_traits>

#include "mx_gemm.h"

namespace {

constexpr int T_NT = 256, T_BM = 128, T_BN = 256;

template <bool MX>
struct Tile {
  static constexpr int BK = MX ? 128 : 64;
  static constexpr int STAGES = MX ? 2 : 3;
  static constexpr int XB = T_BM * 128;              // rows of x: 128 bytes per k-tile
  static constexpr int WR = MX ? 64 : 32;            // bytes of a weight row per k-tile
  static constexpr int WB = T_BN * WR;
  static constexpr int STAGE = XB + WB;
  // Scales of 128 elements, one word per row: weight rows, then x's; two buffers.
  static constexpr int SB = (T_BN + (MX ? T_BM : 0)) * 4;
  static constexpr int LDS = STAGES * STAGE + 2 * SB;
};

// Bytes 0..3 of a scale word: groups past the reduction's end are 127 (their codes are zeros).
__device__ __forceinline__ uint32_t scale_word(const uint8_t* p, int left) {
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) v |= (i < left ? (uint32_t)p[i] : 127u) << (8 * i);
  return v;
}

// KA: K is a multiple of 128 and scales are 4-byte aligned.
template <bool MX, bool GATED, bool OUT8, bool KA>
__global__ __launch_bounds__(T_NT, 2) void mx_tile_kernel(MxArgs p, int tiles_j) {
  typedef Tile<MX> L;
  constexpr int CB = GATED ? T_BN / 2 : T_BN;  // output columns
  constexpr int ES = MX ? 1 : 2;               // bytes of an element of x
  __shared__ __align__(16) char lds_raw[L::LDS];
  RowTile t;
  if (p.counts != nullptr) {
    if (!row_tile<T_BM, T_NT>(p.counts, p.E, tiles_j, lds_raw, t)) return;
    // Counts that sum to more than M end at its last row.
    if (t.seg0 + t.nrows > p.M) t.nrows = p.M - t.seg0;
    if ((int64_t)t.mt * T_BM >= t.nrows) return;
  } else {
    t.e = 0;
    const int tiles_i = (int)((p.M + T_BM - 1) / T_BM);
    const int slot = xcd_remap(blockIdx.x, tiles_i * tiles_j);
    t.mt = slot % tiles_i;
    t.nt = slot / tiles_i;
    t.seg0 = 0;
    t.nrows = p.M;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t K = p.K, i0 = (int64_t)t.mt * T_BM, j0 = (int64_t)t.nt * CB;
  const int64_t rows = t.nrows - i0;  // valid rows of the tile, at least one
  const int groups = (int)(K / MX_GROUP);
  const int nkt = (int)((K + L::BK - 1) / L::BK);
  lds_char* const lds = (lds_char*)lds_raw;
  lds_char* const lds_s = lds + L::STAGES * L::STAGE;

  // x: wave w loads rows 32 w + 8 q + lane / 8, chunk slot lane % 8 holding chunk
  // slot ^ ((row >> 1) & 7). Rows past the expert's read as zeros.
  const bool gather = p.arow != nullptr;
  const int64_t first = t.seg0 + i0;
  const char* const xbase = static_cast<const char*>(p.x) + (gather ? 0 : first * K * ES);
  const i32x4 rx = make_rsrc(xbase, (gather ? p.src_rows : (rows < T_BM ? rows : T_BM)) * K * ES);
  uint32_t xoff[4];
  int xk[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = 32 * wave + 8 * q + (lane >> 3);
    const int c = (lane & 7) ^ ((r >> 1) & 7);
    xk[q] = c * (16 / ES);
    xoff[q] = DM_OOB;
    if (r < rows) xoff[q] = (uint32_t)((gather ? mx_source_row(p, first + r) : r) * K * ES + 16 * c);
  }
  // W: rows of WR bytes. Tile row r is weight row `weight_row(r)`; those past the last read it again
  // (their columns are not stored). A wave's instruction covers 1 KiB.
  const int64_t width = GATED ? 2 * p.N : p.N;
  const uint8_t* const wbase = p.w + (int64_t)t.e * width * (K / 2);
  const uint8_t* const sbase = p.ws + (int64_t)t.e * width * groups;
  const i32x4 rw = make_rsrc(wbase, width * (K / 2));
  const i32x4 rs = make_rsrc(sbase, width * groups);
  auto weight_row = [&](int r) -> int64_t {
    int64_t n = GATED ? j0 + 32 * (r >> 6) + (r & 31) : j0 + r;
    n = n < p.N ? n : p.N - 1;
    return GATED && (r & 32) ? n + p.N : n;
  };
  constexpr int WQ = L::WB / 4096;  // instructions per wave
  constexpr int CW = L::WR / 16;    // chunks of a row
  uint32_t woff[WQ];
  int wk[WQ];
#pragma unroll
  for (int q = 0; q < WQ; ++q) {
    const int r = (64 * wave) + (64 / CW) * q + lane / CW;
    const int c = (lane % CW) ^ (MX ? (r >> 2) & 3 : (r >> 3) & 1);
    wk[q] = 32 * c;
    woff[q] = (uint32_t)(weight_row(r) * (K / 2) + 16 * c);
  }
  // Scales: thread t takes weight row t, and of x row t % 128 (the first 128 threads).
  const int64_t srow = weight_row(tid);
  const uint32_t soff = (uint32_t)(srow * groups);
  const uint8_t* const xsbase = MX ? p.xs + (gather ? 0 : first * groups) : nullptr;
  const i32x4 rxs = make_rsrc(xsbase, MX ? (gather ? p.src_rows : (rows < T_BM ? rows : T_BM)) * groups : 0);
  uint32_t xsoff = DM_OOB;
  if (MX && tid < T_BM && tid < rows)
    xsoff = (uint32_t)((gather ? mx_source_row(p, first + tid) : tid) * groups);

  // The words of 128 elements from group g0 on into scale buffer b.
  auto load_scales = [&](int g0, int b) {
    const uint32_t at = lds_addr_of(lds_s) + (uint32_t)(b * L::SB);
    if constexpr (KA) {
      dma4(soff, advance_rsrc(rs, (uint32_t)g0), at + 256u * wave);
      if (MX && wave < 2)
        dma4(xsoff, advance_rsrc(rxs, (uint32_t)g0), at + T_BN * 4 + 256u * wave);
    } else {
      uint32_t* const to = reinterpret_cast<uint32_t*>(lds_raw + L::STAGES * L::STAGE + b * L::SB);
      to[tid] = scale_word(sbase + soff + g0, groups - g0);
      if constexpr (MX)
        if (tid < T_BM) to[T_BN + tid] = xsoff == DM_OOB ? 0x7f7f7f7fu : scale_word(xsbase + xsoff + g0, groups - g0);
    }
  };
  auto issue = [&](int kt, int stage) {
    const uint32_t base = lds_addr_of(lds) + (uint32_t)(stage * L::STAGE);
    const i32x4 rxk = advance_rsrc(rx, (uint32_t)(kt * L::BK * ES));
    const i32x4 rwk = advance_rsrc(rw, (uint32_t)(kt * (L::BK / 2)));
#pragma unroll
    for (int q = 0; q < 4; ++q)
      dma16(KA || kt * L::BK + xk[q] < (int)K ? xoff[q] : DM_OOB, rxk,
            base + (uint32_t)(4 * wave + q) * 1024u);
#pragma unroll
    for (int q = 0; q < WQ; ++q)
      dma16(KA || kt * L::BK + wk[q] < (int)K ? woff[q] : DM_OOB, rwk,
            base + L::XB + (uint32_t)(WQ * wave + q) * 1024u);
    if (MX || (kt & 1) == 0) load_scales(kt * (L::BK / MX_GROUP), MX ? kt & 1 : (kt >> 1) & 1);
  };

  // Wave w multiplies rows 64 (w / 2) .. + 63 by weight rows 128 (w % 2) .. + 127.
  const int m0 = 64 * (wave >> 1), n0 = 128 * (wave & 1);
  const int r32 = lane & 31, g = lane >> 5;
  f32x16 acc[2][4] = {};
  auto multiply = [&](int kt, int stage) {
    lds_char* const st = lds + stage * L::STAGE;
    const char* const sw = lds_raw + L::STAGES * L::STAGE + (MX ? kt & 1 : (kt >> 1) & 1) * L::SB;
    const int shift = MX ? 8 * g : 8 * (2 * (kt & 1) + g);
    uint32_t ws[4], xs[2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      ws[j] = *reinterpret_cast<const uint32_t*>(sw + 4 * (n0 + 32 * j + r32)) >> shift;
    if constexpr (MX) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        xs[i] = *reinterpret_cast<const uint32_t*>(sw + 4 * (T_BN + m0 + 32 * i + r32)) >> shift;
      auto step = [&](auto sc) {
        constexpr int s = decltype(sc)::value;
        uint4 w[4], x[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = m0 + 32 * i + r32;
          const uint32_t at = (uint32_t)(r * 128), sz = (uint32_t)((r >> 1) & 7);
          x[i][0] = read_k(st, at + (((4 * s + g) ^ sz) << 4));
          x[i][1] = read_k(st, at + (((4 * s + 2 + g) ^ sz) << 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = n0 + 32 * j + r32;
          w[j] = read_k(st, L::XB + (uint32_t)(r * 64 + (((2 * s + g) ^ ((r >> 2) & 3)) << 4)));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            acc[i][j] = mx_mma32<2 * s, 2 * s>(w[j], x[i][0], x[i][1], ws[j], xs[i], acc[i][j]);
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
    } else {
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = n0 + 32 * j + r32;
        w[j] = read_k(st, L::XB + (uint32_t)(r * 32 + ((g ^ ((r >> 3) & 1)) << 4)));
        ws[j] &= 255u;
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint4 x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = m0 + 32 * i + r32;
          x[i] = read_k(st, (uint32_t)(r * 128 + (((4 * g + s) ^ ((r >> 1) & 7)) << 4)));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t q = s == 0 ? w[j].x : s == 1 ? w[j].y : s == 2 ? w[j].z : w[j].w;
          const uint4 a = mx_bf16x8(q, ws[j]);
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[i][j] = Mma<TT_BF16>::run(a, x[i], acc[i][j]);
        }
      }
    }
  };

#pragma unroll
  for (int s = 0; s < L::STAGES - 1; ++s)
    if (s < nkt) issue(s, s);
  int stage = 0;
  for (int kt = 0; kt < nkt; ++kt) {
    // k-tile kt has landed once at most the loads of later ones are outstanding: at least the x and
    // W pieces of kt + 1 where three stages are used.
    if (L::STAGES == 3 && KA && kt + 1 < nkt) TT_WAIT_VMCNT(4 + WQ);
    else TT_WAIT_VMCNT(0);
    TT_LDS_BARRIER();
    const int next = stage == 0 ? L::STAGES - 1 : stage - 1;  // the stage of kt - 1
    if (kt + L::STAGES - 1 < nkt) issue(kt + L::STAGES - 1, next);
    multiply(kt, stage);
    stage = stage == L::STAGES - 1 ? 0 : stage + 1;
  }

  // Epilogue. Register 4 q + e of lane l in block (i, j): row m0 + 32 i + l % 32, weight row
  // n0 + 32 j + 8 q + 4 g + e. A wave's rows go through its own 16 KiB of LDS, in rows of RB bytes,
  // chunk c of row r in slot c ^ (r % (RB / 16)).
  TT_LDS_BARRIER();  // every wave is past its fragment reads
  constexpr int JN = GATED ? 2 : 4;              // 32-column blocks of a wave
  constexpr int RB = 32 * JN * (OUT8 ? 1 : 2);   // bytes of a row
  lds_char* const out = lds + wave * 16384;
  const int64_t c0 = j0 + (GATED ? n0 / 2 : n0);  // the wave's first column
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * i + r32;
    const int64_t row = first + m0 + r;
    const bool valid = m0 + r < rows;
    float f = 1.f;
    if (p.probs != nullptr && valid) f = load_as_f32(p.probs, p.pdt, row);
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if constexpr (GATED) v[e] = mx_act(acc[i][2 * j][e], p.act) * acc[i][2 * j + 1][e];
        else v[e] = mx_act(acc[i][j][e], p.act);
        if (p.probs != nullptr) v[e] *= f;
      }
      if constexpr (OUT8) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, TT_WAVE));
        const uint32_t byte = mx_byte<8>(m);
        const float s = mx_inverse(byte == 255u ? 127u : byte);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t code = byte == 255u ? 0x7f7f7f7fu
                                             : mx_e4m3x4(v[4 * q] * s, v[4 * q + 1] * s,
                                                         v[4 * q + 2] * s, v[4 * q + 3] * s);
          const int c = 2 * j + (q >> 1);
          *reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(
              out + r * RB + ((c ^ (r & (RB / 16 - 1))) << 4) + 8 * (q & 1) + 4 * g) = code;
        }
        if (g == 0 && valid && c0 + 32 * j < p.N)
          p.ys[row * (p.N / MX_GROUP) + (c0 + 32 * j) / MX_GROUP] = (uint8_t)byte;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint2 a = pack4<TT_BF16>(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          const int c = 4 * j + q;
          *reinterpret_cast<lds_u32x2*>(out + r * RB + ((c ^ (r & (RB / 16 - 1))) << 4) + 8 * g) =
              u32x2{a.x, a.y};
        }
      }
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int LR = RB / 16;                      // lanes of a row
  constexpr int PER = OUT8 ? 16 : 8;               // elements of a chunk
  const int64_t col = c0 + PER * (lane % LR);
  const bool whole = OUT8 || (p.N & 7) == 0;
#pragma unroll
  for (int q = 0; q < LR; ++q) {
    const int r = q * (64 / LR) + lane / LR;
    if (m0 + r >= rows || col >= p.N) continue;
    const uint4 v = read_k(out, (uint32_t)(r * RB + (((lane % LR) ^ (r & (LR - 1))) << 4)));
    char* const to = static_cast<char*>(p.y) + ((first + m0 + r) * p.N + col) * (OUT8 ? 1 : 2);
    if (whole) {
      *reinterpret_cast<uint4*>(to) = v;
    } else {
      const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < p.N) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(d[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <bool MX, bool GATED, bool OUT8, bool KA>
int launch(const MxArgs& p, hipStream_t s) {
  constexpr int CB = GATED ? T_BN / 2 : T_BN;
  const int64_t tiles_j = (p.N + CB - 1) / CB;
  int64_t tiles_i = (p.M + T_BM - 1) / T_BM;
  if (p.counts != nullptr) tiles_i = p.M / T_BM + (p.E < p.M ? p.E : p.M);
  TT_REQUIRE(tiles_i * tiles_j < (1ll << 31) && tt_grid_ok(tiles_i * tiles_j, T_NT),
             "mx product: grid too large");
  hipLaunchKernelGGL((mx_tile_kernel<MX, GATED, OUT8, KA>), dim3((unsigned)(tiles_i * tiles_j)),
                     dim3(T_NT), 0, s, p, (int)tiles_j);
  return tt_check_launch("mx_tile");
}

template <bool MX, bool GATED, bool OUT8>
int aligned(const MxArgs& p, hipStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.xs);
  return p.K % 128 == 0 && (at & 3) == 0 ? launch<MX, GATED, OUT8, true>(p, s)
                                         : launch<MX, GATED, OUT8, false>(p, s);
}

template <bool MX, bool GATED>
int out(const MxArgs& p, hipStream_t s) {
  return p.ys != nullptr ? aligned<MX, GATED, true>(p, s) : aligned<MX, GATED, false>(p, s);
}

}  // namespace

bool tt_mx_tile_takes(const MxArgs& p, bool gated) {
  const int64_t es = p.xs != nullptr ? 1 : 2, width = gated ? 2 * p.N : p.N;
  // 32-bit offsets within an expert's weights, a tile's rows, and a gathered source.
  return p.K > 0 && width * (p.K / 2) < (1ll << 31) && T_BM * p.K * es < (1ll << 31) &&
         (p.arow == nullptr || p.src_rows * p.K * es < (1ll << 31)) &&
         (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
}

int tt_mx_tile(const MxArgs& p, bool gated, hipStream_t s) {
  if (p.xs != nullptr) return gated ? out<true, true>(p, s) : out<true, false>(p, s);
  return gated ? out<false, true>(p, s) : out<false, false>(p, s);
}
