// Product of many rows with 4-bit weights (gfx950): prompts, training, experts of many rows.
//
// A block computes 128 rows by 256 weight rows (gated: 128 columns, a wave's blocks of 32 weight
// rows alternating between gates and their ups), four waves of 64 x 128 each on 32-wide matrix
// instructions; 128 x 128 or 64 x 128 where the launch would have too few blocks, and dense products
// of fewer still split their reduction, the parts' sums joined in order by a second kernel. Where
// 128 x 128 gives most CUs one block, two sets of four waves take half of the reduction each. Long
// reductions of E4M3 rows take 256 x 256 in one block of eight waves with three stages: half the
// reads, and loads two k-tiles ahead. k-tiles go from memory straight to LDS, swizzled so that
// fragment reads are free of bank conflicts; otherwise two blocks share a CU, so that one's matrix
// instructions cover the other's waits, prologue and epilogue. Rows of 4-bit weights are a quarter of
// bf16 rows' bytes (half of E4M3 rows'), which is why the tile is twice as wide in them.
//
// Reductions off 128 and scales off four bytes take 128 x 128, unsplit: the scales of a k-tile come by
// single bytes through registers, and every k-tile waits for all of its loads. us at 7136 -> 2 x 2048, for
// those at 7168: 128 rows 116 / 23, 1531 rows 155 / 109, 4096 rows 320 / 214; E4M3 rows 93 / 20, 155 / 64,
// 316 / 105; 32 experts of 64 rows, 2016 -> 2 x 1024, for 2048 52 / 35, of 512 rows 213 / 147.
//
// E4M3 rows: k-tiles of 128, two stages (four of the smallest tile); codes are multiplied as they
// are, with the groups' bytes as the instruction's scales (a row's four bytes of a k-tile are one
// word in LDS).
// bf16 rows: k-tiles of 64, three stages; a lane's 16 bytes of codes are one group of a weight row,
// which it turns into four bf16 fragments with the group's scale. The order of the reduction
// within a k-tile is free as long as both operands agree: lane half g of step s takes elements
// 32 g + 8 s .. + 7.
#include <type_traits>

#include "mx_gemm.h"

namespace {

template <bool MX, int BM_, int BN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_;           // rows of x and of W
  static constexpr int NW = BM == 256 ? 8 : 4;       // waves: MW along the rows, two along W's
  static constexpr int MW = BM == 256 ? 4 : 2, WN = BN / 2;
  static constexpr int BK = MX ? 128 : 64;
  static constexpr int STAGES = !MX || BM == 256 ? 3 : BM == 64 ? 4 : 2;
  static constexpr int XB = BM * 128;                // rows of x: 128 bytes per k-tile
  static constexpr int WR = MX ? 64 : 32;            // bytes of a weight row per k-tile
  static constexpr int WB = BN * WR;
  static constexpr int STAGE = XB + WB;
  // Scales of 128 elements, one word per row: weight rows, then x's. A buffer per stage, or two where
  // a word lasts two k-tiles.
  static constexpr int SB = (BN + (MX ? BM : 0)) * 4;
  static constexpr int SBS = MX ? STAGES : 2;
  static constexpr int LDS = STAGES * STAGE + SBS * SB;
  static constexpr int MI = BM / MW / 32, NJ = WN / 32;   // 32-wide blocks of a wave
};

// Bytes 0..3 of a scale word: groups past the reduction's end are 127 (their codes are zeros).
__device__ __forceinline__ uint32_t scale_word(const uint8_t* p, int left) {
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) v |= (i < left ? (uint32_t)p[i] : 127u) << (8 * i);
  return v;
}

// Epilogue of a wave's MI x NJ blocks: register 4 q + e of lane l in block (i, j) is row
// m0 + MS i + l % 32 of the tile's (`rows` valid, the first is output row `first`), weight row
// 32 j + 8 q + 4 (l / 32) + e of the wave's; gated: odd blocks are the ups of the even ones. Output
// columns from c0. Rows go through the wave's own LDS at `out`, RB bytes each, chunk c of row r in
// slot c ^ (r % (RB / 16)).
template <bool GATED, bool OUT8, int MI, int NJ, int MS>
__device__ __forceinline__ void mx_tile_store(const MxArgs& p, const f32x16 (&acc)[MI][NJ],
                                              lds_char* out, int64_t first, int64_t rows, int m0,
                                              int64_t c0) {
  constexpr int JN = GATED ? NJ / 2 : NJ;        // 32-column blocks of a wave
  constexpr int RB = 32 * JN * (OUT8 ? 1 : 2);   // bytes of a row
  const int lane = lane_id(), r32 = lane & 31, g = lane >> 5;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r = 32 * i + r32;
    const int64_t row = first + m0 + MS * i + r32;
    const bool valid = m0 + MS * i + r32 < rows;
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
  for (int q = 0; q < MI * LR / 2; ++q) {
    const int r = q * (64 / LR) + lane / LR, at = m0 + MS * (r >> 5) + (r & 31);
    if (at >= rows || col >= p.N) continue;
    const uint4 v = read_k(out, (uint32_t)(r * RB + (((lane % LR) ^ (r & (LR - 1))) << 4)));
    char* const to = static_cast<char*>(p.y) + ((first + at) * p.N + col) * (OUT8 ? 1 : 2);
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

// KA: K is a multiple of 128 and scales are 4-byte aligned. KS = 2: two sets of waves with stages of their
// own take a half of the reduction each, and exchange halves of their sums at its end.
template <bool MX, bool GATED, bool OUT8, bool KA, int T_BM, int T_BN, int KS>
__global__ __launch_bounds__((T_BM == 256 || KS == 2 ? 512 : 256), (T_BM == 256 || KS == 2 ? 1 : 2))
void mx_tile_kernel(MxArgs p, int tiles_j, int parts) {
  typedef Tile<MX, T_BM, T_BN> L;
  constexpr int CB = GATED ? T_BN / 2 : T_BN;  // output columns
  constexpr int ES = MX ? 1 : 2;               // bytes of an element of x
  constexpr int MI = L::MI, NJ = L::NJ, NW = L::NW, NT = 64 * NW * KS;
  static_assert(KS == 1 || (KA && MI == 2 && NW == 4), "halves exchange one of two blocks of rows");
  __shared__ __align__(16) char lds_block[KS * L::LDS];
  RowTile t;
  int tile = 0, part = 0;  // of a dense product
  if (p.counts != nullptr) {
    if (!row_tile<T_BM, NT>(p.counts, p.E, tiles_j, lds_block, t)) return;
    // Counts that sum to more than M end at its last row.
    if (t.seg0 + t.nrows > p.M) t.nrows = p.M - t.seg0;
    if ((int64_t)t.mt * T_BM >= t.nrows) return;
  } else {
    t.e = 0;
    const int tiles_i = (int)((p.M + T_BM - 1) / T_BM);
    const int slot = xcd_remap(blockIdx.x, tiles_i * tiles_j * parts);
    part = slot % parts;
    // Eight row tiles at a time: the blocks that an XCD has at work read few panels of either operand.
    const int at = slot / parts, group = 8 * tiles_j, m0 = at / group * 8;
    const int gm = tiles_i - m0 < 8 ? tiles_i - m0 : 8;
    t.mt = m0 + at % group % gm;
    t.nt = at % group / gm;
    tile = t.nt * tiles_i + t.mt;
    t.seg0 = 0;
    t.nrows = p.M;
  }
  const int half = KS == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int tid = threadIdx.x - 256 * half, lane = tid & 63;
  char* const lds_raw = lds_block + half * L::LDS;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t K = p.K, i0 = (int64_t)t.mt * T_BM, j0 = (int64_t)t.nt * CB;
  const int64_t rows = t.nrows - i0;  // valid rows of the tile, at least one
  const int groups = (int)(K / MX_GROUP);
  const int nkt = (int)((K + L::BK - 1) / L::BK);
  lds_char* const lds = (lds_char*)lds_raw;
  lds_char* const lds_s = lds + L::STAGES * L::STAGE;

  // x: wave w loads rows 8 (XQ w + q) + lane / 8, chunk slot lane % 8 holding chunk
  // slot ^ ((row >> 1) & 7). Rows past the expert's read as zeros.
  const bool gather = p.arow != nullptr;
  const int64_t first = t.seg0 + i0;
  const char* const xbase = static_cast<const char*>(p.x) + (gather ? 0 : first * K * ES);
  const i32x4 rx = make_rsrc(xbase, (gather ? p.src_rows : (rows < T_BM ? rows : T_BM)) * K * ES);
  constexpr int XQ = T_BM / 8 / NW;  // instructions per wave
  uint32_t xoff[XQ];
  int xk[XQ];
#pragma unroll
  for (int q = 0; q < XQ; ++q) {
    const int r = 8 * XQ * wave + 8 * q + (lane >> 3);
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
    int64_t n = GATED ? j0 + 32 * (r >> 6) + (r & 31) : j0 + r;  // gated: 32 gates, their 32 ups
    n = n < p.N ? n : p.N - 1;
    return GATED && (r & 32) ? n + p.N : n;
  };
  constexpr int WQ = L::WB / 1024 / NW;  // instructions per wave
  constexpr int CW = L::WR / 16;    // chunks of a row
  uint32_t woff[WQ];
  int wk[WQ];
#pragma unroll
  for (int q = 0; q < WQ; ++q) {
    const int r = (64 / CW) * (WQ * wave + q) + lane / CW;
    const int c = (lane % CW) ^ (MX ? (r >> 2) & 3 : (r >> 3) & 1);
    wk[q] = 32 * c;
    woff[q] = (uint32_t)(weight_row(r) * (K / 2) + 16 * c);
  }
  // Scales: thread t takes weight row t, and row t of x (of eight waves the last four do).
  const int xt = tid - (NW == 8 ? 256 : 0), xw = wave - (NW == 8 ? 4 : 0);
  const uint32_t soff = (uint32_t)(weight_row(tid < T_BN ? tid : 0) * groups);
  const uint8_t* const xsbase = MX ? p.xs + (gather ? 0 : first * groups) : nullptr;
  const i32x4 rxs = make_rsrc(xsbase, MX ? (gather ? p.src_rows : (rows < T_BM ? rows : T_BM)) * groups : 0);
  uint32_t xsoff = DM_OOB;
  if (MX && xt >= 0 && xt < T_BM && xt < rows)
    xsoff = (uint32_t)((gather ? mx_source_row(p, first + xt) : xt) * groups);

  // The words of 128 elements from group g0 on into scale buffer b.
  auto load_scales = [&](int g0, int b) {
    const uint32_t at = lds_addr_of(lds_s) + (uint32_t)(b * L::SB);
    if constexpr (KA) {
      if (wave < T_BN / 64) dma4(soff, advance_rsrc(rs, (uint32_t)g0), at + 256u * wave);
      if (MX && xw >= 0 && xw < T_BM / 64)
        dma4(xsoff, advance_rsrc(rxs, (uint32_t)g0), at + T_BN * 4 + 256u * xw);
    } else {
      uint32_t* const to = reinterpret_cast<uint32_t*>(lds_raw + L::STAGES * L::STAGE + b * L::SB);
      if (tid < T_BN) to[tid] = scale_word(sbase + soff + g0, groups - g0);
      if constexpr (MX)
        if (xt >= 0 && xt < T_BM) to[T_BN + xt] = xsoff == DM_OOB ? 0x7f7f7f7fu : scale_word(xsbase + xsoff + g0, groups - g0);
    }
  };
  auto issue = [&](int kt, int stage) {
    const uint32_t base = lds_addr_of(lds) + (uint32_t)(stage * L::STAGE);
    const i32x4 rxk = advance_rsrc(rx, (uint32_t)(kt * L::BK * ES));
    const i32x4 rwk = advance_rsrc(rw, (uint32_t)(kt * (L::BK / 2)));
#pragma unroll
    for (int q = 0; q < XQ; ++q)
      dma16(KA || kt * L::BK + xk[q] < (int)K ? xoff[q] : DM_OOB, rxk,
            base + (uint32_t)(XQ * wave + q) * 1024u);
#pragma unroll
    for (int q = 0; q < WQ; ++q)
      dma16(KA || kt * L::BK + wk[q] < (int)K ? woff[q] : DM_OOB, rwk,
            base + L::XB + (uint32_t)(WQ * wave + q) * 1024u);
    if (MX || (kt & 1) == 0)
      load_scales(kt * (L::BK / MX_GROUP), MX ? stage : (kt >> 1) & 1);
  };

  // A wave multiplies rows m0 + MS i .. + 31 by its half of the weight rows: the rows of a partial
  // tile spread over all waves, and blocks i past the last one are left out.
  constexpr int MS = 32 * L::MW;
  const int m0 = 32 * (wave >> 1), n0 = L::WN * (wave & 1);
  const int r32 = lane & 31, g = lane >> 5;
  f32x16 acc[MI][NJ] = {};
  auto multiply = [&](int kt, int stage, auto blocks) {
    constexpr int MN = decltype(blocks)::value;
    lds_char* const st = lds + stage * L::STAGE;
    const char* const sw = lds_raw + L::STAGES * L::STAGE + (MX ? stage : (kt >> 1) & 1) * L::SB;
    const int shift = MX ? 8 * g : 8 * (2 * (kt & 1) + g);
    uint32_t ws[NJ], xs[MN];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      ws[j] = *reinterpret_cast<const uint32_t*>(sw + 4 * (n0 + 32 * j + r32)) >> shift;
    if constexpr (MX) {
#pragma unroll
      for (int i = 0; i < MN; ++i)
        xs[i] = *reinterpret_cast<const uint32_t*>(sw + 4 * (T_BN + m0 + MS * i + r32)) >> shift;
      auto step = [&](auto sc) {
        constexpr int s = decltype(sc)::value;
        uint4 w[NJ], x[MN][2];
#pragma unroll
        for (int i = 0; i < MN; ++i) {
          const int r = m0 + MS * i + r32;
          const uint32_t at = (uint32_t)(r * 128), sz = (uint32_t)((r >> 1) & 7);
          x[i][0] = read_k(st, at + (((4 * s + g) ^ sz) << 4));
          x[i][1] = read_k(st, at + (((4 * s + 2 + g) ^ sz) << 4));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int r = n0 + 32 * j + r32;
          w[j] = read_k(st, L::XB + (uint32_t)(r * 64 + (((2 * s + g) ^ ((r >> 2) & 3)) << 4)));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < MN; ++i)
            acc[i][j] = mx_mma32<2 * s, 2 * s>(w[j], x[i][0], x[i][1], ws[j], xs[i], acc[i][j]);
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
    } else {
      uint4 w[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int r = n0 + 32 * j + r32;
        w[j] = read_k(st, L::XB + (uint32_t)(r * 32 + ((g ^ ((r >> 3) & 1)) << 4)));
        ws[j] &= 255u;
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint4 x[MN];
#pragma unroll
        for (int i = 0; i < MN; ++i) {
          const int r = m0 + MS * i + r32;
          x[i] = read_k(st, (uint32_t)(r * 128 + (((4 * g + s) ^ ((r >> 1) & 7)) << 4)));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint32_t q = s == 0 ? w[j].x : s == 1 ? w[j].y : s == 2 ? w[j].z : w[j].w;
          const uint4 a = mx_bf16x8(q, ws[j]);
#pragma unroll
          for (int i = 0; i < MN; ++i) acc[i][j] = Mma<TT_BF16>::run(a, x[i], acc[i][j]);
        }
      }
    }
  };

  // This block's k-tiles: from an even one where the words of scales span two.
  const int pairs = MX ? nkt : (nkt + 1) / 2;
  const int first_pair = (int)((int64_t)pairs * part / parts);
  const int last_pair = (int)((int64_t)pairs * (part + 1) / parts);
  const int mid = KS == 2 ? (first_pair + last_pair + 1) / 2 : last_pair;
  const int k0 = (MX ? 1 : 2) * (half ? mid : first_pair);
  const int k1r = (MX ? 1 : 2) * (half ? last_pair : mid);
  const int k1 = k1r < nkt ? k1r : nkt;
  const int steps = KS == 2 ? (MX ? 1 : 2) * (mid - first_pair) : k1 - k0;  // of both halves
#pragma unroll
  for (int s = 0; s < L::STAGES - 1; ++s)
    if (k0 + s < k1) issue(k0 + s, s);
  auto run = [&](auto blocks) {
    int stage = 0;
    for (int kt = k0; kt < k0 + steps; ++kt) {
      // k-tile kt has landed once at most the loads of later ones are outstanding, at least the x and
      // W pieces of each.
      const int later = KA ? k1 - 1 - kt : 0;
      if (L::STAGES >= 4 && later >= 2) TT_WAIT_VMCNT(2 * (XQ + WQ));
      else if (L::STAGES >= 3 && later >= 1) TT_WAIT_VMCNT(XQ + WQ);
      else TT_WAIT_VMCNT(0);
      TT_LDS_BARRIER();
      const int next = stage == 0 ? L::STAGES - 1 : stage - 1;  // the stage of kt - 1
      if (kt + L::STAGES - 1 < k1) issue(kt + L::STAGES - 1, next);
      if (KS == 1 || kt < k1) multiply(kt, stage, blocks);
      stage = stage == L::STAGES - 1 ? 0 : stage + 1;
    }
  };
  if (MI > 1 && rows <= MS) run(std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, MI>{});

  if (parts > 1) {
    // A part of the reduction: the sums as the registers hold them, for mx_join_kernel.
    float* const to = p.part + (((int64_t)tile * parts + part) * NW + wave) * (MI * NJ * 1024) + lane * 4;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(to + ((i * NJ + j) * 4 + q) * 256) =
              float4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                     acc[i][j][4 * q + 3]};
    return;
  }
  TT_LDS_BARRIER();  // every wave is past its fragment reads
  if constexpr (KS == 2) {
    // A half keeps block `half` of its rows and gives the other one away.
    lds_char* const all = (lds_char*)lds_block;
    constexpr uint32_t BLOCK = NJ * 4096;  // bytes of a wave's block of sums
    const uint32_t to = (4u * (1 - half) + wave) * BLOCK, from = (4u * half + wave) * BLOCK;
    static_assert(8 * BLOCK + 8 * NJ * 2048 <= 2 * L::LDS, "sums and outputs side by side");
    f32x16 sum[1][NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;
        f32x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = half ? acc[0][j][4 * q + e] : acc[1][j][4 * q + e];
          sum[0][j][4 * q + e] = half ? acc[1][j][4 * q + e] : acc[0][j][4 * q + e];
        }
        *reinterpret_cast<lds_f32x4*>(all + to + (4 * j + q) * 1024 + lane * 16) = v;
      }
    TT_LDS_BARRIER();
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t v = __builtin_bit_cast(f32x4_t, read_k(all, from + (4 * j + q) * 1024 + lane * 16));
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[0][j][4 * q + e] += v[e];
      }
    mx_tile_store<GATED, OUT8, 1, NJ, MS>(p, sum, all + 8 * BLOCK + (4 * half + wave) * (NJ * 2048),
                                          t.seg0 + i0, rows, m0 + MS * half,
                                          j0 + (GATED ? n0 / 2 : n0));
    return;
  }
  mx_tile_store<GATED, OUT8, MI, NJ, MS>(p, acc, lds + wave * (MI * NJ * 2048), t.seg0 + i0, rows, m0,
                                     j0 + (GATED ? n0 / 2 : n0));
}

// Sum of a dense product's parts, in order, and the epilogue: a wave per wave of a tile's four.
template <bool GATED, bool OUT8, int T_BM, int T_BN>
__global__ __launch_bounds__(64) void mx_join_kernel(MxArgs p, int tiles_i, int parts) {
  constexpr int MI = T_BM / 64, NJ = T_BN / 64;
  __shared__ __align__(16) char lds_raw[MI * NJ * 2048];
  const int tile = (int)(blockIdx.x >> 2), wave = (int)(blockIdx.x & 3), lane = lane_id();
  const int64_t i0 = (int64_t)(tile % tiles_i) * T_BM;
  const int64_t j0 = (int64_t)(tile / tiles_i) * (GATED ? T_BN / 2 : T_BN);
  f32x16 acc[MI][NJ] = {};
  for (int z = 0; z < parts; ++z) {
    const float* const from =
        p.part + (((int64_t)tile * parts + z) * 4 + wave) * (MI * NJ * 1024) + lane * 4;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 v = *reinterpret_cast<const float4*>(from + ((i * NJ + j) * 4 + q) * 256);
          acc[i][j][4 * q] += v.x;
          acc[i][j][4 * q + 1] += v.y;
          acc[i][j][4 * q + 2] += v.z;
          acc[i][j][4 * q + 3] += v.w;
        }
  }
  const int n0 = T_BN / 2 * (wave & 1);
  mx_tile_store<GATED, OUT8, MI, NJ, 64>(p, acc, (lds_char*)lds_raw, i0, p.M - i0, 32 * (wave >> 1),
                                     j0 + (GATED ? n0 / 2 : n0));
}

template <bool MX, bool GATED, bool OUT8, bool KA, int BM, int BN, int KS = 1>
int launch(const MxArgs& p, int parts, hipStream_t s) {
  constexpr int CB = GATED ? BN / 2 : BN, NT = 64 * Tile<MX, BM, BN>::NW * KS;
  const int64_t tiles_j = (p.N + CB - 1) / CB;
  int64_t tiles_i = (p.M + BM - 1) / BM;
  if (p.counts != nullptr) tiles_i = p.M / BM + (p.E < p.M ? p.E : p.M);
  const int64_t blocks = tiles_i * tiles_j * parts;
  TT_REQUIRE(blocks < (1ll << 31) && tt_grid_ok(blocks, NT), "mx product: grid too large");
  hipLaunchKernelGGL((mx_tile_kernel<MX, GATED, OUT8, KA, BM, BN, KS>), dim3((unsigned)blocks),
                     dim3(NT), 0, s, p, (int)tiles_j, parts);
  const int rc = tt_check_launch("mx_tile");
  if constexpr (BM == 64 && KA) {  // the only tile whose reductions are split
    if (rc != TT_OK || parts == 1) return rc;
    hipLaunchKernelGGL((mx_join_kernel<GATED, OUT8, BM, BN>), dim3((unsigned)(tiles_i * tiles_j * 4)),
                       dim3(64), 0, s, p, (int)tiles_i, parts);
    return tt_check_launch("mx_join");
  }
  return rc;
}

template <bool MX, bool GATED, bool OUT8>
int shaped(const MxArgs& p, MxPlan plan, hipStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.xs);
  if (p.K % 128 != 0 || (at & 3) != 0) return launch<MX, GATED, OUT8, false, 128, 128>(p, 1, s);
  if constexpr (MX)
    if (plan.bm == 256) return launch<MX, GATED, OUT8, true, 256, 256>(p, 1, s);
  if (plan.bm == 64) return launch<MX, GATED, OUT8, true, 64, 128>(p, plan.parts, s);
  if (plan.halves == 2) return launch<MX, GATED, OUT8, true, 128, 128, 2>(p, 1, s);
  if (plan.bn == 128) return launch<MX, GATED, OUT8, true, 128, 128>(p, 1, s);
  return launch<MX, GATED, OUT8, true, 128, 256>(p, 1, s);
}

template <bool MX, bool GATED>
int out(const MxArgs& p, MxPlan plan, hipStream_t s) {
  return p.ys != nullptr ? shaped<MX, GATED, true>(p, plan, s) : shaped<MX, GATED, false>(p, plan, s);
}

}  // namespace

bool tt_mx_tile_takes(const MxArgs& p, bool gated) {
  const int64_t es = p.xs != nullptr ? 1 : 2, width = gated ? 2 * p.N : p.N;
  // 32-bit offsets within an expert's weights, a tile's rows, and a gathered source.
  return p.K > 0 && width * (p.K / 2) < (1ll << 31) && 128 * p.K * es < (1ll << 31) &&
         (p.arow == nullptr || p.src_rows * p.K * es < (1ll << 31)) &&
         (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
}

int tt_mx_tile(const MxArgs& p, bool gated, MxPlan plan, hipStream_t s) {
  if (p.xs != nullptr) return gated ? out<true, true>(p, plan, s) : out<true, false>(p, plan, s);
  return gated ? out<false, true>(p, plan, s) : out<false, false>(p, plan, s);
}
