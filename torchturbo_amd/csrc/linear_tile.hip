// Dense product with an epilogue on the 16-bit matrix instructions (gfx950):
// C [I, J] = sum over r of A(i, r) B(r, j), then what linear.h makes of the fp32 sums.
// Rows of whole aligned 16-byte vectors take linear_big_kernel or linear_mid_kernel,
// all others linear_odd_kernel.
//
// A tile is computed by four waves, two by two, in blocks of v_mfma_f32_16x16x32 (256-row
// tiles) or v_mfma_f32_32x32x16 whose operands are swapped, so that a lane holds four
// consecutive columns of one row. 64-deep k-tiles go from memory straight into LDS.
// LDS layouts: K-major operands: 128 bytes per row, chunk c in slot
// c ^ ((row >> 1) & 7), read with ds_read_b128; the others: k-row by k-row as in
// memory, chunk c in slot c ^ (4 (k-row % 4)), read with the transposing
// ds_read_b64_tr_b16. Resources end with the operand, so rows past it read as
// zeros; a K-major tail (R % 64) is masked per chunk; columns past J are read
// from wherever they lead inside the resource and never stored.
#include "linear.h"

#include <type_traits>

namespace {

constexpr int T_NT = 256, T_BK = 64;

// A buffer resource that walks along an operand a k-tile at a time, in scalar
// registers. MN-major: it ends with the reduction's rows, so it is empty past them (the
// part of a reduction that a block walks is under 4 GiB). K-major: a row's end is
// masked by the loads, the resource keeps ending with the operand's last row.
struct Walk {
  i32x4 r;
  __device__ __forceinline__ void start(const void* base, int64_t left) { r = make_rsrc(base, left); }
  template <bool KM>
  __device__ __forceinline__ void advance(uint32_t by, bool more) {
    const uint32_t lo = (uint32_t)r.x + by;
    r.y += lo < by ? 1 : 0;  // a stride of 0 above the address
    r.x = (int)lo;
    if constexpr (KM) {
      r.z = more ? r.z : 0;
    } else {
      // max(records - by, 0) in scalar instructions (the compiler's is a vector one).
      uint32_t n;
      asm("s_sub_u32 %0, %1, %2\n\ts_cselect_b32 %0, 0, %0" : "=s"(n) : "s"(r.z), "s"(by) : "scc");
      r.z = (int)n;
    }
  }
};

// 16 bytes per lane into LDS at base + at + 16 lane (gemm.h's dma16 with the
// address formed in M0).
template <int AT>
__device__ __forceinline__ void dma16_at(uint32_t voff, const i32x4& rsrc, uint32_t base) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(base), "v"(voff), "s"(rsrc), "i"(AT)
               : "memory", "scc");
}

// Fragment offset of MN-major tiles with RB bytes per k-row: columns c0 .. c0 + 31;
// the second read is at + 4 RB and k-step s adds 16 RB.
template <int RB>
__device__ __forceinline__ uint32_t frag_mn(int c0, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int col = c0 + 16 * (g & 1) + 4 * (i & 3);
  const int kr = 8 * (g >> 1) + (i >> 2);
  return (uint32_t)(kr * RB + (((col >> 3) ^ (4 * (kr & 3) & (RB / 16 - 1))) << 4) + (col & 7) * 2);
}
// The same for 16 columns of a 32-deep k-step (which adds 32 RB): lane l gets column
// c0 + l % 16, k-rows 8 (l / 16) .. + 7.
template <int RB>
__device__ __forceinline__ uint32_t frag_mn16(int c0, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int col = c0 + 4 * (i & 3), kr = 8 * g + (i >> 2);
  return (uint32_t)(kr * RB + (((col >> 3) ^ (4 * (kr & 3) & (RB / 16 - 1))) << 4) + (col & 7) * 2);
}
template <int RB>
__device__ __forceinline__ uint4 read_mn(lds_char* tile, uint32_t off) {
  const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + off));
  const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + off + 4 * RB));
  const uint2 w0 = __builtin_bit_cast(uint2, v0), w1 = __builtin_bit_cast(uint2, v1);
  return uint4{w0.x, w0.y, w1.x, w1.y};
}

// One operand of a tile of BR rows (columns): its loads and its fragments.
// GATE (K-major only): the tile's rows are, per wave column, BR / 4 rows of the
// first half of the operand (from row 0 of the resource) and as many of the second.
// BS: rows of a fragment, 32 (16-deep k-steps) or 16 (32-deep ones).
template <bool KM, int BR, bool GATE, int BS>
struct Operand {
  static constexpr int BYTES = BR * T_BK * 2;
  static constexpr int LOADS = BR / 32;    // per wave and k-tile, 1 KiB each
  static constexpr int FR = BR / 64;       // 32-row blocks of a wave
  static constexpr int RB = BR * 2;        // bytes of a k-row (MN-major)
  static constexpr int KS = BS / 8;        // k-steps of a k-tile
  uint32_t off[LOADS];
  int kof[2];
  uint32_t frag[KM ? KS : FR];

  __device__ __forceinline__ void setup(int wave, int lane, int half, int64_t ld, int64_t rows2) {
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      if constexpr (KM) {
        const int r = (BR / 4) * wave + 8 * q + (lane >> 3);
        const int c = (lane & 7) ^ ((r >> 1) & 7);
        int64_t row = r;
        if constexpr (GATE) {
          const int w = r / (BR / 2), in = r % (BR / 2);
          row = (in / (BR / 4)) * rows2 + w * (BR / 4) + in % (BR / 4);
        }
        off[q] = (uint32_t)((row * ld + 8 * c) * 2);
        kof[q & 1] = 8 * c;
      } else {
        constexpr int LPR = RB / 16;  // lanes per k-row
        const int kr = 16 * wave + (64 / LPR) * q + lane / LPR;
        const int c = (lane % LPR) ^ (4 * (kr & 3) & (LPR - 1));
        off[q] = (uint32_t)((kr * ld + 8 * c) * 2);
      }
    }
    if constexpr (KM) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (BS == 32) {
          frag[s] = fragk64((BR / 2) * half, s, lane);
        } else {  // row lane % 16, chunk 4 s + lane / 16
          const int r = (BR / 2) * half + (lane & 15), c = 4 * s + (lane >> 4);
          frag[s] = (uint32_t)(r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < FR; ++m)
        frag[m] = BS == 32 ? frag_mn<RB>((BR / 2) * half + 32 * m, lane)
                           : frag_mn16<RB>((BR / 2) * half + 32 * m, lane);
    }
  }
  // Load Q of a k-tile of which `valid` reduction elements exist, into the operand's
  // stage; `lds` is the wave's first byte of it.
  template <bool KMASK, int Q>
  __device__ __forceinline__ void load(const i32x4& rs, uint32_t lds, int valid) const {
    uint32_t o = off[Q];
    if constexpr (KM && KMASK) o = kof[Q & 1] >= valid ? DM_OOB : o;
    dma16_at<Q * 1024>(o, rs, lds);
  }
  // Loads FROM .. TO - 1.
  template <bool KMASK, int FROM, int TO>
  __device__ __forceinline__ void loads(const i32x4& rs, uint32_t lds, int valid) const {
    if constexpr (FROM < TO) {
      load<KMASK, FROM>(rs, lds, valid);
      loads<KMASK, FROM + 1, TO>(rs, lds, valid);
    }
  }
  // Fragment m (BS rows) of k-step s.
  __device__ __forceinline__ uint4 read(lds_char* tile, int m, int s) const {
    if constexpr (KM) return read_k(tile, frag[s] + m * (BS * 128));
    else if constexpr (BS == 32) return read_mn<RB>(tile, frag[m] + s * 16 * RB);
    else return read_mn<RB>(tile, frag[m / 2] + (m & 1) * 32 + s * 32 * RB);
  }
};

template <int ET>
struct TypeOf;
template <>
struct TypeOf<TT_BF16> { typedef BF16T type; };
template <>
struct TypeOf<TT_F16> { typedef F16T type; };

typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;

// Eight 16-bit values of four dwords, and back (hardware round to nearest even).
template <int ET>
__device__ __forceinline__ void unpack8(const u32x4& w, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (ET == TT_BF16) {
      o[2 * e] = __uint_as_float(w[e] << 16);
      o[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    } else {
      o[2 * e] = f16_to_f32((uint16_t)(w[e] & 0xffffu));
      o[2 * e + 1] = f16_to_f32((uint16_t)(w[e] >> 16));
    }
  }
}
template <int ET>
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
  const uint2 lo = pack4<ET>(v[0], v[1], v[2], v[3]), hi = pack4<ET>(v[4], v[5], v[6], v[7]);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}

// The wave's rows [i0, I) of a matrix of `ld` elements of `size` bytes per row, from column
// j0 on: rows past I read as zeros, and stores to them are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* m, int64_t i0, int64_t I,
                                                            int64_t ld, int64_t j0, int size) {
  const int64_t at = (i0 * ld + j0) * size, left = m == nullptr ? 0 : I * ld * size - at;
  return __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(m)) + at, (short)0,
      (int)(left <= 0 ? 0u : left < (int64_t)DM_OOB ? (uint32_t)left : DM_OOB), 0x00020000);
}

// The sums of a wave's (32 FM) x (32 FN) part of the tile to what KIND makes of
// them (linear.h), 32 rows at a time through the wave's own LDS, so that a lane gets
// eight consecutive columns, with GATED their ups too. Rows of 128 FN bytes; chunk
// c of row r in slot ((c / 2) ^ r) + (c % 2) CH / 2, which neither the writes (four
// columns of 32 rows) nor the reads (a row's chunks) of eight lanes meet in a bank.
// One wave per SIMD has nothing to hide instructions behind, so memory is reached
// through resources with 32-bit offsets, conversions are the hardware's, and what a
// row needs is fetched 32 rows ahead: 4096 x 4096 x 512 with a residual 48 -> 31 us,
// the gradient with a row scale 73 -> 41.
// stage(mi, put): calls put(row, chunk, four sums) for the lane's part of the 32 rows mi.
template <int KIND, int ET, int FM, int FN, typename F>
__device__ __forceinline__ void tile_finish(const LinArgs& p, F stage, lds_char* region, int64_t i0,
                                            int64_t j0, int lane) {
  typedef typename TypeOf<ET>::type TT;
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int W = 32 * FN, CH = W / 4;       // columns and 16-byte chunks of a row
  constexpr int NG = (GATED ? W / 2 : W) / 8;  // groups of eight outputs of a row
  constexpr int RP = 64 / NG, NP = 32 / RP;    // rows per pass, passes per 32 rows
  constexpr bool SRC = KIND == LIN_RES || KIND == LIN_DROP || KIND == LIN_DGRAD;
  constexpr int BUF = KIND == LIN_DROP ? 1 : 2;  // random words take the registers of one
  const int gi = lane % NG, rr = lane / NG;
  const int64_t j = j0 + 8 * gi, width = GATED ? 2 * p.J : p.J;
  const bool col_ok = j < p.J;
  DropKey dk{};
  if constexpr (KIND == LIN_DROP) dk = load_key(p.key);
  const LinCols<KIND, 8> cols = lin_cols<KIND, 8>(p, j, col_ok ? 8 : 0);
  // Scale of rows lane and lane + 64 of the wave's.
  const bool scaled = SRC && p.scale != nullptr && p.part == nullptr;
  float sc[2] = {1.f, 1.f};
  if (scaled) {
#pragma unroll
    for (int q = 0; q < (FM + 1) / 2; ++q) {
      const int64_t i = i0 + 64 * q + lane;
      if (i < p.I) sc[q] = load_as_f32(p.scale, p.scale_dt, i);
    }
  }
  // Byte offsets of the lane's group in 16-bit rows and in fp32 ones (columns that
  // do not exist get one past any resource).
  const uint32_t off16 = (uint32_t)((rr * p.J + 8 * gi) * 2);
  const uint32_t off32 = (uint32_t)((rr * width + 8 * gi) * 4);
  const uint32_t row16 = (uint32_t)(p.J * 2), row32 = (uint32_t)(width * 4);
  const __amdgpu_buffer_rsrc_t out = rows_rsrc(p.out, i0, p.I, p.J, j0, 2);
  const void* src = KIND == LIN_DGRAD ? (scaled ? p.x : nullptr) : SRC ? p.res : nullptr;
  const __amdgpu_buffer_rsrc_t in = rows_rsrc(src, i0, p.I, p.J, j0, 2);
  const __amdgpu_buffer_rsrc_t xs = rows_rsrc(KIND == LIN_DGRAD ? p.xs : nullptr, i0, p.I, p.J, j0, 2);
  float* const wide = p.part != nullptr ? p.part + (int64_t)blockIdx.y * p.I * width : p.pre;
  const __amdgpu_buffer_rsrc_t w0 = rows_rsrc(wide, i0, p.I, width, j0, 4);
  const __amdgpu_buffer_rsrc_t w1 = rows_rsrc(GATED ? wide : nullptr, i0, p.I, width, p.J + j0, 4);
  const bool keep_sums = wide != nullptr, whole = p.part == nullptr;
  const int nd = (int)((p.J + LIN_DOT - 1) / LIN_DOT);

  auto put32 = [&](const __amdgpu_buffer_rsrc_t& rs, const float (&v)[8], uint32_t off) {
    const f32x4_t lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, lo), rs,
                                           (int)(col_ok ? off : DM_OOB), 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, hi), rs,
                                           (int)(col_ok ? off + 16 : DM_OOB), 0, 0);
  };
  u32x4 rows[BUF][SRC ? NP : 1] = {};
  const bool fetched = SRC && src != nullptr && whole;
  auto fetch = [&](int mi) {
#pragma unroll
    for (int ps = 0; ps < NP; ++ps)
      rows[mi % BUF][ps] = __builtin_amdgcn_raw_buffer_load_b128(
          in, (int)(col_ok ? off16 + (uint32_t)(32 * mi + ps * RP) * row16 : DM_OOB), 0, 0);
  };
  auto pass = [&](int mi, int ps, const u32x4& row) {
    const int r = ps * RP + rr;
    auto chunk = [&](int c) {
      return *reinterpret_cast<const lds_f32x4*>(
          region + r * (W * 4) + ((((c >> 1) ^ (r & (CH / 2 - 1))) + (c & 1) * (CH / 2)) << 4));
    };
    float v[8], u[8];
    const f32x4_t a = chunk(2 * gi), b = chunk(2 * gi + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
    if constexpr (GATED) {
      const f32x4_t c = chunk(CH / 2 + 2 * gi), d = chunk(CH / 2 + 2 * gi + 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[e] = c[e];
        u[4 + e] = d[e];
      }
    }
    const int q = 32 * mi + ps * RP;  // the pass's first row in the wave's
    const uint32_t at16 = off16 + (uint32_t)q * row16, at32 = off32 + (uint32_t)q * row32;
    if (!whole) {  // a split's sums
      put32(w0, v, at32);
      if constexpr (GATED) put32(w1, u, at32);
      return;
    }
    float s = 1.f;
    if (scaled) s = __shfl(sc[FM > 2 ? mi / 2 : 0], 32 * (mi & 1) + ps * RP + rr, 64);
    if constexpr (KIND == LIN_ACT || KIND == LIN_GATED) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] += cols.b[e];
        if constexpr (GATED) u[e] += cols.bu[e];
      }
      if (keep_sums) {
        put32(w0, v, at32);
        if constexpr (GATED) put32(w1, u, at32);
      }
      auto activate = [&](int act) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lin_act<TT>(act, v[e]);
      };
      if (p.act == ACT_SILU) activate(ACT_SILU);
      else if (p.act == ACT_GELU) activate(ACT_GELU);
      if constexpr (GATED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= u[e];
      }
    } else if constexpr (KIND == LIN_RES || KIND == LIN_DROP) {
      uint32_t w[4] = {};
      if constexpr (KIND == LIN_DROP)
        philox(dk, (uint32_t)(j >> 3), (uint32_t)(i0 + q + rr), w);
      float x[8];
      unpack8<ET>(row, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float t = v[e] + cols.b[e];
        if constexpr (KIND == LIN_DROP) t = keeps(w, e, p.threshold) ? t * p.alpha : 0.f;
        v[e] = x[e] + s * t;  // x is zero where there is no residual
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= p.alpha;
      if (KIND == LIN_DGRAD && scaled) {
        float x[8], dot = 0.f;
        unpack8<ET>(row, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dot += x[e] * v[e];
          v[e] *= s;
          x[e] *= s;
        }
        __builtin_amdgcn_raw_buffer_store_b128(pack8<ET>(x), xs, (int)(col_ok ? at16 : DM_OOB), 0, 0);
        if (p.dots != nullptr) {
          static_assert(LIN_DOT == 32, "four lanes of eight columns");
          // Sums past column J are of other rows of B: 0 times an infinite one is no number.
          dot = sum4(col_ok ? dot : 0.f);
          const int64_t i = i0 + q + rr;
          if ((lane & 3) == 0 && i < p.I && col_ok) p.dots[i * nd + j / LIN_DOT] = dot;
        }
      }
    }
    __builtin_amdgcn_raw_buffer_store_b128(pack8<ET>(v), out, (int)(col_ok ? at16 : DM_OOB), 0, 0);
  };
  if (fetched && BUF == 2) fetch(0);
#pragma unroll
  for (int mi = 0; mi < FM; ++mi) {
    if (fetched && mi + BUF - 1 < FM) fetch(mi + BUF - 1);
    stage(mi, [&](int r, int c, const f32x4_t& v) {
      *reinterpret_cast<lds_f32x4*>(
          region + r * (W * 4) + ((((c >> 1) ^ (r & (CH / 2 - 1))) + (c & 1) * (CH / 2)) << 4)) = v;
    });
    if constexpr (SRC) {
#pragma unroll
      for (int ps = 0; ps < NP; ++ps) pass(mi, ps, rows[mi % BUF][ps]);
    } else {
#pragma unroll 2
      for (int ps = 0; ps < NP; ++ps) pass(mi, ps, rows[0][0]);
    }
  }
}

// Tile (row, column) of a block. Consecutive tiles run on one XCD, in groups of
// eight tile rows walked column by column, so that the 32 CUs of an XCD work on an
// 8 x 4 rectangle and share its operand panels in their L2.
__device__ __forceinline__ void tile_of(int ti, int tj, int& i, int& j) {
  const int L = xcd_remap(blockIdx.x, ti * tj);
  const int per = 8 * tj, group = L / per, first = 8 * group;
  const int rows = ti - first < 8 ? ti - first : 8, in = L % per;
  i = first + in % rows;
  j = in / rows;
}

template <int LAYOUT, int KIND, int BM, int BN, int BS>
struct Tile {
  static constexpr bool A_K = LAYOUT != LAY_TN, B_K = LAYOUT == LAY_NT, GATED = KIND == LIN_GATED;
  typedef Operand<A_K, BM, false, BS> OpA;
  typedef Operand<B_K, BN, GATED, BS> OpB;
  static constexpr int STAGE = OpA::BYTES + OpB::BYTES;
  static constexpr int BO = GATED ? BN / 2 : BN;  // output columns
  OpA a;
  OpB b;
  Walk wa, wb;
  uint32_t sa, sb;  // bytes of a k-tile step
  int64_t i0, j0;
  int nkt, kn;  // k-tiles and reduction elements of this block

  __device__ __forceinline__ void setup(const LinArgs& p, int ti, int tj, int wave, int lane) {
    int i, j;
    tile_of(ti, tj, i, j);
    i0 = (int64_t)i * BM;
    j0 = (int64_t)j * BO;
    const int64_t r0 = (int64_t)blockIdx.y * p.rsplit;
    const int64_t n = p.R - r0 < p.rsplit ? p.R - r0 : p.rsplit;
    kn = (int)n;
    nkt = (int)((n + T_BK - 1) / T_BK);
    const char* pa = static_cast<const char*>(p.a);
    const char* pb = static_cast<const char*>(p.b);
    // First byte of the tile's part of the operand, and the bytes from there to
    // the operand's end (of this split's reduction rows where they are MN-major).
    const int64_t oa = A_K ? (i0 * p.lda + r0) * 2 : (r0 * p.lda + i0) * 2;
    wa.start(pa + oa, (A_K ? p.I * p.lda * 2 : (r0 + n) * p.lda * 2) - oa);
    sa = A_K ? T_BK * 2 : (uint32_t)(T_BK * p.lda * 2);
    const int64_t ob = B_K ? (j0 * p.ldb + r0) * 2 : (r0 * p.ldb + j0) * 2;
    wb.start(pb + ob, (B_K ? (GATED ? 2 : 1) * p.J * p.ldb * 2 : (r0 + n) * p.ldb * 2) - ob);
    sb = B_K ? T_BK * 2 : (uint32_t)(T_BK * p.ldb * 2);
    if (nkt == 0) wa.r.z = wb.r.z = 0;
    a.setup(wave, lane, wave >> 1, p.lda, 0);
    b.setup(wave, lane, wave & 1, p.ldb, p.J);
  }
  // The resources of the k-tile after the one they stand at, kt.
  __device__ __forceinline__ void next_a(int kt) { wa.template advance<A_K>(sa, kt + 1 < nkt); }
  __device__ __forceinline__ void next_b(int kt) { wb.template advance<B_K>(sb, kt + 1 < nkt); }
};

// c += a b in the accumulation registers, in its place among the other volatile
// assembly: as a builtin a product has no side effects, and the compiler moved half of
// a k-tile's products behind its barriers, and copied accumulators that it held fixed to
// places (160 moves per k-tile). Nothing but these products touches c before mma_done.
template <int ET>
__device__ __forceinline__ void mma16(f32x4_t& c, const uint4& a, const uint4& b) {
  const u32x4 va = __builtin_bit_cast(u32x4, a), vb = __builtin_bit_cast(u32x4, b);
  if constexpr (ET == TT_BF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(va), "v"(vb));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(va), "v"(vb));
}
// The last product's results may be read: the compiler's padding between a product
// and the use of its result does not see assembly.
__device__ __forceinline__ void mma_done() { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory"); }

// 256 x BN tiles, BN 256 or 128, 128 x BN / 2 per wave (one wave per SIMD), in
// 16x16x32 products. LDS holds SA k-tiles of A and three of B; the k-tile after next is
// loaded while one is multiplied. k-step 0 multiplies and reads the fragments of
// k-step 1. With SA = 2 a barrier then frees A's stage for the loads of k-step 1 (with
// three, the stage of the k-tile before is loaded). Half way through k-step 1 a
// barrier publishes the next k-tile, whose first fragments the other half reads.
// Large products run at the part's power limit, where the 16x16x32 instructions draw less
// than the 32x32x16 ones (2.0 GHz in place of 1.78), and the sums stay in the accumulation
// registers. 4096 x 7168 -> 4096 in bf16, tiles of 256 x 256: NT 159 us (1.51 PFLOP/s),
// NN 163, TN 161; a plain product of torch 151, 177 and 211.
template <int LAYOUT, int KIND, int ET, bool KMASK, int BN>
__global__ __launch_bounds__(T_NT) void linear_big_kernel(LinArgs p, int ti, int tj) {
  typedef Tile<LAYOUT, KIND, 256, BN, 16> TL;
  constexpr int FM = 8, FN = BN / 32, SA = BN == 256 ? 2 : 3;
  constexpr int LA = TL::OpA::LOADS, LB = TL::OpB::LOADS;
  static_assert(LA == 8 && LB == FN, "loads per row of products");
  constexpr uint32_t BA = TL::OpA::BYTES, BB = TL::OpB::BYTES;
  __shared__ __align__(16) char lds_raw[SA * BA + 3 * BB];  // the k-tiles of A, then of B
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TL t;
  t.setup(p, ti, tj, wave, lane);
  lds_char* const lds = (lds_char*)lds_raw;
  const uint32_t lds0 = lds_addr_of(lds);
  const uint32_t wa0 = lds0 + (uint32_t)(LA * wave) * 1024u;            // the wave's part of A's stages
  const uint32_t wb0 = lds0 + SA * BA + (uint32_t)(LB * wave) * 1024u;  // and of B's
  uint4 fa[2][FM], fb[2][FN];
  f32x4_t acc[FM][FN] = {};
  t.a.template loads<KMASK, 0, LA>(t.wa.r, wa0, t.kn);
  t.b.template loads<KMASK, 0, LB>(t.wb.r, wb0, t.kn);
  t.next_a(0);
  t.next_b(0);
  t.b.template loads<KMASK, 0, LB>(t.wb.r, wb0 + BB, t.kn - T_BK);
  t.a.template loads<KMASK, 0, LA>(t.wa.r, wa0 + BA, t.kn - T_BK);
  t.next_a(1);
  t.next_b(1);
  TT_WAIT_VMCNT(LA + LB);
  TT_LDS_BARRIER();
#pragma unroll
  for (int i = 0; i < FM; ++i) fa[0][i] = t.a.read(lds, i, 0);
#pragma unroll
  for (int i = 0; i < FN; ++i) fb[0][i] = t.b.read(lds + SA * BA, i, 0);
  int slot = 0;  // of k-tile kt in a ring of three
  for (int kt = 0; kt < t.nkt; ++kt) {
    const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot == 0 ? 2 : slot - 1;
    const int a0 = SA == 3 ? slot : kt & 1, a1 = SA == 3 ? slot1 : (kt + 1) & 1;
    lds_char* const ca = lds + (uint32_t)a0 * BA;
    lds_char* const na = lds + (uint32_t)a1 * BA;
    lds_char* const cb = lds + SA * BA + (uint32_t)slot * BB;
    lds_char* const nb = lds + SA * BA + (uint32_t)slot1 * BB;
    const uint32_t to_a = wa0 + (uint32_t)(SA == 3 ? slot2 : a0) * BA;
    const uint32_t to_b = wb0 + (uint32_t)slot2 * BB;
    const int valid = t.kn - (kt + 2) * T_BK;
    // Products of row m and columns n, n + 1 of k-step s.
    auto mul = [&](int s, int m, int n) {
      mma16<ET>(acc[m][n], fb[s][n], fa[s][m]);
      mma16<ET>(acc[m][n + 1], fb[s][n + 1], fa[s][m]);
    };
    // k-step 0: row m of the products.
    auto first = [&](auto m_c) {
      constexpr int m = decltype(m_c)::value;
#pragma unroll
      for (int n = 0; n < FN; n += 2) {
        mul(0, m, n);
        if (n == 0 && m < FN) fb[1][m] = t.b.read(cb, m, 1);
        if (n == (FN == 8 ? 4 : m < FN ? 2 : 0)) fa[1][m] = t.a.read(ca, m, 1);
        if (n == FN - 2) {
          if constexpr (m < LB) t.b.template load<KMASK, (m < LB ? m : 0)>(t.wb.r, to_b, valid);
          else t.a.template load<KMASK, m - LB>(t.wa.r, to_a, valid);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // k-step 1, rows 0-3: with the rest of A's loads.
    auto second = [&](auto m_c) {
      constexpr int m = decltype(m_c)::value;
#pragma unroll
      for (int n = 0; n < FN; n += 2) {
        mul(1, m, n);
        if constexpr (FN == 8) {
          if (n == 2) t.a.template load<KMASK, 2 * m>(t.wa.r, to_a, valid);
          if (n == 6) t.a.template load<KMASK, 2 * m + 1>(t.wa.r, to_a, valid);
        } else {
          if (n == 0) t.a.template load<KMASK, 4 + m>(t.wa.r, to_a, valid);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    first(std::integral_constant<int, 0>{});
    first(std::integral_constant<int, 1>{});
    first(std::integral_constant<int, 2>{});
    first(std::integral_constant<int, 3>{});
    first(std::integral_constant<int, 4>{});
    first(std::integral_constant<int, 5>{});
    first(std::integral_constant<int, 6>{});
    first(std::integral_constant<int, 7>{});
    t.next_b(kt + 2);
    if constexpr (SA == 2) TT_LDS_BARRIER();  // every wave has read k-tile kt
    second(std::integral_constant<int, 0>{});
    second(std::integral_constant<int, 1>{});
    second(std::integral_constant<int, 2>{});
    second(std::integral_constant<int, 3>{});
    t.next_a(kt + 2);
    TT_WAIT_VMCNT(LA + LB);  // k-tile kt + 1 has landed
    TT_LDS_BARRIER();
#pragma unroll
    for (int m = 4; m < 8; ++m)
#pragma unroll
      for (int n = 0; n < FN; n += 2) {
        mul(1, m, n);
        constexpr int PS = FN == 8 ? 2 : 3;  // reads per two slots
        const int at = (m - 4) * (FN / 2) + n / 2;
#pragma unroll
        for (int i = at * PS / 2; i < (at + 1) * PS / 2; ++i) {
          if (i < FN) fb[0][i] = t.b.read(nb, i, 0);
          else fa[0][i - FN] = t.a.read(na, i - FN, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    slot = slot1;
  }
  mma_done();
  TT_WAIT_VMCNT(0);
  __syncthreads();  // every wave is past its fragment reads, and every load has landed
  // Lane l holds row 16 m + l % 16, columns 16 n + 4 (l / 16) + 0..3.
  auto stage = [&](auto mi, auto put) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n)
        put(16 * m + (lane & 15), 4 * n + (lane >> 4), acc[2 * mi + m][n]);
  };
  tile_finish<KIND, ET, FM / 2, FN / 2>(p, stage, lds + wave * (32 * (BN / 2) * 4),
                                        t.i0 + (wave >> 1) * 128,
                                        t.j0 + (wave & 1) * (TL::BO / 2), lane);
}

// BT x BT tiles (64 or 128), a quarter per wave, a ring of S stages (16 or 32 KiB) with
// one barrier per k-tile, which publishes k-tile kt and frees the stage of kt - 1. Several
// blocks share a CU and hide one another's waits and epilogues: 512 x 2048 -> 7168 26.1 us
// (0.58 PFLOP/s), 1000 x 704 -> 1024 7.4 us.
template <int LAYOUT, int KIND, int ET, bool KMASK, int BT, int S>
__global__ __launch_bounds__(T_NT) void linear_mid_kernel(LinArgs p, int ti, int tj) {
  typedef Tile<LAYOUT, KIND, BT, BT, 32> TL;
  constexpr int FM = BT / 64, FN = BT / 64;
  constexpr int LA = TL::OpA::LOADS, LB = TL::OpB::LOADS, LD = LA + LB;
  __shared__ __align__(16) char lds_raw[S * TL::STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TL t;
  t.setup(p, ti, tj, wave, lane);
  lds_char* const lds = (lds_char*)lds_raw;
  const uint32_t lds0 = lds_addr_of(lds);
  auto issue = [&](int kt, int slot) {
    const uint32_t at = lds0 + (uint32_t)slot * TL::STAGE;
    const int valid = t.kn - kt * T_BK;
    t.a.template loads<KMASK, 0, LA>(t.wa.r, at + (uint32_t)(LA * wave) * 1024u, valid);
    t.b.template loads<KMASK, 0, LB>(t.wb.r, at + TL::OpA::BYTES + (uint32_t)(LB * wave) * 1024u,
                                     valid);
    t.next_a(kt);
    t.next_b(kt);
  };
  f32x16 acc[FM][FN] = {};
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < t.nkt) issue(i, i);
  int slot = 0;
  for (int kt = 0; kt < t.nkt; ++kt) {
    const int later = t.nkt - 1 - kt;
    if (S >= 4 && later >= 2) TT_WAIT_VMCNT(2 * LD);
    else if (S >= 3 && later >= 1) TT_WAIT_VMCNT(LD);
    else TT_WAIT_VMCNT(0);
    TT_LDS_BARRIER();
    if (kt + S - 1 < t.nkt) issue(kt + S - 1, slot == 0 ? S - 1 : slot - 1);
    lds_char* const stg = lds + slot * TL::STAGE;
    uint4 fa[2][FM], fb[2][FN];
    auto frags = [&](int s) {
#pragma unroll
      for (int m = 0; m < FM; ++m) fa[s & 1][m] = t.a.read(stg, m, s);
#pragma unroll
      for (int n = 0; n < FN; ++n) fb[s & 1][n] = t.b.read(stg + TL::OpA::BYTES, n, s);
    };
    frags(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s < 3) frags(s + 1);
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n)
          acc[m][n] = Mma<ET>::run(fb[s & 1][n], fa[s & 1][m], acc[m][n]);
    }
    slot = slot == S - 1 ? 0 : slot + 1;
  }
  TT_WAIT_VMCNT(0);
  __syncthreads();
  // Lane l holds row 32 mi + l % 32, columns 32 ni + 8 g + 4 (l / 32) + 0..3.
  auto stage = [&](auto mi, auto put) {
#pragma unroll
    for (int ni = 0; ni < FN; ++ni)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        put(lane & 31, 8 * ni + 2 * g + (lane >> 5),
            f32x4_t{acc[mi][ni][4 * g], acc[mi][ni][4 * g + 1], acc[mi][ni][4 * g + 2],
                    acc[mi][ni][4 * g + 3]});
  };
  tile_finish<KIND, ET, FM, FN>(p, stage, lds + wave * (32 * (BT / 2) * 4), t.i0 + (wave >> 1) * (BT / 2),
                                t.j0 + (wave & 1) * (TL::BO / 2), lane);
}

// An operand of linear_odd_kernel, chunks laid out as Operand::setup does. A load is
// always of 16 bytes, at an address moved back where they would pass the operand's
// end, so that it never waits for another; the elements are put in place, and those past
// a row's end cleared, when it has arrived.
// TINY: an operand may have fewer than eight elements in all.
template <bool KM, int BR, bool GATE, bool TINY>
struct OddOperand {
  static constexpr int LOADS = BR / 32;
  const uint16_t* base;
  int64_t last;        // the last element that 16 bytes can start at
  int64_t off[LOADS];  // of the chunk in k-tile 0
  int64_t step;        // elements of a k-tile
  int at[LOADS];       // the chunk's place in the reduction
  int most[LOADS];     // its elements that exist, by the other dimension
  bool inside;         // every row of the tile exists

  // rows x R elements (GATE: 2 x rows), from row `first` and reduction element r0 on.
  __device__ __forceinline__ void setup(const uint16_t* p, int64_t ld, int64_t rows, int64_t R,
                                        int64_t first, int64_t r0, int64_t half, int wave, int lane) {
    base = p;
    last = rows * R * (GATE ? 2 : 1) - 8;
    step = KM ? T_BK : T_BK * ld;
    inside = first + (GATE ? BR / 2 : BR) <= rows;
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      if constexpr (KM) {
        const int r = (BR / 4) * wave + 8 * q + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        int64_t row = r, in = r;
        if constexpr (GATE) {
          in = r / (BR / 2) * (BR / 4) + r % (BR / 2) % (BR / 4);
          row = (r % (BR / 2) / (BR / 4)) * half + in;
        }
        off[q] = (first + row) * ld + r0 + 8 * c;
        at[q] = 8 * c;
        most[q] = first + in < rows ? 8 : 0;
      } else {
        constexpr int LPR = BR / 8;
        const int kr = 16 * wave + (64 / LPR) * q + lane / LPR;
        const int c = (lane % LPR) ^ (4 * (kr & 3) & (LPR - 1));
        const int64_t left = rows - first - 8 * c;
        off[q] = (r0 + kr) * ld + first + 8 * c;
        at[q] = kr;
        most[q] = left <= 0 ? 0 : left < 8 ? (int)left : 8;
      }
    }
  }
  __device__ __forceinline__ int64_t start(int q, int kt) const { return off[q] + kt * step; }
  // Whether all of k-tile kt of kn elements exists.
  __device__ __forceinline__ bool whole(int kt, int kn) const {
    return inside && (kt + 1) * T_BK <= kn;
  }
  __device__ __forceinline__ uint4 load(int q, int kt) const {
    const int64_t o = start(q, kt);
    uint4 v;
    if constexpr (!TINY) {
      __builtin_memcpy(&v, base + (o < last ? o : last), 16);
    } else {
      uint32_t w[4] = {};
      for (int e = 0; e < 8; ++e)
        if (o + e < last + 8) w[e >> 1] |= (uint32_t)base[o + e] << (16 * (e & 1));
      v = uint4{w[0], w[1], w[2], w[3]};
    }
    return v;
  }
  // What `load` brought for k-tile kt, of which kn reduction elements exist from k-tile 0 on.
  __device__ __forceinline__ u32x4 trim(const uint4& v, int q, int kt, int kn) const {
    const int left = kn - kt * T_BK - at[q];
    int n = KM ? (left < most[q] ? left : most[q]) : (left > 0 ? most[q] : 0);
    n = n > 0 ? n : 0;
    const int64_t o = start(q, kt);
    const int moved = !TINY && o > last ? (int)(o - last < 8 ? o - last : 8) : 0;
    uint64_t lo = ((uint64_t)v.y << 32) | v.x, hi = ((uint64_t)v.w << 32) | v.z;
    if (moved != 0) {  // down by `moved` elements
      const int s = 16 * moved;
      lo = s >= 64 ? (s >= 128 ? 0 : hi >> (s - 64)) : (lo >> s) | (hi << (64 - s));
      hi = s >= 64 ? 0 : hi >> s;
    }
    lo = n >= 4 ? lo : lo & ((1ull << (16 * n)) - 1);
    hi = n >= 8 ? hi : n <= 4 ? 0 : hi & ((1ull << (16 * (n - 4))) - 1);
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
};

// Tiles of operands whose rows do not start at multiples of 16 bytes, or end inside a
// vector: BT x BT as in linear_mid_kernel, but a k-tile goes through registers
// (OddOperand) into the same LDS layouts, two stages; and results are stored at any
// address, single elements at a row's end. It is bound by the instructions that move
// k-tiles, not by products: 4001 x 1201 -> 1703 in bf16 62 us NT, 71 NN, 71 TN (0.26
// PFLOP/s; 228, 340 and 366 us on the fp32 matrix instructions).
template <int LAYOUT, int KIND, int ET, int BT, bool TINY>
__global__ __launch_bounds__(T_NT) void linear_odd_kernel(LinArgs p, int ti, int tj) {
  typedef Tile<LAYOUT, KIND, BT, BT, 32> TL;
  typedef typename TypeOf<ET>::type TT;
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int FM = BT / 64, FN = BT / 64;
  constexpr int LA = TL::OpA::LOADS, LB = TL::OpB::LOADS;
  __shared__ __align__(16) char lds_raw[2 * TL::STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TL t;
  t.setup(p, ti, tj, wave, lane);
  lds_char* const lds = (lds_char*)lds_raw;
  const int64_t r0 = (int64_t)blockIdx.y * p.rsplit;
  OddOperand<TL::A_K, BT, false, TINY> oa;
  OddOperand<TL::B_K, BT, GATED, TINY> ob;
  oa.setup(static_cast<const uint16_t*>(p.a), p.lda, p.I, p.R, t.i0, r0, 0, wave, lane);
  ob.setup(static_cast<const uint16_t*>(p.b), p.ldb, p.J, p.R, t.j0, r0, p.J, wave, lane);
  // k-tiles kt + 1 and kt + 2 are on their way while kt is multiplied. Loads past the last
  // one are made all the same (and trimmed to nothing), in whole pairs of k-tiles: where
  // some are skipped, the compiler waits for all of them.
  uint4 va[2][LA], vb[2][LB];
  auto fetch = [&](int kt, int buf) {
#pragma unroll
    for (int q = 0; q < LA; ++q) va[buf][q] = oa.load(q, kt);
#pragma unroll
    for (int q = 0; q < LB; ++q) vb[buf][q] = ob.load(q, kt);
  };
  f32x16 acc[FM][FN] = {};
  auto step = [&](int kt, int buf) {
    // This stage is free: every wave passed the barrier of k-tile kt - 1 after kt - 2.
    lds_char* const stg = lds + buf * TL::STAGE;
    lds_char* const at = stg + lane * 16;
    auto put = [&](auto& op, uint4* v, int first, int loads) {
      const bool all = op.whole(kt, t.kn);
#pragma unroll
      for (int q = 0; q < loads; ++q) {
        u32x4 w = __builtin_bit_cast(u32x4, v[q]);
        if (!all) w = op.trim(v[q], q, kt, t.kn);
        *reinterpret_cast<lds_u32x4*>(at + first + (loads * wave + q) * 1024) = w;
      }
    };
    put(oa, va[buf], 0, LA);
    put(ob, vb[buf], TL::OpA::BYTES, LB);
    fetch(kt + 2, buf);
    TT_LDS_BARRIER();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint4 fa[FM], fb[FN];
#pragma unroll
      for (int m = 0; m < FM; ++m) fa[m] = t.a.read(stg, m, s);
#pragma unroll
      for (int n = 0; n < FN; ++n) fb[n] = t.b.read(stg + TL::OpA::BYTES, n, s);
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = Mma<ET>::run(fb[n], fa[m], acc[m][n]);
    }
  };
  fetch(0, 0);
  fetch(1, 1);
  for (int kt = 0; kt < t.nkt; kt += 2) {
    step(kt, 0);
    step(kt + 1, 1);
  }
  __syncthreads();
  static_assert(LIN_WAVE_FLOATS<FN> * 4 * 4 <= 2 * TL::STAGE, "the waves' rows");
  // Lane l holds row 32 mi + l % 32, columns 32 ni + 8 g + 4 (l / 32) + 0..3.
  auto stage = [&](int mi, auto put) {
#pragma unroll
    for (int ni = 0; ni < FN; ++ni)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        put(lane & 31, 32 * ni + 8 * g + 4 * (lane >> 5),
            f32x4_t{acc[mi][ni][4 * g], acc[mi][ni][4 * g + 1], acc[mi][ni][4 * g + 2],
                    acc[mi][ni][4 * g + 3]});
  };
  lin_finish_wave<KIND, TT, FM, FN>(p, stage, reinterpret_cast<float*>(lds_raw) + wave * LIN_WAVE_FLOATS<FN>,
                                    t.i0 + (wave >> 1) * (BT / 2),
                                    t.j0 + (wave & 1) * (GATED ? BT / 4 : BT / 2), lane);
}

template <int LAYOUT, int KIND, int ET, bool KMASK>
int launch(int tile, const LinArgs& p, hipStream_t s) {
  const int bm = tile == LIN_T64 ? 64 : tile == LIN_T128 ? 128 : 256;
  const int bn = tile == LIN_T64 ? 64 : tile == LIN_T256 ? 256 : 128;
  const int bo = KIND == LIN_GATED ? bn / 2 : bn;
  const int64_t ti = (p.I + bm - 1) / bm, tj = (p.J + bo - 1) / bo;
  TT_REQUIRE(tt_grid_ok(ti * tj, T_NT), "linear: grid too large");
  const dim3 grid((unsigned)(ti * tj), (unsigned)p.splits);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(T_NT), 0, s, p, (int)ti, (int)tj);
    return tt_check_launch("linear");
  };
  if (tile == LIN_T256) return go(&linear_big_kernel<LAYOUT, KIND, ET, KMASK, 256>);
  if (tile == LIN_T256x128) return go(&linear_big_kernel<LAYOUT, KIND, ET, KMASK, 128>);
  if (tile == LIN_T64) return go(&linear_mid_kernel<LAYOUT, KIND, ET, KMASK, 64, 4>);
  // A block has a CU to itself, and all of its memory, in a launch of at most one per CU
  // (four stages / two: 512 x 2048 -> 7168 24.0 / 25.0 us, 2048 cubed 24.8 / 25.6).
  if (ti * tj * p.splits <= 256) return go(&linear_mid_kernel<LAYOUT, KIND, ET, KMASK, 128, 4>);
  return go(&linear_mid_kernel<LAYOUT, KIND, ET, KMASK, 128, 2>);
}

template <int LAYOUT, int KIND, int ET, int BT>
int launch_odd(const LinArgs& p, hipStream_t s) {
  constexpr int BO = KIND == LIN_GATED ? BT / 2 : BT;
  const int64_t ti = (p.I + BT - 1) / BT, tj = (p.J + BO - 1) / BO;
  TT_REQUIRE(tt_grid_ok(ti * tj, T_NT), "linear: grid too large");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(ti * tj), (unsigned)p.splits), dim3(T_NT), 0, s, p,
                       (int)ti, (int)tj);
    return tt_check_launch("linear_odd");
  };
  if constexpr (BT == 64)
    if (p.I * p.R < 8 || p.J * p.R < 8) return go(&linear_odd_kernel<LAYOUT, KIND, ET, BT, true>);
  return go(&linear_odd_kernel<LAYOUT, KIND, ET, BT, false>);
}

template <int LAYOUT, int KIND>
int typed(int tile, int dtype, const LinArgs& p, hipStream_t s) {
  if (tile == LIN_ODD64)
    return dtype == TT_BF16 ? launch_odd<LAYOUT, KIND, TT_BF16, 64>(p, s)
                            : launch_odd<LAYOUT, KIND, TT_F16, 64>(p, s);
  if (tile == LIN_ODD128)
    return dtype == TT_BF16 ? launch_odd<LAYOUT, KIND, TT_BF16, 128>(p, s)
                            : launch_odd<LAYOUT, KIND, TT_F16, 128>(p, s);
  const bool mask = LAYOUT != LAY_TN && p.R % T_BK != 0;
  if (dtype == TT_BF16)
    return mask ? launch<LAYOUT, KIND, TT_BF16, LAYOUT != LAY_TN>(tile, p, s)
                : launch<LAYOUT, KIND, TT_BF16, false>(tile, p, s);
  return mask ? launch<LAYOUT, KIND, TT_F16, LAYOUT != LAY_TN>(tile, p, s)
              : launch<LAYOUT, KIND, TT_F16, false>(tile, p, s);
}

}  // namespace

int tt_linear_tile(int kind, int tile, int dtype, const LinArgs& p, hipStream_t s) {
  switch (kind) {
    case LIN_ACT: return typed<LAY_NT, LIN_ACT>(tile, dtype, p, s);
    case LIN_GATED: return typed<LAY_NT, LIN_GATED>(tile, dtype, p, s);
    case LIN_RES: return typed<LAY_NT, LIN_RES>(tile, dtype, p, s);
    case LIN_DROP: return typed<LAY_NT, LIN_DROP>(tile, dtype, p, s);
    case LIN_DGRAD: return typed<LAY_NN, LIN_DGRAD>(tile, dtype, p, s);
    default: return typed<LAY_TN, LIN_PLAIN>(tile, dtype, p, s);
  }
}
