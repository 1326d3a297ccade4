// Dense product with an epilogue on the 16-bit matrix instructions (gfx950):
// C [I, J] = sum over r of A(i, r) B(r, j), rows of whole aligned 16-byte
// vectors, then what linear.h makes of the fp32 sums.
//
// Both kernels compute a tile with four waves, two by two, in 32x32 blocks of
// v_mfma_f32_32x32x16 whose operands are swapped, so that a lane holds four
// consecutive columns of one row. 64-deep k-tiles go from memory straight into LDS.
// LDS layouts: K-major operands: 128 bytes per row, chunk c in slot
// c ^ ((row >> 1) & 7), read with ds_read_b128; the others: k-row by k-row as in
// memory, chunk c in slot c ^ (4 (k-row % 4)), read with the transposing
// ds_read_b64_tr_b16. Resources end with the operand, so rows past it read as
// zeros; a K-major tail (R % 64) is masked per chunk; columns past J are read
// from wherever they lead inside the resource and never stored.
#include "gemm.h"
#include "linear.h"

namespace {

constexpr int T_NT = 256, T_BK = 64;

// A buffer resource that walks along an operand, 64 bits wide: k-tiles of
// operands of any size.
struct Walk {
  uint64_t base;
  int64_t left;
  __device__ __forceinline__ i32x4 rsrc() const {
    i32x4 r;
    r.x = (int)(uint32_t)base;
    r.y = (int)((uint32_t)(base >> 32) & 0xFFFFu);
    r.z = (int)(left <= 0 ? 0u : left < (int64_t)DM_OOB ? (uint32_t)left : DM_OOB);
    r.w = 0x00020000;
    return r;
  }
  __device__ __forceinline__ void advance(int64_t by) {
    base += (uint64_t)by;
    left -= by;
  }
};

// Fragment offset of MN-major tiles with RB bytes per k-row: columns c0 .. c0 + 31;
// the second read is at + 4 RB and k-step s adds 16 RB.
template <int RB>
__device__ __forceinline__ uint32_t frag_mn(int c0, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int col = c0 + 16 * (g & 1) + 4 * (i & 3);
  const int kr = 8 * (g >> 1) + (i >> 2);
  return (uint32_t)(kr * RB + (((col >> 3) ^ (4 * (kr & 3))) << 4) + (col & 7) * 2);
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
template <bool KM, int BR, bool GATE>
struct Operand {
  static constexpr int BYTES = BR * T_BK * 2;
  static constexpr int LOADS = BR / 32;    // per wave and k-tile, 1 KiB each
  static constexpr int FR = BR / 64;       // 32-row blocks of a wave
  static constexpr int RB = BR * 2;        // bytes of a k-row (MN-major)
  uint32_t off[LOADS];
  int kof[2];
  uint32_t frag[KM ? 4 : FR];

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
        const int c = (lane % LPR) ^ (4 * (kr & 3));
        off[q] = (uint32_t)((kr * ld + 8 * c) * 2);
      }
    }
    if constexpr (KM) {
#pragma unroll
      for (int s = 0; s < 4; ++s) frag[s] = fragk64((BR / 2) * half, s, lane);
    } else {
#pragma unroll
      for (int m = 0; m < FR; ++m) frag[m] = frag_mn<RB>((BR / 2) * half + 32 * m, lane);
    }
  }
  // Load q of a k-tile of which `valid` reduction elements exist.
  template <bool KMASK>
  __device__ __forceinline__ void load(int q, const i32x4& rs, uint32_t lds, int wave, int valid) const {
    uint32_t o = off[q];
    if constexpr (KM && KMASK) o = kof[q & 1] >= valid ? DM_OOB : o;
    dma16(o, rs, lds + (uint32_t)(LOADS * wave + q) * 1024u);
  }
  __device__ __forceinline__ uint4 read(lds_char* tile, int m, int s) const {
    if constexpr (KM) return read_k(tile, frag[s] + m * 4096);
    else return read_mn<RB>(tile, frag[m] + s * 16 * RB);
  }
};

template <int ET>
struct TypeOf;
template <>
struct TypeOf<TT_BF16> { typedef BF16T type; };
template <>
struct TypeOf<TT_F16> { typedef F16T type; };

// The sums of a wave's (32 FM) x (32 FN) part of the tile to what KIND makes of
// them, 32 rows at a time through the wave's own LDS (rows of 128 FN bytes,
// 16-byte chunk c of row r in slot c ^ r), so that a lane gets eight consecutive
// columns, with GATED their ups too.
template <int KIND, int ET, int FM, int FN>
__device__ __forceinline__ void tile_finish(const LinArgs& p, const f32x16 (&acc)[FM][FN],
                                            lds_char* region, int64_t i0, int64_t j0, int lane) {
  typedef typename TypeOf<ET>::type TT;
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int W = 32 * FN, CH = W / 4, MASK = CH - 1;  // columns and 16-byte chunks of a row
  constexpr int NG = (GATED ? W / 2 : W) / 8;            // groups of eight outputs of a row
  constexpr int RP = 64 / NG;                            // rows per pass
  typedef __attribute__((ext_vector_type(4))) float f32x4_t;
  typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;
  const int r_l = lane & 31, h = lane >> 5;
  const int gi = lane % NG, rr = lane / NG;
  const int64_t j = j0 + 8 * gi, width = GATED ? 2 * p.J : p.J;
  DropKey dk{};
  if (KIND == LIN_RES && p.threshold != 0) dk = load_key(p.key);
#pragma unroll
  for (int mi = 0; mi < FM; ++mi) {
#pragma unroll
    for (int ni = 0; ni < FN; ++ni)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 8 * ni + 2 * g + h;
        *reinterpret_cast<lds_f32x4*>(region + r_l * (W * 4) + ((c ^ (r_l & MASK)) << 4)) =
            f32x4_t{acc[mi][ni][4 * g], acc[mi][ni][4 * g + 1], acc[mi][ni][4 * g + 2],
                    acc[mi][ni][4 * g + 3]};
      }
#pragma unroll 1
    for (int ps = 0; ps < 32 / RP; ++ps) {
      const int r = ps * RP + rr;
      const int64_t i = i0 + 32 * mi + r;
      auto chunk = [&](int c) {
        return *reinterpret_cast<const lds_f32x4*>(region + r * (W * 4) + ((c ^ (r & MASK)) << 4));
      };
      float v[8], u[8] = {};
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
      float dot = 0.f;
      if (i < p.I && j < p.J) {
        if (p.part != nullptr) {
          const int64_t at = ((int64_t)blockIdx.y * p.I + i) * width + j;
          lin_store<F32T, 8, true>(p.part, at, 8, v);
          if constexpr (GATED) lin_store<F32T, 8, true>(p.part, at + p.J, 8, u);
        } else {
          dot = lin_finish<KIND, TT, 8, true>(p, i, j, 8, v, u, dk);
        }
      }
      if constexpr (KIND == LIN_DGRAD) {
        if (p.dots != nullptr && p.part == nullptr) {
#pragma unroll
          for (int off = 1; off < LIN_DOT / 8; off <<= 1) dot += __shfl_xor(dot, off, 64);
          if (i < p.I && j < p.J && j % LIN_DOT == 0)
            p.dots[i * ((p.J + LIN_DOT - 1) / LIN_DOT) + j / LIN_DOT] = dot;
        }
      }
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

template <int LAYOUT, int KIND, int BM, int BN>
struct Tile {
  static constexpr bool A_K = LAYOUT != LAY_TN, B_K = LAYOUT == LAY_NT, GATED = KIND == LIN_GATED;
  typedef Operand<A_K, BM, false> OpA;
  typedef Operand<B_K, BN, GATED> OpB;
  static constexpr int STAGE = OpA::BYTES + OpB::BYTES;
  static constexpr int BO = GATED ? BN / 2 : BN;  // output columns
  OpA a;
  OpB b;
  Walk wa, wb;
  int64_t sa, sb;  // bytes of a k-tile step
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
    wa = Walk{reinterpret_cast<uint64_t>(pa) + (uint64_t)oa,
              (A_K ? p.I * p.lda * 2 : (r0 + n) * p.lda * 2) - oa};
    sa = A_K ? T_BK * 2 : T_BK * p.lda * 2;
    const int64_t ob = B_K ? (j0 * p.ldb + r0) * 2 : (r0 * p.ldb + j0) * 2;
    wb = Walk{reinterpret_cast<uint64_t>(pb) + (uint64_t)ob,
              (B_K ? (GATED ? 2 : 1) * p.J * p.ldb * 2 : (r0 + n) * p.ldb * 2) - ob};
    sb = B_K ? T_BK * 2 : T_BK * p.ldb * 2;
    a.setup(wave, lane, wave >> 1, p.lda, 0);
    b.setup(wave, lane, wave & 1, p.ldb, p.J);
  }
};

// 256 x 256 tiles, 128 x 128 per wave (256 accumulators, one wave per SIMD), two
// 64 KiB stages. k-steps 0-2 of a k-tile multiply while they read the next
// k-step's fragments, k-step 0 with the loads of B's next k-tile into the other
// stage between its products; then one barrier, and k-step 3 multiplies while it
// reads the first fragments of the next k-tile and loads A's k-tile after that
// into this stage.
template <int LAYOUT, int KIND, int ET, bool KMASK>
__global__ __launch_bounds__(T_NT) void linear_big_kernel(LinArgs p, int ti, int tj) {
  typedef Tile<LAYOUT, KIND, 256, 256> TL;
  constexpr int FM = 4, FN = 4, NM = FM * FN, NF = FM + FN;
  constexpr int LA = TL::OpA::LOADS, LB = TL::OpB::LOADS;
  __shared__ __align__(16) char lds_raw[2 * TL::STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TL t;
  t.setup(p, ti, tj, wave, lane);
  lds_char* const lds = (lds_char*)lds_raw;
  const uint32_t lds0 = lds_addr_of(lds);
  auto load_a = [&](int q, const i32x4& rs, int kt) {
    t.a.template load<KMASK>(q, rs, lds0 + (uint32_t)(kt & 1) * TL::STAGE, wave, t.kn - kt * T_BK);
  };
  auto load_b = [&](int q, const i32x4& rs, int kt) {
    t.b.template load<KMASK>(q, rs, lds0 + (uint32_t)(kt & 1) * TL::STAGE + TL::OpA::BYTES, wave,
                             t.kn - kt * T_BK);
  };
  // Resource of k-tile kt of a walk that stands there; none past the last.
  auto at = [&](const Walk& w, int kt) {
    i32x4 r = w.rsrc();
    if (kt >= t.nkt) r.z = 0;
    return r;
  };
  uint4 a0[FM], b0[FN], a1[FM], b1[FN];
  auto frag = [&](lds_char* stg, int s, int i, uint4 (&fa)[FM], uint4 (&fb)[FN]) {
    if (i < FM) fa[i] = t.a.read(stg, i, s);
    else fb[i - FM] = t.b.read(stg + TL::OpA::BYTES, i - FM, s);
  };
  f32x16 acc[FM][FN] = {};
  {
    const i32x4 ra = at(t.wa, 0), rb = at(t.wb, 0);
#pragma unroll
    for (int q = 0; q < LA; ++q) load_a(q, ra, 0);
#pragma unroll
    for (int q = 0; q < LB; ++q) load_b(q, rb, 0);
    t.wa.advance(t.sa);
    t.wb.advance(t.sb);
    const i32x4 r1 = at(t.wa, 1);
#pragma unroll
    for (int q = 0; q < LA; ++q) load_a(q, r1, 1);
    t.wa.advance(t.sa);
    TT_WAIT_VMCNT(LA);
    TT_LDS_BARRIER();
#pragma unroll
    for (int i = 0; i < NF; ++i) frag(lds, 0, i, a0, b0);
  }
  for (int kt = 0; kt < t.nkt; ++kt) {
    lds_char* const cur = lds + (kt & 1) * TL::STAGE;
    lds_char* const nxt = lds + ((kt + 1) & 1) * TL::STAGE;
    const i32x4 rb = at(t.wb, kt + 1), ra = at(t.wa, kt + 2);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        f32x16& c = acc[i / FN][i % FN];
        c = (s & 1) ? Mma<ET>::run(b1[i % FN], a1[i / FN], c) : Mma<ET>::run(b0[i % FN], a0[i / FN], c);
        if (i < NF) {
          if (s & 1) frag(cur, s + 1, i, a0, b0);
          else frag(cur, s + 1, i, a1, b1);
        }
        if (s == 0 && (i & 1)) load_b(i / 2, rb, kt + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    TT_WAIT_VMCNT(0);
    TT_LDS_BARRIER();
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      f32x16& c = acc[i / FN][i % FN];
      c = Mma<ET>::run(b1[i % FN], a1[i / FN], c);
      if (i < NF) frag(nxt, 0, i, a0, b0);
      if (i & 1) load_a(i / 2, ra, kt + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    t.wa.advance(t.sa);
    t.wb.advance(t.sb);
  }
  TT_WAIT_VMCNT(0);
  __syncthreads();  // every wave is past its fragment reads, and every load has landed
  tile_finish<KIND, ET, FM, FN>(p, acc, lds + wave * (32 * 128 * 4), t.i0 + (wave >> 1) * 128,
                                t.j0 + (wave & 1) * (TL::BO / 2), lane);
}

// 128 x 128 tiles, 64 x 64 per wave, a ring of S 32 KiB stages with one barrier
// per k-tile, which publishes k-tile kt and frees the stage of kt - 1.
template <int LAYOUT, int KIND, int ET, bool KMASK, int S>
__global__ __launch_bounds__(T_NT) void linear_mid_kernel(LinArgs p, int ti, int tj) {
  typedef Tile<LAYOUT, KIND, 128, 128> TL;
  constexpr int FM = 2, FN = 2;
  constexpr int LA = TL::OpA::LOADS, LB = TL::OpB::LOADS, LD = LA + LB;
  __shared__ __align__(16) char lds_raw[S * TL::STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TL t;
  t.setup(p, ti, tj, wave, lane);
  lds_char* const lds = (lds_char*)lds_raw;
  const uint32_t lds0 = lds_addr_of(lds);
  auto issue = [&](int kt, int slot) {
    const i32x4 ra = t.wa.rsrc(), rb = t.wb.rsrc();
    const uint32_t at = lds0 + (uint32_t)slot * TL::STAGE;
    const int valid = t.kn - kt * T_BK;
#pragma unroll
    for (int q = 0; q < LA; ++q) t.a.template load<KMASK>(q, ra, at, wave, valid);
#pragma unroll
    for (int q = 0; q < LB; ++q) t.b.template load<KMASK>(q, rb, at + TL::OpA::BYTES, wave, valid);
    t.wa.advance(t.sa);
    t.wb.advance(t.sb);
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
  tile_finish<KIND, ET, FM, FN>(p, acc, lds + wave * (32 * 64 * 4), t.i0 + (wave >> 1) * 64,
                                t.j0 + (wave & 1) * (TL::BO / 2), lane);
}

template <int LAYOUT, int KIND, int ET, bool KMASK>
int launch(int tile, const LinArgs& p, hipStream_t s) {
  const int bo = KIND == LIN_GATED ? tile / 2 : tile;
  const int64_t ti = (p.I + tile - 1) / tile, tj = (p.J + bo - 1) / bo;
  TT_REQUIRE(ti * tj < 0x7fffffff, "linear: grid too large");
  const dim3 grid((unsigned)(ti * tj), (unsigned)p.splits), block(T_NT);
  if (tile == 256)
    hipLaunchKernelGGL((linear_big_kernel<LAYOUT, KIND, ET, KMASK>), grid, block, 0, s, p, (int)ti,
                       (int)tj);
  else
    hipLaunchKernelGGL((linear_mid_kernel<LAYOUT, KIND, ET, KMASK, 2>), grid, block, 0, s, p,
                       (int)ti, (int)tj);
  return tt_check_launch("linear");
}

template <int LAYOUT, int KIND>
int typed(int tile, int dtype, const LinArgs& p, hipStream_t s) {
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
    case LIN_DGRAD: return typed<LAY_NN, LIN_DGRAD>(tile, dtype, p, s);
    default: return typed<LAY_TN, LIN_PLAIN>(tile, dtype, p, s);
  }
}
