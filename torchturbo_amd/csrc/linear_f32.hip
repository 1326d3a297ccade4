// Dense product with an epilogue of fp32 tensors, any size and alignment (gfx950).
// Products and sums run in fp32 on v_mfma_f32_32x32x2_f32. 2048 x 8192 -> 2048 613 us (112
// TFLOP/s; a plain product of torch 454), 4096 x 1024 -> 3000 298 us, 512 x 256 -> 512 11 us;
// with 4001 x 1201 -> 1703, whose rows start at no multiple of 16 bytes, 192 us NT, 205 NN
// and 311 TN. Tiles of 128 x 128 are 2 to 7 % faster where they fill the CUs in whole rounds
// (2048 cubed 177 in place of 189) and up to half slower where not (4001 x 1703 -> 1201 313
// us); v_mfma_f32_16x16x4_f32 is 2 to 5 % slower.
#include "linear.h"

namespace {

constexpr int A_NT = 256, A_BT = 64, A_BK = 32, A_CHAIN = 512;

// An operand of a tile of A_BT rows (columns): 32-deep k-tiles in chunks of four elements,
// LOADS of them per thread. A load is always of 16 bytes, at an address moved back where
// they would pass the operand's end, so that it never waits for another; the
// elements are put in place, and those past a row's end cleared, when it has arrived.
// In LDS a K-major operand lies row by row, the other one k-row by k-row, each with a
// stride that spreads a fragment's lanes over all banks.
// GATE: per half of the tile, A_BT / 4 rows of the operand's first half, then their ups.
// FAR: rows too far apart for 32-bit offsets, or an operand of fewer than four elements:
// every element by itself.
template <bool KM, bool GATE, bool FAR>
struct Operand32 {
  static constexpr int LOADS = A_BT / 32;
  static constexpr int LD = KM ? A_BK + 4 : A_BT + 8;
  static constexpr int FLOATS = LD * (KM ? A_BT : A_BK);
  const float* base;
  int64_t last;        // the last element that 16 bytes can start at
  int64_t first_at;    // the tile's first element in k-tile 0
  uint64_t off[LOADS]; // bytes from there to the chunk
  int64_t step;        // elements of a k-tile
  int at[LOADS];       // the chunk's place in the reduction
  int most[LOADS];     // its elements that exist, by the other dimension
  int slot[LOADS];     // its place in LDS
  bool inside;         // every row of the tile exists

  // rows x R elements (GATE: 2 x rows), from row `first` and reduction element r0 on.
  __device__ __forceinline__ void setup(const void* p, int64_t ld, int64_t rows, int64_t R,
                                        int64_t first, int64_t r0) {
    base = static_cast<const float*>(p);
    last = rows * R * (GATE ? 2 : 1) - 4;
    first_at = KM ? first * ld + r0 : r0 * ld + first;
    step = KM ? A_BK : A_BK * ld;
    inside = first + (GATE ? A_BT / 2 : A_BT) <= rows;
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const int id = threadIdx.x + A_NT * q;
      if constexpr (KM) {
        const int r = id / (A_BK / 4), c = id % (A_BK / 4);
        int64_t row = r, in = r;
        if constexpr (GATE) {
          in = r / (A_BT / 2) * (A_BT / 4) + r % (A_BT / 2) % (A_BT / 4);
          row = (r % (A_BT / 2) / (A_BT / 4)) * rows + in;
        }
        off[q] = (uint64_t)(row * ld + 4 * c) * 4;
        at[q] = 4 * c;
        most[q] = first + in < rows ? 4 : 0;
        slot[q] = r * LD + 4 * c;
      } else {
        const int kr = id / (A_BT / 4), c = id % (A_BT / 4);
        const int64_t left = rows - first - 4 * c;
        off[q] = (uint64_t)(kr * ld + 4 * c) * 4;
        at[q] = kr;
        most[q] = left <= 0 ? 0 : left < 4 ? (int)left : 4;
        slot[q] = kr * LD + 4 * c;
      }
    }
  }
  // Whether 32-bit offsets reach a tile's elements.
  static bool near(int64_t ld, int64_t rows) {
    return (KM ? (A_BT + (GATE ? rows : 0)) * ld : (int64_t)A_BK * ld + A_BT) * 4 < (1ll << 32) - 1024;
  }
  __device__ __forceinline__ void load(f32x4_t (&v)[LOADS], int kt) const {
    const int64_t at_kt = first_at + kt * step;
    if constexpr (!FAR) {
      const int64_t from = at_kt < last ? at_kt : last, left = (last - from) * 4;
      const char* const p = reinterpret_cast<const char*>(base + from);
      const uint32_t reach = left < 0xfffffff0ll ? (uint32_t)left : 0xfffffff0u;
#pragma unroll
      for (int q = 0; q < LOADS; ++q) {
        const uint32_t o = (uint32_t)off[q];
        __builtin_memcpy(&v[q], p + (o < reach ? o : reach), 16);
      }
    } else {
#pragma unroll
      for (int q = 0; q < LOADS; ++q) {
        const int64_t o = at_kt + (int64_t)(off[q] / 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q][e] = o + e < last + 4 ? base[o + e] : 0.f;
      }
    }
  }
  // What `load` brought for k-tile kt, of which kn reduction elements exist from k-tile 0 on.
  __device__ __forceinline__ f32x4_t trim(const f32x4_t& v, int q, int kt, int kn) const {
    const int left = kn - kt * A_BK - at[q];
    const int n = KM ? (left < most[q] ? left : most[q]) : (left > 0 ? most[q] : 0);
    const int64_t o = first_at + kt * step + (int64_t)(off[q] / 4);
    const int moved = !FAR && o > last ? (int)(o - last < 4 ? o - last : 4) : 0;
    f32x4_t r{};
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int f = e; f < 4; ++f) r[e] = e < n && e + moved == f ? v[f] : r[e];
    return r;
  }
  // Into LDS.
  __device__ __forceinline__ void put(float* lds, const f32x4_t (&v)[LOADS], int kt, int kn) const {
    if (inside && (kt + 1) * A_BK <= kn) {
#pragma unroll
      for (int q = 0; q < LOADS; ++q) *reinterpret_cast<f32x4_t*>(lds + slot[q]) = v[q];
    } else {
#pragma unroll
      for (int q = 0; q < LOADS; ++q)
        *reinterpret_cast<f32x4_t*>(lds + slot[q]) = trim(v[q], q, kt, kn);
    }
  }
  // Reduction elements 8 s + 4 h + 0..3 of row r.
  static __device__ __forceinline__ f32x4_t fragment(const float* lds, int r, int s, int h) {
    if constexpr (KM) {
      return *reinterpret_cast<const f32x4_t*>(lds + r * LD + 8 * s + 4 * h);
    } else {
      const float* p = lds + (8 * s + 4 * h) * LD + r;
      return f32x4_t{p[0], p[LD], p[2 * LD], p[3 * LD]};
    }
  }
};

// One block computes A_BT x A_BT of C (GATED: A_BT / 2 outputs, each half of the tile's columns
// being gates and their ups), each of the four waves a quarter. While a k-tile is
// multiplied from LDS the next one goes there and the two after it are on their way. Product j of four takes
// reduction elements j and 4 + j of eight, so that a fragment is 16 consecutive bytes of a
// K-major operand.
template <int LAYOUT, int KIND, bool FAR>
__global__ __launch_bounds__(A_NT) void linear_f32_kernel(LinArgs p, int tiles_j) {
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int F = A_BT / 64;             // 32x32 blocks of a wave, each way
  constexpr int BO = GATED ? A_BT / 2 : A_BT;  // output columns of a tile
  typedef Operand32<LAYOUT != LAY_TN, false, FAR> OpA;
  typedef Operand32<LAYOUT == LAY_NT, GATED, FAR> OpB;
  constexpr int FLOATS = 2 * (OpA::FLOATS + OpB::FLOATS);
  __shared__ __align__(16) float lds[FLOATS];
  float* const sa[2] = {lds, lds + OpA::FLOATS};
  float* const sb[2] = {lds + 2 * OpA::FLOATS, lds + 2 * OpA::FLOATS + OpB::FLOATS};
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * (A_BT / 2), wc = (wave & 1) * (A_BT / 2);
  const int l32 = lane & 31, h = lane >> 5;
  const int64_t i0 = (int64_t)(blockIdx.x / tiles_j) * A_BT, j0 = (int64_t)(blockIdx.x % tiles_j) * BO;
  const int64_t r0 = (int64_t)blockIdx.y * p.rsplit;
  const int kn = (int)(r0 + p.rsplit < p.R ? p.rsplit : p.R - r0), nkt = (kn + A_BK - 1) / A_BK;
  OpA oa;
  OpB ob;
  oa.setup(p.a, p.lda, p.I, p.R, i0, r0);
  ob.setup(p.b, p.ldb, p.J, p.R, j0, r0);
  // Loads past the last k-tile are made all the same (and trimmed to nothing), in whole
  // pairs of k-tiles: where some are skipped, the compiler waits for all of them.
  f32x4_t va[2][OpA::LOADS], vb[2][OpB::LOADS];
  auto fetch = [&](int kt, int buf) {
    oa.load(va[buf], kt);
    ob.load(vb[buf], kt);
  };
  // One chain of products is at most A_CHAIN long: a longer reduction adds chains, whose
  // rounding grows with their number instead of its length.
  f32x16 acc[F][F] = {}, total[F][F] = {};
  f32x4_t fa[2][F], fb[2][F];
  auto read = [&](int buf, int s) {
#pragma unroll
    for (int m = 0; m < F; ++m) fa[s & 1][m] = OpA::fragment(sa[buf], wr + 32 * m + l32, s, h);
#pragma unroll
    for (int n = 0; n < F; ++n) fb[s & 1][n] = OpB::fragment(sb[buf], wc + 32 * n + l32, s, h);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n)
          acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[s & 1][n][j], fa[s & 1][m][j],
                                                           acc[m][n], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  // Multiplies k-tile kt, a fragment's eight deep at a time while the next ones are read.
  // After the first, kt + 1 goes to LDS and kt + 3 is asked for; before the last, a barrier
  // publishes kt + 1, and frees kt's stage.
  auto step = [&](int kt, int buf) {
    read(buf, 1);
    multiply(0);
    oa.put(sa[buf ^ 1], va[buf ^ 1], kt + 1, kn);
    ob.put(sb[buf ^ 1], vb[buf ^ 1], kt + 1, kn);
    fetch(kt + 3, buf ^ 1);
    read(buf, 2);
    multiply(1);
    read(buf, 3);
    multiply(2);
    TT_LDS_BARRIER();
    read(buf ^ 1, 0);
    multiply(3);
  };
  fetch(0, 0);
  fetch(1, 1);
  oa.put(sa[0], va[0], 0, kn);
  ob.put(sb[0], vb[0], 0, kn);
  fetch(2, 0);
  TT_LDS_BARRIER();
  read(0, 0);
  for (int first = 0; first < nkt; first += A_CHAIN / A_BK) {
    const int end = first + A_CHAIN / A_BK < nkt ? first + A_CHAIN / A_BK : nkt;
    for (int kt = first; kt < end; kt += 2) {
      step(kt, 0);
      step(kt + 1, 1);
    }
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
      for (int n = 0; n < F; ++n) {
        total[m][n] += acc[m][n];
        acc[m][n] = f32x16{};
      }
  }
  __syncthreads();
  static_assert(LIN_WAVE_FLOATS<F> * 4 <= FLOATS, "the waves' rows");
  // Lane l holds row 32 m + l % 32, columns 32 n + 8 g + 4 (l / 32) + 0..3.
  auto stage = [&](int m, auto put) {
#pragma unroll
    for (int n = 0; n < F; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        put(l32, 32 * n + 8 * g + 4 * h,
            f32x4_t{total[m][n][4 * g], total[m][n][4 * g + 1], total[m][n][4 * g + 2],
                    total[m][n][4 * g + 3]});
  };
  lin_finish_wave<KIND, F32T, F, F>(p, stage, lds + wave * LIN_WAVE_FLOATS<F>, i0 + wr,
                                    j0 + (GATED ? wc / 2 : wc), lane);
}

template <int LAYOUT, int KIND, bool FAR>
int launch(const LinArgs& p, hipStream_t s) {
  const int bo = KIND == LIN_GATED ? A_BT / 2 : A_BT;
  const int64_t ti = (p.I + A_BT - 1) / A_BT, tj = (p.J + bo - 1) / bo;
  TT_REQUIRE(tt_grid_ok(ti * tj, A_NT), "linear: grid too large");
  hipLaunchKernelGGL((linear_f32_kernel<LAYOUT, KIND, FAR>),
                     dim3((unsigned)(ti * tj), (unsigned)p.splits), dim3(A_NT), 0, s, p,
                     (int)tj);
  return tt_check_launch("linear_f32");
}

template <int LAYOUT, int KIND>
int sized(const LinArgs& p, hipStream_t s) {
  constexpr bool GATED = KIND == LIN_GATED;
  typedef Operand32<LAYOUT != LAY_TN, false, false> OpA;
  typedef Operand32<LAYOUT == LAY_NT, GATED, false> OpB;
  if (p.I * p.R < 4 || p.J * p.R < 4 || !OpA::near(p.lda, p.I) || !OpB::near(p.ldb, p.J))
    return launch<LAYOUT, KIND, true>(p, s);
  return launch<LAYOUT, KIND, false>(p, s);
}

}  // namespace

int tt_linear_f32(int kind, const LinArgs& p, hipStream_t s) {
  switch (kind) {
    case LIN_ACT: return sized<LAY_NT, LIN_ACT>(p, s);
    case LIN_GATED: return sized<LAY_NT, LIN_GATED>(p, s);
    case LIN_RES: return sized<LAY_NT, LIN_RES>(p, s);
    case LIN_DROP: return sized<LAY_NT, LIN_DROP>(p, s);
    case LIN_DGRAD: return sized<LAY_NN, LIN_DGRAD>(p, s);
    default: return sized<LAY_TN, LIN_PLAIN>(p, s);
  }
}
