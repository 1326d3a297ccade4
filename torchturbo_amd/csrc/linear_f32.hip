// Dense product with an epilogue of fp32 tensors, any size and alignment (gfx950).
// Products and sums run in fp32 on v_mfma_f32_32x32x2_f32.
#include "linear.h"

namespace {

constexpr int A_NT = 256, A_BK = 32, A_CHAIN = 512;

// One block computes BT x BT of C (GATED: BT / 2 outputs, the tile's columns
// being a gate's and its up's in runs of 32), each of the four waves a quarter.
// The next k-tile is loaded into registers while one is multiplied from LDS
// (k-row-major, so that a fragment is 32 consecutive floats).
template <int LAYOUT, int KIND, int BT>
__global__ __launch_bounds__(A_NT) void linear_f32_kernel(LinArgs p, int tiles_j, int vec) {
  constexpr bool A_K = LAYOUT != LAY_TN, B_K = LAYOUT == LAY_NT;
  constexpr bool GATED = KIND == LIN_GATED;
  constexpr int F = BT / 64;                 // 32x32 blocks of a wave, each way
  constexpr int PER = BT * A_BK / A_NT;      // elements of an operand per thread and k-tile
  constexpr int LD = BT + 4;
  constexpr int BO = GATED ? BT / 2 : BT;    // output columns of a tile
  __shared__ float sa[2][A_BK][LD], sb[2][A_BK][LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = (wave >> 1) * (BT / 2), wc = (wave & 1) * (BT / 2);
  const int l32 = lane & 31, h = lane >> 5;
  const int64_t i0 = (int64_t)(blockIdx.x / tiles_j) * BT, j0 = (int64_t)(blockIdx.x % tiles_j) * BO;
  const int64_t r0 = (int64_t)blockIdx.y * p.rsplit;
  const int64_t r1 = r0 + p.rsplit < p.R ? r0 + p.rsplit : p.R;
  const float* A = static_cast<const float*>(p.a);
  const float* B = static_cast<const float*>(p.b);
  // Column of B that tile column c is, or -1. GATED (F of 32 columns per wave):
  // a wave's first half are gates, its second half their ups.
  auto bcol = [&](int c) -> int64_t {
    if constexpr (GATED) {
      const int w = c / (BT / 2), in = c % (BT / 2), up = in / (BT / 4);
      const int64_t o = j0 + w * (BT / 4) + in % (BT / 4);
      return o < p.J ? o + (up ? p.J : 0) : -1;
    }
    return j0 + c < p.J ? j0 + c : -1;
  };
  // Operand elements of a thread: K-major: PER consecutive k of one row, else
  // PER consecutive rows (columns) of one k.
  constexpr int KT = A_BK / PER > 0 ? A_BK / PER : 1;
  static_assert(PER <= A_BK, "a thread's elements lie in one row");
  const int ar = A_K ? threadIdx.x / KT : (threadIdx.x % (BT / PER)) * PER;
  const int ak = A_K ? (threadIdx.x % KT) * PER : threadIdx.x / (BT / PER);
  const int br = B_K ? threadIdx.x / KT : (threadIdx.x % (BT / PER)) * PER;
  const int bk = B_K ? (threadIdx.x % KT) * PER : threadIdx.x / (BT / PER);
  const int64_t brow = bcol(br);
  float va[PER], vb[PER];
  auto fetch = [&](int64_t k0) {
    if constexpr (A_K) {
      const int64_t i = i0 + ar, k = k0 + ak;
      const float* src = A + i * p.lda + k;
      if (i >= p.I) {
#pragma unroll
        for (int e = 0; e < PER; ++e) va[e] = 0.f;
      } else if (k + PER <= r1) {
        __builtin_memcpy(va, src, sizeof(va));
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) va[e] = k + e < r1 ? src[e] : 0.f;
      }
    } else {
      const int64_t i = i0 + ar, k = k0 + ak;
      const float* src = A + k * p.lda + i;
      if (k >= r1) {
#pragma unroll
        for (int e = 0; e < PER; ++e) va[e] = 0.f;
      } else if (i + PER <= p.I) {
        __builtin_memcpy(va, src, sizeof(va));
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) va[e] = i + e < p.I ? src[e] : 0.f;
      }
    }
    if constexpr (B_K) {
      const int64_t k = k0 + bk;
      const float* src = B + brow * p.ldb + k;
      if (brow < 0) {
#pragma unroll
        for (int e = 0; e < PER; ++e) vb[e] = 0.f;
      } else if (k + PER <= r1) {
        __builtin_memcpy(vb, src, sizeof(vb));
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) vb[e] = k + e < r1 ? src[e] : 0.f;
      }
    } else {
      const int64_t j = j0 + br, k = k0 + bk;
      const float* src = B + k * p.ldb + j;
      if (k >= r1) {
#pragma unroll
        for (int e = 0; e < PER; ++e) vb[e] = 0.f;
      } else if (j + PER <= p.J) {
        __builtin_memcpy(vb, src, sizeof(vb));
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) vb[e] = j + e < p.J ? src[e] : 0.f;
      }
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if constexpr (A_K) sa[buf][ak + e][ar] = va[e];
      else sa[buf][ak][ar + e] = va[e];
      if constexpr (B_K) sb[buf][bk + e][br] = vb[e];
      else sb[buf][bk][br + e] = vb[e];
    }
  };
  // One chain of products is at most A_CHAIN long: a longer reduction adds chains, whose
  // rounding grows with their number instead of its length.
  f32x16 acc[F][F] = {}, total[F][F] = {};
  if (r0 < r1) {
    fetch(r0);
    put(0);
    __syncthreads();
    int buf = 0;
    for (int64_t k0 = r0; k0 < r1; k0 += A_BK) {
      const bool more = k0 + A_BK < r1;
      if (more) fetch(k0 + A_BK);
#pragma unroll
      for (int s = 0; s < A_BK / 2; ++s) {
        float fa[F], fb[F];
#pragma unroll
        for (int m = 0; m < F; ++m) fa[m] = sa[buf][2 * s + h][wr + 32 * m + l32];
#pragma unroll
        for (int m = 0; m < F; ++m) fb[m] = sb[buf][2 * s + h][wc + 32 * m + l32];
#pragma unroll
        for (int m = 0; m < F; ++m)
#pragma unroll
          for (int n = 0; n < F; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[n], fa[m], acc[m][n], 0, 0, 0);
      }
      if (more) put(buf ^ 1);
      if (!more || (k0 - r0) % A_CHAIN == A_CHAIN - A_BK) {
#pragma unroll
        for (int m = 0; m < F; ++m)
#pragma unroll
          for (int n = 0; n < F; ++n) {
            total[m][n] += acc[m][n];
            acc[m][n] = f32x16{};
          }
      }
      __syncthreads();
      buf ^= 1;
    }
  }
  // Lane l holds row 32 m + l % 32, columns 32 n + 8 g + 4 (l / 32) + 0..3 of the wave's.
  DropKey dk{};
  if constexpr (KIND == LIN_DROP) dk = load_key(p.key);
  const int64_t width = GATED ? 2 * p.J : p.J;
#pragma unroll
  for (int m = 0; m < F; ++m) {
    const int64_t i = i0 + wr + 32 * m + l32;
    const bool live = i < p.I;
    float dots[F] = {};  // of each 32 columns
#pragma unroll
    for (int n = 0; n < (GATED ? (F + 1) / 2 : F); ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        // GATED with one block per wave: columns 0-15 of it are gates, 16-31 their ups.
        if (GATED && F == 1 && g >= 2) continue;
        const int64_t j = GATED ? j0 + (wave & 1) * (BT / 4) + 32 * n + 8 * g + 4 * h
                                : j0 + wc + 32 * n + 8 * g + 4 * h;
        if (!live || j >= p.J) continue;
        const int left = p.J - j < 4 ? (int)(p.J - j) : 4;
        float v[4], u[4] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = total[m][n][4 * g + e];
          if constexpr (GATED) u[e] = F == 1 ? total[m][0][4 * ((g + 2) & 3) + e] : total[m][(n + F / 2) % F][4 * g + e];
        }
        if (p.part != nullptr) {
          float* o = p.part + ((int64_t)blockIdx.y * p.I + i) * width + j;
          for (int e = 0; e < left; ++e) {
            o[e] = v[e];
            if (GATED) o[p.J + e] = u[e];
          }
        } else if (p.J % 4 == 0) {
          dots[n] += lin_finish<KIND, F32T, 4, true>(p, i, j, left, v, u, dk, lin_cols<KIND, 4>(p, j, left),
                                             lin_row<KIND, F32T, 4, true>(p, i, j, left));
        } else {
          dots[n] += lin_finish<KIND, F32T, 4, false>(p, i, j, left, v, u, dk, lin_cols<KIND, 4>(p, j, left),
                                             lin_row<KIND, F32T, 4, false>(p, i, j, left));
        }
      }
    if constexpr (KIND == LIN_DGRAD) {
      static_assert(LIN_DOT == 32, "a block's columns");
      if (p.dots != nullptr && p.part == nullptr) {
#pragma unroll
        for (int n = 0; n < F; ++n) {
          const float dot = dots[n] + __shfl_xor(dots[n], 32, 64);
          const int64_t j = j0 + wc + 32 * n;
          if (live && h == 0 && j < p.J)
            p.dots[i * ((p.J + LIN_DOT - 1) / LIN_DOT) + j / LIN_DOT] = dot;
        }
      }
    }
  }
}

template <int LAYOUT, int KIND, int BT>
int launch(const LinArgs& p, hipStream_t s) {
  const int bo = KIND == LIN_GATED ? BT / 2 : BT;
  const int64_t ti = (p.I + BT - 1) / BT, tj = (p.J + bo - 1) / bo;
  TT_REQUIRE(ti * tj < 0x7fffffff, "linear: grid too large");
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.res) |
                       reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.xs) |
                       reinterpret_cast<uintptr_t>(p.pre);
  hipLaunchKernelGGL((linear_f32_kernel<LAYOUT, KIND, BT>),
                     dim3((unsigned)(ti * tj), (unsigned)p.splits), dim3(A_NT), 0, s, p, (int)tj,
                     (int)(at % 16 == 0 && p.J % 4 == 0));
  return tt_check_launch("linear_f32");
}

template <int LAYOUT, int KIND>
int sized(const LinArgs& p, hipStream_t s) {
  // 64-wide tiles while 128-wide ones leave CUs without a block.
  const int64_t width = KIND == LIN_GATED ? 2 * p.J : p.J;
  const int64_t tiles = ((p.I + 127) / 128) * ((width + 127) / 128) * p.splits;
  return tiles >= 256 ? launch<LAYOUT, KIND, 128>(p, s) : launch<LAYOUT, KIND, 64>(p, s);
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
