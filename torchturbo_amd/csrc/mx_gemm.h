// What the products with 4-bit weights share: their arguments, epilogue and the scaled matrix
// instructions.
#pragma once

#include "gemm.h"
#include "mx.h"

// Y [M, N] = epilogue(X W[e]^T), rows [seg_e, seg_e + counts[e]) with expert e's weights.
struct MxArgs {
  const void* x;          // bf16 [*, K], or E4M3 codes
  const uint8_t* xs;      // E8M0 [*, K / 32] of E4M3 rows, NULL: bf16
  const int32_t* arow;    // row r of the product is row arow[r] of x; NULL: r
  int64_t src_rows;       // rows of x
  const uint8_t *w, *ws;  // [E, W, K / 2], [E, W, K / 32]; W = N, or 2 N with the gates' rows first
  int64_t M, K, N;
  int E;
  const int64_t* counts;  // [E], NULL: one expert with all rows
  int act;                // 0 none, 1 SiLU, 2 GELU
  const void* probs;      // [M] or NULL: factor of each row
  int pdt;
  void* y;                // bf16 [M, N], or E4M3 codes
  uint8_t* ys;            // E8M0 [M, N / 32], NULL: bf16
  float* part;            // sums of the parts of a split reduction
};

// Tile of a product of many rows, the parts that its reduction is split into (1: none), and the sets
// of waves that share a block's reduction.
struct MxPlan {
  int bm, bn, parts, halves = 1;
};

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

// Row of x that row r of the product reads. A row past the source (only a wrong map has one)
// reads row 0.
__device__ __forceinline__ int64_t mx_source_row(const MxArgs& p, int64_t r) {
  if (p.arow == nullptr) return r;
  const uint32_t v = (uint32_t)p.arow[r];
  return v < (uint64_t)p.src_rows ? (int64_t)v : 0;
}

// Activation in fp32. The exponential is the hardware's (about 2^-22 relative), the output's
// rounding 2^-9.
__device__ __forceinline__ float mx_act(float a, int act) {
  if (act == 1) return a / (1.f + __expf(-a));
  if (act == 2) return 0.5f * a * (1.f + erff(a * 0.70710678118654752f));
  return a;
}

// The tile of 16 weight rows x 128 reduction elements by 128 x 16 of E4M3 rows, both with their
// groups' powers of two. Lane l holds weight row l % 16, elements 32 g .. + 31 (g = l / 16), and
// of row l % 16 of x elements 16 g .. + 15 and 64 + 16 g .. + 15; both scales are those of group g.
// The result: weight rows 4 g + 0..3 of row l % 16 of x.
//
// The instruction adds the products of eight consecutive elements first and keeps, of each such set,
// what is at least 2^-13 of its largest product; sets and accumulator add in fp32 (measured with
// single elements). A product has at most six significant bits (two by four: 1.5 x 1.875 is 45 / 16), so
// only those below 2^-8 of their set's largest lose any. The sum is off by 2^-10 of the set's magnitudes at most; on normal
// data the outputs are off by 1.6e-4 of their norm, a tenth of what rounding them to bf16 adds (0.0017).
// Products of bf16 rows do not use it.
template <int WSEL, int XSEL>
__device__ __forceinline__ f32x4_t mx_mma16(const uint4& w, const uint4& x0, const uint4& x1,
                                            uint32_t ws, uint32_t xs, const f32x4_t& c) {
  const i32x8 a = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const i32x8 b = {(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w,
                   (int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, WSEL, (int)ws, XSEL,
                                                           (int)xs);
}

// 32 weight rows x 64 elements by 64 x 32: lane l holds weight row l % 32, elements 32 g .. + 31
// (g = l / 32), of x elements 16 g .. + 15 and 32 + 16 g .. + 15, scales of group g. The result:
// register 4 q + e is weight row 8 q + 4 g + e of row l % 32 of x.
template <int WSEL, int XSEL>
__device__ __forceinline__ f32x16 mx_mma32(const uint4& w, const uint4& x0, const uint4& x1,
                                           uint32_t ws, uint32_t xs, const f32x16& c) {
  const i32x8 a = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const i32x8 b = {(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w,
                   (int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 0, WSEL, (int)ws, XSEL,
                                                          (int)xs);
}

// Eight outputs at row r, columns j .. j + 7 (fewer at the row's end).
__device__ __forceinline__ void mx_store_bf16(const MxArgs& p, int64_t r, int64_t j,
                                              const float (&v)[8]) {
  uint16_t* const y = static_cast<uint16_t*>(p.y) + r * p.N + j;
  if ((p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
    const uint2 a = pack4<TT_BF16>(v[0], v[1], v[2], v[3]), b = pack4<TT_BF16>(v[4], v[5], v[6], v[7]);
    *reinterpret_cast<uint4*>(y) = uint4{a.x, a.y, b.x, b.y};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e < p.N) y[e] = f32_to_bf16(v[e]);
  }
}

// The same in 8 bits; four neighbouring lanes hold a group.
__device__ __forceinline__ void mx_store_rows(const MxArgs& p, int64_t r, int64_t j,
                                              const float (&v)[8]) {
  uint32_t byte;
  const uint2 q = mx_rows8(v, byte);
  *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.y) + r * p.N + j) = q;
  if ((j & 31) == 0) p.ys[(r * p.N + j) / MX_GROUP] = (uint8_t)byte;
}

}  // namespace

// Few rows per expert (mx_rows.hip); operands already checked.
int tt_mx_rows(const MxArgs& p, bool gated, hipStream_t s);
// Many rows per expert (mx_tile.hip), and whether the sizes and addresses fit its offsets.
int tt_mx_tile(const MxArgs& p, bool gated, MxPlan plan, hipStream_t s);
bool tt_mx_tile_takes(const MxArgs& p, bool gated);
