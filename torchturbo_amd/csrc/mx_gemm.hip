// Entry points of the products with 4-bit weights.
#include "mx_gemm.h"

namespace {

int64_t tiles(int64_t rows, int64_t cols, int bm, int bn) {
  return (rows + bm - 1) / bm * ((cols + bn - 1) / bn);
}

// Whether a product takes the kernel of few rows, which reads x once per weight tile from memory.
// us, rows / tiles (the plan's), bf16 rows: dense 17 x 7168 -> 2 x 2048 14.6 / 20.5, 64 x 7168 -> 2 x
// 2048 19.3 / 20.8, 24 x 2048 -> 7168 7.3 / 16.1, 32 x 4096 -> 2 x 14336 44 / 31; 128 experts of 2048 ->
// 2 x 768 with 512 rows 50 / 57, with 768 53 / 63, with 1024 62 / 65, of 768 -> 2048 with 512 31 / 32,
// with 1024 38 / 36; 64 of 7168 -> 2 x 2048 with 256 rows 224 / 273. E4M3 rows: 10.9 / 15.5, 13.2 / 15.9,
// 6.0 / 10.0, 31 / 22; 45 / 46, 47 / 52, 55 / 52, 29 / 32, 35 / 36; 205 / 201.
bool few_rows(int64_t M, int64_t W, int E, bool grouped) {
  if (grouped) return M <= (int64_t)6 * E;
  return M <= 16 || (M <= 64 && W < 512 * 16);
}

// Tile and parts. The largest tile reads least, but wants a block for nearly each of the 256 CUs (and
// experts that fill it); then 128 x 128; the smallest, for dense products split until the blocks fill
// the CUs, while a part keeps 1536 elements (the second kernel and its reads cost some 5 us). us, bf16
// rows, 128 x 256 / 128 x 128 / 64 x 128 / 64 x 128 in 2 / in 4 parts: 128 x 7168 -> 2 x 2048 98 / 67 /
// 44 / 30 / 22, 256 rows 99 / 68 / 46 / 31 / 30, 1531 x 5632 -> 2048 92 / 58 / 54 / 61 / 67, 1024 x
// 7168 -> 2 x 2048 100 / 70 / 78 / 93, 2048 rows 112 / 119 / 163, 4096 204 / 264 / 325. 128 experts of
// 2048 -> 2 x 768 with 32 rows each 95 / 96 / 77, with 64 115 / 117 / 104, with 128 148 / 164 / 161; 64
// of 7168 -> 2 x 2048 with 64 479 / 494 / 528, E4M3 rows 375 / 339 / 363, with 256 625 / 714 / 873.
// Dense products of 160 to 256 tiles of 128 x 128 (one for most CUs), two sets of waves with half of the
// reduction each / the better of 128 x 128 and 64 x 128: 1531 x 5632 -> 2048 47 / 56, E4M3 rows 34 / 39,
// 2048 x 2048 -> 2048 23.5 / 24.2, 14.5 / 16.3, 1024 x 7168 -> 2 x 2048 67 / 75, 44 / 50, 128 x 4096 -> 2 x
// 14336 42 / 48, 31 / 35, 1531 x 768 -> 2048 11.6 / 11.7; with 128 tiles (1024 x 5632 -> 2048) 45 / 39,
// with 512 (2048 x 7168 -> 2 x 2048) 129 / 119.
// Long reductions of E4M3 rows, 128 x 256 / 256 x 256: 4096 x 4096 -> 2 x 14336 434 / 403, 4096 x 7168
// -> 2 x 2048 114 / 97, 8192 x 7168 -> 2 x 7168 736 / 657, 4096 x 2048 -> 7168 77 / 83, 64 experts of
// 7168 -> 2 x 2048 with 512 rows each 1020 / 985, with 256 618 / 653; bf16 rows 769 / 762, 198 / 187,
// 1320 / 1305, 120 / 132, 1796 / 1876: not worth a kernel.
MxPlan plan(bool x8, int64_t M, int64_t K, int64_t W, int E, bool grouped) {
  const int64_t per = grouped ? M / E : M;
  if (x8 && K >= 4096 && per >= 384 && tiles(M, W, 256, 256) >= 224) return MxPlan{256, 256, 1};
  if (per > 96 && tiles(M, W, 128, 256) >= 224) return MxPlan{128, 256, 1};
  const int64_t t = tiles(M, W, 128, 128);
  if (!grouped && per > 96 && K >= 1024 && t >= 160 && t <= 256) return MxPlan{128, 128, 1, 2};
  if (per > 48 && t >= 224) return MxPlan{128, 128, 1};
  int parts = 1;
  if (!grouped)
    while (parts < 4 && tiles(M, W, 64, 128) * parts * 2 <= 256 && K / (parts * 2) >= 1536) parts *= 2;
  return MxPlan{64, 128, parts};
}

size_t part_bytes(const MxPlan& pl, int64_t M, int64_t W) {
  if (pl.parts == 1) return 0;
  return (size_t)(tiles(M, W, pl.bm, pl.bn) * pl.parts) * pl.bm * pl.bn * sizeof(float);
}

int check(const MxArgs& p) {
  TT_REQUIRE(p.M >= 0 && p.K >= 0 && p.N >= 0 && p.E > 0, "mx product: bad sizes");
  TT_REQUIRE(p.K % MX_GROUP == 0, "mx product: the reduction is whole groups of 32 elements");
  TT_REQUIRE(p.K < (1ll << 31) && p.N < (1ll << 30) && p.M < (1ll << 31) && p.E <= 65536,
             "mx product: sizes past 2^31");
  TT_REQUIRE(p.counts != nullptr || p.E == 1, "mx product: several experts need their counts");
  TT_REQUIRE(p.act >= 0 && p.act <= 2, "mx product: unknown activation");
  TT_REQUIRE(p.probs == nullptr || p.pdt == TT_F32 || p.pdt == TT_BF16 || p.pdt == TT_F16,
             "mx product: probabilities must be f32, bf16 or f16");
  TT_REQUIRE(p.ys == nullptr || p.N % MX_GROUP == 0,
             "mx product: outputs in 8 bits are whole groups of 32 columns");
  TT_REQUIRE(p.arow == nullptr || p.src_rows > 0 || p.M == 0, "mx product: a row map of no rows");
  if (p.M == 0 || p.N == 0) return TT_OK;
  TT_REQUIRE(p.y != nullptr, "mx product: NULL output");
  TT_REQUIRE(p.K == 0 || (p.x != nullptr && p.w != nullptr && p.ws != nullptr),
             "mx product: NULL tensor");
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w);
  TT_REQUIRE((at & 15) == 0, "mx product: rows and codes must be 16-byte aligned");
  TT_REQUIRE(p.ys == nullptr || (reinterpret_cast<uintptr_t>(p.y) & 7) == 0,
             "mx product: output codes must be 8-byte aligned");
  return TT_OK;
}

}  // namespace

extern "C" int tt_mx_product(const void* x, const uint8_t* x_scales, const int32_t* row_map,
                             int64_t src_rows, const uint8_t* codes, const uint8_t* scales,
                             int64_t M, int64_t K, int64_t N, int32_t num_experts,
                             const int64_t* tokens_per_expert, int32_t gated, int32_t act,
                             const void* probs, int probs_dtype, void* y, uint8_t* y_scales,
                             void* workspace, size_t workspace_bytes, void* stream) {
  MxArgs p = {x, x_scales, row_map, src_rows, codes, scales, M, K, N, num_experts,
                    tokens_per_expert, act, probs, probs_dtype, y, y_scales, nullptr};
  const int rc = check(p);
  if (rc != TT_OK || M == 0 || N == 0) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t W = gated ? 2 * N : N;
  const bool grouped = tokens_per_expert != nullptr;
  if (few_rows(M, W, num_experts, grouped) || !tt_mx_tile_takes(p, gated != 0))
    return tt_mx_rows(p, gated != 0, s);
  MxPlan pl = plan(x_scales != nullptr, M, K, W, num_experts, grouped);
  if (pl.parts > 1) {
    if (workspace != nullptr && workspace_bytes >= part_bytes(pl, M, W) &&
        (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)
      p.part = static_cast<float*>(workspace);
    else
      pl.parts = 1;
  }
  return tt_mx_tile(p, gated != 0, pl, s);
}

extern "C" size_t tt_mx_product_workspace(int64_t M, int64_t K, int64_t N,
                                          int32_t grouped, int32_t gated) {
  // Only reductions in whole steps of 128 are split (mx_tile.hip).
  if (M <= 0 || K <= 0 || K % 128 != 0 || N <= 0 || grouped) return 0;
  const int64_t W = gated ? 2 * N : N;
  if (few_rows(M, W, 1, false)) return 0;
  return part_bytes(plan(false, M, K, W, 1, false), M, W);
}
