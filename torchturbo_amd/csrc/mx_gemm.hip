// Entry points of the products with 4-bit weights.
#include "mx_gemm.h"

namespace {

// Rows per expert on average up to which the weights' stream bounds a product.
constexpr int64_t ROWS_LIMIT = 64;

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
                             void* stream) {
  const MxArgs p = {x, x_scales, row_map, src_rows, codes, scales, M, K, N, num_experts,
                    tokens_per_expert, act, probs, probs_dtype, y, y_scales};
  const int rc = check(p);
  if (rc != TT_OK || M == 0 || N == 0) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t per = M / num_experts;  // rows per expert on average
  if (per > ROWS_LIMIT && tt_mx_tile_takes(p, gated != 0)) return tt_mx_tile(p, gated != 0, s);
  return tt_mx_rows(p, gated != 0, s);
}
