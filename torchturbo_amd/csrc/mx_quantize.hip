// Quantisation to the microscaling formats and back (gfx950): weights to E2M1, rows to E4M3, with
// one E8M0 byte per 32 elements of a row (mx.h).
//
// Bound by memory. A thread holds eight elements, four neighbouring lanes a group, which exchange
// its largest magnitude in two steps; each element is read and each code written once.
#include "mx.h"

namespace {

constexpr int Q_NT = 256;

// Thread i takes elements 8 i .. 8 i + 7 (rows are whole groups, so groups are consecutive).
template <class T, bool VEC, bool FOUR>
__global__ __launch_bounds__(Q_NT) void mx_quantize_kernel(
    const typename T::storage* __restrict__ x, int64_t n8, uint32_t* __restrict__ codes,
    uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * Q_NT + threadIdx.x;
  if (i >= n8) return;  // n8 is a multiple of 4: a group's lanes leave together
  float v[8];
  load8<T, VEC>(v, x + 8 * i, 8);
  uint32_t c;
  if constexpr (FOUR) {
    c = mx_byte<2>(mx_amax4(v));
    codes[i] = c == 255u ? 0u : mx_e2m1x8(v, mx_scale(c));
  } else {
    const uint2 q = mx_rows8(v, c);
    reinterpret_cast<uint2*>(codes)[i] = q;
  }
  if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)c;
}

template <class T, bool VEC>
__global__ __launch_bounds__(Q_NT) void mx_dequantize4_kernel(
    const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n8,
    typename T::storage* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * Q_NT + threadIdx.x;
  if (i >= n8) return;
  const uint4 w = mx_bf16x8(codes[i], scales[i >> 2]);
  if constexpr (VEC && __is_same(T, BF16T)) {
    *reinterpret_cast<uint4*>(out + 8 * i) = w;
  } else {
    const uint32_t p[4] = {w.x, w.y, w.z, w.w};
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(p[j] << 16);
      v[2 * j + 1] = __uint_as_float(p[j] & 0xffff0000u);
    }
    store8<T, VEC>(out + 8 * i, v, 8);
  }
}

template <class T, bool VEC>
__global__ __launch_bounds__(Q_NT) void mx_dequantize8_kernel(
    const uint2* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n8,
    typename T::storage* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * Q_NT + threadIdx.x;
  if (i >= n8) return;
  const uint2 q = codes[i];
  const float s = mx_scale(scales[i >> 2]);
  float v[8];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int w = (int)(j ? q.y : q.x);
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[4 * j] = lo[0] * s;
    v[4 * j + 1] = lo[1] * s;
    v[4 * j + 2] = hi[0] * s;
    v[4 * j + 3] = hi[1] * s;
  }
  store8<T, VEC>(out + 8 * i, v, 8);
}

int check(const char* what, const void* x, int dtype, int64_t rows, int64_t cols, const void* codes,
          const void* scales, int align, int64_t* n8) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16,
             "%s: values must be f32, bf16 or f16", what);
  TT_REQUIRE(rows >= 0 && cols >= 0 && cols % MX_GROUP == 0,
             "%s: rows are whole groups of 32 elements", what);
  TT_REQUIRE(cols == 0 || rows <= (1ll << 42) / cols, "%s: too many elements", what);
  *n8 = rows * cols / 8;
  if (*n8 == 0) return TT_OK;
  TT_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, "%s: NULL tensor", what);
  TT_REQUIRE((reinterpret_cast<uintptr_t>(codes) & (align - 1)) == 0,
             "%s: codes must be %d-byte aligned", what, align);
  TT_REQUIRE(tt_grid_ok((*n8 + Q_NT - 1) / Q_NT, Q_NT), "%s: grid too large", what);
  return TT_OK;
}

template <class T, bool FOUR>
int quantize(const void* x, int64_t n8, void* codes, uint8_t* scales, hipStream_t s) {
  typedef typename T::storage S;
  const dim3 grid((unsigned)((n8 + Q_NT - 1) / Q_NT));
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0)
    hipLaunchKernelGGL((mx_quantize_kernel<T, true, FOUR>), grid, dim3(Q_NT), 0, s,
                       static_cast<const S*>(x), n8, static_cast<uint32_t*>(codes), scales);
  else
    hipLaunchKernelGGL((mx_quantize_kernel<T, false, FOUR>), grid, dim3(Q_NT), 0, s,
                       static_cast<const S*>(x), n8, static_cast<uint32_t*>(codes), scales);
  return tt_check_launch("mx_quantize");
}

template <class T, bool FOUR>
int dequantize(const void* codes, const uint8_t* scales, int64_t n8, void* out, hipStream_t s) {
  typedef typename T::storage S;
  const dim3 grid((unsigned)((n8 + Q_NT - 1) / Q_NT));
  const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  if constexpr (FOUR) {
    const uint32_t* q = static_cast<const uint32_t*>(codes);
    if (vec) hipLaunchKernelGGL((mx_dequantize4_kernel<T, true>), grid, dim3(Q_NT), 0, s, q, scales, n8, static_cast<S*>(out));
    else hipLaunchKernelGGL((mx_dequantize4_kernel<T, false>), grid, dim3(Q_NT), 0, s, q, scales, n8, static_cast<S*>(out));
  } else {
    const uint2* q = static_cast<const uint2*>(codes);
    if (vec) hipLaunchKernelGGL((mx_dequantize8_kernel<T, true>), grid, dim3(Q_NT), 0, s, q, scales, n8, static_cast<S*>(out));
    else hipLaunchKernelGGL((mx_dequantize8_kernel<T, false>), grid, dim3(Q_NT), 0, s, q, scales, n8, static_cast<S*>(out));
  }
  return tt_check_launch("mx_dequantize");
}

template <bool FOUR>
int quantize_typed(const char* what, const void* x, int dtype, int64_t rows, int64_t cols,
                   void* codes, uint8_t* scales, void* stream) {
  int64_t n8;
  const int rc = check(what, x, dtype, rows, cols, codes, scales, FOUR ? 4 : 8, &n8);
  if (rc != TT_OK || n8 == 0) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case TT_BF16: return quantize<BF16T, FOUR>(x, n8, codes, scales, s);
    case TT_F16: return quantize<F16T, FOUR>(x, n8, codes, scales, s);
    default: return quantize<F32T, FOUR>(x, n8, codes, scales, s);
  }
}

template <bool FOUR>
int dequantize_typed(const char* what, const void* codes, const uint8_t* scales, int64_t rows,
                     int64_t cols, void* out, int dtype, void* stream) {
  int64_t n8;
  const int rc = check(what, out, dtype, rows, cols, codes, scales, FOUR ? 4 : 8, &n8);
  if (rc != TT_OK || n8 == 0) return rc;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case TT_BF16: return dequantize<BF16T, FOUR>(codes, scales, n8, out, s);
    case TT_F16: return dequantize<F16T, FOUR>(codes, scales, n8, out, s);
    default: return dequantize<F32T, FOUR>(codes, scales, n8, out, s);
  }
}

}  // namespace

extern "C" int tt_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t cols,
                                 uint8_t* codes, uint8_t* scales, void* stream) {
  return quantize_typed<true>("mxfp4_quantize", x, dtype, rows, cols, codes, scales, stream);
}
extern "C" int tt_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                   int64_t cols, void* out, int dtype, void* stream) {
  return dequantize_typed<true>("mxfp4_dequantize", codes, scales, rows, cols, out, dtype, stream);
}
extern "C" int tt_mxfp8_quantize(const void* x, int dtype, int64_t rows, int64_t cols,
                                 uint8_t* codes, uint8_t* scales, void* stream) {
  return quantize_typed<false>("mxfp8_quantize", x, dtype, rows, cols, codes, scales, stream);
}
extern "C" int tt_mxfp8_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                   int64_t cols, void* out, int dtype, void* stream) {
  return dequantize_typed<false>("mxfp8_dequantize", codes, scales, rows, cols, out, dtype, stream);
}
