// Root-mean-square norm with the residual's addition (gfx950).
//
//   h = x + residual,  rho = (mean(h^2) + eps)^(-1/2),  y = h rho w
//
// and, for the experts' products, y in E4M3 with one power of two per 32 features (mx.h). The
// statistics and the product are formed in fp32 from the unrounded sum; sum and y are rounded once, and
// so are the codes, of the unrounded y or (rounded) of y as it is stored: then they are those that the
// quantiser gives for the stored y.
// The backward, with a = gy w and xh = h rho from the rounded sum that it is given:
//
//   dh = rho (a - xh mean(a xh)) + g_sum,  dw = sum over rows of gy xh.
//
// All of it is bound by memory: every tensor is read or written once (4.3 to 4.9 TB/s up to 8192 bf16
// features, 5.7 in fp32; a large copy on this card reaches 5.1). Rows of features off eight and tensors off
// 16 bytes are read and written by single elements, with no row in flight ahead (16384 x 2047 forward 186 us
// for 56 at 2048, backward 211 for 56; fp32 4096 x 4095 142 for 46 and 131 for 48). A row stays in
// the registers of its threads between the sum of squares and the product: a wave per row up to 2048
// features, 256 threads to 8192, 1024 to 16384; longer rows are read twice. Blocks go on to further rows with the weight kept, so that it is read once per
// block, and dw is summed in registers: one partial row per block, joined by a second kernel in the
// order of the blocks.
#include <initializer_list>

#include "mx.h"

namespace {

// RT threads per row, IT chunks of eight features per thread (chunk c of thread t: c RT + t);
// IT = 0: rows of any length, read again for the second use.
template <int RT>
struct Shape {
  static constexpr int ROWS = RT >= 256 ? 1 : 256 / RT;  // rows of a block
  static constexpr int NT = RT * ROWS;
};

// Sum over the RT threads of a row; every thread gets it. `red`: one float per wave. The waves'
// sums are added in order.
template <int RT>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (RT > TT_WAVE) {
    constexpr int W = RT / TT_WAVE;
    __syncthreads();  // the sums before have been read
    if (lane_id() == 0) red[threadIdx.x / TT_WAVE] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += red[w];
  }
  return v;
}

template <bool VEC>
__device__ __forceinline__ void load_weight(float (&w)[8], const void* p, int dtype, int64_t at,
                                            int64_t left) {
  switch (dtype) {
    case TT_BF16: load8<BF16T, VEC>(w, static_cast<const uint16_t*>(p) + at, left); break;
    case TT_F16: load8<F16T, VEC>(w, static_cast<const uint16_t*>(p) + at, left); break;
    default: load8<F32T, VEC>(w, static_cast<const float*>(p) + at, left); break;
  }
}

// Eight elements as they lie in memory.
template <class T>
struct Raw8 {
  uint4 v[sizeof(typename T::storage) / 2];
  __device__ __forceinline__ void load(const typename T::storage* p) {
    v[0] = *reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(typename T::storage) == 4) v[1] = *reinterpret_cast<const uint4*>(p + 4);
  }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
    typename T::storage s[8];
    __builtin_memcpy(s, v, sizeof(s));
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = T::to_f32(s[j]);
  }
};

struct NormArgs {
  const void *x, *residual, *weight;
  int wdt;
  int64_t T, H;
  float eps;
  void *y, *sum;
  float* rstd;
  uint8_t *codes, *scales;
  int rounded;  // codes of y as rounded to the input's dtype
};

template <class T, bool VEC, int RT, int IT>
__global__ __launch_bounds__(Shape<RT>::NT) void rms_norm_fwd_kernel(NormArgs p) {
  typedef typename T::storage S;
  constexpr int ROWS = Shape<RT>::ROWS, KEEP = IT > 0 ? IT : 1;
  __shared__ float red[16];
  const int t = threadIdx.x % RT;
  const int64_t H = p.H, chunks = (H + 7) / 8;
  const int its = IT > 0 ? IT : (int)((chunks + RT - 1) / RT);
  float w[KEEP][8];
  if constexpr (IT > 0) {
#pragma unroll
    for (int c = 0; c < IT; ++c) {
      const int64_t at = ((int64_t)c * RT + t) * 8;
      if (at < H) load_weight<VEC>(w[c], p.weight, p.wdt, at, H - at);
    }
  }
  auto load_sum = [&](float (&h)[8], int64_t row, int64_t at) {
    load8<T, VEC>(h, static_cast<const S*>(p.x) + row * H + at, H - at);
    if (p.residual != nullptr) {
      float r[8];
      load8<T, VEC>(r, static_cast<const S*>(p.residual) + row * H + at, H - at);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += r[j];
    }
  };
  auto finish = [&](const float (&h)[8], const float (&wc)[8], float rho, int64_t row, int64_t at) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = h[j] * rho * wc[j];
    if (p.sum != nullptr) store8<T, VEC>(static_cast<S*>(p.sum) + row * H + at, h, H - at);
    if (p.y != nullptr) store8<T, VEC>(static_cast<S*>(p.y) + row * H + at, y, H - at);
    if (p.codes != nullptr) {  // H is a multiple of 32: a group's four lanes come together
      if (p.rounded) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = T::to_f32(T::from_f32(y[j]));
      }
      uint32_t byte;
      const uint2 q = mx_rows8(y, byte);
      *reinterpret_cast<uint2*>(p.codes + row * H + at) = q;
      if ((t & 3) == 0) p.scales[(row * H + at) / MX_GROUP] = (uint8_t)byte;
    }
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  // The next row of a thread, in flight while the one before is worked on.
  constexpr bool AHEAD = VEC && IT > 0;
  Raw8<T> xn[AHEAD ? KEEP : 1], en[AHEAD ? KEEP : 1];
  auto fetch = [&](int64_t row) {
    if (row >= p.T) return;
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int64_t at = ((int64_t)c * RT + t) * 8;
      if (at < H) {
        xn[c].load(static_cast<const S*>(p.x) + row * H + at);
        if (p.residual != nullptr) en[c].load(static_cast<const S*>(p.residual) + row * H + at);
      }
    }
  };
  const int64_t row0 = (int64_t)blockIdx.x * ROWS + threadIdx.x / RT;
  if constexpr (AHEAD) fetch(row0);
  for (int64_t row = row0; row < p.T; row += stride) {
    float h[KEEP][8];
    float s = 0.f;
    if constexpr (IT > 0) {
#pragma unroll
      for (int c = 0; c < IT; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at < H) {
          if constexpr (AHEAD) {
            xn[c].unpack(h[c]);
            if (p.residual != nullptr) {
              float r[8];
              en[c].unpack(r);
#pragma unroll
              for (int j = 0; j < 8; ++j) h[c][j] += r[j];
            }
          } else {
            load_sum(h[c], row, at);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) h[c][j] = 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < IT; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += h[c][j] * h[c][j];
      if constexpr (AHEAD) fetch(row + stride);
    } else {
      for (int c = 0; c < its; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at >= H) continue;
        load_sum(h[0], row, at);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += h[0][j] * h[0][j];
      }
    }
    const float rho = 1.f / sqrtf(row_sum<RT>(s, red) / (float)H + p.eps);
    if (p.rstd != nullptr && t == 0) p.rstd[row] = rho;
    if constexpr (IT > 0) {
#pragma unroll
      for (int c = 0; c < IT; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at < H) finish(h[c], w[c], rho, row, at);
      }
    } else {
      for (int c = 0; c < its; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at >= H) continue;
        load_sum(h[0], row, at);
        load_weight<VEC>(w[0], p.weight, p.wdt, at, H - at);
        finish(h[0], w[0], rho, row, at);
      }
    }
  }
}

struct NormBwdArgs {
  const void *h, *weight, *gy, *gsum;
  int wdt;
  const float* rstd;
  int64_t T, H;
  void* dx;
  float* part;  // [blocks, H], or NULL
};

template <class T, bool VEC, int RT, int IT>
__global__ __launch_bounds__(Shape<RT>::NT) void rms_norm_bwd_kernel(NormBwdArgs p) {
  typedef typename T::storage S;
  constexpr int ROWS = Shape<RT>::ROWS, KEEP = IT > 0 ? IT : 1;
  __shared__ float red[16];
  const int t = threadIdx.x % RT;
  const int64_t H = p.H, chunks = (H + 7) / 8;
  const int its = IT > 0 ? IT : (int)((chunks + RT - 1) / RT);
  float w[KEEP][8], dw[KEEP][8];
  if constexpr (IT > 0) {
#pragma unroll
    for (int c = 0; c < IT; ++c) {
      const int64_t at = ((int64_t)c * RT + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) dw[c][j] = w[c][j] = 0.f;
      if (at < H) load_weight<VEC>(w[c], p.weight, p.wdt, at, H - at);
    }
  }
  // The gradient of eight elements, from xh and gy.
  auto finish = [&](const float (&xh)[8], const float (&g)[8], const float (&wc)[8], float rho,
                    float mean, int64_t row, int64_t at) {
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = rho * (g[j] * wc[j] - xh[j] * mean);
    if (p.gsum != nullptr) {
      float e[8];
      load8<T, VEC>(e, static_cast<const S*>(p.gsum) + row * H + at, H - at);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += e[j];
    }
    store8<T, VEC>(static_cast<S*>(p.dx) + row * H + at, d, H - at);
  };
  auto load_pair = [&](float (&xh)[8], float (&g)[8], float rho, int64_t row, int64_t at) {
    load8<T, VEC>(xh, static_cast<const S*>(p.h) + row * H + at, H - at);
    load8<T, VEC>(g, static_cast<const S*>(p.gy) + row * H + at, H - at);
#pragma unroll
    for (int j = 0; j < 8; ++j) xh[j] *= rho;
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  // The next row of a thread, in flight while the one before is worked on.
  constexpr bool AHEAD = VEC && IT > 0;
  Raw8<T> hn[AHEAD ? KEEP : 1], gn[AHEAD ? KEEP : 1];
  float rn = 0.f;
  auto fetch = [&](int64_t row) {
    if (row >= p.T) return;
    rn = p.rstd[row];
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int64_t at = ((int64_t)c * RT + t) * 8;
      if (at < H) {
        hn[c].load(static_cast<const S*>(p.h) + row * H + at);
        gn[c].load(static_cast<const S*>(p.gy) + row * H + at);
      }
    }
  };
  const int64_t row0 = (int64_t)blockIdx.x * ROWS + threadIdx.x / RT;
  if constexpr (AHEAD) fetch(row0);
  for (int64_t row = row0; row < p.T; row += stride) {
    const float rho = AHEAD ? rn : p.rstd[row];
    float xh[KEEP][8], g[KEEP][8];
    float s = 0.f;
    if constexpr (IT > 0) {
#pragma unroll
      for (int c = 0; c < IT; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at < H) {
          if constexpr (AHEAD) {
            hn[c].unpack(xh[c]);
            gn[c].unpack(g[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) xh[c][j] *= rho;
          } else {
            load_pair(xh[c], g[c], rho, row, at);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) xh[c][j] = g[c][j] = 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < IT; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          s += g[c][j] * w[c][j] * xh[c][j];
          dw[c][j] += g[c][j] * xh[c][j];
        }
      if constexpr (AHEAD) fetch(row + stride);
    } else {
      for (int c = 0; c < its; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at >= H) continue;
        load_pair(xh[0], g[0], rho, row, at);
        load_weight<VEC>(w[0], p.weight, p.wdt, at, H - at);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += at + j < H ? g[0][j] * w[0][j] * xh[0][j] : 0.f;
      }
    }
    const float mean = row_sum<RT>(s, red) / (float)H;
    if constexpr (IT > 0) {
      if (p.dx != nullptr) {
#pragma unroll
        for (int c = 0; c < IT; ++c) {
          const int64_t at = ((int64_t)c * RT + t) * 8;
          if (at < H) finish(xh[c], g[c], w[c], rho, mean, row, at);
        }
      }
    } else if (p.dx != nullptr) {
      for (int c = 0; c < its; ++c) {
        const int64_t at = ((int64_t)c * RT + t) * 8;
        if (at >= H) continue;
        load_pair(xh[0], g[0], rho, row, at);
        load_weight<VEC>(w[0], p.weight, p.wdt, at, H - at);
        finish(xh[0], g[0], w[0], rho, mean, row, at);
      }
    }
  }
  if constexpr (IT > 0) {
    if (p.part == nullptr) return;
    // The block's rows, in order, through LDS where several waves have a row each.
    if constexpr (ROWS > 1) {
      __shared__ float sums[RT * IT * 8];
      const int mine = threadIdx.x / RT;
#pragma unroll 1
      for (int r = 0; r < ROWS; ++r) {
        if (mine == r) {
#pragma unroll
          for (int c = 0; c < IT; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float& at = sums[(c * 8 + j) * RT + t];
              at = r == 0 ? dw[c][j] : at + dw[c][j];
            }
        }
        __syncthreads();
      }
      if (mine != 0) return;
#pragma unroll
      for (int c = 0; c < IT; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[c][j] = sums[(c * 8 + j) * RT + t];
    }
#pragma unroll
    for (int c = 0; c < IT; ++c) {
      const int64_t at = ((int64_t)c * RT + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j < H) p.part[(int64_t)blockIdx.x * H + at + j] = dw[c][j];
    }
  }
}

// dw's partial rows for features past the registers' reach: block (x, y) sums feature columns x of
// the rows y, y + gridDim.y, ..., and further columns in turn.
template <class T>
__global__ __launch_bounds__(256) void rms_norm_dw_kernel(NormBwdArgs p) {
  typedef typename T::storage S;
  for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < p.H; j += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int64_t row = blockIdx.y; row < p.T; row += gridDim.y)
      v += T::to_f32(static_cast<const S*>(p.gy)[row * p.H + j]) *
           (T::to_f32(static_cast<const S*>(p.h)[row * p.H + j]) * p.rstd[row]);
    p.part[(int64_t)blockIdx.y * p.H + j] = v;
  }
}

// dw [H] from `parts` partial rows: a block takes 32 features and 32 threads each a share of the
// rows, whose sums are added in order; further features in turn.
__global__ __launch_bounds__(1024) void rms_norm_join_kernel(const float* __restrict__ part,
                                                             int parts, int64_t H,
                                                             void* __restrict__ dw, int dtype) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  for (int64_t j0 = (int64_t)blockIdx.x * 32; j0 < H; j0 += (int64_t)gridDim.x * 32) {
    const int64_t j = j0 + c;
    float v = 0.f;
    if (j < H) {
#pragma unroll 8
      for (int i = r; i < parts; i += 32) v += part[(int64_t)i * H + j];
    }
    __syncthreads();  // the sums before have been read
    sums[r][c] = v;
    __syncthreads();
    if (r == 0 && j < H) {
#pragma unroll
      for (int i = 1; i < 32; ++i) v += sums[i][c];
      store_from_f32(dw, dtype, j, v);
    }
  }
}

// Threads per row for H features, and chunks per thread: at most four (two of 1024 threads, whose
// registers hold no more), 0 past 16384 features.
int row_threads(int64_t H) { return H <= 2048 ? 64 : H <= 8192 ? 256 : 1024; }
int row_chunks(int64_t H) {
  const int rt = row_threads(H);
  return H <= 16384 ? (int)(((H + 7) / 8 + rt - 1) / rt) : 0;
}

// Blocks of a launch: as many as a CU holds with a row in work and the next in flight (more start
// later and wait for their first row; fewer leave memory idle). us at 16384 x 2048 / 4096 x 7168, bf16
// with residual: forward in 512, 768, 2048 blocks 69 / 61 / 59 and 66 / 57 / 58, backward in 256, 512, 640
// blocks 87 / 65 / 87 and 87 / 64 / 87; with no row in flight ahead 60 and 58, 97 and 98. Rows of 1024 threads
// take the same numbers, of which a CU holds fewer at once: 2048 x 16384 56 and 79, 1024 x 32768 75 and 112.
constexpr int64_t FWD_BLOCKS = 256 * 3, BWD_BLOCKS = 256 * 2;
// Blocks along the features in the kernels of the weight's gradient, which keep their launches below
// 2^32 threads (with BWD_BLOCKS parts of 256 threads, and alone of 1024) at any number of features.
constexpr int64_t COLUMN_BLOCKS = 1 << 14;
unsigned column_blocks(int64_t H, int per) {
  const int64_t want = (H + per - 1) / per;
  return (unsigned)(want < COLUMN_BLOCKS ? want : COLUMN_BLOCKS);
}
int64_t blocks_for(int64_t T, int64_t H, int64_t most) {
  const int rows = row_threads(H) >= 256 ? 1 : 256 / row_threads(H);
  const int64_t want = (T + rows - 1) / rows;
  return want < most ? want : most;
}

template <class T, bool VEC, int RT, int IT>
int launch_fwd(const NormArgs& p, hipStream_t s) {
  const int64_t blocks = blocks_for(p.T, p.H, FWD_BLOCKS);
  hipLaunchKernelGGL((rms_norm_fwd_kernel<T, VEC, RT, IT>), dim3((unsigned)blocks),
                     dim3(Shape<RT>::NT), 0, s, p);
  return tt_check_launch("rms_norm_fwd");
}

template <class T, bool VEC, int RT, int IT>
int launch_bwd(const NormBwdArgs& p, hipStream_t s) {
  const int64_t blocks = blocks_for(p.T, p.H, BWD_BLOCKS);
  hipLaunchKernelGGL((rms_norm_bwd_kernel<T, VEC, RT, IT>), dim3((unsigned)blocks),
                     dim3(Shape<RT>::NT), 0, s, p);
  int rc = tt_check_launch("rms_norm_bwd");
  if (IT > 0 || rc != TT_OK || p.part == nullptr) return rc;
  hipLaunchKernelGGL((rms_norm_dw_kernel<T>),
                     dim3(column_blocks(p.H, 256), (unsigned)blocks), dim3(256), 0, s, p);
  return tt_check_launch("rms_norm_dw");
}

#define TT_NORM_SHAPE(fn, p, s)                                            \
  switch (row_threads(p.H)) {                                              \
    case 64:                                                               \
      switch (row_chunks(p.H)) {                                           \
        case 1: return fn<T, VEC, 64, 1>(p, s);                            \
        case 2: return fn<T, VEC, 64, 2>(p, s);                            \
        case 3: return fn<T, VEC, 64, 3>(p, s);                            \
        default: return fn<T, VEC, 64, 4>(p, s);                           \
      }                                                                    \
    case 256:                                                              \
      switch (row_chunks(p.H)) {                                           \
        case 2: return fn<T, VEC, 256, 2>(p, s);                           \
        case 3: return fn<T, VEC, 256, 3>(p, s);                           \
        default: return fn<T, VEC, 256, 4>(p, s);                          \
      }                                                                    \
    default:                                                               \
      switch (row_chunks(p.H)) {                                           \
        case 2: return fn<T, VEC, 1024, 2>(p, s);                          \
        default: return fn<T, VEC, 1024, 0>(p, s);                         \
      }                                                                    \
  }

template <class T, bool VEC>
int fwd_shape(const NormArgs& p, hipStream_t s) { TT_NORM_SHAPE(launch_fwd, p, s) }
template <class T, bool VEC>
int bwd_shape(const NormBwdArgs& p, hipStream_t s) { TT_NORM_SHAPE(launch_bwd, p, s) }

// Whether rows of H elements at these addresses take 16-byte accesses (fp32 rows of eight as two).
bool aligned(int64_t H, std::initializer_list<const void*> ps) {
  uintptr_t bits = (uintptr_t)(H % 8) * 2;
  for (const void* q : ps) bits |= reinterpret_cast<uintptr_t>(q);
  return (bits & 15) == 0;
}

bool is_float(int dtype) { return dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16; }

}  // namespace

namespace {

int norm_fwd(const void* x, const void* residual, const void* weight, int weight_dtype, int dtype,
             int64_t rows, int64_t cols, float eps, void* y, void* sum, float* rstd, uint8_t* codes,
             uint8_t* scales, int rounded, void* stream) {
  TT_REQUIRE(is_float(dtype) && is_float(weight_dtype), "rms_norm: tensors must be f32, bf16 or f16");
  TT_REQUIRE(rows >= 0 && cols >= 0 && cols < (1ll << 31), "rms_norm: bad sizes");
  TT_REQUIRE((codes == nullptr) == (scales == nullptr), "rms_norm: codes and scales, or neither");
  TT_REQUIRE(codes == nullptr || cols % MX_GROUP == 0,
             "rms_norm: rows in 8 bits are whole groups of 32 features");
  if (rows == 0 || cols == 0) return TT_OK;
  TT_REQUIRE(x != nullptr && weight != nullptr, "rms_norm: NULL tensor");
  TT_REQUIRE((residual != nullptr) || (sum == nullptr), "rms_norm: a sum needs a residual");
  TT_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 7) == 0, "rms_norm: codes must be 8-byte aligned");
  const NormArgs p = {x,   residual, weight, weight_dtype, rows,   cols,   eps,
                      y,   sum,      rstd,   codes,        scales, rounded};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool vec = aligned(cols, {x, residual, weight, y, sum});
  switch (dtype) {
    case TT_BF16: return vec ? fwd_shape<BF16T, true>(p, s) : fwd_shape<BF16T, false>(p, s);
    case TT_F16: return vec ? fwd_shape<F16T, true>(p, s) : fwd_shape<F16T, false>(p, s);
    default: return vec ? fwd_shape<F32T, true>(p, s) : fwd_shape<F32T, false>(p, s);
  }
}

}  // namespace

extern "C" int tt_rms_norm_fwd(const void* x, const void* residual, const void* weight,
                               int weight_dtype, int dtype, int64_t rows, int64_t cols, float eps,
                               void* y, void* sum, float* rstd, uint8_t* codes, uint8_t* scales,
                               void* stream) {
  return norm_fwd(x, residual, weight, weight_dtype, dtype, rows, cols, eps, y, sum, rstd, codes,
                  scales, 0, stream);
}

extern "C" int tt_rms_norm_fwd_rounded(const void* x, const void* residual, const void* weight,
                                       int weight_dtype, int dtype, int64_t rows, int64_t cols,
                                       float eps, void* y, void* sum, float* rstd, uint8_t* codes,
                                       uint8_t* scales, void* stream) {
  return norm_fwd(x, residual, weight, weight_dtype, dtype, rows, cols, eps, y, sum, rstd, codes,
                  scales, 1, stream);
}

extern "C" size_t tt_rms_norm_bwd_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)blocks_for(rows, cols, BWD_BLOCKS) * (size_t)cols * sizeof(float);
}

extern "C" int tt_rms_norm_bwd(const void* h, const void* weight, int weight_dtype,
                               const float* rstd, const void* gy, const void* gsum, int dtype,
                               int64_t rows, int64_t cols, void* dx, void* dweight,
                               void* workspace, size_t workspace_bytes, void* stream) {
  TT_REQUIRE(is_float(dtype) && is_float(weight_dtype), "rms_norm: tensors must be f32, bf16 or f16");
  TT_REQUIRE(rows >= 0 && cols >= 0 && cols < (1ll << 31), "rms_norm: bad sizes");
  TT_REQUIRE(rows > 0 && cols > 0, "rms_norm: the backward of no elements is the caller's");
  TT_REQUIRE(h != nullptr && weight != nullptr && rstd != nullptr && gy != nullptr,
             "rms_norm: NULL tensor");
  if (dx == nullptr && dweight == nullptr) return TT_OK;
  TT_REQUIRE(dweight == nullptr || (workspace != nullptr &&
                                    workspace_bytes >= tt_rms_norm_bwd_workspace(rows, cols)),
             "rms_norm: workspace too small");
  const NormBwdArgs p = {h, weight, gy, gsum, weight_dtype, rstd, rows, cols, dx,
                         dweight != nullptr ? static_cast<float*>(workspace) : nullptr};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool vec = aligned(cols, {h, weight, gy, gsum, dx});
  int rc;
  switch (dtype) {
    case TT_BF16: rc = vec ? bwd_shape<BF16T, true>(p, s) : bwd_shape<BF16T, false>(p, s); break;
    case TT_F16: rc = vec ? bwd_shape<F16T, true>(p, s) : bwd_shape<F16T, false>(p, s); break;
    default: rc = vec ? bwd_shape<F32T, true>(p, s) : bwd_shape<F32T, false>(p, s); break;
  }
  if (rc != TT_OK || dweight == nullptr) return rc;
  hipLaunchKernelGGL(rms_norm_join_kernel, dim3(column_blocks(cols, 32)), dim3(1024), 0, s, p.part,
                     (int)blocks_for(rows, cols, BWD_BLOCKS), cols, dweight, weight_dtype);
  return tt_check_launch("rms_norm_join");
}
