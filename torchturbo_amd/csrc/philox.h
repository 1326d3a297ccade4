// Counter-based random numbers: Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
//
// Element (row, col) of a tensor takes 16 bits of its own: with seed and
// offset the two 64-bit words of a key on the device, four 32-bit words come
// from Philox with key `seed` and counter (col / 8, row, offset), and element
// col takes bits 16 (col % 2) .. + 15 of word (col % 8) / 2. It is dropped when
// they are below the threshold. So the mask depends on the key and the position
// alone, not on strides, tiles or the launch, and every kernel that needs it
// computes it again instead of reading it.
#pragma once

#include "common.h"

struct DropKey {
  uint32_t k0, k1, o0, o1;
};

// key: two int64 on the device, the same for every lane.
__device__ __forceinline__ DropKey load_key(const int64_t* __restrict__ key) {
  const uint64_t seed = (uint64_t)key[0], off = (uint64_t)key[1];
  return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

__device__ __forceinline__ void philox(const DropKey& key, uint32_t c0, uint32_t c1,
                                       uint32_t (&w)[4]) {
  uint32_t k0 = key.k0, k1 = key.k1, c2 = key.o0, c3 = key.o1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// Whether element j (0 .. 7) of the words' group of eight is kept.
__device__ __forceinline__ bool keeps(const uint32_t (&w)[4], int j, uint32_t threshold) {
  return ((w[j >> 1] >> (16 * (j & 1))) & 0xffffu) >= threshold;
}

// Word i of a group as a mask of its two 16-bit elements 2 i and 2 i + 1: all ones
// where kept. Thresholds 1 .. 65536.
__device__ __forceinline__ uint32_t keep_mask(uint32_t word, uint32_t threshold) {
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  const unsigned short t = (unsigned short)(threshold - 1);
  // w - (threshold - 1), not below 0, is at least 1 where w >= threshold.
  const u16x2 over = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, word), u16x2{t, t});
  const u16x2 one = __builtin_elementwise_min(over, u16x2{1, 1});
  return __builtin_bit_cast(uint32_t, u16x2{0, 0} - one);
}

// 1 / (share that is kept): thresholds are in steps of 2^-16, 0 (nothing
// dropped) to 65536 (everything dropped).
static inline float keep_inverse(int32_t threshold) {
  return threshold >= 65536 ? 0.0f : (float)(65536.0 / (double)(65536 - threshold));
}
