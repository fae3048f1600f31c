// Dropout's masks from a counter-based generator: nothing of a mask is stored,
// every kernel that needs it forms it again from (seed, stream, element).
//
// Elements are numbered in row-major order. Element i takes the (i mod 8)-th
// 16-bit part, low halves first, of the four words that Philox4x32 makes of the
// counter (i div 8 as 64 bits, stream, 0) and the seed as 64-bit key (Salmon et
// al., "Parallel random numbers: as easy as 1, 2, 3", 2011), and is kept where
// that number is at least T = round(65536 p). 16 bits an element halve the
// integer work against 32 and put the rate within 2^-17 of p; the factor of kept
// elements is 65536 / (65536 - T), the inverse of the rate that is applied, so
// that the mean is kept exactly. Seven rounds are the fewest that the paper
// reports to pass every test of BigCrush.
#pragma once

#include "common.h"

namespace mla {

constexpr int kDropBlock = 8;       // elements per counter
constexpr int kDropAll = 1 << 16;   // T of a rate of 1: nothing is kept

struct DropKey {
  uint32_t k0, k1;
};

// The seed, a 64-bit word in device memory (a captured step changes it between
// replays without a new capture).
__device__ __forceinline__ DropKey drop_key(const int64_t* seed) {
  const uint64_t s = (uint64_t)*seed;
  return DropKey{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)s),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(s >> 32))};
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

// The numbers of elements 8 block .. 8 block + 7, two per word.
__device__ __forceinline__ u32x4_t philox(uint64_t block, uint32_t stream, DropKey key) {
  uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = stream, d = 0;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t u = (uint64_t)a * 0xD2511F53u, v = (uint64_t)c * 0xCD9E8D57u;
    a = xor3((uint32_t)(v >> 32), b, key.k0 + r * 0x9E3779B9u);
    b = (uint32_t)v;
    c = xor3((uint32_t)(u >> 32), d, key.k1 + r * 0xBB67AE85u);
    d = (uint32_t)u;
  }
  return u32x4_t{a, b, c, d};
}

// The rate as the kernels take it: an element is kept where its number exceeds
// T - 1 (as a saturating difference of 16 bits, which also holds at T = 65536),
// or all are (T = 0).
struct DropRate {
  uint32_t below;  // T - 1 in both halves
  uint32_t all;    // all ones for T = 0
};

inline DropRate drop_rate(int64_t threshold) {
  const uint32_t t = threshold > 0 ? (uint32_t)threshold - 1 : 0;
  return DropRate{t | (t << 16), threshold > 0 ? 0u : ~0u};
}

// The factor of kept elements; 0 where nothing is kept.
inline float drop_scale(int64_t threshold) {
  return threshold < kDropAll ? 65536.f / (float)(kDropAll - threshold) : 0.f;
}

// All ones in the halves whose elements are kept, zeros in the others. (Written
// out: from vectors of 16 bits the compiler makes two compares, two selects and a
// permute of it.)
__device__ __forceinline__ uint32_t drop_mask(uint32_t numbers, const DropRate& rate) {
  uint32_t m;
  asm("v_pk_sub_u16 %0, %1, %2 clamp" : "=v"(m) : "v"(numbers), "s"(rate.below));
  asm("v_pk_min_u16 %0, %1, 1 op_sel_hi:[1,0]" : "=v"(m) : "v"(m));
  asm("v_pk_sub_u16 %0, 0, %1" : "=v"(m) : "v"(m));
  return m | rate.all;
}

__device__ __forceinline__ u32x4_t drop_mask(uint64_t block, uint32_t stream, DropKey key,
                                             const DropRate& rate) {
  const u32x4_t w = philox(block, stream, key);
  return u32x4_t{drop_mask(w.x, rate), drop_mask(w.y, rate), drop_mask(w.z, rate),
                 drop_mask(w.w, rate)};
}

// Whether element e (a compile-time index once unrolled) of a block is kept.
__device__ __forceinline__ bool drop_kept(const u32x4_t& mask, int e) {
  return (mask[e >> 1] >> (16 * (e & 1))) & 1;
}

}  // namespace mla
