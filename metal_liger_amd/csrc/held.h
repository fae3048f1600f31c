// Tensors kept in 8 or 16 bits for a backward pass: rows in blocks of 32 elements (a
// row's last block may be shorter), each with one scale 2^e, elements as v / 2^e in
//   8 bits   e4m3 (3 bits of mantissa, smallest step 2^-9), e = floor(log2 m) - 7
//   16 bits  fp16 (10 bits of mantissa),                    e = floor(log2 m) - 14
// for the largest finite magnitude m of the block; e is at least -126, and -126 where
// m = 0; the scale's byte is e + 127. A block's largest element lands in [128, 256) or
// [2^14, 2^15), so nothing saturates (e4m3 ends at 448, fp16 at 65504), and the scale
// is a matter of m's exponent bits alone: 17 octaves below it (fp16: 39) still differ
// from 0. Elements that are not finite do not count for m; e4m3 keeps them as NaN. The
// scale is a power of two, so that v / 2^e rounds nothing; the rounding to e4m3 (half a
// step: 2^-4 of the value) or fp16 (2^-11) is the only one.
// The 16 bits are fp16 with a scale rather than bf16 because a backward multiplies what
// it reads: gate and up in bf16 (2^-8) took the weights' gradients of the gated block
// from 2.4e-3 to 3.5e-3 of their norm off 64 bits, 1.7e-3 being the rounding of the
// result alone; the scales are 32 bytes for 1024 elements.
#pragma once

#include "common.h"

namespace mla {
namespace held {

constexpr int kBlock = 32;

inline int64_t blocks(int64_t cols) { return (cols + kBlock - 1) / kBlock; }

// |v|'s bits where v is finite, else 0 (their order is that of the magnitudes)
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// The scale's byte from the bits of m: its exponent field less TOP, at least 1.
constexpr int kTop8 = 7, kTop16 = 14;

template <int TOP>
__device__ __forceinline__ uint32_t scale_byte(uint32_t max_bits) {
  const int e = (int)(max_bits >> 23) - TOP;
  return (uint32_t)(e > 1 ? e : 1);
}

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

__device__ __forceinline__ float inverse_of(uint32_t byte) {  // byte in 1 .. 247
  return __builtin_bit_cast(float, (254u - byte) << 23);
}

// Largest value over LANES neighbouring lanes (a power of two, aligned).
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t m) {
#pragma unroll
  for (int off = 1; off < LANES; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, off, 64);
    m = m > o ? m : o;
  }
  return m;
}

// Scales of B blocks, as the 32 / VEC neighbouring lanes that hold VEC elements of each
// find them, and whether all of a lane's own elements are finite. They nearly always
// are: the search for the largest finite one is then 1.5 operations an element, and one
// branch for all B blocks.
template <int B>
struct Scales {
  uint32_t byte[B];
  bool finite;
};

template <int TOP, int VEC, int B>
__device__ __forceinline__ Scales<B> block_scales(const float (&v)[B][VEC]) {
  uint32_t m[B], all = 0;
#pragma unroll
  for (int q = 0; q < B; ++q) {
    m[q] = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const uint32_t b = __builtin_bit_cast(uint32_t, v[q][k]) & 0x7FFFFFFFu;
      m[q] = m[q] > b ? m[q] : b;
    }
    all = all > m[q] ? all : m[q];
  }
  Scales<B> s;
  s.finite = all < 0x7F800000u;
  if (!s.finite) {
#pragma unroll
    for (int q = 0; q < B; ++q) {
      m[q] = 0;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const uint32_t b = finite_bits(v[q][k]);
        m[q] = m[q] > b ? m[q] : b;
      }
    }
  }
#pragma unroll
  for (int q = 0; q < B; ++q) s.byte[q] = scale_byte<TOP>(lanes_max<kBlock / VEC>(m[q]));
  return s;
}

__device__ __forceinline__ float finite_or_nan(float v) {
  return finite_bits(v) == (__builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu) ? v : __builtin_nanf("");
}

// Two elements as bytes 0 and 1 of the result.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
}

// VEC elements to q (VEC bytes, aligned to VEC), already divided by their scale and with
// NaN for what is not finite.
template <int VEC>
__device__ __forceinline__ void store(uint8_t* q, const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    *q = (uint8_t)pack2(x[0], 0.f);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      const int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k], x[4 * k + 1], 0, false);
      w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * k + 2], x[4 * k + 3], p, true);
    }
    __builtin_memcpy(__builtin_assume_aligned(q, VEC), w, VEC);
  }
}

// VEC elements of the bytes in w.
template <int VEC>
__device__ __forceinline__ void load(const uint32_t* w, uint32_t byte, float (&v)[VEC]) {
  const float s = scale_of(byte);
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (VEC == 1) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[0], false);
    v[0] = a[0] * s;
  } else {
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false);
      const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
      v[4 * k] = a[0] * s;
      v[4 * k + 1] = a[1] * s;
      v[4 * k + 2] = b[0] * s;
      v[4 * k + 3] = b[1] * s;
    }
  }
}

// VEC elements of the fp16 bits in w.
template <int VEC>
__device__ __forceinline__ void load16(const uint32_t* w, uint32_t byte, float (&v)[VEC]) {
  const float s = scale_of(byte);
#pragma unroll
  for (int k = 0; k < VEC; ++k)
    v[k] = static_cast<float>(__builtin_bit_cast(f16, (uint16_t)(w[k / 2] >> (k % 2 * 16)))) * s;
}

}  // namespace held
}  // namespace mla
