// Copies of matrices of any size and strides to dense ones padded with zeros to sizes in
// multiples of 8, and back without the padding: up to kMaxPads of them in one launch, one
// before and one after a padded call, of which the host's time decides ([100, 333] x 1111
// in bf16 with bias, gelu and residual, forward and backward: 223 us with a fill and a
// copy for every operand, 144 so). A thread moves 8 neighbouring columns of the padded
// side, 16 bytes at a time there, element by element on the other side.
#pragma once

#include "common.h"

namespace mla {
namespace ffn {

constexpr int kMaxPads = 8;

struct PadJob {
  void* any;         // rows x cols, element (r, c) at r * s0 + c * s1
  void* wide;        // wrows x wcols, dense; wcols a multiple of 8
  int64_t rows, cols, s0, s1, wrows, wcols;
  int64_t end;       // groups of 8 columns up to and with this one
};

struct PadJobs {
  PadJob job[kMaxPads];
  int count;
};

template <typename E, bool TO_WIDE>
__global__ __launch_bounds__(256) void pad_kernel(const PadJobs jobs) {
  const int64_t total = jobs.job[jobs.count - 1].end, stride = (int64_t)gridDim.x * 256;
  int j = 0;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += stride) {
    while (u >= jobs.job[j].end) ++j;
    const PadJob& p = jobs.job[j];
    const int64_t g = u - (j ? jobs.job[j - 1].end : 0);
    const uint32_t per = (uint32_t)(p.wcols / 8);  // (a 32-bit division wherever it does)
    const int64_t row = g >> 32 ? g / per : (uint32_t)g / per, c = 8 * (g - row * per);
    if (row >= p.rows && !TO_WIDE) continue;
    E* any = static_cast<E*>(p.any) + (row < p.rows ? row : 0) * p.s0 + c * p.s1;
    E* wide = static_cast<E*>(p.wide) + row * p.wcols + c;
    constexpr int P = 16 / (int)sizeof(E);
    Pack<E, P> v[8 / P];
    if constexpr (TO_WIDE) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e / P].v[e % P] = row < p.rows && c + e < p.cols ? any[e * p.s1] : (E)0;
#pragma unroll
      for (int i = 0; i < 8 / P; ++i) reinterpret_cast<Pack<E, P>*>(wide)[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8 / P; ++i) v[i] = reinterpret_cast<const Pack<E, P>*>(wide)[i];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < p.cols) any[e * p.s1] = v[e / P].v[e % P];
    }
  }
}

inline int launch_pads(PadJobs& jobs, int elem_bytes, bool to_wide, hipStream_t st) {
  int64_t end = 0;
  for (int j = 0; j < jobs.count; ++j) {
    end += jobs.job[j].wrows * (jobs.job[j].wcols / 8);
    jobs.job[j].end = end;
  }
  if (end == 0) return ML_OK;
  const int64_t blocks = (end + 255) / 256;
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
  if (elem_bytes == 2) {
    if (to_wide) pad_kernel<uint16_t, true><<<grid, 256, 0, st>>>(jobs);
    else pad_kernel<uint16_t, false><<<grid, 256, 0, st>>>(jobs);
  } else {
    if (to_wide) pad_kernel<uint32_t, true><<<grid, 256, 0, st>>>(jobs);
    else pad_kernel<uint32_t, false><<<grid, 256, 0, st>>>(jobs);
  }
  ML_LAUNCH_CHECK();
  return ML_OK;
}

}  // namespace ffn
}  // namespace mla
