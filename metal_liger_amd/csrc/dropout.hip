// Dropout, with the add of a residual that follows it, for gfx950 (no reference
// counterpart: nn.Dropout and the adds around it are left to torch there).
//
//   out_i = kept_i ? scale * x_i : 0      (+ residual_i)
//
// with the masks of dropout.h; the gradient is the same kernel over dy, so that
// neither direction stores or reads a mask. A dropped element gives 0 whatever x
// holds there, infinities and NaN included.
#include "dropout.h"

namespace mla {
namespace {

constexpr int kThreads = 256;

// A block of 8 elements at i (the last one may hold fewer), in single accesses.
template <typename T>
__device__ void drop_block(const T* x, const T* res, T* out, int64_t i, int64_t n, DropKey key,
                           uint32_t stream, const DropRate& rate, float scale) {
  const u32x4_t m = drop_mask(i / kDropBlock, stream, key, rate);
#pragma unroll
  for (int e = 0; e < kDropBlock; ++e) {
    if (i + e >= n) break;
    float v = drop_kept(m, e) ? to_f32(x[i + e]) * scale : 0.f;
    if (res) v += to_f32(res[i + e]);
    out[i + e] = from_f32<T>(v);
  }
}

template <typename T, bool RES>
__global__ __launch_bounds__(kThreads) void dropout_scalar(const T* x, const T* res, T* out,
                                                           int64_t n, const int64_t* seed,
                                                           uint32_t stream, DropRate rate, float scale) {
  const DropKey key = drop_key(seed);
  for (int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x; b * kDropBlock < n;
       b += (int64_t)gridDim.x * kThreads)
    drop_block<T>(x, RES ? res : nullptr, out, b * kDropBlock, n, key, stream, rate, scale);
}

}  // namespace
}  // namespace mla

using namespace mla;

extern "C" int ml_dropout(const void* x, const void* residual, void* out, int64_t n,
                          int64_t threshold, float scale, const int64_t* seed, int64_t stream_id,
                          int dtype, void* stream) {
  ML_CHECK(n >= 0, "dropout: negative size");
  ML_CHECK(threshold >= 0 && threshold <= kDropAll, "dropout: threshold %lld outside 0..65536",
           (long long)threshold);
  ML_CHECK(stream_id >= 0 && stream_id <= 0xFFFFFFFFLL, "dropout: stream id outside 32 bits");
  if (n == 0) return ML_OK;
  ML_CHECK(x && out && seed, "dropout: null pointer");
  hipStream_t st = (hipStream_t)stream;
  const DropRate rate = drop_rate(threshold);
  return dispatch_dtype(dtype, [&](auto tv) -> int {
    using T = decltype(tv);
    const int64_t blocks = (n + kDropBlock * kThreads - 1) / (kDropBlock * kThreads);
    const unsigned grid = (unsigned)(blocks < (int64_t)num_cus() * 64 ? blocks : num_cus() * 64);
    const T* xp = static_cast<const T*>(x);
    const T* rp = static_cast<const T*>(residual);
    T* op = static_cast<T*>(out);
    if (residual)
      dropout_scalar<T, true><<<grid, kThreads, 0, st>>>(xp, rp, op, n, seed, (uint32_t)stream_id,
                                                         rate, scale);
    else
      dropout_scalar<T, false><<<grid, kThreads, 0, st>>>(xp, rp, op, n, seed, (uint32_t)stream_id,
                                                          rate, scale);
    ML_LAUNCH_CHECK();
    return ML_OK;
  });
}
