// Dropout, with the add of a residual that follows it, for gfx950 (no reference
// counterpart: nn.Dropout and the adds around it are left to torch there).
//
//   out_i = kept_i ? scale * x_i : 0      (+ residual_i)
//
// with the masks of dropout.h; the gradient is the same kernel over dy, so that
// neither direction stores or reads a mask. A dropped element gives 0 whatever x
// holds there, infinities and NaN included.
#include <algorithm>

#include "dropout.h"

namespace mla {
namespace {

constexpr int kThreads = 256;
// A launch holds fewer than 2^32 threads: longer tensors take several. (A loop in the
// kernel costs shorter ones 0.8 of 31 us at [8192, 6144] bf16.)
constexpr int64_t kMaxBlocks = 1 << 23;

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

// Tensors that are not all 16-byte aligned.
template <typename T, bool RES>
__global__ __launch_bounds__(kThreads) void dropout_scalar(const T* x, const T* res, T* out,
                                                           int64_t n, const int64_t* seed,
                                                           uint32_t stream, DropRate rate,
                                                           float scale) {
  const DropKey key = seed ? drop_key(seed) : DropKey{};  // (none where nothing is dropped)
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kDropBlock; i < n;
       i += (int64_t)gridDim.x * kThreads * kDropBlock)
    drop_block<T>(x, RES ? res : nullptr, out, i, n, key, stream, rate, scale);
}

// VEC elements of a block (8 of 16 bits, or 4 of 32) under their words of the mask.
template <typename T, int VEC>
__device__ __forceinline__ void drop_vec(const Pack<T, VEC>& x, const Pack<T, VEC>& r, bool res,
                                         const uint32_t* m, float scale, T* out) {
  float y[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    // all ones or zeros over the element's half of the word
    const int keep = (e & 1) ? (int)m[e >> 1] >> 16 : (int)(m[e >> 1] << 16) >> 16;
    const float v = to_f32(x.v[e]);
    y[e] = __builtin_bit_cast(float, __builtin_bit_cast(int, v) & keep) * scale;
    if (res) y[e] += to_f32(r.v[e]);
  }
  store_n_nt<T, VEC>(out, y);
}

// 16 bytes a lane, so that a wave's accesses are whole rows of 1 KB: a block of 8
// elements of 16 bits, or half a block of fp32, whose mask both lanes form. The last
// block may hold fewer. [8192, 6144] bf16 33 us (6.1 TB/s; with the residual 48, 6.3),
// as fast with two and four blocks in flight per lane.
template <typename T, bool RES>
__global__ __launch_bounds__(kThreads) void dropout_vec(const T* x, const T* res, T* out,
                                                        int64_t first, int64_t n,
                                                        const int64_t* seed, uint32_t stream,
                                                        DropRate rate, float scale) {
  constexpr int VEC = vec16<T>();
  const int64_t i = first + ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VEC;
  const int64_t block = i / kDropBlock;
  const DropKey key = seed ? drop_key(seed) : DropKey{};  // (none where nothing is dropped)
  if ((block + 1) * kDropBlock <= n) {
    const Pack<T, VEC> v = load_pack_nt<T, VEC>(x + i);
    Pack<T, VEC> r{};
    if constexpr (RES) r = load_pack_nt<T, VEC>(res + i);
    const u32x4_t m = drop_mask((uint64_t)block, stream, key, rate);
    const bool second = VEC == 4 && (threadIdx.x & 1);
    const uint32_t w[4] = {second ? m.z : m.x, second ? m.w : m.y, m.z, m.w};
    drop_vec<T, VEC>(v, r, RES, w, scale, out + i);
  } else if (i % kDropBlock == 0 && i < n) {
    drop_block<T>(x, RES ? res : nullptr, out, i, n, key, stream, rate, scale);
  }
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
  ML_CHECK(x && out && (seed || threshold == 0), "dropout: null pointer");
  ML_CHECK(n < (1LL << 40), "dropout: too many elements (%lld)", (long long)n);
  hipStream_t st = (hipStream_t)stream;
  const DropRate rate = drop_rate(threshold);
  return dispatch_dtype(dtype, [&](auto tv) -> int {
    using T = decltype(tv);
    const T* xp = static_cast<const T*>(x);
    const T* rp = static_cast<const T*>(residual);
    T* op = static_cast<T*>(out);
    const uint32_t sid = (uint32_t)stream_id;
    if (aligned16(x) && aligned16(residual) && aligned16(out)) {
      const int64_t per = (int64_t)kThreads * vec16<T>();
      for (int64_t first = 0; first < n; first += kMaxBlocks * per) {
        const dim3 grid((unsigned)std::min((n - first + per - 1) / per, kMaxBlocks));
        if (residual)
          dropout_vec<T, true><<<grid, kThreads, 0, st>>>(xp, rp, op, first, n, seed, sid, rate,
                                                          scale);
        else
          dropout_vec<T, false><<<grid, kThreads, 0, st>>>(xp, rp, op, first, n, seed, sid, rate,
                                                           scale);
      }
    } else {
      const int64_t per = (int64_t)kThreads * kDropBlock;
      const dim3 grid((unsigned)std::min<int64_t>((n + per - 1) / per, (int64_t)num_cus() * 64));
      if (residual)
        dropout_scalar<T, true><<<grid, kThreads, 0, st>>>(xp, rp, op, n, seed, sid, rate, scale);
      else
        dropout_scalar<T, false><<<grid, kThreads, 0, st>>>(xp, rp, op, n, seed, sid, rate, scale);
    }
    ML_LAUNCH_CHECK();
    return ML_OK;
  });
}
