// Token embedding with scaling, and the gradient of its table, for gfx950 (no
// reference counterpart: nn.Embedding is left to torch there).
//
//   y[n]  = scale * W[id_n]
//   dW[v] = scale * sum over the n with id_n = v, in ascending order, of dy[n]
//
// Sums are held in fp32 and rounded once. An id outside the table gives a row of
// NaN and no gradient; rows of dW that no token names, and the row of the padding
// index, are zero.
#include <math.h>

#include "common.h"

namespace mla {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t id_at(const void* ids, int64_t n, bool wide) {
  return wide ? static_cast<const int64_t*>(ids)[n] : static_cast<const int32_t*>(ids)[n];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void embedding_rows(const void* ids, bool wide, const T* W,
                                                           int64_t ldw, T* y, int64_t V, int64_t H,
                                                           float scale) {
  const int64_t n = blockIdx.x, id = id_at(ids, n, wide);
  const bool ok = id >= 0 && id < V;
  for (int64_t c = threadIdx.x; c < H; c += kThreads)
    y[n * H + c] = from_f32<T>(ok ? to_f32(W[id * ldw + c]) * scale : NAN);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void zero_rows(T* dW, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kThreads)
    dW[i] = from_f32<T>(0.f);
}

// The first token of each id sums the rows of all tokens that name it.
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_rows(const void* ids, bool wide, int64_t N,
                                                     const T* dy, int64_t ldy, T* dW, int64_t V,
                                                     int64_t H, int64_t skip, float scale) {
  const int64_t n = blockIdx.x, id = id_at(ids, n, wide);
  if (id < 0 || id >= V || id == skip) return;
  for (int64_t m = 0; m < n; ++m)
    if (id_at(ids, m, wide) == id) return;
  for (int64_t c = threadIdx.x; c < H; c += kThreads) {
    float s = 0.f;
    for (int64_t m = n; m < N; ++m)
      if (id_at(ids, m, wide) == id) s += to_f32(dy[m * ldy + c]);
    dW[id * H + c] = from_f32<T>(s * scale);
  }
}

}  // namespace
}  // namespace mla

using namespace mla;

static int embedding_sizes(const char* what, int64_t n, int64_t vocab, int64_t hidden, int64_t ld,
                           int id_bytes) {
  ML_CHECK(n >= 0 && n < (1LL << 31), "%s: bad token count %lld", what, (long long)n);
  ML_CHECK(vocab >= 1 && vocab < (1LL << 31) && hidden >= 1 && hidden < (1LL << 31),
           "%s: bad table [%lld, %lld]", what, (long long)vocab, (long long)hidden);
  ML_CHECK(ld >= hidden, "%s: row stride %lld below the width %lld", what, (long long)ld,
           (long long)hidden);
  ML_CHECK(id_bytes == 4 || id_bytes == 8, "%s: ids of 4 or 8 bytes (got %d)", what, id_bytes);
  return ML_OK;
}

extern "C" int ml_embedding_fwd(const void* ids, int id_bytes, int64_t n, const void* weight,
                                int64_t ldw, void* out, int64_t vocab, int64_t hidden, float scale,
                                int dtype, void* stream) {
  int rc = embedding_sizes("embedding", n, vocab, hidden, ldw, id_bytes);
  if (rc) return rc;
  if (n == 0) return ML_OK;
  ML_CHECK(ids && weight && out, "embedding: null pointer");
  return dispatch_dtype(dtype, [&](auto tv) -> int {
    using T = decltype(tv);
    embedding_rows<T><<<dim3((unsigned)n), kThreads, 0, (hipStream_t)stream>>>(
        ids, id_bytes == 8, static_cast<const T*>(weight), ldw, static_cast<T*>(out), vocab, hidden,
        scale);
    ML_LAUNCH_CHECK();
    return ML_OK;
  });
}

extern "C" size_t ml_embedding_bwd_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int ml_embedding_bwd(const void* ids, int id_bytes, int64_t n, const void* dy,
                                int64_t lddy, void* dweight, int64_t vocab, int64_t hidden,
                                int64_t padding_idx, float scale, void* workspace,
                                size_t workspace_bytes, int dtype, void* stream) {
  int rc = embedding_sizes("embedding backward", n, vocab, hidden, lddy, id_bytes);
  if (rc) return rc;
  ML_CHECK(padding_idx >= -1 && padding_idx < vocab, "embedding backward: bad padding index %lld",
           (long long)padding_idx);
  ML_CHECK(dweight && ((ids && dy) || n == 0), "embedding backward: null pointer");
  hipStream_t st = (hipStream_t)stream;
  return dispatch_dtype(dtype, [&](auto tv) -> int {
    using T = decltype(tv);
    zero_rows<T><<<dim3(num_cus() * 16), kThreads, 0, st>>>(static_cast<T*>(dweight),
                                                            vocab * hidden);
    ML_LAUNCH_CHECK();
    if (n == 0) return ML_OK;
    sum_rows<T><<<dim3((unsigned)n), kThreads, 0, st>>>(ids, id_bytes == 8, n,
                                                        static_cast<const T*>(dy), lddy,
                                                        static_cast<T*>(dweight), vocab, hidden,
                                                        padding_idx, scale);
    ML_LAUNCH_CHECK();
    return ML_OK;
  });
}
