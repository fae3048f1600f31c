// Token embedding with scaling, and the gradient of its table, for gfx950 (no
// reference counterpart: nn.Embedding is left to torch there).
//
//   y[n]  = scale * W[id_n]
//   dW[v] = scale * sum over the n with id_n = v, in ascending order, of dy[n]
//
// Sums are held in fp32 and rounded once. An id outside the table gives a row of
// NaN and no gradient; rows of dW that no token names, and the row of the padding
// index, are zero.
//
// The gradient of a table of 151936 rows is mostly zeros (622 MB of bf16 at 2048
// columns, of which 8192 tokens name 33 MB at most), so that its fill is the bound
// and everything else is kept beside it:
//   sort   tiles of 8192 tokens, one workgroup each, by (id, position), while the
//          other workgroups of the launch fill dW with zeros;
//   merge  up to 8 sorted runs at a time (none for one tile);
//   sum    chunks of the sorted order: a run of equal ids inside a chunk is summed
//          and stored; what crosses a chunk's end is left as an fp32 partial;
//   join   the partials of each such run, in the chunks' order.
// Chunks and order follow from the ids alone, so that the sums do too.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace mla {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t id_at(const void* ids, int64_t n, bool wide) {
  return wide ? static_cast<const int64_t*>(ids)[n] : static_cast<const int32_t*>(ids)[n];
}

// ----------------------------------------------------------------- forward --
// A row is VEC-element vectors; LPR lanes (a power of two, 1..256) walk a row and
// 256 / LPR rows go side by side, kRows of them in flight per lane.
constexpr int kRows = 4;

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void embedding_rows(const void* ids, bool wide, int64_t N,
                                                           const T* W, int64_t ldw, T* y, int64_t V,
                                                           int64_t H, int lpr, float scale) {
  const int rows = kThreads / lpr;
  const int64_t n0 = (int64_t)blockIdx.x * rows * kRows + threadIdx.x / lpr;
  const int64_t c = ((int64_t)blockIdx.y * lpr + threadIdx.x % lpr) * VEC;
  if (c >= H) return;
  int64_t id[kRows];
  float x[kRows][VEC];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int64_t n = n0 + k * rows;
    id[k] = n < N ? id_at(ids, n, wide) : 0;
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k)  // rows that are not there read row 0
    load_n<T, VEC>(W + (id[k] >= 0 && id[k] < V ? id[k] : 0) * ldw + c, x[k]);
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int64_t n = n0 + k * rows;
    if (n >= N) break;
    const bool ok = id[k] >= 0 && id[k] < V;
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[k][e] = ok ? x[k][e] * scale : NAN;
    store_n_nt<T, VEC>(y + n * H + c, x[k]);
  }
}

// -------------------------------------------------------------------- sort --
// One workgroup sorts a tile by a radix sort of 6-bit digits in LDS: wave w holds
// elements 512 w .. of the current order, 64 at a time; a lane's rank within its
// digit is the number of lanes below it that share the digit (six ballots) plus
// the wave's count of the digit so far, and a scan over (digit, wave) places them.
constexpr int kTile = 8192, kSortThreads = 1024, kWaves = kSortThreads / 64;
constexpr int kItems = kTile / kSortThreads, kDigitBits = 6, kDigits = 1 << kDigitBits;
static_assert(kWaves * kDigits == kSortThreads, "a counter per thread");

__device__ __forceinline__ void fill_zero(char* p, int64_t bytes, int64_t block, int64_t blocks) {
  const int64_t head = std::min<int64_t>(bytes, (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15);
  const int64_t vecs = (bytes - head) / 16, tail = head + vecs * 16;
  u32x4_t* v = reinterpret_cast<u32x4_t*>(p + head);
  const int64_t stride = blocks * kSortThreads;
  for (int64_t i = block * kSortThreads + threadIdx.x; i < vecs; i += stride)
    __builtin_nontemporal_store(u32x4_t{0, 0, 0, 0}, v + i);
  if (block == 0 && threadIdx.x < 16) {
    if (threadIdx.x < head) p[threadIdx.x] = 0;
    if (tail + threadIdx.x < bytes) p[tail + threadIdx.x] = 0;
  }
}

__global__ __launch_bounds__(kSortThreads) void sort_tiles(const void* ids, bool wide, int64_t N,
                                                           int tiles, int64_t V, int64_t skip,
                                                           int passes, uint64_t* sorted, char* dW,
                                                           int64_t bytes) {
  if ((int)blockIdx.x >= tiles) {
    fill_zero(dW, bytes, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  __shared__ uint32_t keys[kTile];
  __shared__ uint16_t from[kTile];
  __shared__ uint32_t count[kDigits * kWaves];  // [digit][wave]
  __shared__ uint32_t wave_sum_[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)blockIdx.x * kTile;
  const int64_t below = (1ULL << lane) - 1;
  uint32_t key[kItems], pos[kItems], rank[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    pos[r] = wave * (kItems * 64) + r * 64 + lane;
    const int64_t n = first + pos[r];
    key[r] = 0xFFFFFFFFu;  // past the end: after every key of the tile
    if (n < N) {
      const int64_t id = id_at(ids, n, wide);
      key[r] = id >= 0 && id < V && id != skip ? (uint32_t)id : (uint32_t)V;  // no gradient: last
    }
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * kDigitBits;
    count[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const uint32_t d = (key[r] >> shift) & (kDigits - 1);
      uint64_t same = ~0ULL;
#pragma unroll
      for (int b = 0; b < kDigitBits; ++b) {
        const bool bit = (d >> b) & 1;
        const uint64_t has = __ballot(bit);
        same &= bit ? has : ~has;
      }
      volatile uint32_t* c = count + d * kWaves + wave;  // this wave's own, in order
      const uint32_t before = *c;
      rank[r] = before + __popcll(same & below);
      if ((same & below) == 0) *c = before + __popcll(same);
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // exclusive scan of the counters in (digit, wave) order, one per thread
    const uint32_t own = count[tid];
    uint32_t sum = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t up = __shfl_up(sum, off, 64);
      if (lane >= off) sum += up;
    }
    if (lane == 63) wave_sum_[wave] = sum;
    __syncthreads();
    uint32_t base = 0;
    for (int w = 0; w < wave; ++w) base += wave_sum_[w];
    count[tid] = base + sum - own;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const uint32_t at = count[((key[r] >> shift) & (kDigits - 1)) * kWaves + wave] + rank[r];
      keys[at] = key[r];
      from[at] = (uint16_t)pos[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const int i = wave * (kItems * 64) + r * 64 + lane;
      key[r] = keys[i];
      pos[r] = from[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int64_t n = first + wave * (kItems * 64) + r * 64 + lane;
    if (n < N) sorted[n] = (uint64_t)key[r] << 32 | (uint64_t)(first + pos[r]);
  }
}

// Up to kWay neighbouring sorted runs of `run` entries into one: an entry's place is
// its place in its own run plus the number of smaller entries in each other one
// (entries are distinct, their low halves being positions).
constexpr int kWay = 8;

__global__ __launch_bounds__(kThreads) void merge_runs(const uint64_t* in, uint64_t* out, int64_t N,
                                                       int64_t run) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= N) return;
  const uint64_t x = in[i];
  const int64_t own = i / run, group = own / kWay * kWay * run;
  int64_t lo[kWay], len[kWay];
#pragma unroll
  for (int k = 0; k < kWay; ++k) {
    const int64_t s = group + k * run;
    lo[k] = s;
    len[k] = s < N && s != own * run ? std::min(run, N - s) : 0;
  }
  int64_t at = i - own * run;
  for (int64_t step = run; step > 0; step >>= 1) {
#pragma unroll
    for (int k = 0; k < kWay; ++k) {  // lo + len: the end of what is not yet decided
      if (len[k] > 0) {
        const int64_t half = len[k] >> 1;
        const bool less = in[lo[k] + half] < x;
        lo[k] = less ? lo[k] + half + 1 : lo[k];
        len[k] = less ? len[k] - half - 1 : half;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kWay; ++k) {
    const int64_t s = group + k * run;
    if (s < N && s != own * run) at += lo[k] - s;
  }
  out[group + at] = x;
}

// --------------------------------------------------------------------- sum --
__device__ __forceinline__ uint32_t key_of(uint64_t e) { return (uint32_t)(e >> 32); }

// Chunk blockIdx.x of the sorted order, columns of blockIdx.y. parts[chunk][0]: what
// the chunk holds of a run that began before it; [1]: of a run that begins in it and
// goes on after it.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void sum_chunks(const uint64_t* sorted, int64_t N, int chunk,
                                                       const T* dy, int64_t ldy, T* dW, int64_t V,
                                                       int64_t H, float* parts, float scale) {
  constexpr int U = 8;  // rows in flight
  const int64_t s = (int64_t)blockIdx.x * chunk, e = std::min<int64_t>(s + chunk, N);
  const int64_t c = ((int64_t)blockIdx.y * kThreads + threadIdx.x) * VEC;
  const bool live = c < H;
  const uint32_t prev = s > 0 ? key_of(sorted[s - 1]) : 0xFFFFFFFFu;
  const uint32_t next = e < N ? key_of(sorted[e]) : 0xFFFFFFFFu;
  uint32_t cur = key_of(sorted[s]);
  bool entered = cur == prev;  // the current run began in an earlier chunk
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  auto part = [&](int slot) {
    if (live) {
      float* p = parts + ((int64_t)blockIdx.x * 2 + slot) * H + c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) p[j] = acc[j];
    }
  };
  auto finish = [&]() {  // the run ends here
    if (entered) {
      part(0);
    } else if (live) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] *= scale;
      store_n<T, VEC>(dW + cur * H + c, acc);
    }
  };
  for (int64_t i = s; i < e; i += U) {
    uint64_t en[U];
    float x[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) en[u] = sorted[i + u < e ? i + u : e - 1];
    if (key_of(en[0]) >= V) break;  // no gradient from here on
#pragma unroll
    for (int u = 0; u < U; ++u)
      load_n<T, VEC>(dy + (int64_t)(uint32_t)en[u] * ldy + (live ? c : 0), x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < e) {
        const uint32_t k = key_of(en[u]);
        if (k != cur) {
          if (cur < V) finish();
          cur = k;
          entered = false;
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += x[u][j];
      }
    }
  }
  if (cur >= V) return;
  if (cur == next)
    part(entered ? 0 : 1);
  else
    finish();
}

// The runs that cross chunks: the workgroup of the chunk in which a run begins adds
// the partials of the chunks it covers. kJoin groups of lanes take every kJoin-th
// chunk and meet in LDS in a fixed order.
constexpr int kJoin = 8, kJoinCols = 32;  // 4 columns a lane: 128 a workgroup

__device__ __forceinline__ void add4(float (&s)[4], const float* p, int64_t c, int64_t H,
                                     bool vec) {
  if (vec) {
    float x[4];
    load_n<float, 4>(p, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < H) s[j] += p[j];
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void join_chunks(const uint64_t* sorted, int64_t N, int chunk,
                                                        int chunks, T* dW, int64_t V, int64_t H,
                                                        const float* parts, float scale) {
  __shared__ float met[kJoin][kJoinCols * 4];
  const int b = blockIdx.x;
  const int64_t s = (int64_t)b * chunk, e = s + chunk;
  if (e >= N) return;
  const uint32_t key = key_of(sorted[e]);
  if (key >= V || key_of(sorted[e - 1]) != key) return;
  if (s > 0 && key_of(sorted[s - 1]) == key) return;  // it began earlier
  int span = 0;  // chunks after this one that it reaches
  for (;;) {
    const int64_t at = (int64_t)(b + 1 + span + threadIdx.x) * chunk;
    const int n = __syncthreads_count(at < N && key_of(sorted[at]) == key);
    span += n;
    if (n < kThreads) break;
  }
  const int g = threadIdx.x / kJoinCols, l = threadIdx.x % kJoinCols;
  const int64_t c = ((int64_t)blockIdx.y * kJoinCols + l) * 4;
  const bool vec = H % 4 == 0;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < H) {
    if (g == 0) add4(sum, parts + ((int64_t)b * 2 + 1) * H + c, c, H, vec);
#pragma unroll 8
    for (int k = g; k < span; k += kJoin)
      add4(sum, parts + (int64_t)(b + 1 + k) * 2 * H + c, c, H, vec);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) met[g][l * 4 + j] = sum[j];
  __syncthreads();
  const int col = threadIdx.x;
  const int64_t oc = (int64_t)blockIdx.y * kJoinCols * 4 + col;
  if (col < kJoinCols * 4 && oc < H) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) t += met[k][col];
    dW[(int64_t)key * H + oc] = from_f32<T>(t * scale);
  }
}

struct Plan {
  int tiles, chunk, chunks, merges;
  size_t entries, parts;  // bytes of one copy of the sorted entries, and of the partials
};

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// Chunks of 16 tokens until they are 1024, then longer ones: enough workgroups to
// fill the GPU and few enough partials to join.
Plan plan_of(int64_t n, int64_t hidden) {
  Plan p{};
  p.tiles = (int)((n + kTile - 1) / kTile);
  for (int64_t run = kTile; run < n; run *= kWay) ++p.merges;
  p.chunk = (int)std::max<int64_t>(16, (n + 1023) / 1024);
  p.chunks = (int)((n + p.chunk - 1) / p.chunk);
  p.entries = align256((size_t)n * 8);
  p.parts = align256((size_t)p.chunks * 2 * hidden * 4);
  return p;
}

size_t bytes_of(const Plan& p) { return p.entries * (p.merges ? 2 : 1) + p.parts; }

}  // namespace
}  // namespace mla

using namespace mla;

static int embedding_sizes(const char* what, int64_t n, int64_t vocab, int64_t hidden, int64_t ld,
                           int id_bytes) {
  ML_CHECK(n >= 0 && n < (1LL << 31), "%s: bad token count %lld", what, (long long)n);
  ML_CHECK(vocab >= 1 && vocab < (1LL << 31) && hidden >= 1 && hidden < (1LL << 22),
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
    constexpr int VEC = vec16<T>();
    const bool vec = hidden % VEC == 0 && ldw % VEC == 0 && aligned16(weight) && aligned16(out);
    const int64_t per_row = vec ? hidden / VEC : hidden;
    int lpr = 1;
    while (lpr < per_row && lpr < kThreads) lpr *= 2;
    const int rows = kThreads / lpr * kRows;
    const dim3 grid((unsigned)((n + rows - 1) / rows), (unsigned)((per_row + lpr - 1) / lpr));
    const T* w = static_cast<const T*>(weight);
    T* o = static_cast<T*>(out);
    hipStream_t st = (hipStream_t)stream;
    if (vec)
      embedding_rows<T, VEC><<<grid, kThreads, 0, st>>>(ids, id_bytes == 8, n, w, ldw, o, vocab,
                                                        hidden, lpr, scale);
    else
      embedding_rows<T, 1><<<grid, kThreads, 0, st>>>(ids, id_bytes == 8, n, w, ldw, o, vocab,
                                                      hidden, lpr, scale);
    ML_LAUNCH_CHECK();
    return ML_OK;
  });
}

extern "C" size_t ml_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t hidden) {
  if (n <= 0 || vocab <= 0 || hidden <= 0 || n >= (1LL << 31) || hidden >= (1LL << 22)) return 0;
  return bytes_of(plan_of(n, hidden));
}

extern "C" int ml_embedding_bwd(const void* ids, int id_bytes, int64_t n, const void* dy,
                                int64_t lddy, void* dweight, int64_t vocab, int64_t hidden,
                                int64_t padding_idx, float scale, void* workspace,
                                size_t workspace_bytes, int dtype, void* stream) {
  int rc = embedding_sizes("embedding backward", n, vocab, hidden, lddy, id_bytes);
  if (rc) return rc;
  ML_CHECK(padding_idx >= -1 && padding_idx < vocab, "embedding backward: bad padding index %lld",
           (long long)padding_idx);
  ML_CHECK(dweight && ((ids && dy) || n == 0), "embedding backward: null pointer");
  const Plan p = plan_of(n, hidden);
  ML_CHECK(n == 0 || (workspace && aligned16(workspace) && workspace_bytes >= bytes_of(p)),
           "embedding backward: workspace too small or misaligned (%zu < %zu)", workspace_bytes,
           bytes_of(p));
  hipStream_t st = (hipStream_t)stream;
  return dispatch_dtype(dtype, [&](auto tv) -> int {
    using T = decltype(tv);
    constexpr int VEC = vec16<T>();
    T* dw = static_cast<T*>(dweight);
    const int64_t bytes = vocab * hidden * (int64_t)sizeof(T);
    const int64_t per_block = (int64_t)kSortThreads * 16 * 4;
    const int64_t fill = std::min<int64_t>((bytes + per_block - 1) / per_block, num_cus() * 8);
    int passes = 0;
    while (passes * kDigitBits < 32 && (vocab >> (passes * kDigitBits)) > 0) ++passes;
    char* ws = static_cast<char*>(workspace);
    uint64_t* a = reinterpret_cast<uint64_t*>(ws);
    uint64_t* b = reinterpret_cast<uint64_t*>(ws + p.entries);
    float* parts = reinterpret_cast<float*>(ws + p.entries * (p.merges ? 2 : 1));
    sort_tiles<<<dim3((unsigned)(p.tiles + fill)), kSortThreads, 0, st>>>(
        ids, id_bytes == 8, n, p.tiles, vocab, padding_idx, passes, a,
        static_cast<char*>(dweight), bytes);
    ML_LAUNCH_CHECK();
    if (n == 0) return ML_OK;
    int64_t run = kTile;
    for (int k = 0; k < p.merges; ++k, run *= kWay) {
      merge_runs<<<dim3((unsigned)((n + kThreads - 1) / kThreads)), kThreads, 0, st>>>(a, b, n,
                                                                                      run);
      ML_LAUNCH_CHECK();
      std::swap(a, b);
    }
    const T* g = static_cast<const T*>(dy);
    const bool vec = hidden % VEC == 0 && lddy % VEC == 0 && aligned16(dy) && aligned16(dweight);
    const int64_t per = (int64_t)kThreads * (vec ? VEC : 1);
    const dim3 grid((unsigned)p.chunks, (unsigned)((hidden + per - 1) / per));
    if (vec)
      sum_chunks<T, VEC><<<grid, kThreads, 0, st>>>(a, n, p.chunk, g, lddy, dw, vocab, hidden,
                                                    parts, scale);
    else
      sum_chunks<T, 1><<<grid, kThreads, 0, st>>>(a, n, p.chunk, g, lddy, dw, vocab, hidden, parts,
                                                  scale);
    ML_LAUNCH_CHECK();
    if (p.chunks > 1) {
      const dim3 jg((unsigned)p.chunks,
                    (unsigned)((hidden + kJoinCols * 4 - 1) / (kJoinCols * 4)));
      join_chunks<T><<<jg, kThreads, 0, st>>>(a, n, p.chunk, p.chunks, dw, vocab, hidden, parts,
                                              scale);
      ML_LAUNCH_CHECK();
    }
    return ML_OK;
  });
}
