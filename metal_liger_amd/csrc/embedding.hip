// Token embedding with scaling, and the gradient of its table, for gfx950 (no
// reference counterpart: nn.Embedding is left to torch there).
//
//   y[n]  = scale * W[id_n]
//   dW[v] = scale * sum over the n with id_n = v of dy[n]
//
// Sums are held in fp32 and rounded once; their order (below) follows from the ids and
// their number alone. An id outside the table gives a row of
// NaN and no gradient; rows of dW that no token names, and the row of the padding
// index, are zero.
//
// The gradient of a table of 151936 rows is mostly zeros (622 MB of bf16 at 2048
// columns, of which 8192 tokens name 33 MB at most), so that its fill is the bound
// and everything else is kept beside it:
//   sort   tiles of up to 16384 tokens, one workgroup each, by (id, position), while the
//          other workgroups of the launch fill dW with zeros;
//   merge  up to 8 sorted runs at a time (none for one tile);
//   sum    chunks of the sorted order: a run of equal ids inside a chunk is summed
//          and stored; what crosses a chunk's end is left as an fp32 partial;
//   join   the partials of each such run.
// A chunk adds its tokens in ascending order; a run of up to 16 chunks more adds their
// partials two by two, a longer one every 16th chunk to one of 16 sums, then those.
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
constexpr int64_t kMaxBlocks = 1 << 23;  // a launch holds fewer than 2^32 threads along x

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
// One workgroup sorts a tile by a radix sort of 6-bit digits between two buffers of
// LDS, an entry being one word: the id above the position in the tile. Wave w holds
// the w-th part of the current order, 64 entries at a time. A lane's entry goes to
// the number of entries with smaller digits, plus those of the same digit in earlier
// waves (a scan over (digit, wave) of what each wave counted), in the wave's earlier
// rounds and in lower lanes; lanes that share a digit find each other by six ballots.
// (Entries, ranks and predicates held in registers spilled 452 bytes a lane and took
// 95 us for 8192 ids.)
constexpr int kSortThreads = 1024, kWaves = kSortThreads / 64;
constexpr int kDigitBits = 6, kDigits = 1 << kDigitBits;
static_assert(kWaves * kDigits == kSortThreads, "a counter per thread");

// Ids below 2^18 go in 32 bits beside 14 bits of position, others in 64 beside 13.
template <typename W>
constexpr int pos_bits() { return sizeof(W) == 4 ? 14 : 13; }
template <typename W>
constexpr int tile_of() { return 1 << pos_bits<W>(); }
constexpr int64_t kNarrowVocab = (1 << 18) - 1;  // the key of "no gradient" is the vocabulary

// The lanes (of those that are `in`) whose digit is this lane's.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool in) {
  uint64_t same = __ballot(in);
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const bool bit = (d >> b) & 1;
    const uint64_t has = __ballot(bit);
    same &= bit ? has : ~has;
  }
  return same;
}

// Zeros, by one wave in each of `blocks` workgroups. One wave per CU keeps what is
// being written within 256 KB: 622 MB take 100 us beside the sort, and 85 in a launch
// of 64-thread workgroups of their own, which would wait for the sort instead; with
// 512 to 2048 threads per CU, 105 to 140.
__device__ __forceinline__ void fill_zero(char* p, int64_t bytes, int64_t block, int64_t blocks) {
  if (threadIdx.x >= 64) return;
  const int64_t head = std::min<int64_t>(bytes, (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15);
  const int64_t vecs = (bytes - head) / 16, tail = head + vecs * 16;
  u32x4_t* v = reinterpret_cast<u32x4_t*>(p + head);
  for (int64_t i = block * 64 + threadIdx.x; i < vecs; i += blocks * 64)
    __builtin_nontemporal_store(u32x4_t{0, 0, 0, 0}, v + i);
  if (block == 0 && threadIdx.x < 16) {
    if (threadIdx.x < head) p[threadIdx.x] = 0;
    if (tail + threadIdx.x < bytes) p[tail + threadIdx.x] = 0;
  }
}

template <typename W>
__global__ __launch_bounds__(kSortThreads) void sort_tiles(const void* ids, bool wide, int64_t N,
                                                           int tiles, int64_t V, int64_t skip,
                                                           int passes, uint64_t* sorted, char* dW,
                                                           int64_t bytes) {
  if ((int)blockIdx.x >= tiles) {
    fill_zero(dW, bytes, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  constexpr int kTile = tile_of<W>(), kPos = pos_bits<W>();
  __shared__ W buf[2][kTile];
  __shared__ uint32_t count[kDigits * kWaves];  // [digit][wave]
  __shared__ uint32_t totals[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t first = (int64_t)blockIdx.x * kTile;
  const int size = (int)std::min<int64_t>(kTile, N - first);
  const int part = (size + kSortThreads - 1) / kSortThreads * 64;  // entries per wave
  const int begin = wave * part, end = std::min(begin + part, size);
  const uint64_t below = (1ULL << lane) - 1;
  for (int i = tid; i < size; i += kSortThreads) {
    const int64_t id = id_at(ids, first + i, wide);
    const bool ok = id >= 0 && id < V && id != skip;
    buf[0][i] = (W)(ok ? id : V) << kPos | (W)i;  // no gradient: after all others
  }
  W *src = buf[0], *dst = buf[1];
  for (int p = 0; p < passes; ++p) {
    const int shift = kPos + p * kDigitBits;
    count[tid] = 0;
    __syncthreads();
    for (int i = begin; i < end; i += 64) {
      const bool in = i + lane < end;
      const uint32_t d = in ? (uint32_t)(src[i + lane] >> shift) & (kDigits - 1) : 0;
      const uint64_t same = same_digit(d, in);
      volatile uint32_t* c = count + d * kWaves + wave;  // this wave's own, in order
      if (in && (same & below) == 0) *c = *c + __popcll(same);
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
    if (lane == 63) totals[wave] = sum;
    __syncthreads();
    sum -= own;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += w < wave ? totals[w] : 0;
    count[tid] = sum;
    __syncthreads();
    for (int i = begin; i < end; i += 64) {
      const bool in = i + lane < end;
      const W e = in ? src[i + lane] : 0;
      const uint32_t d = (uint32_t)(e >> shift) & (kDigits - 1);
      const uint64_t same = same_digit(d, in);
      volatile uint32_t* c = count + d * kWaves + wave;
      const uint32_t before = *c;
      if (in) {
        if ((same & below) == 0) *c = before + __popcll(same);
        dst[before + __popcll(same & below)] = e;
      }
    }
    __syncthreads();
    W* const done = dst;
    dst = src;
    src = done;
  }
  for (int i = tid; i < size; i += kSortThreads) {
    const W e = src[i];
    sorted[first + i] = (uint64_t)(e >> kPos) << 32 | (uint64_t)(first + (e & (kTile - 1)));
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
__global__ __launch_bounds__(kThreads) void sum_chunks(const uint64_t* __restrict__ sorted,
                                                       int64_t N, int chunk,
                                                       const T* __restrict__ dy, int64_t ldy,
                                                       T* __restrict__ dW, int64_t V, int64_t H,
                                                       float* __restrict__ parts, float scale) {
  constexpr int U = 16;  // rows in flight: the shortest chunk
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
    Pack<T, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) en[u] = sorted[i + u < e ? i + u : e - 1];
    if (key_of(en[0]) >= V) break;  // no gradient from here on
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = *reinterpret_cast<const Pack<T, VEC>*>(dy + (int64_t)(uint32_t)en[u] * ldy +
                                                    (live ? c : 0));
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
        for (int j = 0; j < VEC; ++j) acc[j] += to_f32(x[u].v[j]);
      }
    }
  }
  if (cur >= V) return;
  if (cur == next)
    part(entered ? 0 : 1);
  else
    finish();
}

// The runs that cross chunks: their partials added in a fixed order. Every
// workgroup lists the chunks in which such a run begins (a thread a chunk) and takes
// its share of the (run, column slice) items: a wave sums a run of a few chunks, 256
// columns at a time; a long one (an image's or a padding token) takes the workgroup, 64
// columns at a time, whose waves add every 16th chunk and meet in LDS in a fixed order:
// 9 us after 8192 tokens of text, 10 where one run covers 700 chunks of 16384 tokens.
// (A workgroup for every chunk and slice took 39 us where a run covers 700 chunks of
// 16384 tokens and 7.5 us where it had next to nothing to do.)
constexpr int kJoinThreads = 1024, kJoinWaves = kJoinThreads / 64, kShortCols = 4;
constexpr int kMaxChunks = kJoinThreads, kLongRun = 16;

// Adds the partials k, k + step .. up to `last`, U loads in flight (those past the
// last read it again and add nothing: a loop over what is left would wait for each).
template <int U>
__device__ __forceinline__ void add_parts(float& sum, const float* __restrict__ p, int k, int step,
                                          int last, int64_t H) {
  for (; k <= last; k += U * step) {
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + u * step;
      x[u] = p[(int64_t)(at < last ? at : last) * 2 * H];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) sum += k + u * step <= last ? x[u] : 0.f;
  }
}

template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_chunks(const uint64_t* __restrict__ sorted,
                                                            int64_t N, int chunk, int chunks,
                                                            T* __restrict__ dW, int64_t V,
                                                            int64_t H,
                                                            const float* __restrict__ parts,
                                                            float scale) {
  __shared__ uint32_t first[kMaxChunks + 1];  // a chunk's first key
  __shared__ uint32_t list[2][kMaxChunks];    // chunks in which short / long runs begin
  __shared__ uint16_t spans[kMaxChunks];      // how many chunks more the run reaches
  __shared__ int counts[2][kJoinWaves];
  __shared__ float met[kJoinWaves][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = (int64_t)tid * chunk, e = s + chunk;
  uint32_t before = 0xFFFFFFFFu, last = 0xFFFFFFFFu;
  first[tid] = 0xFFFFFFFFu;
  if (tid < chunks) {
    first[tid] = key_of(sorted[s]);
    if (tid > 0) before = key_of(sorted[s - 1]);
    if (e < N) last = key_of(sorted[e - 1]);
  }
  if (tid == 0) first[kMaxChunks] = 0xFFFFFFFFu;
  __syncthreads();
  // a run goes on after this chunk, and did not come into it
  const bool owner =
      last < V && first[tid + 1] == last && !(first[tid] == last && before == last);
  int span = 0;
  if (owner) {
    int lo = tid + 1, hi = chunks;  // the first chunk after it that begins with another key
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] == last)
        lo = mid + 1;
      else
        hi = mid;
    }
    span = lo - tid - 1;
    spans[tid] = (uint16_t)span;
  }
  // every workgroup makes the same lists, in the chunks' order
  const uint64_t has[2] = {__ballot(owner && span <= kLongRun), __ballot(owner && span > kLongRun)};
  if (lane < 2) counts[lane][wave] = __popcll(lane == 0 ? has[0] : has[1]);
  __syncthreads();
  int found[2] = {0, 0}, at[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int w = 0; w < kJoinWaves; ++w) {
      if (w == wave) at[k] = found[k];
      found[k] += counts[k][w];
    }
  if (owner) {
    const int k = span > kLongRun;
    const uint64_t mine = k ? has[1] : has[0];
    list[k][(k ? at[1] : at[0]) + __popcll(mine & ((1ULL << lane) - 1))] = tid;
  }
  __syncthreads();
  const int wide = (int)((H + 64 * kShortCols - 1) / (64 * kShortCols));
  const int shorts = found[0] * wide;
  for (int i = blockIdx.x * kJoinWaves + wave; i < shorts; i += gridDim.x * kJoinWaves) {
    const int b = list[0][i / wide], span = spans[b];
    const float* p = parts + (int64_t)b * 2 * H;
    int64_t c[kShortCols];
    float sum[kShortCols];
#pragma unroll
    for (int j = 0; j < kShortCols; ++j) {
      c[j] = (int64_t)(i % wide * kShortCols + j) * 64 + lane;
      sum[j] = p[H + (c[j] < H ? c[j] : 0)];
    }
    for (int k = 1; k <= span; k += 2) {  // two chunks of every column in flight
      float x[2][kShortCols];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < kShortCols; ++j)
          x[u][j] = p[(int64_t)(k + u < span ? k + u : span) * 2 * H + (c[j] < H ? c[j] : 0)];
#pragma unroll
      for (int j = 0; j < kShortCols; ++j) sum[j] += x[0][j] + (k < span ? x[1][j] : 0.f);
    }
#pragma unroll
    for (int j = 0; j < kShortCols; ++j)
      if (c[j] < H) dW[(int64_t)first[b + 1] * H + c[j]] = from_f32<T>(sum[j] * scale);
  }
  const int narrow = (int)((H + 63) / 64), longs = found[1] * narrow;
  for (int i = blockIdx.x; i < longs; i += gridDim.x) {
    const int b = list[1][i / narrow], span = spans[b];
    const int64_t c = (int64_t)(i % narrow) * 64 + lane;
    float sum = 0.f;
    if (c < H) {
      if (wave == 0) sum = parts[((int64_t)b * 2 + 1) * H + c];
      add_parts<16>(sum, parts + (int64_t)b * 2 * H + c, 1 + wave, kJoinWaves, span, H);
    }
    __syncthreads();  // the previous item's sums have been read
    met[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < H) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) total += met[w][lane];
      dW[(int64_t)first[b + 1] * H + c] = from_f32<T>(total * scale);
    }
  }
}

struct Plan {
  int tile, tiles, chunk, chunks, merges;
  size_t entries, parts;  // bytes of one copy of the sorted entries, and of the partials
};

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// Chunks of 16 tokens until they are 1024, then longer ones: enough workgroups to
// fill the GPU, and a thread for each in the join.
Plan plan_of(int64_t n, int64_t vocab, int64_t hidden) {
  Plan p{};
  p.tile = vocab <= kNarrowVocab ? tile_of<uint32_t>() : tile_of<uint64_t>();
  p.tiles = (int)((n + p.tile - 1) / p.tile);
  for (int64_t run = p.tile; run < n; run *= kWay) ++p.merges;
  p.chunk = (int)std::max<int64_t>(16, (n + kMaxChunks - 1) / kMaxChunks);
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
    const T* w = static_cast<const T*>(weight);
    hipStream_t st = (hipStream_t)stream;
    for (int64_t first = 0; first < n; first += kMaxBlocks * rows) {
      const int64_t count = std::min(n - first, kMaxBlocks * rows);
      const dim3 grid((unsigned)((count + rows - 1) / rows), (unsigned)((per_row + lpr - 1) / lpr));
      const char* p = static_cast<const char*>(ids) + first * id_bytes;
      T* o = static_cast<T*>(out) + first * hidden;
      if (vec)
        embedding_rows<T, VEC><<<grid, kThreads, 0, st>>>(p, id_bytes == 8, count, w, ldw, o, vocab,
                                                          hidden, lpr, scale);
      else
        embedding_rows<T, 1><<<grid, kThreads, 0, st>>>(p, id_bytes == 8, count, w, ldw, o, vocab,
                                                        hidden, lpr, scale);
    }
    ML_LAUNCH_CHECK();
    return ML_OK;
  });
}

extern "C" size_t ml_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t hidden) {
  if (n <= 0 || vocab <= 0 || hidden <= 0 || n >= (1LL << 31) || hidden >= (1LL << 22)) return 0;
  return bytes_of(plan_of(n, vocab, hidden));
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
  const Plan p = plan_of(n, vocab, hidden);
  ML_CHECK(n == 0 || (workspace && aligned16(workspace) && workspace_bytes >= bytes_of(p)),
           "embedding backward: workspace too small or misaligned (%zu < %zu)", workspace_bytes,
           bytes_of(p));
  hipStream_t st = (hipStream_t)stream;
  return dispatch_dtype(dtype, [&](auto tv) -> int {
    using T = decltype(tv);
    constexpr int VEC = vec16<T>();
    T* dw = static_cast<T*>(dweight);
    const int64_t bytes = vocab * hidden * (int64_t)sizeof(T);
    // one workgroup of this launch fits a CU (its LDS): those that fill leave room for
    // those that sort, so that none starts late
    const int64_t fill = std::min<int64_t>((bytes + 1023) / 1024,
                                           std::max(num_cus() - p.tiles, num_cus() / 4));
    int passes = 0;
    while (passes * kDigitBits < 32 && (vocab >> (passes * kDigitBits)) > 0) ++passes;
    char* ws = static_cast<char*>(workspace);
    uint64_t* a = reinterpret_cast<uint64_t*>(ws);
    uint64_t* b = reinterpret_cast<uint64_t*>(ws + p.entries);
    float* parts = reinterpret_cast<float*>(ws + p.entries * (p.merges ? 2 : 1));
    const dim3 sg((unsigned)(p.tiles + fill));
    if (vocab <= kNarrowVocab)
      sort_tiles<uint32_t><<<sg, kSortThreads, 0, st>>>(ids, id_bytes == 8, n, p.tiles, vocab,
                                                        padding_idx, passes, a,
                                                        static_cast<char*>(dweight), bytes);
    else
      sort_tiles<uint64_t><<<sg, kSortThreads, 0, st>>>(ids, id_bytes == 8, n, p.tiles, vocab,
                                                        padding_idx, passes, a,
                                                        static_cast<char*>(dweight), bytes);
    ML_LAUNCH_CHECK();
    if (n == 0) return ML_OK;
    int64_t run = p.tile;
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
      join_chunks<T><<<dim3((unsigned)num_cus()), kJoinThreads, 0, st>>>(
          a, n, p.chunk, p.chunks, dw, vocab, hidden, parts, scale);
      ML_LAUNCH_CHECK();
    }
    return ML_OK;
  });
}
