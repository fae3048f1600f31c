// Products with fp32 sums of fp32 (or fp16, upcast in registers) operands on the fp32
// matrix cores, for the feed-forward operators' fp32 and fp16 forms:
//
//   out[s][M][N] = the s-th part over K of sum_seg op(A) op(B)       (fp32, dense)
//
// Layouts as in gemm_core.h: K-major element (r, k) at p[r * ld + k], MN-major at p[k *
// ld + r]; up to two K segments.
//
// Bound by the matrix cores (157 TFLOP/s; v_mfma_f32_32x32x2_f32 takes 64 cycles), so
// all that matters is that they never wait and that no CU is left without work:
//   * Tiles of 128 x 128 (4 waves of 64 x 64, 2 x 2 MFMA tiles) or 64 x 64; k-tiles of
//     32 go global to LDS by buffer_load ... lds, two stages, so that a k-tile's loads
//     have a whole k-tile's products (4096 cycles) to land, and two workgroups or more
//     share a CU. Which k an MFMA's operand slot holds does not matter as long as both
//     operands agree: lane group g = lane / 32 takes k = 8 s + 4 g .. + 3 of a step s,
//     one 16-byte read of a K-major row (8 bytes of fp16) for four MFMAs.
//   * K is split over workgroups as an estimate of the rounds finds best; the step that
//     reads the sums joins the parts, in order.
// LDS: K-major tile [rows][32 k], 16-byte chunk c of row r at c ^ (r & 7) (fp16: 64-byte
// rows, c ^ (r / 2 & 3)); MN-major tile [32 k][rows]. Rows past the operand's end and
// k-rows past K read zeros by the buffer's range, K-major chunks past K by an offset past
// every range: sizes and strides are multiples of 8, so that no chunk lies across an end.
// Measured (fp32, forward; a plain library product of the same): [1024, 4352] x 4352 378
// us (318; with an any-size kernel's register tiles 448), [2048, 2048] x 2048 147 (121),
// [8192, 2048] x 2048 527, 130 TFLOP/s (468).
#pragma once

#include "ffn_rows.h"
#include "gemm_core.h"

namespace mla {
namespace ffn {

enum : int { kRowsK = 0, kRowsMN = 1 };  // K-major, MN-major

struct F32Segment {
  const void *a, *b;
  int64_t lda, ldb;
  int K;
};

struct F32Problem {
  F32Segment seg[2];
  int nseg, M, N;
  int tiles_m, tiles_n, splits, kps;  // kps: k-tiles a split
  float* out;                         // [splits][M][N]
};

constexpr int kF32K = 32;  // k of a k-tile
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_a __attribute__((ext_vector_type(4)));

// One operand of a ROWS x 32 tile.
template <typename E, int L, int ROWS>
struct F32Operand {
  static constexpr int kBytes = ROWS * kF32K * (int)sizeof(E);
  static constexpr int kLoads = kBytes / 1024 / 4;             // 1-KB loads a wave
  static constexpr int kRowBytes = L == kRowsK ? kF32K * (int)sizeof(E) : ROWS * (int)sizeof(E);
  static constexpr int kRowsLoad = 1024 / kRowBytes;           // rows (k-rows) a load
  static constexpr int kLanesRow = kRowBytes / 16;
  static_assert(kLoads * 4 * 1024 == kBytes, "whole loads");

  uint64_t base;   // uniform: at the tile's first row and the k-tile's first k
  int64_t range;   // uniform: bytes from base to the end of the tile's valid data
  int64_t step;    // uniform: bytes to the next k-tile
  uint32_t off;    // per lane, of load 0
  uint32_t next;   // uniform: bytes from one load of the wave to its next
  int kb;          // per lane, K-major: k of its chunk within a k-tile

  static __device__ __forceinline__ int swz(int r) {
    if constexpr (L == kRowsMN) return 0;
    return sizeof(E) == 4 ? r & 7 : (r >> 1) & 3;
  }

  __device__ __forceinline__ void setup(const void* p, int64_t ld, int row0, int rows, int k0, int K,
                                        int wave, int lane) {
    const int r = kRowsLoad * wave + lane / kLanesRow, c = lane % kLanesRow;
    const char* q = static_cast<const char*>(p);
    constexpr int64_t S = sizeof(E);
    if constexpr (L == kRowsK) {
      base = gemm::uniform_u64(reinterpret_cast<uint64_t>(q + ((int64_t)row0 * ld + k0) * S));
      range = (int64_t)gemm::uniform_u64((uint64_t)(((int64_t)(rows - row0 - 1) * ld + (K - k0)) * S));
      step = kF32K * S;
      // a load of the wave is 4 kRowsLoad rows further on: the swizzle is the same
      off = (uint32_t)(((int64_t)r * ld) * S + 16 * (c ^ swz(r)));
      kb = (c ^ swz(r)) * (16 / (int)S);
      next = __builtin_amdgcn_readfirstlane((uint32_t)(4 * kRowsLoad * ld * S));
    } else {
      base = gemm::uniform_u64(reinterpret_cast<uint64_t>(q + ((int64_t)k0 * ld + row0) * S));
      range = (int64_t)gemm::uniform_u64((uint64_t)(((int64_t)(K - k0 - 1) * ld + (rows - row0)) * S));
      step = (int64_t)gemm::uniform_u64((uint64_t)(kF32K * ld * S));
      off = (uint32_t)((int64_t)r * ld * S + 16 * c);
      kb = 0;
      next = __builtin_amdgcn_readfirstlane((uint32_t)(4 * kRowsLoad * ld * S));
    }
  }

  // This wave's loads of the k-tile at base; live: there is one; left: K from it on.
  __device__ __forceinline__ void load(char* lds, int wave, bool live, int left) const {
    gemm::rsrc_t rs;
    const int64_t n = !live || range < 0 ? 0 : range < gemm::r4::kRangeMax ? range : gemm::r4::kRangeMax;
    rs[0] = (uint32_t)base;
    rs[1] = (uint32_t)(base >> 32) & 0xFFFFu;
    rs[2] = (uint32_t)__builtin_amdgcn_readfirstlane((int)n);
    rs[3] = (uint32_t)gemm::r4::kRsrcFlags;
    const uint32_t from = L == kRowsMN || kb < left ? off : gemm::r4::kOob;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      gemm::buf_load_lds(rs, from + (uint32_t)i * next, lds + (wave + 4 * i) * 1024);
  }

  // k = 8 s + 4 g .. + 3 of row wbase + 32 i + lane % 32 (s: step of the k-tile)
  static __device__ __forceinline__ void fragment(const char* lds, int row, int g, int s,
                                                  float (&f)[4]) {
    if constexpr (L == kRowsK) {
      const char* p = lds + row * kRowBytes;
      if constexpr (sizeof(E) == 4) {
        const f32x4_a v = *reinterpret_cast<const f32x4_a*>(p + (((2 * s + g) ^ swz(row)) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = v[e];
      } else {
        const Pack<E, 4> v = *reinterpret_cast<const Pack<E, 4>*>(p + ((s ^ swz(row)) << 4) + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = to_f32(v.v[e]);
      }
    } else {
      const E* p = reinterpret_cast<const E*>(lds) + (8 * s + 4 * g) * ROWS + row;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = to_f32(p[e * ROWS]);
    }
  }
};

// Step SumsOnly: the sums (or a split's part of them) to p.out; otherwise, K not split,
// the step takes them from the accumulators: 32 lanes hold a row's 32 columns.
struct SumsOnly {};

template <typename EA, typename EB, int LA, int LB, int T, class Step>
__global__ __launch_bounds__(256, 2) void f32_kernel(const F32Problem p, const Step step) {
  constexpr int TILE = 64 * T, W = 32 * T;
  using OA = F32Operand<EA, LA, TILE>;
  using OB = F32Operand<EB, LB, TILE>;
  constexpr int kStage = OA::kBytes + OB::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[2][kStage];
  // items: the split slowest, tiles row-fastest; XCD b % 8 walks a contiguous range
  const int tiles = p.tiles_m * p.tiles_n, items = tiles * p.splits;
  const int q = items / gemm::kXcds, r = items % gemm::kXcds, xcd = blockIdx.x % gemm::kXcds;
  const int item = xcd * q + min(xcd, r) + (int)blockIdx.x / gemm::kXcds;
  const int split = item / tiles, tile = item - split * tiles;
  const int m0 = tile % p.tiles_m * TILE, n0 = tile / p.tiles_m * TILE;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = (wave >> 1) * W, wn = (wave & 1) * W;

  int nk = 0;
  for (int s = 0; s < p.nseg; ++s) nk += (p.seg[s].K + kF32K - 1) / kF32K;
  int first = split * p.kps, seg = 0;
  nk = nk - first < p.kps ? nk - first : p.kps;
  if (p.nseg > 1) {
    const int n = (p.seg[0].K + kF32K - 1) / kF32K;
    if (first >= n) {
      first -= n;
      seg = 1;
    }
  }

  f32x16 acc[T][T];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;

  OA oa;
  OB ob;
  int k = first * kF32K, K = p.seg[seg].K;
  oa.setup(p.seg[seg].a, p.seg[seg].lda, m0, p.M, k, K, wave, lane);
  ob.setup(p.seg[seg].b, p.seg[seg].ldb, n0, p.N, k, K, wave, lane);
  auto advance = [&]() {  // to the k-tile after the loaded one
    k += kF32K;
    if (k >= K && seg + 1 < p.nseg) {
      ++seg;
      k = 0;
      K = p.seg[seg].K;
      oa.setup(p.seg[seg].a, p.seg[seg].lda, m0, p.M, 0, K, wave, lane);
      ob.setup(p.seg[seg].b, p.seg[seg].ldb, n0, p.N, 0, K, wave, lane);
    } else {
      oa.base += oa.step;
      oa.range -= oa.step;
      ob.base += ob.step;
      ob.range -= ob.step;
    }
  };
  oa.load(lds[0], wave, true, K - k);
  ob.load(lds[0] + OA::kBytes, wave, true, K - k);
  __builtin_amdgcn_s_waitcnt(gemm::big::kWaitVm0);
  gemm::lds_barrier();

  // Fragments are read a step ahead of their products, over the end of a k-tile as well:
  // its last step waits for the next k-tile's loads and the other waves (which frees its
  // stage), reads the next one's first fragments and then multiplies.
  const int fr = lane & 31, g = lane >> 5;
  float a[2][T][4], b[2][T][4];
  auto read = [&](int to, const char* st, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T; ++i) OA::fragment(st, wm + 32 * i + fr, g, s, a[to][i]);
#pragma unroll
    for (int j = 0; j < T; ++j) OB::fragment(st + OA::kBytes, wn + 32 * j + fr, g, s, b[to][j]);
  };
  read(0, lds[0], 0);
  for (int t = 0; t < nk; ++t) {
    const char* st = lds[t & 1];
    char* ld = lds[(t & 1) ^ 1];
    advance();
    oa.load(ld, wave, t + 1 < nk, K - k);
    ob.load(ld + OA::kBytes, wave, t + 1 < nk, K - k);
    constexpr int kSteps = kF32K / 8;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (s + 1 < kSteps) {
        read((s + 1) & 1, st, s + 1);
      } else {
        __builtin_amdgcn_s_waitcnt(gemm::big::kWaitVm0);
        gemm::lds_barrier();
        read((s + 1) & 1, ld, 0);  // (past the last k-tile: zeros)
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = 0; j < T; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s & 1][i][e], b[s & 1][j][e],
                                                             acc[i][j], 0, 0, 0);
    }
  }

  // element v of tile (i, j): row 32 i + 8 (v / 4) + 4 g + v % 4, column 32 j + lane % 32
  if constexpr (std::is_same_v<Step, SumsOnly>) {
    float* out = p.out + (int64_t)split * p.M * p.N;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int n = n0 + wn + 32 * j + fr;
      if (n >= p.N) continue;
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int m = m0 + wm + 32 * i + 8 * (v >> 2) + 4 * g + (v & 3);
          if (m < p.M) out[(int64_t)m * p.N + n] = acc[i][j][v];
        }
    }
  } else {
    constexpr int B = 8;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int n = n0 + wn + 32 * j + fr, nc = n < p.N ? n : 0;
      const typename Step::template Column<1> column = step.template column<1>(nc);
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int v0 = 0; v0 < 16; v0 += B) {
          int64_t m[B];
          bool live[B];
          float x[B][1];
          typename Step::template Fetched<1> f[B];
#pragma unroll
          for (int q = 0; q < B; ++q) {
            const int v = v0 + q, r = m0 + wm + 32 * i + 8 * (v >> 2) + 4 * g + (v & 3);
            m[q] = r;
            live[q] = r < p.M && n < p.N;
            x[q][0] = acc[i][j][v];
            f[q] = step.template fetch<1>(r < p.M ? r : p.M - 1, nc);
          }
          step.template finish<false, 1, B>(m, n, x, column, f, live);
          // (a group's loads are not moved before the last one's: two workgroups a CU
          // need the registers)
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }
}

struct F32Plan {
  int tile, splits, kps;
};

// A CU's matrix cores take c us for a k-tile of a 128 x 128 tile (.28 of it for 64 x 64),
// whichever of its workgroups it is of; parts of K are written once and read once, at 5
// TB/s. Fitted to the times of ten shapes from [128, 512] x 512 to [8192, 2048] x 2048
// with every split (4 % off in the mean; its choice costs 1 % over the best one).
inline F32Plan plan_f32(int64_t M, int64_t N, int64_t ktiles) {
  F32Plan best{128, 1, (int)ktiles};
  double best_us = -1;
  for (int tile = 128; tile >= 64; tile /= 2) {
    const int64_t tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
    const double c = tile == 128 ? 1.9 : 0.535;
    for (int s = 1; s <= 16; ++s) {
      const int64_t kps = (ktiles + s - 1) / s;
      if (s > 1 && (kps < 4 || (ktiles + kps - 1) / kps != s)) continue;
      const int64_t per_cu = (tiles * s + 255) / 256;
      double us = per_cu * c * kps;
      if (s > 1) us += (double)s * M * N * 8 / 5.0e6;
      if (best_us < 0 || us < best_us) {
        best_us = us;
        best = F32Plan{tile, s, (int)kps};
      }
    }
  }
  return best;
}

inline int64_t f32_ktiles(int nseg, const int64_t* K) {
  int64_t n = 0;
  for (int s = 0; s < nseg; ++s) n += (K[s] + kF32K - 1) / kF32K;
  return n;
}

template <typename EA, typename EB, int LA, int LB, class Step>
inline int launch_f32(F32Problem& p, const F32Plan& plan, const Step& step, hipStream_t st) {
  p.tiles_m = (p.M + plan.tile - 1) / plan.tile;
  p.tiles_n = (p.N + plan.tile - 1) / plan.tile;
  p.splits = plan.splits;
  p.kps = plan.kps;
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  ML_CHECK(items <= 0x7fffffffLL, "ffn: too many tiles");
  const dim3 grid((unsigned)items);
  if (plan.tile == 128)
    f32_kernel<EA, EB, LA, LB, 2, Step><<<grid, 256, 0, st>>>(p, step);
  else
    f32_kernel<EA, EB, LA, LB, 1, Step><<<grid, 256, 0, st>>>(p, step);
  ML_LAUNCH_CHECK();
  return ML_OK;
}

}  // namespace ffn
}  // namespace mla
