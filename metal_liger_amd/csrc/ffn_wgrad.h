// Weight gradients: C_g = A_g^T B_g with A_g [K, M_g] and B_g [K, N_g] row-major (K the
// tokens), up to three products of one K in one launch on the 8-wave engine
// (gemm_core.h).
//
// The launch's 256 x 256 tiles rarely come in whole rounds of one per CU: the three of a
// gated block of 2048 x 6144 are 576 tiles, 2.25 rounds, a vision tower's 4304 x 1152
// are 85, a third of one. So the whole rounds run as they are and the tiles of the
// last, partial round are split over K, as many ways as the estimate below finds best;
// their fp32 partials lie in the workspace as the accumulators lie in the lanes (16
// bytes a lane, whatever the tile's edges) and a second kernel sums them in split
// order, eight workgroups a tile. Bound by the matrix cores; [8192, 4304]^T [8192, 1152]:
// 188 us as 85 tiles, 90 split three ways and 17 to join; the gated block's three at 8192
// tokens 660 us one by one, 546 and 16 together.
#pragma once

#include "gemm_core.h"

namespace mla {
namespace ffn {

struct WgradTiles {
  int64_t M, N;
};

struct WgradProduct {
  WgradTiles size;
  const bf16 *a, *b;
  int64_t lda, ldb;
  bf16* c;  // dense
};

constexpr int kMaxWgrads = 3;
constexpr int kTileFloats = 256 * 256;
constexpr int kMaxTailSplit = 16;

struct WgradPlan {
  int tiles, full;  // all tiles; those of whole rounds
  int splits, kps;  // of the others: 64-wide k-tiles per split
  size_t floats;    // of partials
};

// Times on one MI355X: a tile of kt 64-wide k-tiles 10 + 1.6 kt us in a round of 256;
// partials are written and read once (262 KB each way at 4.5 TB/s).
inline WgradPlan plan_wgrads(int count, const WgradTiles* p, int64_t K) {
  WgradPlan w{};
  for (int g = 0; g < count; ++g)
    w.tiles += (int)(((p[g].M + 255) / 256) * ((p[g].N + 255) / 256));
  const int kt = (int)((K + gemm::kBK - 1) / gemm::kBK);
  const int tail = w.tiles % 256;
  w.full = w.tiles - tail;
  w.splits = 1;
  w.kps = kt;
  double best = -1;
  for (int s = 1; tail && s <= kMaxTailSplit; ++s) {
    const int kps = (kt + s - 1) / s;
    if (s > 1 && (kps < 8 || (kt + kps - 1) / kps != s)) continue;  // short, or empty splits
    const double rounds = (tail * s + 255) / 256;
    const double us = rounds * (10 + 1.6 * kps) + (s > 1 ? 4 + 0.117 * tail * s : 0);
    if (best < 0 || us < best) {
      best = us;
      w.splits = s;
      w.kps = kps;
    }
  }
  if (w.splits == 1) w.full = w.tiles;
  w.floats = (size_t)(w.tiles - w.full) * w.splits * kTileFloats * (w.splits > 1);
  return w;
}

struct WgradArgs {
  gemm::Problem pb[kMaxWgrads];
  gemm::EpiStore<bf16> epi[kMaxWgrads];
  int first[kMaxWgrads + 1];  // tiles of the products before
  int count;
  int tiles, full, splits, kps;
  float* partial;
};

// Product and tile of index t (m-fastest within groups, as tile_coords).
__device__ __forceinline__ int wgrad_tile(const WgradArgs& w, int t, int& tm, int& tn) {
  const int g = (w.count > 2 && t >= w.first[2]) ? 2 : (w.count > 1 && t >= w.first[1]) ? 1 : 0;
  const gemm::Problem& pb = w.pb[g];
  t -= w.first[g];
  const int gsize = pb.group_m * pb.tiles_n;
  const int grp = t / gsize, first_m = grp * pb.group_m;
  const int gm = min(pb.tiles_m - first_m, pb.group_m);
  const int within = t - grp * gsize;
  tm = first_m + within % gm;
  tn = within / gm;
  return g;
}

// Blocks 0 .. full - 1 (a multiple of 256 unless nothing is split): a tile each; the
// rest: a tile's split each, the split slowest. Each XCD (block mod 8) walks a
// contiguous range of either part.
__global__ __launch_bounds__(512) void wgrad_kernel(const WgradArgs w) {
  const int bid = blockIdx.x;
  const int tail = w.tiles - w.full;
  const bool whole = bid < w.full;
  const int items = whole ? w.full : tail * w.splits;
  const int b = whole ? bid : bid - w.full;
  // item of block b: XCD b % 8 has the items from (b % 8) * (items / 8) on, the first
  // items % 8 XCDs one more
  const int q = items / gemm::kXcds, r = items % gemm::kXcds, x = b % gemm::kXcds;
  const int item = x * q + min(x, r) + b / gemm::kXcds;
  const int split = whole ? 0 : item / tail;
  const int at = whole ? item : item - split * tail;
  int tm, tn;
  const int g = wgrad_tile(w, whole ? at : w.full + at, tm, tn);
  const gemm::Problem& pb = g == 0 ? w.pb[0] : g == 1 ? w.pb[1] : w.pb[2];
  const gemm::EpiStore<bf16>& epi = g == 0 ? w.epi[0] : g == 1 ? w.epi[1] : w.epi[2];
  __shared__ __attribute__((aligned(16))) char lds[gemm::big::STAGES * gemm::big::STAGE_BYTES];
  gemm::f32x4_t acc[gemm::big::TM][gemm::big::TN];
  gemm::big_mainloop<gemm::kMNMajor, gemm::kMNMajor>(pb, tm, tn, split, lds, acc, 0,
                                                     whole ? 1 : w.splits, w.kps);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (whole) {
    epi(acc, tm * 256 + (wave >> 2) * gemm::big::WM, tn * 256 + (wave & 3) * gemm::big::WN, lane,
        lds + wave * gemm::big::EPI_BYTES, 0);
    return;
  }
  float* p = w.partial + ((int64_t)at * w.splits + split) * kTileFloats +
             (wave * (gemm::big::TM * gemm::big::TN) * 64 + lane) * 4;
#pragma unroll
  for (int i = 0; i < gemm::big::TM; ++i)
#pragma unroll
    for (int j = 0; j < gemm::big::TN; ++j)
      *reinterpret_cast<gemm::f32x4_t*>(p + (i * gemm::big::TN + j) * 256) = acc[i][j];
}

// A wave joins a quarter of one wave's sub-tile (32 x 64): 8 16-byte loads a split in
// flight, 8 workgroups a tile. (One workgroup a tile, 85 tiles of 3 splits: 30 us.)
__global__ __launch_bounds__(256) void wgrad_join_kernel(const WgradArgs w) {
  constexpr int TM = 2, TN = gemm::big::TN;
  const int at = blockIdx.x / 8;
  int tm, tn;
  const int g = wgrad_tile(w, w.full + at, tm, tn);
  const gemm::EpiStore<bf16>& epi = g == 0 ? w.epi[0] : g == 1 ? w.epi[1] : w.epi[2];
  __shared__ __attribute__((aligned(16))) char lds[4 * TM * TN * 512];
  const int part = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wave = blockIdx.x % 8;
  gemm::f32x4_t acc[TM][TN];
  const float* p = w.partial + (int64_t)at * w.splits * kTileFloats +
                   ((wave * gemm::big::TM + part * TM) * TN * 64 + lane) * 4;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
      acc[i][j] = *reinterpret_cast<const gemm::f32x4_t*>(p + (i * TN + j) * 256);
#pragma unroll 2
  for (int s = 1; s < w.splits; ++s) {
    p += kTileFloats;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] += *reinterpret_cast<const gemm::f32x4_t*>(p + (i * TN + j) * 256);
  }
  constexpr int kVecs = TM * TN / 2;
  gemm::stage_rows_bf16<kVecs, TM, TN>(
      lds + part * TM * TN * 512, lane, tm * 256 + (wave >> 2) * gemm::big::WM + part * 16 * TM,
      tn * 256 + (wave & 3) * gemm::big::WN, [&](int i, int j, int v) { return acc[i][j][v]; },
      [&](const int (&m)[kVecs], const int (&n)[kVecs], const float (&x)[kVecs][8]) {
#pragma unroll
        for (int q = 0; q < kVecs; ++q)
          if (m[q] < epi.M && n[q] < epi.N)
            gemm::store_row8_bf16(epi.C + (int64_t)m[q] * epi.ldc + n[q], n[q], epi.N, x[q]);
      });
}

inline int launch_wgrads(int count, const WgradProduct* p, int64_t K, void* ws, size_t wsb,
                         hipStream_t st) {
  WgradTiles sizes[kMaxWgrads];
  for (int g = 0; g < count; ++g) sizes[g] = p[g].size;
  const WgradPlan plan = plan_wgrads(count, sizes, K);
  ML_CHECK(plan.floats * sizeof(float) <= wsb, "ffn: weight gradients' workspace too small");
  WgradArgs w{};
  w.count = count;
  for (int g = 0; g < count; ++g) {
    const gemm::Segment s{{p[g].a, p[g].lda}, {p[g].b, p[g].ldb}, (int)K};
    const int rc = gemm::make_problem<gemm::BigCfg>(w.pb[g], (int)p[g].size.M, (int)p[g].size.N, 1, &s,
                                                    gemm::kMNMajor, gemm::kMNMajor, 0);
    if (rc) return rc;
    w.epi[g] = gemm::EpiStore<bf16>{p[g].c, p[g].size.N, (int)p[g].size.M, (int)p[g].size.N, 1.f, 0.f};
    w.first[g + 1] = w.first[g] + w.pb[g].tiles_m * w.pb[g].tiles_n;
  }
  w.tiles = plan.tiles;
  w.full = plan.full;
  w.splits = plan.splits;
  w.kps = plan.kps;
  w.partial = static_cast<float*>(ws);
  const int tail = w.tiles - w.full;
  wgrad_kernel<<<dim3(w.full + tail * w.splits), 512, 0, st>>>(w);
  ML_LAUNCH_CHECK();
  if (tail) {
    wgrad_join_kernel<<<dim3(8 * tail), 256, 0, st>>>(w);
    ML_LAUNCH_CHECK();
  }
  return ML_OK;
}

}  // namespace ffn
}  // namespace mla
