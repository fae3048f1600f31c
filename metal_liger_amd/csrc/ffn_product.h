// A product on the r4 engine (gemm_core.h) whose epilogue is one of the steps of
// ffn_rows.h, in fp32: nothing is rounded between the sum and the step's outputs.
//
// A wave's sums lie in its registers as columns of 4 rows; the steps take 8
// neighbouring columns of a row (16-byte accesses, and a block of 32 columns in 4
// neighbouring lanes). So the wave stages 64 rows of its sub-tile at a time through
// LDS of its own, in fp32, rows padded by 4 floats: the writes of one instruction (4
// rows of 16 columns) fall into 64 different banks, and 16 lanes' 16-byte reads as
// well. Staging fp32 instead of the rounded result costs twice the LDS traffic (a
// 256 x 256 tile: 512 KB, some 4000 of about 80000 cycles at K = 2048).
#pragma once

#include "ffn_rows.h"
#include "gemm_core.h"

namespace mla {
namespace ffn {

template <int T, bool PAIR>
struct Stager {
  static constexpr int W = 16 * T;                 // a wave's rows and columns
  static constexpr int kPitch = W + 4;             // floats
  static constexpr int kRows = 64;                 // rows staged at a time
  static constexpr int kWaveBytes = kRows * kPitch * 4;
  static constexpr int kCols = PAIR ? W / 2 : W;   // columns of one operand
  static constexpr int kLanes = kCols / 8;         // lanes a row
  static constexpr int kStepRows = 64 / kLanes;    // rows a step of the wave takes
  static constexpr int kSteps = kRows / kStepRows;
  // positions of a lane whose loads are in flight while the last ones are worked on
  static constexpr int kBatch = 4;
  static_assert(kSteps % kBatch == 0, "whole batches");
  static_assert(4 * kWaveBytes <= gemm::r4::Geom<T>::LDS_BYTES, "within the operand slots");

  // Rows m0 .. m0 + W - 1, columns n0 .. n0 + kCols - 1 of this wave (lds: its own).
  // ALL: all of them are within M and N.
  template <bool ALL, class Step>
  static __device__ __forceinline__ void run(gemm::f32x4_t (&acc)[T / 4][T][4], float* lds, int m0,
                                             int n0, int lane, int M, int N, const Step& step) {
    const int G = lane >> 4, c = lane & 15;
    float* wr = lds + 4 * G * kPitch + c;
    const int row = lane / kLanes, col = 8 * (lane % kLanes);
    const float* rd = lds + row * kPitch + col;
    const int n = n0 + col;
    using Fetched = typename Step::template Fetched<8>;
    const int nc = ALL || n < N ? n : 0;  // positions past the edges fetch others, in range
    const typename Step::template Column<8> column = step.template column<8>(nc);
    Fetched next[kBatch];
    auto fetch = [&](Fetched(&f)[kBatch], int m) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = m + k * kStepRows;
        f[k] = step.template fetch<8>(r < M ? r : M - 1, nc);
      }
    };
    fetch(next, m0 + row);
#pragma unroll
    for (int half = 0; half < W / kRows; ++half) {
      const int mh = m0 + half * kRows + row;
#pragma unroll
      for (int i = 0; i < kRows / 16; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            wr[(16 * i + v) * kPitch + 16 * j] = acc[j >> 2][half * (kRows / 16) + i][j & 3][v];
      // the wave's own LDS: its writes before its reads, and these before the next half
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
#pragma unroll 1
      for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
        Fetched now[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) now[k] = next[k];
        const int m1 = mh + (s0 + kBatch) * kStepRows;  // the next batch: of this half, then the next
        fetch(next, s0 + kBatch < kSteps ? m1 : mh + kRows);
        int64_t m[kBatch];
        bool live[kBatch];
        float x[kBatch][8], u[PAIR ? kBatch : 1][8];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int r = (s0 + k) * kStepRows;
          m[k] = mh + r;
          live[k] = ALL || (mh + r < M && n < N);
          load_n<float, 8>(rd + r * kPitch, x[k]);
          if constexpr (PAIR) load_n<float, 8>(rd + r * kPitch + kCols, u[k]);
        }
        if constexpr (PAIR)
          step.template finish<ALL, 8, kBatch>(m, n, x, u, column, now, live);
        else
          step.template finish<ALL, 8, kBatch>(m, n, x, column, now, live);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    }
  }
};

// The tile of a product that carries a step: 256 x 256, or 128 x 128, of which two
// workgroups share a CU, so that one's epilogue runs beside the other's products. Which
// is faster goes by the rounds of tiles, K and the step. Times in us on one MI355X,
// fitted to 152 products each way (rows 130 .. 8192, columns and K 1024 .. 6144; off by
// 2.5-8%; the choice it makes was at most 6% slower than the better tile, 0.2% on
// average, that of the plain products' estimate up to 31%: [8192, 1152] x 4304 with
// gelu_tanh 134 us as 256 x 256 tiles, 102 as 128 x 128; [8192, 2048] x 6144 with both
// of the gated block's products 338 and 436):
//   256: a whole round of 256 tiles of kt 64-wide k-tiles c0 + c1 kt, a partial one of r
//        c2 + c3 kt + (c4 + c5 kt) r / 256
//   128: a whole round of 512 c0 + c1 kt, a partial one c2 + c3 kt, and where it has
//        more than one tile a CU c4 + c5 kt besides
inline double step_us(int tile, int kind, int64_t items, int kt) {
  static const double k256[4][6] = {{12.4, 1.40, 13.3, 1.05, 7.1, 0.11},
                                    {22.7, 1.37, 21.4, 1.11, 8.9, 0.01},
                                    {10.7, 1.40, 14.3, 1.10, 3.9, 0.21},
                                    {38.8, 1.27, 21.9, 1.11, 0.3, 0.38}};
  static const double k128[4][6] = {{0.0, 0.99, 5.6, 0.49, 1.4, 0.32},
                                    {4.5, 0.95, 8.2, 0.49, 1.4, 0.37},
                                    {4.2, 0.88, 7.1, 0.50, 2.1, 0.32},
                                    {17.2, 0.81, 9.2, 0.49, 7.3, 0.17}};
  const double* c = tile == 256 ? k256[kind] : k128[kind];
  const int64_t round = tile == 256 ? 256 : 512, full = items / round, rem = items % round;
  double t = full * (c[0] + c[1] * kt);
  if (rem) {
    t += c[2] + c[3] * kt;
    if (tile == 256) t += (c[4] + c[5] * kt) * rem / 256;
    else if (rem > 256) t += c[4] + c[5] * kt;
  }
  return t;
}

// columns: of both products of a pair together
inline int step_tile(int kind, int64_t M, int64_t columns, int64_t K) {
  const int kt = (int)((K + gemm::kBK - 1) / gemm::kBK);
  double us[2];
  for (int i = 0; i < 2; ++i) {
    const int64_t t = i ? 128 : 256;
    us[i] = step_us((int)t, kind, ((M + t - 1) / t) * ((columns + t - 1) / t), kt);
  }
  return us[0] <= us[1] ? 256 : 128;
}

// C: R4Cfg or R4SCfg; b2: the second operand of a pair.
template <class C, int LB, bool PAIR, class Step>
__global__ __launch_bounds__(C::THREADS) void product_kernel(const gemm::Problem pb,
                                                             const gemm::Operand b2,
                                                             const Step step) {
  constexpr int T = C::BM / 32;
  using G = gemm::r4::Geom<T>;
  using S = Stager<T, PAIR>;
  int tm, tn, split;
  if (!gemm::tile_coords(pb, pb.tiles_m, 1, blockIdx.x, tm, tn, split)) return;
  __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
  gemm::f32x4_t acc[T / 4][T][4];
  gemm::r4_mainloop<gemm::kKMajor, LB, T, false, PAIR>(pb, tm, tn, 0, 1, 0, lds, acc, b2);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  constexpr int kTileN = PAIR ? C::BN / 2 : C::BN;
  float* wl = reinterpret_cast<float*>(lds + w * S::kWaveBytes);
  const int m0 = tm * C::BM + (w >> 1) * S::W, n0 = tn * kTileN + (w & 1) * S::kCols;
  if (m0 + S::W <= pb.M && n0 + S::kCols <= pb.N)  // (wave-uniform)
    S::template run<true>(acc, wl, m0, n0, threadIdx.x & 63, pb.M, pb.N, step);
  else
    S::template run<false>(acc, wl, m0, n0, threadIdx.x & 63, pb.M, pb.N, step);
}

// The product of a [M, K] and b ([N, K], or with LB kMNMajor [K, N]) through the step.
template <class C, int LB, bool PAIR, class Step>
inline int launch_product(int64_t M, int64_t N, const gemm::Segment& s, const gemm::Operand& b2,
                          const Step& step, hipStream_t st) {
  gemm::Problem pb;
  int rc = gemm::make_problem<C>(pb, (int)M, (int)N, 1, &s, gemm::kKMajor, LB, 0);
  if (rc) return rc;
  if constexpr (PAIR) {
    rc = gemm::check_operand(b2, gemm::kKMajor, (int)N, s.k_len, "second B");
    if (rc) return rc;
    pb.tiles_n = (pb.N + C::BN / 2 - 1) / (C::BN / 2);
  }
  product_kernel<C, LB, PAIR, Step><<<dim3(gemm::grid_blocks(pb)), C::THREADS, 0, st>>>(pb, b2, step);
  ML_LAUNCH_CHECK();
  return ML_OK;
}

}  // namespace ffn
}  // namespace mla
