// Products of few rows (single tokens, short prompts) through the steps of ffn_rows.h:
//   C [M, N] = x [M, K] W [N, K]^T, M up to 128.
//
// Bound by W's bytes and by latency: [1, 2048] x 6144 in bf16 are 25 MB, 5 us at the
// rate of a large copy. A workgroup takes 16 NT rows of W and all of K, its 8 waves every
// eighth 64-wide k-chunk each, so that some 8 MB are in flight over the GPU; their sums
// are joined in LDS in wave order (nothing is left to a second launch, and no atomics).
// Per chunk a lane loads 16 neighbouring elements of one row of W (four lanes a row:
// whole 128-byte lines of 16-bit elements) and of x, straight into the operands of
// 16 x 16 MFMAs: which k an operand slot holds does not matter as long as both operands
// agree, so the lane's 16 elements feed the chunk's steps in order.
//   bf16 and fp16 by bf16 or fp16: v_mfma_f32_16x16x32 (exact products, fp32 sums)
//   fp32 by fp32 or fp16: v_mfma_f32_16x16x4_f32, W upcast in registers
// With PAIR a second W of the same shape beside it (gate and up).
// Tiles of 16 rows of x are shared out over workgroups where that gives the CUs more to do
// (plan_skinny); W then comes from the caches again. A workgroup for all of x's rows and
// so: [64, 2048] to 512 columns in bf16 11.0 and 5.8 us, [64, 4304] to 1152 15.7 and 10.6,
// [64, 6144] to 2048 29.4 and 19.2.
#pragma once

#include "ffn_rows.h"

namespace mla {
namespace ffn {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kSkinnyWaves = 8;
constexpr int kSkinnyRows = 128;  // most rows of x
constexpr int kChunk = 64;       // k a chunk

// A lane's 16 elements of a chunk (of one row, from k = 16 (lane / 16)): two halves of 8.
template <typename T>
struct Strip {
  Pack<T, 8> h[2];

  // k0: of the lane; whole: both halves are within K
  __device__ __forceinline__ void load(const T* row, int k0, int K, bool whole) {
    if (whole) {
      load_pack<T, 8>(row + k0, h[0]);
      load_pack<T, 8>(row + k0 + 8, h[1]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool in = k0 + 8 * i < K;
      load_pack<T, 8>(row + (in ? k0 + 8 * i : 0), h[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i].v[e] = in ? h[i].v[e] : (T)0.f;
    }
  }
};

template <typename TX, typename TW>
__device__ __forceinline__ void strip_mma(f32x4& acc, const Strip<TW>& w, const Strip<TX>& x) {
  typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
  typedef f16 f16x8 __attribute__((ext_vector_type(8)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (std::is_same_v<TX, bf16>) {
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.h[i]),
                                                    __builtin_bit_cast(bf16x8, x.h[i]), acc, 0, 0, 0);
    } else if constexpr (std::is_same_v<TX, f16>) {
      acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w.h[i]),
                                                   __builtin_bit_cast(f16x8, x.h[i]), acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.h[i].v[e]), x.h[i].v[e], acc, 0, 0, 0);
    }
  }
}

template <typename TX, typename TW>
struct SkinnyProduct {
  const TX* x;
  const TW *w, *w2;  // w2: PAIR
  int64_t ldx, ldw, ldw2;
  int M, N, K;
};

// MT: tiles of 16 rows of x; NT: of W (2 where the step keeps a tensor: a block of 32
// columns); REGS: registers for loads in flight. (8 rows of W a workgroup, so that 2048
// of them lie on 256 CUs instead of 128, gained nothing, and cost 17% at 6144 pairs.)
template <typename TX, typename TW, int MT, int NT, bool PAIR, int REGS, class Step>
__global__ __launch_bounds__(64 * kSkinnyWaves) void skinny_kernel(
    const SkinnyProduct<TX, TW> p, const Step step) {
  constexpr int kOps = PAIR ? 2 : 1;
  constexpr int kTiles = kOps * NT * MT;
  constexpr int kPitch = 16 * NT + 4;
  __shared__ __attribute__((aligned(16))) float red[kSkinnyWaves][kTiles][64][4];
  __shared__ __attribute__((aligned(16))) float fin[kOps][16 * MT][kPitch];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r = lane & 15, G = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  // rows past the ends read the last one (their results are not used)
  const TW* wr[kOps][NT];
  const TX* xr[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + 16 * j + r < p.N ? n0 + 16 * j + r : p.N - 1;
    wr[0][j] = p.w + n * p.ldw;
    if constexpr (PAIR) wr[1][j] = p.w2 + n * p.ldw2;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + r < p.M ? m0 + 16 * i + r : p.M - 1;
    xr[i] = p.x + m * p.ldx;
  }
  f32x4 acc[kOps][NT][MT];
#pragma unroll
  for (int o = 0; o < kOps; ++o)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[o][j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  // chunks c, c + 8, .. of a batch: every load before the first product
  constexpr int kRegs = 4 * (kOps * NT * (int)sizeof(TW) + MT * (int)sizeof(TX));
  constexpr int kBatch = REGS / kRegs > 0 ? REGS / kRegs : 1;
  const int chunks = (p.K + kChunk - 1) / kChunk;
  for (int c0 = wave; c0 < chunks; c0 += kSkinnyWaves * kBatch) {
    Strip<TW> ws[kBatch][kOps][NT];
    Strip<TX> xs[kBatch][MT];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * kSkinnyWaves;  // (wave-uniform, as the branches on it are)
      if (c >= chunks) break;
      const int k0 = c * kChunk + 16 * G;
      const bool whole = (c + 1) * kChunk <= p.K;
#pragma unroll
      for (int o = 0; o < kOps; ++o)
#pragma unroll
        for (int j = 0; j < NT; ++j) ws[u][o][j].load(wr[o][j], k0, p.K, whole);
#pragma unroll
      for (int i = 0; i < MT; ++i) xs[u][i].load(xr[i], k0, p.K, whole);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (c0 + u * kSkinnyWaves >= chunks) break;
#pragma unroll
      for (int o = 0; o < kOps; ++o)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i) strip_mma<TX, TW>(acc[o][j][i], ws[u][o][j], xs[u][i]);
    }
  }

#pragma unroll
  for (int o = 0; o < kOps; ++o)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        *reinterpret_cast<f32x4*>(red[wave][(o * NT + j) * MT + i][lane]) = acc[o][j][i];
  __syncthreads();
  // element v of a lane of tile (o, j, i): row 16 i + lane % 16 of x, row 16 j + 4 (lane /
  // 16) + v of W
  for (int q = threadIdx.x; q < kTiles * 64; q += 64 * kSkinnyWaves) {
    const int t = q >> 6, l = q & 63;
    f32x4 s = *reinterpret_cast<const f32x4*>(red[0][t][l]);
#pragma unroll
    for (int w = 1; w < kSkinnyWaves; ++w) s += *reinterpret_cast<const f32x4*>(red[w][t][l]);
    const int i = t % MT, j = t / MT % NT, o = t / MT / NT;
    *reinterpret_cast<f32x4*>(&fin[o][16 * i + (l & 15)][16 * j + 4 * (l >> 4)]) = s;
  }
  __syncthreads();
  // 2 NT neighbouring lanes a row
  constexpr int kLanes = 2 * NT;
  constexpr int kPositions = 16 * MT * kLanes;
  for (int q = threadIdx.x; q < (kPositions + 63) / 64 * 64; q += 64 * kSkinnyWaves) {
    const int row = q < kPositions ? q / kLanes : 0, c = 8 * (q % kLanes);
    const int m = m0 + row, n = n0 + c;
    const bool live = m < p.M && n < p.N && q < kPositions;
    typename Step::template Column<8> column;
    typename Step::template Fetched<8> f[1];
    if (live) {
      column = step.template column<8>(n);
      f[0] = step.template fetch<8>(m, n);
    }
    float x[1][8];
    load_n<float, 8>(&fin[0][row][c], x[0]);
    const int64_t ms[1] = {m};
    const bool lives[1] = {live};
    if constexpr (PAIR) {
      float u[1][8];
      load_n<float, 8>(&fin[1][row][c], u[0]);
      step.template finish<false, 8, 1>(ms, n, x, u, column, f, lives);
    } else {
      step.template finish<false, 8, 1>(ms, n, x, column, f, lives);
    }
  }
}

// How many tiles of 16 rows a workgroup takes (mt, up to 4), and the time in us: a round of
// 256 workgroups (one a CU; two that share one take as long as one after the other) goes
// by K and the bytes that they read of W and x. nt: tiles of 16 rows of W; ops: 2 for a
// pair. Fitted to 17 .. 256 rows by six shapes of W, 1152 x 4304 to 16384 x 2048, with
// mt 1, 2 and 4, in bf16 and fp32, with and without a kept tensor.
struct SkinnyPlan {
  int mt;
  double us;
};

inline SkinnyPlan plan_skinny(int x_size, int w_size, int ops, int nt, int64_t M, int64_t N,
                              int64_t K) {
  const int64_t blocks = (N + 16 * nt - 1) / (16 * nt), tiles = (M + 15) / 16;
  SkinnyPlan best{1, -1};
  for (int mt = 1; mt <= 4 && mt <= tiles; ++mt) {
    const int64_t rounds = (blocks * ((tiles + mt - 1) / mt) + 255) / 256;
    const double x_cost = ops * nt > 1 ? 1.2 : 1.0;
    const double us = 2.4 + rounds * 0.43e-3 * K * (ops * nt * w_size + x_cost * mt * x_size);
    if (best.us < 0 || us < best.us) best = {mt, us};
  }
  return best;
}

template <int MT, bool KEEPS, bool PAIR, typename TX, typename TW, class Step>
inline void skinny_launch(const SkinnyProduct<TX, TW>& p, const Step& step, hipStream_t st) {
  constexpr int NT = KEEPS ? 2 : 1, kThreads = 64 * kSkinnyWaves;
  const int blocks = (p.N + 16 * NT - 1) / (16 * NT), parts = (p.M + 16 * MT - 1) / (16 * MT);
  // One workgroup a CU may fill its registers with loads (K = 6144 in one or two
  // batches); where there are more, two share a CU.
  constexpr int kOne = MT > 2 || KEEPS ? 96 : 160;
  const dim3 grid(blocks, parts);
  if (blocks * parts <= num_cus())
    skinny_kernel<TX, TW, MT, NT, PAIR, kOne, Step><<<grid, kThreads, 0, st>>>(p, step);
  else
    skinny_kernel<TX, TW, MT, NT, PAIR, 96, Step><<<grid, kThreads, 0, st>>>(p, step);
}

template <bool KEEPS, bool PAIR, typename TX, typename TW, class Step>
inline int launch_skinny(const SkinnyProduct<TX, TW>& p, const Step& step, hipStream_t st) {
  switch (plan_skinny(sizeof(TX), sizeof(TW), PAIR ? 2 : 1, KEEPS ? 2 : 1, p.M, p.N, p.K).mt) {
    case 1: skinny_launch<1, KEEPS, PAIR>(p, step, st); break;
    case 2: skinny_launch<2, KEEPS, PAIR>(p, step, st); break;
    case 3: skinny_launch<3, KEEPS, PAIR>(p, step, st); break;
    default: skinny_launch<4, KEEPS, PAIR>(p, step, st); break;
  }
  ML_LAUNCH_CHECK();
  return ML_OK;
}

}  // namespace ffn
}  // namespace mla
