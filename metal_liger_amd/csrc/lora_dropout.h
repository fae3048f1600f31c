// LoRA with dropout on the adapters' input: the passes that need the masks. Included
// by lora.hip. For adapter i of n (1..3) that share X [N, IN], M_i its mask (dropout.h,
// stream `first + i` over X's elements), c_i = 65536 / (65536 - T_i):
//   forward    XA_i = c_i (M_i X) A_i^T                    drop_xa_kernel
//   backward   P_i  = c_i s_i dY_i B_i, dB_i               (the dY pass of lora.hip)
//              dX0  = sum_i dY_i W_i                       (one product)
//              dA_i = P_i^T (M_i X)
//              dX   = dX0 + sum_i M_i (P_i A_i)            drop_bwd_kernel
// c_i goes into the rank-r products, so that M_i X is X or 0 and no element is rounded.
// The mask keeps the adapters' part of dX out of the large product (K-concatenated
// there without dropout). It is added to the product's bf16 result, one rounding more
// than without dropout; as an epilogue of the product it would form every mask a second
// time (the pass over X for dA needs them too), while no workgroup multiplies.
#pragma once

constexpr int kDropMaxAdapters = 3;

// A_i is packed in fragment order (frag_offset). frag_size: the elements it takes;
// frag_of: a lane's part of the fragment of its 16-rank slice r at columns 32 s .. 32 s + 31.
__host__ __device__ inline int64_t frag_size(int rank, int K) {
  return (int64_t)rank * ((K + 31) / 32 * 32);
}
template <int RS>
__device__ __forceinline__ bf16x8_t frag_of(const bf16* A, int s, int r, int lane) {
  return *reinterpret_cast<const bf16x8_t*>(A + ((int64_t)(s * RS + r) * 64 + lane) * 8);
}

struct DropRates {
  DropRate rate[kDropMaxAdapters];
  uint32_t stream[kDropMaxAdapters];
  float scale[kDropMaxAdapters];  // c_i
};

__device__ __forceinline__ bf16x8_t masked8(u32x4_t x, u32x4_t m) {
  return __builtin_bit_cast(bf16x8_t, x & m);
}

// ----------------------------------------------------------------- forward --
// As xa_kernel (16 MT rows a workgroup, eight waves splitting K, X loaded in the MFMA
// layout and A lying in it), with every 8 elements of X that a lane holds masked once for each
// of NA adapters: a lane's operand is one counter's block of 8 elements, so that a mask
// costs one Philox call. RS 16-rank tiles per adapter; blockIdx.y takes the next NA.
template <int NA, int RS, int MT>
__global__ __launch_bounds__(64 * kXaWaves) void drop_xa_kernel(
    const bf16* __restrict__ X, int64_t ldx, const bf16* __restrict__ A, int N, int K,
    const int64_t* seed, const DropRates rates, bf16* __restrict__ XA, int64_t ldo) {
  constexpr int NT = NA * RS;
  constexpr int U = 4;                  // k-steps whose loads are in flight
  constexpr int W = 16 * MT * 16 * NT;  // one wave's sums
  __shared__ float red[kXaWaves * W];
  const int ad0 = blockIdx.y * NA;
  A += ad0 * frag_size(16 * RS, K);
  XA += ad0 * 16 * RS;
  const DropKey key = drop_key(seed);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = blockIdx.x * 16 * MT;
  const int ksteps = (K + 31) / 32;
  const int per = (ksteps + kXaWaves - 1) / kXaWaves;
  const int kb = wave * per, ke = kb + per < ksteps ? kb + per : ksteps;
  const int lr = lane & 15, lk = 8 * (lane >> 4);
  const bf16* xp[MT];
  uint64_t block[MT];  // the counter of the row's first 8 elements
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int row = m0 + 16 * t + lr < N ? m0 + 16 * t + lr : N - 1;
    xp[t] = X + (int64_t)row * ldx;
    block[t] = (uint64_t)row * (uint64_t)(K / 8);
  }
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int s0 = kb; s0 < ke; s0 += U) {
    u32x4_t a[U][MT];
    bf16x8_t b[U][NT];
    bool ok[U];
    int kc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 32 * (s0 + u) + lk;
      ok[u] = s0 + u < ke && k < K;
      kc[u] = ok[u] ? k : 0;  // lanes past K read the row's first 8
#pragma unroll
      for (int t = 0; t < MT; ++t) a[u][t] = *reinterpret_cast<const u32x4_t*>(xp[t] + kc[u]);
#pragma unroll
      for (int j = 0; j < NT; ++j)  // zeros past K
        b[u][j] = frag_of<RS>(A + j / RS * frag_size(16 * RS, K), s0 + u < ke ? s0 + u : kb, j % RS,
                              lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= ke) break;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const u32x4_t x = keep16(ok[u], a[u][t]);
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const bf16x8_t xm = masked8(x, drop_mask(block[t] + kc[u] / 8, rates.stream[ad0 + i], key,
                                                   rates.rate[ad0 + i]));
#pragma unroll
          for (int r = 0; r < RS; ++r)
            acc[t][i * RS + r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                xm, b[u][i * RS + r], acc[t][i * RS + r], 0, 0, 0);
        }
      }
    }
  }
  // element v of tile (t, j): row 16 t + 4 (lane / 16) + v, column 16 j + lane % 16
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        red[wave * W + (16 * t + 4 * (lane >> 4) + v) * (16 * NT) + 16 * j + lr] = acc[t][j][v];
  __syncthreads();
  for (int e = tid; e < W; e += 64 * kXaWaves) {
    const int row = m0 + e / (16 * NT), col = e % (16 * NT);
    const float s = ((red[e] + red[W + e]) + (red[2 * W + e] + red[3 * W + e])) +
                    ((red[4 * W + e] + red[5 * W + e]) + (red[6 * W + e] + red[7 * W + e]));
    if (row < N)
      XA[(int64_t)row * ldo + col] = from_f32<bf16>(s * rates.scale[ad0 + col / (16 * RS)]);
  }
}

// NA adapters per workgroup: all where their tiles are at most 4, else one each. 16 rows
// a workgroup until there are 256 workgroups of 32 (three adapters of rank 16 over
// [4096, 2048], again and again over the same X: 8.3 us by 16 rows, 13.4 by 32; one of
// rank 32 over [8192, 6144]: 23.4 and 21.9).
inline int drop_xa_adapters(int n, int rs) { return n * rs <= 4 ? n : 1; }

inline int drop_xa(int N, int K, const bf16* X, int64_t ldx, const bf16* A, int n, int rank,
                   const int64_t* seed, const DropRates& rates, bf16* XA, int64_t ldo,
                   hipStream_t st) {
  const int rs = rank / 16, na = drop_xa_adapters(n, rs), gy = n / na;
  const int mt = (int64_t)((N + 31) / 32) * gy < 256 ? 1 : 2;
  const dim3 grid((unsigned)((N + 16 * mt - 1) / (16 * mt)), (unsigned)gy);
#define ML_DROP_XA(NA, RS)                                                                       \
  if (na == NA && rs == RS) {                                                                    \
    if (mt == 1)                                                                                 \
      drop_xa_kernel<NA, RS, 1><<<grid, 64 * kXaWaves, 0, st>>>(X, ldx, A, N, K, seed, rates,    \
                                                                XA, ldo);                        \
    else                                                                                         \
      drop_xa_kernel<NA, RS, 2><<<grid, 64 * kXaWaves, 0, st>>>(X, ldx, A, N, K, seed, rates,    \
                                                                XA, ldo);                        \
  }
  ML_DROP_XA(1, 1)
  ML_DROP_XA(1, 2)
  ML_DROP_XA(1, 3)
  ML_DROP_XA(1, 4)
  ML_DROP_XA(2, 1)
  ML_DROP_XA(2, 2)
  ML_DROP_XA(3, 1)
#undef ML_DROP_XA
  ML_LAUNCH_CHECK();
  return ML_OK;
}

// ---------------------------------------------------------------- backward --
// One pass over X and dX that forms each mask once for both of its uses. A wave owns
// `trows` rows of 32 columns and walks them 32 rows at a time; a lane holds 8 columns
// (one counter's block) of the rows lane % 16 and lane % 16 + 16, columns 8 (lane / 16).
//   dX: D = A_i^T P_i^T by 16 x 16 x 16 MFMAs, the A fragments' columns permuted (row m
//       of half h: column 8 (m / 4) + 4 h + m % 4) so that the two halves leave a lane
//       with its own 8 columns of its own row; masked, added in fp32, rounded once.
//   dA: the masked X goes through LDS (2 KB an adapter, the wave's own, so that no
//       barrier is needed) and comes back transposed, P^T beside it; fp32 accumulators
//       over the wave's rows, written to the row tile's partial part[rtile][rank][IN].
// LDS of X: 16-byte chunk q of row r at chunk q ^ (r / 4) % 4; of P: per 16 ranks, 32
// bytes a row, row r at r ^ 4 (r / 8 % 2): every half wave's reads touch all banks once.
constexpr int kDbRows = 32, kDbCols = 32, kDbWaves = 4;

inline int drop_bwd_ctiles(int IN) { return (IN + kDbCols * kDbWaves - 1) / (kDbCols * kDbWaves); }
// Rows per wave: 256, fewer (whole steps) while there are not two workgroups per CU. The
// whole backward, by tiles of 32, 128 and 256 rows: [300, 2048] at two adapters of rank
// 32 58, 60 and 65 us; [8192, 2048] 472, 440 and 432. Between them the partials of the
// smaller tile cost up to 5%: [1777, 2048] 139 (32, what is taken), 134 and 138.
inline int drop_bwd_rows(int N, int IN) {
  int rows = 256;
  while (rows > kDbRows && (int64_t)drop_bwd_ctiles(IN) * ((N + rows - 1) / rows) < 512) rows /= 2;
  return rows;
}
inline size_t drop_bwd_ws_bytes(int N, int RT, int IN) {
  const int rows = drop_bwd_rows(N, IN);
  return (size_t)((N + rows - 1) / rows) * RT * IN * sizeof(float);
}

typedef short i16x8v_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i16x4_t tr_read(const char* p) {
  typedef __attribute__((address_space(3))) i16x4_t* lp;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p);
}

__device__ __forceinline__ bf16x8_t tr_pair(const char* lo, const char* hi) {
  const i16x4_t a = tr_read(lo), b = tr_read(hi);
  return __builtin_bit_cast(bf16x8_t,
                            i16x8v_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

template <int NA, int RS>
__global__ __launch_bounds__(64 * kDbWaves) void drop_bwd_kernel(
    const bf16* __restrict__ X, const bf16* __restrict__ P, const bf16* __restrict__ A, bf16* dX,
    int N, int IN, int trows, const int64_t* seed, const DropRates rates,
    float* __restrict__ part) {
  constexpr int S = NA * RS;                   // 16-rank slices
  constexpr int kXBytes = kDbRows * kDbCols * 2;  // of one adapter's masked X
  constexpr int kPBytes = kDbRows * 32;           // of one slice of P
  constexpr int kWaveBytes = NA * kXBytes + S * kPBytes;
  __shared__ __attribute__((aligned(16))) char lds[kDbWaves * kWaveBytes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ctiles = (IN + kDbCols * kDbWaves - 1) / (kDbCols * kDbWaves);
  const int ct = blockIdx.x % ctiles, rt = blockIdx.x / ctiles;
  const int c0 = (ct * kDbWaves + wave) * kDbCols;
  if (c0 >= IN) return;  // (no barrier below: a wave's LDS is its own)
  const int m0 = rt * trows, m1 = m0 + trows < N ? m0 + trows : N;
  const DropKey key = drop_key(seed);
  char* xl = lds + wave * kWaveBytes;
  char* pl = xl + NA * kXBytes;
  const int lr = lane & 15, lg = lane >> 4;
  const int cc = c0 + 8 * lg;
  const bool okc = cc < IN;  // IN % 8 == 0: a lane's columns are all inside or all outside
  const int ccl = okc ? cc : 0;

  // A fragments of the wave's columns, lane (m = lane % 16, k = 4 (lane / 16) + j): the
  // packed ones (rank = lane % 16, 8 columns) laid down in LDS and read transposed
  i16x4_t af[S][2];
#pragma unroll
  for (int s = 0; s < S; ++s)
    *reinterpret_cast<bf16x8_t*>(pl + s * kPBytes + lr * 64 + lg * 16) =
        frag_of<RS>(A + s / RS * frag_size(16 * RS, IN), c0 / kDbCols, s % RS, lane);
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      af[s][h] = tr_read(pl + s * kPBytes + (4 * lg + (lr >> 2)) * 64 + (lr & 3) * 16 + 8 * h);

  // LDS offsets: this lane's 16 bytes of masked X (rows lr and lr + 16: the same chunk
  // swizzle), the transposing reads of X (two column tiles, two groups of 4 rows) and
  // of P, the rows of P for dX.
  const int xw = lr * 64 + ((lg ^ ((lr >> 2) & 3)) << 4);
  int xr[2][2], pr[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = 8 * lg + 4 * h + (lr >> 2), b = lr & 3;
#pragma unroll
    for (int f = 0; f < 2; ++f)
      xr[f][h] = row * 64 + (((2 * f + (b >> 1)) ^ ((row >> 2) & 3)) << 4) + 8 * (b & 1);
    pr[h] = (row ^ (((row >> 3) & 1) << 2)) * 32 + 8 * b;
  }
  const int pd = (lr ^ (((lr >> 3) & 1) << 2)) * 32 + 8 * lg;  // rows lr; + 512: lr + 16
  // this lane's 16-byte pieces of a step's P rows (2 S pieces a row)
  int prow[S], poff[S], plds[S];
#pragma unroll
  for (int k = 0; k < S; ++k) {
    const int q = lane + 64 * k;
    prow[k] = q / (2 * S);
    const int piece = q % (2 * S);
    poff[k] = piece * 8;
    plds[k] = (piece >> 1) * kPBytes + (prow[k] ^ (((prow[k] >> 3) & 1) << 2)) * 32 +
              (piece & 1) * 16;
  }

  u32x4_t vx[2], vd[2], vp[S];
  auto load_step = [&](int m) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = m + 16 * t + lr < m1 ? m + 16 * t + lr : m1 - 1;
      vx[t] = *reinterpret_cast<const u32x4_t*>(X + (int64_t)row * IN + ccl);
      vd[t] = *reinterpret_cast<const u32x4_t*>(dX + (int64_t)row * IN + ccl);
    }
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int row = m + prow[k] < m1 ? m + prow[k] : m1 - 1;
      vp[k] = *reinterpret_cast<const u32x4_t*>(P + (int64_t)row * (16 * S) + poff[k]);
    }
  };

  f32x4_t acc[S][2];
#pragma unroll
  for (int s = 0; s < S; ++s) acc[s][0] = acc[s][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  load_step(m0);
  for (int m = m0; m < m1; m += kDbRows) {
    u32x4_t x[2], d[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x[t] = keep16(okc && m + 16 * t + lr < m1, vx[t]);
      d[t] = vd[t];
    }
#pragma unroll
    for (int k = 0; k < S; ++k)
      *reinterpret_cast<u32x4_t*>(pl + plds[k]) = keep16(m + prow[k] < m1, vp[k]);
    if (m + kDbRows < m1) load_step(m + kDbRows);
    // dX, and the masked X into LDS
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = m + 16 * t + lr;
      const uint64_t block = (uint64_t)row * (uint64_t)(IN / 8) + (uint64_t)(ccl / 8);
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[2 * e] = __builtin_bit_cast(float, d[t][e] << 16);
        y[2 * e + 1] = __builtin_bit_cast(float, d[t][e] & 0xFFFF0000u);
      }
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const u32x4_t mk = drop_mask(block, rates.stream[i], key, rates.rate[i]);
        *reinterpret_cast<u32x4_t*>(xl + i * kXBytes + xw + t * 1024) = x[t] & mk;
        f32x4_t q[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int r = 0; r < RS; ++r) {
          const i16x4_t pf = *reinterpret_cast<const i16x4_t*>(pl + (i * RS + r) * kPBytes + pd +
                                                               t * 512);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            q[h] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(af[i * RS + r][h], pf, q[h], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = mk[e >> 1];
          const uint32_t keep = (uint32_t)((e & 1) ? (int)w >> 16 : (int)(w << 16) >> 16);
          const float v = q[e >> 2][e & 3];  // (bit_cast of the element itself takes the first)
          y[e] += __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & keep);
        }
      }
      if (okc && row < m1) store_n<bf16, 8>(dX + (int64_t)row * IN + cc, y);
    }
    // dA: tokens as k
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      bf16x8_t bx[2];
#pragma unroll
      for (int f = 0; f < 2; ++f)
        bx[f] = tr_pair(xl + i * kXBytes + xr[f][0], xl + i * kXBytes + xr[f][1]);
#pragma unroll
      for (int r = 0; r < RS; ++r) {
        const char* ps = pl + (i * RS + r) * kPBytes;
        const bf16x8_t a = tr_pair(ps + pr[0], ps + pr[1]);
#pragma unroll
        for (int f = 0; f < 2; ++f)
          acc[i * RS + r][f] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, bx[f], acc[i * RS + r][f], 0, 0, 0);
      }
    }
  }
  // element v of tile (s, f): rank 16 s + 4 (lane / 16) + v, column c0 + 16 f + lane % 16
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int col = c0 + 16 * f + lr;
      if (col < IN)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          part[((int64_t)rt * (16 * S) + 16 * s + 4 * lg + v) * IN + col] = acc[s][f][v];
    }
}

// dX [N, IN] += the adapters' part, dA [n rank, IN] (fp32 or bf16, dense).
template <typename TG>
inline int drop_bwd(int N, int IN, const bf16* X, const bf16* P, const bf16* A, int n, int rank,
                    const int64_t* seed, const DropRates& rates, bf16* dX, TG* dA, char* ws,
                    size_t ws_bytes, hipStream_t st) {
  const int rs = rank / 16, RT = n * rank, rows = drop_bwd_rows(N, IN);
  ML_CHECK(drop_bwd_ws_bytes(N, RT, IN) <= ws_bytes, "lora dropout: workspace too small");
  float* part = reinterpret_cast<float*>(ws);
  const int rtiles = (N + rows - 1) / rows;
  const dim3 grid((unsigned)(drop_bwd_ctiles(IN) * rtiles));
#define ML_DROP_BWD(NA, RS)                                                                 \
  if (n == NA && rs == RS)                                                                  \
    drop_bwd_kernel<NA, RS><<<grid, 64 * kDbWaves, 0, st>>>(X, P, A, dX, N, IN, rows, seed, \
                                                            rates, part);
#define ML_DROP_BWD4(NA) ML_DROP_BWD(NA, 1) ML_DROP_BWD(NA, 2) ML_DROP_BWD(NA, 3) ML_DROP_BWD(NA, 4)
  ML_DROP_BWD4(1)
  ML_DROP_BWD4(2)
  ML_DROP_BWD4(3)
#undef ML_DROP_BWD4
#undef ML_DROP_BWD
  ML_LAUNCH_CHECK();
  reduce_partials_kernel<TG><<<dim3(256), 256, 0, st>>>(part, rtiles, RT, IN, dA, IN, 1.0f, 0.f);
  ML_LAUNCH_CHECK();
  return ML_OK;
}
