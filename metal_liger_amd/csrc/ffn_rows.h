// Row-wise steps of the feed-forward operators: what happens between their products,
// on VEC neighbouring columns of a row at a time (8, as 16-byte accesses of 16-bit
// elements; 1 where sizes, strides or bases rule those out). 32 / VEC neighbouring
// lanes hold a block of 32 columns, so that a step can keep a tensor in 8 bits
// (held.h). The same steps run in a product's epilogue and over arrays in memory.
#pragma once

#include "act_math.h"
#include "held.h"

namespace mla {
namespace ffn {

enum : int { kKeepNone = ML_KEEP_NONE, kKeepF32 = ML_KEEP_F32, kKeepFp16 = ML_KEEP_FP16,
             kKeepFp8 = ML_KEEP_FP8 };

// A [rows, cols] tensor kept for the backward, dense: in fp32, or in 16 or 8 bits an
// element with ceil(cols / 32) scale bytes a row (held.h); or not at all. (KIND is a
// template parameter so that fetch's loads stand in no branch.)
template <int KIND>
struct Kept {
  using Elem = std::conditional_t<KIND == kKeepF32, float,
                                  std::conditional_t<KIND == kKeepFp16, f16, uint8_t>>;
  Elem* v;
  uint8_t* scale;
  int64_t cols, nblocks;

  // B positions (rows m[q], columns n on); every lane of a block takes part; live[q]:
  // this lane's position exists (ALL: every one does).
  template <bool ALL, int VEC, int B>
  __device__ __forceinline__ void put(const int64_t (&m)[B], int64_t n, const float (&x)[B][VEC],
                                      const bool (&live)[B]) const {
    if constexpr (KIND == kKeepF32) {
#pragma unroll
      for (int q = 0; q < B; ++q)
        if (ALL || live[q]) store_n<float, VEC>(v + m[q] * cols + n, x[q]);
    } else if constexpr (KIND != kKeepNone) {
      // (a block's columns past the tensor's do not count for its scale)
      float w[B][VEC];
#pragma unroll
      for (int q = 0; q < B; ++q)
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[q][k] = ALL || live[q] ? x[q][k] : 0.f;
      const held::Scales<B> s =
          held::block_scales<KIND == kKeepFp16 ? held::kTop16 : held::kTop8, VEC, B>(w);
#pragma unroll
      for (int q = 0; q < B; ++q) {
        const float inv = held::inverse_of(s.byte[q]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[q][k] = x[q][k] * inv;
      }
      if (KIND == kKeepFp8 && !s.finite) {
#pragma unroll
        for (int q = 0; q < B; ++q)
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            w[q][k] = held::finite_or_nan(x[q][k]) * held::inverse_of(s.byte[q]);
      }
      const int64_t block = n / held::kBlock;
      const bool first = n % held::kBlock == 0;
#pragma unroll
      for (int q = 0; q < B; ++q) {
        if (!(ALL || live[q])) continue;
        if constexpr (KIND == kKeepFp16)
          store_n<f16, VEC>(v + m[q] * cols + n, w[q]);
        else
          held::store<VEC>(v + m[q] * cols + n, w[q]);
      }
      if (first) {
#pragma unroll
        for (int q = 0; q < B; ++q)
          if (ALL || live[q]) scale[m[q] * nblocks + block] = (uint8_t)s.byte[q];
      }
    }
  }

  // Bits of VEC elements as they lie in memory, and their scale's byte: fetched
  // first, decoded when they are needed, so that several are in flight.
  template <int VEC>
  struct Raw {
    uint32_t w[(VEC * sizeof(Elem) + 3) / 4];
    uint32_t byte;
  };

  template <int VEC>
  __device__ __forceinline__ Raw<VEC> fetch(int64_t m, int64_t n) const {
    Raw<VEC> r;
    constexpr int N = VEC * (int)sizeof(Elem);
    const Elem* p = v + m * cols + n;
    if constexpr (N < 4)
      r.w[0] = N == 1 ? *reinterpret_cast<const uint8_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
    else
      __builtin_memcpy(r.w, __builtin_assume_aligned(p, N < 16 ? N : 16), N);
    r.byte = KIND == kKeepF32 ? 0 : scale[m * nblocks + n / held::kBlock];
    return r;
  }

  template <int VEC>
  __device__ __forceinline__ void decode(const Raw<VEC>& r, float (&x)[VEC]) const {
    if constexpr (KIND == kKeepF32)
      __builtin_memcpy(x, r.w, sizeof(x));
    else if constexpr (KIND == kKeepFp16)
      held::load16<VEC>(r.w, r.byte, x);
    else
      held::load<VEC>(r.w, r.byte, x);
  }
};

template <int KIND>
inline Kept<KIND> make_kept(const void* v, const void* scale, int64_t cols) {
  return Kept<KIND>{static_cast<typename Kept<KIND>::Elem*>(const_cast<void*>(v)),
                    static_cast<uint8_t*>(const_cast<void*>(scale)), cols, held::blocks(cols)};
}

// VEC elements of T as they are (16-byte transactions where that is their size or more).
template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, Pack<T, VEC>& r) {
  constexpr int P = VEC * (int)sizeof(T) >= 16 ? 16 / (int)sizeof(T) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += P) {
    const Pack<T, P> q = *reinterpret_cast<const Pack<T, P>*>(p + i);
#pragma unroll
    for (int k = 0; k < P; ++k) r.v[i + k] = q.v[k];
  }
}

template <int ACT, int VEC, int B>
__device__ __forceinline__ void act_fwd_all(float (&x)[B][VEC]) {
#pragma unroll
  for (int q = 0; q < B; ++q)
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[q][k] = act_fwd<ACT>(x[q][k]);
}

template <int VEC, int B>
__device__ __forceinline__ void act_fwd_vec(int act, float (&x)[B][VEC]) {
  switch (act) {  // uniform
    case kActSilu: act_fwd_all<kActSilu>(x); break;
    case kActGelu: act_fwd_all<kActGelu>(x); break;
    case kActGeluTanh: act_fwd_all<kActGeluTanh>(x); break;
    default: break;
  }
}

template <int ACT, int VEC, int B>
__device__ __forceinline__ void act_grad_all(float (&x)[B][VEC]) {
#pragma unroll
  for (int q = 0; q < B; ++q)
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[q][k] = act_grad<ACT>(x[q][k]);
}

template <int VEC, int B>
__device__ __forceinline__ void act_grad_vec(int act, float (&x)[B][VEC]) {
  switch (act) {
    case kActSilu: act_grad_all<kActSilu>(x); break;
    case kActGelu: act_grad_all<kActGelu>(x); break;
    default: act_grad_all<kActGeluTanh>(x); break;
  }
}

// A step: column(n) gives what it needs of a lane's columns, fetch(m, n) issues its
// loads for a position, and finish(...) does the work for B positions of these columns
// at once: straight through, so that a wave on its own has B chains of operations to
// hide latencies in. Every lane of a block takes part in finish; live says whether a
// lane's position exists (ALL: every one does), else what column and fetch gave of it is
// not used.

// data (of the steps whose outputs a product or a backward reads): columns from it on are
// padding beside the operands' own and are written as zeros. The sums there are zeros
// already, unless an infinity met a padded zero: that NaN would reach every column of the
// next product.
template <int VEC, int B>
__device__ __forceinline__ void zero_padding(int64_t n, int64_t data, float (&x)[B][VEC]) {
  if (n + VEC <= data) return;
#pragma unroll
  for (int q = 0; q < B; ++q)
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[q][k] = n + k < data ? x[q][k] : 0.f;
}

// cost: which of the times measured with products it goes by (ffn_product.h).
enum : int { kPlainStep, kActStep, kPairStep, kGradStep };

// z = x + bias; y = act(z) + residual; z kept.
template <typename T, int KIND>
struct LinearStep {
  const T* bias;      // or null
  const T* residual;  // or null
  T* y;
  int64_t ldr, ldy;
  int act;
  Kept<KIND> z;
  int64_t data = INT64_MAX;

  int cost() const { return act == kActNone && KIND == kKeepNone ? kPlainStep : kActStep; }

  template <int VEC>
  struct Column {
    float b[VEC];
  };
  template <int VEC>
  struct Fetched {
    Pack<T, VEC> r;
  };

  template <int VEC>
  __device__ __forceinline__ Column<VEC> column(int64_t n) const {
    Column<VEC> c;
    if (bias) {
      load_n<T, VEC>(bias + n, c.b);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) c.b[k] = 0.f;
    }
    return c;
  }

  template <int VEC>
  __device__ __forceinline__ Fetched<VEC> fetch(int64_t m, int64_t n) const {
    Fetched<VEC> f;
    if (residual) load_pack<T, VEC>(residual + m * ldr + n, f.r);
    return f;
  }

  template <bool ALL, int VEC, int B>
  __device__ __forceinline__ void finish(const int64_t (&m)[B], int64_t n, float (&x)[B][VEC],
                                         const Column<VEC>& c, const Fetched<VEC> (&f)[B],
                                         const bool (&live)[B]) const {
#pragma unroll
    for (int q = 0; q < B; ++q)
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[q][k] += c.b[k];
    if constexpr (KIND != kKeepNone) zero_padding<VEC, B>(n, data, x);
    z.template put<ALL, VEC, B>(m, n, x, live);
    act_fwd_vec<VEC, B>(act, x);
    if (residual) {
#pragma unroll
      for (int q = 0; q < B; ++q)
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[q][k] += to_f32(f[q].r.v[k]);
    }
#pragma unroll
    for (int q = 0; q < B; ++q)
      if (ALL || live[q]) store_n<T, VEC>(y + m[q] * ldy + n, x[q]);
  }
};

// h = silu(g) u; g and u kept.
template <typename T, int KIND>
struct GatedStep {
  T* h;  // dense
  int64_t cols;
  Kept<KIND> gate, up;
  int64_t data = INT64_MAX;

  int cost() const { return kPairStep; }

  template <int VEC>
  struct Column {};
  template <int VEC>
  struct Fetched {};

  template <int VEC>
  __device__ __forceinline__ Column<VEC> column(int64_t) const { return {}; }
  template <int VEC>
  __device__ __forceinline__ Fetched<VEC> fetch(int64_t, int64_t) const { return {}; }

  template <bool ALL, int VEC, int B>
  __device__ __forceinline__ void finish(const int64_t (&m)[B], int64_t n, float (&g)[B][VEC],
                                         float (&u)[B][VEC], const Column<VEC>&,
                                         const Fetched<VEC> (&)[B], const bool (&live)[B]) const {
    zero_padding<VEC, B>(n, data, g);
    zero_padding<VEC, B>(n, data, u);
    gate.template put<ALL, VEC, B>(m, n, g, live);
    up.template put<ALL, VEC, B>(m, n, u, live);
#pragma unroll
    for (int q = 0; q < B; ++q)
#pragma unroll
      for (int k = 0; k < VEC; ++k) g[q][k] = swiglu_fwd_elem(g[q][k], u[q][k]);
#pragma unroll
    for (int q = 0; q < B; ++q)
      if (ALL || live[q]) store_n<T, VEC>(h + m[q] * cols + n, g[q]);
  }
};

// dg, du and (h not null) h again from dh and the kept g, u.
template <typename T, int KIND>
struct GatedGradStep {
  T* dg;
  T* du;
  T* h;  // or null
  int64_t cols;
  Kept<KIND> gate, up;
  int64_t data = INT64_MAX;

  int cost() const { return kGradStep; }

  template <int VEC>
  struct Column {};
  template <int VEC>
  struct Fetched {
    typename Kept<KIND>::template Raw<VEC> g, u;
  };

  template <int VEC>
  __device__ __forceinline__ Column<VEC> column(int64_t) const { return {}; }
  template <int VEC>
  __device__ __forceinline__ Fetched<VEC> fetch(int64_t m, int64_t n) const {
    return {gate.template fetch<VEC>(m, n), up.template fetch<VEC>(m, n)};
  }

  template <bool ALL, int VEC, int B>
  __device__ __forceinline__ void finish(const int64_t (&m)[B], int64_t n, float (&dh)[B][VEC],
                                         const Column<VEC>&, const Fetched<VEC> (&f)[B],
                                         const bool (&live)[B]) const {
    float g[B][VEC], u[B][VEC];
    zero_padding<VEC, B>(n, data, dh);  // (g and u were kept as zeros there)
#pragma unroll
    for (int q = 0; q < B; ++q) {
      gate.template decode<VEC>(f[q].g, g[q]);
      up.template decode<VEC>(f[q].u, u[q]);
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        swiglu_bwd_fwd_elem(g[q][k], u[q][k], dh[q][k], g[q][k], u[q][k], dh[q][k]);
    }
#pragma unroll
    for (int q = 0; q < B; ++q) {
      if (!(ALL || live[q])) continue;
      store_n<T, VEC>(dg + m[q] * cols + n, g[q]);
      store_n<T, VEC>(du + m[q] * cols + n, u[q]);
      if (h) store_n<T, VEC>(h + m[q] * cols + n, dh[q]);
    }
  }
};

// What a kept tensor stands for.
template <typename T, int KIND>
struct ValuesStep {
  T* out;  // dense
  int64_t cols;
  Kept<KIND> v;

  template <int VEC>
  struct Column {};
  template <int VEC>
  using Fetched = typename Kept<KIND>::template Raw<VEC>;

  template <int VEC>
  __device__ __forceinline__ Column<VEC> column(int64_t) const { return {}; }
  template <int VEC>
  __device__ __forceinline__ Fetched<VEC> fetch(int64_t m, int64_t n) const {
    return v.template fetch<VEC>(m, n);
  }

  template <bool ALL, int VEC, int B>
  __device__ __forceinline__ void finish(const int64_t (&m)[B], int64_t n, float (&x)[B][VEC],
                                         const Column<VEC>&, const Fetched<VEC> (&f)[B],
                                         const bool (&live)[B]) const {
#pragma unroll
    for (int q = 0; q < B; ++q) {
      v.template decode<VEC>(f[q], x[q]);
      if (ALL || live[q]) store_n<T, VEC>(out + m[q] * cols + n, x[q]);
    }
  }
};

// ------------------------------------------------------- over arrays in memory --

struct ZeroSource {  // of a step that reads all by itself
  template <int VEC>
  __device__ __forceinline__ void load(int64_t, int64_t, float (&x)[VEC]) const {
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = 0.f;
  }
};

// The sum of S fp32 partials [S][rows][ld], in their order.
struct PartialSource {
  const float* p;
  int splits;
  int64_t stride, ld;

  template <int VEC>
  __device__ __forceinline__ void load(int64_t m, int64_t n, float (&x)[VEC]) const {
    const float* q = p + m * ld + n;
    load_n<float, VEC>(q, x);
    for (int s = 1; s < splits; ++s) {
      float v[VEC];
      load_n<float, VEC>(q + s * stride, v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] += v[k];
    }
  }
};

template <typename T>
struct TypedSource {  // read once
  const T* p;
  int64_t ld;

  template <int VEC>
  __device__ __forceinline__ void load(int64_t m, int64_t n, float (&x)[VEC]) const {
    load_n_nt<T, VEC>(p + m * ld + n, x);
  }
};

constexpr int kThreads = 256;

// One or two sources through a step, a block of 32 columns by 32 / VEC lanes at a time.
// A thread issues the loads of kInFlight positions before it works on the first. The
// index arithmetic is 32-bit where the blocks can be counted in 32 bits (a 64-bit
// division costs more than the rest of a step).
struct NoSource {};
constexpr int kInFlight = 2;

template <int VEC, class Src, class Src2, class Step, typename Index>
__global__ __launch_bounds__(kThreads) void rows_kernel(const Src src, const Src2 src2,
                                                        const Step step, Index rows, int64_t cols,
                                                        Index nb) {
  constexpr int L = held::kBlock / VEC;
  constexpr bool kTwo = !std::is_same_v<Src2, NoSource>;
  const Index groups = rows * nb;
  const Index stride = (Index)gridDim.x * (kThreads / L) * kInFlight;
  const int l = threadIdx.x % L;
  for (Index g0 = (Index)blockIdx.x * (kThreads / L) * kInFlight + threadIdx.x / L; g0 < groups;
       g0 += stride) {
    int64_t m[kInFlight], n[kInFlight];
    bool live[kInFlight];
    float x[kInFlight][VEC], u[kInFlight][VEC];
    typename Step::template Column<VEC> c[kInFlight];
    typename Step::template Fetched<VEC> f[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      // (positions past the last block fetch the last one's; they are not live)
      const Index at = g0 + k * (kThreads / L);
      const Index g = at < groups ? at : groups - 1;
      const Index row = rows == 1 ? 0 : g / nb;
      m[k] = row;
      n[k] = (int64_t)(g - row * nb) * held::kBlock + l * VEC;
      live[k] = n[k] < cols;
      const int64_t nc = live[k] ? n[k] : 0;
      src.template load<VEC>(m[k], nc, x[k]);
      if constexpr (kTwo) src2.template load<VEC>(m[k], nc, u[k]);
      c[k] = step.template column<VEC>(nc);
      f[k] = step.template fetch<VEC>(m[k], nc);
      if (!live[k]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[k][e] = u[k][e] = 0.f;
      }
      live[k] = live[k] && at < groups;
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const int64_t mk[1] = {m[k]};
      const bool lk[1] = {live[k]};
      float(&xk)[1][VEC] = reinterpret_cast<float(&)[1][VEC]>(x[k]);
      typename Step::template Fetched<VEC> fk[1] = {f[k]};
      if constexpr (kTwo)
        step.template finish<false, VEC, 1>(mk, n[k], xk, reinterpret_cast<float(&)[1][VEC]>(u[k]),
                                            c[k], fk, lk);
      else
        step.template finish<false, VEC, 1>(mk, n[k], xk, c[k], fk, lk);
    }
  }
}

template <int VEC, class Src, class Src2, class Step>
inline void rows_launch(const Src& src, const Src2& src2, const Step& step, int64_t rows,
                        int64_t cols, hipStream_t st) {
  const int64_t nb = held::blocks(cols), groups = rows * nb;
  const int per = kThreads / (held::kBlock / VEC) * kInFlight;
  int64_t blocks = (groups + per - 1) / per;
  blocks = blocks < (1 << 20) ? blocks : (1 << 20);
  // (the last stride must not wrap)
  if (groups + blocks * per < (1LL << 32))
    rows_kernel<VEC, Src, Src2, Step, uint32_t><<<dim3((unsigned)blocks), kThreads, 0, st>>>(
        src, src2, step, (uint32_t)rows, cols, (uint32_t)nb);
  else
    rows_kernel<VEC, Src, Src2, Step, int64_t><<<dim3((unsigned)blocks), kThreads, 0, st>>>(
        src, src2, step, rows, cols, nb);
}

template <class Src, class Src2, class Step>
inline int launch_rows(bool vec, const Src& src, const Src2& src2, const Step& step, int64_t rows,
                       int64_t cols, hipStream_t st) {
  if (rows == 0 || cols == 0) return ML_OK;
  if (vec)
    rows_launch<8>(src, src2, step, rows, cols, st);
  else
    rows_launch<1>(src, src2, step, rows, cols, st);
  ML_LAUNCH_CHECK();
  return ML_OK;
}

// ------------------------------------------- the linear layer's backward step --
// dz = dy act'(z) (KIND none: dy, where there is no activation; dz null: not written) and the
// column sums of dz: a workgroup takes 32 VEC columns and a range of rows, its 8
// row lanes' sums are joined in LDS, and the ranges' partial rows are summed in
// their order by a second kernel. fp32 sums; dz is summed as it was before its
// rounding.
template <int VEC, typename T, typename TZ, int KIND>
__global__ __launch_bounds__(kThreads) void linear_grad_kernel(
    const T* __restrict__ dy, int64_t ldy, const Kept<KIND> z, int act, TZ* __restrict__ dz,
    float* __restrict__ partial, int64_t rows, int64_t cols, int64_t rows_per) {
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int64_t n = ((int64_t)blockIdx.x * 32 + cl) * VEC;
  const bool live = n < cols;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per;
  const int64_t r1 = r0 + rows_per < rows ? r0 + rows_per : rows;
  float sum[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
  if (live) {
    constexpr int B = VEC == 8 && sizeof(T) == 2 ? 4 : 2;  // rows of a lane in flight
    for (int64_t m0 = r0 + rl; m0 < r1; m0 += 8 * B) {
      float d[B][VEC], v[B][VEC];
      typename Kept<KIND>::template Raw<VEC> raw[B];
#pragma unroll
      for (int q = 0; q < B; ++q) {  // (rows past the range: the first one's again)
        const int64_t m = m0 + 8 * q < r1 ? m0 + 8 * q : m0;
        load_n_nt<T, VEC>(dy + m * ldy + n, d[q]);
        if constexpr (KIND != kKeepNone) raw[q] = z.template fetch<VEC>(m, n);
      }
      if constexpr (KIND != kKeepNone) {
#pragma unroll
        for (int q = 0; q < B; ++q) z.template decode<VEC>(raw[q], v[q]);
        act_grad_vec<VEC, B>(act, v);
      }
#pragma unroll
      for (int q = 0; q < B; ++q) {
        if (m0 + 8 * q >= r1) break;
        if constexpr (KIND != kKeepNone) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) d[q][k] *= v[q][k];
        }
        if (dz) store_n<TZ, VEC>(dz + (m0 + 8 * q) * cols + n, d[q]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += d[q][k];
      }
    }
  }
  if (!partial) return;
  __shared__ float lds[8][32 * VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) lds[rl][cl * VEC + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * VEC; c += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) s += lds[r][c];
    const int64_t col = (int64_t)blockIdx.x * 32 * VEC + c;
    if (col < cols) partial[(int64_t)blockIdx.y * cols + col] = s;
  }
}

// A workgroup sums 32 columns: 8 lanes a column take every eighth partial row each, and
// are joined in order. (One thread a column, 205 rows of 1152 columns: 48 us.)
template <typename T>
__global__ __launch_bounds__(kThreads) void column_sum_kernel(const float* __restrict__ partial,
                                                              int parts, int64_t cols,
                                                              T* __restrict__ out) {
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + cl;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int p = rl; p < parts; p += 8) s += partial[(int64_t)p * cols + c];
  }
  __shared__ float lds[8][32];
  lds[rl][cl] = s;
  __syncthreads();
  if (rl || c >= cols) return;
#pragma unroll
  for (int r = 1; r < 8; ++r) s += lds[r][cl];
  out[c] = from_f32<T>(s);
}

}  // namespace ffn
}  // namespace mla
