// Row-wise steps of the feed-forward operators: what happens between their products,
// on VEC neighbouring columns of a row at a time (8, as 16-byte accesses of 16-bit
// elements; 1 where sizes, strides or bases rule those out). 32 / VEC neighbouring
// lanes hold a block of 32 columns, so that a step can keep a tensor in 8 bits
// (held8.h). The same steps run in a product's epilogue and over arrays in memory.
#pragma once

#include "act_math.h"
#include "held8.h"

namespace mla {
namespace ffn {

enum : int { kKeepNone = 0, kKeepSame = 1, kKeepFp8 = 2 };

// A [rows, cols] tensor kept for the backward, dense: in T, or its bytes with
// ceil(cols / 32) scale bytes a row.
template <typename T>
struct Kept {
  int kind;
  T* v;
  uint8_t* q;
  uint8_t* scale;
  int64_t cols, nblocks;

  // every lane of a block takes part; live: this lane's columns exist
  template <int VEC>
  __device__ __forceinline__ void put(int64_t m, int64_t n, const float (&x)[VEC],
                                      bool live) const {
    if (kind == kKeepSame) {
      if (live) store_n<T, VEC>(v + m * cols + n, x);
    } else if (kind == kKeepFp8) {
      const uint32_t b = held8::block_byte<VEC>(x);
      if (live) {
        held8::store<VEC>(q + m * cols + n, b, x);
        if (n % held8::kBlock == 0) scale[m * nblocks + n / held8::kBlock] = (uint8_t)b;
      }
    }
  }

  template <int VEC>
  __device__ __forceinline__ void get(int64_t m, int64_t n, float (&x)[VEC]) const {
    if (kind == kKeepSame)
      load_n<T, VEC>(v + m * cols + n, x);
    else
      held8::load<VEC>(q + m * cols + n, scale[m * nblocks + n / held8::kBlock], x);
  }
};

template <typename T>
inline Kept<T> make_kept(int kind, const void* v, const void* scale, int64_t cols) {
  Kept<T> k{};
  k.kind = v ? kind : kKeepNone;
  k.v = kind == kKeepSame ? static_cast<T*>(const_cast<void*>(v)) : nullptr;
  k.q = kind == kKeepFp8 ? static_cast<uint8_t*>(const_cast<void*>(v)) : nullptr;
  k.scale = static_cast<uint8_t*>(const_cast<void*>(scale));
  k.cols = cols;
  k.nblocks = held8::blocks(cols);
  return k;
}

template <int VEC>
__device__ __forceinline__ void act_fwd_vec(int act, float (&x)[VEC]) {
  switch (act) {  // uniform
    case kActSilu:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = act_fwd<kActSilu>(x[k]);
      break;
    case kActGelu:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = act_fwd<kActGelu>(x[k]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = act_fwd<kActGeluTanh>(x[k]);
      break;
    default: break;
  }
}

template <int VEC>
__device__ __forceinline__ void act_grad_vec(int act, float (&x)[VEC]) {
  switch (act) {
    case kActSilu:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = act_grad<kActSilu>(x[k]);
      break;
    case kActGelu:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = act_grad<kActGelu>(x[k]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = act_grad<kActGeluTanh>(x[k]);
      break;
    default:
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = 1.f;
  }
}

// z = x + bias; y = act(z) + residual; z kept.
template <typename T>
struct LinearStep {
  const T* bias;      // or null
  const T* residual;  // or null
  T* y;
  int64_t ldr, ldy;
  int act;
  Kept<T> z;

  template <int VEC>
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, float (&x)[VEC],
                                             bool live) const {
    if (bias && live) {
      float b[VEC];
      load_n<T, VEC>(bias + n, b);
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] += b[k];
    }
    z.template put<VEC>(m, n, x, live);
    if (!live) return;
    act_fwd_vec<VEC>(act, x);
    if (residual) {
      float r[VEC];
      load_n<T, VEC>(residual + m * ldr + n, r);
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] += r[k];
    }
    store_n<T, VEC>(y + m * ldy + n, x);
  }
};

// h = silu(g) u; g and u kept.
template <typename T>
struct GatedStep {
  T* h;  // dense
  int64_t cols;
  Kept<T> gate, up;

  template <int VEC>
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, float (&g)[VEC],
                                             float (&u)[VEC], bool live) const {
    gate.template put<VEC>(m, n, g, live);
    up.template put<VEC>(m, n, u, live);
    if (!live) return;
#pragma unroll
    for (int k = 0; k < VEC; ++k) g[k] = swiglu_fwd_elem(g[k], u[k]);
    store_n<T, VEC>(h + m * cols + n, g);
  }
};

// dg, du and (h not null) h again from dh and the kept g, u.
template <typename T>
struct GatedGradStep {
  T* dg;
  T* du;
  T* h;  // or null
  int64_t cols;
  Kept<T> gate, up;

  template <int VEC>
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, float (&dh)[VEC],
                                             bool live) const {
    if (!live) return;
    float g[VEC], u[VEC], hv[VEC];
    gate.template get<VEC>(m, n, g);
    up.template get<VEC>(m, n, u);
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      swiglu_bwd_fwd_elem(g[k], u[k], dh[k], g[k], u[k], hv[k]);
    store_n<T, VEC>(dg + m * cols + n, g);
    store_n<T, VEC>(du + m * cols + n, u);
    if (h) store_n<T, VEC>(h + m * cols + n, hv);
  }
};

// ------------------------------------------------------- over arrays in memory --

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
struct TypedSource {
  const T* p;
  int64_t ld;

  template <int VEC>
  __device__ __forceinline__ void load(int64_t m, int64_t n, float (&x)[VEC]) const {
    load_n<T, VEC>(p + m * ld + n, x);
  }
};

constexpr int kThreads = 256;

// One or two sources (Src2 void: one) through a step, a block of 32 columns by 32 / VEC
// lanes at a time.
struct NoSource {};

template <int VEC, class Src, class Src2, class Step>
__global__ __launch_bounds__(kThreads) void rows_kernel(const Src src, const Src2 src2,
                                                        const Step step, int64_t rows,
                                                        int64_t cols) {
  constexpr int L = held8::kBlock / VEC;
  const int64_t nb = (cols + held8::kBlock - 1) / held8::kBlock;
  const int64_t groups = rows * nb;
  const int64_t step_groups = (int64_t)gridDim.x * (kThreads / L);
  const int l = threadIdx.x % L;
  for (int64_t g = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L; g < groups;
       g += step_groups) {
    const int64_t m = rows == 1 ? 0 : g / nb;
    const int64_t n = (g - m * nb) * held8::kBlock + l * VEC;
    const bool live = n < cols;
    float x[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = 0.f;
    if (live) src.template load<VEC>(m, n, x);
    if constexpr (std::is_same_v<Src2, NoSource>) {
      step.template operator()<VEC>(m, n, x, live);
    } else {
      float u[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) u[k] = 0.f;
      if (live) src2.template load<VEC>(m, n, u);
      step.template operator()<VEC>(m, n, x, u, live);
    }
  }
}

template <class Src, class Src2, class Step>
inline int launch_rows(bool vec, const Src& src, const Src2& src2, const Step& step, int64_t rows,
                       int64_t cols, hipStream_t st) {
  if (rows == 0 || cols == 0) return ML_OK;
  const int64_t groups = rows * held8::blocks(cols);
  const int per = kThreads / (held8::kBlock / (vec ? 8 : 1));
  int64_t blocks = (groups + per - 1) / per;
  blocks = blocks < (1 << 20) ? blocks : (1 << 20);
  if (vec)
    rows_kernel<8, Src, Src2, Step><<<dim3((unsigned)blocks), kThreads, 0, st>>>(src, src2, step,
                                                                                 rows, cols);
  else
    rows_kernel<1, Src, Src2, Step><<<dim3((unsigned)blocks), kThreads, 0, st>>>(src, src2, step,
                                                                                 rows, cols);
  ML_LAUNCH_CHECK();
  return ML_OK;
}

// ------------------------------------------- the linear layer's backward step --
// dz = dy act'(z) (dz null: not written, as where there is no activation) and the
// column sums of dz: a workgroup takes 32 VEC columns and a range of rows, its 8
// row lanes' sums are joined in LDS, and the ranges' partial rows are summed in
// their order by a second kernel. fp32 sums; dz is summed as it was before its
// rounding.
template <int VEC, typename T>
__global__ __launch_bounds__(kThreads) void linear_grad_kernel(
    const T* __restrict__ dy, int64_t ldy, const Kept<T> z, int act, T* __restrict__ dz,
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
    for (int64_t m = r0 + rl; m < r1; m += 8) {
      float d[VEC];
      load_n<T, VEC>(dy + m * ldy + n, d);
      if (act != kActNone) {
        float v[VEC];
        z.template get<VEC>(m, n, v);
        act_grad_vec<VEC>(act, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[k] *= v[k];
      }
      if (dz) store_n<T, VEC>(dz + m * cols + n, d);
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] += d[k];
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

template <typename T>
__global__ __launch_bounds__(kThreads) void column_sum_kernel(const float* __restrict__ partial,
                                                              int parts, int64_t cols,
                                                              T* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int p = 0; p < parts; ++p) s += partial[(int64_t)p * cols + c];
  out[c] = from_f32<T>(s);
}

}  // namespace ffn
}  // namespace mla
