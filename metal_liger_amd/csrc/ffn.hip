// The feed-forward operators: a linear layer with bias, activation and residual in its
// epilogue, the gated block (both projections, SiLU, the product, the projection
// back), SwiGLU with its inputs kept in 8 bits; forward and backward. The mathematics
// of the steps between the products is in ffn_rows.h, the 8 bits in held.h.
//
//   linear  z = x W^T + b, y = act(z) + residual
//           dz = dy act'(z), dx = dz W, dW = dz^T x, db = column sums of dz
//   gated   g = x Wg^T, u = x Wu^T, h = silu(g) u, y = h Wd^T + residual
//           dh = dy Wd, dg = dh u silu'(g), du = dh silu(g),
//           dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// bf16 runs on the bf16 matrix cores (gemm_core.h), fp32 and fp16 on the fp32 ones
// (ffn_f32.h; what lies between fp16's products is fp32); forwards of few rows (up to
// 128) on kernels of their own (ffn_skinny.h), where products of two fp16 operands run on
// the fp16 matrix cores.
#include <initializer_list>

#include "ffn_f32.h"
#include "ffn_pad.h"
#include "ffn_product.h"
#include "ffn_skinny.h"
#include "ffn_wgrad.h"
#include "gemm_f32.h"

namespace mla {
namespace ffn {
namespace {

using gemm::kKMajor;
using gemm::kMNMajor;

// A workspace taken apart front to back; with a null base it only counts.
struct Arena {
  char* base;
  size_t used = 0;

  template <typename P>
  P* take(size_t n) {
    used = (used + 255) / 256 * 256;
    P* p = base ? reinterpret_cast<P*>(base + used) : nullptr;
    used += n * sizeof(P);
    return p;
  }
};

size_t larger(size_t a, size_t b) { return a > b ? a : b; }

bool aligned_rows(const void* p, int64_t ld) { return !p || (aligned16(p) && ld % 8 == 0); }

// A tile's rows are addressed by 32-bit offsets: at most 256 rows of bf16 or 128 of fp32.
constexpr int64_t kMaxStride = 1 << 21;

struct Checked {
  const void* p;
  int64_t ld, cols;
  const char* what;
};

// 16-bit operands of a product and its step.
int check_operands(std::initializer_list<Checked> list) {
  for (const Checked& c : list)
    ML_CHECK(aligned16(c.p) && c.ld % 8 == 0 && c.cols % 8 == 0 && c.ld <= kMaxStride,
             "ffn: 16-bit %s needs a 16-byte aligned base, and columns and row stride in multiples "
             "of 8, up to %lld (%lld, %lld)", c.what, (long long)kMaxStride, (long long)c.cols,
             (long long)c.ld);
  return ML_OK;
}

int ktiles(int64_t k) { return (int)((k + gemm::kBK - 1) / gemm::kBK); }

// What lies between two products: bf16 as it is, fp32 for fp32 and fp16 (whose range h
// and the gradients of gate, up and z may leave).
template <typename T>
using Inner = std::conditional_t<std::is_same_v<T, bf16>, bf16, float>;

// A weight's gradient C = A^T B, A [K, M], B [K, N]; either may be of the inner type.
struct Wgrad {
  int64_t M, N;
  const void *a, *b;
  int64_t lda, ldb;
  void* c;  // dense
  bool a_inner, b_inner;
};

// The products of each type.
//   raw:     fp32 sums [splits][M][N] of A B^T (B [N, K]) or A B (LB kMNMajor: B [K, N])
//   store:   sum over segments of A_s B_s (B [K_s, N]), rounded to T
//   wgrads:  A^T B of up to three products of one K, rounded to T
// and, where K is not split, a product with its step as its epilogue:
//   through, through_pair
template <typename T>
struct Products;

template <>
struct Products<bf16> {
  static gemm::Plan plan(int64_t M, int64_t N, int64_t K) {
    const int m = (int)M, n = (int)N, kt = ktiles(K);
    return gemm::plan_products(1, &m, &n, &kt, true);
  }

  static size_t raw_floats(int64_t M, int64_t N, int64_t K) {
    return (size_t)plan(M, N, K).ksplit * M * N;
  }

  template <class CF, int LB>
  static int raw_cfg(int64_t M, int64_t N, const gemm::Segment& s, int ksplit, float* out,
                     int& splits, hipStream_t st) {
    gemm::Problem pb;
    const int rc = gemm::make_problem<CF>(pb, (int)M, (int)N, 1, &s, kKMajor, LB, 0, ksplit);
    if (rc) return rc;
    splits = pb.ksplit;
    gemm::gemm_kernel<CF, kKMajor, LB, gemm::EpiPartial>
        <<<dim3(gemm::grid_blocks(pb)), CF::THREADS, 0, st>>>(pb, gemm::EpiPartial{out, pb.M, pb.N});
    ML_LAUNCH_CHECK();
    return ML_OK;
  }

  template <int LB>
  static int raw(int64_t M, int64_t N, int64_t K, const bf16* a, int64_t lda, const bf16* b,
                 int64_t ldb, float* out, int& splits, hipStream_t st) {
    const gemm::Segment s{{a, lda}, {b, ldb}, (int)K};
    const gemm::Plan p = plan(M, N, K);
    return p.tile == 128 ? raw_cfg<gemm::R4SCfg, LB>(M, N, s, p.ksplit, out, splits, st)
                         : raw_cfg<gemm::R4Cfg, LB>(M, N, s, p.ksplit, out, splits, st);
  }

  static bool fused(int64_t M, int64_t N, int64_t K) { return plan(M, N, K).ksplit == 1; }
  static bool fused_pair(int64_t M, int64_t N, int64_t K) { return fused(M, 2 * N, K); }

  template <int LB, class Step>
  static int through(int64_t M, int64_t N, int64_t K, const bf16* a, int64_t lda, const bf16* b,
                     int64_t ldb, const Step& step, hipStream_t st) {
    const gemm::Segment s{{a, lda}, {b, ldb}, (int)K};
    return step_tile(step.cost(), M, N, K) == 128
               ? launch_product<gemm::R4SCfg, LB, false>(M, N, s, gemm::Operand{}, step, st)
               : launch_product<gemm::R4Cfg, LB, false>(M, N, s, gemm::Operand{}, step, st);
  }

  // Both of a's products, with b [N, K] and b2 [N, K].
  template <class Step>
  static int through_pair(int64_t M, int64_t N, int64_t K, const bf16* a, int64_t lda,
                          const bf16* b, int64_t ldb, const bf16* b2, int64_t ldb2,
                          const Step& step, hipStream_t st) {
    const gemm::Segment s{{a, lda}, {b, ldb}, (int)K};
    const gemm::Operand o{b2, ldb2};
    return step_tile(step.cost(), M, 2 * N, K) == 128
               ? launch_product<gemm::R4SCfg, kKMajor, true>(M, N, s, o, step, st)
               : launch_product<gemm::R4Cfg, kKMajor, true>(M, N, s, o, step, st);
  }

  static size_t store_bytes(int64_t M, int64_t N, int nseg, const int64_t* K) {
    int kt = 0;
    for (int i = 0; i < nseg; ++i) kt += ktiles(K[i]);
    return gemm::product_ws_bytes((int)M, (int)N, kt);
  }

  static int store(int64_t M, int64_t N, int nseg, const int64_t* K, const bf16* const* a,
                   const int64_t* lda, const bf16* const* b, const int64_t* ldb, bf16* out,
                   void* ws, size_t wsb, hipStream_t st) {
    gemm::Segment s[2];
    for (int i = 0; i < nseg; ++i) s[i] = gemm::Segment{{a[i], lda[i]}, {b[i], ldb[i]}, (int)K[i]};
    return gemm::run_product((int)M, (int)N, nseg, s, kMNMajor, out, N, 1.f, 0.f,
                             wsb ? static_cast<float*>(ws) : nullptr, wsb, st);
  }

  static size_t wgrads_bytes(int count, const Wgrad* p, int64_t K) {
    WgradTiles t[kMaxWgrads];
    for (int g = 0; g < count; ++g) t[g] = {p[g].M, p[g].N};
    return plan_wgrads(count, t, K).floats * sizeof(float);
  }

  static int wgrads(int count, const Wgrad* p, int64_t K, void* ws, size_t wsb, hipStream_t st) {
    WgradProduct q[kMaxWgrads];
    for (int g = 0; g < count; ++g)
      q[g] = {{p[g].M, p[g].N}, static_cast<const bf16*>(p[g].a), static_cast<const bf16*>(p[g].b),
              p[g].lda, p[g].ldb, static_cast<bf16*>(p[g].c)};
    return launch_wgrads(count, q, K, ws, wsb, st);
  }
};

// fp32 and fp16: fp32 sums on the fp32 matrix cores (ffn_f32.h), joined by the step that
// reads them. fp32 operands whose sizes, strides or bases are not multiples of 8 elements
// and 16 bytes go through the kernels that take any (gemm_f32.hip).
template <typename T>
struct Products {
  using In = float;

  template <typename E>
  static bool regular(const E* p, int64_t ld, int64_t cols) {
    return aligned16(p) && ld % 8 == 0 && cols % 8 == 0 && ld <= kMaxStride;
  }

  static F32Plan plan(int64_t M, int64_t N, int nseg, const int64_t* K) {
    return plan_f32(M, N, f32_ktiles(nseg, K));
  }

  static size_t splits_of(int64_t M, int64_t N, int nseg, const int64_t* K) {
    size_t n = plan(M, N, nseg, K).splits;
    if constexpr (std::is_same_v<T, float>) {
      int64_t sum = 0;
      for (int i = 0; i < nseg; ++i) sum += K[i];
      n = larger(n, gemmf32::sums_splits(M, N, sum));
    }
    return n;
  }

  static size_t raw_floats(int64_t M, int64_t N, int64_t K) {
    return splits_of(M, N, 1, &K) * M * N;
  }

  // out: the sums, in as many parts as splits says; a step (with plan().splits 1) takes
  // them instead
  template <typename EA, typename EB, int LA, int LB, class Step = SumsOnly>
  static int sums(int64_t M, int64_t N, int nseg, const int64_t* K, const EA* const* a,
                  const int64_t* lda, const EB* const* b, const int64_t* ldb, float* out,
                  int& splits, hipStream_t st, const Step& step = {}) {
    F32Problem p{};
    p.nseg = nseg;
    p.M = (int)M;
    p.N = (int)N;
    p.out = out;
    for (int i = 0; i < nseg; ++i) p.seg[i] = F32Segment{a[i], b[i], lda[i], ldb[i], (int)K[i]};
    const F32Plan pl = plan(M, N, nseg, K);
    splits = pl.splits;
    return launch_f32<EA, EB, LA, LB>(p, pl, step, st);
  }

  template <int LB, typename EA, typename EB>
  static int raw(int64_t M, int64_t N, int64_t K, const EA* a, int64_t lda, const EB* b,
                 int64_t ldb, float* out, int& splits, hipStream_t st) {
    if constexpr (std::is_same_v<T, float>) {
      if (!regular(a, lda, K) || !regular(b, ldb, LB == kMNMajor ? N : K) || K % 8)
        return gemmf32::sums(M, N, K, a, lda, b, ldb, LB, out, splits, st);
    }
    return sums<EA, EB, kRowsK, LB>(M, N, 1, &K, &a, &lda, &b, &ldb, out, splits, st);
  }

  // Only steps that keep nothing: those of 128 x 128 tiles that keep a tensor did not fit
  // in two workgroups' registers. (fp32 operands may yet turn out to be of any size:
  // whether a product runs its step itself is known when they are.)
  static bool fused(int64_t M, int64_t N, int64_t K) {
    return !std::is_same_v<T, float> && plan(M, N, 1, &K).splits == 1;
  }

  template <int LB, typename EA, class Step>
  static int through(int64_t M, int64_t N, int64_t K, const EA* a, int64_t lda, const T* b,
                     int64_t ldb, const Step& step, hipStream_t st) {
    int splits;
    return sums<EA, T, kRowsK, LB>(M, N, 1, &K, &a, &lda, &b, &ldb, nullptr, splits, st, step);
  }

  static bool fused_pair(int64_t, int64_t, int64_t) { return false; }

  template <class... Args>
  static int through_pair(const Args&...) { return ML_ERR_INVALID; }

  static LinearStep<T, kKeepNone> store_step(T* out, int64_t N) {
    return {nullptr, nullptr, out, 0, N, kActNone, {}};
  }

  // parts of sums to out, in order
  static int join(const float* sums, int splits, int64_t M, int64_t N, T* out, hipStream_t st) {
    const LinearStep<T, kKeepNone> step = store_step(out, N);
    return launch_rows(N % 8 == 0 && aligned16(out), PartialSource{sums, splits, M * N, N},
                       NoSource{}, step, M, N, st);
  }

  static size_t store_bytes(int64_t M, int64_t N, int nseg, const int64_t* K) {
    return splits_of(M, N, nseg, K) * M * N * sizeof(float);
  }

  template <typename EA>
  static int store(int64_t M, int64_t N, int nseg, const int64_t* K, const EA* const* a,
                   const int64_t* lda, const T* const* b, const int64_t* ldb, T* out, void* ws,
                   size_t wsb, hipStream_t st) {
    if constexpr (std::is_same_v<T, float>) {
      bool any = false;
      for (int i = 0; i < nseg; ++i)
        any = any || !regular(a[i], lda[i], K[i]) || !regular(b[i], ldb[i], N);
      if (any) return any_size(M, N, nseg, K, a, lda, b, ldb, kKMajor, kMNMajor, out, ws, wsb, st);
    }
    return joined<EA, T, kRowsK, kRowsMN>(M, N, nseg, K, a, lda, b, ldb, out, ws, st);
  }

  static size_t wgrads_bytes(int count, const Wgrad* p, int64_t K) {
    size_t n = 0;
    for (int g = 0; g < count; ++g) n = larger(n, store_bytes(p[g].M, p[g].N, 1, &K));
    return n;
  }

  static int wgrads(int count, const Wgrad* p, int64_t K, void* ws, size_t wsb, hipStream_t st) {
    for (int g = 0; g < count; ++g) {
      const Wgrad& w = p[g];
      T* out = static_cast<T*>(w.c);
      int rc;
      if constexpr (std::is_same_v<T, float>) {
        const float *a = static_cast<const float*>(w.a), *b = static_cast<const float*>(w.b);
        rc = regular(a, w.lda, w.M) && regular(b, w.ldb, w.N)
                 ? joined<float, float, kRowsMN, kRowsMN>(w.M, w.N, 1, &K, &a, &w.lda, &b, &w.ldb,
                                                          out, ws, st)
                 : any_size(w.M, w.N, 1, &K, &a, &w.lda, &b, &w.ldb, kMNMajor, kMNMajor, out, ws,
                            wsb, st);
      } else {
        rc = w.a_inner ? wgrad<float, T>(w, K, out, ws, st)
             : w.b_inner ? wgrad<T, float>(w, K, out, ws, st) : wgrad<T, T>(w, K, out, ws, st);
      }
      if (rc) return rc;
    }
    return ML_OK;
  }

 private:
  template <typename EA, typename EB>
  static int wgrad(const Wgrad& w, int64_t K, T* out, void* ws, hipStream_t st) {
    const EA* a = static_cast<const EA*>(w.a);
    const EB* b = static_cast<const EB*>(w.b);
    return joined<EA, EB, kRowsMN, kRowsMN>(w.M, w.N, 1, &K, &a, &w.lda, &b, &w.ldb, out, ws, st);
  }

  template <typename EA, typename EB, int LA, int LB>
  static int joined(int64_t M, int64_t N, int nseg, const int64_t* K, const EA* const* a,
                    const int64_t* lda, const EB* const* b, const int64_t* ldb, T* out, void* ws,
                    hipStream_t st) {
    int splits = 1;
    float* parts = static_cast<float*>(ws);
    if (plan(M, N, nseg, K).splits == 1)
      return sums<EA, EB, LA, LB>(M, N, nseg, K, a, lda, b, ldb, parts, splits, st,
                                  store_step(out, N));
    const int rc = sums<EA, EB, LA, LB>(M, N, nseg, K, a, lda, b, ldb, parts, splits, st);
    return rc ? rc : join(parts, splits, M, N, out, st);
  }

  static int any_size(int64_t M, int64_t N, int nseg, const int64_t* K, const float* const* a,
                      const int64_t* lda, const float* const* b, const int64_t* ldb, int la, int lb,
                      float* out, void* ws, size_t wsb, hipStream_t st) {
    const void *ap[2], *bp[2];
    for (int i = 0; i < nseg; ++i) {
      ap[i] = a[i];
      bp[i] = b[i];
    }
    return ml_gemm_f32_segments_ws(M, N, nseg, K, ap, lda, bp, ldb, la, lb, out, N, 1.f, 0.f, ws,
                                   wsb, st);
  }
};

// Operands of the 16-bit forms (fp32 takes any).
template <typename T>
int check(const void* a, int64_t lda, int64_t cols, const char* what) {
  if constexpr (std::is_same_v<T, float>) return ML_OK;
  return check_operands({{a, lda, cols, what}});
}

template <int KIND>
using Kind = std::integral_constant<int, KIND>;

// How a tensor may be kept where the products are of type T.
template <typename T, typename F>
int dispatch_keep(int keep, F&& f) {
  constexpr int kWhole = std::is_same_v<T, float> ? kKeepF32 : kKeepFp16;
  if (keep == kKeepNone) return f(Kind<kKeepNone>{});
  if (keep == kWhole) return f(Kind<kWhole>{});
  if (keep == kKeepFp8) return f(Kind<kKeepFp8>{});
  set_error("ffn: tensors of this dtype are not kept as %d", keep);
  return ML_ERR_INVALID;
}

// Time in us of a product of up to 128 rows on the tiles (ops: 2 for the gated block's
// pair): latency in bf16, the fp32 matrix cores' time otherwise. Fitted to 96 and 128 rows
// by plan_skinny's shapes. What the two estimates choose, against workgroups for all of up
// to 64 rows and tiles above: [80, 1024] to 1024 through 2816, the gated block in bf16, 44
// -> 21 us, [64, 2048] x 16384 39 -> 19, [96, 4304] x 1152 24 -> 11, in fp16 26 -> 11.
template <typename T>
double tiles_us(int64_t M, int64_t N, int64_t K, int ops) {
  const double all = (double)ops * N;
  return std::is_same_v<T, bf16> ? (ops > 1 ? 19.5 : 11.5) + 1.5e-3 * K + 0.33e-3 * all
                                 : 14 + (M > 64 ? 2e-6 : 1e-6) * all * K;
}

// Whether a forward's product is one of few rows. (Kept tensors do not count, so that a
// workspace goes by the sizes alone.)
template <typename T>
bool few(int64_t M, int64_t N, int64_t K) {
  return M <= kSkinnyRows &&
         plan_skinny(sizeof(T), sizeof(T), 1, 1, M, N, K).us <= tiles_us<T>(M, N, K, 1);
}

template <typename T>
bool few_mlp(int64_t M, int64_t H, int64_t I, int64_t O) {
  return M <= kSkinnyRows &&
         plan_skinny(sizeof(T), sizeof(T), 2, 1, M, I, H).us +
                 plan_skinny(sizeof(Inner<T>), sizeof(T), 1, 1, M, O, I).us <=
             tiles_us<T>(M, I, H, 2) + tiles_us<T>(M, O, I, 1);
}

// Whether such a product's operands can be read so: 16-bit ones always (they qualify as
// they are checked), fp32 ones may not.
bool few_operands(int64_t N, int64_t K, const void* x, int64_t ldx, const void* w, int64_t ldw) {
  return N % 8 == 0 && K % 8 == 0 && aligned16(x) && aligned16(w) && ldx % 4 == 0 && ldw % 4 == 0;
}

// A product of few rows of 16-bit operands needs no workspace, and never comes to run
// on another kernel.
int few_checked(bool run) {
  ML_CHECK(!run, "ffn: operands of few rows that were not checked");
  return ML_OK;
}

int check_sizes(int64_t M, int64_t N, int64_t K) {
  constexpr int64_t kMax = (1LL << 31) - 1024;  // (a last tile's rows are counted in 32 bits)
  ML_CHECK(M > 0 && N > 0 && K > 0 && M < kMax && N < kMax && K < kMax,
           "ffn: bad sizes (rows %lld, columns %lld, %lld)", (long long)M, (long long)N,
           (long long)K);
  return ML_OK;
}

int check_data(int64_t data, int64_t cols) {
  ML_CHECK(data > 0 && data <= cols, "ffn: %lld of %lld columns are not padding", (long long)data,
           (long long)cols);
  return ML_OK;
}

int check_kept(int keep, const void* v, const void* scale, const char* what) {
  ML_CHECK(keep >= kKeepNone && keep <= kKeepFp8, "ffn: bad way to keep %s (%d)", what, keep);
  ML_CHECK(keep == kKeepNone || v, "ffn: %s is kept but its buffer is null", what);
  ML_CHECK(keep < kKeepFp16 || scale, "ffn: %s is kept with scales but they are null", what);
  ML_CHECK(!v || aligned16(v), "ffn: the buffer of %s must be 16-byte aligned", what);
  return ML_OK;
}

// ------------------------------------------------------------------- linear --

template <typename T, int KIND>
int linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
               const LinearStep<T, KIND>& step,
               int64_t M, int64_t N, int64_t K, Arena& ws, bool run, hipStream_t st) {
  const T* xt = static_cast<const T*>(x);
  const T* wt = static_cast<const T*>(w);
  const bool vec = N % 8 == 0 && aligned_rows(step.bias, 0) && aligned_rows(step.residual, step.ldr) &&
                   aligned_rows(step.y, step.ldy);
  const bool rows_few = few<T>(M, N, K);
  if (run && vec && rows_few && few_operands(N, K, x, ldx, w, ldw))
    return launch_skinny<KIND != kKeepNone, false>(
        SkinnyProduct<T, T>{xt, wt, nullptr, ldx, ldw, 0, (int)M, (int)N, (int)K}, step, st);
  if (!std::is_same_v<T, float> && rows_few) return few_checked(run);
  if constexpr (std::is_same_v<T, bf16> || KIND == kKeepNone) {
    if (run && Products<T>::fused(M, N, K))
      return Products<T>::template through<kKMajor>(M, N, K, xt, ldx, wt, ldw, step, st);
  }
  if (std::is_same_v<T, bf16> && Products<T>::fused(M, N, K)) return ML_OK;
  if constexpr (std::is_same_v<T, float> && KIND == kKeepNone) {
    using P = Products<float>;
    if (run && P::regular(xt, ldx, K) && P::regular(wt, ldw, K) &&
        P::plan(M, N, 1, &K).splits == 1)
      return P::through<kKMajor>(M, N, K, xt, ldx, wt, ldw, step, st);
  }
  float* sums = ws.take<float>(Products<T>::raw_floats(M, N, K));
  if (!run) return ML_OK;
  int splits = 1;
  const int rc = Products<T>::template raw<kKMajor>(M, N, K, xt, ldx, wt, ldw, sums, splits, st);
  if (rc) return rc;
  return launch_rows(vec, PartialSource{sums, splits, M * N, N}, NoSource{}, step, M, N, st);
}

struct GradGrid {
  int64_t x, y, rows_per;
};

GradGrid grad_grid(int64_t rows, int64_t cols, bool vec) {
  const int64_t x = (cols + (vec ? 255 : 31)) / (vec ? 256 : 32);
  int64_t want = (4 * 256 + x - 1) / x;  // four workgroups a CU
  const int64_t most = (rows + 7) / 8;
  want = want < most ? want : most;
  want = want > 0 ? want : 1;
  const int64_t per = ((rows + want - 1) / want + 7) / 8 * 8;
  return {x, (rows + per - 1) / per, per};
}

// dz (act) and db; ws counts what the partial sums take.
template <typename T, int KIND>
int linear_grad(const T* dy, int64_t ldy, const Kept<KIND>& z, int act, Inner<T>* dz, T* db,
                int64_t M, int64_t N, Arena& ws, bool run, hipStream_t st) {
  const bool vec = N % 8 == 0 && aligned_rows(dy, ldy) && aligned_rows(dz, 0);
  // (the row ranges of the wider grid: a count that holds for both)
  const int64_t most = grad_grid(M, N, true).y > grad_grid(M, N, false).y
                           ? grad_grid(M, N, true).y : grad_grid(M, N, false).y;
  float* partial = db || !run ? ws.take<float>((size_t)(most * N)) : nullptr;
  if (!run) return ML_OK;
  const GradGrid g = grad_grid(M, N, vec);
  const dim3 grid((unsigned)g.x, (unsigned)g.y);
  if (vec)
    linear_grad_kernel<8, T, Inner<T>, KIND><<<grid, kThreads, 0, st>>>(dy, ldy, z, act, dz, partial, M, N, g.rows_per);
  else
    linear_grad_kernel<1, T, Inner<T>, KIND><<<grid, kThreads, 0, st>>>(dy, ldy, z, act, dz, partial, M, N, g.rows_per);
  ML_LAUNCH_CHECK();
  if (db) {
    column_sum_kernel<T><<<dim3((unsigned)((N + 31) / 32)), kThreads, 0, st>>>(partial, (int)g.y, N,
                                                                               db);
    ML_LAUNCH_CHECK();
  }
  return ML_OK;
}

struct LinearBwd {
  const void *x, *w, *dy;
  int64_t ldx, ldw, ldy;
  int act, keep;
  const void *z, *zscale;
  void *dx, *dw, *db;
  int64_t M, N, K;
};

template <typename T>
int linear_bwd(const LinearBwd& p, Arena& ws, bool run, hipStream_t st) {
  using P = Products<T>;
  const T* dy = static_cast<const T*>(p.dy);
  const bool act = p.act != kActNone;
  Inner<T>* dz = act ? ws.take<Inner<T>>((size_t)(p.M * p.N)) : nullptr;
  if (dz || p.db || !run) {
    const int rc = dispatch_keep<T>(dz ? p.keep : (int)kKeepNone, [&](auto kind) {
      return linear_grad<T>(dy, p.ldy, make_kept<kind.value>(p.z, p.zscale, p.N), p.act, dz,
                            static_cast<T*>(p.db), p.M, p.N, ws, run, st);
    });
    if (rc) return rc;
  }
  const Wgrad wgrad{p.N, p.K, act ? (const void*)dz : p.dy, p.x, act ? p.N : p.ldy, p.ldx, p.dw, act,
                    false};
  const size_t wsb = larger(P::store_bytes(p.M, p.K, 1, &p.N), P::wgrads_bytes(1, &wgrad, p.M));
  char* pws = ws.take<char>(wsb);
  if (!run) return ML_OK;
  if (p.dx) {
    const T* w = static_cast<const T*>(p.w);
    T* dx = static_cast<T*>(p.dx);
    const Inner<T>* z = dz;
    const int rc = act ? P::store(p.M, p.K, 1, &p.N, &z, &p.N, &w, &p.ldw, dx, pws, wsb, st)
                       : P::store(p.M, p.K, 1, &p.N, &dy, &p.ldy, &w, &p.ldw, dx, pws, wsb, st);
    if (rc) return rc;
  }
  return p.dw ? P::wgrads(1, &wgrad, p.M, pws, wsb, st) : (int)ML_OK;
}

// -------------------------------------------------------------- gated block --

struct MlpFwd {
  const void *x, *wg, *wu, *wd, *residual;
  int64_t ldx, ldg, ldu, ldd, ldr;
  void* y;
  int keep;
  void *gate, *gscale, *up, *uscale;
  int64_t M, H, I, O, data;
};

// The block of few rows: weights of T, h of TH (fp32 where T is fp16, whose range h may
// leave).
template <typename T, typename TH, int KIND>
int launch_few_mlp(const MlpFwd& p, const TH* h, const GatedStep<TH, KIND>& step,
            const LinearStep<T, kKeepNone>& out, hipStream_t st) {
  const T *wg = static_cast<const T*>(p.wg), *wu = static_cast<const T*>(p.wu);
  const int rc = launch_skinny<KIND != kKeepNone, true>(
      SkinnyProduct<T, T>{static_cast<const T*>(p.x), wg, wu, p.ldx, p.ldg, p.ldu, (int)p.M,
                          (int)p.I, (int)p.H}, step, st);
  if (rc) return rc;
  return launch_skinny<false, false>(
      SkinnyProduct<TH, T>{h, static_cast<const T*>(p.wd), nullptr, p.I, p.ldd, 0, (int)p.M,
                           (int)p.O, (int)p.I}, out, st);
}

template <typename T, int KIND>
int mlp_fwd(const MlpFwd& p, Arena& ws, bool run, hipStream_t st) {
  using P = Products<T>;
  using In = Inner<T>;
  In* h = ws.take<In>((size_t)(p.M * p.I));
  const T* x = static_cast<const T*>(p.x);
  const T* wg = static_cast<const T*>(p.wg);
  const T* wu = static_cast<const T*>(p.wu);
  const T* wd = static_cast<const T*>(p.wd);
  const GatedStep<In, KIND> step{h, p.I, make_kept<KIND>(p.gate, p.gscale, p.I),
                                make_kept<KIND>(p.up, p.uscale, p.I), p.data};
  const LinearStep<T, kKeepNone> out{nullptr, static_cast<const T*>(p.residual),
                                     static_cast<T*>(p.y), p.ldr, p.O, kActNone, {}};
  const bool vec = p.O % 8 == 0 && aligned_rows(p.residual, p.ldr) && aligned_rows(p.y, p.O);
  const bool rows_few = few_mlp<T>(p.M, p.H, p.I, p.O);
  if (run && vec && rows_few && few_operands(p.I, p.H, x, p.ldx, wg, p.ldg) && aligned16(wu) &&
      p.ldu % 4 == 0 && few_operands(p.O, p.I, h, p.I, wd, p.ldd))
    return launch_few_mlp<T, In>(p, h, step, out, st);
  if (!std::is_same_v<T, float> && rows_few) return few_checked(run);
  const bool fuse_in = P::fused_pair(p.M, p.I, p.H), fuse_out = P::fused(p.M, p.O, p.I);
  const size_t n_in = fuse_in ? 0 : P::raw_floats(p.M, p.I, p.H);
  const size_t n_out = fuse_out ? 0 : P::raw_floats(p.M, p.O, p.I);
  float* sums = ws.take<float>(larger(2 * n_in, n_out));
  if (!run) return ML_OK;
  int splits = 1, rc;
  if (fuse_in) {
    rc = P::through_pair(p.M, p.I, p.H, x, p.ldx, wg, p.ldg, wu, p.ldu, step, st);
  } else {
    int splits_up = 1;  // (the two weights may lie so that their products split differently)
    rc = P::template raw<kKMajor>(p.M, p.I, p.H, x, p.ldx, wg, p.ldg, sums, splits, st);
    if (rc) return rc;
    rc = P::template raw<kKMajor>(p.M, p.I, p.H, x, p.ldx, wu, p.ldu, sums + n_in, splits_up, st);
    if (rc) return rc;
    const int64_t mi = p.M * p.I;
    rc = launch_rows(p.I % 8 == 0, PartialSource{sums, splits, mi, p.I},
                     PartialSource{sums + n_in, splits_up, mi, p.I}, step, p.M, p.I, st);
  }
  if (rc) return rc;
  if (fuse_out) return P::template through<kKMajor>(p.M, p.O, p.I, h, p.I, wd, p.ldd, out, st);
  rc = P::template raw<kKMajor>(p.M, p.O, p.I, h, p.I, wd, p.ldd, sums, splits, st);
  if (rc) return rc;
  return launch_rows(vec, PartialSource{sums, splits, p.M * p.O, p.O}, NoSource{}, out, p.M,
                     p.O, st);
}

struct MlpBwd {
  const void *x, *wg, *wu, *wd, *dy;
  int64_t ldx, ldg, ldu, ldd, ldy;
  int keep;
  const void *gate, *gscale, *up, *uscale;
  void *dx, *dwg, *dwu, *dwd;
  int64_t M, H, I, O, data;
};

template <typename T, int KIND>
int mlp_bwd(const MlpBwd& p, Arena& ws, bool run, hipStream_t st) {
  using P = Products<T>;
  using In = Inner<T>;
  const size_t mi = (size_t)(p.M * p.I);
  In* dg = ws.take<In>(mi);
  In* du = ws.take<In>(mi);
  In* h = ws.take<In>(mi);
  constexpr bool kMayFuse = std::is_same_v<T, bf16>;
  const bool fuse = kMayFuse && P::fused(p.M, p.I, p.O);
  float* sums = ws.take<float>(fuse ? 0 : P::raw_floats(p.M, p.I, p.O));
  const T* dy = static_cast<const T*>(p.dy);
  // the weights' gradients that are wanted (counted for any of them: all three)
  Wgrad wgrad[3];
  int wanted = 0;
  if (p.dwg || !run) wgrad[wanted++] = {p.I, p.H, dg, p.x, p.I, p.ldx, p.dwg, true, false};
  if (p.dwu || !run) wgrad[wanted++] = {p.I, p.H, du, p.x, p.I, p.ldx, p.dwu, true, false};
  if (p.dwd || !run) wgrad[wanted++] = {p.O, p.I, p.dy, h, p.ldy, p.I, p.dwd, false, true};
  const int64_t ks[2] = {p.I, p.I};
  size_t wsb = P::store_bytes(p.M, p.H, 2, ks);
  if (run) {
    wsb = larger(wsb, P::wgrads_bytes(wanted, wgrad, p.M));
  } else {
    // (fewer products may split more)
    for (int first = 0; first < 3; ++first)
      for (int n = 1; first + n <= 3; ++n)
        wsb = larger(wsb, P::wgrads_bytes(n, wgrad + first, p.M));
    const Wgrad outer[2] = {wgrad[0], wgrad[2]};
    wsb = larger(wsb, P::wgrads_bytes(2, outer, p.M));
  }
  char* pws = ws.take<char>(wsb);
  if (!run) return ML_OK;
  const T* wd = static_cast<const T*>(p.wd);
  const GatedGradStep<In, KIND> step{dg, du, p.dwd ? h : nullptr, p.I,
                                    make_kept<KIND>(p.gate, p.gscale, p.I),
                                    make_kept<KIND>(p.up, p.uscale, p.I), p.data};
  int splits = 1, rc = ML_OK;
  if (fuse) {
    if constexpr (kMayFuse)
      rc = P::template through<kMNMajor>(p.M, p.I, p.O, dy, p.ldy, wd, p.ldd, step, st);
  } else {
    rc = P::template raw<kMNMajor>(p.M, p.I, p.O, dy, p.ldy, wd, p.ldd, sums, splits, st);
    if (rc) return rc;
    rc = launch_rows(p.I % 8 == 0, PartialSource{sums, splits, p.M * p.I, p.I}, NoSource{}, step,
                     p.M, p.I, st);
  }
  if (rc) return rc;
  if (p.dx) {
    const int64_t la[2] = {p.I, p.I}, lb[2] = {p.ldg, p.ldu};
    const In* a[2] = {dg, du};
    const T* b[2] = {static_cast<const T*>(p.wg), static_cast<const T*>(p.wu)};
    rc = P::store(p.M, p.H, 2, ks, a, la, b, lb, static_cast<T*>(p.dx), pws, wsb, st);
    if (rc) return rc;
  }
  return wanted ? P::wgrads(wanted, wgrad, p.M, pws, wsb, st) : (int)ML_OK;
}

}  // namespace
}  // namespace ffn
}  // namespace mla

using namespace mla;

#define ML_TRY(call)        \
  do {                      \
    const int rc_ = (call); \
    if (rc_) return rc_;    \
  } while (0)

extern "C" size_t ml_linear_fwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
  if (ffn::check_sizes(M, N, K)) return 0;
  ffn::Arena ws{nullptr};
  dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return ffn::linear_fwd<T>(nullptr, 0, nullptr, 0, ffn::LinearStep<T, ffn::kKeepNone>{}, M, N, K,
                              ws, false, nullptr);
  });
  return ws.used;
}

extern "C" int ml_linear_fwd_padded(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                    const void* bias, const void* residual, int64_t ldr, int act,
                                    void* y, int64_t ldy, int keep, void* z, void* zscale,
                                    int64_t M, int64_t N, int64_t K, int64_t data_n,
                                    void* workspace, size_t workspace_bytes, int dtype,
                                    void* stream) {
  ML_TRY(ffn::check_sizes(M, N, K));
  ML_TRY(ffn::check_data(data_n, N));
  ML_CHECK(x && w && y, "linear: null pointer");
  ML_CHECK(act >= kActNone && act <= kActGeluTanh, "linear: bad activation %d", act);
  ML_CHECK(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), "linear: bad row strides");
  ML_TRY(ffn::check_kept(keep, z, zscale, "z"));
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    ML_TRY(ffn::check<T>(x, ldx, K, "x"));
    ML_TRY(ffn::check<T>(w, ldw, K, "weight"));
    ML_TRY(ffn::check<T>(y, ldy, N, "y"));
    ML_TRY(ffn::check<T>(bias, 0, N, "bias"));
    ML_TRY(ffn::check<T>(residual, residual ? ldr : 0, N, "residual"));
    ffn::Arena ws{static_cast<char*>(workspace)};
    const size_t need = ml_linear_fwd_workspace_bytes(M, N, K, dtype);
    ML_CHECK(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
             "linear: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return ffn::dispatch_keep<T>(keep, [&](auto kind) {
      const ffn::LinearStep<T, kind.value> step{
          static_cast<const T*>(bias), static_cast<const T*>(residual), static_cast<T*>(y), ldr,
          ldy, act, ffn::make_kept<kind.value>(z, zscale, N), data_n};
      return ffn::linear_fwd<T>(x, ldx, w, ldw, step, M, N, K, ws, true, (hipStream_t)stream);
    });
  });
}

extern "C" int ml_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                             const void* bias, const void* residual, int64_t ldr, int act,
                             void* y, int64_t ldy, int keep, void* z, void* zscale, int64_t M,
                             int64_t N, int64_t K, void* workspace, size_t workspace_bytes,
                             int dtype, void* stream) {
  return ml_linear_fwd_padded(x, ldx, w, ldw, bias, residual, ldr, act, y, ldy, keep, z, zscale, M,
                              N, K, N, workspace, workspace_bytes, dtype, stream);
}

extern "C" size_t ml_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int act,
                                                int dtype) {
  if (ffn::check_sizes(M, N, K)) return 0;
  ffn::LinearBwd p{};
  p.act = act;
  p.M = M;
  p.N = N;
  p.K = K;
  ffn::Arena ws{nullptr};
  dispatch_dtype(dtype, [&](auto t) { return ffn::linear_bwd<decltype(t)>(p, ws, false, nullptr); });
  return ws.used;
}

extern "C" int ml_linear_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                             const void* dy, int64_t ldy, int act, int keep, const void* z,
                             const void* zscale, void* dx, void* dw, void* db, int64_t M,
                             int64_t N, int64_t K, void* workspace, size_t workspace_bytes,
                             int dtype, void* stream) {
  ML_TRY(ffn::check_sizes(M, N, K));
  ML_CHECK(act >= kActNone && act <= kActGeluTanh, "linear backward: bad activation %d", act);
  ML_CHECK(dy && (!dx || w) && (!dw || x), "linear backward: null pointer");
  ML_CHECK(ldy >= N && (!dx || ldw >= K) && (!dw || ldx >= K), "linear backward: bad row strides");
  ML_CHECK(act == kActNone || keep != ffn::kKeepNone, "linear backward: no z was kept");
  ML_TRY(ffn::check_kept(act == kActNone ? ffn::kKeepNone : keep, z, zscale, "z"));
  if (!dx && !dw && !db) return ML_OK;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (dx || dw) ML_TRY(ffn::check<T>(act == kActNone ? dy : nullptr, act == kActNone ? ldy : 0, N, "dy"));
    if (dx) {
      ML_TRY(ffn::check<T>(w, ldw, K, "weight"));
      ML_TRY(ffn::check<T>(dx, K, K, "dx"));
    }
    if (dw) {
      ML_TRY(ffn::check<T>(x, ldx, K, "x"));
      ML_TRY(ffn::check<T>(dw, K, K, "dw"));
    }
    ffn::Arena ws{static_cast<char*>(workspace)};
    const size_t need = ml_linear_bwd_workspace_bytes(M, N, K, act, dtype);
    ML_CHECK(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
             "linear backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const ffn::LinearBwd p{x, w, dy, ldx, ldw, ldy, act, keep, z, zscale, dx, dw, db, M, N, K};
    return ffn::linear_bwd<T>(p, ws, true, (hipStream_t)stream);
  });
}

namespace mla {
namespace ffn {
namespace {
int check_mlp(int64_t M, int64_t H, int64_t I, int64_t O) {
  ML_TRY(check_sizes(M, H, I));
  return check_sizes(M, O, 2 * I);
}
}  // namespace
}  // namespace ffn
}  // namespace mla

extern "C" size_t ml_swiglu_mlp_fwd_workspace_bytes(int64_t M, int64_t H, int64_t I, int64_t O,
                                                    int dtype) {
  if (ffn::check_mlp(M, H, I, O)) return 0;
  ffn::MlpFwd p{};
  p.M = M;
  p.H = H;
  p.I = I;
  p.O = O;
  ffn::Arena ws{nullptr};
  dispatch_dtype(dtype, [&](auto t) { return ffn::mlp_fwd<decltype(t), ffn::kKeepNone>(p, ws, false, nullptr); });
  return ws.used;
}

extern "C" int ml_swiglu_mlp_fwd_padded(const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                        const void* wu, int64_t ldu, const void* wd, int64_t ldd,
                                        const void* residual, int64_t ldr, void* y, int keep,
                                        void* gate, void* gate_scale, void* up, void* up_scale,
                                        int64_t M, int64_t H, int64_t I, int64_t O, int64_t data_i,
                                        void* workspace, size_t workspace_bytes, int dtype,
                                        void* stream) {
  ML_TRY(ffn::check_mlp(M, H, I, O));
  ML_TRY(ffn::check_data(data_i, I));
  ML_CHECK(x && wg && wu && wd && y, "swiglu mlp: null pointer");
  ML_CHECK(ldx >= H && ldg >= H && ldu >= H && ldd >= I && (!residual || ldr >= O),
           "swiglu mlp: bad row strides");
  ML_TRY(ffn::check_kept(keep, gate, gate_scale, "gate"));
  ML_TRY(ffn::check_kept(keep, up, up_scale, "up"));
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    ML_TRY(ffn::check<T>(x, ldx, H, "x"));
    ML_TRY(ffn::check<T>(wg, ldg, H, "gate weight"));
    ML_TRY(ffn::check<T>(wu, ldu, H, "up weight"));
    ML_TRY(ffn::check<T>(wd, ldd, I, "down weight"));
    ML_TRY(ffn::check<T>(y, O, O, "y"));
    ML_TRY(ffn::check<T>(residual, residual ? ldr : 0, O, "residual"));
    ffn::Arena ws{static_cast<char*>(workspace)};
    const size_t need = ml_swiglu_mlp_fwd_workspace_bytes(M, H, I, O, dtype);
    ML_CHECK(workspace_bytes >= need && workspace && aligned16(workspace),
             "swiglu mlp: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const ffn::MlpFwd p{x, wg, wu, wd, residual, ldx, ldg, ldu, ldd, ldr, y, keep,
                        gate, gate_scale, up, up_scale, M, H, I, O, data_i};
    return ffn::dispatch_keep<T>(keep, [&](auto kind) {
      return ffn::mlp_fwd<T, kind.value>(p, ws, true, (hipStream_t)stream);
    });
  });
}

extern "C" int ml_swiglu_mlp_fwd(const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                 const void* wu, int64_t ldu, const void* wd, int64_t ldd,
                                 const void* residual, int64_t ldr, void* y, int keep, void* gate,
                                 void* gate_scale, void* up, void* up_scale, int64_t M, int64_t H,
                                 int64_t I, int64_t O, void* workspace, size_t workspace_bytes,
                                 int dtype, void* stream) {
  return ml_swiglu_mlp_fwd_padded(x, ldx, wg, ldg, wu, ldu, wd, ldd, residual, ldr, y, keep, gate,
                                  gate_scale, up, up_scale, M, H, I, O, I, workspace,
                                  workspace_bytes, dtype, stream);
}

extern "C" size_t ml_swiglu_mlp_bwd_workspace_bytes(int64_t M, int64_t H, int64_t I, int64_t O,
                                                    int dtype) {
  if (ffn::check_mlp(M, H, I, O)) return 0;
  ffn::MlpBwd p{};
  p.M = M;
  p.H = H;
  p.I = I;
  p.O = O;
  ffn::Arena ws{nullptr};
  dispatch_dtype(dtype, [&](auto t) { return ffn::mlp_bwd<decltype(t), ffn::kKeepFp8>(p, ws, false, nullptr); });
  return ws.used;
}

extern "C" int ml_swiglu_mlp_bwd_padded(const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                        const void* wu, int64_t ldu, const void* wd, int64_t ldd,
                                        const void* dy, int64_t ldy, int keep, const void* gate,
                                        const void* gate_scale, const void* up,
                                        const void* up_scale, void* dx, void* dwg, void* dwu,
                                        void* dwd, int64_t M, int64_t H, int64_t I, int64_t O,
                                        int64_t data_i, void* workspace, size_t workspace_bytes,
                                        int dtype, void* stream) {
  ML_TRY(ffn::check_mlp(M, H, I, O));
  ML_TRY(ffn::check_data(data_i, I));
  ML_CHECK(wd && dy && (!dx || (wg && wu)) && (!(dwg || dwu) || x),
           "swiglu mlp backward: null pointer");
  ML_CHECK((!x || ldx >= H) && (!wg || ldg >= H) && (!wu || ldu >= H) && ldd >= I && ldy >= O,
           "swiglu mlp backward: bad row strides");
  ML_CHECK(keep != ffn::kKeepNone, "swiglu mlp backward: gate and up were not kept");
  ML_TRY(ffn::check_kept(keep, gate, gate_scale, "gate"));
  ML_TRY(ffn::check_kept(keep, up, up_scale, "up"));
  if (!dx && !dwg && !dwu && !dwd) return ML_OK;
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    ML_TRY(ffn::check<T>(x, x ? ldx : 0, H, "x"));
    ML_TRY(ffn::check<T>(wg, wg ? ldg : 0, H, "gate weight"));
    ML_TRY(ffn::check<T>(wu, wu ? ldu : 0, H, "up weight"));
    ML_TRY(ffn::check<T>(wd, ldd, I, "down weight"));
    ML_TRY(ffn::check<T>(dy, ldy, O, "dy"));
    ML_TRY(ffn::check<T>(dx, H, H, "dx"));
    ML_TRY(ffn::check<T>(dwg, H, H, "gate weight's gradient"));
    ML_TRY(ffn::check<T>(dwu, H, H, "up weight's gradient"));
    ML_TRY(ffn::check<T>(dwd, I, I, "down weight's gradient"));
    ffn::Arena ws{static_cast<char*>(workspace)};
    const size_t need = ml_swiglu_mlp_bwd_workspace_bytes(M, H, I, O, dtype);
    ML_CHECK(workspace_bytes >= need && workspace && aligned16(workspace),
             "swiglu mlp backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const ffn::MlpBwd p{x, wg, wu, wd, dy, ldx, ldg, ldu, ldd, ldy, keep, gate, gate_scale, up,
                        up_scale, dx, dwg, dwu, dwd, M, H, I, O, data_i};
    return ffn::dispatch_keep<T>(keep, [&](auto kind) -> int {
      if constexpr (kind.value == ffn::kKeepNone)
        return ML_ERR_INVALID;  // (refused above)
      else
        return ffn::mlp_bwd<T, kind.value>(p, ws, true, (hipStream_t)stream);
    });
  });
}

extern "C" int ml_swiglu_mlp_bwd(const void* x, int64_t ldx, const void* wg, int64_t ldg,
                                 const void* wu, int64_t ldu, const void* wd, int64_t ldd,
                                 const void* dy, int64_t ldy, int keep, const void* gate,
                                 const void* gate_scale, const void* up, const void* up_scale,
                                 void* dx, void* dwg, void* dwu, void* dwd, int64_t M, int64_t H,
                                 int64_t I, int64_t O, void* workspace, size_t workspace_bytes,
                                 int dtype, void* stream) {
  return ml_swiglu_mlp_bwd_padded(x, ldx, wg, ldg, wu, ldu, wd, ldd, dy, ldy, keep, gate,
                                  gate_scale, up, up_scale, dx, dwg, dwu, dwd, M, H, I, O, I,
                                  workspace, workspace_bytes, dtype, stream);
}

// ----------------------------------------------------------------- padding --

extern "C" int ml_pad_matrices(int count, void* const* any, const int64_t* strides,
                               const int64_t* sizes, void* const* wide, const int64_t* wide_sizes,
                               int to_wide, int dtype, void* stream) {
  ML_CHECK(count >= 1 && count <= ffn::kMaxPads, "pad: %d matrices, 1 to %d at a time", count,
           ffn::kMaxPads);
  ML_CHECK(any && strides && sizes && wide && wide_sizes, "pad: null pointer");
  ffn::PadJobs jobs{};
  jobs.count = count;
  for (int j = 0; j < count; ++j) {
    ffn::PadJob& p = jobs.job[j];
    p.any = any[j];
    p.wide = wide[j];
    p.s0 = strides[2 * j];
    p.s1 = strides[2 * j + 1];
    p.rows = sizes[2 * j];
    p.cols = sizes[2 * j + 1];
    p.wrows = wide_sizes[2 * j];
    p.wcols = wide_sizes[2 * j + 1];
    ML_CHECK(p.rows >= 0 && p.cols >= 0 && p.wrows >= p.rows && p.wcols >= p.cols &&
                 p.wcols % 8 == 0 && p.wrows < (1LL << 31) && p.wcols < (1LL << 31),
             "pad: [%lld, %lld] in [%lld, %lld]", (long long)p.rows, (long long)p.cols,
             (long long)p.wrows, (long long)p.wcols);
    ML_CHECK((p.any || p.rows == 0 || p.cols == 0) && (p.wide || p.wrows == 0 || p.wcols == 0),
             "pad: null pointer");
    ML_CHECK(aligned16(p.wide), "pad: the padded matrix must be 16-byte aligned");
  }
  return dispatch_dtype(dtype, [&](auto t) {
    return ffn::launch_pads(jobs, (int)sizeof(t), to_wide != 0, (hipStream_t)stream);
  });
}

// ------------------------------------------------- SwiGLU kept in 8 bits --

extern "C" int ml_swiglu_kept_fwd(const void* gate, const void* up, void* out, void* gate_q,
                                  void* gate_scale, void* up_q, void* up_scale, int64_t rows,
                                  int64_t cols, int dtype, void* stream) {
  ML_CHECK(rows >= 0 && cols >= 0, "swiglu kept: negative size");
  if (rows == 0 || cols == 0) return ML_OK;
  ML_CHECK(gate && up && out, "swiglu kept: null pointer");
  ML_TRY(ffn::check_kept(ffn::kKeepFp8, gate_q, gate_scale, "gate"));
  ML_TRY(ffn::check_kept(ffn::kKeepFp8, up_q, up_scale, "up"));
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const bool vec = cols % 8 == 0 && aligned16(gate) && aligned16(up) && aligned16(out);
    // whole blocks: one long row
    const bool flat = cols % held::kBlock == 0;
    const int64_t r = flat ? 1 : rows, c = flat ? rows * cols : cols;
    const ffn::GatedStep<T, ffn::kKeepFp8> step{
        static_cast<T*>(out), c, ffn::make_kept<ffn::kKeepFp8>(gate_q, gate_scale, c),
        ffn::make_kept<ffn::kKeepFp8>(up_q, up_scale, c)};
    return ffn::launch_rows(vec, ffn::TypedSource<T>{static_cast<const T*>(gate), c},
                            ffn::TypedSource<T>{static_cast<const T*>(up), c}, step, r, c,
                            (hipStream_t)stream);
  });
}

extern "C" int ml_swiglu_kept_bwd(const void* gate_q, const void* gate_scale, const void* up_q,
                                  const void* up_scale, const void* dy, void* dgate, void* dup,
                                  int64_t rows, int64_t cols, int dtype, void* stream) {
  ML_CHECK(rows >= 0 && cols >= 0, "swiglu kept backward: negative size");
  if (rows == 0 || cols == 0) return ML_OK;
  ML_CHECK(dy && dgate && dup, "swiglu kept backward: null pointer");
  ML_TRY(ffn::check_kept(ffn::kKeepFp8, gate_q, gate_scale, "gate"));
  ML_TRY(ffn::check_kept(ffn::kKeepFp8, up_q, up_scale, "up"));
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const bool vec = cols % 8 == 0 && aligned16(dy) && aligned16(dgate) && aligned16(dup);
    const bool flat = cols % held::kBlock == 0;
    const int64_t r = flat ? 1 : rows, c = flat ? rows * cols : cols;
    const ffn::GatedGradStep<T, ffn::kKeepFp8> step{
        static_cast<T*>(dgate), static_cast<T*>(dup), nullptr, c,
        ffn::make_kept<ffn::kKeepFp8>(gate_q, gate_scale, c),
        ffn::make_kept<ffn::kKeepFp8>(up_q, up_scale, c)};
    return ffn::launch_rows(vec, ffn::TypedSource<T>{static_cast<const T*>(dy), c}, ffn::NoSource{},
                            step, r, c, (hipStream_t)stream);
  });
}

extern "C" int ml_held_values(const void* q, const void* scale, void* out, int64_t rows,
                              int64_t cols, int dtype, void* stream) {
  ML_CHECK(rows >= 0 && cols >= 0, "held values: negative size");
  if (rows == 0 || cols == 0) return ML_OK;
  ML_CHECK(out, "held values: null pointer");
  ML_TRY(ffn::check_kept(ffn::kKeepFp8, q, scale, "the tensor"));
  return dispatch_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const bool flat = cols % held::kBlock == 0;
    const int64_t r = flat ? 1 : rows, c = flat ? rows * cols : cols;
    const ffn::ValuesStep<T, ffn::kKeepFp8> step{static_cast<T*>(out), c,
                                                 ffn::make_kept<ffn::kKeepFp8>(q, scale, c)};
    return ffn::launch_rows(cols % 8 == 0 && aligned16(out), ffn::ZeroSource{}, ffn::NoSource{},
                            step, r, c, (hipStream_t)stream);
  });
}
