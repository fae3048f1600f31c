// The fp32 product's sums before they are joined, for a caller whose next step reads
// them (gemm_f32.hip).
#pragma once

#include "common.h"

namespace mla {
namespace gemmf32 {

// out [splits][M][N] = the parts of a [M, K] times b ([N, K], or [K, N] where b_layout is
// 1): splits of K as the entry points choose them given a workspace.
int sums(int64_t M, int64_t N, int64_t K, const float* a, int64_t lda, const float* b, int64_t ldb,
         int b_layout, float* out, int& splits, hipStream_t st);
int sums_splits(int64_t M, int64_t N, int64_t K);

}  // namespace gemmf32
}  // namespace mla
