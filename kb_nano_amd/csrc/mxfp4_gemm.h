// Arguments of the MXFP4 product's kernels (mxfp4_gemm.hip).
#pragma once

#include "mxfp4.h"

namespace kbn {

struct MxGemmArgs {
    const uint8_t* A;    // codes [M, K/2]
    int64_t lda;
    const uint8_t* sA;   // scale bytes [M, K/32]
    int64_t ld_sa;
    const uint8_t* W;    // codes [N, K/2]
    int64_t ldw;
    const uint8_t* sW;
    int64_t ld_sw;
    uint16_t* D;
    int64_t ldd;
    int M, N, K;
    int tiles_m, tiles_n;
    int splits, groups_per_split;   // K split in runs of whole 512-K groups
    float* P;                       // [splits][tiles][BM][BN] partial sums (splits > 1)
    const void* X;                  // bf16 or fp16 rows, quantized by the kernel itself (lda: their stride)
};

// What a call launches: the tiled kernel (rf = 0), or the one for few rows with
// 16 rf weight rows a workgroup.
struct MxPlan {
    int bm, bn, splits, rf;
};
MxPlan mxfp4_plan(int64_t M, int64_t N, int64_t K);
// Bytes of the partial sums.
int64_t mxfp4_plan_bytes(const MxPlan& plan, int64_t M, int64_t N);

// Rows of values that the few-rows kernel's variant for M of them holds.
inline int mxfp4_value_rows(int64_t M) { return M <= 2 ? 2 : M <= 4 ? 4 : M <= 8 ? 8 : 16; }

int mxfp4_rows_launch(const MxGemmArgs& p, int rf, int x_dtype, hipStream_t st);
int mxfp4_gemm_launch(MxGemmArgs& p, float* slabs, hipStream_t st);

}  // namespace kbn
