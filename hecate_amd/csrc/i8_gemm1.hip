// i8_gemm1.hip - the 8-bit product of one matrix: the tile shapes of i8_gemm.h and the rule that chooses one.
#include "i8_gemm.h"

namespace hmoe {

// Measured on full grids of 256 workgroups (one a CU) at depths 1024 and 6144, weights from memory: the time of a tile is f + s
// depth / 6144 microseconds. Small tiles spread few rows over the chip and split the depth over the waves of a workgroup; large
// ones read each operand less often. 16 x 16: 5.8 us at depth 6144 on 256 tiles (with 32 x 64 tiles the same product takes a
// quarter of the workgroups and 11.8); 2048 x 4096 outputs of depth 6144: 57.8 us in 128 x 256 tiles, 70 in 192 x 256 (176 of
// them), 78 in 128 x 128; 8192 x 6144 of depth 2048: 115 in 192 x 256, 130 in 128 x 256, 190 in 128 x 128 (on the same operands again
// and again). The constants rank the shapes; they are no launch's duration. A profiler shows 2 to 4 us more for the small ones: 9.1 us
// for 61 x 2048 of depth 6144 (5.2 here), 9.5 for 333 x 1501 of depth 1360 (6.1), 9.7 for 77 x 6144 of depth 2048 (7.4); large ones
// are within a tenth.
#define HMOE_I8_SHAPES(X)                                                                                              \
    X(1, 1, 1, 1, 8, 3, 1.5f, 2.4f) X(2, 1, 1, 1, 8, 3, 2.2f, 3.0f) X(1, 2, 1, 1, 8, 3, 2.4f, 3.2f)                    \
    X(2, 2, 1, 1, 4, 4, 2.7f, 5.0f)                                                                                    \
    X(1, 4, 2, 1, 4, 3, 2.8f, 7.0f) X(2, 4, 2, 1, 4, 2, 3.5f, 11.7f) X(2, 4, 2, 2, 2, 3, 5.1f, 16.9f)                  \
    X(4, 4, 2, 2, 2, 2, 7.2f, 35.1f) X(4, 4, 2, 4, 1, 3, 8.3f, 49.8f) X(6, 4, 2, 4, 1, 2, 11.5f, 64.7f)

int i8_product(const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, int M, int N, int K, const I8Out& o, hipStream_t st)
{
    I8Pick p;
#define HMOE_COST(TM, TN, WM, WN, WK, NST, F, S) p.offer(16 * WM * TM, 16 * WN * TN, F, S, M, N, K);
    HMOE_I8_SHAPES(HMOE_COST)
#undef HMOE_COST
    int i = 0;
#define HMOE_RUN(TM, TN, WM, WN, WK, NST, F, S)                                                                        \
    if (p.best == i++)                                                                                                 \
        i8_gemm_kernel<1, TM, TN, WM, WN, WK, NST><<<p.grid, 64 * WM * WN * WK, 0, st>>>(q, ldq, w, nullptr, ldw, M, N, K, o);
    HMOE_I8_SHAPES(HMOE_RUN)
#undef HMOE_RUN
    return HMOE_LAUNCHED("i8 product");
}

}  // namespace hmoe
