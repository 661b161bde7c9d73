// i8_gemm2.hip - gate and up in one 8-bit product whose epilogue writes silu(gate) up in fp32: the tile shapes of i8_gemm.h (TM
// counts the tiles of both matrices) and the rule that chooses one.
#include "i8_gemm.h"

namespace hmoe {

// as in i8_gemm1.hip, channels counted in pairs: 2048 tokens, 2048 pairs of depth 6144 take 58 us in 64 x 256 tiles and 59 in
// 128 x 128; 77 tokens 19 us in 16 x 48, 30 in 32 x 128 (by the constants 10.1; 14.3 as the profiler times the kernel alone)
#define HMOE_I8_SHAPES(X)                                                                                              \
    X(2, 1, 1, 1, 8, 3, 2.2f, 3.2f) X(2, 2, 1, 1, 4, 4, 2.6f, 5.2f) X(2, 3, 1, 1, 4, 3, 3.5f, 6.6f)                    \
    X(2, 4, 1, 1, 4, 3, 4.1f, 7.6f) X(2, 4, 2, 1, 4, 2, 3.0f, 11.6f) X(2, 4, 2, 2, 2, 3, 4.4f, 16.8f)                  \
    X(4, 4, 2, 2, 2, 2, 7.2f, 35.1f) X(4, 4, 2, 4, 1, 3, 7.3f, 49.2f) X(6, 4, 2, 4, 1, 2, 10.5f, 64.7f)

int i8_gated(const int8_t* q, int64_t ldq, const int8_t* wg, const int8_t* wu, int64_t ldw, int M, int N, int K, const I8Out& o,
             hipStream_t st)
{
    I8Pick p;
#define HMOE_COST(TM, TN, WM, WN, WK, NST, F, S) p.offer(8 * WM * TM, 16 * WN * TN, F, S, M, N, K);
    HMOE_I8_SHAPES(HMOE_COST)
#undef HMOE_COST
    int i = 0;
#define HMOE_RUN(TM, TN, WM, WN, WK, NST, F, S)                                                                        \
    if (p.best == i++)                                                                                                 \
        i8_gemm_kernel<2, TM, TN, WM, WN, WK, NST><<<p.grid, 64 * WM * WN * WK, 0, st>>>(q, ldq, wg, wu, ldw, M, N, K, o);
    HMOE_I8_SHAPES(HMOE_RUN)
#undef HMOE_RUN
    return HMOE_LAUNCHED("i8 gate and up");
}

}  // namespace hmoe
