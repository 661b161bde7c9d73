// i8_few.hip - the 8-bit products of few rows in one launch: every workgroup brings the rows into 8 bits for itself.
#include "i8_gemm.h"

namespace hmoe {

// y[m][n] of M <= 16 rows (NMAT 2: silu(gate) up in fp32). SRC: the type of x, or 3: x is in 8 bits already, its scales xs.
//
// With few rows the time is that of fetching the weights once, and of everything that comes before and after it. So a workgroup
// asks for x (out of the caches, a few KB) and its weights at once: 16 rows of them (NMAT 2: 8 of gate and 8 of up) by 8 waves that
// share the depth, up to 12 loads of 1 KB a wave. While the weights are on their way it takes each row's largest magnitude and
// leaves its whole numbers in LDS. Then one matrix instruction a load, 16 tokens wide whatever M is, and the 8 waves' sums are
// joined in LDS. A launch of its own for the rows costs about 3 us; in each workgroup they cost M K / 512 values a thread.
//
// HALF (M <= 8): a tile has 8 weight rows, and a load takes 128 bytes of each, whole lines, where 16 rows leave 64 to each. Rows and
// columns 8 .. 15 of the matrix instruction then stand for the second 64 bytes of the same channels and tokens, so that its
// upper left and lower right 8 x 8 are the sums of the one half of the depth and of the other (the rest is not used). 1 token, depth
// 6144: 20000 channels 22.0 us (5.6 TB/s) and 28.1 in 16 rows, 6144 channels 9.5 and 12.3, 256 channels 4.3 and 6.0.
constexpr int FEW_T = 16, FEW_LDS = 48 * 1024, FEW_NW = 8;
template <int NMAT, int SRC, int HALF, int NL>
__global__ void __launch_bounds__(64 * FEW_NW) __attribute__((amdgpu_waves_per_eu(4, 4)))
i8_few_kernel(const void* __restrict__ x, int64_t ldx, const int8_t* __restrict__ w, const int8_t* __restrict__ w2, int64_t ldw, int M, int N,
              int K, I8Out o)
{
    extern __shared__ __attribute__((aligned(16))) int8_t xl[];         // [M][XP]
    __shared__ __attribute__((aligned(16))) i32x4 red[FEW_NW][64];
    __shared__ uint32_t top[FEW_T];
    __shared__ float sx[FEW_T];
    constexpr int TR = 16 >> HALF, TN = TR / NMAT, SB = 64 << HALF;     // weight rows and channels of a tile; depth of a step
    const int t = threadIdx.x, l = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), row = l & (TR - 1);
    const int C = cdiv(K, SB * FEW_NW * NL), S = C * NL;                 // a wave's steps, NL at a time
    const int XP = SB * FEW_NW * S + 16;                                // (+ 16: the 16 rows of a fragment read on distinct banks)
    const int tiles = cdiv(N, TN);
    const int k0 = SB * S * wv + 16 * (l >> 4) + (HALF ? 8 * (l & 8) : 0);
    u32x4 a[NL];
    const int8_t* wr;
    const int om = t / TN, oc = t % TN;                                 // the output of a tile that this thread finishes
    float f1 = 0.f, f2 = 0.f;                                           // its channel's scale, and the second one or the bias
    auto place = [&](int tile) __attribute__((always_inline)) {
        const int n = min(TN * tile + row % TN, N - 1), no = min(TN * tile + oc, N - 1);
        f1 = ldg<float>(o.ws + no);
        if (NMAT == 2) f2 = ldg<float>(o.ws2 + no);
        else if (o.bias) f2 = ldg<float>(o.bias + no);
        wr = (NMAT == 2 && row >= TN ? w2 : w) + (size_t) n * ldw;
    };
    // step s of the wave's slice; a piece behind the depth re-reads the row's last 16 bytes, against values that are zero
    auto fetch = [&](int i, int s) __attribute__((always_inline)) {
        a[i] = __builtin_nontemporal_load((const HMOE_GLOBAL u32x4*) (wr + min(k0 + SB * s, K - 16)));
    };
    auto load = [&]() __attribute__((always_inline)) {
        #pragma unroll
        for (int i = 0; i < NL; ++i) fetch(i, i);
    };
    // (LDS in order, and the loads left on their way)
    auto sync = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const int per = K / 16, pieces = M * per;
    if constexpr (SRC == 3)
    {
        place(blockIdx.x);
        load();
        for (int i = t; i < pieces; i += 64 * FEW_NW)
        {
            const int r = i / per, k = i - r * per;
            *(u32x4*) (xl + r * XP + 16 * k) = ld16((const int8_t*) x + (size_t) r * ldx + 16 * k);
        }
        if (t < M) sx[t] = o.xs[t];
    }
    else
    {
        constexpr int HOLD = NL == 12 ? 1 : 2;                          // pieces of 16 values a thread keeps from one pass to the next
        const size_t lb = (size_t) ldx * (SRC == HMOE_DT_F32 ? 4 : 2);
        float v[HOLD][16];
        #pragma unroll
        for (int h = 0; h < HOLD; ++h)
        {
            const int i = min(t + 64 * FEW_NW * h, pieces - 1), r = i / per;
            load16<SRC>((const uint8_t*) x + r * lb, i - r * per, v[h]);
        }
        __builtin_amdgcn_sched_barrier(0);                              // (loads come back in order: x is not to wait for the weights)
        place(blockIdx.x);
        load();
        __builtin_amdgcn_sched_barrier(0);
        if (t < M) top[t] = 0;
        sync();
        auto largest = [&](const float (&u)[16], int r, bool on) __attribute__((always_inline)) {
            uint32_t m = 0;
            #pragma unroll
            for (int j = 0; j < 16; ++j) m = max(m, mag(u[j]));
            m = on ? m : 0u;
            if (__all(r == __builtin_amdgcn_readfirstlane(r)))
            {
                m = wave_ext_u32<true>(m);
                if (l == 0) atomicMax(&top[r], m);
            }
            else if (on) atomicMax(&top[r], m);
        };
        auto put = [&](const float (&u)[16], int r, int k) __attribute__((always_inline)) {
            const RowQ q = row_q(top[r]);
            if (k == 0) sx[r] = q.s;
            *(u32x4*) (xl + r * XP + 16 * k) = quant16<SRC>(u, q);
        };
        #pragma unroll
        for (int h = 0; h < HOLD; ++h) largest(v[h], min(t + 64 * FEW_NW * h, pieces - 1) / per, t + 64 * FEW_NW * h < pieces);
        for (int i0 = 64 * FEW_NW * HOLD; i0 < pieces; i0 += 64 * FEW_NW)
        {
            const int i = min(i0 + t, pieces - 1), r = i / per;
            float u[16];
            load16<SRC>((const uint8_t*) x + r * lb, i - r * per, u);
            largest(u, r, i0 + t < pieces);
        }
        sync();
        #pragma unroll
        for (int h = 0; h < HOLD; ++h)
        {
            const int i = t + 64 * FEW_NW * h, r = i / per;
            if (i < pieces) put(v[h], r, i - r * per);
        }
        for (int i = 64 * FEW_NW * HOLD + t; i < pieces; i += 64 * FEW_NW)
        {
            const int r = i / per;
            float u[16];
            load16<SRC>((const uint8_t*) x + r * lb, i - r * per, u);
            put(u, r, i - r * per);
        }
    }
    const int pad = XP / 16 - 1 - per;                                  // zeros behind the depth
    for (int i = t; i < M * pad; i += 64 * FEW_NW)
    {
        const int r = i / pad;
        *(u32x4*) (xl + r * XP + 16 * (per + i - r * pad)) = (u32x4) {0u, 0u, 0u, 0u};
    }
    sync();
    const int8_t* xr = xl + min(row, M - 1) * XP + k0;                  // (columns behind the rows: any row, not stored)
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    {
        i32x4 acc = {0, 0, 0, 0};
        const int8_t* xc = xr;
        for (int c = 1; c < C; ++c, xc += SB * NL)
        {
            #pragma unroll
            for (int i = 0; i < NL; ++i)
            {
                acc = mfma_i8(a[i], *(const u32x4*) (xc + SB * i), acc);
                fetch(i, NL * c + i);
            }
        }
        #pragma unroll
        for (int i = 0; i < NL; ++i) acc = mfma_i8(a[i], *(const u32x4*) (xc + SB * i), acc);
        const float g1 = f1, g2 = f2;
        if (tile + (int) gridDim.x < tiles) { place(tile + gridDim.x); load(); }
        red[wv][l] = acc;
        sync();
        const int m = om, n = TN * tile + oc;
        if (m < M && n < N)
        {
            auto sum = [&](int ch) __attribute__((always_inline)) {
                int v = 0;
                #pragma unroll
                for (int k = 0; k < FEW_NW; ++k)
                {
                    v += ((const int*) &red[k][16 * (ch >> 2) + m])[ch & 3];
                    if (HALF) v += ((const int*) &red[k][32 + 16 * (ch >> 2) + 8 + m])[ch & 3];
                }
                return (float) v;
            };
            float v = sum(oc) * sx[m] * g1;
            if (NMAT == 2) v = swiglu(v, sum(TN + oc) * sx[m] * g2);
            else if (o.bias) v += g2;
            store_out(o.y, (size_t) m * o.ldy + n, v, NMAT == 2 ? HMOE_DT_F32 : o.dt);
        }
        sync();
    }
}

struct FewPlan { int half, nl, grid; size_t lds; };
static FewPlan few_plan(int nmat, int M, int N, int K)
{
    FewPlan p;
    p.half = M <= 8;
    // the steps of a wave: at most 12 (half: 6) at a time, in as few turns as that allows
    const int sb = 64 << p.half, top = 12 >> p.half, s = cdiv(K, sb * FEW_NW), per = cdiv(s, cdiv(s, top));
    p.nl = (p.half ? per <= 1 ? 1 : per <= 2 ? 2 : per <= 4 ? 4 : 6 : per <= 2 ? 2 : per <= 4 ? 4 : per <= 8 ? 8 : 12);
    p.lds = (size_t) M * (sb * FEW_NW * p.nl * cdiv(K, sb * FEW_NW * p.nl) + 16);
    // a CU holds two workgroups: two each, or one where that leaves less to the CU with the most
    const int tiles = cdiv(N, (16 >> p.half) / nmat), g = cdiv(tiles, 256) < 2 * cdiv(tiles, 512) ? 256 : 512;
    p.grid = tiles < g ? tiles : g;
    return p;
}

// Where every workgroup's own quantisation costs less than a launch for it. Against that launch and the tiles of i8_gemm1.hip (us,
// N = 6144, depth 2048): 1 row of bf16 5.9 and 9.1, 8 rows 6.7 and 9.5, 12 rows 9.0 and 9.6, 16 rows 10.8 and 9.7; of fp32 (in 64 bits:
// twice the work) 8 rows 8.3 and 9.6, 12 rows 11.6 and 9.7; 16 rows that are in 8 bits already 6.3 and 7.1. Of depth 4096, 8 rows of
// fp32 12.2 and 12.2; of depth 6144, 6 rows of bf16 12.7 and 14.6, 6 of fp32 15.1 and 14.8. The bounds do not look at N: both sides were
// measured at 6144 channels only.
bool i8_few(int M, int N, int K, int src)
{
    if (M > FEW_T || few_plan(1, M, N, K).lds > FEW_LDS) return false;
    if (src == 3) return true;
    return src == HMOE_DT_F32 ? M * K <= (M <= 8 ? 24576 : 16384) : M <= 8 || M * K <= 24576;
}

template <int NMAT>
static int launch_few(const void* x, int src, int64_t ldx, const int8_t* w, const int8_t* w2, int64_t ldw, int M, int N, int K, const I8Out& o,
                      hipStream_t st)
{
    const FewPlan p = few_plan(NMAT, M, N, K);
#define HMOE_N(S, H, L)                                                                                                \
    if (p.half == H && p.nl == L)                                                                                      \
        i8_few_kernel<NMAT, S, H, L><<<p.grid, 64 * FEW_NW, p.lds, st>>>(x, ldx, w, w2, ldw, M, N, K, o);
#define HMOE_F(S)                                                                                                      \
    {                                                                                                                  \
        HMOE_N(S, 0, 2) HMOE_N(S, 0, 4) HMOE_N(S, 0, 8) HMOE_N(S, 0, 12)                                               \
        HMOE_N(S, 1, 1) HMOE_N(S, 1, 2) HMOE_N(S, 1, 4) HMOE_N(S, 1, 6)                                                \
    }
    if (src == 3)
    {
        if constexpr (NMAT == 1) HMOE_F(3)
    }
    else if (src == HMOE_DT_F32) HMOE_F(HMOE_DT_F32)
    else if (src == HMOE_DT_BF16) HMOE_F(HMOE_DT_BF16)
    else HMOE_F(HMOE_DT_F16)
#undef HMOE_F
#undef HMOE_N
    return HMOE_LAUNCHED("i8 few rows");
}

int i8_few_product(const void* x, int src, int64_t ldx, const int8_t* w, int64_t ldw, int M, int N, int K, const I8Out& o, hipStream_t st)
{
    return launch_few<1>(x, src, ldx, w, nullptr, ldw, M, N, K, o, st);
}
int i8_few_gated(const void* x, int src, int64_t ldx, const int8_t* wg, const int8_t* wu, int64_t ldw, int M, int N, int K, const I8Out& o,
                 hipStream_t st)
{
    return launch_few<2>(x, src, ldx, wg, wu, ldw, M, N, K, o, st);
}

}  // namespace hmoe
