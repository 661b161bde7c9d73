// i8_gemm.h - the 8-bit products y[m][n] = sum_k q[m][k] w[n][k] on the integer matrix instructions, both operands through LDS.
//
// Workgroup = WM x WN x WK waves (WM along the channels n, WN along the tokens m, WK along the depth); a wave holds TM x TN tiles
// of 16 x 16 in its accumulators (NMAT = 2: TM / 2 tiles of gate and the same of up, whose epilogue joins them). The depth runs
// in stages of 128 WK bytes: both operands' rows of a stage go to LDS by direct loads, whole 128-byte lines, in a ring of NST
// stages issued NST - 1 ahead; one wait and barrier a stage. A stage holds each 8 rows' 128 bytes as a 1 KB block (block b: lane
// l of its load takes row l / 8's 16-byte chunk (l % 8) ^ (l / 8) ^ 4 (b % 2), stored at 16 l), so that the 16 rows x 16 bytes
// of a channel fragment's read lie on distinct banks where a wave has pairs of channel tiles. The other fragments' reads (the tokens',
// and the channels' without pairs) take two lanes to each bank they touch: 4 cycles of conflict a read. Each 64-k step's fragments
// are read one step ahead of its products. With WK > 1 the waves' sums are joined in LDS.
//
// 8192 x 6144 of depth 2048 takes 122 us a call on operands that change from call to call (1.69 POP/s; 112 on the same ones again and
// again, 134 as the profiler times the kernel), 2048 x 4096 of depth 6144 58 to 64 on different cards (1.6 to 1.8): the matrix pipes are
// busy a third of that, the rest is fragment reads out of LDS and the stages' barriers. With few tiles the stages' round trips bound
// it: 61 rows, 2048 channels, depth 6144 9.1 us, of which the bytes are 2.4.
//
// Where a wave has an even number of channel tiles, tiles 2 p and 2 p + 1 share 32 channels so that a lane's 4 rows of the one
// and 4 of the other are 8 consecutive channels, stored at once.
#pragma once
#include "i8_dev.h"

namespace hmoe {

struct I8Out
{
    void* y; int64_t ldy; int dt;
    const float* xs; const float* ws; const float* ws2; const float* bias;
};

// y = the product of one matrix (i8_gemm1.hip), or silu(gate) up in fp32 (i8_gemm2.hip); ldq and ldw below 2^28
int i8_product(const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, int M, int N, int K, const I8Out& o, hipStream_t st);
int i8_gated(const int8_t* q, int64_t ldq, const int8_t* wg, const int8_t* wu, int64_t ldw, int M, int N, int K, const I8Out& o,
             hipStream_t st);

// the same of few rows (i8_few.hip), of x as it is (src: its type; 3: in 8 bits, with the scales o.xs), where i8_few() holds
bool i8_few(int M, int N, int K, int src);
int i8_few_product(const void* x, int src, int64_t ldx, const int8_t* w, int64_t ldw, int M, int N, int K, const I8Out& o, hipStream_t st);
int i8_few_gated(const void* x, int src, int64_t ldx, const int8_t* wg, const int8_t* wu, int64_t ldw, int M, int N, int K, const I8Out& o,
                 hipStream_t st);

// the tile shape of least estimated time: rounds of 256 workgroups, one a CU, each of the tile's f + s depth / 6144
struct I8Pick
{
    int best = -1, grid = 0, seen = 0;
    float least = 0.f;
    void offer(int bn, int bm, float f, float s, int M, int N, int K)
    {
        const int64_t tiles = (int64_t) cdiv(N, bn) * cdiv(M, bm);
        const float t = (float) ((tiles + 255) / 256) * (f + s * (float) K / 6144.0f);
        if (best < 0 || t < least) { best = seen; least = t; grid = (int) (tiles < 256 ? tiles : 256); }
        ++seen;
    }
};

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// C (4 or 8) consecutive channels n .. of token m, at once whatever the row's alignment
template <int DT, int C, typename V>
__device__ __forceinline__ void store_row(const I8Out& o, int m, int n, int N, const V& v)
{
    const size_t at = (size_t) m * o.ldy + n;
    if (n + C <= N)
    {
        if constexpr (DT == HMOE_DT_F32)
        {
            #pragma unroll
            for (int c = 0; c < C; c += 4)
                *(HMOE_GLOBAL f32x4_4*) ((HMOE_GLOBAL float*) o.y + at + c) = (f32x4_4) {v[c], v[c + 1], v[c + 2], v[c + 3]};
        }
        else
        {
            HMOE_GLOBAL uint16_t* to = (HMOE_GLOBAL uint16_t*) o.y + at;
            if constexpr (C == 8)
            {
                if constexpr (DT == HMOE_DT_BF16) *(HMOE_GLOBAL u32x4_2*) to = __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8));
                else *(HMOE_GLOBAL u32x4_2*) to = __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8));
            }
            else
            {
                if constexpr (DT == HMOE_DT_BF16) *(HMOE_GLOBAL u32x2_2*) to = __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4));
                else *(HMOE_GLOBAL u32x2_2*) to = __builtin_bit_cast(u32x2, __builtin_convertvector(v, f16x4));
            }
        }
        return;
    }
    #pragma unroll
    for (int e = 0; e < C; ++e)
        if (n + e < N) store_out(o.y, at + e, v[e], DT);
}

template <int NMAT, int TM, int TN, int WM, int WN, int WK, int NST>
__global__ void __launch_bounds__(64 * WM * WN * WK) __attribute__((amdgpu_waves_per_eu(WM * WN * WK / 4, WM * WN * WK / 4)))
i8_gemm_kernel(const int8_t* __restrict__ q, int64_t ldq, const int8_t* __restrict__ w, const int8_t* __restrict__ w2, int64_t ldw,
               int M, int N, int K, I8Out o)
{
    constexpr int TMO = TM / NMAT, NW = WM * WN * WK, AT = WM * TM, BT = WN * TN, DK = 128 * WK;
    constexpr int NBK = (AT + BT) * 2, NB = NBK * WK, SL = NB / NW;      // 1 KB blocks of 128 bytes of depth and of a stage; a wave's share
    constexpr int BN = 16 * WM * TMO, BM = 16 * WN * TN;
    constexpr bool PAIR = TMO % 2 == 0;
    constexpr int C = PAIR ? 8 : 4;                                      // consecutive channels of a lane
    static_assert(NB % NW == 0 && NW % 2 == 0 && TM % NMAT == 0, "the waves share the staging evenly");
    static_assert(WK == 1 || NW * TM * TN <= NST * NB, "the joined sums take the staging's place");
    __shared__ __attribute__((aligned(16))) u32x4 lds[NST][NB * 64];
    __shared__ __attribute__((aligned(16))) float lxs[BM], lws[NMAT + 1][BN];      // the tile's scales (and bias)
    const int t = threadIdx.x, l = t & 63, row = l & 15;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6), wm = wv % WM, wn = wv / WM % WN, wk = wv / (WM * WN);
    // tiles: each of the 8 XCDs (workgroups go to them in turn) takes a run of neighbouring tiles, GM token tiles deep, so that
    // its L2 holds what they share
    constexpr int GM = 4;
    const int nn = cdiv(N, BN), nm = cdiv(M, BM), total = nn * nm;
    const int KS = cdiv(K, DK);
    const int klast = K - DK * (KS - 1);
    const uint32_t chunk = 16u * (uint32_t) ((l & 7) ^ (l >> 3) ^ ((wv & 1) << 2));
    // the blocks this wave stages, b = wv + NW i: a scalar address of the block's first row (held to the last row of the matrix)
    // and how many of its rows there are; a row or chunk that is not there re-reads the last that is
    const uint8_t* sb[SL];
    int lim[SL];
    const uint32_t vw = (uint32_t) (l >> 3) * (uint32_t) ldw + chunk, vq = (uint32_t) (l >> 3) * (uint32_t) ldq + chunk;
    bool whole = false;
    auto is_w = [&](int i) { return (wv + NW * i) % NBK < 2 * AT; };
    auto place = [&](int tile, int& m0, int& n0) {
        const int per = total >> 3, rest = total & 7, xcd = tile & 7;
        tile = xcd * per + min(xcd, rest) + (tile >> 3);
        const int gsz = GM * nn, grp = tile / gsz, gm = min(GM, nm - grp * GM), in = tile - grp * gsz;
        m0 = (grp * GM + in % gm) * BM;
        n0 = (in / gm) * BN;
        whole = m0 + BM <= M && n0 + BN <= N;
        #pragma unroll
        for (int i = 0; i < SL; ++i)
        {
            const int b = wv + NW * i, tl = (b % NBK) >> 1, r = 8 * (b & 1);
            if (tl < AT)
            {
                const int mat = tl / (WM * TMO), rr = min(n0 + 16 * (tl % (WM * TMO)) + r, N - 1);
                sb[i] = (const uint8_t*) (mat == 0 ? w : w2) + (size_t) rr * ldw;
                lim[i] = min(N - 1 - rr, 7);
            }
            else
            {
                const int rr = min(m0 + 16 * (tl - AT) + r, M - 1);
                sb[i] = (const uint8_t*) q + (size_t) rr * ldq;
                lim[i] = min(M - 1 - rr, 7);
            }
        }
    };
    auto stage = [&](int s) {
        if (s >= KS) return;
        u32x4* buf = lds[s % NST];
        auto put = [&](auto plain) {
            #pragma unroll
            for (int i = 0; i < SL; ++i)
            {
                const int b = wv + NW * i;
                const uint8_t* base = sb[i] + (size_t) DK * s + (decltype(plain)::value ? 128 * (b / NBK) : 0);
                uint32_t v = is_w(i) ? vw : vq;
                if (!decltype(plain)::value)
                {
                    // (the offset is unsigned: the slice's 128 bytes are in it here, so that it stays in the row)
                    const int ld = (int) (is_w(i) ? ldw : ldq), k = 128 * (b / NBK) + (int) chunk;
                    v = (uint32_t) (min(l >> 3, lim[i]) * ld + (s < KS - 1 ? k : min(k, klast - 16)));
                }
                const uint32_t la = __builtin_amdgcn_readfirstlane(
                    (uint32_t) (uintptr_t) (__attribute__((address_space(3))) void*) (buf + b * 64));
    #pragma clang diagnostic push
    #pragma clang diagnostic ignored "-Winline-asm"
                // (an SALU write of M0 needs one wait state before an LDS-DMA load reads it: the s_nop)
                asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(v), "s"(base), "s"(la)
                             : "memory", "m0");
    #pragma clang diagnostic pop
            }
        };
        if (whole && (klast == DK || s < KS - 1)) put(ic<1>{});
        else put(ic<0>{});
    };
    // a token fragment's lane l: row l % 16 of the tile; a channel fragment's the same, or row 8 (r / 4) + r % 4 (+ 4: the odd
    // tile) of the pair's 32, r = l % 16; chunk 4 ks + l / 16
    int fo[2], fa[2];
    #pragma unroll
    for (int ks = 0; ks < 2; ++ks)
    {
        const int ch = 4 * ks + (l >> 4);
        fo[ks] = 64 * (row >> 3) + 8 * (l & 7) + (ch ^ (l & 7) ^ (4 * (row >> 3)));
        fa[ks] = PAIR ? 64 * (row >> 2) + 8 * (row & 3) + (ch ^ (row & 3) ^ (4 * ((row >> 2) & 1))) : fo[ks];
    }
    // (the odd tile's rows are 4 on in their blocks: 32 units, and the chunk's bit 2 the other way)
    const int odd[2] = {32 + ((fa[0] & 4) ? -4 : 4), 32 + ((fa[1] & 4) ? -4 : 4)};
    i32x4 acc[TM][TN];
    u32x4 a[2][TM], bv[2][TN];
    auto read = [&](int s, int ks) {
        const u32x4* cur = lds[s % NST] + wk * NBK * 64;
        #pragma unroll
        for (int i = 0; i < TM; ++i)
        {
            const int tl = (i / TMO) * WM * TMO + wm * TMO + i % TMO;
            a[ks][i] = PAIR ? cur[(tl & ~1) * 128 + fa[ks] + ((i & 1) ? odd[ks] : 0)] : cur[tl * 128 + fa[ks]];
        }
        #pragma unroll
        for (int j = 0; j < TN; ++j) bv[ks][j] = cur[(AT + wn * TN + j) * 128 + fo[ks]];
    };
    auto cut = [&](int ks) {                                       // what lies behind the depth
        const bool z = 128 * wk + 64 * ks + 16 * (l >> 4) >= klast;
        #pragma unroll
        for (int i = 0; i < TM; ++i)
            #pragma unroll
            for (int e = 0; e < 4; ++e) a[ks][i][e] = z ? 0u : a[ks][i][e];
    };
    auto mul = [&](int ks) {
        #pragma unroll
        for (int i = 0; i < TM; ++i)
            #pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = mfma_i8(a[ks][i], bv[ks][j], acc[i][j]);
    };
    // at stage s's barrier stage s + 1 has to have arrived: of the loads issued after it, NST - 2 stages may be under way
    auto arrive = [&](int s) {
        if (NST > 2 && s + NST - 1 < KS) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((NST - 2) * SL) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    int m0, n0;
    place(blockIdx.x, m0, n0);
    #pragma unroll
    for (int s = 0; s < NST - 1; ++s) stage(s);
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x)
    {
        // the tile's scales, in LDS before the stages' barriers and read behind them
        for (int i = t; i < BM + BN; i += 64 * NW)
        {
            if (i < BM) lxs[i] = o.xs[min(m0 + i, M - 1)];
            else
            {
                const int n = min(n0 + i - BM, N - 1);
                lws[0][i - BM] = o.ws[n];
                if (NMAT == 2) lws[1][i - BM] = o.ws2[n];
                lws[NMAT][i - BM] = NMAT == 1 && o.bias ? o.bias[n] : 0.f;
            }
        }
        #pragma unroll
        for (int i = 0; i < TM; ++i)
            #pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = (i32x4) {0, 0, 0, 0};
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        stage(NST - 1);
        read(0, 0);
        if (klast < DK && KS == 1) cut(0);
        for (int s = 0; s < KS; ++s)
        {
            read(s, 1);
            if (klast < DK && s == KS - 1) cut(1);
            mul(0);
            __builtin_amdgcn_sched_group_barrier(0x100, TM + TN, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, TM * TN, 0);
            if (s + 1 < KS)
            {
                arrive(s);                                         // every wave holds stage s in registers; stage s + 1 is here
                stage(s + NST);
                read(s + 1, 0);
                if (klast < DK && s + 1 == KS - 1) cut(0);
            }
            mul(1);
            __builtin_amdgcn_sched_group_barrier(0x100, TM + TN, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, TM * TN, 0);
        }
        __syncthreads();
        const int tm0 = m0, tn0 = n0;
        // the sums of channel group u (of TMO tiles, or pairs) and token tile j become C outputs of one token
        constexpr int UM = PAIR ? TMO / 2 : TMO;
        auto finish = [&](auto dt, int u, int j, const i32x4 (&c)[NMAT][C / 4]) {
            const int lm = 16 * (wn * TN + j) + row, ln = 16 * wm * TMO + 4 * C * u + C * (l >> 4);
            const float xs = lxs[lm];
            typedef float vec __attribute__((ext_vector_type(C)));
            vec v;
            #pragma unroll
            for (int e = 0; e < C; ++e)
            {
                v[e] = (float) c[0][e >> 2][e & 3] * xs * lws[0][ln + e];
                if (NMAT == 2) v[e] = swiglu(v[e], (float) c[NMAT - 1][e >> 2][e & 3] * xs * lws[1][ln + e]);
                else if (o.bias) v[e] += lws[NMAT][ln + e];
            }
            if (tm0 + lm < M && tn0 + ln < N) store_row<decltype(dt)::value, C>(o, tm0 + lm, tn0 + ln, N, v);
        };
        if constexpr (WK > 1)
        {
            // the WK waves' sums of wave column (wm, wn), joined in turn; wave wk finishes groups wk, wk + WK, ..
            i32x4* red = (i32x4*) lds;
            #pragma unroll
            for (int i = 0; i < TM; ++i)
                #pragma unroll
                for (int j = 0; j < TN; ++j) red[(wv * TM * TN + i * TN + j) * 64 + l] = acc[i][j];
            __syncthreads();
            for (int g = wk; g < UM * TN; g += WK)
            {
                const int u = g / TN, j = g % TN;
                i32x4 c[NMAT][C / 4];
                #pragma unroll
                for (int a2 = 0; a2 < NMAT; ++a2)
                    #pragma unroll
                    for (int h = 0; h < C / 4; ++h)
                    {
                        c[a2][h] = (i32x4) {0, 0, 0, 0};
                        #pragma unroll
                        for (int k = 0; k < WK; ++k)
                            c[a2][h] += red[((wm + WM * (wn + WN * k)) * TM * TN + (a2 * TMO + C / 4 * u + h) * TN + j) * 64 + l];
                    }
                if (NMAT == 2 || o.dt == HMOE_DT_F32) finish(ic<HMOE_DT_F32>{}, u, j, c);
                else if (o.dt == HMOE_DT_BF16) finish(ic<HMOE_DT_BF16>{}, u, j, c);
                else finish(ic<HMOE_DT_F16>{}, u, j, c);
            }
            __syncthreads();
        }
        // the next tile's first stages are under way while this one is written
        if (tile + (int) gridDim.x < total)
        {
            place(tile + gridDim.x, m0, n0);
            #pragma unroll
            for (int s = 0; s < NST - 1; ++s) stage(s);
        }
        if constexpr (WK == 1)
        {
            auto all = [&](auto dt) {
                #pragma unroll
                for (int j = 0; j < TN; ++j)
                    #pragma unroll
                    for (int u = 0; u < UM; ++u)
                    {
                        i32x4 c[NMAT][C / 4];
                        #pragma unroll
                        for (int a2 = 0; a2 < NMAT; ++a2)
                            #pragma unroll
                            for (int h = 0; h < C / 4; ++h) c[a2][h] = acc[a2 * TMO + C / 4 * u + h][j];
                        finish(dt, u, j, c);
                    }
            };
            if (NMAT == 2 || o.dt == HMOE_DT_F32) all(ic<HMOE_DT_F32>{});
            else if (o.dt == HMOE_DT_BF16) all(ic<HMOE_DT_BF16>{});
            else all(ic<HMOE_DT_F16>{});
            __syncthreads();                                       // (the scales are read)
        }
    }
}

}  // namespace hmoe
