// moe8.hip - a whole mixture-of-experts layer for up to 16 tokens, its experts in 8 bits (hmoe_moe8_layer): scores and
// selection, then for each distinct selected expert that is resident (and the shared expert) the gated MLP of i8.hip on the
// tokens that chose it, joined with the routing weights.
#include "i8_dev.h"

namespace hmoe {

constexpr int M8_T = 16, M8_K = 16, M8_E = 512, M8_SIZE = 8192;       // tokens, picks, experts, hidden / intermediate size
constexpr int M8_SLOTS = M8_T * M8_K + 1;                             // distinct experts of a call, the shared one first
constexpr int M8_ROWS = M8_T * (M8_K + 1);                            // (expert, token) rows of a call

struct M8Args
{
    const void* x; int64_t ldx; int xdt;
    const float* wr; const float* bias;
    const int8_t* wg; const int8_t* wu; const int8_t* wd; const float* sg; const float* su; const float* sd;
    const int8_t* hg; const int8_t* hu; const int8_t* hd; const float* hsg; const float* hsu; const float* hsd;   // shared, or null
    int T, H, I, E, n, lo, topk;
    double scale;
    int64_t* sel; float* rw; void* y; int64_t ldy; int ydt;
    // workspace
    double* logits;                 // [T][E]
    int8_t* xq; float* xs;          // [T][up128(H)], [T]
    float* act;                     // [rows][I]: silu(gate) up
    int8_t* qa; float* sa;          // [rows][up128(I)], [rows]
    int* nrows;
};

// ---- scores: one workgroup an expert, sums in 64 bits (scores next to each other decide the selection); behind them one
// workgroup a token, that quantises its row ----
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) m8_route_kernel(M8Args p)
{
    __shared__ double part[4][M8_T];
    __shared__ uint32_t wmax[4];
    const int t = threadIdx.x, es = DT == HMOE_DT_F32 ? 4 : 2;
    const uint8_t* x = (const uint8_t*) p.x;
    if ((int) blockIdx.x >= p.E)
    {
        const int row = blockIdx.x - p.E;
        const uint8_t* xr = x + (size_t) row * p.ldx * es;
        uint32_t m = 0;
        for (int i = t; i < p.H / 16; i += 256)
        {
            float v[16];
            load16<DT, VEC>(xr, i, v);
            #pragma unroll
            for (int j = 0; j < 16; ++j) m = max(m, mag(v[j]));
        }
        m = wave_ext_u32<true>(m);
        if ((t & 63) == 0) wmax[t >> 6] = m;
        __syncthreads();
        const RowQ q = row_q(max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3])));
        if (t == 0) p.xs[row] = q.s;
        for (int i = t; i < p.H / 16; i += 256)
        {
            float v[16];
            load16<DT, VEC>(xr, i, v);
            *(u32x4*) (p.xq + (size_t) row * up128(p.H) + 16 * i) = quant16<DT>(v, q);
        }
        return;
    }
    const float* w = p.wr + (size_t) blockIdx.x * p.H;
    double acc[M8_T];
    #pragma unroll
    for (int r = 0; r < M8_T; ++r) acc[r] = 0.0;
    for (int i = t; i < p.H / 4; i += 256)
    {
        const f32x4 wv = ldg<f32x4>(w + 4 * i);
        #pragma unroll
        for (int r = 0; r < M8_T; ++r)
        {
            if (r >= p.T) break;
            const uint8_t* xr = x + (size_t) r * p.ldx * es;
            #pragma unroll
            for (int j = 0; j < 4; ++j) acc[r] = __builtin_fma((double) load1<DT>(xr, 4 * i + j), (double) wv[j], acc[r]);
        }
    }
    #pragma unroll
    for (int r = 0; r < M8_T; ++r)
    {
        if (r >= p.T) break;
        double v = acc[r];
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
        if ((t & 63) == 0) part[t >> 6][r] = v;
    }
    __syncthreads();
    if (t < p.T) p.logits[(size_t) t * p.E + blockIdx.x] = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
}

// ---- selection: every workgroup of the launches below forms it for itself ----
struct M8Plan
{
    unsigned long long key[M8_E];
    double score[M8_E];
    int sel[M8_T][M8_K];
    double top[M8_T][M8_K];
    int mask[M8_E];                 // tokens that chose a resident expert
    uint16_t slot_of[M8_E];
    uint16_t expert[M8_SLOTS];      // slot -> local id; slot 0 is the shared expert's where there is one
    uint16_t tokens[M8_SLOTS];      // its tokens, a bit each
    uint16_t row0[M8_SLOTS + 1];    // its first row: the row of its token t is row0 + the set bits below t
    float weight[M8_ROWS];
    int slots;
};

__device__ inline unsigned long long order_key(double v)
{
    const unsigned long long b = (unsigned long long) __double_as_longlong(v);
    if (v != v) return 0ull;                                             // NaN behind everything
    return (b >> 63) ? ~b : b | (1ull << 63);
}

// The topk largest score + bias of each token, equal ones in the order of their ids: an expert's place is the number of
// experts before it, counted by the thread that has it
__device__ inline void m8_plan(const M8Args& p, M8Plan& s, bool write)
{
    const int t = threadIdx.x, nt = blockDim.x;
    for (int e = t; e < M8_E; e += nt) s.mask[e] = 0;
    for (int r = 0; r < p.T; ++r)
    {
        __syncthreads();
        for (int e = t; e < p.E; e += nt)
        {
            const double a = 1.0 / (1.0 + exp(-p.logits[(size_t) r * p.E + e]));
            s.score[e] = a;
            s.key[e] = order_key(p.bias ? a + (double) p.bias[e] : a);
        }
        __syncthreads();
        for (int e = t; e < p.E; e += nt)
        {
            const unsigned long long k = s.key[e];
            int place = 0;
            for (int f = 0; f < p.E; ++f) place += s.key[f] > k || (s.key[f] == k && f < e);
            if (place < p.topk)
            {
                s.sel[r][place] = e;
                s.top[r][place] = s.score[e];
                const int id = e - p.lo;
                if (id >= 0 && id < p.n) atomicOr(&s.mask[id], 1 << r);
            }
        }
    }
    __syncthreads();
    if (t == 0)
    {
        int m = 0, row = 0;
        if (p.hg)
        {
            s.expert[0] = 0; s.tokens[0] = (uint16_t) ((1u << p.T) - 1u); s.row0[0] = 0;
            for (int r = 0; r < p.T; ++r) s.weight[r] = 1.0f;
            m = 1; row = p.T;
        }
        for (int id = 0; id < p.n; ++id)
            if (s.mask[id])
            {
                s.expert[m] = (uint16_t) id; s.tokens[m] = (uint16_t) s.mask[id]; s.row0[m] = (uint16_t) row;
                s.slot_of[id] = (uint16_t) m;
                row += __popc(s.mask[id]);
                ++m;
            }
        s.row0[m] = (uint16_t) row;
        s.slots = m;
    }
    __syncthreads();
    for (int i = t; i < p.T * p.topk; i += nt)
    {
        const int r = i / p.topk, j = i - r * p.topk, e = s.sel[r][j], id = e - p.lo;
        double sum = 0.0;
        for (int k = 0; k < p.topk; ++k) sum += s.top[r][k];
        const float w = (float) (p.scale * s.top[r][j] / (sum + 1e-20));
        if (write) { p.sel[i] = e; p.rw[i] = w; }
        if (id >= 0 && id < p.n)
        {
            const int sl = s.slot_of[id];
            s.weight[s.row0[sl] + __popc(s.tokens[sl] & ((1 << r) - 1))] = w;
        }
    }
    __syncthreads();
}

// the sum over the 8 lanes of a group, in each of them
__device__ __forceinline__ int sum8(int v)
{
    v += __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);     // quad_perm [1,0,3,2]
    v += __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);     // quad_perm [2,3,0,1]
    v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);    // row_half_mirror
    return v;
}

// ---- gate and up: tile = 8 gated values of one expert ----
__global__ void __launch_bounds__(512) m8_gate_up_kernel(M8Args p)
{
    __shared__ M8Plan s;
    __shared__ int red[8][2][8][M8_T];
    m8_plan(p, s, blockIdx.x == 0);
    const int t = threadIdx.x, l = t & 63, w = t >> 6, r = l >> 3, pc = l & 7;
    if (blockIdx.x == 0 && t == 0) *p.nrows = s.row0[s.slots];
    const int NB = cdiv(p.I, 8), NC = cdiv(p.H, 128);
    for (int tile = blockIdx.x; tile < s.slots * NB; tile += gridDim.x)
    {
        const int sl = tile / NB, n0 = 8 * (tile - sl * NB), n = min(n0 + r, p.I - 1);
        const bool sh = p.hg && sl == 0;
        const size_t wo = (sh ? 0 : (size_t) s.expert[sl] * p.I * p.H) + (size_t) n * p.H;
        const int8_t* wg = (sh ? p.hg : p.wg) + wo;
        const int8_t* wu = (sh ? p.hu : p.wu) + wo;
        int k = 0;
        for (uint32_t m = s.tokens[sl]; m; m &= m - 1, ++k)
        {
            const int8_t* xr = p.xq + (size_t) __builtin_ctz(m) * up128(p.H);
            int ag = 0, au = 0;
            for (int c = w; c < NC; c += 8)
            {
                const int off = 128 * c + 16 * pc;
                if (off < p.H)
                {
                    const u32x4 xv = ld16(xr + off);
                    ag = dot16(ld16(wg + off), xv, ag);
                    au = dot16(ld16(wu + off), xv, au);
                }
            }
            ag = sum8(ag); au = sum8(au);
            if (pc == 0) { red[w][0][r][k] = ag; red[w][1][r][k] = au; }
        }
        __syncthreads();
        if (t < 8 * k)
        {
            const int rr = t & 7, kk = t >> 3, nn = n0 + rr;
            if (nn < p.I)
            {
                int ag = 0, au = 0;
                for (int v = 0; v < 8; ++v) { ag += red[v][0][rr][kk]; au += red[v][1][rr][kk]; }
                uint32_t m = s.tokens[sl];
                for (int i = 0; i < kk; ++i) m &= m - 1;
                const float xs = p.xs[__builtin_ctz(m)];
                const size_t so = (sh ? 0 : (size_t) s.expert[sl] * p.I) + nn;
                const float g = (float) ag * xs * (sh ? p.hsg : p.sg)[so], u = (float) au * xs * (sh ? p.hsu : p.su)[so];
                p.act[(size_t) (s.row0[sl] + kk) * p.I + nn] = swiglu(g, u);
            }
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) m8_quant_kernel(M8Args p)
{
    __shared__ uint32_t wmax[4];
    const int t = threadIdx.x, row = blockIdx.x;
    if (row >= *p.nrows) return;
    const float* a = p.act + (size_t) row * p.I;
    uint32_t m = 0;
    for (int i = t; i < p.I; i += 256) m = max(m, mag(a[i]));
    m = wave_ext_u32<true>(m);
    if ((t & 63) == 0) wmax[t >> 6] = m;
    __syncthreads();
    const RowQ q = row_q(max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3])));
    if (t == 0) p.sa[row] = q.s;
    for (int i = t; i < p.I / 16; i += 256)
    {
        float v[16];
        load16<HMOE_DT_F32, true>(a, i, v);
        *(u32x4*) (p.qa + (size_t) row * up128(p.I) + 16 * i) = quant16<HMOE_DT_F32>(v, q);
    }
}

// ---- down: tile = 8 output columns, over every expert in the order of its slot ----
__global__ void __launch_bounds__(512) m8_down_kernel(M8Args p)
{
    __shared__ M8Plan s;
    __shared__ float acc[8][8][M8_T];
    m8_plan(p, s, false);
    const int t = threadIdx.x, l = t & 63, w = t >> 6, r = l >> 3, pc = l & 7;
    const int NB = cdiv(p.H, 8), NC = cdiv(p.I, 128);
    for (int tile = blockIdx.x; tile < NB; tile += gridDim.x)
    {
        const int n0 = 8 * tile, n = min(n0 + r, p.H - 1);
        for (int i = t; i < 8 * 8 * M8_T; i += 512) (&acc[0][0][0])[i] = 0.f;
        __syncthreads();
        for (int sl = 0; sl < s.slots; ++sl)
        {
            const bool sh = p.hg && sl == 0;
            const int8_t* wd = (sh ? p.hd : p.wd + (size_t) s.expert[sl] * p.H * p.I) + (size_t) n * p.I;
            const float sd = (sh ? p.hsd : p.sd + (size_t) s.expert[sl] * p.H)[n];
            int row = s.row0[sl];
            for (uint32_t m = s.tokens[sl]; m; m &= m - 1, ++row)
            {
                int a = 0;
                for (int c = w; c < NC; c += 8)
                {
                    const int off = 128 * c + 16 * pc;
                    if (off < p.I) a = dot16(ld16(wd + off), ld16(p.qa + (size_t) row * up128(p.I) + off), a);
                }
                a = sum8(a);
                if (pc == 0) acc[w][r][__builtin_ctz(m)] += (float) a * (p.sa[row] * sd) * s.weight[row];
            }
        }
        __syncthreads();
        if (t < 8 * p.T)
        {
            const int rr = t & 7, tk = t >> 3;
            float v = 0.f;
            for (int k = 0; k < 8; ++k) v += acc[k][rr][tk];
            if (n0 + rr < p.H) store_out(p.y, (size_t) tk * p.ldy + n0 + rr, v, p.ydt);
        }
        __syncthreads();
    }
}

// workspace layout; the parts' offsets into o (or null) and the whole size
static size_t m8_layout(int T, int H, int I, int E, int topk, size_t* o)
{
    const size_t rows = (size_t) T * (topk + 1);
    const size_t part[] = {(size_t) T * E * 8, (size_t) T * up128(H), (size_t) T * 4, rows * I * 4, rows * up128(I), rows * 4, 128};
    size_t at = 0;
    for (int i = 0; i < 7; ++i)
    {
        if (o) o[i] = at;
        at += up128(part[i]);
    }
    return at;
}

}  // namespace hmoe

using namespace hmoe;

extern "C" size_t hmoe_moe8_work_bytes(int T, int H, int I, int E, int topk)
{
    if (T < 1 || T > M8_T || H < 16 || H > M8_SIZE || I < 16 || I > M8_SIZE || E < 1 || E > M8_E || topk < 1 || topk > M8_K) return 0;
    return m8_layout(T, H, I, E, topk, nullptr);
}

extern "C" int hmoe_moe8_layer(const void* x, int x_dtype, int64_t ldx, int T, const float* wr, const float* bias, int E, int topk,
                               double scale, const int8_t* wg, const int8_t* wu, const int8_t* wd, const float* sg, const float* su,
                               const float* sd, int n, int lo, int H, int I, const int8_t* const* sh_w, const float* const* sh_s,
                               int64_t* sel, float* rw, void* y, int y_dtype, int64_t ldy, void* work, void* stream)
{
    if (T == 0) return HMOE_OK;
    const auto dt_ok = [](int d) { return d == HMOE_DT_F32 || d == HMOE_DT_BF16 || d == HMOE_DT_F16; };
    const auto at = [](const void* q, int a) { return q && ((uintptr_t) q & (a - 1)) == 0; };
    HMOE_REQUIRE(T > 0 && T <= M8_T, "moe8_layer: %d tokens: up to %d", T, M8_T);
    HMOE_REQUIRE(H >= 16 && H <= M8_SIZE && H % 16 == 0 && I >= 16 && I <= M8_SIZE && I % 16 == 0,
                 "moe8_layer: hidden size %d, intermediate size %d: multiples of 16 up to %d", H, I, M8_SIZE);
    HMOE_REQUIRE(E >= 1 && E <= M8_E && topk >= 1 && topk <= M8_K && topk <= E, "moe8_layer: %d of %d experts: up to %d of %d", topk, E,
                 M8_K, M8_E);
    HMOE_REQUIRE(n >= 0 && lo >= 0 && lo <= E - n, "moe8_layer: resident experts [%d, %d + %d) of %d", lo, lo, n, E);
    HMOE_REQUIRE(dt_ok(x_dtype) && dt_ok(y_dtype), "moe8_layer: dtype codes %d, %d", x_dtype, y_dtype);
    HMOE_REQUIRE(at(x, x_dtype == HMOE_DT_F32 ? 4 : 2) && ldx >= H && ldx < (1ll << 40) && at(y, y_dtype == HMOE_DT_F32 ? 4 : 2) && ldy >= H &&
                 ldy < (1ll << 40), "moe8_layer: x or output address or row stride (%lld, %lld)", (long long) ldx, (long long) ldy);
    HMOE_REQUIRE(at(wr, 16) && ((uintptr_t) bias & 3) == 0, "moe8_layer: router weights null or not 16-byte aligned, or bias alignment");
    HMOE_REQUIRE(n == 0 || (at(wg, 16) && at(wu, 16) && at(wd, 16) && at(sg, 4) && at(su, 4) && at(sd, 4)),
                 "moe8_layer: expert weights or scales null or not aligned");
    HMOE_REQUIRE((sh_w != nullptr) == (sh_s != nullptr), "moe8_layer: the shared expert's weights without its scales, or the reverse");
    for (int i = 0; sh_w && i < 3; ++i)
        HMOE_REQUIRE(at(sh_w[i], 16) && at(sh_s[i], 4), "moe8_layer: shared expert: weights or scales null or not aligned");
    HMOE_REQUIRE(at(sel, 8) && at(rw, 4) && at(work, 128), "moe8_layer: sel, rw or workspace null or not aligned");
    {
        const int ex = x_dtype == HMOE_DT_F32 ? 4 : 2, ey = y_dtype == HMOE_DT_F32 ? 4 : 2;
        const uintptr_t x0 = (uintptr_t) x, x1 = x0 + ((T - 1) * ldx + H) * ex, y0 = (uintptr_t) y, y1 = y0 + ((T - 1) * ldy + H) * ey;
        HMOE_REQUIRE(x1 <= y0 || y1 <= x0, "moe8_layer: the output overlaps x");
    }
    size_t o[7];
    m8_layout(T, H, I, E, topk, o);
    uint8_t* b = (uint8_t*) work;
    M8Args p = {x, ldx, x_dtype, wr, bias, wg, wu, wd, sg, su, sd,
                sh_w ? sh_w[0] : nullptr, sh_w ? sh_w[1] : nullptr, sh_w ? sh_w[2] : nullptr,
                sh_s ? sh_s[0] : nullptr, sh_s ? sh_s[1] : nullptr, sh_s ? sh_s[2] : nullptr,
                T, H, I, E, n, lo, topk, scale, sel, rw, y, ldy, y_dtype,
                (double*) (b + o[0]), (int8_t*) (b + o[1]), (float*) (b + o[2]), (float*) (b + o[3]), (int8_t*) (b + o[4]),
                (float*) (b + o[5]), (int*) (b + o[6])};
    const hipStream_t st = (hipStream_t) stream;
    const bool vec = ((uintptr_t) x & 15) == 0 && (ldx * (x_dtype == HMOE_DT_F32 ? 4 : 2)) % 16 == 0;
#define HMOE_R(D, V) m8_route_kernel<D, V><<<E + T, 256, 0, st>>>(p)
    if (x_dtype == HMOE_DT_F32) { if (vec) HMOE_R(HMOE_DT_F32, true); else HMOE_R(HMOE_DT_F32, false); }
    else if (x_dtype == HMOE_DT_BF16) { if (vec) HMOE_R(HMOE_DT_BF16, true); else HMOE_R(HMOE_DT_BF16, false); }
    else { if (vec) HMOE_R(HMOE_DT_F16, true); else HMOE_R(HMOE_DT_F16, false); }
#undef HMOE_R
    m8_gate_up_kernel<<<1024, 512, 0, st>>>(p);
    m8_quant_kernel<<<T * (topk + 1), 256, 0, st>>>(p);
    m8_down_kernel<<<cdiv(H, 8), 512, 0, st>>>(p);
    return HMOE_LAUNCHED("moe8 layer");
}
