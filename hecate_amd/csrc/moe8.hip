// moe8.hip - a whole mixture-of-experts layer for up to 16 tokens, its experts in 8 bits (hmoe_moe8_layer), in two launches:
// the scores and the tokens in 8 bits; then the selection, and for each distinct selected expert that is resident (and the
// shared expert) the gated MLP of i8.hip on the tokens that chose it, joined with the routing weights.
#include "i8_dev.h"

namespace hmoe {

constexpr int M8_T = 16, M8_K = 16, M8_E = 512, M8_H = 7168, M8_I = 4096;      // tokens, picks, experts, hidden and intermediate size
constexpr int M8_SLOTS = M8_T * M8_K + 1;                             // distinct experts of a call, the shared one first
constexpr int M8_ROWS = M8_T * (M8_K + 1);                            // (expert, token) rows of a call
constexpr int M8_SUB = 8, M8_COPY = 32;                               // parts of a slot's count, copies of the rows' scales
constexpr int M8_SYNC = 32 + 32 * M8_SUB * M8_SLOTS + M8_COPY * M8_ROWS;         // the claim counter, the slots' counts (a line each), the scales

struct M8Args
{
    const void* x; int64_t ldx; int xdt;
    const float* wr; const float* bias;
    const int8_t* wg; const int8_t* wu; const int8_t* wd; const float* sg; const float* su; const float* sd;
    const int8_t* hg; const int8_t* hu; const int8_t* hd; const float* hsg; const float* hsu; const float* hsd;   // shared, or null
    int64_t dg, du, dd, dsd;        // the shared expert's hg - wg, hu - wu, hd - wd, hsd - sd, in bytes
    int T, H, I, E, n, lo, topk;
    double scale;
    int64_t* sel; float* rw; void* y; int64_t ldy; int ydt;
    // workspace
    double* logits;                 // [T][E]
    int8_t* xq; float* xs;          // [T][up128(H)], [T]
    float* act;                     // [rows][I]: silu(gate) up
    int8_t* qa;                     // [rows][up128(I)]
    int* ticket; int* count;        // the next claim; of each slot, gate/up tiles done, in M8_SUB parts, a line each
    uint32_t* up;                   // [M8_COPY][M8_ROWS]: a quantised row's scale with the sign set, 0 before
};

// ---- scores: one workgroup an expert, sums in 64 bits (scores next to each other decide the selection); behind them one
// workgroup a token, that quantises its row. Bound by the round trip of the router's rows (6.3 MB of 256 x 6144): 5.2 us at one
// token, 9.3 at 16 ----
template <int DT, int NI>
__global__ void __launch_bounds__(256) m8_route_kernel(M8Args p)
{
    __shared__ double part[4][M8_T];
    __shared__ uint32_t wmax[4];
    const int t = threadIdx.x, es = DT == HMOE_DT_F32 ? 4 : 2;
    const uint8_t* x = (const uint8_t*) p.x;
    // (ticket, count, up: one array; by every workgroup: the tokens' own took 6 us for it at one token)
    for (int i = blockIdx.x * 256 + t; i < M8_SYNC; i += gridDim.x * 256) p.ticket[i] = 0;
    if ((int) blockIdx.x >= p.E)
    {
        const int row = blockIdx.x - p.E;
        const uint8_t* xr = x + (size_t) row * p.ldx * es;
        uint32_t m = 0;
        for (int i = t; i < p.H / 16; i += 256)
        {
            float v[16];
            load16<DT>(xr, i, v);
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
            load16<DT>(xr, i, v);
            *(u32x4*) (p.xq + (size_t) row * up128(p.H) + 16 * i) = quant16<DT>(v, q);
        }
        return;
    }
    // the expert's whole row is asked for at once (NI = H / 1024 rounded up loads a thread; a load at a time took 10.5 us of 256 x 6144
    // and one token), then four tokens at a time
    const float* w = p.wr + (size_t) blockIdx.x * p.H;
    const bool last = t + 256 * (NI - 1) < p.H / 4;                      // whether this thread has a part in the last load
    f32x4 wv[NI];
    #pragma unroll
    for (int g = 0; g < NI; ++g) wv[g] = ldg<f32x4>(w + 4 * min(t + 256 * g, p.H / 4 - 1));
    auto tokens = [&](auto many, int r0) __attribute__((always_inline)) {
        constexpr int R = decltype(many)::value;
        float v[R][NI][4];
        #pragma unroll
        for (int k = 0; k < R; ++k)
            #pragma unroll
            for (int g = 0; g < NI; ++g)
                load4<DT>(x + (size_t) min(r0 + k, p.T - 1) * p.ldx * es, min(t + 256 * g, p.H / 4 - 1), v[k][g]);
        double acc[R];
        #pragma unroll
        for (int k = 0; k < R; ++k)
        {
            acc[k] = 0.0;
            #pragma unroll
            for (int g = 0; g < NI; ++g)
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const double c = __builtin_fma((double) v[k][g][j], (double) wv[g][j], acc[k]);
                    acc[k] = g < NI - 1 || last ? c : acc[k];
                }
        }
        for (int o = 32; o > 0; o >>= 1)
        {
            #pragma unroll
            for (int k = 0; k < R; ++k) acc[k] += __shfl_xor(acc[k], o);
        }
        if ((t & 63) == 0)
        {
            #pragma unroll
            for (int k = 0; k < R; ++k)
                part[t >> 6][r0 + k] = acc[k];
        }
    };
    if (p.T == 1) tokens(ic<1>{}, 0);
    else
        for (int r0 = 0; r0 < p.T; r0 += 4) tokens(ic<4>{}, r0);
    static_assert(M8_T % 4 == 0, "part's room");
    __syncthreads();
    if (t < p.T) p.logits[(size_t) t * p.E + blockIdx.x] = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
}

// ---- the plan: which experts run on which tokens; every workgroup of the experts' kernel forms it for itself ----
struct M8Plan
{
    int sel[M8_T][M8_K];
    double top[M8_T][M8_K];
    int mask[M8_E];                 // tokens that chose a resident expert
    uint16_t slot_of[M8_E];
    uint16_t expert[M8_SLOTS];      // slot -> local id; slot 0 is the shared expert's where there is one
    uint16_t tokens[M8_SLOTS];      // its tokens, a bit each
    uint16_t row0[M8_SLOTS + 1];    // its first row: the row of its token t is row0 + the set bits below t
    float weight[M8_ROWS];
    float xs[M8_T];
    uint32_t scan[8];
    uint16_t batch[M8_SLOTS + 2];   // a down tile's batches: batch b holds the slots from batch[b] to batch[b + 1]
    int slots, batches;
};

// a number ordered as the scores are, NaN behind everything
__device__ inline unsigned long long order_key(double v)
{
    const unsigned long long b = (unsigned long long) __double_as_longlong(v);
    if (v != v) return 0ull;
    return (b >> 63) ? ~b : b | (1ull << 63);
}

// The topk largest score + bias of token r by one wave: expert e is with lane e % 64, and each round takes the largest key left
// and of equal ones the lowest id
template <int EL>
__device__ inline void m8_select(const M8Args& p, M8Plan& s, int r)
{
    const int l = threadIdx.x & 63;
    double a[EL];
    float bs[EL];
    unsigned long long k[EL];
    // (every load asked for before any is used: a round trip each would be most of the plan's time)
    #pragma unroll
    for (int i = 0; i < EL; ++i)
    {
        const int e = min(64 * i + l, p.E - 1);
        a[i] = ldg<double>(p.logits + (size_t) r * p.E + e);
        bs[i] = ldg<float>(p.bias ? p.bias + e : p.wr);
    }
    #pragma unroll
    for (int i = 0; i < EL; ++i) asm volatile("" : "+v"(a[i]), "+v"(bs[i]));
    #pragma unroll
    for (int i = 0; i < EL; ++i)
    {
        a[i] = 1.0 / (1.0 + exp(-a[i]));
        const unsigned long long o = order_key(p.bias ? a[i] + (double) bs[i] : a[i]);
        k[i] = 64 * i + l < p.E ? o + 1ull : 0ull;                       // (the largest key is infinity's: + 1 does not wrap)
    }
    for (int j = 0; j < p.topk; ++j)
    {
        // the lane's best (of equal keys the lowest id, 0: none left), then the wave's: by the keys' upper halves, where those tie
        // by the lower ones, and then by the ids
        unsigned long long bk = k[0];
        double ba = a[0];
        int bi = 0;
        #pragma unroll
        for (int i = 1; i < EL; ++i)
        {
            const bool gt = k[i] > bk;
            bk = gt ? k[i] : bk; ba = gt ? a[i] : ba; bi = gt ? i : bi;
        }
        const uint32_t hi = wave_ext_u32<true>((uint32_t) (bk >> 32));
        bool c = (uint32_t) (bk >> 32) == hi;
        unsigned long long who = __ballot(c);
        if (who & (who - 1))
        {
            const uint32_t lo = wave_ext_u32<true>(c ? (uint32_t) bk : 0u);
            c = c && (uint32_t) bk == lo;
            const int e = (int) wave_ext_u32<false>(c ? (uint32_t) (64 * bi + l) : 0x7fffffffu);
            who = 1ull << (e & 63);
        }
        if (l == __builtin_ctzll(who))
        {
            s.sel[r][j] = 64 * bi + l;
            s.top[r][j] = ba;
            #pragma unroll
            for (int i = 0; i < EL; ++i) k[i] = i == bi ? 0ull : k[i];
        }
    }
}

__device__ inline void m8_plan(const M8Args& p, M8Plan& s, bool write)
{
    const int t = threadIdx.x, l = t & 63, nw = blockDim.x / 64;
    for (int e = t; e < M8_E; e += blockDim.x) s.mask[e] = 0;
    const int lt = t - (int) blockDim.x + 64;
    if (lt >= 0 && lt < p.T) s.xs[lt] = p.xs[lt];                        // (the last wave too)
    for (int r = nw - 1 - (t >> 6); r < p.T; r += nw)                    // (the last waves first: they stream nothing)
    {
        if (p.E <= 256) m8_select<4>(p, s, r);
        else m8_select<8>(p, s, r);
    }
    __syncthreads();
    for (int i = t; i < p.T * p.topk; i += blockDim.x)
    {
        const int r = i / p.topk, id = s.sel[r][i - r * p.topk] - p.lo;
        if (id >= 0 && id < p.n) atomicOr(&s.mask[id], 1 << r);
    }
    __syncthreads();
    // slots in the order of the ids: a running count of (experts, rows) over them
    const int m = t < M8_E ? s.mask[t] : 0;
    uint32_t c = t < M8_E ? ((m != 0 ? 1u : 0u) << 16) + (uint32_t) __popc(m) : 0u;
    const uint32_t own = c;
    for (int o = 1; o < 64; o <<= 1)
    {
        const uint32_t v = __shfl_up(c, o);
        c += l >= o ? v : 0u;
    }
    if (l == 63 && t < M8_E) s.scan[t >> 6] = c;
    __syncthreads();
    uint32_t before = 0, all = 0;
    #pragma unroll
    for (int i = 0; i < M8_E / 64; ++i)
    {
        before += i < (t >> 6) ? s.scan[i] : 0u;
        all += s.scan[i];
    }
    const int s0 = p.hg ? 1 : 0, r0 = p.hg ? p.T : 0;
    if (t < M8_E && m)
    {
        const uint32_t at = before + c - own;
        const int sl = s0 + (int) (at >> 16);
        s.expert[sl] = (uint16_t) t; s.tokens[sl] = (uint16_t) m; s.row0[sl] = (uint16_t) (r0 + (int) (at & 0xffffu));
        s.slot_of[t] = (uint16_t) sl;
    }
    if (t == 0)
    {
        s.slots = s0 + (int) (all >> 16);
        s.row0[s.slots] = (uint16_t) (r0 + (int) (all & 0xffffu));
        if (p.hg) { s.expert[0] = 0; s.tokens[0] = (uint16_t) ((1u << p.T) - 1u); s.row0[0] = 0; }
    }
    if (p.hg && t < p.T) s.weight[t] = 1.0f;
    __syncthreads();
    for (int i = t; i < p.T * p.topk; i += blockDim.x)
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

// the sum over the 8 lanes of a group, in each of them. v comes out of integer dot products, whose result another instruction
// may read three wait states later at the earliest. The compiler sees to that, copies that it makes itself included; the wait is
// written out as well, from when a sum came out without its last product. (Followed along every path of the assembly of all the
// kernels here, no result of a dot product is read earlier, with this wait or without it)
__device__ __forceinline__ int sum8(int v)
{
    asm volatile("s_nop 2" : "+v"(v));
    v += __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);     // quad_perm [1,0,3,2]
    v += __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);     // quad_perm [2,3,0,1]
    v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);    // row_half_mirror
    return v;
}

// an address that is the same in every lane, in scalar registers
template <typename T> __device__ __forceinline__ const T* scalar(const T* q)
{
    const uint64_t v = (uint64_t) (uintptr_t) q;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t) v), hi = __builtin_amdgcn_readfirstlane((uint32_t) (v >> 32));
    return (const T*) (uintptr_t) (lo | ((uint64_t) hi << 32));
}
// 16 bytes of a weight, read once, at a scalar address and the lane's offset
__device__ __forceinline__ u32x4 ldw16_at(const void* base, uint32_t off)
{
    return __builtin_nontemporal_load((const HMOE_GLOBAL u32x4*) ((const HMOE_GLOBAL char*) base + off));
}

// ---- the experts, gate and up to the weighted sum, in one launch ----
// One workgroup a CU: 8 waves that stream weights, one that finishes what they sum and one that brings what they need next. The
// work is a list of tickets, taken in order through one counter: first the gate/up tiles (8 TR gated values of one expert: slot
// after slot, the shared expert first), then the down tiles (8 output columns, over every slot, a batch of slots at a time).
//
// Once a slot's gate/up tiles are counted, its rows are quantised, each by one workgroup, and their scales shown; a down batch waits
// for its rows' scales. Those come from earlier claims alone, which are held by workgroups that run already; a workgroup waits for
// none before all its gate/up tiles are counted, and quantises what is left to it while it waits. So every wait ends, whatever else is
// on the card and however many of this launch's workgroups have started (all the same it is bounded: past the bound the output is
// NaN).
//
// Weights are read 8 rows x 128 bytes a load, each wave its own slice of the depth, and multiplied by 4-wide integer dot
// products with the tokens' values out of LDS: an expert has one or two tokens of a step, for which a matrix instruction would
// be mostly empty, and whole lines arrive faster from memory than a matrix fragment's order (16 rows x 64 bytes): 7.0 against
// 5.7 TB/s over 3.2 GB. A wave holds one item's loads (8 to 14 KB) and asks for the next item's line as soon as it has used
// one. Two items deep it is no faster (7.1 TB/s either way over 2.5 GB of expert tiles), and a round trip of the other two
// waves, whose loads return in the order of the workgroup's, takes 6 us in place of 1.4: longer than an item. The streaming
// waves load nothing else for the same reason, and the other two use what they ask for an item later.
//
// Measured with 256 experts of 6144 x 2048, top 8 and a shared one: 1 token 69 us of 340 MB (6.5 TB/s while it streams; 9 us go
// before the first bytes, 5 between gate/up and down), 16 tokens 536 us of the 3.3 GB of 86 distinct experts (6.1 TB/s).
// With 5 tokens and experts of 2048 x 1408 (100 MB) the two gaps are half of 43 us.
//
// A wave's whole numbers are exact; those of a down tile are scaled and added slot by slot in fp32, then over the 8 waves: the
// same order every time.
constexpr int M8_ARENA = 148 * 1024, M8_RQ = 32;                        // LDS of x, sums and quantised rows; rows of a batch

template <int NS, int TR, int NSD>
__global__ void __launch_bounds__(640) m8_experts_kernel(M8Args p)
{
    constexpr int NG2 = 2 * NS * TR, SU = NG2 / NSD < 6 ? (NG2 / NSD > 0 ? NG2 / NSD : 1) : 6;     // (slot, 8 rows) pairs of a down item
    constexpr int NL = NG2;                                             // loads of an item
    static_assert(SU * NSD <= NL, "a down item fits the registers of a gate/up one");
    constexpr int XP = 1024 * NS, ROWS = 16 * TR, QP = 1024 * NSD;      // LDS row of x; rows of a gate/up tile; LDS row of a batch
    constexpr int RDM = NSD == 4 ? 2 : SU < 3 ? SU : 3;                 // 8-row groups of a down tile, at most
    static_assert(M8_T * (XP + 64 * ROWS) <= M8_ARENA && M8_T * (2 * QP + 512 * RDM) <= M8_ARENA, "LDS");
    __shared__ M8Plan s;
    __shared__ __attribute__((aligned(16))) int8_t arena[M8_ARENA];
    __shared__ float fq[2][M8_RQ];
    __shared__ uint16_t duty[M8_ROWS];                                  // the rows this workgroup is to quantise: M8_T slot + its number there
    __shared__ int tk[8], late;
    const int t = threadIdx.x, l = t & 63, r = l >> 3, pc = l & 7;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int T = p.T, IP = (int) up128(p.I), HP = (int) up128(p.H);
    // x [T][XP] and partial sums [2][8][ROWS][T]; a down tile's sums [2][8][8 RD][T] and the batches' rows [2][rq][QP]: side by
    // side, or the later ones in the earlier ones' place
    const int xr_bytes = T * (XP + 64 * ROWS), acc_bytes = 512 * min(cdiv(p.H, 8 * 256), RDM) * T;
    const bool apart = xr_bytes + acc_bytes + 2 * T * QP <= M8_ARENA;
    const int after = (apart ? xr_bytes : 0) + acc_bytes;
    int8_t* xl = arena;
    int* red = (int*) (arena + T * XP);
    float* accl = (float*) (arena + after - acc_bytes);
    int8_t* qb = arena + after;
    const int rq = min((M8_ARENA - after) / (2 * QP), M8_RQ);
    auto claim = [&]() { return __hip_atomic_fetch_add(p.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    if (t == 0) tk[0] = claim();
    for (int i = t; i < T * (XP / 16); i += 640)
    {
        const int tok = i / (XP / 16), k = 16 * (i - tok * (XP / 16));
        *(u32x4*) (xl + tok * XP + k) = k < p.H ? ld16(p.xq + (size_t) tok * HP + k) : (u32x4) {0u, 0u, 0u, 0u};
    }
    const int NB = cdiv(p.I, 8 * TR);
    // a streaming wave's slice of the depth is NS (gate, up) or NSD (down) lines of 128 bytes from line w NS (w NSD) on; a piece
    // behind the depth re-reads the row's last 16 bytes, against values that are zero. Rows come in whole groups of 8 (H and I
    // are multiples of 16), so that a load is a scalar address and one of these lane offsets
    uint32_t vo[NS], vd[NSD];
    #pragma unroll
    for (int i = 0; i < NS; ++i) vo[i] = (uint32_t) (r * p.H + min(128 * (w * NS + i) + 16 * pc, p.H - 16));
    #pragma unroll
    for (int i = 0; i < NSD; ++i) vd[i] = (uint32_t) (r * p.I + min(128 * (w * NSD + i) + 16 * pc, p.I - 16));
    u32x4 a[NL];
    float sd[SU];
    // (the shared expert's matrices as distances from the others: a choice between two kernel arguments became a choice of which to
    // load, and that load went the weights' way, behind all of them)
    struct GuAt { const int8_t* g[TR]; const int8_t* u[TR]; };
    auto gu_at = [&](int expert, int blk) {                              // expert -1: the shared one
        GuAt o;
        const int64_t eo = (int64_t) expert * p.I * p.H;
        const uintptr_t g = (uintptr_t) p.wg + (expert < 0 ? p.dg : eo), u = (uintptr_t) p.wu + (expert < 0 ? p.du : eo);
        #pragma unroll
        for (int tr = 0; tr < TR; ++tr)
        {
            const size_t ro = (size_t) min(TR * blk + tr, p.I / 8 - 1) * 8 * p.H;
            o.g[tr] = scalar((const int8_t*) (g + ro));
            o.u[tr] = scalar((const int8_t*) (u + ro));
        }
        return o;
    };
    auto load_gu = [&](const GuAt& at, int i, int tr) {                  // line i of group tr of both
        a[tr * NS + i] = ldw16_at(at.g[tr], vo[i]);
        a[(TR + tr) * NS + i] = ldw16_at(at.u[tr], vo[i]);
    };
    __syncthreads();
    // the shared expert's first tiles need no plan: their weights come while it is made
    const int first = __builtin_amdgcn_readfirstlane(tk[0]);
    const bool early = p.hg && T <= 2 && first < min(NB, 256);           // (more tokens are selected by the streaming waves too)
    if (early && w < 8)
    {
        const GuAt at = gu_at(-1, first);
        #pragma unroll
        for (int i = 0; i < NS; ++i)
            #pragma unroll
            for (int tr = 0; tr < TR; ++tr) load_gu(at, i, tr);
    }
    m8_plan(p, s, blockIdx.x == 0);
    const int slots = __builtin_amdgcn_readfirstlane(s.slots);
    // a down tile: as many 8-row groups as give each of 256 workgroups one, so that the slots quantised last come last in it
    const int RD = min(cdiv(p.H, 8 * 256), RDM);
    const int NG = slots * NB, total = NG + cdiv(p.H, 8 * RD);
    // claims, one atomic each: the first 256 stand for `run` gate/up tiles, 256 apart (so that all work on the same slot), the
    // others for one ticket. (A claim for each tile from every workgroup kept one line of memory busy for longer than the tile)
    const int run = max(NG / 256 - 1, 1);
    auto ticket_of = [&](int c) { return c < 256 ? c : 256 * (run - 1) + c; };
    int nb = 0;                                                         // batches of a down tile (from the first barrier below on)

    // an item: a gate/up tile (batch < 0) or one batch of a down tile; d counts the down items
    struct Item { int ticket, seq, slot, blk, batch, d; };
    auto item = [&](int ticket, int seq, int d) {
        Item it = {ticket, seq, 0, 0, -1, d};
        if (ticket < NG) { it.slot = (int) ((uint32_t) ticket / (uint32_t) NB); it.blk = ticket - it.slot * NB; }
        else { it.blk = ticket - NG; it.batch = 0; ++it.d; }
        return it;
    };
    auto next = [&](const Item& c) {
        if (c.batch >= 0 && c.batch + 1 < nb) { Item it = c; ++it.batch; ++it.d; return it; }
        return item(__builtin_amdgcn_readfirstlane(tk[(c.seq + 1) & 7]), c.seq + 1, c.d);
    };
    // between the last gate/up tile and the first down batch: what was not ready then is brought, and may wait for this
    // workgroup's own tiles
    auto turns = [&](const Item& c, const Item& n) { return c.batch < 0 && n.batch >= 0 && n.ticket < total; };
    auto turn = [&](const Item& c, const Item& n) {
        if (!turns(c, n) || !__builtin_amdgcn_readfirstlane(late)) return;
        if (!apart) __syncthreads();
        __syncthreads();
    };
    const int start = ticket_of(first);
    Item cur = item(start, 0, 0);

    if (w == 9)
    {
        // the bringing wave: tickets, and the rows of the next down batch
        // (each workgroup looks at one of 32 copies of the rows' scales: a line that all of them read past their caches is served to
        // one after the other)
        const uint32_t* up = p.up + (blockIdx.x % M8_COPY) * M8_ROWS;
        bool lost = false;
        auto ask = [&](const Item& it, uint32_t& v) __attribute__((always_inline)) {                    // whether the batch's rows are there; their scales
            const int r0 = s.row0[s.batch[it.batch]], n = s.row0[s.batch[it.batch + 1]] - r0;
            v = l < n ? __hip_atomic_load(up + r0 + l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 1u;
            return __ballot(v == 0u) == 0ull;
        };
        // The workgroup that took one certain tile of a slot, another one for each of its rows, brings that row into 8 bits once all
        // the slot's tiles are counted. (Left to whoever counts the last tile, the slowest workgroup gets every slot, and is slower
        // for it.) The values come past this XCD's caches, as they were stored, and go the same way
        int head = 0, tail = 0;
        auto take = [&](const Item& it) __attribute__((always_inline)) {
            const int m = __builtin_amdgcn_readfirstlane(s.row0[it.slot + 1] - s.row0[it.slot]);
            const int at = it.ticket - it.slot * NB, step = max(NB / M8_T, 1);
            for (int j = 0; j < m; ++j)
                if (at == (int) ((uint32_t) (37 * it.slot + step * j) % (uint32_t) NB)) duty[tail++] = (uint16_t) (it.slot * M8_T + j);
        };
        auto serve = [&]() __attribute__((always_inline)) {
            if (head == tail) return;
            const int d = __builtin_amdgcn_readfirstlane((int) duty[head]), slot = d / M8_T, row = __builtin_amdgcn_readfirstlane(s.row0[slot] + d % M8_T);
            const int c = l < M8_SUB ? __hip_atomic_load(p.count + 32 * (M8_SUB * slot + l), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
            static_assert(M8_SUB == 8, "one 8-lane sum");
            if (__builtin_amdgcn_readfirstlane(sum8(c)) != NB) return;
            asm volatile("" ::: "memory");
            constexpr int G = M8_I / 16 / 64;
            const unsigned long long* h = (const unsigned long long*) (p.act + (size_t) row * p.I);
            float v[G][16];
            uint32_t top = 0;
            #pragma unroll
            for (int g = 0; g < G; ++g)
                if (1024 * g < p.I)
                {
                    #pragma unroll
                    for (int j = 0; j < 8; ++j)
                    {
                        const unsigned long long u = __hip_atomic_load(h + 8 * min(l + 64 * g, p.I / 16 - 1) + j, __ATOMIC_RELAXED,
                                                                       __HIP_MEMORY_SCOPE_AGENT);
                        v[g][2 * j] = __uint_as_float((uint32_t) u);
                        v[g][2 * j + 1] = __uint_as_float((uint32_t) (u >> 32));
                    }
                }
            #pragma unroll
            for (int g = 0; g < G; ++g)
                if (1024 * g < p.I)
                {
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) top = max(top, mag(v[g][j]));
                }
            const RowQ q = row_q(wave_ext_u32<true>(top));
            #pragma unroll
            for (int g = 0; g < G; ++g)
                if (1024 * g < p.I && l + 64 * g < p.I / 16)
                {
                    // (sixteen values at a time: all of a row's quotients in 64 bits at once spill the streaming waves' registers)
                    __builtin_amdgcn_sched_barrier(0);
                    const u32x4 o = quant16<HMOE_DT_F32>(v[g], q);
                    __builtin_amdgcn_sched_barrier(0);
                    unsigned long long* to = (unsigned long long*) (p.qa + (size_t) row * IP + 16 * (l + 64 * g));
                    #pragma unroll
                    for (int j = 0; j < 2; ++j)
                        __hip_atomic_store(to + j, (unsigned long long) o[2 * j] | ((unsigned long long) o[2 * j + 1] << 32), __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
                }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (l < M8_COPY)
                __hip_atomic_store(p.up + l * M8_ROWS + row, __float_as_uint(q.s) | 0x80000000u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            ++head;
        };
        auto bring = [&](const Item& it) __attribute__((always_inline)) {
            if (it.batch < 0 || it.ticket >= total || slots == 0) return;
            const int r0 = s.row0[s.batch[it.batch]], n = s.row0[s.batch[it.batch + 1]] - r0;
            uint32_t v;
            for (int polls = 0; !ask(it, v) && !lost; ++polls)
            {
                serve();
                __builtin_amdgcn_s_sleep(2);
                lost = polls > (1 << 22);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
            int8_t* q = qb + (it.d & 1) * rq * QP;
            const int pieces = n * (QP / 16);
            for (int i0 = 0; i0 < pieces; i0 += 512)
            {
                u32x4 e[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                {
                    const int i = min(i0 + 64 * j + l, pieces - 1);
                    e[j] = ld16(p.qa + (size_t) (r0 + i / (QP / 16)) * IP + min(16 * (i % (QP / 16)), p.I - 16));
                }
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                {
                    const int i = i0 + 64 * j + l;
                    if (i < pieces) *(u32x4*) (q + 16 * i) = 16 * (i % (QP / 16)) < p.I ? e[j] : (u32x4) {0u, 0u, 0u, 0u};
                }
            }
            if (l < n) fq[it.d & 1][l] = lost ? __uint_as_float(0x7fc00000u) : __uint_as_float(v & 0x7fffffffu) * s.weight[r0 + l];
        };
        // the tickets to come: what is left of the run, then the claim that was made meanwhile
        int left = first < 256 ? run - 1 : 0, last = start, nc = 0;
        bool asked = false;
        auto ticket = [&]() __attribute__((always_inline)) {
            if (left > 0) { --left; last += 256; }
            else
            {
                if (!asked && l == 0) nc = claim();
                const int c = __builtin_amdgcn_readfirstlane(nc);
                asked = false;
                last = ticket_of(c);
                left = c < 256 ? run - 1 : 0;
            }
            if (left <= 2 && last < NG && !asked)                        // (a down ticket takes long: no claim ahead of one)
            {
                if (l == 0) nc = claim();
                asked = true;
            }
            return last;
        };
        // the batches of a down tile: up to SU / RD slots and rq rows (a slot has at most 16 of these). (With as many slots as would fit
        // if every token were in each of them, 16 tokens over 102 experts of 6144 x 2048 took 708 us in place of 582, over 47 of
        // 1840 x 288 146 in place of 84)
        for (int at = 0; at < slots; ++nb)
        {
            const int c = min(at + 1 + l, slots);
            const unsigned long long fit = __ballot(l < SU / RD && at + 1 + l <= slots && (int) s.row0[c] - (int) s.row0[at] <= rq);
            if (l == 0) s.batch[nb] = (uint16_t) at;
            at = __builtin_amdgcn_readfirstlane(at + max(__popcll(fit), 1));
        }
        if (l == 0)
        {
            s.batch[nb] = s.batch[nb + 1] = (uint16_t) slots;
            s.batches = max(nb, 1);
        }
        nb = max(nb, 1);
        if (cur.batch < 0 || nb == 1) tk[1] = ticket();
        bring(cur);
        __syncthreads();
        while (cur.ticket < total)
        {
            // the ticket after the next; behind a down tile of several batches in its last but one
            const Item nx = next(cur);
            if (cur.batch < 0) take(cur);
            serve();
            if (cur.batch < 0 ? nx.batch < 0 || nb == 1 : nb == 1) tk[(cur.seq + 2) & 7] = ticket();
            else if (cur.batch >= 0 && cur.batch == nb - 2) tk[(cur.seq + 1) & 7] = ticket();
            const bool tn = turns(cur, nx);
            uint32_t v;
            const bool now = !tn || (apart && ask(nx, v));
            if (now) bring(nx);
            if (tn && l == 0) late = !now;
            __syncthreads();
            if (!now)
            {
                if (!apart) __syncthreads();
                bring(nx);
                __syncthreads();
            }
            cur = nx;
        }
        // what is left to quantise: its tiles are counted, or will be by workgroups that wait for nothing
        for (int polls = 0; head < tail && polls < (1 << 22); ++polls) serve();
        return;
    }
    if (w == 8)
    {
        // the finishing wave. A tile's values are stored in its item and counted in the next (behind the wait for that one's
        // scales, which were asked for after them)
        float sg = 0.f, su = 0.f;
        auto scales = [&](const Item& it) {
            if (it.batch >= 0 || it.ticket >= total || l >= 8 * TR) return;
            const bool sh = p.hg && it.slot == 0;
            const size_t so = (sh ? 0 : (size_t) s.expert[it.slot] * p.I) + min(8 * TR * it.blk + l, p.I - 1);
            sg = (sh ? p.hsg : p.sg)[so];
            su = (sh ? p.hsu : p.su)[so];
        };
        int stored = -1;                                                 // the ticket of the tile stored last
        auto count = [&]() {
            if (stored >= 0 && l == 0)
                (void) __hip_atomic_fetch_add(p.count + 32 * (M8_SUB * (int) ((uint32_t) stored / (uint32_t) NB) + stored % M8_SUB), 1,
                                              __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            stored = -1;
        };
        scales(cur);
        __syncthreads();
        nb = __builtin_amdgcn_readfirstlane(s.batches);
        while (cur.ticket < total)
        {
            const Item nx = next(cur);
            __syncthreads();
            if (cur.batch < 0)
            {
                const uint32_t mask = s.tokens[cur.slot];
                const int m = __popc(mask), row0 = s.row0[cur.slot];
                const int* rd = red + (cur.seq & 1) * 8 * ROWS * T;
                // (values stored at the agent's scope go past the XCD's own L2: once the wait is over they can be seen, without
                // writing the L2's lines back, which takes longer than a tile)
                asm volatile("s_waitcnt vmcnt(0)" : "+v"(sg), "+v"(su) : : "memory");
                count();
                for (int i0 = 0; i0 < 8 * TR * m; i0 += 64)
                {
                    const int i = min(i0 + l, 8 * TR * m - 1), k = i / (8 * TR), rr = i - k * 8 * TR, n = 8 * TR * cur.blk + rr;
                    int ag = 0, au = 0;
                    #pragma unroll
                    for (int v = 0; v < 8; ++v)
                    {
                        ag += rd[(v * ROWS + rr) * T + k];
                        au += rd[(v * ROWS + 8 * TR + rr) * T + k];
                    }
                    uint32_t mm = mask;
                    for (int j = 0; j < k; ++j) mm &= mm - 1;
                    const float xs = s.xs[__builtin_ctz(mm)];
                    const float g = (float) ag * xs * __shfl(sg, rr), u = (float) au * xs * __shfl(su, rr);
                    if (i0 + l < 8 * TR * m && n < p.I)
                        __hip_atomic_store(p.act + (size_t) (row0 + k) * p.I + n, swiglu(g, u), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                stored = cur.ticket;
                scales(nx);
                if (nx.batch >= 0 || nx.ticket >= total)
                {
                    // the last of this workgroup's gate/up tiles
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    count();
                }
            }
            else if (cur.batch + 1 == nb)
            {
                const float* ac = accl + (cur.seq & 1) * 64 * RD * T;
                for (int i = l; i < 8 * RD * T; i += 64)
                {
                    const int tok = i / (8 * RD), rr = i - tok * 8 * RD;
                    float v = 0.f;
                    #pragma unroll
                    for (int k = 0; k < 8; ++k) v += ac[(k * 8 * RD + rr) * T + tok];
                    // (a token that is not finite and has no expert here has no term that says so)
                    const float xs = s.xs[tok];
                    v = xs == xs ? v : xs;
                    if (8 * RD * cur.blk + rr < p.H) store_out(p.y, (size_t) tok * p.ldy + 8 * RD * cur.blk + rr, v, p.ydt);
                }
            }
            turn(cur, nx);
            cur = nx;
        }
        return;
    }

    // a streaming wave
    auto expert_of = [&](int slot) { return p.hg && slot == 0 ? -1 : __builtin_amdgcn_readfirstlane((int) s.expert[slot]); };
    struct DnAt { const int8_t* w[SU]; const float* s[SU]; int live; };
    auto dn_at = [&](const Item& it) {
        // (a pair behind the batch's last asks for one piece of x: every item has the same number of loads to wait for)
        DnAt o;
        o.live = 0;
        int sl = __builtin_amdgcn_readfirstlane((int) s.batch[it.batch]), og = 0;
        const int s1 = __builtin_amdgcn_readfirstlane((int) s.batch[it.batch + 1]);
        #pragma unroll
        for (int b = 0; b < SU; ++b)
        {
            const int8_t* wb = p.xq;
            const float* sb = p.xs;
            if (sl < s1)
            {
                const int e = expert_of(sl), n0 = 8 * min(RD * it.blk + og, p.H / 8 - 1);
                wb = (const int8_t*) ((uintptr_t) p.wd + (e < 0 ? p.dd : (int64_t) e * p.H * p.I) + (size_t) n0 * p.I);
                sb = (const float*) ((uintptr_t) p.sd + (e < 0 ? p.dsd : (int64_t) e * p.H * 4) + (size_t) n0 * 4);
                o.live = b + 1;
            }
            o.w[b] = scalar(wb);
            o.s[b] = scalar(sb);
            if (++og == RD) { og = 0; ++sl; }
        }
        return o;
    };
    auto load_dn = [&](const DnAt& at, int j) {                          // load j of a down item
        const int b = j / NSD, i = j % NSD;
        const uint32_t is = b < at.live ? ~0u : 0u;
        a[j] = ldw16_at(at.w[b], vd[i] & is);
        if (i == NSD - 1) sd[b] = *(const HMOE_GLOBAL float*) ((const HMOE_GLOBAL char*) at.s[b] + (4u * r & is));
    };
    // two tokens of a gate/up item (or one, twice), the k-th on; KIND: the next item, whose loads take the place of what is used:
    // gate/up 0, down 1, none 2. (One form for one token and for two: what is loaded on two ways that meet is moved where they
    // do, and waited for)
    auto tokens = [&](const Item& it, int t0, int t1, int k0, int k1, auto kind, const GuAt& ng, const DnAt& nd) {
        constexpr int KIND = decltype(kind)::value;
        int* rd = red + ((it.seq & 1) * 8 + w) * ROWS * T;
        const int8_t* x[2] = {xl + t0 * XP + 128 * w * NS + 16 * pc, xl + t1 * XP + 128 * w * NS + 16 * pc};
        int g[2][TR], u[2][TR];
        #pragma unroll
        for (int n = 0; n < 2; ++n)
            #pragma unroll
            for (int tr = 0; tr < TR; ++tr) g[n][tr] = u[n][tr] = 0;
        #pragma unroll
        for (int i = 0; i < NS; ++i)
        {
            u32x4 xv[2];
            #pragma unroll
            for (int n = 0; n < 2; ++n) xv[n] = *(const u32x4*) (x[n] + 128 * i);
            #pragma unroll
            for (int tr = 0; tr < TR; ++tr)
            {
                #pragma unroll
                for (int n = 0; n < 2; ++n)
                {
                    g[n][tr] = dot16(a[tr * NS + i], xv[n], g[n][tr]);
                    u[n][tr] = dot16(a[(TR + tr) * NS + i], xv[n], u[n][tr]);
                }
                if constexpr (KIND < 2)
                {
                    // (the products stand here: where they are put off, the loads below get other registers, and the moves back wait
                    // for them)
                    #pragma unroll
                    for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(g[n][tr]), "+v"(u[n][tr]));
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (KIND == 0) load_gu(ng, i, tr);
                    else
                    {
                        if (tr * NS + i < SU * NSD) load_dn(nd, tr * NS + i);
                        if ((TR + tr) * NS + i < SU * NSD) load_dn(nd, (TR + tr) * NS + i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        const int kk[2] = {k0, k1};
        #pragma unroll
        for (int n = 0; n < 2; ++n)
            #pragma unroll
            for (int tr = 0; tr < TR; ++tr)
            {
                const int gs = sum8(g[n][tr]), us = sum8(u[n][tr]);
                if (pc == 0)
                {
                    rd[(8 * tr + r) * T + kk[n]] = gs;
                    rd[(8 * (TR + tr) + r) * T + kk[n]] = us;
                }
            }
    };
    auto gate_up = [&](const Item& it, auto kind, const GuAt& ng, const DnAt& nd) {
        uint32_t m = __builtin_amdgcn_readfirstlane((int) s.tokens[it.slot]);
        int k = 0;
        for (; __popc(m) > 2; k += 2)
        {
            const uint32_t m1 = m & (m - 1);
            tokens(it, __builtin_ctz(m), __builtin_ctz(m1), k, k + 1, ic<2>{}, ng, nd);
            m = m1 & (m1 - 1);
        }
        const uint32_t m1 = m & (m - 1);
        tokens(it, __builtin_ctz(m), __builtin_ctz(m1 ? m1 : m), k, k + (m1 ? 1 : 0), kind, ng, nd);
    };
    auto down = [&](const Item& it, auto kind, const DnAt& nd) {
        constexpr int KIND = decltype(kind)::value;
        float* acc = accl + ((it.seq & 1) * 8 + w) * 8 * RD * T;
        if (it.batch == 0)
            for (int i = l; i < 8 * RD * T; i += 64) acc[i] = 0.f;
        int sl = __builtin_amdgcn_readfirstlane((int) s.batch[it.batch]), og = 0;
        const int s1 = __builtin_amdgcn_readfirstlane((int) s.batch[it.batch + 1]), r0 = s.row0[sl];
        const int8_t* qr = qb + (it.d & 1) * rq * QP + 128 * w * NSD + 16 * pc;
        const float* f = fq[it.d & 1];
        #pragma unroll
        for (int b = 0; b < SU; ++b)
        {
            if (sl < s1)
            {
                int row = s.row0[sl] - r0;
                for (uint32_t m = __builtin_amdgcn_readfirstlane((int) s.tokens[sl]); m; m &= m - 1, ++row)
                {
                    int v = 0;
                    #pragma unroll
                    for (int i = 0; i < NSD; ++i) v = dot16(a[b * NSD + i], *(const u32x4*) (qr + row * QP + 128 * i), v);
                    v = sum8(v);
                    if (pc == 0) acc[(8 * og + r) * T + __builtin_ctz(m)] += (float) v * (f[row] * sd[b]);
                }
            }
            if (++og == RD) { og = 0; ++sl; }
            if constexpr (KIND == 1)
            {
                __builtin_amdgcn_sched_barrier(0);
                #pragma unroll
                for (int i = 0; i < NSD; ++i) load_dn(nd, b * NSD + i);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    GuAt ng;
    DnAt nd;
    if (!early && cur.batch < 0)
    {
        ng = gu_at(expert_of(cur.slot), cur.blk);
        #pragma unroll
        for (int i = 0; i < NS; ++i)
            #pragma unroll
            for (int tr = 0; tr < TR; ++tr) load_gu(ng, i, tr);
    }
    __syncthreads();
    nb = __builtin_amdgcn_readfirstlane(s.batches);
    if (cur.batch >= 0 && cur.ticket < total)
    {
        nd = dn_at(cur);
        #pragma unroll
        for (int j = 0; j < SU * NSD; ++j) load_dn(nd, j);
    }
    Item nx = cur.ticket < total ? next(cur) : cur;
    if (cur.ticket < total && cur.batch < 0)
    {
        while (nx.batch < 0)                                             // (every ticket behind the gate/up ones is a down one)
        {
            ng = gu_at(expert_of(nx.slot), nx.blk);
            gate_up(cur, ic<0>{}, ng, nd);
            __syncthreads();
            cur = nx;
            nx = next(cur);
        }
        if (nx.ticket < total)
        {
            nd = dn_at(nx);
            gate_up(cur, ic<1>{}, ng, nd);
        }
        else gate_up(cur, ic<2>{}, ng, nd);
        __syncthreads();
        turn(cur, nx);
        cur = nx;
        if (cur.ticket < total) nx = next(cur);
    }
    if (cur.ticket >= total) return;
    while (nx.ticket < total)
    {
        nd = dn_at(nx);
        down(cur, ic<1>{}, nd);
        __syncthreads();
        cur = nx;
        nx = next(cur);
    }
    down(cur, ic<2>{}, nd);
    __syncthreads();
}

template <int NS, int TR>
static void m8_launch(const M8Args& p, hipStream_t st)
{
    if (p.I <= 1024) m8_experts_kernel<NS, TR, 1><<<256, 640, 0, st>>>(p);
    else if (p.I <= 2048) m8_experts_kernel<NS, TR, 2><<<256, 640, 0, st>>>(p);
    else m8_experts_kernel<NS, TR, 4><<<256, 640, 0, st>>>(p);
}

// workspace layout; the parts' offsets into o (or null) and the whole size
static size_t m8_layout(int T, int H, int I, int E, int topk, size_t* o)
{
    const size_t rows = (size_t) T * (topk + 1);
    const size_t part[] = {(size_t) T * E * 8, (size_t) T * up128(H), (size_t) T * 4, rows * I * 4, rows * up128(I), M8_SYNC * 4};
    size_t at = 0;
    for (int i = 0; i < 6; ++i)
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
    if (T < 1 || T > M8_T || H < 16 || H > M8_H || I < 16 || I > M8_I || E < 1 || E > M8_E || topk < 1 || topk > M8_K) return 0;
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
    HMOE_REQUIRE(H >= 16 && H <= M8_H && H % 16 == 0 && I >= 16 && I <= M8_I && I % 16 == 0,
                 "moe8_layer: hidden size %d, intermediate size %d: multiples of 16 up to %d and %d", H, I, M8_H, M8_I);
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
    HMOE_REQUIRE(!rows_meet(T, x, ldx, H, x_dtype == HMOE_DT_F32 ? 4 : 2, y, ldy, H, y_dtype == HMOE_DT_F32 ? 4 : 2),
                 "moe8_layer: the output overlaps x");
    size_t o[6];
    m8_layout(T, H, I, E, topk, o);
    uint8_t* b = (uint8_t*) work;
    M8Args p = {x, ldx, x_dtype, wr, bias, wg, wu, wd, sg, su, sd,
                sh_w ? sh_w[0] : nullptr, sh_w ? sh_w[1] : nullptr, sh_w ? sh_w[2] : nullptr,
                sh_s ? sh_s[0] : nullptr, sh_s ? sh_s[1] : nullptr, sh_s ? sh_s[2] : nullptr,
                0, 0, 0, 0, T, H, I, E, n, lo, topk, scale, sel, rw, y, ldy, y_dtype,
                (double*) (b + o[0]), (int8_t*) (b + o[1]), (float*) (b + o[2]), (float*) (b + o[3]), (int8_t*) (b + o[4]),
                (int*) (b + o[5]), (int*) (b + o[5]) + 32, (uint32_t*) (b + o[5]) + 32 + 32 * M8_SUB * M8_SLOTS};
    p.dg = (int64_t) ((uintptr_t) p.hg - (uintptr_t) wg);
    p.du = (int64_t) ((uintptr_t) p.hu - (uintptr_t) wu);
    p.dd = (int64_t) ((uintptr_t) p.hd - (uintptr_t) wd);
    p.dsd = (int64_t) ((uintptr_t) p.hsd - (uintptr_t) sd);
    const hipStream_t st = (hipStream_t) stream;
    const int ni = cdiv(H, 1024);
#define HMOE_N(D, N) if (ni == N) m8_route_kernel<D, N><<<E + T, 256, 0, st>>>(p);
#define HMOE_R(D) { HMOE_N(D, 1) HMOE_N(D, 2) HMOE_N(D, 3) HMOE_N(D, 4) HMOE_N(D, 5) HMOE_N(D, 6) HMOE_N(D, 7) }
    if (x_dtype == HMOE_DT_F32) HMOE_R(HMOE_DT_F32)
    else if (x_dtype == HMOE_DT_BF16) HMOE_R(HMOE_DT_BF16)
    else HMOE_R(HMOE_DT_F16)
#undef HMOE_R
#undef HMOE_N
    // the lines of a hidden row that a wave takes, and as many 8-row groups as make 8 to 14 loads of an item with them
    if (H <= 1024) m8_launch<1, 6>(p, st);
    else if (H <= 2048) m8_launch<2, 3>(p, st);
    else if (H <= 4096) m8_launch<4, 1>(p, st);
    else if (H <= 6144) m8_launch<6, 1>(p, st);
    else m8_launch<7, 1>(p, st);
    return HMOE_LAUNCHED("moe8 layer");
}
