// i8.hip - products in 8-bit integers with a scale for each token and each output channel, and the gated MLP made of them
// (hmoe_i8_quantize, hmoe_i8_matmul, hmoe_i8_linear, hmoe_i8_mlp):
//   y[m][n] = s_x[m] s_w[n] sum_k q[m][k] w[n][k] (+ bias[n]), the sum exact in int32, the rest fp32, rounded once to y's type.
// Few rows are brought into 8 bits by the product's own workgroups (i8_few.hip), others by a launch before it (i8_gemm1.hip,
// i8_gemm2.hip: tiles out of LDS).
#include "i8_gemm.h"

namespace hmoe {

// ---- rows to 8 bits ----------------------------------------------------------------------------------------------
// One workgroup a row: the row's largest magnitude, then its values as whole numbers. HOLD: the 16 values a thread of a row of
// up to 4096 HOLD stay in registers between the two; a longer row (0) is read again, out of the caches. Bound by the bytes: 2048 rows
// of 6144 in bf16 8 us (4.7 TB/s), fp32 rows of 2048 6 us; 61 rows 3.2 us, the launch and one round trip.
template <int DT, int HOLD>
__global__ void __launch_bounds__(256) i8_quant_kernel(const void* __restrict__ x, int64_t ldx, int K, int8_t* __restrict__ q,
                                                       int64_t ldq, float* __restrict__ s)
{
    __shared__ uint32_t wmax[4];
    constexpr int G = HOLD > 0 ? HOLD : 1;
    const int t = threadIdx.x, pieces = K / 16;
    const size_t row = blockIdx.x;
    const uint8_t* xr = (const uint8_t*) x + row * (size_t) ldx * (DT == HMOE_DT_F32 ? 4 : 2);
    int8_t* qr = q + row * (size_t) ldq;
    float v[G][16];
    uint32_t m = 0;
    auto largest = [&](const float (&u)[16]) __attribute__((always_inline)) {
        #pragma unroll
        for (int j = 0; j < 16; ++j) m = max(m, mag(u[j]));
    };
    if constexpr (HOLD > 0)
    {
        #pragma unroll
        for (int g = 0; g < G; ++g) load16<DT>(xr, min(t + 256 * g, pieces - 1), v[g]);      // (past the row: its last values)
        #pragma unroll
        for (int g = 0; g < G; ++g) largest(v[g]);
    }
    else
        for (int i = t; i < pieces; i += 256)
        {
            load16<DT>(xr, i, v[0]);
            largest(v[0]);
        }
    m = wave_ext_u32<true>(m);
    if ((t & 63) == 0) wmax[t >> 6] = m;
    __syncthreads();
    const RowQ p = row_q(max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3])));
    if (t == 0) s[row] = p.s;
    if constexpr (HOLD > 0)
    {
        #pragma unroll
        for (int g = 0; g < G; ++g)
            if (t + 256 * g < pieces) *(u32x4*) (qr + 16 * (t + 256 * g)) = quant16<DT>(v[g], p);
    }
    else
        for (int i = t; i < pieces; i += 256)
        {
            load16<DT>(xr, i, v[0]);
            *(u32x4*) (qr + 16 * (size_t) i) = quant16<DT>(v[0], p);
        }
}

constexpr int I8_MAXK = 131056;              // 128 x 128 x K stays below 2^31
constexpr int64_t I8_MAXLD = 1 << 28;        // the product's kernel steps over 8 rows in 32 bits

static int launch_quant(const void* x, int dt, int64_t ldx, int M, int K, int8_t* q, int64_t ldq, float* s, hipStream_t st)
{
#define HMOE_Q(D)                                                                                                      \
    do                                                                                                                 \
    {                                                                                                                  \
        if (K <= 4096) i8_quant_kernel<D, 1><<<M, 256, 0, st>>>(x, ldx, K, q, ldq, s);                                 \
        else if (K <= 8192) i8_quant_kernel<D, 2><<<M, 256, 0, st>>>(x, ldx, K, q, ldq, s);                            \
        else i8_quant_kernel<D, 0><<<M, 256, 0, st>>>(x, ldx, K, q, ldq, s);                                           \
    } while (0)
    if (dt == HMOE_DT_F32) HMOE_Q(HMOE_DT_F32);
    else if (dt == HMOE_DT_BF16) HMOE_Q(HMOE_DT_BF16);
    else HMOE_Q(HMOE_DT_F16);
#undef HMOE_Q
    return HMOE_LAUNCHED("i8 quantize");
}

static I8Out out_of(void* y, int64_t ldy, int dt, const float* xs, const float* ws, const float* ws2, const float* bias)
{
    return {y, ldy, dt, xs, ws, ws2, bias};
}

static bool is_dt(int dt) { return dt == HMOE_DT_F32 || dt == HMOE_DT_BF16 || dt == HMOE_DT_F16; }
// rows [n][cols] of a matrix with a row stride, at least cols, in elements of es bytes: does its last byte's offset fit?
static bool rows_ok(int64_t n, int64_t ld, int64_t cols) { return ld >= cols && n <= INT64_MAX / 8 / (ld > 0 ? ld : 1); }

static int check_x(const char* what, const void* x, int dt, int64_t ldx, int M, int K)
{
    HMOE_REQUIRE(is_dt(dt), "%s: x dtype code %d", what, dt);
    HMOE_REQUIRE(K >= 16 && K % 16 == 0 && K <= I8_MAXK, "%s: depth %d: a multiple of 16 up to %d", what, K, I8_MAXK);
    HMOE_REQUIRE(M >= 0 && M <= (1 << 20), "%s: %d rows: up to %d", what, M, 1 << 20);
    HMOE_REQUIRE(x && ((uintptr_t) x & (dt == HMOE_DT_F32 ? 3 : 1)) == 0 && rows_ok(M, ldx, K), "%s: x address or row stride %lld", what,
                 (long long) ldx);
    return HMOE_OK;
}

static int check_w(const char* what, const int8_t* w, const float* ws, int64_t ldw, int N, int K)
{
    HMOE_REQUIRE(N >= 1 && N <= (1 << 20), "%s: %d output channels: 1 to %d", what, N, 1 << 20);
    HMOE_REQUIRE(w && ws && ((uintptr_t) w & 15) == 0 && ((uintptr_t) ws & 3) == 0 && ldw % 16 == 0 && ldw < I8_MAXLD && rows_ok(N, ldw, K),
                 "%s: weights: null, not 16-byte aligned, or row stride %lld for depth %d", what, (long long) ldw, K);
    return HMOE_OK;
}

static int check_y(const char* what, const void* y, int dt, int64_t ldy, int M, int N)
{
    HMOE_REQUIRE(is_dt(dt), "%s: output dtype code %d", what, dt);
    HMOE_REQUIRE(y && ((uintptr_t) y & (dt == HMOE_DT_F32 ? 3 : 1)) == 0 && rows_ok(M, ldy, N), "%s: output address or row stride %lld", what,
                 (long long) ldy);
    return HMOE_OK;
}

static int dt_size(int dt) { return dt == HMOE_DT_F32 ? 4 : 2; }

}  // namespace hmoe

using namespace hmoe;

extern "C" int hmoe_i8_quantize(const void* x, int x_dtype, int64_t ldx, int M, int K, int8_t* q, int64_t ldq, float* s,
                                void* stream)
{
    if (M == 0) return HMOE_OK;
    if (int rc = check_x("i8_quantize", x, x_dtype, ldx, M, K)) return rc;
    HMOE_REQUIRE(q && s && ((uintptr_t) q & 15) == 0 && ((uintptr_t) s & 3) == 0 && ldq % 16 == 0 && rows_ok(M, ldq, K),
                 "i8_quantize: q: null, not 16-byte aligned, or row stride %lld", (long long) ldq);
    HMOE_REQUIRE(!rows_meet(M, x, ldx, K, dt_size(x_dtype), q, ldq, K, 1), "i8_quantize: q overlaps x");
    return launch_quant(x, x_dtype, ldx, M, K, q, ldq, s, (hipStream_t) stream);
}

extern "C" int hmoe_i8_matmul(const int8_t* q, int64_t ldq, const float* s, int M, const int8_t* w, int64_t ldw, const float* ws,
                              int N, int K, const float* bias, void* y, int y_dtype, int64_t ldy, void* stream)
{
    if (M == 0) return HMOE_OK;
    HMOE_REQUIRE(K >= 16 && K % 16 == 0 && K <= I8_MAXK, "i8_matmul: depth %d: a multiple of 16 up to %d", K, I8_MAXK);
    HMOE_REQUIRE(M > 0 && M <= (1 << 20), "i8_matmul: %d rows: up to %d", M, 1 << 20);
    HMOE_REQUIRE(q && s && ((uintptr_t) q & 15) == 0 && ((uintptr_t) s & 3) == 0 && ldq % 16 == 0 && ldq < I8_MAXLD && rows_ok(M, ldq, K),
                 "i8_matmul: q: null, not 16-byte aligned, or row stride %lld", (long long) ldq);
    if (int rc = check_w("i8_matmul", w, ws, ldw, N, K)) return rc;
    HMOE_REQUIRE(((uintptr_t) bias & 3) == 0, "i8_matmul: bias alignment");
    if (int rc = check_y("i8_matmul", y, y_dtype, ldy, M, N)) return rc;
    HMOE_REQUIRE(!rows_meet(M, q, ldq, K, 1, y, ldy, N, dt_size(y_dtype)), "i8_matmul: the output overlaps q");
    const I8Out o = out_of(y, ldy, y_dtype, s, ws, nullptr, bias);
    if (i8_few(M, N, K, 3)) return i8_few_product(q, 3, ldq, w, ldw, M, N, K, o, (hipStream_t) stream);
    return i8_product(q, ldq, w, ldw, M, N, K, o, (hipStream_t) stream);
}

extern "C" size_t hmoe_i8_linear_work_bytes(int M, int N, int K)
{
    (void) N;
    if (M < 0 || K < 0) return 0;
    return up128((size_t) M * K) + up128((size_t) M * 4);
}

extern "C" int hmoe_i8_linear(const void* x, int x_dtype, int64_t ldx, int M, const int8_t* w, int64_t ldw, const float* ws, int N,
                              int K, const float* bias, void* y, int y_dtype, int64_t ldy, void* work, void* stream)
{
    if (M == 0) return HMOE_OK;
    if (int rc = check_x("i8_linear", x, x_dtype, ldx, M, K)) return rc;
    if (int rc = check_w("i8_linear", w, ws, ldw, N, K)) return rc;
    HMOE_REQUIRE(((uintptr_t) bias & 3) == 0, "i8_linear: bias alignment");
    if (int rc = check_y("i8_linear", y, y_dtype, ldy, M, N)) return rc;
    HMOE_REQUIRE(!rows_meet(M, x, ldx, K, dt_size(x_dtype), y, ldy, N, dt_size(y_dtype)), "i8_linear: the output overlaps x");
    HMOE_REQUIRE(work && ((uintptr_t) work & 15) == 0, "i8_linear: workspace null or not 16-byte aligned");
    const hipStream_t st = (hipStream_t) stream;
    int8_t* q = (int8_t*) work;
    float* s = (float*) (q + up128((size_t) M * K));
    const I8Out o = out_of(y, ldy, y_dtype, s, ws, nullptr, bias);
    if (i8_few(M, N, K, x_dtype)) return i8_few_product(x, x_dtype, ldx, w, ldw, M, N, K, o, st);
    if (int rc = launch_quant(x, x_dtype, ldx, M, K, q, K, s, st)) return rc;
    return i8_product(q, K, w, ldw, M, N, K, o, st);
}

// workspace: x in 8 bits and its scales, the gated rows in fp32, then in 8 bits with their scales
extern "C" size_t hmoe_i8_mlp_work_bytes(int M, int Hd, int Id)
{
    if (M < 0 || Hd < 0 || Id < 0) return 0;
    return up128((size_t) M * Hd) + 2 * up128((size_t) M * 4) + up128((size_t) M * Id * 4) + up128((size_t) M * Id);
}

extern "C" int hmoe_i8_mlp(const void* x, int x_dtype, int64_t ldx, int M, int Hd, int Id, const int8_t* wg, const int8_t* wu,
                           const int8_t* wd, const float* sg, const float* su, const float* sd, void* y, int y_dtype, int64_t ldy,
                           void* work, void* stream)
{
    if (M == 0) return HMOE_OK;
    if (int rc = check_x("i8_mlp", x, x_dtype, ldx, M, Hd)) return rc;
    HMOE_REQUIRE(Id >= 16 && Id % 16 == 0 && Id <= I8_MAXK, "i8_mlp: intermediate size %d: a multiple of 16 up to %d", Id, I8_MAXK);
    if (int rc = check_w("i8_mlp", wg, sg, Hd, Id, Hd)) return rc;
    if (int rc = check_w("i8_mlp", wu, su, Hd, Id, Hd)) return rc;
    if (int rc = check_w("i8_mlp", wd, sd, Id, Hd, Id)) return rc;
    if (int rc = check_y("i8_mlp", y, y_dtype, ldy, M, Hd)) return rc;
    HMOE_REQUIRE(!rows_meet(M, x, ldx, Hd, dt_size(x_dtype), y, ldy, Hd, dt_size(y_dtype)), "i8_mlp: the output overlaps x");
    HMOE_REQUIRE(work && ((uintptr_t) work & 15) == 0, "i8_mlp: workspace null or not 16-byte aligned");
    const hipStream_t st = (hipStream_t) stream;
    int8_t* q = (int8_t*) work;
    float* s = (float*) (q + up128((size_t) M * Hd));
    float* act = (float*) ((uint8_t*) s + up128((size_t) M * 4));
    int8_t* qa = (int8_t*) act + up128((size_t) M * Id * 4);
    float* sa = (float*) (qa + up128((size_t) M * Id));
    const I8Out up = out_of(act, Id, HMOE_DT_F32, s, sg, su, nullptr), down = out_of(y, ldy, y_dtype, sa, sd, nullptr, nullptr);
    if (i8_few(M, Id, Hd, x_dtype))
    {
        if (int rc = i8_few_gated(x, x_dtype, ldx, wg, wu, Hd, M, Id, Hd, up, st)) return rc;
    }
    else
    {
        if (int rc = launch_quant(x, x_dtype, ldx, M, Hd, q, Hd, s, st)) return rc;
        if (int rc = i8_gated(q, Hd, wg, wu, Hd, M, Id, Hd, up, st)) return rc;
    }
    if (i8_few(M, Hd, Id, HMOE_DT_F32)) return i8_few_product(act, HMOE_DT_F32, Id, wd, Id, M, Hd, Id, down, st);
    if (int rc = launch_quant(act, HMOE_DT_F32, Id, M, Id, qa, Id, sa, st)) return rc;
    return i8_product(qa, Id, wd, Id, M, Hd, Id, down, st);
}
