// i8_dev.h - gfx950 device helpers of the 8-bit integer operators (i8.hip, moe8.hip): quantising a row, the integer
// products, storing an output row in its type.
//
// A row x of K values is held as whole numbers q in [-127, 127] and one fp32 scale: a = max |x|, s = a / 127,
// q = 127 x / a rounded half to even. A row of zeros has s = 0 and q = 0; a row with a NaN or an infinity s = NaN and
// q = 0, so that every product of it is NaN.
#pragma once
#include "hmoe_dev.h"

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

namespace hmoe {

// |v| as an unsigned number: ordered as the magnitudes are, infinities above every finite value and NaN above those
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// What a row's quantisation needs of its largest magnitude. With a' = a 2^-e and c = 127 2^-e, e the exponent of a (held
// above -118, where 2^-e would overflow), x c is exact for a 16-bit x (11 + 7 bits) and its quotient by a' is the true
// one 127 x / a, without overflow at either end of the type.
struct RowQ { float c, a, r, s; };
__device__ __forceinline__ RowQ row_q(uint32_t amax)
{
    RowQ o = {0.f, 0.f, 0.f, 0.f};
    if (amax >= 0x7f800000u) { o.s = __uint_as_float(0x7fc00000u); return o; }
    if (amax == 0u) return o;
    const float a = __uint_as_float(amax);
    int e = 0;
    (void) __builtin_frexpf(a, &e);
    e = max(e, -118);
    o.c = __builtin_ldexpf(127.0f, -e);
    o.a = __builtin_ldexpf(a, -e);
    o.r = 1.0f / o.a;
    o.s = a / 127.0f;
    return o;
}

// The quantised value in the low byte of the result (the other bits are the exponent of the 1.5 2^23 it was rounded
// against). The quotient t / a' is formed as t r with one correction by its exact remainder. For a 16-bit x that is the
// correctly rounded quotient, and rounding it to a whole number is rounding the true one: where 127 x / a is not half way
// between whole numbers it is at least 2^-19 (relative) off, and where it is, the fp32 quotient is exactly that half.
__device__ __forceinline__ uint32_t q8(float x, const RowQ& p)
{
    const float t = x * p.c;
    const float q0 = t * p.r;
    const float q1 = __builtin_fmaf(__builtin_fmaf(-q0, p.a, t), p.r, q0);
    return __float_as_uint(q1 + 12582912.0f);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                 0x05040100u);
}
// the same of a 32-bit x, whose 127 x has 31 bits: in 64 bits, where the argument above holds again
__device__ __forceinline__ uint32_t q8_wide(float x, const RowQ& p, double rd)
{
    const double t = (double) x * (double) p.c;
    const double q0 = t * rd;
    const double q1 = __builtin_fma(__builtin_fma(-q0, (double) p.a, t), rd, q0);
    return (uint32_t) (int) __builtin_rint(q1);
}

// ---- values of a row as fp32 ----
template <int DT> __device__ __forceinline__ void widen2(uint32_t v, float& lo, float& hi)
{
    if constexpr (DT == HMOE_DT_BF16) { lo = __uint_as_float(v << 16); hi = __uint_as_float(v & 0xffff0000u); }
    else
    {
        const f16x2 h = __builtin_bit_cast(f16x2, v);
        lo = (float) h[0]; hi = (float) h[1];
    }
}
// 16-byte and 8-byte accesses at an element's own alignment (the hardware takes them at any; a row of an odd stride in 4-byte pieces
// takes 3 times as long)
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));

// 16 (4) values at element 16 i (4 i) of a row
template <int DT> __device__ __forceinline__ void load16(const void* row, int i, float (&v)[16])
{
    if constexpr (DT == HMOE_DT_F32)
    {
        #pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const f32x4_4 u = *(const HMOE_GLOBAL f32x4_4*) ((const HMOE_GLOBAL float*) row + (size_t) 16 * i + 4 * j);
            #pragma unroll
            for (int k = 0; k < 4; ++k) v[4 * j + k] = u[k];
        }
    }
    else
    {
        #pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            const u32x4_2 u = *(const HMOE_GLOBAL u32x4_2*) ((const HMOE_GLOBAL uint16_t*) row + (size_t) 16 * i + 8 * j);
            #pragma unroll
            for (int k = 0; k < 4; ++k) widen2<DT>(u[k], v[8 * j + 2 * k], v[8 * j + 2 * k + 1]);
        }
    }
}
template <int DT> __device__ __forceinline__ void load4(const void* row, int i, float (&v)[4])
{
    if constexpr (DT == HMOE_DT_F32)
    {
        const f32x4_4 u = *(const HMOE_GLOBAL f32x4_4*) ((const HMOE_GLOBAL float*) row + (size_t) 4 * i);
        #pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = u[k];
    }
    else
    {
        const u32x2_2 u = *(const HMOE_GLOBAL u32x2_2*) ((const HMOE_GLOBAL uint16_t*) row + (size_t) 4 * i);
        widen2<DT>(u[0], v[0], v[1]);
        widen2<DT>(u[1], v[2], v[3]);
    }
}
template <int DT> __device__ __forceinline__ u32x4 quant16(const float (&v)[16], const RowQ& p)
{
    u32x4 o;
    if constexpr (DT == HMOE_DT_F32)
    {
        const double rd = p.a > 0.f ? 1.0 / (double) p.a : 0.0;
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            o[j] = pack4(q8_wide(v[4 * j], p, rd), q8_wide(v[4 * j + 1], p, rd), q8_wide(v[4 * j + 2], p, rd),
                         q8_wide(v[4 * j + 3], p, rd));
    }
    else
    {
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            o[j] = pack4(q8(v[4 * j], p), q8(v[4 * j + 1], p), q8(v[4 * j + 2], p), q8(v[4 * j + 3], p));
    }
    // (a row that is not finite: t is 0 x inf or 0 x NaN there)
    if (!(p.r > 0.f)) o = (u32x4) {0u, 0u, 0u, 0u};
    return o;
}

// ---- products ----
// D = A(16 x 64) B(64 x 16) + C of 8-bit integers, exact in int32. Lane l: A row l % 16 and B column l % 16, each at
// k = 16 (l / 16) .. + 16; D rows 4 (l / 16) .. + 4 of column l % 16.
__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ int dot16(u32x4 a, u32x4 b, int c)
{
    #pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_sdot4((int) a[j], (int) b[j], c, false);
    return c;
}

// silu(g) u in fp32. Of a g below -88, e^-g is infinite and its reciprocal 0: silu = -0, as in the limit; a g of -inf
// gives NaN (inf 0), as g sigmoid(g) does.
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

// fp32 to a 16-bit type, to the nearest, ties to even (the hardware's conversions)
__device__ __forceinline__ uint16_t to16(float v, int dt)
{
    return dt == HMOE_DT_BF16 ? __builtin_bit_cast(uint16_t, (__bf16) v) : __builtin_bit_cast(uint16_t, (_Float16) v);
}
__device__ __forceinline__ void store_out(void* out, size_t i, float v, int dt)
{
    if (dt == HMOE_DT_F32) ((float*) out)[i] = v;
    else ((uint16_t*) out)[i] = to16(v, dt);
}

// whether M rows of ca values at a (row stride lda, ea bytes a value) and M rows at b share a byte: exactly where the rows lie the same
// distance apart (column ranges of one buffer do), otherwise by their whole spans
inline bool rows_meet(int64_t M, const void* a, int64_t lda, int64_t ca, int ea, const void* b, int64_t ldb, int64_t cb, int eb)
{
    const int64_t pa = lda * ea, pb = ldb * eb, wa = ca * ea, wb = cb * eb;
    const uintptr_t a0 = (uintptr_t) a, b0 = (uintptr_t) b;
    if (a0 + (uintptr_t) ((M - 1) * pa + wa) <= b0 || b0 + (uintptr_t) ((M - 1) * pb + wb) <= a0) return false;
    if (M == 1 || pa != pb) return true;
    // row j of b begins d + (j - i) pa bytes behind row i of a, and meets it if that is in (-wb, wa): the one distance in [0, pa), or
    // the one before
    const int64_t d = (int64_t) (b0 - a0), r = (d % pa + pa) % pa, k = (r - d) / pa;
    return (r < wa && k > -M && k < M) || (r - pa > -wb && k - 1 > -M && k - 1 < M);
}

__host__ __device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ __forceinline__ size_t up128(size_t n) { return (n + 127) & ~(size_t) 127; }

}  // namespace hmoe
