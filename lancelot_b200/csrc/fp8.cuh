// 8-bit floating point: e4m3 (three bits behind the point, up to 448) and e5m2 (two bits, up to 57344).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace lb {

namespace {

template <bool E5M2> struct Fp8 {
    static constexpr int kBits = E5M2 ? 2 : 3;
    static constexpr float kMost = E5M2 ? 57344.0f : 448.0f;
    static constexpr float kNormal = E5M2 ? 6.103515625e-05f : 0.015625f; // the least normal number: 2^-14, 2^-6
    static constexpr unsigned kLow = (1u << (23 - kBits)) - 1;           // the bits of a 32-bit number that such a type does not have
    static constexpr unsigned kHalf = 1u << (22 - kBits);                // the first of them: half way between two neighbours
};

// two 32-bit floats to codes, to nearest, ties to even, at most the type's largest value; `a` in the low byte
template <bool E5M2> __device__ __forceinline__ unsigned to_codes2(float a, float b)
{
    unsigned short v;
    if (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(v) : "f"(b), "f"(a));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(b), "f"(a));
    return v;
}
// two codes (of the low 16 bits) to the values that they stand for; both types are part of half
template <bool E5M2> __device__ __forceinline__ float2 from_codes2(unsigned v)
{
    unsigned h;
    if (E5M2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((unsigned short)v));
    else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)v));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Two 32-bit floats in a register pair
__device__ __forceinline__ unsigned long long pair(float a, float b)
{
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ unsigned long long pair(int a, int b)
{
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b));
    return v;
}
__device__ __forceinline__ void unpair(unsigned long long v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b)
{
    unsigned long long v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ void fma2(unsigned long long &c, unsigned long long a, unsigned long long b)
{
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
__device__ __forceinline__ unsigned long long fma2_of(unsigned long long a, unsigned long long b, unsigned long long c)
{
    unsigned long long v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ unsigned long long fma2_towards_zero(unsigned long long a, unsigned long long b, unsigned long long c)
{
    unsigned long long v;
    asm("fma.rz.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ float fma_sat(float a, float b, float c) // cut to [0, 1]
{
    float v;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}

// The code nearest to m / s, m >= 0, decided exactly.  q = m * (1 / s) in 32 bits is within two steps of the quotient.  The codes on either side of q
// have the border h between them, of five bits at most, and the sign of d = m - h s, exact in one fused multiply-add for s >= 2^-80, says on which
// side of it the quotient lies, 0 that it lies on it.  So what is rounded to a code is not q but h (1 - 2^-10), h or h (1 + 2^-10): a tie goes to the
// even code.  (Where q itself lies next to a code, on the wrong side of it, the border next to q still sends it to that code.)  Below the
// least normal number the codes are evenly spaced; that number added to q brings their borders to the same bits (rounded towards zero: the last q below it,
// rounded to nearest, would make twice that number, where borders are spaced twice as far).  Choices are made by
// multiply-adds cut to [0, 1], which cost half of what comparisons do, and nothing depends on how often values lie next to a border: 16-bit
// values often lie on one.
constexpr float kTinyScale = 0x1p-80f;

template <bool E5M2> __device__ __forceinline__ unsigned long long beside_border(unsigned long long m, unsigned long long s, unsigned long long f)
{
    using F = Fp8<E5M2>;
    const unsigned long long q = mul2(m, f);
    float q0, q1, w0, w1, d0, d1;
    unpair(q, q0, q1);
    const unsigned long long y = pair(fma_sat(q0, -0x1p60f, F::kNormal * 0x1p60f), fma_sat(q1, -0x1p60f, F::kNormal * 0x1p60f)); // 1: below the normal numbers
    unpair(fma2_towards_zero(y, pair(F::kNormal, F::kNormal), q), w0, w1);
    // -h, which spares turning m
    const unsigned long long h = fma2_of(y, pair(F::kNormal, F::kNormal), pair(__uint_as_float((__float_as_uint(w0) & ~F::kLow) | (F::kHalf | 0x80000000u)),
                                                                               __uint_as_float((__float_as_uint(w1) & ~F::kLow) | (F::kHalf | 0x80000000u))));
    unpair(fma2_of(h, s, m), d0, d1);
    const unsigned long long z = pair(fma_sat(d0, 0x1p125f, 0.5f), fma_sat(d1, 0x1p125f, 0.5f)); // d is a multiple of 2^-120
    return mul2(h, fma2_of(z, pair(-0x1p-9f, -0x1p-9f), pair(-1.f + 0x1p-10f, -1.f + 0x1p-10f)));
}
// smaller scales: a quotient of 64 bits, rounded to 24 in a way that keeps what lies beyond them in the last bit, so that rounding once more is
// right.  0 where the scale is not finite
__device__ __noinline__ float quotient_of_tiny(float m, float s)
{
    if (!(s > 0.f)) return 0.f;
    const double q = (double)m / (double)s;
    const float f = __double2float_rz(q);
    return (double)f == q ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ float inverse_of(float s) { return s >= kTinyScale ? __frcp_rn(s) : 0.f; }
// whether a block's codes cannot be had with that
__device__ __forceinline__ bool odd_scale(float s) { return !(s >= kTinyScale); }

// The codes of four magnitudes (bits), of one scale or of a scale each (s), with the factors to their quotients (f).  ODD: one of the scales may be
template <bool E5M2, bool ODD> __device__ __forceinline__ unsigned codes4(const uint4 &m, const float4 &s, const float4 &f)
{
    const float a = __uint_as_float(m.x), b = __uint_as_float(m.y), c = __uint_as_float(m.z), d = __uint_as_float(m.w);
    float q0, q1, q2, q3;
    unpair(beside_border<E5M2>(pair(a, b), pair(s.x, s.y), pair(f.x, f.y)), q0, q1);
    unpair(beside_border<E5M2>(pair(c, d), pair(s.z, s.w), pair(f.z, f.w)), q2, q3);
    if constexpr (ODD) {
        if (!(s.x >= kTinyScale)) q0 = quotient_of_tiny(a, s.x);
        if (!(s.y >= kTinyScale)) q1 = quotient_of_tiny(b, s.y);
        if (!(s.z >= kTinyScale)) q2 = quotient_of_tiny(c, s.z);
        if (!(s.w >= kTinyScale)) q3 = quotient_of_tiny(d, s.w);
    }
    return to_codes2<E5M2>(q0, q1) | to_codes2<E5M2>(q2, q3) << 16;
}

} // namespace

} // namespace lb
