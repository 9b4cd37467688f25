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

// The code nearest to t / s, decided exactly, with one product.  q = t * (1 / s) in 32 bits is within two steps (2^-22 relative) of the quotient, so its
// code is right unless q lies that near to a border between two codes.  There the border h, which has five bits at most, is
// compared itself: the sign of h s - |t| is exact in one fused multiply-add for s >= 2^-100.  Below the least normal number the codes are evenly
// spaced; adding that number brings their borders to the same bits of the sum.
template <bool E5M2> __device__ __forceinline__ bool near_border(float q)
{
    using F = Fp8<E5M2>;
    const float m = fabsf(q);
    const unsigned u = __float_as_uint(m < F::kNormal ? m + F::kNormal : m);
    return ((u & F::kLow) - (F::kHalf - 4)) <= 8u;
}
template <bool E5M2> __device__ __forceinline__ float settled(float q, float t, float s) // q, moved off the border to its right side, or onto it
{
    using F = Fp8<E5M2>;
    if (!near_border<E5M2>(q)) return q;
    const float m = fabsf(q);
    const bool low = m < F::kNormal;
    float h = __uint_as_float((__float_as_uint(low ? m + F::kNormal : m) & ~F::kLow) | F::kHalf);
    if (low) h -= F::kNormal;
    const float d = fmaf(h, s, -fabsf(t));
    if (d != 0.f) h *= d > 0.f ? 1.f - 0x1p-12f : 1.f + 0x1p-12f;
    return copysignf(h, t);
}
// scales below that (1 / s may pass the range, and h s the smallest numbers): a quotient of 64 bits, rounded to 24 in a way that keeps
// what lies beyond them in the last bit, so that rounding once more is right
__device__ __noinline__ float quotient_of_tiny(float t, float s)
{
    const double q = (double)t / (double)s;
    const float f = __double2float_rz(q);
    return (double)f == q ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

constexpr float kTinyScale = 0x1p-100f;

// the factor that takes a value to its quotient; 0 where the codes are 0 (a block of zeros, one that is not finite), and for the scales
// that quotient_of_tiny serves
__device__ __forceinline__ float inverse_of(float s) { return s >= kTinyScale ? __frcp_rn(s) : 0.f; }

// four codes of one scale, or of a scale each
template <bool E5M2> __device__ __forceinline__ unsigned codes4(const float *t, float s0, float s1, float s2, float s3, float i0, float i1, float i2, float i3)
{
    float a = t[0] * i0, b = t[1] * i1, c = t[2] * i2, d = t[3] * i3;
    if (i0 == 0.f || i1 == 0.f || i2 == 0.f || i3 == 0.f) { // seldom: none of this is on the way of ordinary blocks
        a = i0 != 0.f ? settled<E5M2>(a, t[0], s0) : s0 > 0.f ? quotient_of_tiny(t[0], s0) : 0.f;
        b = i1 != 0.f ? settled<E5M2>(b, t[1], s1) : s1 > 0.f ? quotient_of_tiny(t[1], s1) : 0.f;
        c = i2 != 0.f ? settled<E5M2>(c, t[2], s2) : s2 > 0.f ? quotient_of_tiny(t[2], s2) : 0.f;
        d = i3 != 0.f ? settled<E5M2>(d, t[3], s3) : s3 > 0.f ? quotient_of_tiny(t[3], s3) : 0.f;
    } else if (near_border<E5M2>(a) | near_border<E5M2>(b) | near_border<E5M2>(c) | near_border<E5M2>(d)) {
        a = settled<E5M2>(a, t[0], s0);
        b = settled<E5M2>(b, t[1], s1);
        c = settled<E5M2>(c, t[2], s2);
        d = settled<E5M2>(d, t[3], s3);
    }
    return to_codes2<E5M2>(a, b) | to_codes2<E5M2>(c, d) << 16;
}

} // namespace

} // namespace lb
