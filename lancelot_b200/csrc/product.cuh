// What the matrix products share (int8_product.cu, fp8_product.cu): results of either type, operands off a 16-byte boundary.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "context.h"

namespace lb {

namespace {

// ---- results ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }

// 32 results of a row, column n0 on
__device__ __forceinline__ void put32(float *p, const float (&v)[32], int valid, int align)
{
    if (valid >= 32 && align == 32) {
#pragma unroll
        for (int e = 0; e < 32; e += 8)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p + e), "r"(__float_as_uint(v[e])), "r"(__float_as_uint(v[e + 1])),
                         "r"(__float_as_uint(v[e + 2])), "r"(__float_as_uint(v[e + 3])), "r"(__float_as_uint(v[e + 4])),
                         "r"(__float_as_uint(v[e + 5])), "r"(__float_as_uint(v[e + 6])), "r"(__float_as_uint(v[e + 7]))
                         : "memory");
    } else if (valid >= 32 && align >= 16) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4 *>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else {
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if (e < valid) p[e] = v[e];
    }
}
__device__ __forceinline__ unsigned pack2(const __nv_bfloat16 *, float a, float b)
{
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<unsigned *>(&v);
}
__device__ __forceinline__ unsigned pack2(const __half *, float a, float b)
{
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<unsigned *>(&v);
}
template <typename T> __device__ __forceinline__ void put32(T *p, const float (&v)[32], int valid, int align)
{
    if (valid >= 32 && align >= 16) {
        unsigned w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack2(p, v[2 * e], v[2 * e + 1]);
        if (align == 32) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p + 2 * e), "r"(w[e]), "r"(w[e + 1]), "r"(w[e + 2]),
                             "r"(w[e + 3]), "r"(w[e + 4]), "r"(w[e + 5]), "r"(w[e + 6]), "r"(w[e + 7])
                             : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4) *reinterpret_cast<uint4 *>(p + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if (e < valid) put(p + e, v[e]);
    }
}

// ---- rows off a 16-byte boundary --------------------------------------------------------------------------------------------
// 16 codes from p on, zeros from `left` codes on.  Not aligned: out of the two aligned lines that they lie in, the second one only where it
// holds one of them.  What else such a line holds is dropped; it lies in the same 16 bytes as a code of the operand, so it can be read.
template <bool ALIGNED> __device__ __forceinline__ uint4 load16(const signed char *p, int left)
{
    if (left <= 0) return make_uint4(0, 0, 0, 0);
    if (ALIGNED) return __ldg(reinterpret_cast<const uint4 *>(p));
    const unsigned shift = (unsigned)(uintptr_t)p & 15;
    const uint4 *line = reinterpret_cast<const uint4 *>(p - shift);
    const uint4 x = __ldg(line);
    uint4 y = make_uint4(0, 0, 0, 0);
    if ((int)shift + min(left, 16) > 16) y = __ldg(line + 1);
    unsigned v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) v[i] = shift & 8 ? v[i + 2] : v[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) v[i] = shift & 4 ? v[i + 1] : v[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = __funnelshift_r(v[i], v[i + 1], 8 * (shift & 3));
        const int keep = left - 4 * i;
        if (keep < 4) v[i] = keep <= 0 ? 0 : v[i] & ((1u << 8 * keep) - 1);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Operands of the tiles whose rows start off a 16-byte boundary are copied once, zeros up to the pitch: a TMA row has to start on such a
// boundary.  Both operands go in one launch; 2^log_lanes threads take a row together.  333 x 1111 x 2047 takes 10.6 us with it, 8.0 us with
// k = 2048 (13.0 us where each thread put four bytes together one by one).
struct Packed {
    const signed char *src;
    long stride, rows;
    signed char *dst;
};
__global__ void __launch_bounds__(256) pack_kernel(const Packed one, const Packed two, const int cols, const int pitch, const int log_lanes)
{
    const int lane = threadIdx.x & ((1 << log_lanes) - 1);
    const long step = (long)gridDim.x << (8 - log_lanes);
    for (long i = ((long)blockIdx.x << (8 - log_lanes)) + (threadIdx.x >> log_lanes); i < one.rows + two.rows; i += step) {
        const bool first = i < one.rows;
        const long r = first ? i : i - one.rows;
        const signed char *p = first ? one.src + r * one.stride : two.src + r * two.stride;
        signed char *to = (first ? one.dst : two.dst) + r * pitch;
        for (int c = lane * 16; c < pitch; c += 16 << log_lanes) *reinterpret_cast<uint4 *>(to + c) = load16<false>(p + c, cols - c);
    }
}

} // namespace

} // namespace lb
