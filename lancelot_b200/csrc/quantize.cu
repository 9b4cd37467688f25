// The 8-bit cache of client updates: rows of values are written as codes with a scale per group of columns and read back.
//
//   t = value + residual (32 bits; 0 behind a row's length)    s = max|t| / 127 over the group, rounded to 32 bits
//   q = the integer nearest to t / s, ties to even             what the rounding lost: t - q s
//
// The reference has no 8-bit form of an update: its driver holds every client's values in the clear as lists of doubles
// (lancelot-main-GPU/utils/byzantine_fl.py:478-490).
//
// The nearest integer is found without a division.  q0 = rint(t * (1 / s)) is off by at most one, and only next to a border
// between two codes; r = fma(-q0, s, t) is exact there (both terms are multiples of the smaller of their units in the last
// place, and |r| is about s / 2, so it has at most 24 bits), and comparing 2 |r| with s settles the border, ties included.
// The same r is what the rounding lost, exactly: error feedback adds no error of its own.
//
// All kernels stream: bound by HBM at (value bytes + 1 + 8 with a residual) per value.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "context.h"

namespace lb {

namespace {

constexpr unsigned kInfBits = 0x7f800000u;

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four consecutive values as 32-bit floats.  `valid`: how many of them lie inside the row (<= 0: none)
template <bool VEC> __device__ __forceinline__ float4 load4(const float *p, long valid)
{
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && valid >= 4) return __ldcs(reinterpret_cast<const float4 *>(p));
    if (valid > 0) v.x = __ldcs(p);
    if (valid > 1) v.y = __ldcs(p + 1);
    if (valid > 2) v.z = __ldcs(p + 2);
    if (valid > 3) v.w = __ldcs(p + 3);
    return v;
}
template <bool VEC> __device__ __forceinline__ float4 load4(const __nv_bfloat16 *p, long valid)
{
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && valid >= 4) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(p));
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xffff0000u));
    }
    if (valid > 0) v.x = __bfloat162float(p[0]);
    if (valid > 1) v.y = __bfloat162float(p[1]);
    if (valid > 2) v.z = __bfloat162float(p[2]);
    if (valid > 3) v.w = __bfloat162float(p[3]);
    return v;
}
template <bool VEC> __device__ __forceinline__ float4 load4(const __half *p, long valid)
{
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && valid >= 4) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(p));
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    if (valid > 0) v.x = __half2float(p[0]);
    if (valid > 1) v.y = __half2float(p[1]);
    if (valid > 2) v.z = __half2float(p[2]);
    if (valid > 3) v.w = __half2float(p[3]);
    return v;
}

template <bool VEC> __device__ __forceinline__ void store4(float *p, float4 v, long valid)
{
    if (VEC && valid >= 4) {
        __stcs(reinterpret_cast<float4 *>(p), v);
        return;
    }
    if (valid > 0) p[0] = v.x;
    if (valid > 1) p[1] = v.y;
    if (valid > 2) p[2] = v.z;
    if (valid > 3) p[3] = v.w;
}
template <bool VEC> __device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v, long valid)
{
    if (VEC && valid >= 4) {
        __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        __stcs(reinterpret_cast<uint2 *>(p), make_uint2(*reinterpret_cast<unsigned *>(&a), *reinterpret_cast<unsigned *>(&b)));
        return;
    }
    if (valid > 0) p[0] = __float2bfloat16_rn(v.x);
    if (valid > 1) p[1] = __float2bfloat16_rn(v.y);
    if (valid > 2) p[2] = __float2bfloat16_rn(v.z);
    if (valid > 3) p[3] = __float2bfloat16_rn(v.w);
}
template <bool VEC> __device__ __forceinline__ void store4(__half *p, float4 v, long valid)
{
    if (VEC && valid >= 4) {
        __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        __stcs(reinterpret_cast<uint2 *>(p), make_uint2(*reinterpret_cast<unsigned *>(&a), *reinterpret_cast<unsigned *>(&b)));
        return;
    }
    if (valid > 0) p[0] = __float2half_rn(v.x);
    if (valid > 1) p[1] = __float2half_rn(v.y);
    if (valid > 2) p[2] = __float2half_rn(v.z);
    if (valid > 3) p[3] = __float2half_rn(v.w);
}

// Rows that start off a 16-byte boundary (an odd number of values a row is the rule for updates).  The warp's run of columns
// is still contiguous, so it moves in aligned pieces and the lanes hand the values on to where they belong: `off` values of a piece
// belong to the lane before.  All 32 lanes take part; lane l stands for columns col .. col + 3, col = (lane 0's) + 4 l.  Only values with
// 0 <= column < limit are touched.
template <typename T> __device__ __forceinline__ float4 load_piece(const T *row, long at, long limit)
{
    if (at >= 0 && at + 4 <= limit) return load4<true>(row + at, 4);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= 0 && at < limit) v.x = (float)row[at];
    if (at + 1 >= 0 && at + 1 < limit) v.y = (float)row[at + 1];
    if (at + 2 >= 0 && at + 2 < limit) v.z = (float)row[at + 2];
    if (at + 3 >= 0 && at + 3 < limit) v.w = (float)row[at + 3];
    return v;
}
template <typename T> __device__ __forceinline__ float4 load_shifted(const T *row, long col, long limit)
{
    const int off = (int)((uintptr_t)(row + col) / sizeof(T)) & 3;
    const float4 a = load_piece(row, col - off, limit);
    if (off == 0) return a;
    float4 next = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool last = (threadIdx.x & 31) == 31;
    if (last) next = load_piece(row, col - off + 4, limit);
    const float x = __shfl_down_sync(0xffffffffu, a.x, 1), y = __shfl_down_sync(0xffffffffu, a.y, 1), z = __shfl_down_sync(0xffffffffu, a.z, 1);
    if (!last) next = make_float4(x, y, z, 0.f);
    if (off == 1) return make_float4(a.y, a.z, a.w, next.x);
    if (off == 2) return make_float4(a.z, a.w, next.x, next.y);
    return make_float4(a.w, next.x, next.y, next.z);
}
template <typename T> __device__ __forceinline__ void store_shifted(T *row, long col, float4 v, long limit)
{
    const int off = (int)((uintptr_t)(row + col) / sizeof(T)) & 3;
    if (off == 0) {
        store4<true>(row + col, v, limit - col);
        return;
    }
    const float y = __shfl_up_sync(0xffffffffu, v.y, 1), z = __shfl_up_sync(0xffffffffu, v.z, 1), w = __shfl_up_sync(0xffffffffu, v.w, 1);
    const int lane = threadIdx.x & 31;
    const float4 piece = off == 1 ? make_float4(w, v.x, v.y, v.z) : off == 2 ? make_float4(z, w, v.x, v.y) : make_float4(y, z, w, v.x);
    if (lane == 0) store4<false>(row + col, v, min(limit - col, 4L - off)); // the rest of the piece is not this warp's
    else store4<true>(row + col - off, piece, limit - col + off);
    if (lane == 31) {
        const float4 rest = off == 1 ? make_float4(v.w, 0.f, 0.f, 0.f) : off == 2 ? make_float4(v.z, v.w, 0.f, 0.f) : make_float4(v.y, v.z, v.w, 0.f);
        store4<false>(row + col + 4 - off, rest, min(limit - col - 4 + off, (long)off));
    }
}

// The scale of a group from the bits of its largest magnitude.  The bit patterns of magnitudes are ordered like the magnitudes
// with infinities and NaN above all numbers, so an integer maximum carries them along: such a group gets NaN
__device__ __forceinline__ float scale_of(unsigned most)
{
    return most >= kInfBits ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(most), 127.0f);
}

// the code of t in a group of scale s (inv = 1 / s); t <- what the rounding lost
__device__ __forceinline__ int code_of(float &t, float s, float inv)
{
    float q = rintf(t * inv);
    float r = fmaf(-q, s, t);
    const float twice = fabsf(r + r);
    // past the border, or on it with an odd code: the neighbour on the side of r
    if (twice > s || (twice == s && ((int)q & 1))) {
        q += copysignf(1.0f, r);
        r = fmaf(-q, s, t);
    }
    t = r;
    return (int)q;
}
// Groups without a normal scale: empty (0), not finite (NaN), or so small that 1 / s overflows and the rounding of s itself
// moves codes past 127; a quotient of 64 bits decides a border between 32-bit numbers rightly
__device__ __noinline__ float2 code_of_odd(float t, float s) // (code, what was lost)
{
    if (!(s > 0.0f)) return make_float2(0.0f, s == s ? t : 0.0f);
    const double q = fmin(fmax(rint((double)t / (double)s), -127.0), 127.0);
    return make_float2((float)q, (float)((double)t - q * (double)s));
}

// codes of four values, packed; v <- what was lost
__device__ __forceinline__ unsigned codes4(float4 &v, float s)
{
    int a, b, c, d;
    if (s >= 1.17549435e-38f) {
        const float inv = __frcp_rn(s);
        a = code_of(v.x, s, inv);
        b = code_of(v.y, s, inv);
        c = code_of(v.z, s, inv);
        d = code_of(v.w, s, inv);
    } else {
        const float2 x = code_of_odd(v.x, s), y = code_of_odd(v.y, s), z = code_of_odd(v.z, s), w = code_of_odd(v.w, s);
        v = make_float4(x.y, y.y, z.y, w.y);
        a = (int)x.x;
        b = (int)y.x;
        c = (int)z.x;
        d = (int)w.x;
    }
    return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)d << 24;
}

__device__ __forceinline__ unsigned most4(const float4 &v)
{
    return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
}

struct QuantizeArgs {
    const void *values;
    long value_stride;
    const int *lengths;
    const float *residual;
    float *residual_out;
    long residual_stride;
    long n_cols;
    int page, pages; // columns of a page, pages of a row
    const int *slots;
    long n_slots;
    signed char *codes;
    long code_stride;
    float *scales;
    long scale_stride;
    int group, groups; // columns of a group, groups of a page
};

// where a page's codes go; false: the page is skipped
__device__ __forceinline__ bool page_slot(const QuantizeArgs &a, long page_index, long &slot)
{
    slot = a.slots ? (long)a.slots[page_index] : page_index;
    return slot >= 0 && slot < a.n_slots;
}
__device__ __forceinline__ long row_limit(const QuantizeArgs &a, long row)
{
    return a.lengths ? min((long)max(a.lengths[row], 0), a.n_cols) : a.n_cols;
}

// t for columns col .. col + 3 of a row, 0 from column `limit` on.  VEC: all rows start on the boundary of a vector
template <typename T, bool VEC> __device__ __forceinline__ float4 load_sum(const QuantizeArgs &a, long row, long col, long limit)
{
    const T *values = reinterpret_cast<const T *>(a.values) + row * a.value_stride;
    float4 v = VEC ? load4<true>(values + col, limit - col) : load_shifted(values, col, limit);
    if (a.residual) {
        const float *res = a.residual + row * a.residual_stride;
        const float4 r = VEC ? load4<true>(res + col, limit - col) : load_shifted(res, col, limit);
        v.x += r.x;
        v.y += r.y;
        v.z += r.z;
        v.w += r.w;
    }
    return v;
}
template <bool VEC> __device__ __forceinline__ void store_lost(const QuantizeArgs &a, long row, long col, const float4 &v, long limit)
{
    if (!a.residual_out) return;
    float *out = a.residual_out + row * a.residual_stride;
    if (VEC) store4<true>(out + col, v, limit - col);
    else store_shifted(out, col, v, limit);
}

// ---- groups of 32 to 512 columns: a warp takes 512 columns, four of each lane's values side by side -------------------
// Every load and store of a warp is one contiguous run (512 bytes of 32-bit values, 128 bytes of codes); a group's maximum
// never leaves the warp.
template <typename T, bool VEC, int LOG_G>
__global__ void __launch_bounds__(256) quantize_warp_kernel(const QuantizeArgs a, const unsigned tiles, const unsigned total)
{
    const unsigned w = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (w >= total) return;
    const int lane = threadIdx.x & 31;
    const unsigned page_index = w / tiles, tile = w - page_index * tiles;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    long slot;
    if (!page_slot(a, page_index, slot)) return;
    const long limit = min(row_limit(a, row), (long)(page + 1) * a.page);
    const int in_page = tile * 512 + lane * 4;
    const long col = (long)page * a.page + in_page;
    float4 v[4];
    unsigned m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load_sum<T, VEC>(a, row, col + j * 128, limit);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = most4(v[j]);
        if (LOG_G >= 7) {
            m[j] = __reduce_max_sync(0xffffffffu, m[j]);
        } else {
            if (LOG_G >= 6) m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
            m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 4));
            m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 2));
            m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 1));
        }
    }
    if (LOG_G >= 8) {
        m[0] = m[1] = max(m[0], m[1]);
        m[2] = m[3] = max(m[2], m[3]);
    }
    if (LOG_G >= 9) m[0] = m[1] = m[2] = m[3] = max(m[0], m[2]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = in_page + j * 128;
        const float s = scale_of(m[j]);
        const unsigned q = codes4(v[j], s);
        if (c < a.page) {
            if ((c & ((1 << LOG_G) - 1)) == 0) a.scales[slot * a.scale_stride + (c >> LOG_G)] = s;
            *reinterpret_cast<unsigned *>(a.codes + slot * a.code_stride + c) = q;
        }
        store_lost<VEC>(a, row, col + j * 128, v[j], limit);
    }
}

// ---- groups of up to 32768 columns: a block holds the group in registers ----------------------------------------------
template <typename T, bool VEC, int THREADS, int V>
__global__ void __launch_bounds__(THREADS) quantize_block_kernel(const QuantizeArgs a)
{
    __shared__ unsigned warp_most[32];
    const unsigned page_index = blockIdx.x / (unsigned)a.groups, g = blockIdx.x - page_index * (unsigned)a.groups;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    long slot;
    if (!page_slot(a, page_index, slot)) return;
    const int first = g * a.group, end = min(a.page, first + a.group); // columns of the group inside the page
    const long limit = min(row_limit(a, row), (long)page * a.page + end);
    const int in_page = first + threadIdx.x * 4;
    const long col = (long)page * a.page + in_page;
    float4 v[V];
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = load_sum<T, VEC>(a, row, col + j * THREADS * 4, limit);
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, most4(v[j]));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = m;
    __syncthreads();
    m = (threadIdx.x & 31) < THREADS / 32 ? warp_most[threadIdx.x & 31] : 0;
    m = __reduce_max_sync(0xffffffffu, m);
    const float s = scale_of(m);
    if (threadIdx.x == 0) a.scales[slot * a.scale_stride + g] = s;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = in_page + j * THREADS * 4;
        const unsigned q = codes4(v[j], s);
        if (c < end) *reinterpret_cast<unsigned *>(a.codes + slot * a.code_stride + c) = q;
        store_lost<VEC>(a, row, col + j * THREADS * 4, v[j], limit);
    }
}

// ---- longer groups: the maxima of parts of 32768 columns first, then the codes -----------------------------------------
constexpr int kPart = 32768;

template <typename T, bool VEC, bool WRITE>
__global__ void __launch_bounds__(1024) quantize_part_kernel(const QuantizeArgs a, unsigned *__restrict__ part_most, const unsigned parts)
{
    __shared__ unsigned warp_most[32];
    const unsigned group_index = blockIdx.x / parts, part = blockIdx.x - group_index * parts;
    const unsigned page_index = group_index / (unsigned)a.groups, g = group_index - page_index * (unsigned)a.groups;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    long slot;
    if (!page_slot(a, page_index, slot)) return;
    const long first = (long)g * a.group;
    const long end = min((long)a.page, first + a.group);
    const long limit = min(row_limit(a, row), (long)page * a.page + end);
    const long in_page = first + (long)part * kPart + threadIdx.x * 4;
    const long col = (long)page * a.page + in_page;
    unsigned m = 0;
    if (WRITE) {
        for (unsigned p = threadIdx.x & 31; p < parts; p += 32) m = max(m, part_most[(size_t)group_index * parts + p]);
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const float s = scale_of(m);
    if (WRITE && part == 0 && threadIdx.x == 0) a.scales[slot * a.scale_stride + g] = s;
#pragma unroll 4
    for (int j = 0; j < kPart / 4096; ++j) {
        const long c = in_page + j * 4096;
        float4 v = load_sum<T, VEC>(a, row, col + j * 4096, limit);
        if (WRITE) {
            const unsigned q = codes4(v, s);
            if (c < end) *reinterpret_cast<unsigned *>(a.codes + slot * a.code_stride + c) = q;
            store_lost<VEC>(a, row, col + j * 4096, v, limit);
        } else {
            m = max(m, most4(v));
        }
    }
    if (!WRITE) {
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = m;
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, warp_most[threadIdx.x & 31]);
        if (threadIdx.x == 0) part_most[(size_t)group_index * parts + part] = m;
    }
}

template <typename T, bool VEC>
int quantize_typed(const QuantizeArgs &a, long n_rows, void *workspace, double bytes, cudaStream_t stream)
{
    const long n_pages = n_rows * a.pages;
    const int longest = a.group < a.page ? a.group : a.page; // columns of the longest group
    count_launch("quantize", stream, bytes);
    if (longest <= 512) {
        const unsigned tiles = (a.page + 511) / 512, total = (unsigned)(n_pages * tiles);
        const unsigned grid = (total + 7) / 8;
        switch (a.group) {
        case 32: quantize_warp_kernel<T, VEC, 5><<<grid, 256, 0, stream>>>(a, tiles, total); break;
        case 64: quantize_warp_kernel<T, VEC, 6><<<grid, 256, 0, stream>>>(a, tiles, total); break;
        case 128: quantize_warp_kernel<T, VEC, 7><<<grid, 256, 0, stream>>>(a, tiles, total); break;
        case 256: quantize_warp_kernel<T, VEC, 8><<<grid, 256, 0, stream>>>(a, tiles, total); break;
        default: quantize_warp_kernel<T, VEC, 9><<<grid, 256, 0, stream>>>(a, tiles, total); break; // 512, or one group in a page of at most 512
        }
    } else if (longest <= kPart) {
        const unsigned grid = (unsigned)(n_pages * a.groups);
        if (longest <= 1024) quantize_block_kernel<T, VEC, 256, 1><<<grid, 256, 0, stream>>>(a);
        else if (longest <= 4096) quantize_block_kernel<T, VEC, 256, 4><<<grid, 256, 0, stream>>>(a);
        else if (longest <= 8192) quantize_block_kernel<T, VEC, 512, 4><<<grid, 512, 0, stream>>>(a);
        else if (longest <= 16384) quantize_block_kernel<T, VEC, 1024, 4><<<grid, 1024, 0, stream>>>(a);
        else quantize_block_kernel<T, VEC, 1024, 8><<<grid, 1024, 0, stream>>>(a);
    } else {
        const unsigned parts = (unsigned)((longest + kPart - 1) / kPart);
        const unsigned grid = (unsigned)(n_pages * a.groups * parts);
        quantize_part_kernel<T, VEC, false><<<grid, 1024, 0, stream>>>(a, (unsigned *)workspace, parts);
        LB_CUDA(cudaGetLastError());
        count_launch("quantize", stream);
        quantize_part_kernel<T, VEC, true><<<grid, 1024, 0, stream>>>(a, (unsigned *)workspace, parts);
    }
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

// ---- reading back ------------------------------------------------------------------------------------------------------
struct DequantizeArgs {
    const signed char *codes;
    long code_stride;
    const float *scales;
    long scale_stride;
    long n_slots;
    int page, pages, log_group; // log_group 31: one group in a page
    const int *slots;
    long n_cols;
    void *out;
    long out_stride;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantizeArgs a, const unsigned tiles, const unsigned total)
{
    const unsigned w = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (w >= total) return;
    const int lane = threadIdx.x & 31;
    const unsigned page_index = w / tiles, tile = w - page_index * tiles;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    const long slot = a.slots ? (long)a.slots[page_index] : (long)page_index;
    const bool there = slot >= 0 && slot < a.n_slots; // a page that is not in the cache reads as zeros
    const int in_page = tile * 512 + lane * 4;
    const long col = (long)page * a.page + in_page;
    unsigned q[4] = {0, 0, 0, 0};
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = in_page + j * 128;
        if (there && c < a.page && col + j * 128 < a.n_cols) {
            q[j] = __ldcs(reinterpret_cast<const unsigned *>(a.codes + slot * a.code_stride + c));
            s[j] = __ldg(a.scales + slot * a.scale_stride + (c >> a.log_group));
        }
    }
    T *out = reinterpret_cast<T *>(a.out) + (long)row * a.out_stride;
    const long limit = min(a.n_cols, (long)(page + 1) * a.page);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float4 v = make_float4(s[j] * (float)(signed char)(q[j] & 255), s[j] * (float)(signed char)(q[j] >> 8 & 255),
                                     s[j] * (float)(signed char)(q[j] >> 16 & 255), s[j] * (float)(signed char)(q[j] >> 24));
        if (VEC) store4<true>(out + col + j * 128, v, limit - col - j * 128);
        else store_shifted(out, col + j * 128, v, limit);
    }
}

template <typename T> bool aligned4(const void *p, long stride) { return (uintptr_t)p % (4 * sizeof(T)) == 0 && stride % 4 == 0; }

} // namespace

size_t quantize_workspace_bytes(long n_rows, long n_cols, int page, int group)
{
    const int longest = group == 0 || group > page ? page : group;
    if (longest <= kPart) return 0;
    const long pages = (n_cols + page - 1) / page, groups = (page + longest - 1) / longest;
    return sizeof(unsigned) * (size_t)(n_rows * pages * groups * ((longest + kPart - 1) / kPart));
}

int quantize_rows(const void *values, int dtype, long n_rows, long n_cols, long value_stride, const int *lengths, const float *residual,
                  float *residual_out, long residual_stride, const int *slots, long n_slots, int page, int group, signed char *codes,
                  long code_stride, float *scales, long scale_stride, void *workspace, cudaStream_t stream)
{
    QuantizeArgs a;
    a.values = values;
    a.value_stride = value_stride;
    a.lengths = lengths;
    a.residual = residual;
    a.residual_out = residual_out;
    a.residual_stride = residual_stride;
    a.n_cols = n_cols;
    a.page = page;
    a.pages = (int)((n_cols + page - 1) / page);
    a.slots = slots;
    a.n_slots = n_slots;
    a.codes = codes;
    a.code_stride = code_stride;
    a.scales = scales;
    a.scale_stride = scale_stride;
    // one group in a page: a power of two that covers it, as far as the warp kernel goes
    a.group = group == 0 || group >= page ? (page <= 512 ? 512 : page) : group;
    a.groups = (page + a.group - 1) / a.group;
    const bool res = (!residual || aligned4<float>(residual, residual_stride)) && (!residual_out || aligned4<float>(residual_out, residual_stride));
    const double bytes = (double)n_rows * n_cols * ((dtype == 1 ? 4 : 2) + 1 + (residual ? 4 : 0) + (residual_out ? 4 : 0));
    switch (dtype) {
    case 1:
        return res && aligned4<float>(values, value_stride) ? quantize_typed<float, true>(a, n_rows, workspace, bytes, stream)
                                                            : quantize_typed<float, false>(a, n_rows, workspace, bytes, stream);
    case 3:
        return res && aligned4<__nv_bfloat16>(values, value_stride) ? quantize_typed<__nv_bfloat16, true>(a, n_rows, workspace, bytes, stream)
                                                                    : quantize_typed<__nv_bfloat16, false>(a, n_rows, workspace, bytes, stream);
    default:
        return res && aligned4<__half>(values, value_stride) ? quantize_typed<__half, true>(a, n_rows, workspace, bytes, stream)
                                                             : quantize_typed<__half, false>(a, n_rows, workspace, bytes, stream);
    }
}

int dequantize_rows(const signed char *codes, long code_stride, const float *scales, long scale_stride, long n_slots, int page, int group,
                    const int *slots, long n_rows, long n_cols, void *out, int dtype, long out_stride, cudaStream_t stream)
{
    DequantizeArgs a;
    a.codes = codes;
    a.code_stride = code_stride;
    a.scales = scales;
    a.scale_stride = scale_stride;
    a.n_slots = n_slots;
    a.page = page;
    a.pages = (int)((n_cols + page - 1) / page);
    a.log_group = 31;
    if (group > 0 && group < page) a.log_group = __builtin_ctz((unsigned)group);
    a.slots = slots;
    a.n_cols = n_cols;
    a.out = out;
    a.out_stride = out_stride;
    const unsigned tiles = (page + 511) / 512, total = (unsigned)(n_rows * a.pages * tiles), grid = (total + 7) / 8;
    count_launch("dequantize", stream, (double)n_rows * n_cols * (1 + (dtype == 1 ? 4 : 2)));
    if (dtype == 1) {
        if (aligned4<float>(out, out_stride)) dequantize_kernel<float, true><<<grid, 256, 0, stream>>>(a, tiles, total);
        else dequantize_kernel<float, false><<<grid, 256, 0, stream>>>(a, tiles, total);
    } else if (dtype == 3) {
        if (aligned4<__nv_bfloat16>(out, out_stride)) dequantize_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(a, tiles, total);
        else dequantize_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(a, tiles, total);
    } else {
        if (aligned4<__half>(out, out_stride)) dequantize_kernel<__half, true><<<grid, 256, 0, stream>>>(a, tiles, total);
        else dequantize_kernel<__half, false><<<grid, 256, 0, stream>>>(a, tiles, total);
    }
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

} // namespace lb
