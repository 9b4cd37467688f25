// Matrices in 8-bit floating point with a scale for each block of 128: 128 columns of a row, 128 rows of a column, 128 x 128, or both of the
// first two in one pass.
//
//   s = max|v| / M over the block, rounded to 32 bits (M: the type's largest value)     code = the type's value nearest to v / s, ties to even
//
// The reference has no 8-bit form of anything; products of such matrices (fp8_product.cu) sum over the axis along which a block
// has 128 values, so the operand of a product and that of its gradient are the same matrix in two kinds of blocks.
//
// Both kernels work on tiles of 128 x 128 and are bound by their instructions (some 20 a value and kind of blocks, issued in 70 % of the cycles) rather than by memory:
// 8192 x 4096 in bf16 in rows 31 us (3.2 TB/s), in columns 32, in squares 28.5, in both kinds 50; in 32 bits 34, 35, 33.5 and 54 (3.7 to 4.9 TB/s); 4096 x 11008
// in 32 bits in squares 43.5 us (5.2 TB/s).  Read back to bf16 20 to 24 us (4.3 TB/s).  Rows off their alignment: 8192 x 4095 in bf16 52 and 40 us.
#include <type_traits>

#include "fp8.cuh"
#include "product.cuh"

namespace lb {

namespace {

constexpr int kB = 128;
constexpr unsigned kInf = 0x7f800000u;

// blocks, as the C ABI numbers them
constexpr int kRows = 1, kColumns = 2, kBoth = 3, kSquare = 4;

__device__ __forceinline__ float number(float v) { return v; }
__device__ __forceinline__ float number(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float number(__half v) { return __half2float(v); }

// Four values of a row as they lie.  Magnitudes are ordered like their bit patterns, with infinities and NaN above all numbers, in each of the types:
// an integer maximum carries those along
template <typename T> struct Four { // 16-bit types
    using Raw = uint2;
    static __device__ __forceinline__ Raw load(const T *p) { return __ldg(reinterpret_cast<const uint2 *>(p)); }
    static __device__ __forceinline__ Raw make(const float (&v)[4]) { return make_uint2(pack2((T *)nullptr, v[0], v[1]), pack2((T *)nullptr, v[2], v[3])); }
    static __device__ __forceinline__ unsigned wide(unsigned v) // the 32-bit float's bits of one of the type's in the upper half
    {
        if (sizeof(T) == 2 && std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)(v >> 16))));
        return v;
    }
    static __device__ __forceinline__ uint4 magnitudes(const Raw &x)
    {
        const unsigned a = x.x & 0x7fff7fffu, b = x.y & 0x7fff7fffu;
        if (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a)), g = __half22float2(*reinterpret_cast<const __half2 *>(&b));
            return make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(g.x), __float_as_uint(g.y));
        }
        return make_uint4(a << 16, a & 0x7fff0000u, b << 16, b & 0x7fff0000u);
    }
    static __device__ __forceinline__ unsigned signs(const Raw &x) { return __byte_perm(x.x, x.y, 0x7531) & 0x80808080u; }
    // the largest magnitudes of several: column by column
    using Most = uint2;
    static __device__ __forceinline__ Most none() { return make_uint2(0, 0); }
    static __device__ __forceinline__ Most more(const Most &m, const Raw &x) { return make_uint2(__vmaxu2(m.x, x.x & 0x7fff7fffu), __vmaxu2(m.y, x.y & 0x7fff7fffu)); }
    static __device__ __forceinline__ uint4 columns(const Most &m) { return make_uint4(wide(m.x << 16), wide(m.x & 0xffff0000u), wide(m.y << 16), wide(m.y & 0xffff0000u)); }
    static __device__ __forceinline__ unsigned all(const Most &m)
    {
        const unsigned v = __vmaxu2(m.x, m.y);
        return wide(max(v << 16, v & 0xffff0000u));
    }
};
template <> struct Four<float> {
    using Raw = uint4;
    static __device__ __forceinline__ Raw load(const float *p) { return __ldg(reinterpret_cast<const uint4 *>(p)); }
    static __device__ __forceinline__ Raw make(const float (&v)[4]) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
    static __device__ __forceinline__ uint4 magnitudes(const Raw &x) { return make_uint4(x.x & 0x7fffffffu, x.y & 0x7fffffffu, x.z & 0x7fffffffu, x.w & 0x7fffffffu); }
    static __device__ __forceinline__ unsigned signs(const Raw &x) { return __byte_perm(__byte_perm(x.x, x.y, 0x0073), __byte_perm(x.z, x.w, 0x0073), 0x5410) & 0x80808080u; }
    using Most = uint4;
    static __device__ __forceinline__ Most none() { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ Most more(const Most &m, const Raw &x)
    {
        const uint4 a = magnitudes(x);
        return make_uint4(max(m.x, a.x), max(m.y, a.y), max(m.z, a.z), max(m.w, a.w));
    }
    static __device__ __forceinline__ uint4 columns(const Most &m) { return m; }
    static __device__ __forceinline__ unsigned all(const Most &m) { return max(max(m.x, m.y), max(m.z, m.w)); }
};
template <typename T, bool VEC> __device__ __forceinline__ typename Four<T>::Raw load4(const T *p, int n) // the first n of them, zeros for the others
{
    if (VEC && n >= 4) return Four<T>::load(p);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? number(p[e]) : 0.f;
    return Four<T>::make(v);
}
template <bool E5M2> __device__ __forceinline__ float scale_of(unsigned most)
{
    return most >= kInf ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(most), Fp8<E5M2>::kMost);
}
// What codes are decided by: the scale, and for a block without one (of zeros, or of values so small that their scale rounds to 0) any that makes its codes 0
__device__ __forceinline__ float divisor_of(float scale) { return scale == 0.f ? 1.f : scale; }
__device__ __forceinline__ float4 all(float v) { return make_float4(v, v, v, v); }

struct QuantizeFp8Args {
    const void *values;
    long stride, rows;
    int cols;
    unsigned tiles_c; // tiles of 128 columns
    unsigned char *codes, *down; // blocks along rows (or square ones); along columns
    long code_stride, down_stride;
    float *scales, *down_scales;
    long scale_stride, down_scale_stride;
};

__device__ __forceinline__ void put4(unsigned char *p, unsigned q, int n, bool vec)
{
    if (vec && n >= 4) {
        *reinterpret_cast<unsigned *>(p) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = (unsigned char)(q >> 8 * e);
    }
}
__device__ __forceinline__ bool four_aligned(const unsigned char *p, long stride) { return stride % 4 == 0 && (uintptr_t)p % 4 == 0; }

// A block takes a tile of 128 x 128, a warp eight of its rows, a lane four columns: the values of a row's block are one warp's, and
// a thread's maxima along columns cover its eight rows and then go through shared memory.
constexpr int kWarps = 16, kRowsOf = kB / kWarps;
template <typename T, bool E5M2, int MODE, bool VEC> __global__ void __launch_bounds__(kWarps * 32, 2) quantize_fp8_kernel(const QuantizeFp8Args a)
{
    __shared__ unsigned part[kWarps][kB];
    __shared__ float column[kB];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long tr = blockIdx.x / a.tiles_c;
    const int tc = blockIdx.x - (unsigned)tr * a.tiles_c;
    const int c0 = tc * kB + lane * 4, n = a.cols - c0;
    const long r0 = tr * kB + warp;
    const int rows = (int)min((long)kRowsOf, max(0l, (a.rows - r0 + kWarps - 1) / kWarps)); // of this warp: r0, r0 + 16, ...
    const T *p = reinterpret_cast<const T *>(a.values) + r0 * a.stride + c0;
    typename Four<T>::Raw raw[kRowsOf];
#pragma unroll
    for (int i = 0; i < kRowsOf; ++i, p += kWarps * a.stride) raw[i] = load4<T, VEC>(p, i < rows ? n : 0);
    using V = Four<T>;
    // a whole tile of ordinary scales goes without a question asked for each of its rows
    const bool whole = rows == kRowsOf && tc * kB + kB <= a.cols;
    auto put_rows = [&](unsigned char *to, long stride, auto scale_of_row, bool odd) {
        to += r0 * stride + c0;
        const long step = kWarps * stride;
        if (whole && !odd && four_aligned(to - c0 - r0 * stride, stride)) {
#pragma unroll
            for (int i = 0; i < kRowsOf; ++i, to += step) {
                float4 s, f;
                scale_of_row(i, s, f);
                *reinterpret_cast<unsigned *>(to) = codes4<E5M2, false>(V::magnitudes(raw[i]), s, f) | V::signs(raw[i]);
            }
        } else if (!odd) {
            const bool vec = four_aligned(to - c0 - r0 * stride, stride);
#pragma unroll
            for (int i = 0; i < kRowsOf; ++i, to += step) {
                if (i >= rows) break;
                float4 s, f;
                scale_of_row(i, s, f);
                put4(to, codes4<E5M2, false>(V::magnitudes(raw[i]), s, f) | V::signs(raw[i]), n, vec);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < kRowsOf; ++i, to += step) {
                float4 s, f;
                scale_of_row(i, s, f);
                typename V::Raw x = raw[0];
#pragma unroll
                for (int j = 1; j < kRowsOf; ++j)
                    if (i == j) x = raw[j];
                if (i < rows) put4(to, codes4<E5M2, true>(V::magnitudes(x), s, f) | V::signs(x), n, false);
            }
        }
    };
    if (MODE == kRows || MODE == kBoth) {
        // lane i finds the scale of row i, for all lanes
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < kRowsOf; ++i) {
            const unsigned most = __reduce_max_sync(0xffffffffu, V::all(V::more(V::none(), raw[i])));
            if (lane == i) mine = most;
        }
        const float scale = scale_of<E5M2>(mine), divisor = divisor_of(scale), inverse = inverse_of(divisor);
        if (lane < rows) a.scales[(r0 + lane * kWarps) * a.scale_stride + tc] = scale;
        put_rows(a.codes, a.code_stride, [&](int i, float4 &s, float4 &f) { s = all(__shfl_sync(0xffffffffu, divisor, i)), f = all(__shfl_sync(0xffffffffu, inverse, i)); },
                 __any_sync(0xffffffffu, odd_scale(divisor)));
    }
    if constexpr (MODE == kSquare || MODE == kColumns || MODE == kBoth) {
        typename V::Most most = V::none();
#pragma unroll
        for (int i = 0; i < kRowsOf; ++i) most = V::more(most, raw[i]);
        if constexpr (MODE == kSquare) {
            unsigned m = __reduce_max_sync(0xffffffffu, V::all(most));
            if (lane == 0) part[0][warp] = m;
            __syncthreads();
            m = __reduce_max_sync(0xffffffffu, part[0][lane & (kWarps - 1)]);
            const float scale = scale_of<E5M2>(m), divisor = divisor_of(scale), inverse = inverse_of(divisor);
            if (threadIdx.x == 0) a.scales[tr * a.scale_stride + tc] = scale;
            put_rows(a.codes, a.code_stride, [&](int, float4 &s, float4 &f) { s = all(divisor), f = all(inverse); }, odd_scale(divisor));
        } else {
            *reinterpret_cast<uint4 *>(&part[warp][lane * 4]) = V::columns(most);
            __syncthreads();
            if (threadIdx.x < kB) {
                unsigned m = 0;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = max(m, part[w][threadIdx.x]);
                const float s = scale_of<E5M2>(m);
                column[threadIdx.x] = divisor_of(s);
                if (tc * kB + (int)threadIdx.x < a.cols) a.down_scales[tr * a.down_scale_stride + tc * kB + threadIdx.x] = s;
            }
            __syncthreads();
            const float4 c = *reinterpret_cast<const float4 *>(column + lane * 4);
            const float4 inverse = make_float4(inverse_of(c.x), inverse_of(c.y), inverse_of(c.z), inverse_of(c.w));
            put_rows(a.down, a.down_stride, [&](int, float4 &s, float4 &f) { s = c, f = inverse; },
                     __any_sync(0xffffffffu, odd_scale(c.x) || odd_scale(c.y) || odd_scale(c.z) || odd_scale(c.w)));
        }
    }
}

struct DequantizeFp8Args {
    const unsigned char *codes;
    long code_stride, rows;
    int cols;
    unsigned tiles_c;
    const float *scales;
    long scale_stride;
    int row_shift, col_shift; // 7: a block spans 128 rows, 128 columns; 0: one
    void *out;
    long out_stride;
};

// the same tiles: the scales of a lane's four columns serve its eight rows
template <typename T, bool E5M2, bool VEC> __global__ void __launch_bounds__(kWarps * 32) dequantize_fp8_kernel(const DequantizeFp8Args a)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long tr = blockIdx.x / a.tiles_c;
    const int tc = blockIdx.x - (unsigned)tr * a.tiles_c;
    const int c0 = tc * kB + lane * 4, n = a.cols - c0;
    const long r0 = tr * kB + warp;
    const int rows = (int)min((long)kRowsOf, max(0l, (a.rows - r0 + kWarps - 1) / kWarps));
    if (!VEC) { // rows off their alignment: a lane takes every 32nd column, so that a warp's loads and stores are runs all the same
        const int first = tc * kB + lane;
        float s[4];
        if (!a.col_shift) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = first + 32 * e < a.cols ? __ldg(a.scales + tr * a.scale_stride + first + 32 * e) : 0.f;
        }
        const unsigned char *p = a.codes + r0 * a.code_stride + first;
        T *to = reinterpret_cast<T *>(a.out) + r0 * a.out_stride + first;
#pragma unroll 4
        for (int i = 0; i < rows; ++i) {
            const unsigned char *at = p + i * kWarps * a.code_stride;
            unsigned q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = first + 32 * e < a.cols ? __ldg(at + 32 * e) : 0;
            const float2 x = from_codes2<E5M2>(q[0] | q[1] << 8), y = from_codes2<E5M2>(q[2] | q[3] << 8);
            const float v[4] = {x.x, x.y, y.x, y.y};
            const float one = a.col_shift ? __ldg(a.scales + ((r0 + i * kWarps) >> a.row_shift) * a.scale_stride + tc) : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (first + 32 * e < a.cols) put(to + i * kWarps * a.out_stride + 32 * e, v[e] * (a.col_shift ? one : s[e]));
        }
        return;
    }
    if (n <= 0) return;
    const unsigned char *p = a.codes + r0 * a.code_stride + c0;
    T *to = reinterpret_cast<T *>(a.out) + r0 * a.out_stride + c0;
    const long step = kWarps * a.code_stride, out_step = kWarps * a.out_stride;
    float4 s[kRowsOf];
    if (!a.col_shift) {
        const float *of = a.scales + tr * a.scale_stride + c0;
        s[0] = make_float4(__ldg(of), n > 1 ? __ldg(of + 1) : 0.f, n > 2 ? __ldg(of + 2) : 0.f, n > 3 ? __ldg(of + 3) : 0.f);
#pragma unroll
        for (int i = 1; i < kRowsOf; ++i) s[i] = s[0];
    } else if (a.row_shift) {
        s[0] = all(__ldg(a.scales + tr * a.scale_stride + tc));
#pragma unroll
        for (int i = 1; i < kRowsOf; ++i) s[i] = s[0];
    } else {
        const float *of = a.scales + r0 * a.scale_stride + tc;
#pragma unroll
        for (int i = 0; i < kRowsOf; ++i, of += kWarps * a.scale_stride) s[i] = all(i < rows ? __ldg(of) : 0.f);
    }
    auto value = [&](unsigned q, const float4 &f, float (&v)[4]) {
        const float2 x = from_codes2<E5M2>(q), y = from_codes2<E5M2>(q >> 16);
        v[0] = x.x * f.x, v[1] = x.y * f.y, v[2] = y.x * f.z, v[3] = y.y * f.w;
    };
    if (rows == kRowsOf && tc * kB + kB <= a.cols) { // a whole tile
        unsigned q[kRowsOf];
#pragma unroll
        for (int i = 0; i < kRowsOf; ++i, p += step) q[i] = __ldg(reinterpret_cast<const unsigned *>(p));
#pragma unroll
        for (int i = 0; i < kRowsOf; ++i, to += out_step) {
            float v[4];
            value(q[i], s[i], v);
            *reinterpret_cast<typename Four<T>::Raw *>(to) = Four<T>::make(v);
        }
        return;
    }
    unsigned q[kRowsOf];
#pragma unroll
    for (int i = 0; i < kRowsOf; ++i, p += step) {
        q[i] = 0;
        if (i >= rows) break;
        if (n >= 4) {
            q[i] = __ldg(reinterpret_cast<const unsigned *>(p));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) q[i] |= (unsigned)__ldg(p + e) << 8 * e;
        }
    }
#pragma unroll
    for (int i = 0; i < kRowsOf; ++i, to += out_step) {
        if (i >= rows) break;
        float v[4];
        value(q[i], s[i], v);
        if (n >= 4) {
            *reinterpret_cast<typename Four<T>::Raw *>(to) = Four<T>::make(v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) put(to + e, v[e]);
        }
    }
}

template <typename T, bool E5M2, int MODE> int launch_quantize(const QuantizeFp8Args &a, cudaStream_t stream)
{
    const long tiles = ((a.rows + kB - 1) / kB) * a.tiles_c;
    const long unit = 4 * (long)sizeof(T);
    const bool vec = (uintptr_t)a.values % unit == 0 && (a.rows == 1 || a.stride * (long)sizeof(T) % unit == 0);
    if (vec) quantize_fp8_kernel<T, E5M2, MODE, true><<<(unsigned)tiles, kWarps * 32, 0, stream>>>(a);
    else quantize_fp8_kernel<T, E5M2, MODE, false><<<(unsigned)tiles, kWarps * 32, 0, stream>>>(a);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}
template <typename T, bool E5M2> int quantize_typed(const QuantizeFp8Args &a, int mode, cudaStream_t stream)
{
    switch (mode) {
    case kRows: return launch_quantize<T, E5M2, kRows>(a, stream);
    case kColumns: return launch_quantize<T, E5M2, kColumns>(a, stream);
    case kBoth: return launch_quantize<T, E5M2, kBoth>(a, stream);
    default: return launch_quantize<T, E5M2, kSquare>(a, stream);
    }
}
template <typename T, bool E5M2> int launch_dequantize(const DequantizeFp8Args &a, cudaStream_t stream)
{
    const long tiles = ((a.rows + kB - 1) / kB) * a.tiles_c, unit = 4 * (long)sizeof(T);
    const bool vec = (uintptr_t)a.codes % 4 == 0 && (uintptr_t)a.out % unit == 0 && (a.rows == 1 || (a.code_stride % 4 == 0 && a.out_stride * (long)sizeof(T) % unit == 0));
    if (vec) dequantize_fp8_kernel<T, E5M2, true><<<(unsigned)tiles, kWarps * 32, 0, stream>>>(a);
    else dequantize_fp8_kernel<T, E5M2, false><<<(unsigned)tiles, kWarps * 32, 0, stream>>>(a);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

} // namespace

int quantize_fp8(const void *values, int dtype, long rows, int cols, long stride, int blocks, int code_type, unsigned char *codes, long code_stride,
                 float *scales, long scale_stride, unsigned char *down, long down_stride, float *down_scales, long down_scale_stride, cudaStream_t stream)
{
    QuantizeFp8Args a;
    a.values = values;
    a.stride = stride;
    a.rows = rows;
    a.cols = cols;
    a.tiles_c = (unsigned)((cols + kB - 1) / kB);
    a.codes = codes;
    a.code_stride = code_stride;
    a.scales = scales;
    a.scale_stride = scale_stride;
    a.down = down;
    a.down_stride = down_stride;
    a.down_scales = down_scales;
    a.down_scale_stride = down_scale_stride;
    count_launch("fp8_quantize", stream, (double)rows * cols * ((dtype == 1 ? 4 : 2) + (blocks == kBoth ? 2 : 1)));
    const bool e5m2 = code_type == 6;
    switch (dtype) {
    case 1: return e5m2 ? quantize_typed<float, true>(a, blocks, stream) : quantize_typed<float, false>(a, blocks, stream);
    case 3: return e5m2 ? quantize_typed<__nv_bfloat16, true>(a, blocks, stream) : quantize_typed<__nv_bfloat16, false>(a, blocks, stream);
    default: return e5m2 ? quantize_typed<__half, true>(a, blocks, stream) : quantize_typed<__half, false>(a, blocks, stream);
    }
}

int dequantize_fp8(const unsigned char *codes, int code_type, long code_stride, const float *scales, long scale_stride, int blocks,
                   long rows, int cols, void *out, int dtype, long out_stride, cudaStream_t stream)
{
    DequantizeFp8Args a;
    a.codes = codes;
    a.code_stride = code_stride;
    a.rows = rows;
    a.cols = cols;
    a.tiles_c = (unsigned)((cols + kB - 1) / kB);
    a.scales = scales;
    a.scale_stride = scale_stride;
    a.row_shift = blocks == kRows ? 0 : 7;
    a.col_shift = blocks == kColumns ? 0 : 7;
    a.out = out;
    a.out_stride = out_stride;
    count_launch("fp8_dequantize", stream, (double)rows * cols * (1 + (dtype == 1 ? 4 : 2)));
    const bool e5m2 = code_type == 6;
    switch (dtype) {
    case 1: return e5m2 ? launch_dequantize<float, true>(a, stream) : launch_dequantize<float, false>(a, stream);
    case 3: return e5m2 ? launch_dequantize<__nv_bfloat16, true>(a, stream) : launch_dequantize<__nv_bfloat16, false>(a, stream);
    default: return e5m2 ? launch_dequantize<__half, true>(a, stream) : launch_dequantize<__half, false>(a, stream);
    }
}

} // namespace lb
