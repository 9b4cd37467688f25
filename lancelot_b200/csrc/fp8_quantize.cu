// Matrices in 8-bit floating point with a scale for each block of 128: 128 columns of a row, 128 rows of a column, 128 x 128, or both of the
// first two in one pass.
//
//   s = max|v| / M over the block, rounded to 32 bits (M: the type's largest value)     code = the type's value nearest to v / s, ties to even
//
// The reference has no 8-bit form of anything; products of such matrices (fp8_product.cu) sum over the axis along which a block
// has 128 values, so the operand of a product and that of its gradient are the same matrix in two kinds of blocks.
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

// 16 values on a 16-byte boundary
__device__ __forceinline__ void load16v(const float *p, float *v)
{
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4 *>(p + e));
        v[e] = x.x, v[e + 1] = x.y, v[e + 2] = x.z, v[e + 3] = x.w;
    }
}
__device__ __forceinline__ void load16v(const __nv_bfloat16 *p, float *v)
{
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
        const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p + e));
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e + 2 * i] = __uint_as_float(w[i] << 16), v[e + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load16v(const __half *p, float *v)
{
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
        const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p + e));
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[e + 2 * i] = f.x, v[e + 2 * i + 1] = f.y;
        }
    }
}

// magnitudes are ordered like their bit patterns, with infinities and NaN above all numbers: an integer maximum carries them along
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
template <bool E5M2> __device__ __forceinline__ float scale_of(unsigned most)
{
    return most >= kInf ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(most), Fp8<E5M2>::kMost);
}

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

__device__ __forceinline__ void put16(unsigned char *p, const unsigned (&q)[4], int n, bool vec)
{
    if (vec && n >= 16) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < n) p[e] = (unsigned char)(q[e / 4] >> 8 * (e & 3));
    }
}

// A block takes a tile of 128 x 128: eight threads a row, 16 columns each, four rows a thread.  Maxima along a row stay in the eight threads,
// those along a column go through shared memory.
template <typename T, bool E5M2, int MODE, bool VEC> __global__ void __launch_bounds__(256) quantize_fp8_kernel(const QuantizeFp8Args a)
{
    __shared__ unsigned part[8][kB];
    __shared__ float2 column[kB]; // scale and its inverse
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const long tr = blockIdx.x / a.tiles_c;
    const int tc = blockIdx.x - (unsigned)tr * a.tiles_c;
    const int c0 = tc * kB + (t & 7) * 16, n = min(16, a.cols - c0);
    const long r0 = tr * kB + (t >> 3);
    float v[4][16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long r = r0 + 32 * i;
        const T *p = reinterpret_cast<const T *>(a.values) + r * a.stride + c0;
        if (VEC && r < a.rows && n == 16) {
            load16v(p, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[i][e] = r < a.rows && e < n ? number(p[e]) : 0.f;
        }
    }
    const bool code_vec = a.code_stride % 16 == 0 && (uintptr_t)a.codes % 16 == 0, down_vec = a.down_stride % 16 == 0 && (uintptr_t)a.down % 16 == 0;
    if (MODE == kRows || MODE == kBoth) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long r = r0 + 32 * i;
            unsigned m = 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) m = max(m, magnitude(v[i][e]));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
            const float s = scale_of<E5M2>(m), inv = inverse_of(s);
            if (r >= a.rows || n <= 0) continue;
            if ((t & 7) == 0) a.scales[r * a.scale_stride + tc] = s;
            unsigned q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = codes4<E5M2>(v[i] + 4 * e, s, s, s, s, inv, inv, inv, inv);
            put16(a.codes + r * a.code_stride + c0, q, n, code_vec);
        }
    }
    if constexpr (MODE == kSquare) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = max(m, magnitude(v[i][e]));
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) part[0][warp] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) m = max(m, part[0][w]);
        const float s = scale_of<E5M2>(m), inv = inverse_of(s);
        if (t == 0) a.scales[tr * a.scale_stride + tc] = s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long r = r0 + 32 * i;
            if (r >= a.rows || n <= 0) continue;
            unsigned q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = codes4<E5M2>(v[i] + 4 * e, s, s, s, s, inv, inv, inv, inv);
            put16(a.codes + r * a.code_stride + c0, q, n, code_vec);
        }
    }
    if constexpr (MODE == kColumns || MODE == kBoth) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            unsigned m = max(max(magnitude(v[0][e]), magnitude(v[1][e])), max(magnitude(v[2][e]), magnitude(v[3][e])));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if (lane < 8) part[warp][lane * 16 + e] = m;
        }
        __syncthreads();
        if (t < kB) {
            unsigned m = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) m = max(m, part[w][t]);
            const float s = scale_of<E5M2>(m);
            column[t] = make_float2(s, inverse_of(s));
            if (tc * kB + t < a.cols) a.down_scales[tr * a.down_scale_stride + tc * kB + t] = s;
        }
        __syncthreads();
        unsigned q[4][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 *s = column + (t & 7) * 16 + 4 * e;
            const float2 s0 = s[0], s1 = s[1], s2 = s[2], s3 = s[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i][e] = codes4<E5M2>(v[i] + 4 * e, s0.x, s1.x, s2.x, s3.x, s0.y, s1.y, s2.y, s3.y);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long r = r0 + 32 * i;
            if (r < a.rows && n > 0) put16(a.down + r * a.down_stride + c0, q[i], n, down_vec);
        }
    }
}

struct DequantizeFp8Args {
    const unsigned char *codes;
    long code_stride, rows;
    int cols, groups; // groups of 16 columns in a row
    const float *scales;
    long scale_stride;
    int row_shift, col_shift; // 7: a block spans 128 rows, 128 columns; 0: one
    void *out;
    long out_stride;
};

// a thread takes 16 codes of a row
template <typename T, bool E5M2, bool VEC> __global__ void __launch_bounds__(256) dequantize_fp8_kernel(const DequantizeFp8Args a)
{
    const long total = a.rows * a.groups, step = (long)gridDim.x * 256;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const long r = i / a.groups;
        const int c = (int)(i - r * a.groups) * 16, n = min(16, a.cols - c);
        const unsigned char *p = a.codes + r * a.code_stride + c;
        const float *s = a.scales + (r >> a.row_shift) * a.scale_stride;
        T *to = reinterpret_cast<T *>(a.out) + r * a.out_stride + c;
        unsigned w[4] = {0, 0, 0, 0};
        if (VEC && n == 16) {
            const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e < n) w[e / 4] |= (unsigned)p[e] << 8 * (e & 3);
        }
        float v[16];
        const float one = a.col_shift ? __ldg(s + (c >> 7)) : 0.f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float2 f = from_codes2<E5M2>(w[e / 4] >> 8 * (e & 3));
            v[e] = f.x * (a.col_shift ? one : e < n ? __ldg(s + c + e) : 0.f);
            v[e + 1] = f.y * (a.col_shift ? one : e + 1 < n ? __ldg(s + c + e + 1) : 0.f);
        }
        if (VEC && n == 16) {
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4 *>(to + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; e += 8)
                    *reinterpret_cast<uint4 *>(to + e) = make_uint4(pack2((T *)nullptr, v[e], v[e + 1]), pack2((T *)nullptr, v[e + 2], v[e + 3]),
                                                                    pack2((T *)nullptr, v[e + 4], v[e + 5]), pack2((T *)nullptr, v[e + 6], v[e + 7]));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e < n) put(to + e, v[e]);
        }
    }
}

template <typename T, bool E5M2, int MODE> int launch_quantize(const QuantizeFp8Args &a, cudaStream_t stream)
{
    const long tiles = ((a.rows + kB - 1) / kB) * a.tiles_c;
    const bool vec = (uintptr_t)a.values % 16 == 0 && (a.rows == 1 || a.stride * (long)sizeof(T) % 16 == 0);
    if (vec) quantize_fp8_kernel<T, E5M2, MODE, true><<<(unsigned)tiles, 256, 0, stream>>>(a);
    else quantize_fp8_kernel<T, E5M2, MODE, false><<<(unsigned)tiles, 256, 0, stream>>>(a);
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
template <typename T, bool E5M2> int launch_dequantize(const Context *ctx, const DequantizeFp8Args &a, cudaStream_t stream)
{
    const long blocks = (a.rows * a.groups + 255) / 256, most = (long)ctx->sm_count * 32;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    const bool vec = (uintptr_t)a.codes % 16 == 0 && (uintptr_t)a.out % 16 == 0 && (a.rows == 1 || (a.code_stride % 16 == 0 && a.out_stride * (long)sizeof(T) % 16 == 0));
    if (vec) dequantize_fp8_kernel<T, E5M2, true><<<grid, 256, 0, stream>>>(a);
    else dequantize_fp8_kernel<T, E5M2, false><<<grid, 256, 0, stream>>>(a);
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

int dequantize_fp8(const Context *ctx, const unsigned char *codes, int code_type, long code_stride, const float *scales, long scale_stride, int blocks,
                   long rows, int cols, void *out, int dtype, long out_stride, cudaStream_t stream)
{
    DequantizeFp8Args a;
    a.codes = codes;
    a.code_stride = code_stride;
    a.rows = rows;
    a.cols = cols;
    a.groups = (cols + 15) / 16;
    a.scales = scales;
    a.scale_stride = scale_stride;
    a.row_shift = blocks == kRows ? 0 : 7;
    a.col_shift = blocks == kColumns ? 0 : 7;
    a.out = out;
    a.out_stride = out_stride;
    count_launch("fp8_dequantize", stream, (double)rows * cols * (1 + (dtype == 1 ? 4 : 2)));
    const bool e5m2 = code_type == 6;
    switch (dtype) {
    case 1: return e5m2 ? launch_dequantize<float, true>(ctx, a, stream) : launch_dequantize<float, false>(ctx, a, stream);
    case 3: return e5m2 ? launch_dequantize<__nv_bfloat16, true>(ctx, a, stream) : launch_dequantize<__nv_bfloat16, false>(ctx, a, stream);
    default: return e5m2 ? launch_dequantize<__half, true>(ctx, a, stream) : launch_dequantize<__half, false>(ctx, a, stream);
    }
}

} // namespace lb
