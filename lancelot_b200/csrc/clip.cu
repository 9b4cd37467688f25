// The norms of clients' updates, each over many tensors, and the updates scaled down to a largest norm:
//
//   norm = sqrt(sum of v^2 over all tensors of a client)     f = min(1, most / norm), rounded to 32 bits; NaN where the norm is not finite     out = v * f
//
// A bound on the norm is the plain defence against an update that outweighs the others, next to the selection by distances
// (lancelot-main-GPU/utils/byzantine_fl.py:162-171,527-536); the reference has none.
//
// Squares of 32-bit floats are exact in 64 bits, and so are summed there: no sum passes the range, and small entries are not lost behind
// large ones.  The tensors are cut into pieces; a piece's sum goes to its own place, and every block that needs a client's norm adds
// its pieces up in the same order, so that results do not depend on which block was first.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "product.cuh"

namespace lb {

namespace {

constexpr int kThreads = 256;
constexpr int kMostTensors = 800; // of one launch: they travel as its argument

struct Part {
    const void *in;
    void *out; // NULL: nothing is written
    long n;
    int first;      // of the call's pieces
    int begin, end; // the client's pieces
    int client : 24, in_type : 4, out_type : 4;
};
template <int MOST> struct ClipArgs {
    Part tensor[MOST];
    int n_tensors, n_pieces; // of this launch
    int piece;               // elements of a piece, a multiple of 64
    bool sums, writes;       // whether this launch forms the pieces' sums, and whether it goes on to norms and results
    double most;
    double *partial, *norms;
};

template <typename T> struct Pack; // values in 16 bytes
template <> struct Pack<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void open(const uint4 &w, float *v)
    {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ float one(float v) { return v; }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void open(const uint4 &w, float *v)
    {
        const unsigned x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(x[i] << 16), v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct Pack<__half> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void open(const uint4 &w, float *v)
    {
        const unsigned x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
};

// the sum of a block's values, in every thread; the order is fixed
__device__ __forceinline__ double block_sum(double v, double *shared)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += shared[i];
    return v;
}

// the tensor that holds a piece
template <int MOST> __device__ __forceinline__ int tensor_of(const ClipArgs<MOST> &a, int piece)
{
    int lo = 0, hi = a.n_tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.tensor[mid].first <= piece) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T> __device__ __forceinline__ double squares(const T *p, int n)
{
    constexpr int N = Pack<T>::kN;
    double sum = 0.0;
    int done = 0;
    if ((uintptr_t)p % 16 == 0) {
        done = n / N * N;
#pragma unroll 4
        for (int i = threadIdx.x * N; i < done; i += kThreads * N) {
            float v[N];
            Pack<T>::open(__ldg(reinterpret_cast<const uint4 *>(p + i)), v);
#pragma unroll
            for (int e = 0; e < N; ++e) sum = fma((double)v[e], (double)v[e], sum);
        }
    }
#pragma unroll 4
    for (int i = done + threadIdx.x; i < n; i += kThreads) {
        const double v = Pack<T>::one(p[i]);
        sum = fma(v, v, sum);
    }
    return sum;
}

template <typename T, typename O> __device__ __forceinline__ void scaled(const T *p, O *out, int n, float f)
{
    constexpr int N = Pack<T>::kN;
    int done = 0;
    if ((uintptr_t)p % 16 == 0 && (uintptr_t)out % 16 == 0) {
        done = n / N * N;
#pragma unroll 4
        for (int i = threadIdx.x * N; i < done; i += kThreads * N) {
            float v[N];
            Pack<T>::open(__ldcs(reinterpret_cast<const uint4 *>(p + i)), v);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] *= f;
            if constexpr (sizeof(O) == 4) {
#pragma unroll
                for (int e = 0; e < N; e += 4) __stcs(reinterpret_cast<float4 *>(out + i + e), make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]));
            } else if constexpr (N == 8) {
                __stcs(reinterpret_cast<uint4 *>(out + i), make_uint4(pack2(out, v[0], v[1]), pack2(out, v[2], v[3]), pack2(out, v[4], v[5]), pack2(out, v[6], v[7])));
            } else {
                __stcs(reinterpret_cast<uint2 *>(out + i), make_uint2(pack2(out, v[0], v[1]), pack2(out, v[2], v[3])));
            }
        }
    }
#pragma unroll 8
    for (int i = done + threadIdx.x; i < n; i += kThreads) put(out + i, Pack<T>::one(p[i]) * f);
}

__device__ __forceinline__ double squares(const void *in, int type, long at, int n)
{
    return type == 1 ? squares(reinterpret_cast<const float *>(in) + at, n)
         : type == 3 ? squares(reinterpret_cast<const __nv_bfloat16 *>(in) + at, n)
                     : squares(reinterpret_cast<const __half *>(in) + at, n);
}
template <typename T> __device__ __forceinline__ void scaled(const T *in, void *out, int type, long at, int n, float f)
{
    if (type == 1) scaled(in, reinterpret_cast<float *>(out) + at, n, f);
    else if (type == 3) scaled(in, reinterpret_cast<__nv_bfloat16 *>(out) + at, n, f);
    else scaled(in, reinterpret_cast<__half *>(out) + at, n, f);
}

template <int MOST> __global__ void __launch_bounds__(kThreads, 4) clip_kernel(const __grid_constant__ ClipArgs<MOST> a)
{
    __shared__ double shared[kThreads / 32];
    const int piece0 = a.tensor[0].first;
    if (a.sums)
        for (int i = piece0 + blockIdx.x; i < piece0 + a.n_pieces; i += gridDim.x) {
            const Part &t = a.tensor[tensor_of(a, i)];
            const long at = (long)(i - t.first) * a.piece;
            const double sum = block_sum(squares(t.in, t.in_type, at, (int)min((long)a.piece, t.n - at)), shared);
            if (threadIdx.x == 0) a.partial[i] = sum;
        }
    if (!a.writes) return;
    if (a.sums) cooperative_groups::this_grid().sync();
    int client = -1;
    float f = 1.0f;
    for (int i = piece0 + blockIdx.x; i < piece0 + a.n_pieces; i += gridDim.x) {
        const Part &t = a.tensor[tensor_of(a, i)];
        if (t.client != client) {
            client = t.client;
            double sum = 0.0;
            for (int j = t.begin + (int)threadIdx.x; j < t.end; j += kThreads) sum += __ldcg(a.partial + j);
            const double norm = sqrt(block_sum(sum, shared));
            f = !isfinite(norm) ? __int_as_float(0x7fc00000) : norm > a.most ? (float)(a.most / norm) : 1.0f;
            if (i == t.begin && threadIdx.x == 0) a.norms[client] = norm;
        }
        if (!t.out || (f == 1.0f && t.out == t.in)) continue;
        const long at = (long)(i - t.first) * a.piece;
        const int n = (int)min((long)a.piece, t.n - at);
        if (t.in_type == 1) scaled(reinterpret_cast<const float *>(t.in) + at, t.out, t.out_type, at, n, f);
        else if (t.in_type == 3) scaled(reinterpret_cast<const __nv_bfloat16 *>(t.in) + at, t.out, t.out_type, at, n, f);
        else scaled(reinterpret_cast<const __half *>(t.in) + at, t.out, t.out_type, at, n, f);
    }
}

template <int MOST> int launch_clip(const Context *ctx, const ClipPart *parts, int n_tensors, int n_pieces, int piece, bool sums, bool writes, double most,
                                    double *partial, double *norms, cudaStream_t stream)
{
    static std::atomic<int> known{0};
    int per_sm = known;
    if (!per_sm) {
        LB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, clip_kernel<MOST>, kThreads, 0));
        known = per_sm;
    }
    ClipArgs<MOST> a;
    for (int i = 0; i < n_tensors; ++i) {
        const ClipPart &p = parts[i];
        Part &t = a.tensor[i];
        t.in = p.in;
        t.out = p.out;
        t.n = p.n;
        t.first = p.first;
        t.begin = p.begin;
        t.end = p.end;
        t.client = p.client;
        t.in_type = p.in_type;
        t.out_type = p.out_type;
    }
    a.n_tensors = n_tensors;
    a.n_pieces = n_pieces;
    a.piece = piece;
    a.sums = sums;
    a.writes = writes;
    a.most = most;
    a.partial = partial;
    a.norms = norms;
    const int blocks = per_sm * ctx->sm_count;
    void *args[] = {&a};
    LB_CUDA(cudaLaunchCooperativeKernel(reinterpret_cast<const void *>(clip_kernel<MOST>), dim3((unsigned)(n_pieces < blocks ? n_pieces : blocks)), dim3(kThreads), args, 0,
                                        stream));
    return LB_OK;
}

} // namespace

int clip_piece(const Context *ctx, double elements)
{
    const double even = elements / (8.0 * ctx->sm_count);
    return even <= 1024 ? 1024 : even >= 32768 ? 32768 : ((int)even + 63) / 64 * 64;
}

int clip_updates(const Context *ctx, const ClipPart *parts, int n_parts, int piece, double most, double *partial, double *norms, cudaStream_t stream)
{
    double bytes = 0.0;
    for (int i = 0; i < n_parts; ++i) bytes += (double)parts[i].n * ((parts[i].in_type == 1 ? 4 : 2) + (!parts[i].out ? 0 : parts[i].out_type == 1 ? 4 : 2));
    const bool one = n_parts <= kMostTensors;
    for (int pass = one ? 1 : 0; pass < 2; ++pass) // more tensors than one launch holds: all sums first
        for (int i = 0; i < n_parts; i += kMostTensors) {
            const int n = n_parts - i < kMostTensors ? n_parts - i : kMostTensors;
            const ClipPart &last = parts[i + n - 1];
            const int pieces = last.first + (last.n > piece ? (int)((last.n + piece - 1) / piece) : 1) - parts[i].first;
            count_launch("clip_updates", stream, i ? 0.0 : bytes);
            const auto launch = n <= 16 ? launch_clip<16> : n <= 96 ? launch_clip<96> : launch_clip<kMostTensors>;
            const int rc = launch(ctx, parts + i, n, pieces, piece, one || pass == 0, pass == 1, most, partial, norms, stream);
            if (rc) return rc;
        }
    return LB_OK;
}

} // namespace lb
