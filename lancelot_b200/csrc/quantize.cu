// The 8-bit cache of client updates: rows of values are written as codes with a scale per group of columns and read back.
//
//   t = value + residual (32 bits; 0 behind a row's length)    s = max|t| / 127 over the group, rounded to 32 bits
//   q = the integer nearest to t / s, ties to even             what the rounding lost: t - q s
//
// The reference has no 8-bit form of an update: its driver holds every client's values in the clear as lists of doubles
// (lancelot-main-GPU/utils/byzantine_fl.py:478-490).
//
// The nearest integer is found without a division.  q0 = t * (1 / s), rounded, is off by at most one, and only next to a border
// between two codes; r = fma(-q0, s, t) is exact there (both terms are multiples of the smaller of their units in the last
// place, and |r| is about s / 2, so it has at most 24 bits), and comparing 2 |r| with s settles the border, ties included.
// The same r is what the rounding lost, exactly: error feedback adds no error of its own.
//
// All kernels stream, (value bytes + 1 + 8 with a residual) per value.  Bound by HBM with 32-bit values and residuals: 20 rows of 11 M, one
// B200 that copies at 6.5 TB/s: groups of 128 in 496 us (5.9 TB/s), one scale for 32768 columns in 479 us (6.1), for 131072 columns in
// 856 us, where every value is read twice; read back in 179 us (6.3 TB/s).  With fewer bytes a value the instructions bound
// it: 32-bit values without residuals 271 us (one scale for 32768 columns), 338 us (groups of 128), 16-bit ones 266 and 341 us (2.5 and 2.0
// TB/s, with instructions issued in 65 and 81 % of the cycles).  Moves of 16 bytes are what it takes, for rows off their alignment too:
// these are taken in the values' aligned pieces and the codes are shifted, not the values.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "context.h"
#include "tcgen05.cuh"

namespace lb {

namespace {

constexpr unsigned kInfBits = 0x7f800000u;

// Four consecutive values on their piece's boundary, as 32-bit floats
__device__ __forceinline__ float4 load4(const float *p) { return __ldcs(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p)
{
    const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(p));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ float4 load4(const __half *p)
{
    const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ void store4(float *p, float4 v) { __stcs(reinterpret_cast<float4 *>(p), v); }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v)
{
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    __stcs(reinterpret_cast<uint2 *>(p), make_uint2(*reinterpret_cast<unsigned *>(&a), *reinterpret_cast<unsigned *>(&b)));
}
__device__ __forceinline__ void store4(__half *p, float4 v)
{
    __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    __stcs(reinterpret_cast<uint2 *>(p), make_uint2(*reinterpret_cast<unsigned *>(&a), *reinterpret_cast<unsigned *>(&b)));
}

// Four values at positions at .. at + 3 of a run, of which only [lo, hi) exist or are wanted
template <bool VEC, typename T> __device__ __forceinline__ float4 load_piece(const T *p, int at, int lo, int hi)
{
    if (VEC && at >= lo && at + 4 <= hi) return load4(p + at);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= lo && at < hi) v.x = (float)p[at];
    if (at + 1 >= lo && at + 1 < hi) v.y = (float)p[at + 1];
    if (at + 2 >= lo && at + 2 < hi) v.z = (float)p[at + 2];
    if (at + 3 >= lo && at + 3 < hi) v.w = (float)p[at + 3];
    return v;
}
__device__ __forceinline__ void set(float *p, float v) { *p = v; }
__device__ __forceinline__ void set(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void set(__half *p, float v) { *p = __float2half_rn(v); }
template <bool VEC, typename T> __device__ __forceinline__ void store_piece(T *p, int at, const float4 &v, int lo, int hi)
{
    if (VEC && at >= lo && at + 4 <= hi) {
        store4(p + at, v);
        return;
    }
    if (at >= lo && at < hi) set(p + at, v.x);
    if (at + 1 >= lo && at + 1 < hi) set(p + at + 1, v.y);
    if (at + 2 >= lo && at + 2 < hi) set(p + at + 2, v.z);
    if (at + 3 >= lo && at + 3 < hi) set(p + at + 3, v.w);
}
template <typename T> __device__ __forceinline__ int offset_of(const T *p) { return (int)((uintptr_t)p / sizeof(T)) & 3; }
// the first n elements, or those from n on; the others 0
__device__ __forceinline__ float4 first_of(const float4 &v, int n) { return make_float4(n > 0 ? v.x : 0.f, n > 1 ? v.y : 0.f, n > 2 ? v.z : 0.f, n > 3 ? v.w : 0.f); }
__device__ __forceinline__ float4 from_of(const float4 &v, int n) { return make_float4(n > 0 ? 0.f : v.x, n > 1 ? 0.f : v.y, n > 2 ? 0.f : v.z, n > 3 ? 0.f : v.w); }

// The scale of a group from the bits of its largest magnitude.  The bit patterns of magnitudes are ordered like the magnitudes
// with infinities and NaN above all numbers, so an integer maximum carries them along: such a group gets NaN
__device__ __forceinline__ float scale_of(unsigned most)
{
    return most >= kInfBits ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(most), 127.0f);
}

// Codes of four values in a group of scale s (inv = 1 / s), packed; v <- what the rounding lost.  Adding 1.5 * 2^23 rounds a
// product to an integer, ties to even, and leaves its last eight bits as the code.
constexpr float kMagic = 12582912.0f;
__device__ __forceinline__ void settle(float &y, float &t, float r, float s) // the neighbour on the side of r, past the border, or on it from an odd code
{
    const float twice = fabsf(r + r);
    if (twice > s || (twice == s && (__float_as_int(y) & 1))) {
        y += copysignf(1.0f, r);
        r = fmaf(-(y - kMagic), s, t);
    }
    t = r;
}
__device__ __forceinline__ unsigned codes4_normal(float4 &v, const float4 &s, const float4 &inv)
{
    float a = fmaf(v.x, inv.x, kMagic), b = fmaf(v.y, inv.y, kMagic), c = fmaf(v.z, inv.z, kMagic), d = fmaf(v.w, inv.w, kMagic);
    const float p = fmaf(kMagic - a, s.x, v.x), q = fmaf(kMagic - b, s.y, v.y), r = fmaf(kMagic - c, s.z, v.z), u = fmaf(kMagic - d, s.w, v.w);
    if (fabsf(p + p) >= s.x || fabsf(q + q) >= s.y || fabsf(r + r) >= s.z || fabsf(u + u) >= s.w) { // seldom: one of the four lies next to a border
        settle(a, v.x, p, s.x);
        settle(b, v.y, q, s.y);
        settle(c, v.z, r, s.z);
        settle(d, v.w, u, s.w);
    } else {
        v = make_float4(p, q, r, u);
    }
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
// Groups whose scale is below the normal numbers: 1 / s overflows, and the rounding of s itself moves codes past 127.  A quotient of
// 64 bits decides a border between 32-bit numbers rightly
__device__ __noinline__ float2 code_of_tiny(float t, float s) // (code, what was lost)
{
    const double q = fmin(fmax(rint((double)t / (double)s), -127.0), 127.0);
    return make_float2((float)q, (float)((double)t - q * (double)s));
}
__device__ __forceinline__ unsigned codes4(float4 &v, float s)
{
    if (s >= 1.17549435e-38f) {
        const float inv = __frcp_rn(s);
        return codes4_normal(v, make_float4(s, s, s, s), make_float4(inv, inv, inv, inv));
    }
    if (!(s > 0.0f)) { // an empty group, or one that is not finite
        if (s != s) v = make_float4(0.f, 0.f, 0.f, 0.f);
        return 0;
    }
    const float2 x = code_of_tiny(v.x, s), y = code_of_tiny(v.y, s), z = code_of_tiny(v.z, s), w = code_of_tiny(v.w, s);
    v = make_float4(x.y, y.y, z.y, w.y);
    return ((unsigned)(int)x.x & 255) | ((unsigned)(int)y.x & 255) << 8 | ((unsigned)(int)z.x & 255) << 16 | (unsigned)(int)w.x << 24;
}
// the first `off` of the four belong to the group before, of scale `before`
__device__ __forceinline__ unsigned codes4_across(float4 &v, float before, float s, int off)
{
    if (before >= 1.17549435e-38f && s >= 1.17549435e-38f) {
        const float i = __frcp_rn(before), j = __frcp_rn(s);
        return codes4_normal(v, make_float4(off > 0 ? before : s, off > 1 ? before : s, off > 2 ? before : s, s),
                             make_float4(off > 0 ? i : j, off > 1 ? i : j, off > 2 ? i : j, j));
    }
    float4 head = first_of(v, off);
    v = from_of(v, off);
    const unsigned mask = (1u << 8 * off) - 1, q = codes4(head, before) & mask, r = codes4(v, s) & ~mask;
    v = make_float4(off > 0 ? head.x : v.x, off > 1 ? head.y : v.y, off > 2 ? head.z : v.z, v.w);
    return q | r;
}

// the largest magnitude, NaN if one is NaN
__device__ __forceinline__ float max_nan(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ unsigned most4(const float4 &v)
{
    return __float_as_uint(max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w)))) & 0x7fffffffu;
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
    int *status;
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

// A run of columns of one row, as its warps see it.  Rows seldom start on a 16-byte boundary (an update has an odd number of values as
// often as not), so the values move in aligned pieces of four that begin `off` columns early: piece i holds the columns 4 i - off to
// 4 i + 3 - off of the run.  A piece across the border of two groups is rounded with both scales, and the codes, which are aligned to
// the columns, are put together from two pieces.  VEC: values and residuals have the same offset; otherwise off is 0 and everything
// moves value by value.
template <typename T> struct Run {
    const T *values;
    const float *residual;
    float *lost;
    int off;
    int hi;    // columns [0, hi) exist
    bool full; // the whole run does, and the row goes on by a piece on either side
};
template <typename T, bool VEC> __device__ __forceinline__ Run<T> run_of(const QuantizeArgs &a, long row, long col, long limit, int length)
{
    Run<T> r;
    r.values = reinterpret_cast<const T *>(a.values) + row * a.value_stride + col;
    r.residual = a.residual ? a.residual + row * a.residual_stride + col : nullptr;
    r.lost = a.residual_out ? a.residual_out + row * a.residual_stride + col : nullptr;
    r.off = VEC ? offset_of(r.values) : 0;
    r.hi = (int)max(0l, min(limit - col, 1l << 30));
    r.full = VEC && r.hi >= length && (r.off == 0 || (col >= 4 && col + length + 4 <= a.n_cols));
    return r;
}
template <bool FULL, bool VEC, typename T> __device__ __forceinline__ float4 load_sum(const Run<T> &r, int at)
{
    float4 v = FULL ? load4(r.values + at) : load_piece<VEC>(r.values, at, 0, r.hi);
    if (r.residual) {
        const float4 w = FULL ? load4(r.residual + at) : load_piece<VEC>(r.residual, at, 0, r.hi);
        v.x += w.x;
        v.y += w.y;
        v.z += w.z;
        v.w += w.w;
    }
    return v;
}

// ---- groups of 32 to 512 columns: a warp takes 512 columns ------------------------------------------------------------
// Every load and store of a warp is one contiguous run (512 bytes of 32-bit values, 128 bytes of codes); a group's maximum never
// leaves the warp.
template <typename T, bool VEC, int LOG_G, bool FULL>
__device__ __forceinline__ void quantize_tile(const Run<T> &r, signed char *codes, float *scales, int in_page, int page)
{
    const int lane = threadIdx.x & 31, off = r.off, first = lane * 4 - off;
    float4 v[4], last = make_float4(0.f, 0.f, 0.f, 0.f); // of lane 0: the end of the run
    unsigned m[4], q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load_sum<FULL, VEC>(r, first + j * 128);
    if (off) {
        if (lane == 0) {
            last = first_of(load_sum<FULL, VEC>(r, 512 - off), off);
            v[0] = from_of(v[0], off);
        }
        unsigned head[5];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            head[j] = most4(first_of(v[j], off));
            m[j] = most4(from_of(v[j], off));
        }
        head[4] = most4(last);
#pragma unroll
        for (int j = 0; j < 4; ++j) { // the columns of a lane: the rest of its piece and the head of the next lane's
            const unsigned next = __shfl_down_sync(0xffffffffu, head[j], 1), wrap = __shfl_sync(0xffffffffu, head[j + 1], 0);
            m[j] = max(m[j], lane == 31 ? wrap : next);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = most4(v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
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
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s[j] = scale_of(m[j]);
        const int c = in_page + lane * 4 + j * 128;
        if (c < page && (c & ((1 << LOG_G) - 1)) == 0) scales[c >> LOG_G] = s[j];
    }
    if (off) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float before = __shfl_up_sync(0xffffffffu, s[j], 1);
            const float wrap = __shfl_sync(0xffffffffu, s[j > 0 ? j - 1 : 0], 31);
            if (lane == 0) before = wrap;
            q[j] = codes4_across(v[j], before, s[j], off);
        }
        const float end = __shfl_sync(0xffffffffu, s[3], 31);
        unsigned tail = 0;
        if (lane == 0) tail = codes4(last, end);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned next = __shfl_down_sync(0xffffffffu, q[j], 1), wrap = __shfl_sync(0xffffffffu, j < 3 ? q[j < 3 ? j + 1 : 3] : tail, 0);
            q[j] = __funnelshift_r(q[j], lane == 31 ? wrap : next, 8 * off);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = codes4(v[j], s[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = lane * 4 + j * 128;
        if (in_page + c < page) *reinterpret_cast<unsigned *>(codes + c) = q[j];
    }
    if (!r.lost) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (FULL && (j > 0 || off == 0 || lane > 0)) store4(r.lost + first + j * 128, v[j]);
        else store_piece<VEC>(r.lost, first + j * 128, v[j], 0, r.hi);
    }
    if (off && lane == 0) store_piece<false>(r.lost, 512 - off, last, 0, min(r.hi, 512));
}

template <typename T, bool VEC, int LOG_G>
__global__ void __launch_bounds__(256) quantize_warp_kernel(const QuantizeArgs a, const unsigned tiles, const unsigned total)
{
    const unsigned w = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (w >= total) return;
    const unsigned page_index = w / tiles, tile = w - page_index * tiles;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    long slot;
    if (!page_slot(a, page_index, slot)) return;
    const long limit = min(row_limit(a, row), (long)(page + 1) * a.page), col = (long)page * a.page + tile * 512;
    const Run<T> r = run_of<T, VEC>(a, row, col, limit, 512);
    signed char *codes = a.codes + slot * a.code_stride + tile * 512;
    float *scales = a.scales + slot * a.scale_stride;
    if (r.full) quantize_tile<T, VEC, LOG_G, true>(r, codes, scales, tile * 512, a.page);
    else quantize_tile<T, VEC, LOG_G, false>(r, codes, scales, tile * 512, a.page);
}

// ---- groups of up to 65536 columns: a block, or a cluster of blocks, holds the group in registers ---------------------
// A block of 256 threads holds up to 8192 columns.  One of 1024 threads for 32768 columns would be alone on its SM, and all of it would
// wait for its loads, then compute, then store; the blocks of a cluster do these at different times from those of others on the SM.  They
// send their maxima to one another, each to an mbarrier of its own, so that nobody waits for stores or for a barrier of the whole cluster.
//
// Bound by HBM, less what the wait for the slowest block costs: 20 x 11 M with one scale for 32768 columns takes 479 us with residuals (6.1
// of 6.5 TB/s), 271 us without (4.1 TB/s; four loads of 16 bytes a thread, or as many blocks as 64 registers allow, gave 287 and 271,
// and 497 and 520 with residuals; a barrier of the cluster instead of the messages 592 and 317); 100 x 1.6 M with groups of 4096, which
// one block holds, 345 us (6.3 TB/s).
template <int V> struct GroupShared {
    unsigned most[32 + 8]; // of the warps; of the cluster's blocks
    unsigned heads[V * 8 + 1]; // the first codes of every warp's pieces, in the order of their columns
    unsigned long long arrived; // the cluster's maxima
    int failed;
};
template <typename T, bool VEC, int V, bool FULL>
__device__ __forceinline__ void quantize_group(const Run<T> &r, signed char *codes, float *scale, int length, GroupShared<V> &shared, int peer, int peers, int *status)
{
    constexpr int kThreads = 256, kRun = kThreads * V * 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, off = r.off, first = threadIdx.x * 4 - off;
    float4 v[V], last = make_float4(0.f, 0.f, 0.f, 0.f); // of thread 0: the end of the run
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = load_sum<FULL, VEC>(r, first + j * kThreads * 4);
    if (off && threadIdx.x == 0) {
        last = first_of(load_sum<FULL, VEC>(r, kRun - off), off);
        v[0] = from_of(v[0], off);
    }
    unsigned m = most4(last);
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, most4(v[j]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) shared.most[warp] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? shared.most[lane] : 0);
    if (peers > 1) { // the other blocks' maxima, by way of their shared memory
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // all of them have begun
        const unsigned arrived = smem_u32(&shared.arrived);
        if (threadIdx.x < (unsigned)peers)
            asm volatile("{\n\t.reg .b32 to, bar;\n\tmapa.shared::cluster.u32 to, %0, %2;\n\tmapa.shared::cluster.u32 bar, %1, %2;\n\t"
                         "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [to], %3, [bar];\n\t}" ::"r"(smem_u32(shared.most + 32 + peer)),
                         "r"(arrived), "r"(threadIdx.x), "r"(m)
                         : "memory");
        if (!mbar_wait(arrived, 0, &shared.failed)) atomicOr(status, 2); // a block leaves when all maxima are there: none is sent to one that has left
        __syncwarp();
        m = __reduce_max_sync(0xffffffffu, lane < peers ? shared.most[32 + lane] : 0);
    }
    const float s = scale_of(m);
    if (peer == 0 && threadIdx.x == 0) *scale = s;
    unsigned q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = codes4(v[j], s);
    if (off) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (lane == 0) shared.heads[j * 8 + warp] = q[j];
        if (threadIdx.x == 0) shared.heads[V * 8] = codes4(last, s);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const unsigned next = __shfl_down_sync(0xffffffffu, q[j], 1);
            q[j] = __funnelshift_r(q[j], lane == 31 ? shared.heads[j * 8 + warp + 1] : next, 8 * off);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = threadIdx.x * 4 + j * kThreads * 4;
        if (c < length) *reinterpret_cast<unsigned *>(codes + c) = q[j];
    }
    if (!r.lost) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (FULL && (j > 0 || off == 0 || threadIdx.x > 0)) store4(r.lost + first + j * kThreads * 4, v[j]);
        else store_piece<VEC>(r.lost, first + j * kThreads * 4, v[j], 0, r.hi);
    }
    if (off && threadIdx.x == 0) store_piece<false>(r.lost, kRun - off, last, 0, min(r.hi, kRun));
}

template <typename T, bool VEC, int V> __global__ void __launch_bounds__(256, V == 8 ? 3 : 5) quantize_block_kernel(const QuantizeArgs a, const int peers)
{
    __shared__ GroupShared<V> shared;
    const unsigned group_index = blockIdx.x / peers, peer = blockIdx.x - group_index * peers;
    const unsigned page_index = group_index / (unsigned)a.groups, g = group_index - page_index * (unsigned)a.groups;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    long slot;
    if (!page_slot(a, page_index, slot)) return; // all blocks of a cluster alike
    if (peers > 1) {
        if (threadIdx.x == 0) {
            mbar_init(smem_u32(&shared.arrived), 1);
            mbar_expect(smem_u32(&shared.arrived), peers * 4);
            shared.failed = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }
    constexpr int kRun = 256 * V * 4;
    const int first = g * a.group + peer * kRun, end = min(a.page, (int)(g + 1) * a.group); // columns inside the page
    const long limit = min(row_limit(a, row), (long)page * a.page + end), col = (long)page * a.page + first;
    const Run<T> r = run_of<T, VEC>(a, row, col, limit, kRun);
    signed char *codes = a.codes + slot * a.code_stride + first;
    float *scale = a.scales + slot * a.scale_stride + g;
    if (r.full) quantize_group<T, VEC, V, true>(r, codes, scale, end - first, shared, (int)peer, peers, a.status);
    else quantize_group<T, VEC, V, false>(r, codes, scale, end - first, shared, (int)peer, peers, a.status);
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
    const long first = (long)g * a.group + (long)part * kPart, end = min((long)a.page, (long)(g + 1) * a.group);
    const long limit = min(row_limit(a, row), (long)page * a.page + end), col = (long)page * a.page + first;
    Run<T> r = run_of<T, VEC>(a, row, col, limit, kPart);
    const bool vec = VEC && r.off == 0; // other rows value by value: such groups are rare
    unsigned m = 0;
    if (WRITE) {
        for (unsigned p = threadIdx.x & 31; p < parts; p += 32) m = max(m, part_most[(size_t)group_index * parts + p]);
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const float s = scale_of(m);
    if (WRITE && part == 0 && threadIdx.x == 0) a.scales[slot * a.scale_stride + g] = s;
#pragma unroll 4
    for (int j = 0; j < kPart / 4096; ++j) {
        const int c = threadIdx.x * 4 + j * 4096;
        float4 v = vec ? load_sum<false, true>(r, c) : load_sum<false, false>(r, c);
        if (WRITE) {
            const unsigned q = codes4(v, s);
            if (first + c < end) *reinterpret_cast<unsigned *>(a.codes + slot * a.code_stride + first + c) = q;
            if (r.lost && vec) store_piece<true>(r.lost, c, v, 0, r.hi);
            else if (r.lost) store_piece<false>(r.lost, c, v, 0, r.hi);
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

constexpr int kBlock = 8192, kCluster = 8; // columns that a block holds; blocks of a cluster, at most

template <typename T, bool VEC, int V> int launch_block(const QuantizeArgs &a, long groups, int peers, cudaStream_t stream)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(groups * peers));
    config.blockDim = dim3(256);
    config.stream = stream;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim = {(unsigned)peers, 1, 1};
    config.attrs = &cluster;
    config.numAttrs = peers > 1 ? 1 : 0;
    LB_CUDA(cudaLaunchKernelEx(&config, quantize_block_kernel<T, VEC, V>, a, peers));
    return LB_OK;
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
    } else if (longest <= kBlock * kCluster) {
        const long groups = n_pages * a.groups;
        if (longest <= 1024) return launch_block<T, VEC, 1>(a, groups, 1, stream);
        if (longest <= 4096) return launch_block<T, VEC, 4>(a, groups, 1, stream);
        return launch_block<T, VEC, 8>(a, groups, (longest + kBlock - 1) / kBlock, stream);
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

// Four codes as floats: a byte below the exponent of 2^23 is 2^23 + the byte
__device__ __forceinline__ float4 floats_of(unsigned x)
{
    const unsigned u = x ^ 0x80808080u; // code + 128
    return make_float4(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - 8388736.0f, __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - 8388736.0f,
                       __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - 8388736.0f, __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - 8388736.0f);
}

// A warp takes 512 columns of a page: 20 x 11 M in 179 us (6.3 TB/s) as 32-bit floats, 132 us (5.1 TB/s) as bf16.  The results are
// written in aligned pieces of four (see Run), whose codes are put together from two words.  ONE: one scale in a page
template <typename T, bool ONE>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantizeArgs a, const unsigned tiles, const unsigned total)
{
    const unsigned w = blockIdx.x * 8u + (threadIdx.x >> 5);
    if (w >= total) return;
    const int lane = threadIdx.x & 31;
    const unsigned page_index = w / tiles, tile = w - page_index * tiles;
    const unsigned row = page_index / (unsigned)a.pages, page = page_index - row * (unsigned)a.pages;
    const long slot = a.slots ? (long)a.slots[page_index] : (long)page_index;
    const bool there = slot >= 0 && slot < a.n_slots; // a page that is not in the cache reads as zeros
    const long col = (long)page * a.page + tile * 512;
    T *out = reinterpret_cast<T *>(a.out) + (long)row * a.out_stride + col;
    const int off = offset_of(out), hi = (int)max(0l, min(min(a.n_cols - col, 512l), (long)a.page - tile * 512));
    const signed char *codes = a.codes + (there ? slot : 0) * a.code_stride + tile * 512 + lane * 4;
    const float *scales = a.scales + (there ? slot : 0) * a.scale_stride;
    const int end = there ? hi : 0; // columns whose codes are read, in words
    unsigned q[4];
    float s[4];
    if (ONE) s[0] = s[1] = s[2] = s[3] = end ? __ldg(scales) : 0.f;
    if (end == 512) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q[j] = __ldcs(reinterpret_cast<const unsigned *>(codes + j * 128));
            if (!ONE) s[j] = __ldg(scales + ((int)(tile * 512 + lane * 4 + j * 128) >> a.log_group));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool inside = lane * 4 + j * 128 < end;
            q[j] = 0;
            if (inside) q[j] = __ldcs(reinterpret_cast<const unsigned *>(codes + j * 128));
            if (!ONE) {
                s[j] = 0.f;
                if (inside) s[j] = __ldg(scales + ((int)(tile * 512 + lane * 4 + j * 128) >> a.log_group));
            }
        }
    }
    if (off == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 f = floats_of(q[j]);
            store_piece<true>(out, lane * 4 + j * 128, make_float4(s[j] * f.x, s[j] * f.y, s[j] * f.z, s[j] * f.w), 0, hi);
        }
        return;
    }
    // the words and scales of the lane before; lane 0's are of the run before, or of the j before
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned before = __shfl_up_sync(0xffffffffu, q[j], 1), wrap = __shfl_sync(0xffffffffu, q[j > 0 ? j - 1 : 0], 31);
        const float4 f = floats_of(__funnelshift_r(lane ? before : wrap, q[j], 32 - 8 * off));
        float b = s[j];
        if (!ONE) {
            const float up = __shfl_up_sync(0xffffffffu, s[j], 1), down = __shfl_sync(0xffffffffu, s[j > 0 ? j - 1 : 0], 31);
            b = lane ? up : down;
        }
        const float4 v = make_float4(b * f.x, (off > 1 ? b : s[j]) * f.y, (off > 2 ? b : s[j]) * f.z, s[j] * f.w);
        if (hi == 512 && (j > 0 || lane > 0)) store4(out + lane * 4 + j * 128 - off, v);
        else store_piece<true>(out, lane * 4 + j * 128 - off, v, 0, hi);
    }
    if (hi > 512 - off && lane == 31) { // the columns before the next run's first piece
        const float4 f = floats_of(q[3] >> (32 - 8 * off));
        store_piece<false>(out, 512 - off, make_float4(s[3] * f.x, s[3] * f.y, s[3] * f.z, 0.f), 0, hi);
    }
}

template <typename T> int phase_of(const void *p) { return (int)((uintptr_t)p / sizeof(T)) & 3; }

} // namespace

size_t quantize_workspace_bytes(long n_rows, long n_cols, int page, int group)
{
    const int longest = group == 0 || group > page ? page : group;
    if (longest <= kBlock * kCluster) return 0;
    const long pages = (n_cols + page - 1) / page, groups = (page + longest - 1) / longest;
    return sizeof(unsigned) * (size_t)(n_rows * pages * groups * ((longest + kPart - 1) / kPart));
}

int quantize_rows(const void *values, int dtype, long n_rows, long n_cols, long value_stride, const int *lengths, const float *residual,
                  float *residual_out, long residual_stride, const int *slots, long n_slots, int page, int group, signed char *codes,
                  long code_stride, float *scales, long scale_stride, void *workspace, int *status, cudaStream_t stream)
{
    QuantizeArgs a;
    a.status = status;
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
    // whether values and residuals lie at the same offset from an aligned piece in every row
    auto same = [&](int phase) {
        const bool strides = n_rows == 1 || (value_stride - residual_stride) % 4 == 0;
        return (!residual && !residual_out) || (strides && (!residual || phase_of<float>(residual) == phase) && (!residual_out || phase_of<float>(residual_out) == phase));
    };
    const double bytes = (double)n_rows * n_cols * ((dtype == 1 ? 4 : 2) + 1 + (residual ? 4 : 0) + (residual_out ? 4 : 0));
    switch (dtype) {
    case 1:
        return same(phase_of<float>(values)) ? quantize_typed<float, true>(a, n_rows, workspace, bytes, stream)
                                                            : quantize_typed<float, false>(a, n_rows, workspace, bytes, stream);
    case 3:
        return same(phase_of<__nv_bfloat16>(values)) ? quantize_typed<__nv_bfloat16, true>(a, n_rows, workspace, bytes, stream)
                                                                    : quantize_typed<__nv_bfloat16, false>(a, n_rows, workspace, bytes, stream);
    default:
        return same(phase_of<__half>(values)) ? quantize_typed<__half, true>(a, n_rows, workspace, bytes, stream)
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
    const bool one = a.log_group == 31;
    if (dtype == 1) (one ? dequantize_kernel<float, true> : dequantize_kernel<float, false>)<<<grid, 256, 0, stream>>>(a, tiles, total);
    else if (dtype == 3) (one ? dequantize_kernel<__nv_bfloat16, true> : dequantize_kernel<__nv_bfloat16, false>)<<<grid, 256, 0, stream>>>(a, tiles, total);
    else (one ? dequantize_kernel<__half, true> : dequantize_kernel<__half, false>)<<<grid, 256, 0, stream>>>(a, tiles, total);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

} // namespace lb
