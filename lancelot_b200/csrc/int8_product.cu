// Matrix product of 8-bit integers with a scale per row of either operand:
//   out[m][n] = (sum over k of a[m][k] b[n][k]) * a_scale[m] * b_scale[n]
// Sums are exact 32-bit integers; the two scales are applied in 32-bit floats and the result is rounded once to its type.
// The reference has no integer matrix product; updates of low rank are formed with it from their two factors before they are
// encrypted (the mean of products is not the product of means, so the factors themselves cannot be averaged).
//
// Two kernels.  With few rows on one side the other side is read once and that bounds the call: rows go from memory straight into
// the registers of the warp's matrix instruction.  Otherwise the tiles run on the tensor cores' own memory: operands by TMA
// into 128-byte swizzled shared memory, tcgen05.mma into TMEM, results out of TMEM while the next tile is being multiplied.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "tcgen05.cuh"

namespace lb {

namespace {

// ---- results ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float scaled(int sum, float sa, float sb) { return __int2float_rn(sum) * sa * sb; }

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

// ---- few rows on one side -------------------------------------------------------------------------------------------------
// A block forms 16 rows of the long side (the rows of A of m16n8k32) against up to 32 rows of the short side; its 16 warps split k
// and add up through shared memory (so many, because a round of loads is what a small call waits for: k = 4096 takes one).  As in the
// pair distances, the order of k inside a product is free, so lane (g, t) loads 16 consecutive bytes of a row and uses them as four
// k-slots on either side.  Bound by the latency of its loads: 1 x 4096 x 4096 in 4.5 us, 3.4 us where L2 still holds the long side
// (2.6 us at the copy rate; 7.6 us with 8 warps), 1 x 4096 x 4095, whose rows are taken off their alignment, in 6.7 us (18.5 us where they
// were copied to aligned ones first), 16 x 11008 x 4096 in 13.5 us (3.3 TB/s).
constexpr int kSkinnyWarps = 16;

struct SkinnyArgs {
    const signed char *w, *x; // long side [rows][k], short side [cols][k]
    long w_stride, x_stride;
    const float *w_scale, *x_scale;
    int rows, cols, k;
    void *out;
    long row_step, col_step; // of the result
};

template <typename T, int NB, bool ALIGNED> __global__ void __launch_bounds__(kSkinnyWarps * 32, 2) skinny_kernel(const SkinnyArgs a)
{
    __shared__ int part[kSkinnyWarps][16][NB * 8 + 1];
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
    const long r0 = (long)blockIdx.x * 16;
    const bool in0 = r0 + g < a.rows, in1 = r0 + g + 8 < a.rows;
    const signed char *w0 = a.w + (r0 + g) * a.w_stride, *w1 = w0 + 8 * a.w_stride;
    int acc[NB][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0;
#pragma unroll(ALIGNED ? 4 : 2)
    for (int k = warp * 64 + t * 16; k < a.k + t * 16; k += kSkinnyWarps * 64) { // the warp stays together: mma.sync wants all lanes
        const int left = a.k - k;
        const uint4 u = load16<ALIGNED>(w0 + k, in0 ? left : 0);
        const uint4 v = load16<ALIGNED>(w1 + k, in1 ? left : 0);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const uint4 x = load16<ALIGNED>(a.x + (j * 8 + g) * a.x_stride + k, j * 8 + g < a.cols ? left : 0);
            mma_s8(acc[j], u.x, v.x, u.y, v.y, x.x, x.y);
            mma_s8(acc[j], u.z, v.z, u.w, v.w, x.z, x.w);
        }
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[warp][g + (e >> 1) * 8][j * 8 + t * 2 + (e & 1)] = acc[j][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NB * 8; i += kSkinnyWarps * 32) {
        const int r = i & 15, c = i >> 4;
        if (r0 + r >= a.rows || c >= a.cols) continue;
        int sum = 0;
#pragma unroll
        for (int s = 0; s < kSkinnyWarps; ++s) sum += part[s][r][c];
        put(reinterpret_cast<T *>(a.out) + (r0 + r) * a.row_step + c * a.col_step, scaled(sum, a.w_scale[r0 + r], a.x_scale[c]));
    }
}

template <typename T, bool ALIGNED> int launch_skinny(const SkinnyArgs &a, cudaStream_t stream)
{
    const unsigned grid = (unsigned)((a.rows + 15) / 16);
    if (a.cols <= 8) skinny_kernel<T, 1, ALIGNED><<<grid, kSkinnyWarps * 32, 0, stream>>>(a);
    else if (a.cols <= 16) skinny_kernel<T, 2, ALIGNED><<<grid, kSkinnyWarps * 32, 0, stream>>>(a);
    else skinny_kernel<T, 4, ALIGNED><<<grid, kSkinnyWarps * 32, 0, stream>>>(a);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

// ---- tiles on tcgen05 -------------------------------------------------------------------------------------------------------
// One CTA per SM walks over tiles of 128 x BN.  Warp 0 brings 128-byte wide blocks of k by TMA into a ring of stages, warp 1
// issues the products (four of k = 32 a stage), warps 2 to 5 take a finished tile out of TMEM.  TMEM holds two tiles, so
// a tile leaves while the next one is being formed.  Bound by the tensor cores where k is long: 8192 x 8192 x 8192 in 372 us, 2.95 P
// operations a second (0.91 of twice the rate that bf16 products reach), in a burst; one such product after the other takes some 430 us (2.56 P)
// under the power cap.  Bound by the results where it is short: 4096 x 4096 x 16 in 18 us
// (67 MB).  All of warp 1 comes to the instruction and one lane is elected, instead of a branch for lane 0: the operands are then in
// uniform registers (64 x 64 x 131056: 230 us, 300 us before).
constexpr int kTileM = 128, kTileK = 128;

// SHORT: few blocks of k, so that the results are what takes time: eight warps instead of four take them out, and fewer stages leave
// shared memory for them to leave by TMA
template <int BN, bool SHORT> struct Tile {
    static constexpr int kOutWarps = SHORT ? 8 : 4, kThreads = 64 + kOutWarps * 32;
    static constexpr int kStageBytes = (kTileM + BN) * kTileK;
    static constexpr int kStages = SHORT ? 3 : BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kOutBytes = SHORT ? 2 * 4096 : 0; // of a warp: two boxes of 32 rows of 128 bytes
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kOutWarps * (kOutBytes + BN * 4) + 256;
    // D 32-bit signed, A and B 8-bit signed, both k-major
    static constexpr unsigned kDesc = 2u << 4 | 1u << 7 | 1u << 10 | (unsigned)(BN >> 3) << 17 | (unsigned)(kTileM >> 4) << 24;
};

struct ProductArgs {
    int m, n, k_blocks;
    int tiles_m, tiles_n, band; // tiles are walked in bands of `band` rows of tiles, so that a wave reads few distinct rows of a and b
    const float *a_scale, *b_scale;
    void *out;
    long out_stride;
    int align; // 32, 16: the result's rows start on such a boundary; 0: on none; 1: the results leave by TMA
    int *status;
};

__device__ __forceinline__ void tile_at(const ProductArgs &a, int t, int &tm, int &tn)
{
    const int per_band = a.band * a.tiles_n, b = t / per_band, in = t - b * per_band;
    const int rows = min(a.band, a.tiles_m - b * a.band);
    tn = in / rows;
    tm = b * a.band + (in - tn * rows);
}

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

__device__ __forceinline__ void tma_store(const CUtensorMap *map, int x, int y, unsigned src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <typename T, int BN, bool SHORT>
__global__ void __launch_bounds__(Tile<BN, SHORT>::kThreads, 1) product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                               const __grid_constant__ CUtensorMap map_out, const ProductArgs a)
{
    using C = Tile<BN, SHORT>;
    extern __shared__ unsigned char raw[];
    unsigned char *stages = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    unsigned char *boxes = stages + C::kStages * C::kStageBytes;                           // [warp][2][32][128]
    float *scales = reinterpret_cast<float *>(boxes + C::kOutWarps * C::kOutBytes);        // [warp][BN]
    unsigned char *tail = reinterpret_cast<unsigned char *>(scales + C::kOutWarps * BN);
    unsigned long long *bars = reinterpret_cast<unsigned long long *>(tail); // full[stages], empty[stages], done[2], freed[2], drained
    unsigned *tmem_at = reinterpret_cast<unsigned *>(bars + 2 * C::kStages + 5);
    volatile int *failed = reinterpret_cast<volatile int *>(tmem_at + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned full = smem_u32(bars), empty = full + 8 * C::kStages, done = empty + 8 * C::kStages, freed = done + 16, drained = freed + 16;
    const unsigned stage0 = smem_u32(stages);

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(done + 8 * i, 1);
            mbar_init(freed + 8 * i, C::kOutWarps * 32);
        }
        mbar_init(drained, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "n"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = *tmem_at;
    const int tiles = a.tiles_m * a.tiles_n;

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                int tm, tn;
                tile_at(a, t, tm, tn);
                for (int k = 0; k < a.k_blocks && ok; ++k, ++it) {
                    const int s = it % C::kStages;
                    if (it >= C::kStages) ok = mbar_wait(empty + 8 * s, (it / C::kStages - 1) & 1, failed);
                    if (!ok) break;
                    mbar_expect(full + 8 * s, C::kStageBytes);
                    tma_load(stage0 + s * C::kStageBytes, &map_a, k * kTileK, tm * kTileM, full + 8 * s);
                    tma_load(stage0 + s * C::kStageBytes + kTileM * kTileK, &map_b, k * kTileK, tn * BN, full + 8 * s);
                }
            }
            // nothing may be in flight into shared memory when the block ends; after a success the products have waited for it
            if (!ok) {
                for (int i = it > C::kStages ? it - C::kStages : 0; i < it; ++i)
                    for (int n = 0; n < 1 << 20; ++n)
                        if (mbar_try(full + 8 * (i % C::kStages), (i / C::kStages) & 1)) break;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const unsigned elected = elect_one();
        int it = 0, done_tiles = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++done_tiles) {
            const int buf = done_tiles & 1;
            if (done_tiles >= 2) ok = mbar_wait_warp(freed + 8 * buf, (done_tiles / 2 - 1) & 1, failed);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int k = 0; k < a.k_blocks; ++k, ++it) {
                const int s = it % C::kStages;
                ok = mbar_wait_warp(full + 8 * s, (it / C::kStages) & 1, failed);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned at = stage0 + s * C::kStageBytes;
                const unsigned long long da = operand_desc(at), db = operand_desc(at + kTileM * kTileK);
#pragma unroll
                for (int e = 0; e < kTileK / 32; ++e) mma_i8(elected, tmem + buf * BN, da + 2 * e, db + 2 * e, C::kDesc, k > 0 || e > 0);
                mma_commit(elected, empty + 8 * s);
            }
            if (ok) mma_commit(elected, done + 8 * buf);
        }
        if (!ok) { // products that are still under way end before their memory is given back
            mma_commit(elected, drained);
            for (int n = 0; n < 1 << 20; ++n)
                if (mbar_try(drained, 0)) break;
        }
    } else {
        // a warp sees the 32 lanes of TMEM of its quarter; the warps of a quarter take their runs of 32 columns by turns
        constexpr int kTurns = C::kOutWarps / 4, kCols = SHORT && sizeof(T) == 2 ? 64 : 32; // columns of a run: a box of 128 bytes
        const int quarter = warp & 3, turn = (warp - 2) / 4;
        float *sb = scales + (warp - 2) * BN;
        unsigned char *box = boxes + (warp - 2) * C::kOutBytes;
        int done_tiles = 0, sent = 0;
        bool ok = true;
        float next_a, next_b[BN / 32]; // the scales of the next tile, on their way while this one is taken out
        auto fetch = [&](int t) {
            int tm, tn;
            tile_at(a, min(t, tiles - 1), tm, tn);
            const int row = tm * kTileM + quarter * 32 + lane;
            next_a = row < a.m ? __ldg(a.a_scale + row) : 0.f;
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) next_b[c] = tn * BN + c * 32 + lane < a.n ? __ldg(a.b_scale + tn * BN + c * 32 + lane) : 0.f;
        };
        fetch(blockIdx.x);
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++done_tiles) {
            const int buf = done_tiles & 1;
            int tm, tn;
            tile_at(a, t, tm, tn);
            const int row = tm * kTileM + quarter * 32 + lane;
            const float sa = next_a;
            __syncwarp();
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) sb[c * 32 + lane] = next_b[c];
            __syncwarp();
            fetch(t + gridDim.x);
            ok = mbar_wait(done + 8 * buf, (done_tiles / 2) & 1, failed);
            if (!__all_sync(0xffffffffu, ok)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            T *out = reinterpret_cast<T *>(a.out) + (long)row * a.out_stride + tn * BN;
            // A quarter wholly behind the last row has nothing to send.  It must not walk the boxes either: one that is passed without a store
            // leaves the wait below one store short of the box that it is about to write
            const int columns = tm * kTileM + quarter * 32 < a.m ? min(BN, a.n - tn * BN) : 0;
#pragma unroll 1
            for (int c0 = turn * kCols; c0 < columns; c0 += kTurns * kCols) {
                const bool by_tma = SHORT && a.align == 1;
                unsigned char *to = box + (sent & 1) * 4096;
                if (by_tma) { // all stores but the last one have been read out of their boxes
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    __syncwarp();
                }
#pragma unroll
                for (int c = c0; c < c0 + kCols; c += 32) {
                    int v[32];
                    tmem_load32(tmem + buf * BN + c + ((unsigned)quarter << 21), v);
                    float f[32];
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 s4 = *reinterpret_cast<const float4 *>(sb + c + e);
                        f[e] = scaled(v[e], sa, s4.x);
                        f[e + 1] = scaled(v[e + 1], sa, s4.y);
                        f[e + 2] = scaled(v[e + 2], sa, s4.z);
                        f[e + 3] = scaled(v[e + 3], sa, s4.w);
                    }
                    if (by_tma) { // 16-byte pieces where the 128-byte swizzle wants them
                        if constexpr (sizeof(T) == 4) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                *reinterpret_cast<float4 *>(to + lane * 128 + ((e / 4 ^ (lane & 7)) << 4)) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; e += 8)
                                *reinterpret_cast<uint4 *>(to + lane * 128 + ((((c - c0) / 8 + e / 8) ^ (lane & 7)) << 4)) =
                                    make_uint4(pack2((T *)nullptr, f[e], f[e + 1]), pack2((T *)nullptr, f[e + 2], f[e + 3]), pack2((T *)nullptr, f[e + 4], f[e + 5]),
                                               pack2((T *)nullptr, f[e + 6], f[e + 7]));
                        }
                    } else if (SHORT && a.align == 0) { // rows off their alignment: a row of the run at a time
                        // (through the box, 32 rows of 32 floats with the columns turned by the row, so that neither side meets a bank twice)
                        float *turned = reinterpret_cast<float *>(box);
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 32; ++e) turned[lane * 32 + ((e + lane) & 31)] = f[e];
                        __syncwarp();
                        const int first = tm * kTileM + quarter * 32, rows = min(32, a.m - first), col = tn * BN + c + lane;
                        T *p = reinterpret_cast<T *>(a.out) + (long)first * a.out_stride + col;
                        if (col < a.n)
                            for (int i = 0; i < rows; ++i) put(p + i * a.out_stride, turned[i * 32 + ((lane + i) & 31)]);
                    } else if (row < a.m) {
                        put32(out + c, f, a.n - tn * BN - c, a.align);
                    }
                }
                if (by_tma) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tma_store(&map_out, tn * BN + c0, tm * kTileM + quarter * 32, smem_u32(to));
                    ++sent;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(freed + 8 * buf);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (threadIdx.x == 0 && *failed) atomicOr(a.status, 2);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * BN) : "memory");
}

template <typename T, int BN, bool SHORT>
int launch_tiles(const Context *ctx, const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mo, const ProductArgs &a, cudaStream_t stream)
{
    using C = Tile<BN, SHORT>;
    static std::atomic<bool> set[64]; // host threads that come here first at once all set the same attribute
    if (ctx->device >= 64 || !set[ctx->device]) {
        LB_CUDA(cudaFuncSetAttribute(product_kernel<T, BN, SHORT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (ctx->device < 64) set[ctx->device] = true;
    }
    const int tiles = a.tiles_m * a.tiles_n;
    product_kernel<T, BN, SHORT><<<tiles < ctx->sm_count ? tiles : ctx->sm_count, C::kThreads, C::kSmem, stream>>>(ma, mb, mo, a);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

constexpr int kShort = 8;   // blocks of k up to which the results are what takes time
constexpr int kSkinny = 32; // rows on the short side up to which the long side is streamed

struct ProductPlan {
    bool off_a, off_b;   // rows off a 16-byte boundary
    bool pack_a, pack_b;
    int pitch;      // of packed rows
    size_t a_bytes; // of packed a
    size_t bytes;
};
ProductPlan product_plan(int m, int n, int k, const void *a, long a_stride, const void *b, long b_stride)
{
    ProductPlan p;
    auto off = [&](const void *x, long stride, int rows) { return (uintptr_t)x % 16 != 0 || (rows > 1 && stride % 16 != 0) || k % 16 != 0 || k == 0; };
    p.off_a = off(a, a_stride, m);
    p.off_b = off(b, b_stride, n);
    const bool skinny = m <= kSkinny || n <= kSkinny;
    p.pack_a = p.off_a && !skinny;
    p.pack_b = p.off_b && !skinny;
    p.pitch = k ? (k + 15) / 16 * 16 : 16;
    p.a_bytes = p.pack_a ? ((size_t)m * p.pitch + 255) / 256 * 256 : 0;
    p.bytes = p.a_bytes + (p.pack_b ? (size_t)n * p.pitch : 0);
    return p;
}

template <typename T>
int product_typed(Context *ctx, int m, int n, int k, bool aligned, const signed char *a, long a_stride, const float *a_scale, const signed char *b, long b_stride,
                  const float *b_scale, void *out, long out_stride, cudaStream_t stream)
{
    const double bytes = (double)m * k + (double)n * k + (double)m * n * sizeof(T);
    if (m <= kSkinny || n <= kSkinny) {
        SkinnyArgs s;
        const bool turned = m > n; // the long side is the rows of a
        s.w = turned ? a : b;
        s.x = turned ? b : a;
        s.w_stride = turned ? a_stride : b_stride;
        s.x_stride = turned ? b_stride : a_stride;
        s.w_scale = turned ? a_scale : b_scale;
        s.x_scale = turned ? b_scale : a_scale;
        s.rows = turned ? m : n;
        s.cols = turned ? n : m;
        s.k = k;
        s.out = out;
        s.row_step = turned ? out_stride : 1;
        s.col_step = turned ? 1 : out_stride;
        count_launch("int8_skinny", stream, bytes);
        return aligned ? launch_skinny<T, true>(s, stream) : launch_skinny<T, false>(s, stream);
    }
    ProductArgs p;
    p.m = m;
    p.n = n;
    p.k_blocks = (k + kTileK - 1) / kTileK;
    p.tiles_m = (m + kTileM - 1) / kTileM;
    p.a_scale = a_scale;
    p.b_scale = b_scale;
    p.out = out;
    p.out_stride = out_stride;
    const uintptr_t at = (uintptr_t)out | (uintptr_t)(out_stride * (long)sizeof(T));
    p.align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 0;
    p.status = ctx->d_status;
    p.band = 8;
    // Up to kShort blocks of k, and where rows are off their alignment, the form that takes results out faster (4096 x 4096 x 1024 in bf16:
    // 19.0 us instead of 24.6; from k = 2048 on its three stages cost more: 8192 x 8192 x 4096 205 us instead of 188).
    const bool quick = p.k_blocks <= kShort || p.align == 0;
    // The tile whose waves over the SMs take least: a block of k costs what its (128 + bn) x 128 bytes take from L2 to the SM, some
    // 58 bytes a cycle (0.22, 0.29, 0.43 us), a tile about a microsecond and the time of its results beside that.
    int bn = 64;
    double least = 0.0;
    for (int b = 64; b <= 256; b *= 2) {
        const long tiles = (long)p.tiles_m * ((n + b - 1) / b), waves = (tiles + ctx->sm_count - 1) / ctx->sm_count;
        const double us = (double)waves * ((double)p.k_blocks * (128 + b) * 1.15e-3 + 0.7 + b * 6e-3);
        if (least == 0.0 || us < least) {
            least = us;
            bn = b;
        }
    }
    p.tiles_n = (n + bn - 1) / bn;
    CUtensorMap ma, mb, mo;
    int rc = encode_map(&ma, a, m, k, a_stride, kTileK, kTileM);
    if (rc) return rc;
    if ((rc = encode_map(&mb, b, n, k, b_stride, kTileK, bn))) return rc;
    mo = ma; // not used where results do not leave by TMA
    if (quick && p.align >= 16) {
        if ((long)n * (long)sizeof(T) % 16 != 0) { // a TMA store would write the rest of a row's last 16 bytes, which is not the result's
            p.align = 0;
        } else {
            if ((rc = encode_map(&mo, out, m, (long)n * (long)sizeof(T), out_stride * (long)sizeof(T), 128, 32, sizeof(T)))) return rc;
            p.align = 1;
        }
    }
    count_launch("int8_tiles", stream, bytes);
    if (quick && bn == 256) return launch_tiles<T, 256, true>(ctx, ma, mb, mo, p, stream);
    if (quick) return bn == 128 ? launch_tiles<T, 128, true>(ctx, ma, mb, mo, p, stream) : launch_tiles<T, 64, true>(ctx, ma, mb, mo, p, stream);
    if (bn == 256) return launch_tiles<T, 256, false>(ctx, ma, mb, mo, p, stream);
    if (bn == 128) return launch_tiles<T, 128, false>(ctx, ma, mb, mo, p, stream);
    return launch_tiles<T, 64, false>(ctx, ma, mb, mo, p, stream);
}

} // namespace

size_t int8_matmul_workspace_bytes(int m, int n, int k, const void *a, long a_stride, const void *b, long b_stride)
{
    return product_plan(m, n, k, a, a_stride, b, b_stride).bytes;
}

int int8_matmul(Context *ctx, int m, int n, int k, const signed char *a, long a_stride, const float *a_scale, const signed char *b, long b_stride,
                const float *b_scale, void *out, int dtype, long out_stride, void *workspace, cudaStream_t stream)
{
    const ProductPlan p = product_plan(m, n, k, a, a_stride, b, b_stride);
    signed char *ws = reinterpret_cast<signed char *>(workspace);
    if (p.pack_a || p.pack_b) {
        const Packed one = {a, a_stride, p.pack_a ? m : 0, ws}, two = {b, b_stride, p.pack_b ? n : 0, ws + p.a_bytes};
        int log_lanes = 0;
        while (log_lanes < 8 && 16 << log_lanes < p.pitch) ++log_lanes;
        const long blocks = (one.rows + two.rows + (256 >> log_lanes) - 1) >> (8 - log_lanes), most = (long)ctx->sm_count * 32;
        count_launch("int8_pack", stream, 2.0 * (one.rows + two.rows) * k);
        pack_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(one, two, k, p.pitch, log_lanes);
        LB_CUDA(cudaGetLastError());
        if (p.pack_a) a = one.dst, a_stride = p.pitch;
        if (p.pack_b) b = two.dst, b_stride = p.pitch;
    }
    const bool aligned = !p.off_a && !p.off_b;
    if (p.pack_a || p.pack_b) k = p.pitch; // k itself where only one side is packed: a ragged k packs both
    switch (dtype) {
    case 1: return product_typed<float>(ctx, m, n, k, aligned, a, a_stride, a_scale, b, b_stride, b_scale, out, out_stride, stream);
    case 3: return product_typed<__nv_bfloat16>(ctx, m, n, k, aligned, a, a_stride, a_scale, b, b_stride, b_scale, out, out_stride, stream);
    default: return product_typed<__half>(ctx, m, n, k, aligned, a, a_stride, a_scale, b, b_stride, b_scale, out, out_stride, stream);
    }
}

} // namespace lb
