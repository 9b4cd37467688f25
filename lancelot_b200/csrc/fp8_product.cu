// Matrix product of 8-bit floating point with a scale for each block of 128 of the summed axis:
//   out[m][n] = sum over blocks p of (sum over k in p of a[m][k] b[n][k]) * a_scale[m][p] * b_scale[n][p]
// A block's sum is formed by the tensor cores in 32-bit floats, scaled, and added to the result in 32-bit floats; the result is rounded once to
// its type.  With a scale for 128 rows of b the two scales are multiplied first, elsewhere the sum by a's scale and then by b's: so both the product of the
// scales and the sum times a's scale have to be normal numbers or 0.  Kernels that multiply twice where the product of the scales is none were right for more
// scales and slower for all: a look at the scales and a vote a block 485 -> 508 us for 8192 x 8192 x 8192, a second multiplication for all 605 us.  Either operand may lie with the summed axis across its rows: the gradients of a product y = x w^T read x, w and the
// gradient of y as they are.  The reference has no such product.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "fp8.cuh"
#include "product.cuh"
#include "tcgen05.cuh"

namespace lb {

namespace {

constexpr int kM = 128, kK = 128; // rows of a tile, the summed axis of a block

struct Scales {
    const float *at;
    long row, block; // from one row (or block of 128 rows) to the next; from one block of the summed axis to the next
    int shift;       // 7: a scale for 128 rows
};

// ---- few rows on one side -------------------------------------------------------------------------------------------------
// Where both operands lie with the summed axis along their rows and one has up to eight of them, the other's bytes bound the call: they go
// from memory straight into the registers of the warp's matrix instruction, as in the 8-bit integer product.  A block forms 16 rows of the long side
// (the rows of A of m16n8k32) against the short side; its 16 warps take runs of 128 of the summed axis by turns, two steps of 64, and add up
// through shared memory.  The order of the summed axis inside a product is free, so lane (g, t) loads 16 consecutive bytes of a row and uses them as four
// k-slots on either side.  1 x 4096 x 4096 takes 4.8 us, 1 x 11008 x 4096 10.1 us (4.5 TB/s); 16 x 4096 x 4096 takes 10.2 us so, and
// 8 us by tiles.
constexpr int kSkinnyWarps = 16, kSkinny = 8;

template <bool WIDE_A, bool WIDE_B> // e5m2
__device__ __forceinline__ void mma_fp8(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
#define LB_MMA(A, B)                                                                                                                                  \
    asm("mma.sync.aligned.m16n8k32.row.col.f32." A "." B ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                                 \
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                                                              \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if (WIDE_A && WIDE_B) LB_MMA("e5m2", "e5m2");
    else if (WIDE_A) LB_MMA("e5m2", "e4m3");
    else if (WIDE_B) LB_MMA("e4m3", "e5m2");
    else LB_MMA("e4m3", "e4m3");
#undef LB_MMA
}

struct SkinnyFp8Args {
    const signed char *w, *x; // long side [rows][k], short side [cols][k]
    long w_stride, x_stride;
    Scales ws, xs;
    int rows, cols, k;
    bool w_first; // the long side is a, whose scale comes first
    void *out;
    long row_step, col_step; // of the result
};

template <typename T, bool ALIGNED, bool WIDE_W, bool WIDE_X>
__global__ void __launch_bounds__(kSkinnyWarps * 32, 2) fp8_skinny_kernel(const SkinnyFp8Args a)
{
    __shared__ float part[kSkinnyWarps][16][kSkinny + 1];
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
    const long r0 = (long)blockIdx.x * 16;
    const bool in0 = r0 + g < a.rows, in1 = r0 + g + 8 < a.rows;
    const signed char *w0 = a.w + (r0 + g) * a.w_stride, *w1 = w0 + 8 * a.w_stride;
    const float *s0 = a.ws.at + ((min(r0 + g, (long)a.rows - 1)) >> a.ws.shift) * a.ws.row, *s1 = a.ws.at + ((min(r0 + g + 8, (long)a.rows - 1)) >> a.ws.shift) * a.ws.row;
    const signed char *x0 = a.x + g * a.x_stride;
    const float *x_s0 = a.xs.at + (long)(min(t * 2, a.cols - 1) >> a.xs.shift) * a.xs.row, *x_s1 = a.xs.at + (long)(min(t * 2 + 1, a.cols - 1) >> a.xs.shift) * a.xs.row;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll(ALIGNED ? 2 : 1)
    for (int k0 = warp * kK; k0 < a.k; k0 += kSkinnyWarps * kK) { // the warp stays together: mma.sync wants all lanes
        uint4 u[2], v[2], x[2];
        const int at = k0 + t * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u[h] = load16<ALIGNED>(w0 + at + h * 64, in0 ? a.k - at - h * 64 : 0);
            v[h] = load16<ALIGNED>(w1 + at + h * 64, in1 ? a.k - at - h * 64 : 0);
            x[h] = load16<ALIGNED>(x0 + at + h * 64, g < a.cols ? a.k - at - h * 64 : 0);
        }
        const long p = k0 / kK;
        const float sw0 = __ldg(s0 + p * a.ws.block), sw1 = __ldg(s1 + p * a.ws.block), sx0 = __ldg(x_s0 + p * a.xs.block), sx1 = __ldg(x_s1 + p * a.xs.block);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mma_fp8<WIDE_W, WIDE_X>(c, u[h].x, v[h].x, u[h].y, v[h].y, x[h].x, x[h].y);
            mma_fp8<WIDE_W, WIDE_X>(c, u[h].z, v[h].z, u[h].w, v[h].w, x[h].z, x[h].w);
        }
        acc[0] = fmaf(c[0] * (a.w_first ? sw0 : sx0), a.w_first ? sx0 : sw0, acc[0]);
        acc[1] = fmaf(c[1] * (a.w_first ? sw0 : sx1), a.w_first ? sx1 : sw0, acc[1]);
        acc[2] = fmaf(c[2] * (a.w_first ? sw1 : sx0), a.w_first ? sx0 : sw1, acc[2]);
        acc[3] = fmaf(c[3] * (a.w_first ? sw1 : sx1), a.w_first ? sx1 : sw1, acc[3]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][g + (e >> 1) * 8][t * 2 + (e & 1)] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * kSkinny; i += kSkinnyWarps * 32) {
        const int r = i & 15, c = i >> 4;
        if (r0 + r >= a.rows || c >= a.cols) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kSkinnyWarps; ++w) sum += part[w][r][c];
        put(reinterpret_cast<T *>(a.out) + (r0 + r) * a.row_step + c * a.col_step, sum);
    }
}

template <typename T, bool ALIGNED, bool WIDE_W, bool WIDE_X> int launch_skinny(const SkinnyFp8Args &a, cudaStream_t stream)
{
    const unsigned grid = (unsigned)((a.rows + 15) / 16);
    fp8_skinny_kernel<T, ALIGNED, WIDE_W, WIDE_X><<<grid, kSkinnyWarps * 32, 0, stream>>>(a);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}
template <typename T, bool ALIGNED> int launch_skinny(const SkinnyFp8Args &a, bool wide_w, bool wide_x, cudaStream_t stream)
{
    if (wide_w) return wide_x ? launch_skinny<T, ALIGNED, true, true>(a, stream) : launch_skinny<T, ALIGNED, true, false>(a, stream);
    return wide_x ? launch_skinny<T, ALIGNED, false, true>(a, stream) : launch_skinny<T, ALIGNED, false, false>(a, stream);
}

// ---- tiles on tcgen05 -------------------------------------------------------------------------------------------------------
template <int BN, bool OFF> struct TileFp8 {
    static constexpr int kOutWarps = 8, kThreads = 128 + kOutWarps * 32;
    static constexpr int kCols = BN / 2; // columns of a thread: the warps of a quarter of TMEM's lanes take a half each
    static constexpr int kStageBytes = (kM + BN) * kK;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kBufs = BN == 256 ? 2 : 4; // block sums in TMEM
    static constexpr int kPitch = BN + 4;           // of a tile's results in shared memory, in floats
    static constexpr int kScaleStages = 8;          // blocks of the summed axis whose scales are on their way
    static constexpr int kRun = kCols / 4 + 4;      // scales of every fourth pair of columns, and a gap that keeps the four runs in different banks
    static constexpr int kScaleFloats = kM + 8 * kRun; // of a stage: of the rows; of the columns of each half
    static constexpr int kBars = 2 * kStages + 2 * kBufs + 2 * kScaleStages + 1;
    static constexpr int kTurn = OFF ? 16 * 33 : 0; // of a warp: 16 rows of 32 results, to be written row by row
    static constexpr int kSmem = 1024 + kStages * kStageBytes + (kScaleStages * kScaleFloats + kOutWarps * kTurn) * 4 + 8 * kBars + 16;
};

struct Fp8Args {
    int m, n, k_blocks;
    int tiles_m, tiles_n, band; // tiles are walked in bands of `band` rows of tiles, so that a wave reads few distinct rows of a and b
    int a_across, b_across;     // the summed axis lies across the operand's rows
    unsigned desc;
    Scales a, b;
    void *out;
    long out_stride;
    int align; // 32, 16: the result's rows start on such a boundary; 0: on none
    int *status;
};

__device__ __forceinline__ void tile_at(const Fp8Args &a, int t, int &tm, int &tn)
{
    const int per_band = a.band * a.tiles_n, b = t / per_band, in = t - b * per_band;
    const int rows = min(a.band, a.tiles_m - b * a.band);
    tn = in / rows;
    tm = b * a.band + (in - tn * rows);
}

// Threads of the warps that take results out need more registers than an even share, those of the first warpgroup fewer: with 128 results each
// 56 + 2 x 224 of the 3 x 168 that the block has (launch_tiles sees that it has them: the second call waits for what the first one gives up).
constexpr int kEven = 168, kFew = 56, kMany = 224;

__device__ __forceinline__ void copy4(unsigned to, const float *from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory"); }

// One CTA per SM walks over tiles of 128 x BN.  Warp 0 brings 128 bytes of the summed axis of either operand by TMA into a ring of stages, warp 1 issues the
// products (four of k = 32 a block) into one of two or four places in TMEM, and warps 4 to 11 scale a block's sums and add them to results that they keep
// in registers: a scale is for 128 of the summed axis, so the sums have to leave TMEM that often.  A block of a tile 256 wide takes some 1050 cycles, of which the
// products are 512 (the tensor cores are active in 51 % of the cycles): what bounds it is the 96 KB that shared memory takes in and gives out a block, and the chain from
// the products' end over the sums' way to the registers to the next products, with two places for the sums.  8192 x 8192 x 8192 takes 480 to 500 us (2.2 P
// operations a second; among others of its kind 570 to 597 us, under the power cap), without the accumulating warps' work 423 us, without the products 323 us,
// without either 281 us.  Two CTAs on
// a tile of 256 x 256, which move 64 KB a block, wait longer for one another than that saves (732 us).  With a scale per row of b there is a product
// more for every sum, and TMEM is read 16 registers at a time: 4096 x 11008 x 4096 in 307 us, without that product 276, without the accumulating warps' work 169.  Everything in the accumulating warps' chain costs what it takes: a vote a block 3 %,
// scales through shared memory instead of a load ahead 25 % (with a scale per row, where loads are many, they gain 8 %).
//
// PER_ROW: b has a scale for each of its rows, otherwise one for 128.
// SPLIT: few tiles and a long summed axis.  The blocks of a cluster take a tile together, a run of the axis each, and add up through one another's
// shared memory, in the order of the runs: no second kernel, no atomics.  333 x 1111 x 2047 takes 8.2 us with it, 25.7 us without.
// OFF: the result's rows start on no 16-byte boundary: results are turned through shared memory, so that a warp writes 32 of a row at a time.
// 8000 x 7999 x 1024 in bf16 takes 146 us so, 680 us where every thread writes its own row, and with 8000 columns 82 us.
template <typename T, int BN, bool PER_ROW, bool SPLIT, bool OFF>
__global__ void __launch_bounds__(TileFp8<BN, OFF>::kThreads, 1) fp8_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                              const Fp8Args a)
{
    using C = TileFp8<BN, OFF>;
    extern __shared__ unsigned char raw[];
    unsigned char *stages = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    float *scales = reinterpret_cast<float *>(stages + C::kStages * C::kStageBytes); // [scale stage][kScaleFloats]
    float *turns = scales + C::kScaleStages * C::kScaleFloats; // [warp][kTurn]
    unsigned long long *bars = reinterpret_cast<unsigned long long *>(turns + C::kOutWarps * C::kTurn);
    unsigned *tmem_at = reinterpret_cast<unsigned *>(bars + C::kBars);
    volatile int *failed = reinterpret_cast<volatile int *>(tmem_at + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // stages of the operands, block sums in TMEM, stages of the scales: filled, and free again
    const unsigned full = smem_u32(bars), empty = full + 8 * C::kStages, done = empty + 8 * C::kStages, freed = done + 8 * C::kBufs, known = freed + 8 * C::kBufs,
                   used = known + 8 * C::kScaleStages, drained = used + 8 * C::kScaleStages;
    const unsigned stage0 = smem_u32(stages);

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < C::kBufs; ++i) {
            mbar_init(done + 8 * i, 1);
            mbar_init(freed + 8 * i, C::kOutWarps);
        }
        for (int i = 0; i < C::kScaleStages; ++i) {
            mbar_init(known + 8 * i, 64);
            mbar_init(used + 8 * i, C::kOutWarps);
        }
        mbar_init(drained, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "n"(C::kBufs * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = *tmem_at;
    unsigned rank = 0, ranks = 1;
    if (SPLIT) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    }
    const int tiles = SPLIT ? (int)(blockIdx.x / ranks) + 1 : a.tiles_m * a.tiles_n, tile0 = SPLIT ? (int)(blockIdx.x / ranks) : (int)blockIdx.x;
    const int k0 = SPLIT ? (int)((long)a.k_blocks * rank / ranks) : 0, k1 = SPLIT ? (int)((long)a.k_blocks * (rank + 1) / ranks) : a.k_blocks;

    if (warp < 4) {
        if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFew));
        if (warp == 0) {
            if (lane == 0) {
                int it = 0;
                bool ok = true;
                for (int t = tile0; t < tiles && ok; t += gridDim.x) {
                    int tm, tn;
                    tile_at(a, t, tm, tn);
                    for (int k = k0; k < k1; ++k, ++it) {
                        const int s = it % C::kStages;
                        if (it >= C::kStages) ok = mbar_wait(empty + 8 * s, (it / C::kStages - 1) & 1, failed);
                        if (!ok) break;
                        mbar_expect(full + 8 * s, C::kStageBytes);
                        const unsigned to = stage0 + s * C::kStageBytes;
                        tma_load(to, &map_a, a.a_across ? tm * kM : k * kK, a.a_across ? k * kK : tm * kM, full + 8 * s);
                        if (!a.b_across) {
                            tma_load(to + kM * kK, &map_b, k * kK, tn * BN, full + 8 * s);
                        } else { // boxes are 128 bytes wide: a run of 128 places at a time
#pragma unroll
                            for (int i = 0; i < BN / 128; ++i) tma_load(to + kM * kK + i * 128 * kK, &map_b, tn * BN + i * 128, k * kK, full + 8 * s);
                        }
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
            int it = 0;
            bool ok = true;
            for (int t = tile0; t < tiles && ok; t += gridDim.x) {
                for (int k = k0; k < k1; ++k, ++it) {
                    const int s = it % C::kStages, buf = it % C::kBufs;
                    if (it >= C::kBufs) ok = mbar_wait_warp(freed + 8 * buf, (it / C::kBufs - 1) & 1, failed);
                    if (ok) ok = mbar_wait_warp(full + 8 * s, (it / C::kStages) & 1, failed);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned at = stage0 + s * C::kStageBytes;
                    const unsigned long long da = a.a_across ? operand_desc_across(at, 128 * kK) : operand_desc(at);
                    const unsigned long long db = a.b_across ? operand_desc_across(at + kM * kK, 128 * kK) : operand_desc(at + kM * kK);
                    const int step_a = a.a_across ? 32 * 128 / 16 : 2, step_b = a.b_across ? 32 * 128 / 16 : 2; // 32 of the summed axis, in units of 16 bytes
#pragma unroll
                    for (int e = 0; e < kK / 32; ++e) mma_f8(elected, tmem + buf * BN, da + e * step_a, db + e * step_b, a.desc, e > 0);
                    mma_commit(elected, empty + 8 * s);
                    mma_commit(elected, done + 8 * buf);
                }
            }
            if (!ok) { // products that are still under way end before their memory is given back
                mma_commit(elected, drained);
                for (int n = 0; n < 1 << 20; ++n)
                    if (mbar_try(drained, 0)) break;
            }
        } else if (PER_ROW) { // the scales, blocks ahead of their use: of the rows, and of the columns
            int it = 0;
            bool ok = true;
            for (int t = tile0; t < tiles && ok; t += gridDim.x) {
                int tm, tn;
                tile_at(a, t, tm, tn);
                constexpr int kMine = BN / 32;
                const float *from[kMine > 4 ? kMine : 4];
                unsigned to[kMine > 4 ? kMine : 4];
                const long step = warp == 2 ? a.a.block : a.b.block;
                if (warp == 2) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        from[i] = a.a.at + (long)(min(tm * kM + i * 32 + lane, a.m - 1) >> a.a.shift) * a.a.row + k0 * step;
                        to[i] = i * 32 + lane;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
                        const int c = i * 32 + lane, in = c % C::kCols; // of each half of the columns four runs of every fourth pair
                        from[i] = a.b.at + (long)(min(tn * BN + c, a.n - 1) >> a.b.shift) * a.b.row + k0 * step;
                        to[i] = kM + c / C::kCols * 4 * C::kRun + (in >> 1 & 3) * C::kRun + (in >> 3) * 2 + (in & 1);
                    }
                }
                for (int k = k0; k < k1; ++k, ++it) {
                    const int s = it % C::kScaleStages;
                    if (it >= C::kScaleStages) ok = mbar_wait_warp(used + 8 * s, (it / C::kScaleStages - 1) & 1, failed);
                    if (!ok) break;
                    const unsigned at = smem_u32(scales + s * C::kScaleFloats);
                    if (warp == 2) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) copy4(at + 4 * to[i], from[i]), from[i] += step;
                    } else {
#pragma unroll
                        for (int i = 0; i < kMine; ++i) copy4(at + 4 * to[i], from[i]), from[i] += step;
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(known + 8 * s) : "memory");
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMany));
        // A warp sees the 32 lanes of TMEM of its quarter, and takes half of the tile's columns.  With one scale for them a thread has a row; with a
        // scale each it has, as in the results of a warp's own matrix instruction, two columns of every eight in four rows, so that it
        // needs a quarter of the scales.
        const int quarter = warp & 3, half = (warp - 4) / 4;
        constexpr int kRows = PER_ROW ? 4 : 1;
        int it = 0;
        bool ok = true;
        for (int t = tile0; t < tiles && ok; t += gridDim.x) {
            int tm, tn;
            tile_at(a, t, tm, tn);
            const int row = tm * kM + quarter * 32 + (PER_ROW ? lane >> 2 : lane), col = tn * BN + half * C::kCols;
            unsigned long long acc[C::kCols / 2];
#pragma unroll
            for (int e = 0; e < C::kCols / 2; ++e) acc[e] = 0;
            // One scale for the columns: every thread fetches the two that it needs, a block ahead.  A scale each: two warps bring them into shared memory
            const float *pa = a.a.at + (long)(min(row, a.m - 1) >> a.a.shift) * a.a.row + k0 * a.a.block, *pb = a.b.at + (long)(min(col, a.n - 1) >> a.b.shift) * a.b.row + k0 * a.b.block;
            float next_row = 0.f, next_col = 0.f;
            if (!PER_ROW && k0 < k1) next_row = __ldg(pa), next_col = __ldg(pb);
            for (int k = k0; k < k1; ++k, ++it) {
                const int buf = it % C::kBufs, stage = it % C::kScaleStages;
                const float *row_scales = scales + stage * C::kScaleFloats + quarter * 32 + (lane >> 2);
                const float *col_scales = scales + stage * C::kScaleFloats + kM + half * 4 * C::kRun + (lane & 3) * C::kRun;
                unsigned long long ss[kRows];
                if (PER_ROW) {
                    ok &= mbar_wait_inline(known + 8 * stage, (it / C::kScaleStages) & 1, failed);
#pragma unroll
                    for (int r = 0; r < kRows; ++r) ss[r] = pair(row_scales[8 * r], row_scales[8 * r]);
                } else {
                    ss[0] = pair(next_row * next_col, next_row * next_col);
                    if (k + 1 < k1) next_row = __ldg(pa += a.a.block), next_col = __ldg(pb += a.b.block);
                }
                ok &= mbar_wait_inline(done + 8 * buf, (it / C::kBufs) & 1, failed); // a warp whose wait ran out goes on to the tile's end
                __syncwarp(); // every lane has waited for itself, in as many turns as it took: loads out of TMEM want the whole warp at once
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned from = tmem + buf * BN + half * C::kCols + ((unsigned)quarter << 21);
                constexpr int kW = PER_ROW || OFF ? 16 : 32;
                int v[2][kW];
                auto begin = [&](int step, int (&w)[kW]) { // 32 columns of 16 rows, the upper ones and then the lower ones; or 16 columns of all rows
                    if constexpr (PER_ROW) tmem_begin_tiles(from + (step >> 1) * 32 + ((unsigned)(step & 1) << 20), w);
                    else tmem_begin(from + step * kW, w);
                };
                begin(0, v[0]);
#pragma unroll
                for (int step = 0; step < C::kCols / kW; ++step) {
                    int(&w)[kW] = v[step & 1];
                    tmem_ready(w);
                    if (step + 1 < C::kCols / kW) begin(step + 1, v[(step & 1) ^ 1]);
                    if constexpr (PER_ROW) {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) { // eight columns, and the next eight
                            const int eight = (step >> 1) * 4 + i, at = ((step & 1) * (C::kCols / 8) + eight) * 2, r = (step & 1) * 2;
                            const ulonglong2 s4 = *reinterpret_cast<const ulonglong2 *>(col_scales + eight * 2);
                            fma2(acc[at], mul2(pair(w[4 * i], w[4 * i + 1]), ss[r]), s4.x);
                            fma2(acc[at + 1], mul2(pair(w[4 * i + 2], w[4 * i + 3]), ss[r + 1]), s4.x);
                            fma2(acc[at + 2], mul2(pair(w[4 * i + 4], w[4 * i + 5]), ss[r]), s4.y);
                            fma2(acc[at + 3], mul2(pair(w[4 * i + 6], w[4 * i + 7]), ss[r + 1]), s4.y);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < kW; e += 2) fma2(acc[step * kW / 2 + e / 2], pair(w[e], w[e + 1]), ss[0]);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(freed + 8 * buf);
                    if (PER_ROW) mbar_arrive(used + 8 * stage);
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (SPLIT) { // all products have been formed, so the stages are free
                float *to = reinterpret_cast<float *>(stages) + (quarter * 32 + (PER_ROW ? lane >> 2 : lane)) * C::kPitch + half * C::kCols + (PER_ROW ? (lane & 3) * 2 : 0);
#pragma unroll
                for (int e = 0; e < C::kCols / 2; ++e) {
                    float2 x;
                    unpair(acc[e], x.x, x.y);
                    *reinterpret_cast<float2 *>(PER_ROW ? to + ((e & 1) * 8 + e / (C::kCols / 4) * 16) * C::kPitch + (e % (C::kCols / 4) >> 1) * 8 : to + 2 * e) = x;
                }
            } else if (OFF) { // turned through shared memory, so that a warp writes 32 results of a row at a time
                float *turn = turns + (warp - 4) * C::kTurn;
                const int first = tm * kM + quarter * 32;
#pragma unroll
                for (int c = 0; c < C::kCols; c += 32) {
#pragma unroll
                    for (int upper = 0; upper < 2; ++upper) {
                        __syncwarp();
                        if (PER_ROW) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int r = 0; r < 2; ++r) {
                                    float x, y;
                                    unpair(acc[(upper * (C::kCols / 8) + c / 8 + i) * 2 + r], x, y);
                                    float *to = turn + ((lane >> 2) + 8 * r) * 33 + i * 8 + (lane & 3) * 2;
                                    to[0] = x, to[1] = y;
                                }
                        } else if ((lane >> 4) == upper) {
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                float x, y;
                                unpair(acc[(c + e) / 2], x, y);
                                turn[(lane & 15) * 33 + e] = x, turn[(lane & 15) * 33 + e + 1] = y;
                            }
                        }
                        __syncwarp();
                        const int rows = min(16, a.m - first - upper * 16);
                        T *to = reinterpret_cast<T *>(a.out) + (long)(first + upper * 16) * a.out_stride + col + c + lane;
                        if (col + c + lane < a.n)
                            for (int i = 0; i < rows; ++i, to += a.out_stride) put(to, turn[i * 33 + lane]);
                    }
                }
            } else if (PER_ROW) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (row + 8 * r >= a.m) continue;
                    T *out = reinterpret_cast<T *>(a.out) + (long)(row + 8 * r) * a.out_stride + col + (lane & 3) * 2;
#pragma unroll
                    for (int i = 0; i < C::kCols / 8; ++i) {
                        float x, y;
                        unpair(acc[((r >> 1) * (C::kCols / 8) + i) * 2 + (r & 1)], x, y);
                        const int left = a.n - col - (lane & 3) * 2 - i * 8;
                        if (left >= 2) {
                            if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(out + i * 8) = make_float2(x, y);
                            else *reinterpret_cast<unsigned *>(out + i * 8) = pack2(out, x, y);
                        } else if (left == 1) {
                            put(out + i * 8, x);
                        }
                    }
                }
            } else if (row < a.m) {
                T *out = reinterpret_cast<T *>(a.out) + (long)row * a.out_stride + col;
#pragma unroll
                for (int c = 0; c < C::kCols; c += 32) {
                    float f[32];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) unpair(acc[(c + e) / 2], f[e], f[e + 1]);
                    if (col + c < a.n) put32(out + c, f, a.n - col - c, a.align);
                }
            }
        }
    }
    if (SPLIT) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        int tm, tn;
        tile_at(a, tile0, tm, tn);
        const int rows = min(kM, a.m - tm * kM), cols = min(BN, a.n - tn * BN), all = rows * (BN / 4);
        for (int i = (int)((long)all * rank / ranks) + (int)threadIdx.x; i < (int)((long)all * (rank + 1) / ranks); i += C::kThreads) {
            const int r = i / (BN / 4), c = i % (BN / 4) * 4;
            if (c >= cols) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (unsigned from = 0; from < ranks; ++from) {
                unsigned at;
                float4 v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(stage0 + (r * C::kPitch + c) * 4), "r"(from));
                asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
                sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
            }
            T *out = reinterpret_cast<T *>(a.out) + (long)(tm * kM + r) * a.out_stride + tn * BN + c;
            if (a.align && c + 4 <= cols) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(out) = sum;
                else *reinterpret_cast<uint2 *>(out) = make_uint2(pack2(out, sum.x, sum.y), pack2(out, sum.z, sum.w));
            } else {
                put(out, sum.x);
                if (c + 1 < cols) put(out + 1, sum.y);
                if (c + 2 < cols) put(out + 2, sum.z);
                if (c + 3 < cols) put(out + 3, sum.w);
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); // nobody leaves while it is read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (threadIdx.x == 0 && *failed) atomicOr(a.status, 2);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kBufs * BN) : "memory");
}

template <typename T, int BN, bool PER_ROW, bool SPLIT, bool OFF>
int launch_tiles(const Context *ctx, const CUtensorMap &ma, const CUtensorMap &mb, const Fp8Args &a, int split, cudaStream_t stream)
{
    using C = TileFp8<BN, OFF>;
    const auto kernel = fp8_product_kernel<T, BN, PER_ROW, SPLIT, OFF>;
    static std::atomic<bool> set[64]; // host threads that come here first at once all set the same attribute
    if (ctx->device >= 64 || !set[ctx->device]) {
        LB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (BN == 256) {
            cudaFuncAttributes has;
            LB_CUDA(cudaFuncGetAttributes(&has, kernel));
            if (has.numRegs < kEven) {
                set_error("the product's kernel was built with too few registers");
                return LB_ERR_LOGIC;
            }
        }
        if (ctx->device < 64) set[ctx->device] = true;
    }
    const int tiles = a.tiles_m * a.tiles_n;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)(SPLIT ? tiles * split : tiles < ctx->sm_count ? tiles : ctx->sm_count));
    c.blockDim = dim3(C::kThreads);
    c.dynamicSmemBytes = C::kSmem;
    c.stream = stream;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = (unsigned)split;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    c.attrs = &cluster;
    c.numAttrs = SPLIT ? 1 : 0;
    LB_CUDA(cudaLaunchKernelEx(&c, kernel, ma, mb, a));
    return LB_OK;
}
template <typename T, int BN, bool PER_ROW> int launch_whole(const Context *ctx, const CUtensorMap &ma, const CUtensorMap &mb, const Fp8Args &a, cudaStream_t stream)
{
    return a.align ? launch_tiles<T, BN, PER_ROW, false, false>(ctx, ma, mb, a, 1, stream) : launch_tiles<T, BN, PER_ROW, false, true>(ctx, ma, mb, a, 1, stream);
}
template <typename T, bool PER_ROW> int launch_any(const Context *ctx, int bn, const CUtensorMap &ma, const CUtensorMap &mb, const Fp8Args &a, int split, cudaStream_t stream)
{
    if (split > 1) return bn == 128 ? launch_tiles<T, 128, PER_ROW, true, false>(ctx, ma, mb, a, split, stream) : launch_tiles<T, 64, PER_ROW, true, false>(ctx, ma, mb, a, split, stream);
    if (bn == 256) return launch_whole<T, 256, PER_ROW>(ctx, ma, mb, a, stream);
    return bn == 128 ? launch_whole<T, 128, PER_ROW>(ctx, ma, mb, a, stream) : launch_whole<T, 64, PER_ROW>(ctx, ma, mb, a, stream);
}

// an operand as it lies: rows of `cols` bytes
struct Stored {
    long rows;
    int cols;
    bool off; // rows off a 16-byte boundary: TMA cannot read them
    int pitch;
};
Stored stored(const Fp8Operand &o, int along, int k)
{
    Stored s;
    s.rows = o.across ? k : along;
    s.cols = o.across ? along : k;
    s.off = (uintptr_t)o.codes % 16 != 0 || (s.rows > 1 && o.stride % 16 != 0);
    s.pitch = (s.cols + 15) / 16 * 16;
    return s;
}
size_t packed_bytes(const Stored &s) { return s.off ? ((size_t)s.rows * s.pitch + 255) / 256 * 256 : 0; }

bool skinny(int m, int n, const Fp8Operand &a, const Fp8Operand &b) { return !a.across && !b.across && (m <= kSkinny || n <= kSkinny); }

template <typename T> int product_typed(Context *ctx, int m, int n, int k, const Fp8Operand &a, const Fp8Operand &b, void *out, long out_stride, cudaStream_t stream)
{
    if (skinny(m, n, a, b)) {
        const bool turned = m > n; // the long side is the rows of a
        const Fp8Operand &w = turned ? a : b, &x = turned ? b : a;
        SkinnyFp8Args s;
        s.w = reinterpret_cast<const signed char *>(w.codes);
        s.x = reinterpret_cast<const signed char *>(x.codes);
        s.w_stride = w.stride;
        s.x_stride = x.stride;
        s.ws = {w.scales, w.scale_row, w.scale_block, w.scale_shift};
        s.xs = {x.scales, x.scale_row, x.scale_block, x.scale_shift};
        s.rows = turned ? m : n;
        s.cols = turned ? n : m;
        s.k = k;
        s.w_first = turned;
        s.out = out;
        s.row_step = turned ? out_stride : 1;
        s.col_step = turned ? 1 : out_stride;
        count_launch("fp8_skinny", stream, (double)m * k + (double)n * k + (double)m * n * sizeof(T));
        const bool off = k % 16 != 0 || stored(a, m, k).off || stored(b, n, k).off;
        return off ? launch_skinny<T, false>(s, w.type == 6, x.type == 6, stream) : launch_skinny<T, true>(s, w.type == 6, x.type == 6, stream);
    }
    Fp8Args p;
    p.m = m;
    p.n = n;
    p.k_blocks = (k + kK - 1) / kK;
    p.tiles_m = (m + kM - 1) / kM;
    p.a_across = a.across;
    p.b_across = b.across;
    p.a = {a.scales, a.scale_row, a.scale_block, a.scale_shift};
    p.b = {b.scales, b.scale_row, b.scale_block, b.scale_shift};
    p.out = out;
    p.out_stride = out_stride;
    const uintptr_t at = (uintptr_t)out | (uintptr_t)(out_stride * (long)sizeof(T));
    p.align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 0;
    p.status = ctx->d_status;
    p.band = 8;
    // The tile, and the CTAs that share one, that take least, in microseconds as measured: waves over the SMs, in each a block of the summed axis at
    // what one takes (by shared memory and the accumulating warps; with a scale per row of b by the latter), and a tile's results; a split adds two.
    // 2048 x 2048 x 2048 takes 12.7 us with tiles 256 wide and 16.3 with 128, 4096 x 4096 x 64 14.3 and 13.5; 100 x 100 x 4096 7.0 us split
    // over eight and 18.8 by one.  Results off a 16-byte boundary, which take longer to write, get the same tiles: the times are those of aligned ones.
    int bn = 128, split = 1;
    double least = 0.0;
    const bool per_row = b.scale_shift == 0;
    for (int w = b.across ? 128 : 64; w <= 256; w *= 2)
        for (int parts = 1; parts <= 8 && parts <= p.k_blocks; ++parts) {
            const long tiles = (long)p.tiles_m * ((n + w - 1) / w), blocks = tiles * parts, waves = (blocks + ctx->sm_count - 1) / ctx->sm_count;
            if (parts > 1 && (w == 256 || blocks > ctx->sm_count - ctx->sm_count / 8)) break; // clusters do not fill every group of SMs
            const int k = (p.k_blocks + parts - 1) / parts;
            const double block = per_row ? 0.06 + w * 3.3e-3 : w == 64 ? 0.3 : 0.16 + w * 1.33e-3;
            const double us = (double)waves * (k * block + w * 14e-3) + (parts > 1 ? 2.0 : 0.0);
            if (least == 0.0 || us < least) {
                least = us;
                bn = w;
                split = parts;
            }
        }
    p.tiles_n = (n + bn - 1) / bn;
    // D 32-bit floats; the operands' types, and bits 15 and 16 where the summed axis lies across their rows
    p.desc = (unsigned)(bn >> 3) << 17 | (unsigned)(kM >> 4) << 24 | 1u << 4 | (unsigned)(a.type == 6) << 7 | (unsigned)(b.type == 6) << 10 | (unsigned)a.across << 15 |
             (unsigned)b.across << 16;
    const Stored sa = stored(a, m, k), sb = stored(b, n, k);
    CUtensorMap ma, mb;
    int rc = encode_map(&ma, a.codes, sa.rows, sa.cols, sa.rows > 1 ? a.stride : sa.pitch, 128, 128);
    if (rc) return rc;
    if ((rc = encode_map(&mb, b.codes, sb.rows, sb.cols, sb.rows > 1 ? b.stride : sb.pitch, 128, b.across ? 128 : bn))) return rc;
    count_launch("fp8_tiles", stream, (double)m * k + (double)n * k + (double)m * n * sizeof(T));
    return per_row ? launch_any<T, true>(ctx, bn, ma, mb, p, split, stream) : launch_any<T, false>(ctx, bn, ma, mb, p, split, stream);
}

} // namespace

size_t fp8_matmul_workspace_bytes(int m, int n, int k, const Fp8Operand &a, const Fp8Operand &b)
{
    return skinny(m, n, a, b) ? 0 : packed_bytes(stored(a, m, k)) + packed_bytes(stored(b, n, k));
}

int fp8_matmul(Context *ctx, int m, int n, int k, Fp8Operand a, Fp8Operand b, void *out, int dtype, long out_stride, void *workspace, cudaStream_t stream)
{
    signed char *ws = reinterpret_cast<signed char *>(workspace);
    for (int i = 0; i < 2; ++i) { // operands that TMA cannot read
        Fp8Operand &o = i ? b : a;
        const Stored s = stored(o, i ? n : m, k);
        if (!s.off || skinny(m, n, a, b)) continue;
        const Packed one = {reinterpret_cast<const signed char *>(o.codes), o.stride, s.rows, ws}, none = {nullptr, 0, 0, nullptr};
        int log_lanes = 0;
        while (log_lanes < 8 && 16 << log_lanes < s.pitch) ++log_lanes;
        const long blocks = (s.rows + (256 >> log_lanes) - 1) >> (8 - log_lanes), most = (long)ctx->sm_count * 32;
        count_launch("fp8_pack", stream, 2.0 * s.rows * s.cols);
        pack_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(one, none, s.cols, s.pitch, log_lanes);
        LB_CUDA(cudaGetLastError());
        o.codes = reinterpret_cast<unsigned char *>(ws);
        o.stride = s.pitch;
        ws += packed_bytes(s);
    }
    switch (dtype) {
    case 1: return product_typed<float>(ctx, m, n, k, a, b, out, out_stride, stream);
    case 3: return product_typed<__nv_bfloat16>(ctx, m, n, k, a, b, out, out_stride, stream);
    default: return product_typed<__half>(ctx, m, n, k, a, b, out, out_stride, stream);
    }
}

} // namespace lb
