// Matrix product of 8-bit floating point with a scale for each block of 128 of the summed axis:
//   out[m][n] = sum over blocks p of (sum over k in p of a[m][k] b[n][k]) * a_scale[m][p] * b_scale[n][p]
// A block's sum is formed by the tensor cores in 32-bit floats, scaled, and added to the result in 32-bit floats; the result is rounded once to
// its type.  Either operand may lie with the summed axis across its rows: the gradients of a product y = x w^T read x, w and the
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

template <int BN> struct TileFp8 {
    static constexpr int kOutWarps = 8, kThreads = 128 + kOutWarps * 32;
    static constexpr int kCols = BN / 2; // columns of a thread: the warps of a quarter of TMEM's lanes take a half each
    static constexpr int kStageBytes = (kM + BN) * kK;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kBufs = BN == 256 ? 2 : 4; // block sums in TMEM
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kOutWarps * kCols * 4 + 256;
};

struct Scales {
    const float *at;
    long row, block; // from one row (or block of 128 rows) to the next; from one block of the summed axis to the next
    int shift;       // 7: a scale for 128 rows
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
constexpr int kChunk = 16;
constexpr int kEven = 168, kFew = 56, kMany = 224;

// PER_ROW: b has a scale for each of its rows, otherwise one for 128
template <typename T, int BN, bool PER_ROW>
__global__ void __launch_bounds__(TileFp8<BN>::kThreads, 1) fp8_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                              const Fp8Args a)
{
    using C = TileFp8<BN>;
    extern __shared__ unsigned char raw[];
    unsigned char *stages = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    float *scales = reinterpret_cast<float *>(stages + C::kStages * C::kStageBytes); // [warp][kCols]
    unsigned char *tail = reinterpret_cast<unsigned char *>(scales + C::kOutWarps * C::kCols);
    unsigned long long *bars = reinterpret_cast<unsigned long long *>(tail); // full[stages], empty[stages], done[bufs], freed[bufs], drained
    unsigned *tmem_at = reinterpret_cast<unsigned *>(bars + 2 * C::kStages + 2 * C::kBufs + 1);
    volatile int *failed = reinterpret_cast<volatile int *>(tmem_at + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned full = smem_u32(bars), empty = full + 8 * C::kStages, done = empty + 8 * C::kStages, freed = done + 8 * C::kBufs, drained = freed + 8 * C::kBufs;
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
    const int tiles = a.tiles_m * a.tiles_n;

    if (warp < 4) {
    if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFew));
    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                int tm, tn;
                tile_at(a, t, tm, tn);
                for (int k = 0; k < a.k_blocks; ++k, ++it) {
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
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            for (int k = 0; k < a.k_blocks; ++k, ++it) {
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
    }
    } else {
        if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMany));
        // a warp sees the 32 lanes of TMEM of its quarter; a thread has a row and half of the tile's columns
        const int quarter = warp & 3, half = (warp - 4) / 4;
        float *sb = scales + (warp - 4) * C::kCols;
        int it = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            int tm, tn;
            tile_at(a, t, tm, tn);
            const int row = tm * kM + quarter * 32 + lane, col = tn * BN + half * C::kCols;
            const float *pa = a.a.at + (long)(min(row, a.m - 1) >> a.a.shift) * a.a.row;
            const float *pb = a.b.at + (long)(min(col, a.n - 1) >> a.b.shift) * a.b.row;
            unsigned long long acc[C::kCols / 2];
#pragma unroll
            for (int e = 0; e < C::kCols / 2; ++e) acc[e] = 0;
            float sa = __ldg(pa), one = 0.f, many[C::kCols / 32];
            auto fetch_b = [&](int k) { // the scales of block k of b
                if (PER_ROW) {
#pragma unroll
                    for (int c = 0; c < C::kCols / 32; ++c)
                        many[c] = __ldg(a.b.at + (long)min(col + c * 32 + lane, a.n - 1) * a.b.row + (long)k * a.b.block);
                } else {
                    one = __ldg(pb + (long)k * a.b.block);
                }
            };
            fetch_b(0);
            for (int k = 0; k < a.k_blocks; ++k, ++it) {
                const int buf = it % C::kBufs;
                const float s = PER_ROW ? sa : sa * one;
                const unsigned long long ss = pair(s, s);
                if (PER_ROW) {
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < C::kCols / 32; ++c) sb[c * 32 + lane] = many[c];
                    __syncwarp();
                }
                if (k + 1 < a.k_blocks) { // those of the next block, on their way while this one is added up
                    sa = __ldg(pa + (long)(k + 1) * a.a.block);
                    fetch_b(k + 1);
                }
                ok = mbar_wait_inline(done + 8 * buf, (it / C::kBufs) & 1, failed);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned from = tmem + buf * BN + half * C::kCols + ((unsigned)quarter << 21);
                int v[2][kChunk];
                tmem_begin(from, v[0]);
#pragma unroll
                for (int c = 0; c < C::kCols; c += kChunk) {
                    int(&w)[kChunk] = v[c / kChunk & 1];
                    tmem_ready(w);
                    if (c + kChunk < C::kCols) tmem_begin(from + c + kChunk, v[(c / kChunk & 1) ^ 1]);
#pragma unroll
                    for (int e = 0; e < kChunk; e += 4) {
                        if (PER_ROW) {
                            const ulonglong2 s4 = *reinterpret_cast<const ulonglong2 *>(sb + c + e);
                            fma2(acc[(c + e) / 2], mul2(pair(w[e], w[e + 1]), ss), s4.x);
                            fma2(acc[(c + e) / 2 + 1], mul2(pair(w[e + 2], w[e + 3]), ss), s4.y);
                        } else {
                            fma2(acc[(c + e) / 2], pair(w[e], w[e + 1]), ss);
                            fma2(acc[(c + e) / 2 + 1], pair(w[e + 2], w[e + 3]), ss);
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(freed + 8 * buf);
            }
            if (!ok) break;
            if (row < a.m) {
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
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (threadIdx.x == 0 && *failed) atomicOr(a.status, 2);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kBufs * BN) : "memory");
}

template <typename T, int BN, bool PER_ROW> int launch_tiles(const Context *ctx, const CUtensorMap &ma, const CUtensorMap &mb, const Fp8Args &a, cudaStream_t stream)
{
    using C = TileFp8<BN>;
    static std::atomic<bool> set[64]; // host threads that come here first at once all set the same attribute
    if (ctx->device >= 64 || !set[ctx->device]) {
        LB_CUDA(cudaFuncSetAttribute(fp8_product_kernel<T, BN, PER_ROW>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (BN == 256) {
            cudaFuncAttributes has;
            LB_CUDA(cudaFuncGetAttributes(&has, fp8_product_kernel<T, BN, PER_ROW>));
            if (has.numRegs < kEven) {
                set_error("the product's kernel was built with too few registers");
                return LB_ERR_LOGIC;
            }
        }
        if (ctx->device < 64) set[ctx->device] = true;
    }
    const int tiles = a.tiles_m * a.tiles_n;
    fp8_product_kernel<T, BN, PER_ROW><<<tiles < ctx->sm_count ? tiles : ctx->sm_count, C::kThreads, C::kSmem, stream>>>(ma, mb, a);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
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

template <typename T> int product_typed(Context *ctx, int m, int n, int k, const Fp8Operand &a, const Fp8Operand &b, void *out, long out_stride, cudaStream_t stream)
{
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
    int bn = 128;
    double least = 0.0;
    for (int w = b.across ? 128 : 64; w <= 256; w *= 2) {
        const long tiles = (long)p.tiles_m * ((n + w - 1) / w), waves = (tiles + ctx->sm_count - 1) / ctx->sm_count;
        const double us = (double)waves * ((double)p.k_blocks * (128 + w) * 1.15e-3 + 0.7 + w * 6e-3);
        if (least == 0.0 || us < least) {
            least = us;
            bn = w;
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
    const bool per_row = b.scale_shift == 0;
    if (bn == 256) return per_row ? launch_tiles<T, 256, true>(ctx, ma, mb, p, stream) : launch_tiles<T, 256, false>(ctx, ma, mb, p, stream);
    if (bn == 128) return per_row ? launch_tiles<T, 128, true>(ctx, ma, mb, p, stream) : launch_tiles<T, 128, false>(ctx, ma, mb, p, stream);
    return per_row ? launch_tiles<T, 64, true>(ctx, ma, mb, p, stream) : launch_tiles<T, 64, false>(ctx, ma, mb, p, stream);
}

} // namespace

size_t fp8_matmul_workspace_bytes(int m, int n, int k, const Fp8Operand &a, const Fp8Operand &b)
{
    return packed_bytes(stored(a, m, k)) + packed_bytes(stored(b, n, k));
}

int fp8_matmul(Context *ctx, int m, int n, int k, Fp8Operand a, Fp8Operand b, void *out, int dtype, long out_stride, void *workspace, cudaStream_t stream)
{
    signed char *ws = reinterpret_cast<signed char *>(workspace);
    for (int i = 0; i < 2; ++i) {
        Fp8Operand &o = i ? b : a;
        const Stored s = stored(o, i ? n : m, k);
        if (!s.off) continue;
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
