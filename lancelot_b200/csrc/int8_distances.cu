// Squared distances between all pairs of cached 8-bit updates, the plaintext selection rule of the reference's driver
// (lancelot-main-GPU/utils/byzantine_fl.py:162-171, 527-536) without the updates ever being expanded.
//
//   D_ij = |x_i|^2 + |x_j|^2 - 2 <x_i, x_j>,   <x_i, x_j> = sum over groups g of s_ig s_jg (sum of q_ik q_jk inside g)
//
// The inner sums are integer products on the tensor cores and exact; the scales are applied, and the groups added, in 64-bit
// floats, so that the three terms of D_ij may cancel by nine digits before a 32-bit result would suffer.  Two equal updates
// give exactly 0: the same warps add the same numbers in the same order for ii, ij and jj.
//
// Bound by reading the codes once.  The rows of a tile of clients go from memory straight into the registers of the matrix
// instruction: a row of A and a column of B are both "a client's codes along k", and the order of k inside the product does not
// matter as long as both sides agree, so lane (g, t) loads 16 consecutive bytes of client g and uses them as four k-slots of A and
// of B at once.  No shared memory, no transposition, one load per code.
#include "context.h"

namespace lb {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct DistanceArgs {
    const signed char *codes;
    long code_stride;
    const float *scales;
    long scale_stride;
    long n_slots;
    const int *slots; // [n][pages]; nullptr: in order
    int n, pages, page;
    int group;          // columns of a group; page for one group in a page
    int unit;           // columns a warp takes at a time, within a page
    unsigned units_per_page, units;
    int blocks; // blocks per tile
    double *partial; // [tile][block][32][32]
};

__device__ __forceinline__ long slot_of(const DistanceArgs &a, int row, unsigned page)
{
    const long i = (long)row * a.pages + page;
    return a.slots ? (long)a.slots[i] : i;
}

// tile t of the upper triangle of row blocks -> (i, j), i <= j
__device__ __forceinline__ void tile_of(int t, int n_blocks, int &i, int &j)
{
    i = 0;
    while (t >= n_blocks - i) {
        t -= n_blocks - i;
        ++i;
    }
    j = i + t;
}

// the products of one tile of client blocks: DIAG: RB blocks of 8 clients with themselves; otherwise 4 blocks with RB others
template <int RB, bool DIAG, int BYTES>
__device__ void gram_tile(const DistanceArgs &a, const int row_a, const int row_b, double *sum, double *out)
{
    constexpr int RA = DIAG ? RB : 4;        // blocks of 8 rows
    constexpr int RP = (RA + 1) / 2;         // pairs of them: the 16 rows of A
    constexpr int NL = DIAG ? RB : 4 + RB;   // blocks to load
    constexpr int STEP = BYTES * 4, W = BYTES / 4;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;

    double total[RP][RB][4];
#pragma unroll
    for (int p = 0; p < RP; ++p)
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[p][j][e] = 0.0;

    int rows[NL];
#pragma unroll
    for (int r = 0; r < NL; ++r) {
        rows[r] = (r < RA ? row_a + r * 8 : row_b + (r - RA) * 8) + g;
        if (rows[r] >= a.n) rows[r] = -1;
    }
    const unsigned stride = a.blocks * kWarps;
    const int step_cols = a.group < a.unit ? a.group : a.unit; // columns between two applications of the scales
    unsigned u = blockIdx.y * kWarps + warp;
    long slot[NL];
#pragma unroll
    for (int r = 0; r < NL; ++r) slot[r] = u < a.units && rows[r] >= 0 ? slot_of(a, rows[r], u / a.units_per_page) : -1;
    for (; u < a.units; u += stride) {
        const unsigned part = u % a.units_per_page;
        const signed char *src[NL];
        const float *scl[NL];
#pragma unroll
        for (int r = 0; r < NL; ++r) {
            const bool there = slot[r] >= 0 && slot[r] < a.n_slots;
            src[r] = there ? a.codes + slot[r] * a.code_stride : nullptr;
            scl[r] = there ? a.scales + slot[r] * a.scale_stride : nullptr;
        }
        const unsigned next = u + stride; // the slots of the next unit are on their way while this one is computed
#pragma unroll
        for (int r = 0; r < NL; ++r) slot[r] = next < a.units && rows[r] >= 0 ? slot_of(a, rows[r], next / a.units_per_page) : -1;
        const int begin = part * a.unit, end = min(begin + a.unit, a.page);
        for (int c0 = begin; c0 < end; c0 += step_cols) {
            const int c1 = min(c0 + step_cols, end);
            float s[NL];
#pragma unroll
            for (int r = 0; r < NL; ++r) s[r] = scl[r] ? __ldg(scl[r] + c0 / a.group) : 0.f;
            int acc[RP][RB][4];
#pragma unroll
            for (int p = 0; p < RP; ++p)
#pragma unroll
                for (int j = 0; j < RB; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[p][j][e] = 0;
#pragma unroll 2
            for (int c = c0; c < c1; c += STEP) {
                const int at = c + t * BYTES;
                unsigned w[NL + 1][W];
#pragma unroll
                for (int r = 0; r < NL; ++r) {
                    if constexpr (BYTES == 16) {
                        const uint4 x = src[r] && at < c1 ? __ldg(reinterpret_cast<const uint4 *>(src[r] + at)) : make_uint4(0, 0, 0, 0);
                        w[r][0] = x.x;
                        w[r][1] = x.y;
                        w[r][2] = x.z;
                        w[r][3] = x.w;
                    } else {
                        const uint2 x = src[r] && at < c1 ? __ldg(reinterpret_cast<const uint2 *>(src[r] + at)) : make_uint2(0, 0);
                        w[r][0] = x.x;
                        w[r][1] = x.y;
                    }
                }
#pragma unroll
                for (int k = 0; k < W; ++k) w[NL][k] = 0;
#pragma unroll
                for (int k = 0; k < W; k += 2)
#pragma unroll
                    for (int p = 0; p < RP; ++p) {
                        const int hi = 2 * p + 1 < RA ? 2 * p + 1 : NL;
#pragma unroll
                        for (int j = DIAG ? 2 * p : 0; j < RB; ++j) {
                            const int b = DIAG ? j : RA + j;
                            mma_s8(acc[p][j], w[2 * p][k], w[hi][k], w[2 * p][k + 1], w[hi][k + 1], w[b][k], w[b][k + 1]);
                        }
                    }
            }
            // accumulator e of a lane: row g (+ 8 for e >= 2) of A, column 2 t + (e & 1) of B
#pragma unroll
            for (int j = 0; j < RB; ++j) {
                const float sj = s[DIAG ? j : RA + j];
                const double s0 = __shfl_sync(0xffffffffu, sj, t * 8), s1 = __shfl_sync(0xffffffffu, sj, t * 8 + 4);
#pragma unroll
                for (int p = 0; p < RP; ++p) {
                    if (DIAG && j < 2 * p) continue;
                    const double lo = s[2 * p], hi = 2 * p + 1 < RA ? s[2 * p + 1] : 0.f;
                    total[p][j][0] += (lo * s0) * (double)acc[p][j][0];
                    total[p][j][1] += (lo * s1) * (double)acc[p][j][1];
                    if (2 * p + 1 < RA) {
                        total[p][j][2] += (hi * s0) * (double)acc[p][j][2];
                        total[p][j][3] += (hi * s1) * (double)acc[p][j][3];
                    }
                }
            }
        }
    }
    // the block's warps one after the other: the order of the additions is fixed
    for (int k = 0; k < kWarps; ++k) {
        if (warp == k) {
#pragma unroll
            for (int p = 0; p < RP; ++p)
#pragma unroll
                for (int j = 0; j < RB; ++j) {
                    if (DIAG && j < 2 * p) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        double *at = sum + (p * 16 + g + (e >> 1) * 8) * 32 + j * 8 + t * 2 + (e & 1);
                        *at = k ? *at + total[p][j][e] : total[p][j][e];
                    }
                }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < RP * 16 * 32; i += kWarps * 32) {
        const int p = i >> 9, j = (i & 31) >> 3;
        if (j < RB && (!DIAG || j >= 2 * p)) out[i] = sum[i];
    }
}

template <int RB, bool DIAG_ONLY, int BYTES>
__global__ void __launch_bounds__(kWarps * 32) gram_kernel(const DistanceArgs a, const int n_blocks)
{
    __shared__ double sum[32 * 32];
    int i = 0, j = 0;
    if (!DIAG_ONLY) tile_of(blockIdx.x, n_blocks, i, j);
    double *out = a.partial + ((size_t)blockIdx.x * a.blocks + blockIdx.y) * 1024;
    if (DIAG_ONLY || i == j) gram_tile<RB, true, BYTES>(a, i * 32, j * 32, sum, out);
    else gram_tile<RB, false, BYTES>(a, i * 32, j * 32, sum, out);
}

// a warp per pair i <= j: the partial sums of the blocks, then the distance
__global__ void __launch_bounds__(256) distance_finish_kernel(const double *__restrict__ partial, const int n, const int n_blocks, const int blocks,
                                                              double *__restrict__ out)
{
    const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int i = (int)(w / n), j = (int)(w - (long)i * n);
    if (i >= n || j < i) return;
    auto dot = [&](int x, int y) {
        const int bi = x >> 5, bj = y >> 5;
        const long tile = (long)bi * n_blocks - (long)bi * (bi - 1) / 2 + (bj - bi);
        const double *p = partial + tile * blocks * 1024 + (x & 31) * 32 + (y & 31);
        double v = 0.0;
        for (int b = lane; b < blocks; b += 32) v += p[(size_t)b * 1024];
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    double d = 0.0;
    if (i != j) {
        const double x = dot(i, i), y = dot(j, j), z = dot(i, j);
        d = (x - z) + (y - z);
        if (d < 0.0) d = 0.0; // rounding of nearly equal updates; NaN stays
    }
    if (lane == 0) {
        out[(long)i * n + j] = d;
        out[(long)j * n + i] = d;
    }
}

struct DistancePlan {
    int n_blocks, tiles, blocks, unit;
    long units;
};

DistancePlan distance_plan(int sm_count, int n, long pages, int page)
{
    DistancePlan p;
    p.n_blocks = (n + 31) / 32;
    p.tiles = p.n_blocks * (p.n_blocks + 1) / 2;
    // a warp takes 1024 columns of a page at a time; fewer where that would leave warps without work
    p.unit = 1024;
    while (p.unit > 128 && pages * ((page + p.unit - 1) / p.unit) * p.tiles < (long)sm_count * 2 * kWarps) p.unit >>= 1;
    p.units = pages * ((page + p.unit - 1) / p.unit);
    const long want = (p.units + kWarps - 1) / kWarps, most = (sm_count * 2 + p.tiles - 1) / p.tiles;
    p.blocks = (int)(want < most ? want : most);
    if (p.blocks < 1) p.blocks = 1;
    return p;
}

template <int BYTES> void launch_gram(const DistanceArgs &a, const DistancePlan &p, cudaStream_t stream)
{
    const dim3 grid((unsigned)p.tiles, (unsigned)p.blocks);
    if (p.n_blocks > 1) gram_kernel<4, false, BYTES><<<grid, kWarps * 32, 0, stream>>>(a, p.n_blocks);
    else if (a.n > 24) gram_kernel<4, true, BYTES><<<grid, kWarps * 32, 0, stream>>>(a, 1);
    else if (a.n > 16) gram_kernel<3, true, BYTES><<<grid, kWarps * 32, 0, stream>>>(a, 1);
    else if (a.n > 8) gram_kernel<2, true, BYTES><<<grid, kWarps * 32, 0, stream>>>(a, 1);
    else gram_kernel<1, true, BYTES><<<grid, kWarps * 32, 0, stream>>>(a, 1);
}

} // namespace

size_t int8_distances_workspace_bytes(const Context *ctx, int n, long pages, int page)
{
    const DistancePlan p = distance_plan(ctx->sm_count, n, pages, page);
    return (size_t)p.tiles * p.blocks * 1024 * sizeof(double);
}

int int8_distances(Context *ctx, const signed char *codes, long code_stride, const float *scales, long scale_stride, long n_slots, int page,
                   int group, const int *slots, int n, int pages, double *out, void *workspace, cudaStream_t stream)
{
    const DistancePlan p = distance_plan(ctx->sm_count, n, pages, page);
    DistanceArgs a;
    a.codes = codes;
    a.code_stride = code_stride;
    a.scales = scales;
    a.scale_stride = scale_stride;
    a.n_slots = n_slots;
    a.slots = slots;
    a.n = n;
    a.pages = pages;
    a.page = page;
    a.group = group == 0 || group > page ? page : group;
    a.unit = p.unit;
    a.units_per_page = (unsigned)((page + p.unit - 1) / p.unit);
    a.units = (unsigned)p.units;
    a.blocks = p.blocks;
    a.partial = reinterpret_cast<double *>(workspace);
    count_launch("int8_gram", stream, (double)n * pages * page);
    if (a.group % 64 == 0 || a.group == a.page) launch_gram<16>(a, p, stream);
    else launch_gram<8>(a, p, stream);
    LB_CUDA(cudaGetLastError());
    count_launch("int8_distances", stream, 8.0 * n * n);
    distance_finish_kernel<<<(unsigned)(((long)n * n + 7) / 8), 256, 0, stream>>>(a.partial, n, p.n_blocks, p.blocks, out);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

} // namespace lb
