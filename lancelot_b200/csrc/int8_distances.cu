// Squared distances between all pairs of cached 8-bit updates, the plaintext selection rule of the reference's driver
// (lancelot-main-GPU/utils/byzantine_fl.py:162-171, 527-536) without the updates ever being expanded.
//
//   D_ij = |x_i|^2 + |x_j|^2 - 2 <x_i, x_j>,   <x_i, x_j> = sum over groups g of s_ig s_jg (sum of q_ik q_jk inside g)
//
// The inner sums are integer products on the tensor cores and exact; the scales are applied, and the groups added, in 64-bit
// floats, so that the three terms of D_ij may cancel by nine digits before a 32-bit result would suffer.  Two equal updates
// give exactly 0: the same warps add the same numbers in the same order for ii, ij and jj.
//
// A row of A and a column of B are both "a client's codes along k", and the order of k inside a product does not matter as long as
// both sides agree: lane (g, t) of the matrix instruction takes 16 consecutive bytes of client g and uses them as four k-slots of A
// and of B at once, without a transposition.
//
// What was measured on the way (20 x 11 M, groups of 128; 36 us at the copy rate).  m16n8k32 takes 8 cycles of a quarter of the SM, so
// that 20 clients keep it busy for a fifth of the time that their codes take to come in: the warp's own instruction is the right
// one.  tcgen05 took 148 us: one thread issues for all, its results leave TMEM group by group, and a product of few columns costs as
// much as a wide one.  A ring of shared memory filled by a warp of its own took 123 us (a bulk copy or a gathered TMA load of four rows
// holds its warp up for 70 cycles), filled by all warps 96 us (instructions); registers 56 us.  Beyond 32 clients the registers of a
// warp do not hold what it would have to read, and the ring is used after all.
#include <atomic>
#include <type_traits>

#include "tcgen05.cuh"

namespace lb {

namespace {

constexpr int kWarps = 8;

struct DistanceArgs {
    const signed char *codes;
    long code_stride;
    const float *scales;
    long scale_stride;
    long n_slots;
    const int *slots; // [n][pages]; nullptr: in order
    int n, pages, page;
    int group;          // columns of a group; 2^30 for one group in a page
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

// ---- more than 128 clients -------------------------------------------------------------------------------------------------------
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

// More than 128 clients: 32 by 32 of them a block, whose codes come from L2 once for each of the n / 32 blocks they meet.  (The ring below
// keeps the 64-bit sums of all pairs in one block's registers: 20 warps for 128 clients; 160 would take 30 of 64 registers, half of them
// sums.)  Bound by instructions and the latency of loads with two warps a quarter: 200 x 1.6 M takes 605 us with one scale a page, 1.6 ms with
// groups of 64 (64-bit operations of all pairs; 52 us at the copy rate).  At the border, 1.67 M values with one scale a page and with groups
// of 64: 129 clients 305 and 780 us here, 128 clients 142 and 202 us in the ring.
template <int BYTES> __global__ void __launch_bounds__(kWarps * 32) gram_kernel(const DistanceArgs a, const int n_blocks)
{
    __shared__ double sum[32 * 32];
    int i, j;
    tile_of(blockIdx.x, n_blocks, i, j);
    double *out = a.partial + ((size_t)blockIdx.x * a.blocks + blockIdx.y) * 1024;
    if (i == j) gram_tile<4, true, BYTES>(a, i * 32, j * 32, sum, out);
    else gram_tile<4, false, BYTES>(a, i * 32, j * 32, sum, out);
}

// ---- pieces of the kernels for up to 128 clients ----------------------------------------------------------------------------------
constexpr int kRingBytes = 226 * 1024;
constexpr int kSlotStages = 16; // stages whose slots are held; at least twice the ring's

// An integer sum as a 64-bit float, without the conversion unit (which takes 8 cycles for what the FP64 pipe does in 2): sums start
// from -2^31 instead of 0, and 2^52 + 2^31 + x has just those bits below an exponent of 52.
constexpr int kBias = (int)0x80000000;
__device__ __forceinline__ double unbiased(int x) { return __hiloint2double(0x43300000, x) - 4503601774854144.0; }

struct Ring {
    int rows;        // of clients, rounded up to eight: what a stage has room for
    int groups;      // scales of a row in a stage
    int stage_bytes; // codes [rows][pitch], then scales [rows][groups] in 32 bits
    int stages;
    int spare;       // bytes behind the ring that a read of rows beyond `rows` may reach
    int wide;        // bytes of the scales in 64 bits and of the slots
};

// Eight rows of codes at columns `at` of a stage, as four (two) k-slots of the matrix instruction
template <int BYTES> __device__ __forceinline__ void load_rows(unsigned (&w)[BYTES / 4], const unsigned char *at)
{
    if constexpr (BYTES == 16) {
        const uint4 x = *reinterpret_cast<const uint4 *>(at);
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2 *>(at);
        w[0] = x.x;
        w[1] = x.y;
    }
}

__device__ __forceinline__ void apply_scales(double (&total)[4], const int (&acc)[4], double lo, double hi, double2 col)
{
    total[0] += (lo * col.x) * unbiased(acc[0]);
    total[1] += (lo * col.y) * unbiased(acc[1]);
    total[2] += (hi * col.x) * unbiased(acc[2]);
    total[3] += (hi * col.y) * unbiased(acc[3]);
}

// All pairs of up to 32 clients.  The 8 x 8 blocks of pairs that are wanted come in twos: the instruction forms 16 rows against 8
// columns, and block (i, j) serves as (j, i).  Three blocks of clients take three instructions this way instead of four for the
// upper triangle as it stands.
template <int TILES, unsigned LO, unsigned HI, unsigned COL> struct Tiles { // one hexadecimal digit per instruction, the first one last
    static constexpr int kTiles = TILES;
    static constexpr __host__ __device__ int lo(int v) { return LO >> 4 * v & 15; }                                     // block of rows 0 to 7
    static constexpr __host__ __device__ int hi(int v) { return (HI >> 4 * v & 15) == 15 ? -1 : (int)(HI >> 4 * v & 15); } // of rows 8 to 15; f: none
    static constexpr __host__ __device__ int col(int v) { return COL >> 4 * v & 15; }                                   // of the columns
};
template <int NB> struct Cover;
template <> struct Cover<1> : Tiles<1, 0x0, 0xf, 0x0> {};
template <> struct Cover<2> : Tiles<2, 0x00, 0xf1, 0x01> {};
template <> struct Cover<3> : Tiles<3, 0x100, 0x212, 0x210> {};
template <> struct Cover<4> : Tiles<6, 0x103210, 0xff0321, 0x320321> {};

// 16 clients (`codes`, `scales` at the first) with BLOCKS x 8 clients `apart` rows further down: columns [begin, end), one scale each.
// BLOCKS is a constant so that all loads of a step are on their way before its first product.
template <int BYTES, int BLOCKS>
__device__ __forceinline__ void strip(double (&total)[4][4], const unsigned char *codes, const double *scales, int apart, int pitch, int begin, int end)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const unsigned char *at = codes + g * pitch + t * BYTES, *other = at + apart * pitch;
    int acc[BLOCKS][4];
    auto step = [&](int c, auto first) {
        unsigned lo[BYTES / 4], hi[BYTES / 4], b[BLOCKS][BYTES / 4];
        load_rows<BYTES>(lo, at + c);
        load_rows<BYTES>(hi, at + 8 * pitch + c);
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) load_rows<BYTES>(b[j], other + j * 8 * pitch + c);
#pragma unroll
        for (int k = 0; k < BYTES / 4; k += 2)
#pragma unroll
            for (int j = 0; j < BLOCKS; ++j) {
                if (decltype(first)::value && k == 0) mma_s8_from(acc[j], kBias, lo[k], hi[k], lo[k + 1], hi[k + 1], b[j][k], b[j][k + 1]);
                else mma_s8(acc[j], lo[k], hi[k], lo[k + 1], hi[k + 1], b[j][k], b[j][k + 1]);
            }
    };
    step(begin, std::true_type());
    for (int c = begin + 4 * BYTES; c < end; c += 4 * BYTES) step(c, std::false_type());
    const double lo = scales[g], hi = scales[8 + g];
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) apply_scales(total[j], acc[j], lo, hi, *reinterpret_cast<const double2 *>(scales + apart + j * 8 + t * 2));
}

// ---- up to 32 clients: no shared memory ----------------------------------------------------------------------------------------
// A warp takes a unit of a page's columns, CHUNK columns at a time, the next ones on their way in registers while these are multiplied.
// 16 warps an SM, none of which waits for another: 20 x 11 M in 56 us (4.2 TB/s), of which some 8 us are the first loads, the sums of the
// blocks and the second kernel.  More bytes on their way would take more registers; loads that also bring the next chunk into L2 gained
// 6 us of the 62.  Above 24 clients the sums leave room for 8 warps: 32 x 11 M in 136 us, 156 us with half the columns a chunk; scales
// applied at the end of a group of several chunks gained 12 us there with one scale a page and cost up to 12 us below.  A client
// that is not there (or a page of one) is read as the cache's first slot with scales of 0, so that no load needs a condition.

// 16 bytes of codes; the 256 bytes around them are brought into L2, for the next chunk
__device__ __forceinline__ uint4 load_and_next(const signed char *at)
{
    uint4 x;
    asm volatile("ld.global.nc.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(at));
    return x;
}

template <int NB, int BYTES, int CHUNK, int GROUPS> // GROUPS: scales of a chunk
__global__ void __launch_bounds__(kWarps * 32, NB == 4 ? 1 : 2) gram_direct_kernel(const DistanceArgs a)
{
    using V = Cover<NB>;
    constexpr int STEP = BYTES * 4, STEPS = CHUNK / STEP, W = BYTES / 4;
    __shared__ double sum[NB * 8][NB * 8];
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
    const int log_group = 31 - __clz(a.group), code_stride = (int)a.code_stride, scale_stride = (int)a.scale_stride;
    double total[V::kTiles][4];
#pragma unroll
    for (int v = 0; v < V::kTiles; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[v][e] = 0.0;

    // where the next chunk lies
    const unsigned stride = a.blocks * kWarps;
    unsigned u = blockIdx.x * kWarps + warp;
    int at = 0, end = 0; // columns of the page
    int entry[NB], slot[NB];
    const signed char *src[NB];
    const float *scl[NB];
    unsigned there = 0;
#pragma unroll
    for (int r = 0; r < NB; ++r) entry[r] = min(r * 8 + g, a.n - 1) * a.pages;
    auto look_up = [&](unsigned unit) {
        const int page = (int)(min(unit, a.units - 1) / a.units_per_page);
        if (a.slots) { // (not a choice for each slot: that would wait for it)
#pragma unroll
            for (int r = 0; r < NB; ++r) slot[r] = __ldg(a.slots + entry[r] + page);
        } else {
#pragma unroll
            for (int r = 0; r < NB; ++r) slot[r] = entry[r] + page;
        }
    };
    auto enter = [&]() {
        there = 0;
        at = (int)(u % a.units_per_page) * a.unit;
        end = min(at + a.unit, a.page);
#pragma unroll
        for (int r = 0; r < NB; ++r) {
            const bool is = r * 8 + g < a.n && (unsigned)slot[r] < (unsigned)a.n_slots;
            there |= (unsigned)is << r;
            const int s = is ? slot[r] : 0;
            src[r] = a.codes + (long)s * code_stride + t * BYTES;
            scl[r] = a.scales + (long)s * scale_stride;
        }
        look_up(u + stride); // on their way while this unit is multiplied
    };
    struct Chunk {
        unsigned w[NB][STEPS][W];
        float s[NB][GROUPS];
    };
    auto load = [&](Chunk &k) {
        const bool whole = at + CHUNK <= end;
#pragma unroll
        for (int r = 0; r < NB; ++r) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const bool inside = whole || at + i * STEP + t * BYTES < end;
                if constexpr (BYTES == 16) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (inside) x = load_and_next(src[r] + at + i * STEP);
                    k.w[r][i][0] = x.x;
                    k.w[r][i][1] = x.y;
                    k.w[r][i][2] = x.z;
                    k.w[r][i][3] = x.w;
                } else {
                    uint2 x = make_uint2(0, 0);
                    if (inside) x = __ldg(reinterpret_cast<const uint2 *>(src[r] + at + i * STEP));
                    k.w[r][i][0] = x.x;
                    k.w[r][i][1] = x.y;
                }
            }
#pragma unroll
            for (int q = 0; q < GROUPS; ++q) {
                k.s[r][q] = 0.f;
                if ((there >> r & 1) && (q == 0 || at + q * (CHUNK / GROUPS) < end)) k.s[r][q] = __ldg(scl[r] + (at >> log_group) + q);
            }
        }
        at += CHUNK;
        if (at >= end) {
            u += stride;
            if (u < a.units) enter();
        }
    };
    auto multiply = [&](const Chunk &k) {
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            int acc[V::kTiles][4];
#pragma unroll
            for (int i = q * STEPS / GROUPS; i < (q + 1) * STEPS / GROUPS; ++i)
#pragma unroll
                for (int j = 0; j < W; j += 2)
#pragma unroll
                    for (int v = 0; v < V::kTiles; ++v) {
                        const int lo = V::lo(v), hi = V::hi(v) >= 0 ? V::hi(v) : 0, col = V::col(v);
                        const unsigned h0 = V::hi(v) >= 0 ? k.w[hi][i][j] : 0, h1 = V::hi(v) >= 0 ? k.w[hi][i][j + 1] : 0;
                        if (i == q * STEPS / GROUPS && j == 0) mma_s8_from(acc[v], kBias, k.w[lo][i][j], h0, k.w[lo][i][j + 1], h1, k.w[col][i][j], k.w[col][i][j + 1]);
                        else mma_s8(acc[v], k.w[lo][i][j], h0, k.w[lo][i][j + 1], h1, k.w[col][i][j], k.w[col][i][j + 1]);
                    }
            // accumulator e of a lane: row g (+ 8 for e >= 2) of A, column 2 t + (e & 1) of B
            double row[NB];
            double2 col[NB];
#pragma unroll
            for (int r = 0; r < NB; ++r) {
                row[r] = k.s[r][q];
                col[r].x = __shfl_sync(0xffffffffu, k.s[r][q], t * 8);
                col[r].y = __shfl_sync(0xffffffffu, k.s[r][q], t * 8 + 4);
            }
#pragma unroll
            for (int v = 0; v < V::kTiles; ++v) apply_scales(total[v], acc[v], row[V::lo(v)], V::hi(v) >= 0 ? row[V::hi(v) >= 0 ? V::hi(v) : 0] : 0.0, col[V::col(v)]);
        }
    };

    look_up(u);
    if (u < a.units) {
        enter();
        Chunk one, two;
        load(one);
        while (true) {
            const bool more = u < a.units;
            if (more) load(two);
            multiply(one);
            if (!more) break;
            const bool again = u < a.units;
            if (again) load(one);
            multiply(two);
            if (!again) break;
        }
    }
    // the block's warps one after the other: the order of the additions is fixed
    for (int k = 0; k < kWarps; ++k) {
        if (warp == k) {
#pragma unroll
            for (int v = 0; v < V::kTiles; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int block = e < 2 ? V::lo(v) : V::hi(v);
                    if (block < 0) continue;
                    const int x = block * 8 + g, y = V::col(v) * 8 + t * 2 + (e & 1);
                    if (block == V::col(v) && x > y) continue;
                    double *to = &sum[min(x, y)][max(x, y)];
                    *to = k ? *to + total[v][e] : total[v][e];
                }
        }
        __syncthreads();
    }
    constexpr int kRows = NB * 8;
    double *out = a.partial + (size_t)blockIdx.x * (kRows * kRows + kRows);
    for (int i = threadIdx.x; i < kRows * kRows; i += kWarps * 32) {
        const int x = i / kRows, y = i % kRows;
        if (x <= y) {
            out[i] = sum[x][y];
            if (x == y) out[kRows * kRows + x] = sum[x][x];
        }
    }
}

// ---- up to 128 clients: a ring of shared memory --------------------------------------------------------------------------------
// One CTA per SM.  All its warps together copy the codes and scales of some hundred columns of all clients into the ring, several stages
// ahead (cp.async; one barrier a stage), and each warp multiplies 16 clients with 32.  Rows lie 64 bytes off a multiple of 128 apart, so
// that the 16-byte loads of eight rows fall on different banks.
//
// Bound by the warps' own work, which is most of the time even without the copies: 100 x 1.6 M takes 94 us with one scale a page, 147 us
// with groups of 64 (26 us at the copy rate).  Each group costs three 64-bit operations a pair and group, 50 us at their rate; a step's six
// 512-byte rows of loads and up to eight products wait for one another.  Stages of 256 columns took 124, 161 us, loads next to their products
// 142, 186 us; 32 by 32 clients a warp, which read less, left too few warps (162, 219 us); a barrier for each stage and warp instead of one
// for all took 152, 245 us.
//
// NB: blocks of eight clients: 8, 12 or 16.  SETS warps split the columns of a stage, 2^LOG_UNIT, for the same pairs.  Sizes are constants
// because divisions by a unit of run-time size took more instructions than all the rest.
template <int NB, int LOG_UNIT, int BYTES, int WARPS, int SETS>
__global__ void __launch_bounds__(WARPS * 32, 1) gram_ring_kernel(const DistanceArgs a, const Ring r)
{
    constexpr int kThreads = WARPS * 32;
    constexpr int kUnit = 1 << LOG_UNIT, kPitch = kUnit + 64, kWide = NB * 8;
    constexpr int kLanes = kUnit < 512 ? kUnit / 16 : 32;                         // that copy one row together
    constexpr int kRowsACopy = 32 / kLanes, kCopiesARow = kUnit / (kLanes * 16); // of a warp
    constexpr int kFill = (kWide / kRowsACopy * kCopiesARow + WARPS - 1) / WARPS; // copies that a warp makes for one stage, at most
    extern __shared__ __align__(128) unsigned char ring[];
    double *wide_scales = reinterpret_cast<double *>(ring + r.stages * r.stage_bytes + r.spare); // [2][groups][kWide]: of this stage and the next
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int code_bytes = r.rows * kPitch;
    const int log_group = 31 - __clz(a.group), log_groups = 31 - __clz(r.groups), scales_a_stage = a.n << log_groups;

    // where a unit lies; units are taken in turn by the CTAs
    const int page_step = (int)(gridDim.x / a.units_per_page), part_step = (int)(gridDim.x % a.units_per_page);
    struct Place {
        int page, begin;
    };
    auto advance = [&](Place &p) {
        p.page += page_step;
        p.begin += part_step << LOG_UNIT;
        if (p.begin >= a.page) {
            ++p.page;
            p.begin -= (int)a.units_per_page << LOG_UNIT;
        }
    };
    Place now = {(int)(blockIdx.x / a.units_per_page), (int)(blockIdx.x % a.units_per_page) << LOG_UNIT};
    Place ahead = now; // the next unit to be copied

    // What this thread copies of every stage: 16 bytes of the same columns of every kRowsApart-th row, some scales, and the slots of a stage
    // further on, so that these are in shared memory when that stage is copied
    static_assert(WARPS % kCopiesARow == 0, "a warp's copies are of the same columns");
    constexpr int kRowsApart = WARPS / kCopiesARow * kRowsACopy;
    const int first_row = warp / kCopiesARow * kRowsACopy + lane / kLanes, column = warp % kCopiesARow * 512 + lane % kLanes * 16;
    const unsigned first_to = smem_u32(ring) + first_row * kPitch + column;
    const int n_slots = (int)a.n_slots, code_stride = (int)a.code_stride, scale_stride = (int)a.scale_stride;
    int *slots = reinterpret_cast<int *>(wide_scales + 2 * r.groups * kWide); // [kSlotStages][kWide]
    auto look_up = [&](int page, int at) { // entry `at` of the slots
        const int i = (int)threadIdx.x * a.pages + min(page, a.pages - 1);
        if ((int)threadIdx.x < a.n) {
            if (a.slots) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(slots + at * kWide + threadIdx.x)), "l"(a.slots + i));
            else slots[at * kWide + threadIdx.x] = i;
        }
    };
    auto fill = [&](const Place &p, int stage, int at) { // a page that is not there leaves old codes, and scales of 0
        if (p.page < a.pages) {
            const int *slot = slots + at * kWide;
            const unsigned to = first_to + stage * r.stage_bytes;
            const signed char *from = a.codes + p.begin + column;
            const bool inside = p.begin + column < a.page;
#pragma unroll
            for (int k = 0; k < kFill; ++k) {
                const int row = first_row + k * kRowsApart;
                if (row >= a.n) break;
                const int here = slot[row];
                if ((unsigned)here < (unsigned)n_slots) {
                    if (inside) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * kRowsApart * kPitch), "l"(from + (long)here * code_stride));
                    else asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(to + k * kRowsApart * kPitch), "r"(0) : "memory"); // behind the page's end
                }
            }
            const unsigned scales_to = smem_u32(ring) + stage * r.stage_bytes + code_bytes;
            for (int i = threadIdx.x; i < scales_a_stage; i += kThreads) {
                const int q = (p.begin >> log_group) + (i & (r.groups - 1)), here = slot[i >> log_groups];
                const bool there = (unsigned)here < (unsigned)n_slots && (long)q << log_group < a.page;
                const float *src = there ? a.scales + (long)here * scale_stride + q : a.scales;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(scales_to + i * 4), "l"(src), "r"(there ? 4 : 0));
            }
        }
    };
    auto commit = [&]() { asm volatile("cp.async.commit_group;" ::: "memory"); };
    auto widen = [&](int stage, int parity) { // a stage's scales as 64-bit floats, [group][client]
        const float *from = reinterpret_cast<const float *>(ring + (size_t)stage * r.stage_bytes + code_bytes);
        double *to = wide_scales + parity * r.groups * kWide;
        for (int i = threadIdx.x; i < scales_a_stage; i += kThreads) to[(i & (r.groups - 1)) * kWide + (i >> log_groups)] = from[i];
    };

    // the pairs of this warp: 16 rows from row0 on with up to 32 from col0 on; two warps make a pair of groups
    const int set = warp % SETS, pair = warp / SETS / 2, half = (warp / SETS & 1) ^ (NB == 8 ? pair >> 1 & 1 : pair >> 2 & 1); // (the quarters of
    int row0 = 0, col0 = pair;                                                    // an SM, warps modulo 4, get equal numbers of products this way)
    constexpr int kGroups = NB / 4;
    while (col0 >= kGroups - row0) col0 -= kGroups - row0++;
    const bool same = col0 == 0; // a group with itself: the lower half has nothing to do with the upper
    col0 = (row0 + col0) * 32 + (same ? half * 16 : 0);
    row0 = row0 * 32 + half * 16;
    const int col_blocks = min(same && half ? 2 : 4, (a.n - col0 + 7) / 8);
    constexpr int kPer = kUnit / SETS; // columns of a warp
    const int step = min(a.group, kPer);
    double total[4][4];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[v][e] = 0.0;

    // The slots of unit u stand at u % kSlotStages.  They come with the copies of unit u - (stages - 1), which are complete when
    // unit u is copied; those of the first units are waited for here
    Place looked = now;
    int look_at = 0, fill_at = 0;
    auto look_further = [&]() {
        look_up(looked.page, look_at);
        advance(looked);
        look_at = (look_at + 1) % kSlotStages;
    };
    for (int u = 0; u < r.stages - 1; ++u) look_further();
    commit();
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    for (int s = 0; s < r.stages - 1; ++s) {
        fill(ahead, s, fill_at);
        fill_at = (fill_at + 1) % kSlotStages;
        advance(ahead);
        look_further();
        commit();
    }
    // a stage and the next one have come in when all but the last stages - 3 copies have
    auto wait = [&]() {
        switch (r.stages) {
        case 3: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 5: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 6: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        case 7: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
        }
    };
    wait();
    __syncthreads();
    widen(0, 0);
    int s = 0, parity = 0;
    for (; now.page < a.pages; advance(now)) {
        wait();
        __syncthreads(); // this stage and the next have come in, the last one has been read
        const int next = s + 1 == r.stages ? 0 : s + 1;
        fill(ahead, s ? s - 1 : r.stages - 1, fill_at);
        fill_at = (fill_at + 1) % kSlotStages;
        advance(ahead);
        look_further();
        commit();
        widen(next, parity ^ 1); // (behind the last unit: old scales, and nobody reads them)
        const int columns = min(kUnit, a.page - now.begin);
        const unsigned char *codes = ring + (size_t)s * r.stage_bytes;
        const int to = min((set + 1) * kPer, columns);
        const double *scales = wide_scales + parity * r.groups * kWide;
        auto all = [&](auto blocks) {
            for (int c = set * kPer; c < to; c += step) {
                const double *sc = scales + (c >> log_group) * kWide; // a stage begins where a group does, or has only one
                strip<BYTES, decltype(blocks)::value>(total, codes + row0 * kPitch, sc + row0, col0 - row0, kPitch, c, c + step);
            }
        };
        switch (col_blocks) {
        case 4: all(std::integral_constant<int, 4>()); break;
        case 3: all(std::integral_constant<int, 3>()); break;
        case 2: all(std::integral_constant<int, 2>()); break;
        case 1: all(std::integral_constant<int, 1>()); break;
        }
        s = next;
        parity ^= 1;
    }
    // the ring's memory takes the sums now; the order in which the warps of a set add them up is fixed
    asm volatile("cp.async.wait_all;" ::: "memory");
    double *sums = reinterpret_cast<double *>(ring);
    const int g = lane >> 2, t = lane & 3;
    for (int k = 0; k < SETS; ++k) {
        __syncthreads();
        if (set != k) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int x = row0 + (e >> 1) * 8 + g, y = col0 + j * 8 + t * 2 + (e & 1);
                if (j >= col_blocks || x > y) continue;
                double *at = sums + x * kWide + y;
                *at = k ? *at + total[j][e] : total[j][e];
            }
    }
    __syncthreads();
    double *out = a.partial + (size_t)blockIdx.x * (kWide * kWide + kWide);
    for (int i = threadIdx.x; i < kWide * kWide; i += kThreads) {
        const int x = i / kWide, y = i - x * kWide;
        if (x <= y && y < a.n) {
            out[i] = sums[i];
            if (x == y) out[kWide * kWide + x] = sums[i];
        }
    }
}

// A block per row i: the sums of all blocks, then the distances of row i.  LANES clients side by side, and as many slices of the blocks
// as the 1024 threads give, the same ones for every sum
template <int LANES>
__global__ void __launch_bounds__(1024) distance_rows_kernel(const double *__restrict__ partial, const int n, const int rows, const int blocks, double *__restrict__ out)
{
    constexpr int kSlices = 1024 / LANES;
    __shared__ double dots[kSlices][LANES], norms[kSlices][LANES];
    const int i = blockIdx.x, j = threadIdx.x % LANES, slice = threadIdx.x / LANES;
    const long pitch = (long)rows * rows + rows;
    double dot = 0.0, norm = 0.0;
    if (j < n) {
        const double *p = partial + (long)min(i, j) * rows + max(i, j), *q = partial + (long)rows * rows + j;
#pragma unroll 8
        for (int b = slice; b < blocks; b += kSlices) {
            dot += p[b * pitch];
            norm += q[b * pitch];
        }
    }
    dots[slice][j] = dot;
    norms[slice][j] = norm;
    __syncthreads();
    for (int half = kSlices / 2; half; half /= 2) {
        if (slice < half) {
            dots[slice][j] += dots[slice + half][j];
            norms[slice][j] += norms[slice + half][j];
        }
        __syncthreads();
    }
    if (slice || j >= n) return;
    const double x = norms[0][i], y = norms[0][j], z = dots[0][j], d = (x - z) + (y - z);
    out[(long)i * n + j] = i == j ? 0.0 : d < 0.0 ? 0.0 : d; // below 0: rounding of nearly equal updates; NaN stays
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
    int n_blocks, tiles, blocks; // gram_kernel: blocks of 32 clients, pairs of them, blocks per pair
    int unit, least_unit;        // columns taken at a time
    int rows;                          // gram_ring_kernel: its rows; 0: gram_kernel
    long units;
    size_t bytes;
};

Ring ring_shape(int blocks, int unit, int n, int group) // blocks of eight clients
{
    Ring r;
    r.rows = (n + 7) / 8 * 8;
    r.groups = group < unit ? unit / group : 1;
    r.stage_bytes = (r.rows * (unit + 64) + r.rows * r.groups * 4 + 127) / 128 * 128;
    r.spare = r.rows % 16 * (unit + 64); // a warp reads 16 rows from a multiple of 16 below n on
    r.wide = 2 * r.groups * blocks * 8 * 8 + kSlotStages * blocks * 8 * 4;
    r.stages = (kRingBytes - r.spare - r.wide) / r.stage_bytes;
    if (r.stages > 8) r.stages = 8;
    return r;
}

// A smaller group never takes larger units, nor fewer blocks
DistancePlan distance_plan(int sm_count, int n, long pages, int page, int group)
{
    DistancePlan p;
    p.n_blocks = (n + 31) / 32;
    p.tiles = p.n_blocks * (p.n_blocks + 1) / 2;
    p.rows = n <= 32 ? (n + 7) / 8 * 8 : n <= 128 ? (n + 31) / 32 * 32 : 0;
    // what a warp (gram_ring_kernel: a CTA) takes at a time: as much as leaves all of them work
    const bool ring = n > 32 && n <= 128;
    const int warp_blocks = p.rows ? (p.rows == 32 ? 1 : 2) * sm_count : (2 * sm_count + p.tiles - 1) / p.tiles;
    const long takers = ring ? sm_count : (long)warp_blocks * kWarps;
    p.unit = !ring ? 1024 : ring_shape(p.rows / 8, 512, n, group).stages >= 3 ? 512 : 256; // of 100 x 1.6 M: 153 us with 512, 161 us with 256
    p.least_unit = !ring ? 128 : 256;
    while (p.unit > p.least_unit && pages * ((page + p.unit - 1) / p.unit) < takers) p.unit >>= 1;
    p.units = pages * ((page + p.unit - 1) / p.unit);
    if (p.rows) {
        const long want = ring ? p.units : (p.units + kWarps - 1) / kWarps, most = ring ? sm_count : warp_blocks;
        p.blocks = (int)(want < most ? want : most);
        if (p.blocks < 1) p.blocks = 1;
        p.bytes = (size_t)p.blocks * (p.rows * p.rows + p.rows) * sizeof(double);
    } else {
        const long want = (p.units + kWarps - 1) / kWarps, most = (sm_count * 2 + p.tiles - 1) / p.tiles;
        p.blocks = (int)(want < most ? want : most);
        if (p.blocks < 1) p.blocks = 1;
        p.bytes = (size_t)p.tiles * p.blocks * 1024 * sizeof(double);
    }
    return p;
}

template <int NB, int LOG_UNIT, int BYTES, int WARPS, int SETS> int launch_ring(Context *ctx, const DistanceArgs &a, const DistancePlan &p, cudaStream_t stream)
{
    const Ring r = ring_shape(NB, 1 << LOG_UNIT, a.n, a.group);
    static std::atomic<bool> set[64]; // host threads that come here first at once all set the same attribute
    if (ctx->device >= 64 || !set[ctx->device]) {
        LB_CUDA(cudaFuncSetAttribute(gram_ring_kernel<NB, LOG_UNIT, BYTES, WARPS, SETS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
        if (ctx->device < 64) set[ctx->device] = true;
    }
    gram_ring_kernel<NB, LOG_UNIT, BYTES, WARPS, SETS><<<p.blocks, WARPS * 32, r.stages * r.stage_bytes + r.spare + r.wide, stream>>>(a, r);
    return LB_OK;
}

template <int NB, int BYTES, int CHUNK> int launch_direct(const DistanceArgs &a, const DistancePlan &p, cudaStream_t stream)
{
    if constexpr (BYTES == 8) {
        gram_direct_kernel<NB, 8, CHUNK, CHUNK / 32><<<p.blocks, kWarps * 32, 0, stream>>>(a);
    } else if constexpr (CHUNK == 256) {
        if (a.group < 128) gram_direct_kernel<NB, 16, CHUNK, 4><<<p.blocks, kWarps * 32, 0, stream>>>(a);
        else if (a.group < CHUNK) gram_direct_kernel<NB, 16, CHUNK, 2><<<p.blocks, kWarps * 32, 0, stream>>>(a);
        else gram_direct_kernel<NB, 16, CHUNK, 1><<<p.blocks, kWarps * 32, 0, stream>>>(a);
    } else {
        if (a.group < CHUNK) gram_direct_kernel<NB, 16, CHUNK, 2><<<p.blocks, kWarps * 32, 0, stream>>>(a);
        else gram_direct_kernel<NB, 16, CHUNK, 1><<<p.blocks, kWarps * 32, 0, stream>>>(a);
    }
    return LB_OK;
}

template <int BYTES> int launch_gram(Context *ctx, const DistanceArgs &a, const DistancePlan &p, cudaStream_t stream)
{
    const bool small = p.unit == p.least_unit;
    switch (p.rows / 8) {
    case 1: return launch_direct<1, BYTES, 256>(a, p, stream);
    case 2: return launch_direct<2, BYTES, BYTES == 8 ? 128 : 256>(a, p, stream);
    case 3: return launch_direct<3, BYTES, 128>(a, p, stream);
    case 4: return launch_direct<4, BYTES, BYTES == 8 ? 64 : 128>(a, p, stream);
    case 8: return small ? launch_ring<8, 8, BYTES, 12, 2>(ctx, a, p, stream) : launch_ring<8, 9, BYTES, 12, 2>(ctx, a, p, stream); // three pairs of groups of 32, two warps each
    case 12: return small ? launch_ring<12, 8, BYTES, 12, 1>(ctx, a, p, stream) : launch_ring<12, 9, BYTES, 12, 1>(ctx, a, p, stream); // six
    case 16: return small ? launch_ring<16, 8, BYTES, 20, 1>(ctx, a, p, stream) : launch_ring<16, 9, BYTES, 20, 1>(ctx, a, p, stream); // ten
    }
    gram_kernel<BYTES><<<dim3((unsigned)p.tiles, (unsigned)p.blocks), kWarps * 32, 0, stream>>>(a, p.n_blocks);
    return LB_OK;
}

} // namespace

size_t int8_distances_workspace_bytes(const Context *ctx, int n, long pages, int page) { return distance_plan(ctx->sm_count, n, pages, page, 32).bytes; }

int int8_distances(Context *ctx, const signed char *codes, long code_stride, const float *scales, long scale_stride, long n_slots, int page,
                   int group, const int *slots, int n, int pages, double *out, void *workspace, cudaStream_t stream)
{
    if (n_slots == 0) pages = 0; // no page is there: all distances are 0
    if (n == 1 || pages == 0) {
        LB_CUDA(cudaMemsetAsync(out, 0, (size_t)n * n * sizeof(double), stream));
        return LB_OK;
    }
    if (group == 0 || group >= page) group = 1 << 30;
    const DistancePlan p = distance_plan(ctx->sm_count, n, pages, page, group);
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
    a.group = group;
    a.unit = p.unit;
    a.units_per_page = (unsigned)((page + p.unit - 1) / p.unit);
    a.units = (unsigned)p.units;
    a.blocks = p.blocks;
    a.partial = reinterpret_cast<double *>(workspace);
    count_launch("int8_gram", stream, (double)n * pages * page);
    // 16 bytes a lane cover 64 columns, which have to share their scale; 8 bytes cover 32
    int rc = a.group % 64 == 0 ? launch_gram<16>(ctx, a, p, stream) : launch_gram<8>(ctx, a, p, stream);
    if (rc) return rc;
    LB_CUDA(cudaGetLastError());
    count_launch("int8_distances", stream, 8.0 * n * n);
    if (p.rows && n <= 32) distance_rows_kernel<32><<<n, 1024, 0, stream>>>(a.partial, n, p.rows, p.blocks, out);
    else if (p.rows) distance_rows_kernel<128><<<n, 1024, 0, stream>>>(a.partial, n, p.rows, p.blocks, out);
    else distance_finish_kernel<<<(unsigned)(((long)n * n + 7) / 8), 256, 0, stream>>>(a.partial, n, p.n_blocks, p.blocks, out);
    LB_CUDA(cudaGetLastError());
    return LB_OK;
}

} // namespace lb
