// What the kernels on Blackwell's tensor memory share: bounded mbarrier waits, TMA loads, tcgen05 in its 8-bit integer and 8-bit floating-point forms.
#pragma once
#include <cuda.h>

#include <atomic>

#include "context.h"

namespace lb {

namespace {

// the warp's own matrix instruction, for operands that stay in registers
__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same, starting from `c` in all four accumulators
__device__ __forceinline__ void mma_s8_from(int (&d)[4], int c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c));
}

constexpr long long kWaitCycles = 4000000000ll; // a wait gives up after some two seconds

__device__ __forceinline__ unsigned smem_u32(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity)
{
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done;
}
// false: the wait ran out, here or in another warp of the block
__device__ __noinline__ bool mbar_wait_slow(unsigned bar, unsigned parity, volatile int *failed)
{
    const long long began = clock64();
    while (!*failed) {
        for (int i = 0; i < 64; ++i)
            if (mbar_try(bar, parity)) return true;
        if (clock64() - began > kWaitCycles) {
            *failed = 1;
            break;
        }
    }
    return false;
}
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int *failed)
{
    for (int i = 0; i < 16; ++i)
        if (mbar_try(bar, parity)) return true;
    return mbar_wait_slow(bar, parity, failed);
}
// the same without a call, for warps whose registers are full
__device__ __forceinline__ bool mbar_wait_inline(unsigned bar, unsigned parity, volatile int *failed)
{
    if (mbar_try(bar, parity)) return true;
    const long long began = clock64();
    while (!mbar_try(bar, parity)) {
        if (*failed) return false;
        if (clock64() - began > kWaitCycles) {
            *failed = 1;
            return false;
        }
    }
    return true;
}
// the same for a whole warp
__device__ __forceinline__ bool mbar_wait_warp(unsigned bar, unsigned parity, volatile int *failed)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, failed));
}
__device__ __forceinline__ void tma_load(unsigned dst, const CUtensorMap *map, int x, int y, unsigned bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap *map, int x, int y, unsigned src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// rows of 128 bytes, 128-byte swizzle: groups of eight rows 1024 bytes apart
__device__ __forceinline__ unsigned long long operand_desc(unsigned addr)
{
    return (unsigned long long)((addr & 0x3ffff) >> 4) | 1ull << 16 | (unsigned long long)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// The same bytes with the summed axis across the rows: a row holds 128 places along the other axis, eight rows (of the summed axis) lie 1024 bytes
// before the next eight; runs of 128 places are `run` bytes apart
__device__ __forceinline__ unsigned long long operand_desc_across(unsigned addr, unsigned run)
{
    return (unsigned long long)((addr & 0x3ffff) >> 4) | (unsigned long long)(run >> 4) << 16 | (unsigned long long)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// One lane issues (`elected`, from elect_one), but the whole warp comes here, and without divergence: the operands are uniform
// registers, which the compiler only uses where the warp provably stays together.
__device__ __forceinline__ unsigned elect_one()
{
    unsigned is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is;
}
__device__ __forceinline__ void mma_i8(unsigned elected, unsigned d, unsigned long long a, unsigned long long b, unsigned desc, bool add)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(desc), "r"((unsigned)add), "r"(elected)
                 : "memory");
}
__device__ __forceinline__ void mma_f8(unsigned elected, unsigned d, unsigned long long a, unsigned long long b, unsigned desc, bool add)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(desc), "r"((unsigned)add), "r"(elected)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned elected, unsigned bar)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(elected) : "memory");
}
__device__ __forceinline__ void tmem_load32(unsigned addr, int (&v)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
                   "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
                   "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(addr)
                 : "memory");
}
// The same in two steps, so that the next columns are on their way while these are used: tmem_ready names the values that it waits for, so that
// none is used before
// 16 lanes of 32 columns: of eight columns, lane l of the warp gets two (2 (l % 4) on) of rows l / 4 and l / 4 + 8
__device__ __forceinline__ void tmem_begin_tiles(unsigned addr, int (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_begin(unsigned addr, int (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_begin(unsigned addr, int (&v)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ready(int (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ready(int (&v)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Rows of `cols` bytes, `stride` apart, in boxes of box_cols bytes x box_rows with a 128-byte swizzle; outside the matrix lie zeros.
// size: bytes of an element, which coordinates count in
inline int encode_map(CUtensorMap *map, const void *base, long rows, long cols, long stride, int box_cols, int box_rows, int size = 1)
{
    static std::atomic<EncodeTiled> known; // host threads that come here first at once all find the same function
    EncodeTiled encode = known;
    if (!encode) {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        LB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !f) {
            set_error("the driver has no cuTensorMapEncodeTiled");
            return LB_ERR_CUDA;
        }
        known = encode = reinterpret_cast<EncodeTiled>(f);
    }
    const cuuint64_t dims[2] = {(cuuint64_t)(cols / size), (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)(box_cols / size), (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUresult r = encode(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
        return LB_ERR_CUDA;
    }
    return LB_OK;
}

} // namespace

} // namespace lb
