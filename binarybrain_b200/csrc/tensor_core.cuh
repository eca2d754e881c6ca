// The fifth-generation tensor cores as inline PTX for sm_100a: tiled TMA loads, shared-memory descriptors, products of 8-bit integers and of bf16 into TMEM,
// and the bounded waits around them.
//
// Rules kept here: a tiled copy starts on a 16-byte boundary of a row; one thread issues all products and commits of a CTA; every wait has a limit, and
// the first one that runs out sets the CTA's flag, which all others look at, so that no role waits for another that has left.
#pragma once

#include <cuda.h>

#include "async_copy.cuh"

namespace bb200 {

constexpr int kDrainSpins = 1 << 16;

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory"); }

// at most `spins` attempts
__device__ __forceinline__ bool mbar_wait_some(uint64_t *bar, uint32_t parity, int spins)
{
    for (int i = 0; i < spins; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

// One thread's wait: false, with the flag set, when the phase did not complete in time or another thread's did not.
__device__ __forceinline__ bool mbar_wait_one(uint64_t *bar, uint32_t parity, volatile int *gave_up)
{
    for (int i = 0; i < kWaitSpins; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*gave_up) return false;
    }
    *gave_up = 1;
    return false;
}

// the same for a whole warp, with one outcome for all lanes
__device__ __forceinline__ bool mbar_wait_warp(uint64_t *bar, uint32_t parity, volatile int *gave_up)
{
    return __all_sync(0xffffffffu, mbar_wait_one(bar, parity, gave_up));
}

__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

__device__ __forceinline__ void tma_load_2d(void *smem_dst, const CUtensorMap *map, int x, int row, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_addr(smem_dst)), "l"(map), "r"(x), "r"(row), "r"(smem_addr(bar)) : "memory");
}

// the same by one CTA of a pair, whose bytes count at a barrier of either (a cluster address)
__device__ __forceinline__ void tma_load_2d_pair(void *smem_dst, const CUtensorMap *map, int x, int row, uint32_t cluster_bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_addr(smem_dst)), "l"(map), "r"(x), "r"(row), "r"(cluster_bar) : "memory");
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t *smem_out, int columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_out)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_free(uint32_t tmem, int columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// for a pair of CTAs, by a warp of each
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *smem_out, int columns)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_out)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_free_pair(uint32_t tmem, int columns)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

__device__ __forceinline__ void tcgen05_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_fence_after()  { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// the barrier is arrived at when all products issued so far by this thread are done
__device__ __forceinline__ void tcgen05_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// the same for a pair's products: at this place in both CTAs, or in this one alone
__device__ __forceinline__ void tcgen05_commit_pair(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tcgen05_commit_pair_own(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Rows of 128 bytes (k) in groups of eight, 128-byte swizzled, 1024 bytes a group: start address, group distance, version 1, swizzle mode 2.  32 bytes
// of k further on are two units of the address field.
__device__ __forceinline__ uint64_t smem_descriptor_128b(uint32_t addr)
{
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// The same rows along m or n, 64 of them (128 bytes) a row of k, eight rows of k a group of 1024 bytes: 64 further ones lie `next` bytes on.  16 rows of k
// further on are 128 units of the address field.
__device__ __forceinline__ uint64_t smem_descriptor_128b_across(uint32_t addr, uint32_t next)
{
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// what a product of bf16 with sums of 32 bits is told about its operands; across: their rows lie along m or n instead of k
__host__ __device__ constexpr uint32_t mma_bf16_instruction(int m, int n, bool a_across, bool b_across)
{
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_across << 15) | ((uint32_t)b_across << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <bool PAIR> __device__ __forceinline__ void mma_bf16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t instr, bool accumulate)
{
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)accumulate) : "memory");
}

// A warp's own product in registers, 16 rows x 16 of k times 16 of k x 8 columns: for operands that come once and are not worth the way through shared memory.
// Lane 4 g + t has the pairs t and t + 4 of k of rows g and g + 8 (a) and of column g (b), and columns 2 t and 2 t + 1 of those rows of the sums.
__device__ __forceinline__ void mma_rows_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t instr, bool accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)accumulate) : "memory");
}

// both CTAs of a pair, each with half of the rows of either operand at the same place of its shared memory
__device__ __forceinline__ void mma_i8_pair(uint32_t tmem, uint64_t a, uint64_t b, uint32_t instr, bool accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)accumulate) : "memory");
}

// 32 columns of this warp's 32 lanes, complete on return
__device__ __forceinline__ void tmem_load_32(uint32_t tmem, int (&v)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
                 "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(tmem) : "memory");
}

__device__ __forceinline__ void tmem_load_16(uint32_t tmem, int (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(tmem) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t tmem, int (&v)[32]) { tmem_load_32(tmem, v); }
__device__ __forceinline__ void tmem_load(uint32_t tmem, int (&v)[16]) { tmem_load_16(tmem, v); }

__device__ __forceinline__ int4 peer_load_v4(uint32_t own_smem, uint32_t rank)
{
    uint32_t at;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(own_smem), "r"(rank));
    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// cuTensorMapEncodeTiled of the driver, looked up once; null where there is none
using TensorMapEncode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                     const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorMapEncode tensor_map_encode()
{
    static const TensorMapEncode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return reinterpret_cast<TensorMapEncode>(fn);
    }();
    return encode;
}

// Rows of `size` elements as TMA sees them: 128-byte swizzled boxes of 128 bytes x `box_rows` rows; what lies beyond the elements or the rows reads as zero.
// The rows start on 16-byte boundaries.
inline CUresult tensor_map_rows(TensorMapEncode encode, CUtensorMap *map, CUtensorMapDataType type, int element, const void *p, long long size, long long rows,
                                long long stride_bytes, int box_rows)
{
    const cuuint64_t extent[2] = {(cuuint64_t)size, (cuuint64_t)rows}, pitch[1] = {(cuuint64_t)stride_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / element), (cuuint32_t)box_rows}, unit[2] = {1, 1};
    return encode(map, type, 2, const_cast<void *>(p), extent, pitch, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

}   // namespace bb200
