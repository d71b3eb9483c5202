// Fifth-generation tensor cores in inline PTX: barriers in shared memory, tensor memory, 16-bit products of tiles in shared memory
// (fp32 accumulators), and the layout of the tiles.
//
// A tile in shared memory is made of blocks of 64 elements (128 bytes) wide rows; the 16-byte pieces of row r of a block stand at places
// piece ^ (r % 8), so that neither rows nor columns of pieces meet in one bank (the hardware's 128-byte swizzle).  A block read along its
// rows ("K-major") has rows = the index that is kept and columns = the index that is summed; read the other way ("MN-major") it is
// the transpose.  Blocks start on 1024 bytes.
#pragma once

#include "common.cuh"

namespace dynb {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ uint64_t timer_ns()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits at most two seconds for the phase; false when they have passed.  All lanes of a warp call it and get the same answer, which the compiler can
// see from the vote: what follows stays uniform, and with it the operands of the products.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity)
{
    uint64_t from = 0;
    for (uint32_t i = 0; i < (1u << 30); i++) {
        if (__all_sync(0xffffffffu, bar_try(bar, parity))) return true;
        if ((i & 1023u) != 1023u) continue;
        const uint64_t now = timer_ns();
        if (from == 0) from = now;
        if (__any_sync(0xffffffffu, now - from > 2000000000ull)) return false;
    }
    return false;
}
// The number of this warp, and one of its lanes, in ways that the compiler knows to be uniform.
__device__ __forceinline__ int warp_number() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
__device__ __forceinline__ bool elected()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// What this thread wrote to shared memory becomes visible to the tensor cores.
__device__ __forceinline__ void fence_to_tensor() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Tensor memory: `columns` a power of two from 32 to 512; the whole warp calls these.
__device__ __forceinline__ void tensor_alloc(uint32_t* at, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tensor_free(uint32_t at, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}

// 32 columns of this warp's 32 lanes of tensor memory (warp w of a group of four reads lanes 32 (w % 4) and on): lane l gets row l.
__device__ __forceinline__ void tensor_load_32(uint32_t at, uint32_t (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(at));
}
__device__ __forceinline__ void tensor_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// d (+)= a b: 128 rows, `n` columns from the descriptor of the instruction, 16 summed elements.  One thread issues it.
__device__ __forceinline__ void tensor_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(what), "r"((uint32_t)add)
        : "memory");
}
// The same, keeping the tile of `a` at the multipliers for the next product with it (KEEP 1: from shared memory, 2: kept before, 3: kept before
// and not after).
template <int KEEP>
__device__ __forceinline__ void tensor_mma_keep(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add)
{
    if constexpr (KEEP == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(what), "r"((uint32_t)add)
                     : "memory");
    else if constexpr (KEEP == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16.collector::a::use [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(what), "r"((uint32_t)add)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                     "l"(b), "r"(what), "r"((uint32_t)add)
                     : "memory");
}
// The barrier gets one arrival when all products issued so far by this thread are done.
__device__ __forceinline__ void tensor_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// 128 x n products of fp16 (or bf16) tiles in fp32; `columns`: both operands are read along their columns (MN-major).
__host__ __device__ constexpr uint32_t mma_what(bool bf16, int n, bool a_columns, bool b_columns)
{
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_columns ? 1u : 0u) << 15) | ((b_columns ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// Descriptor of an operand of blocks of 128-byte rows with the 128-byte swizzle.  Read along rows: `lead` is not used (1), `stride` is the
// distance of groups of eight rows (1024).  Read along columns: `lead` is the distance of blocks of 64 columns, `stride` that of groups of
// eight rows.  Bytes.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t at, uint32_t lead, uint32_t stride)
{
    return (uint64_t)((at & 0x3ffffu) >> 4) | ((uint64_t)((lead & 0x3ffffu) >> 4) << 16) | ((uint64_t)((stride & 0x3ffffu) >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// Byte offset of 16-byte piece `piece` of row `row` in a block.
__device__ __forceinline__ uint32_t tile_piece(int row, int piece) { return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4)); }

}  // namespace dynb
