// PTX wrappers of the 5th-generation tensor core instructions (sm_100a): TMEM allocation, the
// bf16 / fp16 matrix product on shared-memory operands, its completion on an mbarrier, and the
// loads and stores of accumulators.
#pragma once

#include "common.cuh"

namespace dflash {
namespace tc5 {

// Warp-wide: allocates `columns` (a power of two from 32 to 512) of TMEM and writes the base
// address to shared memory; no other kernel of this library that uses TMEM fits beside one
// that does, so the allocation never waits.
__device__ __forceinline__ void alloc(uint32_t smem_dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(columns));
}

// True on one lane of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand in 128-byte swizzled rows (1024-byte aligned tiles of 8 rows).  lead: byte
// step between 64-element blocks along a transposed operand's M or N; step: bytes between 8-row
// groups.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead, uint32_t step) {
    return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 |
           static_cast<uint64_t>(step >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor: fp32 accumulators, both operands bf16 or both fp16, M = 128, N columns;
// transposed: both operands are stored along M / N instead of along K.
__device__ __forceinline__ uint32_t shape(bool bf16, bool transposed, uint32_t n) {
    const uint32_t type = bf16 ? 1u : 0u, major = transposed ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | major << 15 | major << 16 | (n >> 3) << 17 | (128u >> 4) << 24;
}

// D[tmem] (+)= A B, one thread.
__device__ __forceinline__ void mma(uint32_t tmem, uint64_t a, uint64_t b, uint32_t desc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(a), "l"(b), "r"(desc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// Arrives on the mbarrier once every product that this thread has issued is complete.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// 32 (16) consecutive columns of the warp's 32 lanes, a register per column.  The wait is part of
// the statement, so no use of the registers can be scheduled before it.
__device__ __forceinline__ void ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}

}  // namespace tc5
}  // namespace dflash
