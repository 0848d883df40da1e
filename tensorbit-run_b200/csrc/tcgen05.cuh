// tcgen05.cuh -- the fifth-generation tensor core instructions that the kernels
// use: f16 products with f32 sums in tensor memory, issued by one thread, their
// right operand in shared memory, the left one there or in tensor memory.
//
// Operand tiles in shared memory have rows of 128 bytes (64 f16), the 16-byte
// piece c of row r at c ^ (r & 7), on 1024-byte boundaries:
//   K-major   a row is one of the operand's M or N indices, 64 of K; the next 8
//             rows 1024 bytes on; 16 of K further is 32 bytes further;
//   MN-major  a row is one of K, 64 M or N indices; the next 8 rows 1024 bytes
//             on, the next 64 indices `lead` bytes on; 16 of K further is 2048.
#pragma once

#include <stdint.h>

#include "tma.cuh"

namespace tc {

__device__ __forceinline__ uint64_t tile_descriptor(uint32_t smem, uint32_t lead) {
    return (uint64_t)((smem >> 4) & 0x3fff) |      // start
           (uint64_t)((lead >> 4) & 0x3fff) << 16 |  // leading dimension offset
           (uint64_t)(1024 >> 4) << 32 |             // 8 rows further
           1ull << 46 |                              // the descriptor's version
           2ull << 61;                               // 128-byte swizzle
}

// f16 x f16 -> f32, M = 128; the right operand MN-major or K-major.
constexpr uint32_t f16_instruction(int n, bool right_mn_major) {
    return 1u << 4 | (right_mn_major ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 |
           (uint32_t)(128 / 16) << 24;
}

// The instructions below are for a whole warp, whose lane `leader` issues them:
// the operands stay uniform, and no lane waits for another's branch.
//
// d (tensor memory) = a b, or += if `add`; a in shared memory.
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction,
                                    bool add, bool leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add), "r"((uint32_t)leader)
        : "memory");
}
// The same, a in tensor memory (two f16 a column).
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t instruction,
                                         bool add, bool leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(instruction), "r"((uint32_t)add), "r"((uint32_t)leader)
        : "memory");
}
// Arrive on bar when the products issued so far by the leader are done.
__device__ __forceinline__ void commit(uint64_t* bar, bool leader) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(
            tbk::smem_addr(bar)),
        "r"((uint32_t)leader)
        : "memory");
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Whole-warp: allocate `columns` of tensor memory, the address into *smem_out.
__device__ __forceinline__ void allocate(uint32_t* smem_out, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tbk::smem_addr(smem_out)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void release(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address),
                 "r"(columns)
                 : "memory");
}

// COLUMNS columns (a multiple of 32) of the warp's 32 rows, a row a lane: asked
// for all at once, waited for once.  The values pass through the wait, so that
// nothing computes with them before it.
template <int COLUMNS>
__device__ __forceinline__ void load(uint32_t address, float (&v)[COLUMNS]) {
#pragma unroll
    for (int i = 0; i < COLUMNS; i += 32) {
        float* r = v + i;
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
              "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]),
              "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]),
              "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
              "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]),
              "=f"(r[31])
            : "r"(address + i));
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < COLUMNS; i += 8) {
        float* r = v + i;
        asm volatile(""
                     : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]),
                       "+f"(r[6]), "+f"(r[7]));
    }
}
__device__ __forceinline__ void store32(uint32_t address, const float (&v)[32]) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void store16(uint32_t address, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}
// The warpgroup's registers per thread; the shares add up to the launch's.
template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void wait_store() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

}  // namespace tc
