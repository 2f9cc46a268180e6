// Fifth-generation tensor core instructions (tcgen05) as the kernels use them.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace aion {

// UMMA shared-memory matrix descriptor, K-major with the 128-byte swizzle:
// rows of 128 bytes, 8-row groups 1024 bytes apart (SBO), version 1.  Only
// the low word depends on the address (umma_lo), in units of 16 bytes.
__device__ __forceinline__ uint32_t umma_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | (1u << 16); }
constexpr uint32_t kUmmaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr) {
    return (uint64_t)umma_lo(saddr) | ((uint64_t)kUmmaDescHi << 32);
}

// One tcgen05.mma of kind::f16 with both operands in shared memory: D (TMEM)
// += A B^T, M and N and the operands' type (bf16 or fp16, the same for both)
// by `idesc`, K = 16.
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
        : "memory");
}

__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}

// A run of tcgen05.mma issued by one elected lane of a converged warp, in one
// piece: D (TMEM) (+)= A B^T over `steps` (1..8) k-steps of 16 fp16 or bf16
// values (the type by `idesc`), both operands in shared memory, in the
// 128-byte-swizzled halves of 64 values that umma_lo points to; `half_a` and
// `half_b` (in 16 bytes) lead to the second halves.
// One piece, because the operands of each MMA pass through uniform registers,
// and an election for each took longer than the MMA itself.
#define UMMA_STEP(K, A, B)                                                     \
    "setp.gt.and.s32 on, %6, " K ", lead;\n\t"                                 \
    "add.u32 al, " A ";\n\tadd.u32 bl, " B ";\n\t"                             \
    "mov.b64 ad, {al, %7};\n\tmov.b64 bd, {bl, %7};\n\t"                       \
    "@on tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %3, one;\n\t"
__device__ __forceinline__ void umma_run_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t half_a, uint32_t half_b,
                                            uint32_t idesc, int steps, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred lead, acc, one, on;\n\t.reg .b32 al, bl;\n\t.reg .b64 ad, bd;\n\t"
        "elect.sync _|lead, 0xffffffff;\n\t"
        "setp.ne.b32 acc, %5, 0;\n\t"
        "setp.eq.b32 one, 0, 0;\n\t"
        "mov.b64 ad, {%1, %7};\n\tmov.b64 bd, {%2, %7};\n\t"
        "@lead tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %3, acc;\n\t"
        UMMA_STEP("1", "%1, 2", "%2, 2") UMMA_STEP("2", "%1, 4", "%2, 4") UMMA_STEP("3", "%1, 6", "%2, 6")
        UMMA_STEP("4", "%4, 0", "%8, 0") UMMA_STEP("5", "%4, 2", "%8, 2") UMMA_STEP("6", "%4, 4", "%8, 4")
        UMMA_STEP("7", "%4, 6", "%8, 6") "}"
        ::"r"(tmem_d), "r"(a), "r"(b), "r"(idesc), "r"(a + half_a), "r"(accumulate), "r"(steps), "r"(kUmmaDescHi),
        "r"(b + half_b)
        : "memory");
}
#undef UMMA_STEP
// The same with A in TMEM (lanes are rows, a column holds two values along K)
// and four k-steps, in one half of B.
__device__ __forceinline__ void umma_run4_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred lead, acc, one;\n\t.reg .b32 al, bl;\n\t.reg .b64 bd;\n\t"
        "elect.sync _|lead, 0xffffffff;\n\t"
        "setp.ne.b32 acc, %4, 0;\n\t"
        "setp.eq.b32 one, 0, 0;\n\t"
        "mov.b64 bd, {%2, %5};\n\t"
        "@lead tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %3, acc;\n\t"
        "add.u32 al, %1, 8;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 bd, {bl, %5};\n\t"
        "@lead tcgen05.mma.cta_group::1.kind::f16 [%0], [al], bd, %3, one;\n\t"
        "add.u32 al, %1, 16;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 bd, {bl, %5};\n\t"
        "@lead tcgen05.mma.cta_group::1.kind::f16 [%0], [al], bd, %3, one;\n\t"
        "add.u32 al, %1, 24;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 bd, {bl, %5};\n\t"
        "@lead tcgen05.mma.cta_group::1.kind::f16 [%0], [al], bd, %3, one;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kUmmaDescHi)
        : "memory");
}
__device__ __forceinline__ void umma_commit_warp(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

}  // namespace aion
