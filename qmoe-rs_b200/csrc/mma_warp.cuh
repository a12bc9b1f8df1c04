// mma_warp.cuh -- tcgen05.mma and commit issued by a converged warp, one elected
// lane of it acting.  A whole warp runs the code around them, so descriptors
// and addresses stay in uniform registers; from a one-lane branch every MMA
// first moves each of them there.  The elected lane is the same every time
// (full membership mask), so a commit covers the MMAs before it.
#pragma once

#include "sm100.cuh"

namespace qmoe {
namespace sm100 {

// mbar_wait_warp whose probes suspend for up to two microseconds each: warps
// that wait for long leave the issue slots to the others.
QMOE_DEV bool wait_long(uint64_t *bar, uint32_t parity, volatile int *abort, int *err) {
    for (uint32_t n = 0; n < kMaxWaitProbes; ++n) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
            : "memory");
        if (__all_sync(0xffffffffu, done)) return true;
        if (__any_sync(0xffffffffu, *abort != 0)) return false;
    }
    if ((threadIdx.x & 31) == 0) {
        *abort = 1;
        atomicOr(err, kErrWaitTimeout);
    }
    __syncwarp();
    return false;
}

#define QMOE_MMA_WARP(kind, a_decl, a_op)                                                           \
    "{\n .reg .pred p, e;\n .reg .b64 ad, bd;\n setp.ne.b32 p, %5, 0;\n elect.sync _|e, 0xffffffff;\n" \
    a_decl " mov.b64 bd, {%2, %3};\n"                                                              \
    " @e tcgen05.mma.cta_group::1.kind::" kind " [%0], " a_op ", bd, %4, {%6, %6, %6, %6}, p;\n}"

// D[tmem] (+)= A[smem] * B[smem]^T; lo, hi: halves of the descriptors (hi the same).
QMOE_DEV void warp_mma_f16_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(QMOE_MMA_WARP("f16", " mov.b64 ad, {%1, %3};\n", "ad") ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi),
                 "r"(idesc), "r"(accumulate), "r"(0u)
                 : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T.
QMOE_DEV void warp_mma_f16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(QMOE_MMA_WARP("f16", "", "[%1]") ::"r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate),
                 "r"(0u)
                 : "memory");
}

// 8-bit integers, 32-bit sums.
QMOE_DEV void warp_mma_i8_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(QMOE_MMA_WARP("i8", " mov.b64 ad, {%1, %3};\n", "ad") ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi),
                 "r"(idesc), "r"(accumulate), "r"(0u)
                 : "memory");
}

#undef QMOE_MMA_WARP

// Arrive on `bar` once every MMA the warp issued so far is done.
QMOE_DEV void warp_commit(uint64_t *bar) {
    asm volatile(
        "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
        : "memory");
}

}  // namespace sm100
}  // namespace qmoe
