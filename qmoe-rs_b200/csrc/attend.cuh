// attend.cuh -- what the two attention kernels over the 8-bit cache share
// (attend.cu, attend_prompt.cu).
#pragma once

#include <cuda_fp16.h>

#include "code8.cuh"
#include "kernels.h"

namespace qmoe {

constexpr float kLog2e = 1.44269504088896340736f;

QMOE_DEV float neg_inf() { return __int_as_float(0xff800000); }

QMOE_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

QMOE_DEV uint32_t h2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

QMOE_DEV float h_lo(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v & 0xffff))); }
QMOE_DEV float h_hi(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }

// Four codes as fp16, exactly: as 1152 + c (0x6400 | (c + 128)) first.
QMOE_DEV void codes_to_half(uint32_t v, uint32_t &lo, uint32_t &hi) {
    v ^= 0x80808080u;
    const uint32_t a = __byte_perm(v, 0x64646464u, 0x4140), b = __byte_perm(v, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
}

// tok / block for a multiple of 16: per_block = ceil(2^36 / (block / 16)); exact
// below 2^31, since the error of the product is below 2^27 * 16 < 2^36 / 16.
QMOE_DEV int block_index(const AttendParams &p, int tok) {
    return (int)(((uint64_t)(uint32_t)(tok >> 4) * p.per_block) >> 36);
}

// Four elements of q; the type and the form of the load are the caller's
// constants, so that several calls' loads are in flight together (a test of
// either between them had each wait for the one before).
template <bool BF16, bool VEC>
QMOE_DEV float4 load_q4(const AttendParams &p, int64_t at) {
    if (VEC) return load_act4(p.q, BF16 ? 1 : 0, at);
    return make_float4(load_act(p.q, BF16 ? 1 : 0, at), load_act(p.q, BF16 ? 1 : 0, at + 1),
                       load_act(p.q, BF16 ? 1 : 0, at + 2), load_act(p.q, BF16 ? 1 : 0, at + 3));
}

// A row of q whose largest magnitude is m goes to fp16 times 2^(14 - e): below
// 2^15 and, but for elements 2^-28 below the largest, with all of bf16's bits.
// No row is above f32's 2^128; those below 2^-100 are as good as 0.
QMOE_DEV int q_exponent(float m) {
    const int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;
    return e < -100 ? -100 : e;
}

}  // namespace qmoe
