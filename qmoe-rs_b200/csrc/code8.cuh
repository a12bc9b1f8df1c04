// code8.cuh -- the 8-bit code of a value on a symmetric range, shared by the
// row quantiser (int8.cu) and the append to the 8-bit cache (kv.cu).
//
//   r     = max(max |x|, 127 * 2^-64), NaN when an element is not finite
//   code  = 127 x / r rounded to the nearest whole number, ties to even
//   value = code * (r / 127)
//
// The rounding is that of the real quotient, not of a rounded one: the f32
// estimate decides unless it lies within 2^-14 of a border between two codes
// (its error is below 2^-16: two roundings of a value of at most 127), and
// the f64 quotient decides there.  The f64 products a * m are exact (24 + 24
// bits), and a quotient of 24-bit numbers that is not on a border is further
// from it than f64's rounding, so a code is the same whatever computes it.
#pragma once

#include "common.cuh"

namespace qmoe {

constexpr float kRangeFloor = 127.0f * 5.42101086242752217e-20f;   // a scale of 2^-64

// Out of line: rare, and an f64 division at every use would fill the
// instruction cache (64 single tokens' append took 23 us with it inlined, see
// kv.cu).
static __device__ __noinline__ int code8_exact(float a, float m, float r) {
    return (int)rint((double)a * (double)m / (double)r);
}

// a * m / r as a code, |a * m| <= 127 r; mi = m / r in f32.
QMOE_DEV int code8(float a, float m, float r, float mi) {
    const float q = __fmul_rn(a, mi);
    const float c = rintf(q);
    if (fabsf(fabsf(__fsub_rn(q, c)) - 0.5f) < 6.103515625e-05f)
        return code8_exact(a, m, r);
    return (int)c;                                                 // NaN gives 0
}

// The range of values whose largest magnitude is `m`, when `finite`.
QMOE_DEV float range8(float m, bool finite) {
    return finite ? fmaxf(m, kRangeFloor) : __int_as_float(0x7fc00000);
}

QMOE_DEV float max_abs(float m, float v) { return fmaxf(m, fabsf(v)); }   // NaN is looked for apart

// Four codes as bytes, the first in the lowest.
QMOE_DEV uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

static __device__ __noinline__ uint32_t codes4_exact(float a, float b, float c, float d, float m, float r) {
    if (r != r) return 0;
    return pack4(code8_exact(a, m, r), code8_exact(b, m, r), code8_exact(c, m, r), code8_exact(d, m, r));
}

// code8 of four values as bytes, with one branch for the four of them and no
// conversions (16 lanes a cycle an SM, where additions have 128): 1.5 * 2^23
// added to a value of at most 127 rounds it to a whole number, ties to even,
// that stands in the sum's low byte.  NaN, all four alike, takes the branch.
QMOE_DEV uint32_t codes4(float a, float b, float c, float d, float m, float r, float mi) {
    constexpr float kWhole = 12582912.0f;
    const float v[4] = {__fmul_rn(a, mi), __fmul_rn(b, mi), __fmul_rn(c, mi), __fmul_rn(d, mi)};
    uint32_t w[4];
    float far[4];                                 // from the whole number
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = __fadd_rn(v[i], kWhole);
        w[i] = __float_as_uint(t);
        far[i] = fabsf(__fsub_rn(v[i], __fsub_rn(t, kWhole)));
    }
    if (!(fmaxf(fmaxf(far[0], far[1]), fmaxf(far[2], far[3])) <= 0.5f - 6.103515625e-05f))
        return codes4_exact(a, b, c, d, m, r);
    return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

}  // namespace qmoe
