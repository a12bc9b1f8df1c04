// attend_prompt.cu -- attention over the 8-bit cache for prompts: requests with
// more tokens than attend.cu's rows hold, bf16 activations.
//
// The arithmetic is attend.cu's (its head says how): scores on codes, the
// blocks' scales folded into t = (q . ck) * f + log2(rv / 127), P = 2^(t - M) in
// fp16, f32 sums.  What differs is where it runs.  A CTA takes 256 query rows
// (two tiles of 128: tq tokens by the heads that share a kv head) and goes once
// over their keys in tiles of 64 tokens:
//
//   warps 0-3, 4-7   one row of a query tile a thread: q to fp16 in shared
//                    memory, then per key tile the scores from tensor memory,
//                    the running maximum and sum, P back to tensor memory
//   warps 8-14       codes from the cache to fp16 operands in shared memory (K
//                    [token][dim], V [dim][token]; 128-byte swizzle) and the
//                    scales; the eight 16-token groups of K and V of a tile go
//                    round the seven warps
//   warp 15          tcgen05: S = q K^T (both operands in shared memory), then
//                    O += P V (P from tensor memory)
//
// Tensor memory holds two score tiles and O of each query tile.  The scores of
// a tile are asked for two tiles ahead, so a softmax waits for no MMA, and the
// two query tiles' softmaxes run side by side.  O is scaled to a maximum that a
// row's own may outgrow by 2^8: P is made with it before the tile's maximum is
// known and made again, with O rescaled, only where that was too small (P then
// reaches 2^(8 + 6), which fp16 holds; its rounding, 2^-11 of P or 2^-31 of that
// maximum, is below that of the bf16 output; the sum takes P in f32).  For 256
// rows by 128 keys of 128 dims the exponentials take 2048 cycles of an SM (16 a
// cycle) and the MMAs as many.
// Measured: three prompts of up to 2048 tokens after up to 6000, 32 query and 8 kv
// heads of 128, 355 us = 700 TFLOP/s, the tensor pipe busy 38 % of the time: the
// chain score, softmax, P V of two query tiles and the barriers between its warps
// bound it, then the tail of 256 long items on 148 SMs.
#include "attend.cuh"
#include "kernels.h"
#include "mma_warp.cuh"

namespace qmoe {
namespace {

using namespace sm100;

constexpr int kSoftWarps = 8, kCodeWarps = 7, kMmaWarp = 15;
constexpr int kThreads = 16 * 32;
constexpr int KT = 64;                        // keys a tile
constexpr float kGrow = 8.0f;                 // log2 of how far a maximum may outgrow the scaling
constexpr float kShift = 6.0f;                // P = 2^6 at the scaling's maximum
// Tiles whose scales are kept.  Those of tile u are written once the scores
// of tile u - stages are done; these were asked for after P of tile u - stages -
// 2, so the softmax is done with the slot's tile u - 8.
constexpr int kScaleRing = 8;

template <int DK, int DV>
struct Shared {
    static constexpr int kStages = DK > 128 ? 3 : 4;
    static constexpr int kQ = 128 * DK * 2, kK = KT * DK * 2, kV = DV * KT * 2;
    static_assert(kStages + 2 <= kScaleRing, "scales");
    uint8_t q[2][kQ];
    uint8_t k[kStages][kK];
    uint8_t v[kStages][kV];
    float f[kScaleRing][KT / 16], lv[kScaleRing][KT / 16], iv[kScaleRing][KT / 16];
    uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2];
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) {
    return (1u << 4)          // D = f32; A, B = f16 (format 0)
           | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Four bf16; `vec`: the address is a multiple of 8.
QMOE_DEV uint2 load_bf16x4(const uint16_t *at, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const uint2 *>(at));
    return make_uint2(at[0] | (uint32_t)at[1] << 16, at[2] | (uint32_t)at[3] << 16);
}
QMOE_DEV float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
QMOE_DEV float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// Pairs of f32 in one instruction each, every half rounded as the single form.
QMOE_DEV uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
QMOE_DEV void unpair(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
QMOE_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
QMOE_DEV uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
QMOE_DEV float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

QMOE_DEV uint4 ldg_code(const int8_t *at) { return __ldg(reinterpret_cast<const uint4 *>(at)); }

// Sixteen codes as fp16 to units `unit` and unit + 1 (16 bytes each) of row r of
// a 128-byte swizzled operand.  A quarter warp's units are distinct banks: two
// rows of four even units (K), or eight rows of one (V).
QMOE_DEV void store_codes(uint8_t *row, int unit, int r, const uint4 &v) {
    uint4 a, b;
    codes_to_half(v.x, a.x, a.y);
    codes_to_half(v.y, a.z, a.w);
    codes_to_half(v.z, b.x, b.y);
    codes_to_half(v.w, b.z, b.w);
    *reinterpret_cast<uint4 *>(row + ((unit ^ (r & 7)) << 4)) = a;
    *reinterpret_cast<uint4 *>(row + (((unit + 1) ^ (r & 7)) << 4)) = b;
}

// `span` tokens of a request (both query tiles', or the first one's) that begin
// in a window of rows of q.
struct Item {
    int64_t request;
    int t0, cnt;                              // first row of q, tokens
    int pos0;                                 // last key of the first token
    int keys;                                 // of the last token
};

// The item of the first request from `r` on that has one in the window; false
// when there is none.  Requests of up to `few` tokens are attend.cu's.  The
// whole warp alike.
QMOE_DEV bool next_item(const AttendParams &p, int64_t lo, int64_t hi, int span, int few, int64_t &r, Item &it) {
    const int lane = threadIdx.x & 31;
    for (; r < p.R; r += 32) {
        const int64_t mine = r + lane;
        int64_t s0 = 0, n = 0, at = -1;
        if (mine < p.R) {
            s0 = p.q_start[mine];
            n = p.q_start[mine + 1] - s0;
            if (n > few && s0 >= 0) {
                at = s0 >= lo ? s0 : s0 + (lo - s0 + span - 1) / span * span;
                if (at >= hi || at >= s0 + n) at = -1;
            }
        }
        const unsigned some = __ballot_sync(0xffffffffu, at >= 0);
        if (some) {
            const int f = __ffs(some) - 1;
            s0 = __shfl_sync(0xffffffffu, s0, f);
            n = __shfl_sync(0xffffffffu, n, f);
            at = __shfl_sync(0xffffffffu, at, f);
            it.request = r + f;
            it.t0 = (int)at;
            const int64_t end = s0 + n < p.T ? s0 + n : p.T;   // rows that the buffer does not hold
            it.cnt = (int)(end - at < span ? end - at : span);
            const int64_t most = p.max_blocks * p.c.block, kv0 = p.kv_lens[it.request];
            const int64_t kv = kv0 < 0 ? 0 : kv0;
            const int64_t pos0 = kv - n + (at - s0), keys = pos0 + it.cnt;
            it.pos0 = (int)(pos0 < -(1 << 30) ? -(1 << 30) : pos0);
            it.keys = (int)(keys < 0 ? 0 : keys < most ? keys : most);
            r = it.request + 1;
            return true;
        }
        // past the window: starts never fall
        if (__shfl_sync(0xffffffffu, mine < p.R ? s0 : hi, 31) >= hi) break;
    }
    return false;
}

// The first request whose rows reach past row `lo`.
QMOE_DEV int64_t first_request(const int32_t *start, int64_t R, int64_t lo) {
    const int lane = threadIdx.x & 31;
    int64_t at = 0, n = R;                    // the last r with start[r] <= lo, or 0
    while (n > 1) {
        const int64_t step = (n + 31) / 32, i = at + lane * step;
        const bool le = lane == 0 || (i < at + n && start[i] <= lo);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
        const int64_t next = at + last * step;
        n = at + n - next < step ? at + n - next : step;
        at = next;
    }
    return at;
}

template <int DK, int DV>
__global__ void __launch_bounds__(kThreads, 1)
attend_prompt_kernel(const AttendParams p, const int tq, const int span, const int rows, const int gq, const int hgroups,
                     const int few) {
    using Sm = Shared<DK, DV>;
    constexpr int kStages = Sm::kStages;
    extern __shared__ uint8_t smem_raw[];
    Sm &S = *reinterpret_cast<Sm *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // late windows of all heads first: their rows see the most keys
    const int groups = p.c.heads * hgroups, windows = gridDim.x / groups;
    const int window = blockIdx.x / groups, hh = blockIdx.x - window * groups;
    const int64_t lo = (int64_t)(windows - 1 - window) * rows, hi = lo + rows < p.T ? lo + rows : p.T;
    const int h = hh / hgroups, hg = hh - h * hgroups, G = p.heads / p.c.heads;
    const int head0 = h * G + hg * gq, heads_here = G - hg * gq < gq ? G - hg * gq : gq;
    int64_t r = first_request(p.q_start, p.R, lo);
    const int64_t r0 = r;
    Item it;
    if (!next_item(p, lo, hi, span, few, r, it)) {            // the whole CTA alike
        QMOE_PDL_TRIGGER();
        QMOE_PDL_WAIT();
        return;
    }

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.q_full[i], 4);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&S.s_full[i][b], 2);        // the MMAs, and the warp that issued them
                mbar_init(&S.p_full[i][b], 4);
                mbar_init(&S.pv_done[i][b], 1);
            }
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&S.k_full[i], 4);
            mbar_init(&S.k_empty[i], 1);
            mbar_init(&S.v_full[i], 4);
            mbar_init(&S.v_empty[i], 1);
        }
        mbar_init(&S.drain, 1);
        S.abort = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&S.tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Beside the launch before (attend.cu): the wait is at the end.  A later
    // kernel that holds TMEM while it waits must find this one's columns taken.
    QMOE_PDL_TRIGGER();
    const uint32_t tmem = S.tmem_base;
    // columns: scores (P in a tile's first half) of query tile m, buffer b at
    // 128 m + 64 b; O of query tile m at 256 + 128 m
    constexpr uint32_t kOCol = 256;
    volatile int *abort = &S.abort;
    bool ok = true;
    r = r0;

    if (warp < kSoftWarps) {
        // ---------------------------------------------------------- softmax
        const int m = warp >> 2, q = warp & 3, row = q * 32 + lane;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const uint32_t s_at = tmem + lanes + m * 128, o_at = tmem + lanes + kOCol + m * 128;
        const float scale = fabsf(p.scale) * kLog2e, sign = p.scale < 0.0f ? -1.0f : 1.0f;
        uint32_t u = 0, n = 0;                        // key tiles of the CTA, and those with this query tile, so far
        while (ok && next_item(p, lo, hi, span, few, r, it)) {
            const int cnt = it.cnt - m * tq < tq ? it.cnt - m * tq : tq;      // tokens of this query tile
            const int nt = (it.keys + KT - 1) / KT;
            const int i = row / gq, gg = row - i * gq;
            const bool live = i < cnt && gg < heads_here;
            const int64_t tok = (int64_t)it.t0 + m * tq + i;
            const int64_t out_at = tok * p.ldo + (int64_t)(head0 + gg) * DV;
            if (nt == 0 || cnt <= 0) {
                // nothing to see: zeros, a row a warp at a time
                for (int x = 0; x < 32 && cnt > 0; ++x) {
                    const int64_t at = __shfl_sync(0xffffffffu, live ? out_at : -1, x);
                    if (at >= 0)
                        for (int d = lane; d < DV; d += 32) reinterpret_cast<__nv_bfloat16 *>(p.out)[at + d] = __float2bfloat16_rn(0.0f);
                }
                u += nt;
                continue;
            }
            // q: rows by a power of two (and the scale's sign), as fp16, 64 dims a
            // 128-byte row; some of the warp's rows at a time, four dims a lane
            float back = 0.0f;
            constexpr int kRep = (DK + 127) / 128, kAtOnce = 8 / kRep;
#pragma unroll 1
            for (int x = 0; x < 32; x += kAtOnce) {
                uint2 raw[kAtOnce][kRep];                                    // all in flight at once
                const int64_t mine = live ? tok * p.ldq + (int64_t)(head0 + gg) * DK : -1;
#pragma unroll
                for (int y = 0; y < kAtOnce; ++y) {
                    const int64_t at = __shfl_sync(0xffffffffu, mine, x + y);
#pragma unroll
                    for (int z = 0; z < kRep; ++z) {
                        const int d = 4 * lane + 128 * z;
                        const bool some = at >= 0 && d < DK;
                        raw[y][z] = load_bf16x4(reinterpret_cast<const uint16_t *>(p.q) + (some ? at + d : 0), p.vec_q);
                        if (!some) raw[y][z] = make_uint2(0, 0);
                    }
                }
#pragma unroll
                for (int y = 0; y < kAtOnce; ++y) {
                    float mx = 0.0f;
#pragma unroll
                    for (int z = 0; z < kRep; ++z)
                        mx = max_abs(max_abs(max_abs(max_abs(mx, bf_lo(raw[y][z].x)), bf_hi(raw[y][z].x)), bf_lo(raw[y][z].y)),
                                     bf_hi(raw[y][z].y));
                    const int e = q_exponent(warp_max(mx)), at = q * 32 + x + y;
                    const float up = sign * pow2i(14 - e);
#pragma unroll
                    for (int z = 0; z < kRep; ++z) {
                        const int d = 4 * lane + 128 * z;
                        const uint2 f = make_uint2(h2(bf_lo(raw[y][z].x) * up, bf_hi(raw[y][z].x) * up),
                                                   h2(bf_lo(raw[y][z].y) * up, bf_hi(raw[y][z].y) * up));
                        if (d < DK)
                            *reinterpret_cast<uint2 *>(S.q[m] + (d >> 6) * (128 * 128) + at * 128 +
                                                       ((((d >> 3) & 7) ^ (at & 7)) << 4) + 2 * (d & 4)) = f;
                    }
                    if (lane == x + y) back = pow2i(e - 14);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.q_full[m]);
            back *= scale;
            const int last = live ? it.pos0 + m * tq + i : -1;               // this row's last key
            const int first_last = it.pos0 + m * tq;                         // the first token's
            float mx = neg_inf(), sum = 0.0f;                                // mx: what O and sum are scaled to
            for (int j = 0; j < nt; ++j, ++u, ++n) {
                const uint32_t at = s_at + 64 * (n & 1);
                if (!(ok = wait_long(&S.s_full[m][n & 1], (n >> 1) & 1, abort, p.err))) break;
                tc_fence_after();
                const int see = last - j * KT;                               // columns 0 .. see are visible
                const bool whole = j * KT + KT - 1 <= first_last && j * KT + KT <= it.keys;
                uint32_t t[2][32];                                           // scores; dead once P is made
                auto load_scores = [&] {
                    tmem_ld_x32(at, t[0]);
                    tmem_ld_x32(at + 32, t[1]);
                    tmem_wait_ld();
                    if (!whole) {
#pragma unroll
                        for (int x = 0; x < 64; ++x)
                            if (x > see) t[x >> 5][x & 31] = 0xff800000u;    // -inf
                    }
                };
                load_scores();
                uint32_t w[2][16];
                // P, its sum, and the largest exponent of the tile over `base`
                auto exponentials = [&](float base, float &top) {
                    float total = 0.0f, m4[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        // the group's factors: a > 0, so that a masked score of -inf stays one (a
                        // poisoned group's NaN is in lv).  A row that sees none of the group takes
                        // neither its lv nor its iv, which may be NaN.
                        const bool seen = 16 * x <= see;
                        const float a = fmaxf(S.f[u % kScaleRing][x] * back, 1.17549435e-38f);
                        const float b = (seen ? S.lv[u % kScaleRing][x] : neg_inf()) - base;
                        const uint64_t aa = pair(a, a), bb = pair(b, b);
                        uint64_t acc = pair(0.0f, 0.0f);
                        m4[x] = neg_inf();
#pragma unroll
                        for (int y = 0; y < 16; y += 2) {
                            const int z = 16 * (x & 1) + y;
                            float t0, t1;
                            unpair(fma2(pair(__uint_as_float(t[x >> 1][z]), __uint_as_float(t[x >> 1][z + 1])), aa, bb), t0, t1);
                            m4[x] = max3(m4[x], t0, t1);
                            const float e0 = ex2(t0), e1 = ex2(t1);
                            acc = add2(acc, pair(e0, e1));
                            w[x >> 1][z / 2] = h2(e0, e1);
                        }
                        float p0, p1;
                        unpair(acc, p0, p1);
                        total = __fmaf_rn(p0 + p1, seen ? S.iv[u % kScaleRing][x] : 0.0f, total);
                    }
                    top = max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]);
                    return total;
                };
                float top, add = exponentials(mx == neg_inf() ? 0.0f : mx - kShift, top);
                // too small a scaling; the first tile's is none at all
                const bool grow = mx == neg_inf() ? top != neg_inf() : top > kGrow + kShift;
                if (__any_sync(0xffffffffu, grow)) {
                    const float to = top + (mx == neg_inf() ? 0.0f : mx - kShift);   // the tile's largest
                    const float now = grow ? to : mx;    // a row's bits do not depend on the warp's other rows
                    const float by = now == neg_inf() ? 1.0f : ex2(mx - now);
                    mx = now;
                    sum *= by;
                    if (j > 0) {                                             // O is the last tile's product's until it is done
                        if (!(ok = wait_long(&S.pv_done[m][(n - 1) & 1], ((n - 1) >> 1) & 1, abort, p.err))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DV; c += 16) {
                            uint32_t o[16];
                            tmem_ld_x16(o_at + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * by);
                            tmem_st_x16(o_at + c, o);
                        }
                    }
                    load_scores();
                    add = exponentials(mx == neg_inf() ? 0.0f : mx - kShift, top);
                }
                sum += add;
                tmem_st_x16(at, w[0]);
                tmem_st_x16(at + 16, w[1]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.p_full[m][n & 1]);
            }
            if (!ok) break;
            if (!(ok = wait_long(&S.pv_done[m][(n - 1) & 1], ((n - 1) >> 1) & 1, abort, p.err))) break;
            tc_fence_after();
            const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
            const bool wide = p.vec_out;
#pragma unroll 1
            for (int c = 0; c < DV; c += 32) {
                uint32_t o[32];
                tmem_ld_x32(o_at + c, o);
                tmem_wait_ld();
                if (live) {
                    __nv_bfloat16 *to = reinterpret_cast<__nv_bfloat16 *>(p.out) + out_at + c;
#pragma unroll
                    for (int x = 0; x < 32; x += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(
                                sum == 0.0f ? 0.0f : __uint_as_float(o[x + 2 * y]) * inv,
                                sum == 0.0f ? 0.0f : __uint_as_float(o[x + 2 * y + 1]) * inv);
                            w[y] = *reinterpret_cast<const uint32_t *>(&v);
                        }
                        if (wide) {
                            *reinterpret_cast<uint4 *>(to + x) = make_uint4(w[0], w[1], w[2], w[3]);
                        } else {
#pragma unroll
                            for (int y = 0; y < 8; ++y)
                                reinterpret_cast<unsigned short *>(to)[x + y] = (unsigned short)(w[y >> 1] >> (16 * (y & 1)));
                        }
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
        }
    } else if (warp < kMmaWarp) {
        // ---------------------------------------------------------- codes to operands
        // Unit 8 u + x is group x of K (x < 4; loads of 8 tokens by 64 dims) or x - 4 of V
        // (32 dims) of tile u.  The codes of a warp's next unit are loaded while this
        // one's wait for their stage; blocks are looked up two units ahead.
        const int g = lane >> 2, c = lane & 3, bs = p.c.block;
        constexpr int kKLoads = 2 * (DK / 64), kVLoads = DV / 32, kLoads = kKLoads > kVLoads ? kKLoads : kVLoads;
        uint32_t first = 0;                           // unit of the item's first tile
        uint32_t unit = warp - kSoftWarps;            // this warp's next
        while (ok && next_item(p, lo, hi, span, few, r, it)) {
            const int nt = (it.keys + KT - 1) / KT;
            const uint32_t end = first + 8 * nt;
            const int32_t *table = p.table + it.request * p.max_blocks;
            auto token_of = [&](uint32_t x) { return (int)((x - first) >> 3) * KT + (int)(x & 3) * 16; };
            auto block_of = [&](uint32_t x) -> int64_t {
                const int tok = token_of(x);
                if (x >= end || tok >= it.keys) return -1;
                const int64_t b = table[block_index(p, tok)];
                return b >= 0 && b < p.c.num_blocks ? b * p.c.heads + h : -1;
            };
            uint4 codes[kLoads];
            float kr = 0.0f, vr = -1.0f;              // ranges of a K unit's group; vr -1: no group
            auto load = [&](uint32_t x, int64_t bh) {
                const bool is_v = x & 4;
                const int tok = token_of(x), off = tok - block_index(p, tok) * bs;
                const int8_t *at = is_v ? p.c.v + ((bh * (bs / 16) + off / 16) * DV + lane) * 16
                                        : p.c.k + (bh * (DK / 64) * bs + off + g) * 64 + c * 16;
#pragma unroll
                for (int y = 0; y < kLoads; ++y) {
                    const int step = is_v ? y * 512 : (y >> 1) * bs * 64 + (y & 1) * 512;
                    codes[y] = bh >= 0 && y < (is_v ? kVLoads : kKLoads) ? ldg_code(at + step) : make_uint4(0, 0, 0, 0);
                }
                kr = bh >= 0 && !is_v ? p.c.k_range[bh] : 0.0f;
                vr = bh >= 0 && !is_v ? p.c.v_range[bh] : -1.0f;
            };
            if (unit < end) load(unit, block_of(unit));
            int64_t b1 = block_of(unit + kCodeWarps);
            for (; unit < end; unit += kCodeWarps) {
                const bool is_v = unit & 4;
                const uint32_t u = unit >> 3, st = u % kStages, phase = (u / kStages) & 1, grp = unit & 3;
                const int64_t b2 = block_of(unit + 2 * kCodeWarps);
                if (!(ok = wait_long(is_v ? &S.v_empty[st] : &S.k_empty[st], phase ^ 1, abort, p.err))) break;
                if (is_v) {
#pragma unroll
                    for (int y = 0; y < kVLoads; ++y)
                        store_codes(S.v[st] + (32 * y + lane) * 128, 2 * grp, lane, codes[y]);
                } else {
#pragma unroll
                    for (int y = 0; y < kKLoads; ++y)
                        store_codes(S.k[st] + (y >> 1) * (KT * 128) + (grp * 16 + (y & 1) * 8 + g) * 128, 2 * c, g, codes[y]);
                    if (lane == 0) {
                        const float v1 = vr < kRangeFloor ? kRangeFloor : vr;
                        S.f[u % kScaleRing][grp] = __fdiv_rn(kr, 127.0f);
                        S.lv[u % kScaleRing][grp] = vr == -1.0f ? neg_inf() : kr != kr ? kr : log2f(__fdiv_rn(v1, 127.0f));
                        S.iv[u % kScaleRing][grp] = vr == -1.0f ? 0.0f : __fdiv_rn(127.0f, v1);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(is_v ? &S.v_full[st] : &S.k_full[st]);
                if (unit + kCodeWarps < end) load(unit + kCodeWarps, b1);
                b1 = b2;
            }
            first = end;
        }
    } else {
        // ---------------------------------------------------------- MMA
        // Counts come through warp reductions: uniform registers, which the MMAs take
        // (an MMA whose descriptors sit in ordinary registers takes 100 cycles to issue,
        // twice its time).
        constexpr uint32_t is = idesc_f16(128, KT), io = idesc_f16(128, DV);
        const uint64_t q0 = smem_desc(smem_u32(S.q[0]), 16, 1024, 2);
        const uint32_t desc_hi = (uint32_t)(q0 >> 32), q_lo = (uint32_t)q0,
                       k_lo = q_lo + (uint32_t)((S.k[0] - S.q[0]) >> 4), v_lo = q_lo + (uint32_t)((S.v[0] - S.q[0]) >> 4);
        bool issued = false;
        uint32_t u = 0, items[2] = {0, 0}, asked[2] = {0, 0}, used[2] = {0, 0};   // tiles whose scores / P of m, so far
        auto scores = [&](int m, uint32_t st) {
            const uint32_t b = asked[m]++ & 1, d = tmem + m * 128 + 64 * b;
            const uint32_t qa = q_lo + ((m * Sm::kQ) >> 4), ka = k_lo + st * (Sm::kK >> 4);
#pragma unroll
            for (int x = 0; x < DK / 16; ++x)
                warp_mma_f16_ss(d, qa + ((x >> 2) * (128 * 128) >> 4) + 2 * (x & 3),
                                ka + ((x >> 2) * (KT * 128) >> 4) + 2 * (x & 3), desc_hi, is, x != 0);
            warp_commit(&S.s_full[m][b]);
            // this warp has seen the stage's codes: its arrival passes the scales on too
            if (lane == 0) mbar_arrive(&S.s_full[m][b]);
            issued = true;
        };
        while (ok && next_item(p, lo, hi, span, few, r, it)) {
            const int nt = __reduce_max_sync(0xffffffffu, (it.keys + KT - 1) / KT);
            const bool two = __any_sync(0xffffffffu, it.cnt > tq);           // both query tiles have tokens
            for (int j = 0; j < 2 && j < nt && ok; ++j) {          // the first two tiles' scores
                const uint32_t st = (u + j) % kStages;
                if (!(ok = wait_long(&S.k_full[st], ((u + j) / kStages) & 1, abort, p.err))) break;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    if (!ok || (m == 1 && !two)) break;
                    if (j == 0 && !(ok = wait_long(&S.q_full[m], items[m]++ & 1, abort, p.err))) break;
                    tc_fence_after();
                    scores(m, st);
                }
                if (ok) warp_commit(&S.k_empty[st]);
            }
            for (int j = 0; j < nt && ok; ++j, ++u) {
                const uint32_t st = u % kStages, st2 = (u + 2) % kStages;
                if (!(ok = wait_long(&S.v_full[st], (u / kStages) & 1, abort, p.err))) break;
                if (j + 2 < nt && !(ok = wait_long(&S.k_full[st2], ((u + 2) / kStages) & 1, abort, p.err))) break;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    if (m == 1 && !two) break;
                    const uint32_t b = used[m] & 1;
                    if (!(ok = wait_long(&S.p_full[m][b], (used[m] >> 1) & 1, abort, p.err))) break;
                    ++used[m];
                    tc_fence_after();
                    const uint32_t d = tmem + kOCol + m * 128, pa = tmem + m * 128 + 64 * b, va = v_lo + st * (Sm::kV >> 4);
#pragma unroll
                    for (int x = 0; x < KT / 16; ++x)
                        warp_mma_f16_ts(d, pa + 8 * x, va + 2 * x, desc_hi, io, (j | x) != 0);
                    warp_commit(&S.pv_done[m][b]);
                    issued = true;
                    if (j + 2 < nt) scores(m, st2);                // in order after P V: its buffer is free
                }
                if (!ok) break;
                warp_commit(&S.v_empty[st]);
                if (j + 2 < nt) warp_commit(&S.k_empty[st2]);
            }
        }
        // every MMA issued so far completes before TMEM is freed
        if (issued) {
            warp_commit(&S.drain);
            for (uint32_t n = 0; n < kMaxWaitProbes; ++n)
                if (__all_sync(0xffffffffu, mbar_try_wait(&S.drain, 0))) break;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    QMOE_PDL_WAIT();
}

template <int DK, int DV>
cudaError_t launch_dims(const AttendParams &p, int few, cudaStream_t s) {
    const int G = p.heads / p.c.heads, gq = G < 128 ? G : 128, tq = 128 / gq, hgroups = (G + gq - 1) / gq;
    const size_t smem = sizeof(Shared<DK, DV>) + 1024;
    auto kernel = attend_prompt_kernel<DK, DV>;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    // Batches that leave SMs idle: one query tile an item, windows of fewer rows
    // (649 tokens after 1112, 8 kv heads 48 -> 40 us; 2 requests of some 20 tokens
    // 29 -> 19 us; nothing where the SMs are full).
    const int64_t groups = (int64_t)p.c.heads * hgroups, sms = device_sm_count();
    const int span = p.T * groups <= sms * tq ? tq : 2 * tq;
    const int64_t even = (p.T * groups + sms - 1) / sms;
    // never above span: a window holds one item of a request
    const int rows = even >= span || span < 16 ? span : even < 16 ? 16 : (int)even;
    const int64_t windows = (p.T + rows - 1) / rows;
    return launch_pdl(kernel, dim3((unsigned)(windows * groups)), dim3(kThreads), smem, s, p, tq, span, rows, gq, hgroups,
                      few);
}

}  // namespace

cudaError_t launch_attend_prompt(const AttendParams &p, int few, cudaStream_t s) {
    if (p.c.k_dim == 64) return launch_dims<64, 64>(p, few, s);
    if (p.c.k_dim == 128) return launch_dims<128, 128>(p, few, s);
    return launch_dims<192, 128>(p, few, s);
}

}  // namespace qmoe
