// attend_prompt.cu -- attention over the 8-bit cache for prompts: requests with
// more tokens than attend.cu's rows hold, bf16 activations.
//
// The arithmetic is attend.cu's (its head says how): scores on codes, the
// blocks' scales folded into t = (q . ck) * f + log2(rv / 127), P = 2^(t - M) in
// fp16, f32 sums.  What differs is where it runs.  A CTA takes 256 query rows
// (two tiles of 128: tq tokens by the heads that share a kv head) and goes once
// over their keys in tiles of KT tokens:
//
//   warps 0-3, 4-7   one row of a query tile a thread: q to fp16 in shared
//                    memory, then per key tile the scores from tensor memory,
//                    the running maximum and sum, P back to tensor memory
//   warps 8-11       codes from the cache to fp16 operands in shared memory
//                    (K [token][dim], V [dim][token], 128-byte swizzle), the
//                    16-token groups' scales beside them
//   warp 12          tcgen05: S = q K^T (both operands in shared memory), then
//                    O += P V (P from tensor memory), the two query tiles in
//                    turn, so that one's softmax runs under the other's MMAs
//
// O stays in tensor memory.  It is rescaled only where a row's maximum has
// grown by more than 2^8 since it was last scaled; until then P may reach
// 2^(8 + 6), which fp16 holds.  Work is bound by the exponentials (a quarter of
// an MMA's elements a cycle) and the MMAs alike: 2048 cycles each for 256 rows
// by 128 keys of 128 dims.
#include "attend.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace qmoe {
namespace {

using namespace sm100;

constexpr int kSoftWarps = 8;
constexpr int kCodeWarp0 = 8, kCodeWarps = 4;
constexpr int kMmaWarp = 12;
constexpr int kThreads = 13 * 32;
constexpr float kGrow = 8.0f;                 // log2 of how far a maximum may outgrow the scaling
constexpr float kShift = 6.0f;                // P = 2^6 at the scaling's maximum
constexpr int kScaleRing = 4;                 // tiles whose scales are kept: the codes run at most
                                              // two tiles ahead of the softmax

template <int DK, int DV, int KT>
struct Shared {
    static constexpr int kQ = 128 * DK * 2, kK = KT * DK * 2, kV = DV * KT * 2;
    uint8_t q[2][kQ];
    uint8_t k[2][kK];
    uint8_t v[2][kV];
    float f[kScaleRing][KT / 16], lv[kScaleRing][KT / 16], iv[kScaleRing][KT / 16];
    uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t scale_full[kScaleRing];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) {
    return (1u << 4)          // D = f32; A, B = f16 (format 0)
           | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

QMOE_DEV void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T.
QMOE_DEV void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    mma_bf16_ts(d_tmem, a_tmem, b_desc, idesc, accumulate);   // kind::f16; idesc says which type
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

// 2 * tq tokens of a request that begin in a window of as many rows of q.
struct Item {
    int64_t request;
    int t0, cnt;                              // first row of q, tokens
    int pos0;                                 // last key of the first token
    int keys;                                 // of the last token
};

// The item of the first request from `r` on that has one in the window; false
// when there is none.  Requests of up to `few` tokens are attend.cu's.  The
// whole warp alike.
QMOE_DEV bool next_item(const AttendParams &p, int64_t lo, int span, int few, int64_t &r, Item &it) {
    const int lane = threadIdx.x & 31;
    const int64_t hi = lo + span < p.T ? lo + span : p.T;
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

template <int DK, int DV, int KT>
__global__ void __launch_bounds__(kThreads, 1)
attend_prompt_kernel(const AttendParams p, const int tq, const int gq, const int hgroups, const int few) {
    using Sm = Shared<DK, DV, KT>;
    extern __shared__ uint8_t smem_raw[];
    Sm &S = *reinterpret_cast<Sm *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    // late windows first: their rows see the most keys
    const int span = 2 * tq;
    const int64_t lo = (int64_t)(gridDim.x - 1 - blockIdx.x) * span;
    const int h = blockIdx.y / hgroups, hg = blockIdx.y - h * hgroups, G = p.heads / p.c.heads;
    const int head0 = h * G + hg * gq, heads_here = G - hg * gq < gq ? G - hg * gq : gq;
    int64_t r = first_request(p.q_start, p.R, lo);
    const int64_t r0 = r;
    Item it;
    if (!next_item(p, lo, span, few, r, it)) return;      // the whole CTA alike

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.q_full[i], 4);
            mbar_init(&S.s_full[i], 1);
            mbar_init(&S.p_full[i], 4);
            mbar_init(&S.o_full[i], 1);
            mbar_init(&S.k_full[i], kCodeWarps);
            mbar_init(&S.k_empty[i], 1);
            mbar_init(&S.v_full[i], kCodeWarps);
            mbar_init(&S.v_empty[i], 1);
        }
        for (int i = 0; i < kScaleRing; ++i) mbar_init(&S.scale_full[i], 1);
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
    const uint32_t tmem = S.tmem_base;
    constexpr uint32_t kSCol = 128, kOCol = 256;      // S (and P in its first half) of tile m at 128 m, O at 256 + 128 m
    volatile int *abort = &S.abort;
    bool ok = true;
    uint32_t u = 0;                                   // key tiles so far
    uint32_t items[2] = {0, 0};                       // items with query tile m so far
    uint32_t tiles[2] = {0, 0};                       // key tiles with query tile m so far
    r = r0;

    if (warp < kSoftWarps) {
        // ---------------------------------------------------------- softmax
        const int m = warp >> 2, q = warp & 3, row = q * 32 + lane;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const uint32_t s_at = tmem + lanes + m * kSCol, o_at = tmem + lanes + kOCol + m * 128;
        while (ok && next_item(p, lo, span, few, r, it)) {
            const int cnt = it.cnt - m * tq < tq ? it.cnt - m * tq : tq;      // tokens of this query tile
            const int nt = (it.keys + KT - 1) / KT;
            const int i = row / gq, gg = row - i * gq;
            const bool live = i < cnt && gg < heads_here;
            const int64_t tok = (int64_t)it.t0 + m * tq + i;
            const int64_t out_at = tok * p.ldo + (int64_t)(head0 + gg) * DV;
            if (nt == 0 || cnt <= 0) {
                if (live)
                    for (int d = 0; d < DV; ++d) reinterpret_cast<__nv_bfloat16 *>(p.out)[out_at + d] = __float2bfloat16_rn(0.0f);
                u += nt;
                continue;
            }
            // q: the row by a power of two, as fp16, 64 dims a 128-byte row
            float back;
            {
                const int64_t at = live ? tok * p.ldq + (int64_t)(head0 + gg) * DK : 0;
                float mx = 0.0f;
                if (live)
                    for (int d = 0; d < DK; d += 4) {
                        const float4 v = load_q4(p, at + d);
                        mx = max_abs(max_abs(max_abs(max_abs(mx, v.x), v.y), v.z), v.w);
                    }
                const int e = q_exponent(mx);
                const float up = pow2i(14 - e);
                back = pow2i(e - 14);
                for (int d = 0; d < DK; d += 8) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (live) {
                        const float4 a = load_q4(p, at + d), b = load_q4(p, at + d + 4);
                        w = make_uint4(h2(a.x * up, a.y * up), h2(a.z * up, a.w * up), h2(b.x * up, b.y * up),
                                       h2(b.z * up, b.w * up));
                    }
                    *reinterpret_cast<uint4 *>(S.q[m] + (d >> 6) * (128 * 128) + row * 128 +
                                               ((((d >> 3) & 7) ^ (row & 7)) << 4)) = w;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.q_full[m]);
            const int last = live ? it.pos0 + m * tq + i : -1;               // this row's last key
            const int first_last = it.pos0 + m * tq;                         // the first token's
            float mx = neg_inf(), sum = 0.0f;                                // mx: what O and sum are scaled to
            for (int j = 0; j < nt; ++j, ++u, ++tiles[m]) {
                if (!(ok = mbar_wait_warp(&S.s_full[m], tiles[m] & 1, abort, p.err))) break;
                // complete by now (the codes came after it): the wait orders the reads behind it
                if (!(ok = mbar_wait_warp(&S.scale_full[u % kScaleRing], (u / kScaleRing) & 1, abort, p.err))) break;
                tc_fence_after();
                const float *f = S.f[u % kScaleRing], *lv = S.lv[u % kScaleRing], *iv = S.iv[u % kScaleRing];
                const int see = last - j * KT;                               // columns 0 .. see are visible
                const bool whole = j * KT + KT - 1 <= first_last && j * KT + KT <= it.keys;
                float top = neg_inf();
#pragma unroll
                for (int c = 0; c < KT; c += 32) {
                    uint32_t v[32];
                    tmem_ld_x32(s_at + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float a = f[c / 16 + half] * back, b = lv[c / 16 + half];
                        if (whole) {
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                top = fmaxf(top, __fmaf_rn(__uint_as_float(v[16 * half + x]), a, b));
                        } else {
#pragma unroll
                            for (int x = 0; x < 16; ++x) {
                                const float t = __fmaf_rn(__uint_as_float(v[16 * half + x]), a, b);
                                top = c + 16 * half + x <= see ? fmaxf(top, t) : top;
                            }
                        }
                    }
                }
                if (__any_sync(0xffffffffu, top > mx + kGrow)) {             // also the first tile: mx is -inf
                    const float to = top > mx ? top : mx;
                    const float by = to == neg_inf() ? 1.0f : ex2(mx - to);
                    mx = to;
                    sum *= by;
                    if (j > 0) {
#pragma unroll
                        for (int c = 0; c < DV; c += 32) {
                            uint32_t o[32];
                            tmem_ld_x32(o_at + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * by);
                            tmem_st_x32(o_at + c, o);
                        }
                    }
                }
                const float base = mx == neg_inf() ? 0.0f : mx - kShift;
#pragma unroll
                for (int c = 0; c < KT; c += 32) {
                    uint32_t v[32], w[16];
                    tmem_ld_x32(s_at + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float a = f[c / 16 + half] * back, b = lv[c / 16 + half] - base;
                        float part = 0.0f;
#pragma unroll
                        for (int x = 0; x < 16; x += 2) {
                            float t0 = __fmaf_rn(__uint_as_float(v[16 * half + x]), a, b);
                            float t1 = __fmaf_rn(__uint_as_float(v[16 * half + x + 1]), a, b);
                            if (!whole) {
                                t0 = c + 16 * half + x <= see ? t0 : neg_inf();
                                t1 = c + 16 * half + x + 1 <= see ? t1 : neg_inf();
                            }
                            t0 = ex2(t0);
                            t1 = ex2(t1);
                            part += t0 + t1;
                            w[8 * half + x / 2] = h2(t0, t1);
                        }
                        sum = __fmaf_rn(part, iv[c / 16 + half], sum);
                    }
                    tmem_st_x16(s_at + c / 2, w);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.p_full[m]);
            }
            if (!ok) break;
            if (!(ok = mbar_wait_warp(&S.o_full[m], items[m] & 1, abort, p.err))) break;
            ++items[m];
            tc_fence_after();
            const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
            const bool wide = p.vec_out;
#pragma unroll
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
                            const __nv_bfloat162 b = __floats2bfloat162_rn(
                                sum == 0.0f ? 0.0f : __uint_as_float(o[x + 2 * y]) * inv,
                                sum == 0.0f ? 0.0f : __uint_as_float(o[x + 2 * y + 1]) * inv);
                            w[y] = *reinterpret_cast<const uint32_t *>(&b);
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
        constexpr int kKLoads = KT / 8 / kCodeWarps * (DK / 64);   // 8 tokens by 64 dims a load of the warp
        constexpr int kVLoads = KT / 16 * (DV / 32) / kCodeWarps;  // 32 dims of a group of 16 tokens
        const int w = warp - kCodeWarp0, g = lane >> 2, c = lane & 3;
        while (ok && next_item(p, lo, span, few, r, it)) {
            const int nt = (it.keys + KT - 1) / KT;
            const int32_t *table = p.table + it.request * p.max_blocks;
            auto block_of = [&](int tok) -> int64_t {
                if (tok >= it.keys) return -1;
                const int64_t b = table[block_index(p, tok)];
                return b >= 0 && b < p.c.num_blocks ? b * p.c.heads + h : -1;
            };
            // lane x's group x of a tile: its block, one tile ahead
            int64_t ahead = lane < KT / 16 ? block_of(16 * lane) : -1;
            for (int j = 0; j < nt; ++j, ++u) {
                const int64_t mine = ahead;
                ahead = lane < KT / 16 && j + 1 < nt ? block_of((j + 1) * KT + 16 * lane) : -1;
                uint4 kc[kKLoads], vc[kVLoads];
#pragma unroll
                for (int x = 0; x < kKLoads; ++x) {
                    const int J = x % (DK / 64), t = (w + kCodeWarps * (x / (DK / 64))) * 8 + g;   // dims 64 J, token t
                    const int64_t bh = __shfl_sync(0xffffffffu, mine, t >> 4);
                    const int tok = j * KT + t, off = tok - block_index(p, tok) * p.c.block;
                    kc[x] = bh >= 0 ? ldg_code(p.c.k + ((bh * (DK / 64) + J) * p.c.block + off) * 64 + c * 16)
                                    : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int x = 0; x < kVLoads; ++x) {
                    const int grp = w + kCodeWarps * (x / (DV / 32)), d = (x % (DV / 32)) * 32 + lane;
                    const int64_t bh = __shfl_sync(0xffffffffu, mine, grp);
                    const int tok = j * KT + 16 * grp, off = tok - block_index(p, tok) * p.c.block;
                    vc[x] = bh >= 0 ? ldg_code(p.c.v + ((bh * (p.c.block / 16) + off / 16) * DV + d) * 16)
                                    : make_uint4(0, 0, 0, 0);
                }
                // The groups' scales.  Their slot was the tile's four back: the softmax is done
                // with it, since this warp has seen the scores of the tile three back finished
                // (the last wait for an empty K), and those wait for that tile's P.
                if (w == 0) {
                    float kr = 0.0f, vr = 127.0f;
                    if (mine >= 0) {
                        kr = p.c.k_range[mine];
                        vr = p.c.v_range[mine];
                    }
                    vr = vr < kRangeFloor ? kRangeFloor : vr;
                    if (lane < KT / 16) {
                        S.f[u % kScaleRing][lane] = __fdiv_rn(kr, 127.0f) * (p.scale * kLog2e);
                        S.lv[u % kScaleRing][lane] = mine >= 0 ? log2f(__fdiv_rn(vr, 127.0f)) : neg_inf();
                        S.iv[u % kScaleRing][lane] = mine >= 0 ? __fdiv_rn(127.0f, vr) : 0.0f;
                    }
                    __syncwarp();
                }
                const uint32_t st = u & 1;
                if (!(ok = mbar_wait_warp(&S.k_empty[st], ((u >> 1) & 1) ^ 1, abort, p.err))) break;
                if (w == 0 && lane == 0) mbar_arrive(&S.scale_full[u % kScaleRing]);
#pragma unroll
                for (int x = 0; x < kKLoads; ++x) {
                    const int J = x % (DK / 64), t = (w + kCodeWarps * (x / (DK / 64))) * 8 + g;
                    store_codes(S.k[st] + J * (KT * 128) + t * 128, 2 * c, t, kc[x]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.k_full[st]);
                if (!(ok = mbar_wait_warp(&S.v_empty[st], ((u >> 1) & 1) ^ 1, abort, p.err))) break;
#pragma unroll
                for (int x = 0; x < kVLoads; ++x) {
                    const int grp = w + kCodeWarps * (x / (DV / 32)), d = (x % (DV / 32)) * 32 + lane;
                    store_codes(S.v[st] + (grp >> 2) * (DV * 128) + d * 128, 2 * (grp & 3), d, vc[x]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.v_full[st]);
            }
        }
    } else {
        // ---------------------------------------------------------- MMA
        const uint32_t is = idesc_f16(128, KT), io = idesc_f16(128, DV);
        const uint64_t q0 = smem_desc(smem_u32(S.q[0]), 16, 1024, 2), k0 = smem_desc(smem_u32(S.k[0]), 16, 1024, 2),
                       v0 = smem_desc(smem_u32(S.v[0]), 16, 1024, 2);
        bool issued = false;
        auto scores = [&](int m, uint32_t st) {
            if (lane == 0) {
#pragma unroll
                for (int x = 0; x < DK / 16; ++x)
                    mma_f16_ss(tmem + m * kSCol, q0 + ((m * Sm::kQ + (x >> 2) * (128 * 128)) >> 4) + 2 * (x & 3),
                               k0 + ((st * Sm::kK + (x >> 2) * (KT * 128)) >> 4) + 2 * (x & 3), is, x != 0);
                mma_commit(&S.s_full[m]);
            }
            issued = true;
        };
        while (ok && next_item(p, lo, span, few, r, it)) {
            const int nt = (it.keys + KT - 1) / KT;
            const int both = it.cnt > tq ? 2 : 1;                  // query tiles with tokens
            for (int j = 0; j < nt && ok; ++j, ++u) {
                const uint32_t st = u & 1, st1 = st ^ 1;
                if (j == 0) {
                    if (!(ok = mbar_wait_warp(&S.k_full[st], (u >> 1) & 1, abort, p.err))) break;
                    for (int m = 0; m < both; ++m) {
                        if (!(ok = mbar_wait_warp(&S.q_full[m], items[m] & 1, abort, p.err))) break;
                        tc_fence_after();
                        scores(m, st);
                    }
                    if (!ok) break;
                    if (lane == 0) mma_commit(&S.k_empty[st]);
                }
                if (!(ok = mbar_wait_warp(&S.v_full[st], (u >> 1) & 1, abort, p.err))) break;
                for (int m = 0; m < both; ++m) {
                    if (!(ok = mbar_wait_warp(&S.p_full[m], tiles[m] & 1, abort, p.err))) break;
                    ++tiles[m];
                    tc_fence_after();
                    if (lane == 0)
#pragma unroll
                        for (int x = 0; x < KT / 16; ++x)
                            mma_f16_ts(tmem + kOCol + m * 128, tmem + m * kSCol + 8 * x,
                                       v0 + ((st * Sm::kV + (x >> 2) * (DV * 128)) >> 4) + 2 * (x & 3), io, (j | x) != 0);
                    if (j + 1 < nt) {
                        if (m == 0 && !(ok = mbar_wait_warp(&S.k_full[st1], ((u + 1) >> 1) & 1, abort, p.err))) break;
                        tc_fence_after();
                        scores(m, st1);
                    } else {
                        if (lane == 0) mma_commit(&S.o_full[m]);
                        ++items[m];
                    }
                }
                if (!ok) break;
                if (lane == 0) {
                    mma_commit(&S.v_empty[st]);
                    if (j + 1 < nt) mma_commit(&S.k_empty[st1]);
                }
            }
        }
        // every MMA issued so far completes before TMEM is freed
        if (issued) {
            if (lane == 0) mma_commit(&S.drain);
            __syncwarp();
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
}

template <int DK, int DV, int KT>
cudaError_t launch_dims(const AttendParams &p, int few, cudaStream_t s) {
    const int G = p.heads / p.c.heads, gq = G < 128 ? G : 128, tq = 128 / gq, hgroups = (G + gq - 1) / gq;
    const size_t smem = sizeof(Shared<DK, DV, KT>) + 1024;
    auto kernel = attend_prompt_kernel<DK, DV, KT>;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)((p.T + 2 * tq - 1) / (2 * tq)), (unsigned)(p.c.heads * hgroups)),
                      dim3(kThreads), smem, s, p, tq, gq, hgroups, few);
}

}  // namespace

cudaError_t launch_attend_prompt(const AttendParams &p, int few, cudaStream_t s) {
    if (p.c.k_dim == 64) return launch_dims<64, 64, 128>(p, few, s);
    if (p.c.k_dim == 128) return launch_dims<128, 128, 128>(p, few, s);
    return launch_dims<192, 128, 64>(p, few, s);   // q of two tiles takes 96 KB
}

}  // namespace qmoe
