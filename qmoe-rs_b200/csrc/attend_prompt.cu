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
#include "mma_warp.cuh"

namespace qmoe {
namespace {

using namespace sm100;

constexpr int kSoftWarps = 8;
constexpr int kCodeWarp0 = 8, kCodeWarps = 4;
constexpr int kMmaWarp = 12;
constexpr int kThreads = 16 * 32;             // warps 13-15 only give their registers up
// Registers a thread: the softmax holds a row's scores of a tile.  Of the 128 a
// thread that the CTA is launched with, 2 * 168 + 112 + 64 = 4 * 128.
constexpr int kSoftRegs = 168, kCodeRegs = 112, kMmaRegs = 64;
static_assert(2 * kSoftRegs + kCodeRegs + kMmaRegs <= 512, "registers of the CTA");
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

template <int N>
QMOE_DEV void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
QMOE_DEV void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
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
        for (int i = 0; i < kScaleRing; ++i) mbar_init(&S.scale_full[i], kCodeWarps);
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
        more_registers<kSoftRegs>();
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
                // nothing to see: zeros, a row a warp at a time
                for (int x = 0; x < 32 && cnt > 0; ++x) {
                    const int64_t at = __shfl_sync(0xffffffffu, live ? out_at : -1, x);
                    if (at >= 0)
                        for (int d = lane; d < DV; d += 32) reinterpret_cast<__nv_bfloat16 *>(p.out)[at + d] = __float2bfloat16_rn(0.0f);
                }
                u += nt;
                continue;
            }
            // q: rows by a power of two, as fp16, 64 dims a 128-byte row; four of the
            // warp's rows at a time, four dims a lane
            float back = 0.0f;
            constexpr int kRep = (DK + 127) / 128;
#pragma unroll 1
            for (int x = 0; x < 32; x += 4) {
                float4 v[4][kRep];
                const int64_t mine = live ? tok * p.ldq + (int64_t)(head0 + gg) * DK : -1;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int64_t at = __shfl_sync(0xffffffffu, mine, x + y);
#pragma unroll
                    for (int z = 0; z < kRep; ++z) {
                        const int d = 4 * lane + 128 * z;
                        v[y][z] = at >= 0 && d < DK ? load_q4(p, at + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    float mx = 0.0f;
#pragma unroll
                    for (int z = 0; z < kRep; ++z)
                        mx = max_abs(max_abs(max_abs(max_abs(mx, v[y][z].x), v[y][z].y), v[y][z].z), v[y][z].w);
                    const int e = q_exponent(warp_max(mx)), at = q * 32 + x + y;
                    const float up = pow2i(14 - e);
                    if (lane == x + y) back = pow2i(e - 14);
#pragma unroll
                    for (int z = 0; z < kRep; ++z) {
                        const int d = 4 * lane + 128 * z;
                        if (d < DK)
                            *reinterpret_cast<uint2 *>(S.q[m] + (d >> 6) * (128 * 128) + at * 128 +
                                                       ((((d >> 3) & 7) ^ (at & 7)) << 4) + 2 * (d & 4)) =
                                make_uint2(h2(v[y][z].x * up, v[y][z].y * up), h2(v[y][z].z * up, v[y][z].w * up));
                    }
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
                uint32_t t[KT / 32][32];
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) tmem_ld_x32(s_at + 32 * c, t[c]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < KT / 32; ++c)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float a = f[2 * c + half] * back, b = lv[2 * c + half];
#pragma unroll
                        for (int x = 16 * half; x < 16 * half + 16; ++x)
                            t[c][x] = __float_as_uint(__fmaf_rn(__uint_as_float(t[c][x]), a, b));
                    }
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c)
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (32 * c + x > see) t[c][x] = 0xff800000u;     // -inf
                }
                float tops[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
                for (int c = 0; c < KT / 32; ++c)
#pragma unroll
                    for (int x = 0; x < 32; ++x) tops[x & 3] = fmaxf(tops[x & 3], __uint_as_float(t[c][x]));
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                if (__any_sync(0xffffffffu, top > mx + kGrow)) {             // also the first tile: mx is -inf
                    const float to = top > mx ? top : mx;
                    const float by = to == neg_inf() ? 1.0f : ex2(mx - to);
                    mx = to;
                    sum *= by;
                    if (j > 0) {
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
                }
                const float base = mx == neg_inf() ? 0.0f : mx - kShift;
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float part = 0.0f;
#pragma unroll
                        for (int x = 16 * half; x < 16 * half + 16; x += 2) {
                            const float t0 = ex2(__uint_as_float(t[c][x]) - base), t1 = ex2(__uint_as_float(t[c][x + 1]) - base);
                            part += t0 + t1;
                            w[x / 2] = h2(t0, t1);
                        }
                        sum = __fmaf_rn(part, iv[2 * c + half], sum);
                    }
                    tmem_st_x16(s_at + 16 * c, w);
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
        fewer_registers<kCodeRegs>();
        // Warp w has groups kOwn w .. of 16 tokens: of each the loads are 8 tokens by 64
        // dims of K, 32 dims of V.  K of the next tile is loaded while V of this one is
        // converted, and V while K is; the blocks are looked up two tiles ahead.
        constexpr int kOwn = KT / 16 / kCodeWarps, kKLoads = 2 * (DK / 64), kVLoads = DV / 32;
        const int w = warp - kCodeWarp0, g = lane >> 2, c = lane & 3;
        const int bs = p.c.block;
        while (ok && next_item(p, lo, span, few, r, it)) {
            const int nt = (it.keys + KT - 1) / KT;
            const int32_t *table = p.table + it.request * p.max_blocks;
            // the block and head of this warp's group x of tile j
            auto block_of = [&](int j, int x) -> int64_t {
                const int tok = j * KT + (w * kOwn + x) * 16;
                if (tok >= it.keys) return -1;
                const int64_t b = table[block_index(p, tok)];
                return b >= 0 && b < p.c.num_blocks ? b * p.c.heads + h : -1;
            };
            auto off_of = [&](int j, int x) {
                const int tok = j * KT + (w * kOwn + x) * 16;
                return tok - block_index(p, tok) * bs;
            };
            uint4 kc[kOwn][kKLoads], vc[kOwn][kVLoads];
            auto load_k = [&](int j, const int64_t (&bh)[kOwn]) {
#pragma unroll
                for (int x = 0; x < kOwn; ++x) {
                    const int8_t *at = p.c.k + (bh[x] * (DK / 64) * bs + off_of(j, x) + g) * 64 + c * 16;
#pragma unroll
                    for (int y = 0; y < kKLoads; ++y)
                        kc[x][y] = bh[x] >= 0 ? ldg_code(at + (y >> 1) * bs * 64 + (y & 1) * 512) : make_uint4(0, 0, 0, 0);
                }
            };
            auto load_v = [&](int j, const int64_t (&bh)[kOwn]) {
#pragma unroll
                for (int x = 0; x < kOwn; ++x) {
                    const int8_t *at = p.c.v + ((bh[x] * (bs / 16) + off_of(j, x) / 16) * DV + lane) * 16;
#pragma unroll
                    for (int y = 0; y < kVLoads; ++y)
                        vc[x][y] = bh[x] >= 0 ? ldg_code(at + y * 512) : make_uint4(0, 0, 0, 0);
                }
            };
            int64_t b0[kOwn], b1[kOwn], b2[kOwn];                    // of this tile, the next, the one after
#pragma unroll
            for (int x = 0; x < kOwn; ++x) {
                b0[x] = block_of(0, x);
                b1[x] = block_of(1, x);
            }
            float kr = 0.0f, vr = 127.0f;                           // ranges of group `lane` of the warp's
            auto load_ranges = [&](const int64_t (&bh)[kOwn]) {
                int64_t mine = -1;
#pragma unroll
                for (int x = 0; x < kOwn; ++x) mine = lane == x ? bh[x] : mine;
                kr = mine >= 0 ? p.c.k_range[mine] : 0.0f;
                vr = mine >= 0 ? p.c.v_range[mine] : -1.0f;          // none
            };
            if (nt > 0) {
                load_k(0, b0);
                load_v(0, b0);
                load_ranges(b0);
            }
            for (int j = 0; j < nt; ++j, ++u) {
                const uint32_t st = u & 1;
#pragma unroll
                for (int x = 0; x < kOwn; ++x) b2[x] = block_of(j + 2, x);
                // The groups' scales.  Their slot was the tile's four back: the softmax is done
                // with it, since this warp has seen the scores of the tile three back finished
                // (the last wait for an empty K), and those wait for that tile's P.
                if (lane < kOwn) {
                    const bool none = vr == -1.0f;
                    const float v1 = vr < kRangeFloor ? kRangeFloor : vr;
                    S.f[u % kScaleRing][w * kOwn + lane] = __fdiv_rn(kr, 127.0f) * (p.scale * kLog2e);
                    S.lv[u % kScaleRing][w * kOwn + lane] = none ? neg_inf() : log2f(__fdiv_rn(v1, 127.0f));
                    S.iv[u % kScaleRing][w * kOwn + lane] = none ? 0.0f : __fdiv_rn(127.0f, v1);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.scale_full[u % kScaleRing]);
                if (!(ok = mbar_wait_warp(&S.k_empty[st], ((u >> 1) & 1) ^ 1, abort, p.err))) break;
#pragma unroll
                for (int x = 0; x < kOwn; ++x)
#pragma unroll
                    for (int y = 0; y < kKLoads; ++y) {
                        const int t = (w * kOwn + x) * 16 + (y & 1) * 8 + g;
                        store_codes(S.k[st] + (y >> 1) * (KT * 128) + t * 128, 2 * c, g, kc[x][y]);
                    }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.k_full[st]);
                if (j + 1 < nt) {
                    load_k(j + 1, b1);
                    load_ranges(b1);
                }
                if (!(ok = mbar_wait_warp(&S.v_empty[st], ((u >> 1) & 1) ^ 1, abort, p.err))) break;
#pragma unroll
                for (int x = 0; x < kOwn; ++x)
#pragma unroll
                    for (int y = 0; y < kVLoads; ++y) {
                        const int grp = w * kOwn + x, d = 32 * y + lane;
                        store_codes(S.v[st] + (grp >> 2) * (DV * 128) + d * 128, 2 * (grp & 3), lane, vc[x][y]);
                    }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.v_full[st]);
                if (j + 1 < nt) load_v(j + 1, b1);
#pragma unroll
                for (int x = 0; x < kOwn; ++x) {
                    b0[x] = b1[x];
                    b1[x] = b2[x];
                }
            }
        }
    } else if (fewer_registers<kMmaRegs>(), warp == kMmaWarp) {
        // ---------------------------------------------------------- MMA
        const uint32_t is = idesc_f16(128, KT), io = idesc_f16(128, DV);
        const uint64_t q0 = smem_desc(smem_u32(S.q[0]), 16, 1024, 2);
        const uint32_t desc_hi = (uint32_t)(q0 >> 32), q_lo = (uint32_t)q0,
                       k_lo = q_lo + (uint32_t)((S.k[0] - S.q[0]) >> 4), v_lo = q_lo + (uint32_t)((S.v[0] - S.q[0]) >> 4);
        bool issued = false;
        auto scores = [&](int m, uint32_t st) {
            const uint32_t d = tmem + m * kSCol, a = q_lo + ((m * Sm::kQ) >> 4), b = k_lo + ((st * Sm::kK) >> 4);
#pragma unroll
            for (int x = 0; x < DK / 16; ++x)
                warp_mma_f16_ss(d, a + ((x >> 2) * (128 * 128) >> 4) + 2 * (x & 3),
                                b + ((x >> 2) * (KT * 128) >> 4) + 2 * (x & 3), desc_hi, is, x != 0);
            warp_commit(&S.s_full[m]);
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
                    warp_commit(&S.k_empty[st]);
                }
                if (!(ok = mbar_wait_warp(&S.v_full[st], (u >> 1) & 1, abort, p.err))) break;
                for (int m = 0; m < both; ++m) {
                    if (!(ok = mbar_wait_warp(&S.p_full[m], tiles[m] & 1, abort, p.err))) break;
                    ++tiles[m];
                    tc_fence_after();
                    const uint32_t d = tmem + kOCol + m * 128, a = tmem + m * kSCol, b = v_lo + ((st * Sm::kV) >> 4);
#pragma unroll
                    for (int x = 0; x < KT / 16; ++x)
                        warp_mma_f16_ts(d, a + 8 * x, b + ((x >> 2) * (DV * 128) >> 4) + 2 * (x & 3), desc_hi, io, (j | x) != 0);
                    if (j + 1 < nt) {
                        if (m == 0 && !(ok = mbar_wait_warp(&S.k_full[st1], ((u + 1) >> 1) & 1, abort, p.err))) break;
                        tc_fence_after();
                        scores(m, st1);
                    } else {
                        warp_commit(&S.o_full[m]);
                        ++items[m];
                    }
                }
                if (!ok) break;
                warp_commit(&S.v_empty[st]);
                if (j + 1 < nt) warp_commit(&S.k_empty[st1]);
            }
        }
        // every MMA issued so far completes before TMEM is freed
        if (issued) {
            warp_commit(&S.drain);
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
