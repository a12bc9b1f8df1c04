// attend.cu -- attention over the 8-bit paged cache.
//
//   o[i] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j),
//   j <= kv_len - n + i for query i of the n of its request
//
// with k_j = ck_j * rk / 127 and v_j = cv_j * rv / 127, rk and rv constant over
// a block of tokens and head.  One pass over the keys with the running maximum
// and sum of the softmax.  The codes go to the tensor cores as fp16, exactly;
// the block's scales never multiply an element of K or V:
//   t = (q . ck) * (scale * log2(e) * rk / 127) + log2(rv / 127)
//   P = 2^(t - M), M the running maximum of t;  o = sum P cv / sum P * 127 / rv
// so each tile costs one FMA and one exp2 an element.  q is brought to fp16 by
// a power of two a row (exact for bf16 unless 2^-28 below the row's largest);
// with f32 activations q and P are the sums of two fp16 terms (22 bits).  The
// 64-token sums of P cv are added to the running ones in f32.
//
// The tensor cores form S^T = K q^T and O^T = V^T P^T (mma.m16n8k16): tokens,
// then dims, are the 16 rows, query rows (tokens x heads that share a kv head)
// the 8 columns, so that a single token with a few heads wastes little.  The
// layout of the cache is the operands': of a 64-token tile, lane 4 g + c takes
// the 16 bytes of K that are dims 16 c .. 16 c + 15 (of each 64) of its tokens
// and the 16 bytes of V that are tokens 16 c .. 16 c + 15 of its dims, and every
// 4 bytes of them are half of an A fragment.  Row r of token tile u is token
// 16 ((r % 8) / 2) + 4 u + 2 (r / 8) + r % 2: transposed eight by eight
// (movmatrix), the scores' fragments are then P^T's for those bytes of V, and a
// lane's scores all lie in one group of 16 tokens, hence in one block.
#include "attend.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace qmoe {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kPShift = 14.0f;              // P up to 2^14: fp16 keeps 2^-38 of the largest

QMOE_DEV void mma_f16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// 32-bit word t of v (t a constant after unrolling).
QMOE_DEV uint32_t word_of(const uint4 &v, int t) { return t == 0 ? v.x : t == 1 ? v.y : t == 2 ? v.z : v.w; }

// The request whose tiles of tq tokens hold slot `slot`.  With one token a tile
// the slots are the tokens: the last request that starts at or before it.  Else
// the tiles of request r start at start[r] / tq + r, which leaves each request
// room for a part of a tile more.  Both never fall with r; a warp looks at 32
// places at a time.
QMOE_DEV int64_t first_slot(const int32_t *start, int64_t r, int tq) { return tq == 1 ? start[r] : start[r] / tq + r; }

QMOE_DEV int64_t find_request(const int32_t *start, int64_t R, int64_t slot, int tq) {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, n = R;                       // the answer is in [lo, lo + n)
    while (n > 1) {
        const int64_t step = (n + 31) / 32;
        const int64_t i = lo + lane * step;
        const bool le = lane == 0 || (i < lo + n && first_slot(start, i, tq) <= slot);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
        const int64_t at = lo + last * step;
        n = lo + n - at < step ? lo + n - at : step;
        lo = at;
    }
    return lo;
}

// What the slots of a launch are: tokens, of requests with up to cut.few;
// requests with one token; `tiles` tiles of tq tokens for each request, of those
// with that many tokens at most; tiles of tq tokens of the requests with
// more than cut.few; tokens, of which every tq-th of such a request is one's.
enum class Slots { kTokens, kSingles, kFew, kTiles, kEvery };

struct Rows {                                    // of one CTA: rows of one request and kv head
    int64_t t0;                                  // token of row 0
    int tokens, head0;                           // row i * gq + g: token t0 + i, head head0 + g
    int pos0;                                    // last key of token t0 (may be negative)
    int keys;                                    // keys of the last token
    int64_t request;
    int64_t scratch;                             // row of scratch of token t0
};

QMOE_DEV bool find_rows(const AttendParams &p, int64_t slot, int tq, Slots kind, int tiles, Rows &w) {
    const bool by_request = kind == Slots::kSingles || kind == Slots::kFew;
    const int each = kind == Slots::kEvery ? 1 : tq;
    const int64_t r = kind == Slots::kFew ? slot / tiles : by_request ? slot : find_request(p.q_start, p.R, slot, each);
    const int64_t s0 = p.q_start[r], n = p.q_start[r + 1] - s0;
    if (kind == Slots::kSingles  ? n != 1
        : kind == Slots::kFew    ? n < 2 || n > tiles * tq
        : kind == Slots::kTokens ? n > p.cut.few
                                 : n <= p.cut.few)
        return false;
    const int64_t i0 = kind == Slots::kFew ? slot % tiles * tq : by_request ? 0 : (slot - (each == 1 ? s0 : s0 / tq + r)) * each;
    if (i0 < 0 || i0 >= n || s0 < 0 || (kind == Slots::kEvery && i0 % tq)) return false;
    int64_t cnt = n - i0 < tq ? n - i0 : tq;
    w.t0 = s0 + i0;
    if (w.t0 + cnt > p.T) cnt = p.T - w.t0;      // rows that the buffer does not hold
    if (cnt <= 0) return false;
    const int64_t most = p.max_blocks * p.c.block;
    const int64_t kv = p.kv_lens[r];
    const int64_t pos0 = (kv < 0 ? 0 : kv) - n + i0;
    const int64_t keys = pos0 + cnt;             // one past the last token's last key
    w.request = r;
    w.scratch = p.cut.by_token ? w.t0 : r * p.cut.few + i0;
    w.tokens = (int)cnt;
    w.pos0 = (int)(pos0 < -(1 << 30) ? -(1 << 30) : pos0);
    w.keys = (int)(keys < 0 ? 0 : keys > most ? most : keys);
    return true;
}

// Every warp keeps a ring of its own in shared memory: halves of a tile (the K
// of 64 tokens, then their V), fetched by bulk copies a 16-token group each,
// the next ones in flight while one is worked on.  16 tokens of V start 32
// bytes off a multiple of 128 from the ones before, so the lanes of a quarter
// warp (two dims, four groups) read 128 bytes of distinct banks.  Two halves a
// warp are enough with eight or twelve warps an SM (64 KB and more in flight);
// a third slot gained nothing.
constexpr int kSlots = 2;

template <int DK, int DV, int NT>
struct Shared {
    static constexpr int kVGroup = DV * 16 + 32;
    static constexpr int kSlot = (64 * DK > 4 * kVGroup ? 64 * DK : 4 * kVGroup);
    union {
        uint8_t ring[kWarps][kSlots][kSlot];
        float o[kWarps][8 * NT][DV + 4];         // once the ring is done with
    };
    float m[kWarps][8 * NT], l[kWarps][8 * NT];
    uint64_t full[kWarps][kSlots];
    int abort;
};

QMOE_DEV void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     sm100::smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
                 : "memory");
}

// Eight by eight 16-bit values, transposed.
QMOE_DEV uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Dims 64 J + 0 .. 15 from q[at] on.
template <int DK, bool BF16, bool VEC>
QMOE_DEV void load_row(const AttendParams &p, int64_t at, float (&v)[DK / 64][16]) {
#pragma unroll
    for (int J = 0; J < DK / 64; ++J)
#pragma unroll
        for (int d = 0; d < 16; d += 4) {
            const float4 f = load_q4<BF16, VEC>(p, at + 64 * J + d);
            v[J][d] = f.x;
            v[J][d + 1] = f.y;
            v[J][d + 2] = f.z;
            v[J][d + 3] = f.w;
        }
}

// A CTA's rows on NT * 8 columns: row i * gq + g of w.
template <int DK, int DV, bool BF16, int NT>
QMOE_DEV void attend_rows(const AttendParams &p, const Rows &w, int h, int split, int gq, int heads_here, Shared<DK, DV, NT> &S,
                          uint32_t &done) {
    constexpr int kTerms = BF16 ? 1 : 2;
    using Sm = Shared<DK, DV, NT>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int bs = p.c.block;

    const int tiles = (w.keys + 63) / 64;
    // pieces of cut.chunk tiles, larger where the request is longer than the host was told
    const int even = (tiles + p.splits - 1) / p.splits, chunk = p.cut.chunk > even ? p.cut.chunk : even;
    const int t_lo = split * chunk, t_hi = t_lo + chunk < tiles ? t_lo + chunk : tiles;
    const int mine = t_hi > t_lo + warp ? (t_hi - t_lo - warp + kWarps - 1) / kWarps : 0;   // tiles of this warp
    const int32_t *row_table = p.table + w.request * p.max_blocks;
    const int grp = g >> 1;                       // this lane's group of 16 tokens in a tile
    // the block and head of this lane's group of the warp's k-th tile, -1 past
    // the keys and where the table's entry is none
    auto block_of = [&](int k) -> int64_t {
        if (k >= mine) return -1;
        const int tok = (t_lo + warp + k * kWarps) * 64 + 16 * grp;
        if (tok >= w.keys) return -1;
        const int64_t b = row_table[block_index(p, tok)];
        return b >= 0 && b < p.c.num_blocks ? b * p.c.heads + h : -1;
    };
    // copies of item n (K of tile n / 2, or its V) into its slot (`done` items were
    // worked on before): an even lane g a piece of 64 dims each of K, or c = 0 its
    // group of V
    auto fetch = [&](int n, int64_t bh) {
        if (n >= 2 * mine) return;
        const int tok = (t_lo + warp + (n >> 1) * kWarps) * 64 + 16 * grp, off = tok - block_index(p, tok) * bs;
        uint8_t *dst = S.ring[warp][(done + n) % kSlots];
        uint64_t *bar = &S.full[warp][(done + n) % kSlots];
        const bool is_v = n & 1;
        const bool copy = bh >= 0 && (g & 1) == 0 && c < (is_v ? 1 : DK / 64);
        const uint32_t bytes = is_v ? DV * 16 : 1024;
        const uint32_t count = __popc(__ballot_sync(0xffffffffu, copy));
        if (lane == 0) sm100::mbar_arrive_expect_tx(bar, count * bytes);
        __syncwarp();
        if (copy) {
            if (is_v)
                bulk_load(dst + grp * Sm::kVGroup, p.c.v + (bh * (bs / 16) + off / 16) * (DV * 16), bytes, bar);
            else
                bulk_load(dst + c * 4096 + grp * 1024, p.c.k + ((bh * (DK / 64) + c) * bs + off) * 64, bytes, bar);
        }
    };

    int64_t blk = block_of(0), blk1 = block_of(1), blk2 = block_of(2);
    fetch(0, blk);
    fetch(1, blk);
    float kr = blk >= 0 ? p.c.k_range[blk] : 0.0f, vr = blk >= 0 ? p.c.v_range[blk] : 127.0f;

    // ---- q: rows brought to fp16 by a power of two, as B fragments: lane 4 g + c
    // has dims 64 J + 16 c + 4 t + {0, 1 | 2, 3} of row 8 x + g for step 4 J + t
    uint32_t qf[kTerms][NT][DK / 16][2];
    float back[NT][2];                            // scores to exponents, of this lane's columns 2 c, 2 c + 1
    int last[NT][2];                              // their last keys
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        const int row = 8 * x + g, i = row / gq, gg = row - i * gq;
        const bool live = i < w.tokens && gg < heads_here;
        const int64_t at = (live ? (w.t0 + i) * p.ldq + (int64_t)(w.head0 + gg) * DK : w.t0 * p.ldq) + 16 * c;
        float v[DK / 64][16];
        if (p.vec_q) load_row<DK, BF16, true>(p, at, v);
        else load_row<DK, BF16, false>(p, at, v);
        float m = 0.0f;
#pragma unroll
        for (int J = 0; J < DK / 64; ++J)
#pragma unroll
            for (int d = 0; d < 16; ++d) {
                v[J][d] = live ? v[J][d] : 0.0f;
                m = max_abs(m, v[J][d]);
            }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = q_exponent(m);
        const float up = pow2i(14 - e);
#pragma unroll
        for (int J = 0; J < DK / 64; ++J)
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float a = __fmul_rn(v[J][2 * t], up), b = __fmul_rn(v[J][2 * t + 1], up);
                const uint32_t hi = h2(a, b);
                qf[0][x][4 * J + t / 2][t & 1] = hi;
                if (kTerms == 2)
                    qf[kTerms - 1][x][4 * J + t / 2][t & 1] = h2(__fsub_rn(a, h_lo(hi)), __fsub_rn(b, h_hi(hi)));
            }
        const float down = pow2i(e - 14);
#pragma unroll
        for (int i = 0; i < 2; ++i) {             // row g's lanes 4 g .. have it: fetch those of the columns
            back[x][i] = __shfl_sync(0xffffffffu, down, 4 * (2 * c + i)) * (p.scale * kLog2e);
            last[x][i] = w.pos0 + (8 * x + 2 * c + i) / gq;
        }
    }

    float acc[DV / 16][NT][4];
#pragma unroll
    for (int t = 0; t < DV / 16; ++t)
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][x][i] = 0.0f;
    float mx[NT][2], sum[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[x][i] = neg_inf();
            sum[x][i] = 0.0f;
        }

    bool ok = true;
    int n = 0;                                    // items worked on
    for (int k = 0; k < mine; ++k) {
        const int tg = (t_lo + warp + k * kWarps) * 64 + 16 * grp + (g & 1);   // token of row g, tile u: tg + 4 u
        const float kr1 = blk1 >= 0 ? p.c.k_range[blk1] : 0.0f, vr1 = blk1 >= 0 ? p.c.v_range[blk1] : 127.0f;
        const int64_t blk3 = block_of(k + 3);
        // ---- scores, on the codes themselves.  (Left as 1152 + c, less 1152 sum q at
        // the end, they cost two instructions less for four: 64 ragged requests 96 us
        // instead of 100.  But the f32 sums then round at 1152 sum q, which for rows of
        // q with a mean is far above the score: up to 1 % in P.)  Two terms: the small
        // one first, and each 64 dims in sums of their own, added in f32.
        if (!(ok = sm100::mbar_wait_warp(&S.full[warp][(done + n) % kSlots], ((done + n) / kSlots) & 1, &S.abort, p.err))) break;
        const uint8_t *slot = S.ring[warp][(done + n) % kSlots] + (16 * grp + (g & 1)) * 64 + c * 16;
        float s[4][NT][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[u][x][i] = 0.0f;
#pragma unroll
        for (int J = 0; J < DK / 64; ++J) {
            uint4 kc[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) kc[j] = *reinterpret_cast<const uint4 *>(slot + J * 4096 + j * 128);
            if (kTerms == 1) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint4 a;
                        codes_to_half(word_of(kc[2 * u], t), a.x, a.z);
                        codes_to_half(word_of(kc[2 * u + 1], t), a.y, a.w);
#pragma unroll
                        for (int x = 0; x < NT; ++x) mma_f16(s[u][x], a, qf[0][x][4 * J + t][0], qf[0][x][4 * J + t][1]);
                    }
            } else {
                float part[4][NT][4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) part[u][x][i] = 0.0f;
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint4 a;
                        codes_to_half(word_of(kc[2 * u], t & 3), a.x, a.z);
                        codes_to_half(word_of(kc[2 * u + 1], t & 3), a.y, a.w);
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            const uint32_t(&b)[2] = qf[t < 4 ? kTerms - 1 : 0][x][4 * J + (t & 3)];
                            mma_f16(part[u][x], a, b[0], b[1]);
                        }
                    }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[u][x][i] += part[u][x][i];
            }
        }
        __syncwarp();
        fetch(n + 2, blk1);                       // K of the next tile
        ++n;
        // ---- softmax
        vr = vr < kRangeFloor ? kRangeFloor : vr; // a block of zeros of another writer; NaN stays
        const float ks = __fdiv_rn(kr, 127.0f);
        const float lv = log2f(__fdiv_rn(vr, 127.0f)), iv = __fdiv_rn(127.0f, vr);
        // a tile that every row sees whole needs no mask
        const bool whole = __all_sync(0xffffffffu, blk >= 0 && tg + 15 < w.keys && tg + 15 <= w.pos0);
        float fix[NT][2];
        uint32_t pb[kTerms][NT][4][2];            // P^T: row 8 x + g, tokens 16 c + 4 u + {0, 1 | 2, 3}
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            float top[2] = {neg_inf(), neg_inf()};
            const float f[2] = {ks * back[x][0], ks * back[x][1]};
            float ic[2] = {iv, iv};               // NaN for a poisoned group: 0 where this lane's rows see nothing of it
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[u][x][i] = __fmaf_rn(s[u][x][i], f[i & 1], lv);
            if (!whole) {
                int see[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    see[i] = blk >= 0 ? (last[x][i] < w.keys - 1 ? last[x][i] : w.keys - 1) - tg : -1;
                    ic[i] = see[i] < 0 ? 0.0f : iv;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * u + (i & 2) > see[i & 1]) s[u][x][i] = neg_inf();
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) top[i & 1] = fmaxf(top[i & 1], s[u][x][i]);
            float base[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
                const float m = fmaxf(mx[x][i], top[i]);
                fix[x][i] = m == neg_inf() ? 1.0f : ex2(mx[x][i] - m);
                base[i] = m == neg_inf() ? 0.0f : m - kPShift;
                mx[x][i] = m;
                sum[x][i] *= fix[x][i];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[u][x][i] = ex2(s[u][x][i] - base[i & 1]);
                    sum[x][i & 1] = __fmaf_rn(s[u][x][i], ic[i & 1], sum[x][i & 1]);
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float a = s[u][x][2 * half], b = s[u][x][2 * half + 1];
                    const uint32_t hi = h2(a, b);
                    pb[0][x][u][half] = transpose8(hi);
                    if (kTerms == 2) pb[kTerms - 1][x][u][half] = transpose8(h2(a - h_lo(hi), b - h_hi(hi)));
                }
            }
        }
        // ---- P V
        if (!(ok = sm100::mbar_wait_warp(&S.full[warp][(done + n) % kSlots], ((done + n) / kSlots) & 1, &S.abort, p.err))) break;
        slot = S.ring[warp][(done + n) % kSlots] + c * Sm::kVGroup + g * 16;
        constexpr int kSide = NT >= 4 ? 2 : 4;    // 16-dim tiles side by side
#pragma unroll
        for (int t0 = 0; t0 < DV / 16; t0 += kSide) {
            uint4 va[kSide], vb[kSide];
            float o[kSide][NT][4];
#pragma unroll
            for (int t = 0; t < kSide; ++t) {
                va[t] = *reinterpret_cast<const uint4 *>(slot + (t0 + t) * 256);
                vb[t] = *reinterpret_cast<const uint4 *>(slot + (t0 + t) * 256 + 128);
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[t][x][i] = 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 4 * kTerms; ++u)
#pragma unroll
                for (int t = 0; t < kSide; ++t) {
                    uint4 a;
                    codes_to_half(word_of(va[t], u & 3), a.x, a.z);
                    codes_to_half(word_of(vb[t], u & 3), a.y, a.w);
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        const uint32_t(&b)[2] = pb[u < 4 ? kTerms - 1 : 0][x][u & 3];
                        mma_f16(o[t][x], a, b[0], b[1]);
                    }
                }
#pragma unroll
            for (int t = 0; t < kSide; ++t)
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[t0 + t][x][i] = __fmaf_rn(acc[t0 + t][x][i], fix[x][i & 1], o[t][x][i]);
        }
        __syncwarp();
        fetch(n + 2, blk1);                       // its V
        ++n;
        blk = blk1;
        blk1 = blk2;
        blk2 = blk3;
        kr = kr1;
        vr = vr1;
    }
    if (!ok) {                                    // let the copies already issued land before the CTA exits
        for (int i = n; i < n + kSlots && i < 2 * mine; ++i)
            for (uint32_t tries = 0; tries < sm100::kMaxWaitProbes; ++tries)
                if (sm100::mbar_try_wait(&S.full[warp][(done + i) % kSlots], ((done + i) / kSlots) & 1)) break;
    }
    done += 2 * mine;
    __syncthreads();                              // the ring is free

    // ---- join the warps
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum[x][i] += __shfl_xor_sync(0xffffffffu, sum[x][i], o);
            if (g == 0) {
                S.m[warp][8 * x + 2 * c + i] = mx[x][i];
                S.l[warp][8 * x + 2 * c + i] = sum[x][i];
            }
        }
#pragma unroll
        for (int t = 0; t < DV / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) S.o[warp][8 * x + 2 * c + (i & 1)][16 * t + g + 4 * (i & 2)] = acc[t][x][i];
    }
    __syncthreads();
    for (int row = warp; row < w.tokens * gq; row += kWarps) {
        const int i = row / gq, gg = row - i * gq;
        if (gg >= heads_here) continue;
        float m = neg_inf(), f[kWarps], l = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) m = fmaxf(m, S.m[k][row]);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            f[k] = m == neg_inf() ? 1.0f : ex2(S.m[k][row] - m);
            l = __fmaf_rn(S.l[k][row], f[k], l);
        }
        const int64_t t = w.t0 + i;
        const int head = w.head0 + gg;
        for (int d = lane; d < DV; d += 32) {
            float o = 0.0f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) o = __fmaf_rn(S.o[k][row][d], f[k], o);
            if (p.splits == 1) {
                const float y = l == 0.0f ? 0.0f : __fdiv_rn(o, l);
                const int64_t at = t * p.ldo + (int64_t)head * DV + d;
                if (BF16) reinterpret_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(y);
                else reinterpret_cast<float *>(p.out)[at] = y;
            } else {
                const int64_t at = ((w.scratch + i) * p.heads + head) * p.splits + split;
                float *ml = p.ws + at * 2;
                if (d == 0) {
                    ml[0] = m;
                    ml[1] = l;
                }
                p.ws[p.cut.rows * p.heads * p.splits * 2 + at * DV + d] = o;
            }
        }
    }
}

// Columns of a request's several tokens, as many as the registers hold: the
// more, the less often the keys are read.
__host__ __device__ constexpr int most_columns(bool bf16) { return bf16 ? 4 : 2; }

// CTAs an SM holds: three where the registers of a single token's few columns
// allow it, which evens out batches of ragged lengths (64 requests 106 -> 100 us).
__host__ __device__ constexpr int ctas_per_sm(int dk, bool bf16, int nt) { return bf16 && nt == 1 && dk <= 128 ? 3 : 2; }

// Up to tq tokens of a request by gq heads of a kv head, on NT * 8 columns.
template <int DK, int DV, bool BF16, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(DK, BF16, NT))
attend_kernel(const AttendParams p, int tq, int gq, int hgroups, Slots kind, int tiles, int64_t slots,
              bool beside) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared<DK, DV, NT> &S = *reinterpret_cast<Shared<DK, DV, NT> *>(smem_raw);
    if (!beside) QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int h = blockIdx.y / hgroups, hg = blockIdx.y % hgroups;
    const int G = p.heads / p.c.heads;
    const int heads_here = G - hg * gq < gq ? G - hg * gq : gq;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kWarps * kSlots; ++i) sm100::mbar_init(&S.full[0][0] + i, 1);
        S.abort = 0;
        sm100::fence_mbar_init();
    }
    __syncthreads();
    uint32_t done = 0;                            // items of this warp's ring so far
    for (int64_t slot = blockIdx.x; slot < slots; slot += gridDim.x) {
        Rows w;
        if (!find_rows(p, slot, tq, kind, tiles, w)) continue;           // the whole CTA alike
        w.head0 = h * G + hg * gq;
        attend_rows<DK, DV, BF16, NT>(p, w, h, blockIdx.z, gq, heads_here, S, done);
        if (slot + gridDim.x < slots) {           // the ring is written by copies again
            sm100::fence_proxy_async_smem();
            __syncthreads();
        }
    }
    if (beside) QMOE_PDL_WAIT();
}

// Joins the pieces, one CTA per (token, head): thread s weighs piece s, the
// warps share the pieces' sums out.
constexpr int kJoinWarps = 4;
constexpr int kMaxSplits = 256;

// How a CTA finds its tokens: every gridDim.x / R-th one of a request of up to
// cut.few; token blockIdx.x; or that token, whose request says which of the two
// kinds of pieces it has (`tile`: the second kind).
enum class Joins { kRequests, kTokens, kBoth };

template <int DV, bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const AttendParams p, const AttendParams tile,
                                                                       Joins kind) {
    constexpr int kPer = DV / 32;
    __shared__ float weight[kMaxSplits];
    __shared__ float red[kJoinWarps], part_sum[kJoinWarps][DV];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // Before the wait: q_start was written in front of this call's first launch,
    // and this one starts after that has waited for it.
    const int64_t rows = p.q_start[p.R] < p.T ? p.q_start[p.R] : p.T;
    int64_t t = blockIdx.x, t_hi = t + 1, step = 1, scratch = t, scratch_rows = p.cut.rows;
    int splits = p.splits;
    const float *ws = p.ws;
    if (kind == Joins::kRequests) {
        step = gridDim.x / p.R;
        const int64_t r = blockIdx.x / step, first = p.q_start[r], i = blockIdx.x % step;
        t = first + i;
        t_hi = p.q_start[r + 1];
        if (t_hi - first > p.cut.few || first < 0) t_hi = 0;
        scratch = p.cut.by_token ? t : r * p.cut.few + i;
    } else if (t < p.q_start[0]) {                // nobody's: no piece was written
        t_hi = 0;
    } else if (kind == Joins::kBoth) {
        const int64_t r = find_request(p.q_start, p.R, t, 1), first = p.q_start[r];
        if (p.q_start[r + 1] - first > p.cut.few) {
            splits = tile.splits;
            ws = tile.ws;
            scratch_rows = tile.cut.rows;
            if (splits == 1) t_hi = 0;            // written in one piece
        } else if (!p.cut.by_token) {
            scratch = r * p.cut.few + t - first;
        }
    }
    t_hi = t_hi < rows ? t_hi : rows;
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    for (; t < t_hi; t += step, scratch += step) {
    const int64_t row = scratch * p.heads + blockIdx.y;
    const float2 *ml = reinterpret_cast<const float2 *>(ws) + row * splits;
    const float *part = ws + scratch_rows * p.heads * splits * 2 + row * splits * DV;
    float2 v[kMaxSplits / (kJoinWarps * 32)];
    float m = neg_inf();
#pragma unroll
    for (int k = 0; k < kMaxSplits / (kJoinWarps * 32); ++k) {
        const int s = k * kJoinWarps * 32 + tid;
        v[k] = s < splits ? ml[s] : make_float2(neg_inf(), 0.0f);
        m = fmaxf(m, v[k].x);
    }
    m = warp_max(m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kJoinWarps; ++k) m = fmaxf(m, red[k]);
    __syncthreads();
    float l = 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxSplits / (kJoinWarps * 32); ++k) {
        const int s = k * kJoinWarps * 32 + tid;
        const float f = m == neg_inf() ? 1.0f : ex2(v[k].x - m);
        if (s < splits) weight[s] = f;
        l = __fmaf_rn(v[k].y, f, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[warp] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoinWarps; ++k) l += red[k];
    float o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) o[j] = 0.0f;
#pragma unroll 4
    for (int s = warp; s < splits; s += kJoinWarps) {
        const float f = weight[s];
#pragma unroll
        for (int j = 0; j < kPer; ++j) o[j] = __fmaf_rn(part[(int64_t)s * DV + 32 * j + lane], f, o[j]);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) part_sum[warp][32 * j + lane] = o[j];
    __syncthreads();
    const int64_t at = t * p.ldo + (int64_t)blockIdx.y * DV;
    for (int d = tid; d < DV; d += kJoinWarps * 32) {
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < kJoinWarps; ++k) y += part_sum[k][d];
        y = l == 0.0f ? 0.0f : __fdiv_rn(y, l);
        if (BF16) reinterpret_cast<__nv_bfloat16 *>(p.out)[at + d] = __float2bfloat16_rn(y);
        else reinterpret_cast<float *>(p.out)[at + d] = y;
    }
    __syncthreads();
    }
}

struct RowShape {
    int nt, gq, tq, hgroups;
};
// gq heads by tq tokens on nt * 8 columns: one token, or several.
RowShape row_shape(bool single, int G, int dtype) {
    const int most = most_columns(dtype != 0);
    RowShape r;
    r.gq = G < 8 * most ? G : 8 * most;
    r.nt = !single ? most : r.gq <= 8 ? 1 : r.gq <= 16 ? 2 : most;
    r.tq = single ? 1 : 8 * most / r.gq;
    r.hgroups = (G + r.gq - 1) / r.gq;
    return r;
}

template <int DK, int DV, bool BF16, int NT>
cudaError_t launch_nt(const AttendParams &p, const RowShape &r, Slots kind, int tiles, int64_t slots, int64_t grid, bool beside,
                      cudaStream_t s) {
    const size_t smem = sizeof(Shared<DK, DV, NT>);
    auto kernel = attend_kernel<DK, DV, BF16, NT>;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)grid, (unsigned)(p.c.heads * r.hgroups), (unsigned)p.splits), dim3(kThreads),
                      smem, s, p, r.tq, r.gq, r.hgroups, kind, tiles, slots, beside);
}

template <int DK, int DV, bool BF16>
cudaError_t launch_dims(const AttendParams &p, cudaStream_t s) {
    const int G = p.heads / p.c.heads;
    constexpr int kMost = most_columns(BF16);
    const RowShape one = row_shape(true, G, p.dtype), more = row_shape(false, G, p.dtype);
    const bool several = p.cut.several;
    const Slots kind = several ? Slots::kSingles : Slots::kTokens;
    const int64_t slots = several ? p.R : p.T;
    cudaError_t e = one.nt == 1   ? launch_nt<DK, DV, BF16, 1>(p, one, kind, 1, slots, slots, false, s)
                    : one.nt == 2 ? launch_nt<DK, DV, BF16, 2>(p, one, kind, 1, slots, slots, false, s)
                                  : launch_nt<DK, DV, BF16, kMost>(p, one, kind, 1, slots, slots, false, s);
    // The kinds of requests are launches side by side: a launch may start once
    // every CTA of the one before has, which the first does only after its wait
    // for what came before this call; so the others read nothing too early.  They
    // wait for the launch before them at their end, so that what comes after the
    // last has all of them behind it.
    const bool prompts = p.cut.mixed && BF16;     // the requests of more than cut.few tokens
    AttendParams tile = p;                        // those in f32: pieces of their own
    tile.splits = p.cut.tile_splits;
    tile.ws = p.ws ? p.ws + p.cut.rows * p.heads * p.splits * (DV + 2) : nullptr;
    tile.cut.rows = p.T;
    tile.cut.by_token = true;
    if (e == cudaSuccess && prompts) e = launch_attend_prompt(p, p.cut.few, s);
    if (e == cudaSuccess && (several || (p.cut.mixed && !BF16))) {
        // often none: a bounded grid looks through the slots (eight CTAs an SM: 5
        // requests of 2 tokens after 4000, 256 heads to 16, 80 us, with two 82)
        const int64_t n = BF16 ? p.R * p.cut.tiles : several ? p.T / more.tq + p.R : p.T, cap = 8 * (int64_t)device_sm_count();
        const AttendParams &q = BF16 ? p : tile;
        int64_t grid = (p.cut.tiles > 1 ? 2 * cap : cap) / ((int64_t)p.c.heads * more.hgroups * q.splits);
        grid = grid < 1 ? 1 : grid < n ? grid : n;
        e = launch_nt<DK, DV, BF16, kMost>(q, more, BF16 ? Slots::kFew : several ? Slots::kTiles : Slots::kEvery, p.cut.tiles, n,
                                          grid, true, s);
    }
    if (e == cudaSuccess && p.splits > 1) {
        int64_t grid = p.T;
        const bool by_request = several && BF16;
        if (by_request) {                         // a request's tokens side by side while the device has room
            const int64_t room = 8 * (int64_t)device_sm_count() / (p.R * p.heads);
            grid = p.R * (room < 1 ? 1 : room < p.cut.few ? room : p.cut.few);
        }
        e = launch_pdl(attend_join_kernel<DV, BF16>, dim3((unsigned)grid, (unsigned)p.heads), dim3(kJoinWarps * 32), 0, s, p,
                       tile, by_request ? Joins::kRequests : p.cut.mixed ? Joins::kBoth : Joins::kTokens);
    }
    return e;
}

}  // namespace

// A batch of few CTAs is cut so that two an SM fill the device once (a request
// of the longest length each); one of many into a piece's quarter of that,
// since its requests may be of any length.
//
// Scratch has rows for the requests that are cut this way only: few tokens of
// each, a few ten MB whatever the batch (a row for every token of it was 5 GB at
// 8192 tokens, 32 heads of 128 and a table of 131072 tokens).  Longer requests
// have CTAs enough of their own in bf16 (attend_prompt.cu); in f32 they are cut
// into as many pieces as kTileScratch holds, which is all of them while their
// rows are too few to fill the device.
constexpr size_t kTileScratch = (size_t)128 << 20;

// A batch without more tokens than requests is taken for single tokens, but one
// of a captured step's many places may hold a prompt.  Requests of up to this many
// tokens go a token at a time there: their keys come from L2 after the first, and
// they are cut into pieces (33 tokens after 30000, 32 heads to 8: 242 us, by tiles
// 552).  Longer ones go by tiles (256 after 1000 38 us, a token at a time 90, and
// ever more the longer); the launch that looks for them costs a batch of 200
// single tokens 2 us of 44, smaller batches nothing.
constexpr int kPerToken = 128;

AttendCut attend_cut(const KvCacheDev &c, int64_t T, int64_t R, int heads, int dtype, int64_t max_kv) {
    const RowShape r = row_shape(true, heads / c.heads, dtype), more = row_shape(false, heads / c.heads, dtype);
    const int64_t rows = T <= R ? T : R;
    const int64_t ctas = (rows < 1 ? 1 : rows) * c.heads * r.hgroups;
    const int64_t sms = device_sm_count(), fill = 2 * sms;
    const int64_t tiles = max_kv < 1 ? 1 : (max_kv + 63) / 64;
    int64_t s = 4 * ctas <= fill ? fill / ctas : (4 * fill + ctas - 1) / ctas;
    int64_t ch = (tiles + s - 1) / s;
    ch = ch < 2 * kWarps ? 2 * kWarps : (ch + kWarps - 1) / kWarps * kWarps;
    s = (tiles + ch - 1) / ch;
    if (s > kMaxSplits) {
        s = kMaxSplits;
        ch = (tiles + s - 1) / s;
    }
    AttendCut cut{};
    cut.splits = (int)s;
    cut.chunk = (int)ch;
    cut.several = T > R;
    cut.mixed = cut.several || T > kPerToken;
    cut.tiles = 1;
    cut.few = cut.several ? 1 : cut.mixed ? kPerToken : INT32_MAX;
    if (cut.several && dtype != 0) {
        // Up to 32 tokens (a tile of the prompts' kernel at most) stay here, where their
        // keys are cut into pieces, while the batch is small: 6 requests of up to 9
        // tokens after 3756, 8 heads to one kv head, 28 us, by the prompts' kernel 114.
        // In larger ones only a tile does: with up to 32 tokens here 64 single tokens of
        // up to 8192 keys, 32 heads to 8, take 105 us instead of 100 for the search, and
        // 63 requests of up to 231 after 500 287 instead of 246.
        cut.tiles = more.tq >= 32 ? 1 : more.tq > 8 ? 32 / more.tq : 4;
        if (R * cut.tiles * c.heads * more.hgroups * s > 16 * sms) cut.tiles = 1;
        cut.few = cut.tiles * more.tq;
    }
    cut.by_token = T <= R * cut.few;
    cut.rows = cut.by_token ? T : R * cut.few;
    const size_t row = (size_t)heads * (c.v_dim + 2);                 // floats of a piece of a row
    cut.tile_splits = 1;
    if (cut.mixed && dtype == 0 && s > 1) {
        const int64_t room = (int64_t)(kTileScratch / (sizeof(float) * row * T));
        cut.tile_splits = (int)(room < 1 ? 1 : room < s ? room : s);
    }
    cut.floats = s > 1 ? row * (cut.rows * s + (cut.tile_splits > 1 ? T * cut.tile_splits : 0)) : 0;
    return cut;
}

cudaError_t launch_attend(const AttendParams &params, cudaStream_t s) {
    if (params.T == 0 || params.R == 0) return cudaSuccess;
    AttendParams p = params;
    const uint64_t d = (uint64_t)p.c.block / 16;
    p.per_block = ((1ull << 36) + d - 1) / d;
    p.splits = p.cut.splits;
    const bool bf = p.dtype != 0;
    if (p.c.k_dim == 64 && p.c.v_dim == 64) return bf ? launch_dims<64, 64, true>(p, s) : launch_dims<64, 64, false>(p, s);
    if (p.c.k_dim == 128 && p.c.v_dim == 128)
        return bf ? launch_dims<128, 128, true>(p, s) : launch_dims<128, 128, false>(p, s);
    return bf ? launch_dims<192, 128, true>(p, s) : launch_dims<192, 128, false>(p, s);
}

}  // namespace qmoe
