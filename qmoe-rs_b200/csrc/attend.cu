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
// The layout of the cache is the operands': within 64 tokens, lane 4 g + c of
// a warp takes the 16 bytes of K that are dims 16 c .. 16 c + 15 of a token and
// the 16 bytes of V that are tokens 16 c .. 16 c + 15 of a dim, and each 4 bytes
// of them are one B fragment of mma.m16n8k16.  Column 2 c + i of score tile j
// is token 16 c + 2 j + i, so a lane's scores all lie in one block.
#include "code8.cuh"
#include "kernels.h"

#include <cuda_fp16.h>

namespace qmoe {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kPShift = 14.0f;              // P up to 2^14: fp16 keeps 2^-38 of the largest

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

// Four codes -> two fp16 pairs: 0x6400 | (c + 128) is 1152 + c, exactly.
QMOE_DEV void codes_to_half(uint32_t v, uint32_t &lo, uint32_t &hi) {
    v ^= 0x80808080u;
    const uint32_t a = __byte_perm(v, 0x64646464u, 0x4140), b = __byte_perm(v, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
}

QMOE_DEV void mma_f16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The largest r in [0, R) with start[r] / tq + r <= slot.  Tiles of request r
// take the slots from there on; start never falls, so neither does that.  A
// warp looks at 32 places at a time.
QMOE_DEV int64_t find_request(const int32_t *start, int64_t R, int64_t slot, int tq) {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, n = R;                       // the answer is in [lo, lo + n)
    while (n > 1) {
        const int64_t step = (n + 31) / 32;
        const int64_t i = lo + lane * step;
        const bool le = lane == 0 || (i < lo + n && start[i] / tq + i <= slot);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
        const int64_t at = lo + last * step;
        n = lo + n - at < step ? lo + n - at : step;
        lo = at;
    }
    return lo;
}

struct Rows {                                    // of one CTA: up to 16 rows of one request and kv head
    int64_t t0;                                  // token of row 0
    int tokens, gq, head0;                       // row i * gq + g: token t0 + i, head head0 + g
    int pos0;                                    // last key of token t0 (may be negative)
    int keys;                                    // keys of the last token
    int64_t request;
};

QMOE_DEV bool find_rows(const AttendParams &p, int64_t slot, int tq, int gq, int hg, Rows &w) {
    const int64_t r = find_request(p.q_start, p.R, slot, tq);
    const int64_t s0 = p.q_start[r], n = p.q_start[r + 1] - s0;
    const int64_t i0 = (slot - (s0 / tq + r)) * tq;
    if (i0 < 0 || i0 >= n || s0 < 0) return false;
    int64_t cnt = n - i0 < tq ? n - i0 : tq;
    w.t0 = s0 + i0;
    if (w.t0 + cnt > p.T) cnt = p.T - w.t0;      // rows that the buffer does not hold
    if (cnt <= 0) return false;
    const int64_t most = p.max_blocks * p.c.block;
    const int64_t kv = p.kv_lens[r];
    const int64_t pos0 = (kv < 0 ? 0 : kv) - n + i0;
    const int64_t keys = pos0 + cnt;             // one past the last token's last key
    w.request = r;
    w.tokens = (int)cnt;
    w.gq = gq;
    w.pos0 = (int)(pos0 < -(1 << 30) ? -(1 << 30) : pos0);
    w.keys = (int)(keys < 0 ? 0 : keys > most ? most : keys);
    return true;
}

template <int DK, int DV, bool BF16>
struct Shared {
    static constexpr int kTerms = BF16 ? 1 : 2;
    uint4 q[kTerms][DK / 16][32];                // A fragments of q
    float back[16];                              // 2^-k of the row's scaling
    float m[kWarps][16], l[kWarps][16];
    float o[kWarps][16][DV];
};

template <int DK, int DV, bool BF16>
__global__ void __launch_bounds__(kThreads) attend_kernel(const AttendParams p, int tq, int gq, int hgroups) {
    constexpr int kTerms = BF16 ? 1 : 2;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    using Sm = Shared<DK, DV, BF16>;
    Sm &S = *reinterpret_cast<Sm *>(smem_raw);
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int h = blockIdx.y / hgroups, hg = blockIdx.y % hgroups, split = blockIdx.z;
    const int G = p.heads / p.c.heads;
    Rows w;
    if (!find_rows(p, blockIdx.x, tq, gq, hg, w)) return;        // the whole CTA alike
    w.head0 = h * G + hg * 16;
    const int heads_here = G - hg * 16 < gq ? G - hg * 16 : gq;
    const int bs = p.c.block;

    // ---- q: scale rows by a power of two, lay out the A fragments
    for (int row = warp; row < 16; row += kWarps) {
        const int i = row / gq, gg = row - i * gq;
        const bool live = i < w.tokens && gg < heads_here;
        float m = 0.0f;
        const int64_t at = live ? (w.t0 + i) * p.ldq + (int64_t)(w.head0 + gg) * DK : 0;
        if (live)
            for (int d = lane; d < DK; d += 32) m = fmaxf(m, fabsf(load_act(p.q, p.dtype, at + d)));
        m = warp_max(m);
        int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;
        e = e < -100 ? -100 : e > 100 ? 100 : e;
        const float up = pow2i(14 - e);
        if (lane == 0) S.back[row] = pow2i(e - 14);
        for (int d = 4 * lane; d < DK; d += 128) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = live ? __fmul_rn(load_act(p.q, p.dtype, at + d + j), up) : 0.0f;
            // dims 64 J + 16 c + 4 t + {0,1 | 2,3} are k = {2c, 2c+1 | 2c+8, 2c+9} of step 4 J + t
            const int step = (d >> 6) * 4 + ((d >> 2) & 3), cc = (d >> 4) & 3;
            uint32_t lo = h2(v[0], v[1]), hi = h2(v[2], v[3]);
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
                uint32_t *f = reinterpret_cast<uint32_t *>(&S.q[term][step][4 * (row & 7) + cc]) + (row >> 3);
                f[0] = lo;
                f[2] = hi;
                if (kTerms == 2) {
                    lo = h2(__fsub_rn(v[0], h_lo(lo)), __fsub_rn(v[1], h_hi(lo)));
                    hi = h2(__fsub_rn(v[2], h_lo(hi)), __fsub_rn(v[3], h_hi(hi)));
                }
            }
        }
    }
    __syncthreads();

    float acc[DV / 8][4];
#pragma unroll
    for (int t = 0; t < DV / 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][j] = 0.0f;
    float mx[2] = {neg_inf(), neg_inf()}, sum[2] = {0.0f, 0.0f};
    const float back[2] = {S.back[g], S.back[g + 8]};
    int last[2];                                  // last key of rows g, g + 8
#pragma unroll
    for (int a = 0; a < 2; ++a) last[a] = w.pos0 + (g + 8 * a) / gq;

    const int tiles = (w.keys + 63) / 64, per = (tiles + p.splits - 1) / p.splits;
    const int t_lo = split * per, t_hi = t_lo + per < tiles ? t_lo + per : tiles;
    const int32_t *row_table = p.table + w.request * p.max_blocks;
    // the block of 16 tokens from `tok` on, -1 past the keys and where the entry is none
    auto block_of = [&](int tok) -> int64_t {
        if (tok >= w.keys) return -1;
        const int64_t b = row_table[tok / bs];
        return b >= 0 && b < p.c.num_blocks ? b * p.c.heads + h : -1;
    };
    for (int tile = t_lo + warp; tile < t_hi; tile += kWarps) {
        const int tk = tile * 64 + 16 * (g >> 1), tv = tile * 64 + 16 * c;
        const int64_t bk = block_of(tk), bv = block_of(tv);
        // ---- scores
        float s[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = 0.0f;
#pragma unroll
        for (int J = 0; J < DK / 64; ++J) {
            uint4 kc[8];
            const int8_t *src = p.c.k + ((bk * (DK / 64) + J) * bs + tk % bs + (g & 1)) * 64 + c * 16;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                kc[j] = bk >= 0 ? *reinterpret_cast<const uint4 *>(src + j * 128) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint4 a0 = S.q[0][4 * J + t][lane];
                const uint4 a1 = kTerms == 2 ? S.q[kTerms - 1][4 * J + t][lane] : a0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t word = t == 0 ? kc[j].x : t == 1 ? kc[j].y : t == 2 ? kc[j].z : kc[j].w;
                    uint32_t b0, b1;
                    codes_to_half(word, b0, b1);
                    mma_f16(s[j], a0, b0, b1);
                    if (kTerms == 2) mma_f16(s[j], a1, b0, b1);
                }
            }
        }
        // ---- softmax
        const float kr = bv >= 0 ? p.c.k_range[bv] : 0.0f;
        float vr = bv >= 0 ? p.c.v_range[bv] : 127.0f;
        vr = vr < kRangeFloor ? kRangeFloor : vr;              // a block of zeros of another writer; NaN stays
        const float ks = __fdiv_rn(kr, 127.0f) * (p.scale * kLog2e);
        const float lv = log2f(__fdiv_rn(vr, 127.0f)), iv = __fdiv_rn(127.0f, vr);
        float top[2] = {neg_inf(), neg_inf()};
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int a = i >> 1, tok = tv + 2 * j + (i & 1);
                const float v = __fmaf_rn(s[j][i], ks * back[a], lv);
                s[j][i] = bv >= 0 && tok < w.keys && tok <= last[a] ? v : neg_inf();
                top[a] = fmaxf(top[a], s[j][i]);
            }
        float fix[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            top[a] = fmaxf(top[a], __shfl_xor_sync(0xffffffffu, top[a], 1));
            top[a] = fmaxf(top[a], __shfl_xor_sync(0xffffffffu, top[a], 2));
            const float m = fmaxf(mx[a], top[a]);
            fix[a] = m == neg_inf() ? 1.0f : ex2(mx[a] - m);
            mx[a] = m;
            sum[a] *= fix[a];
        }
        const float base[2] = {mx[0] == neg_inf() ? 0.0f : mx[0] - kPShift, mx[1] == neg_inf() ? 0.0f : mx[1] - kPShift};
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int a = i >> 1;
                s[j][i] = ex2(s[j][i] - base[a]);
                sum[a] = __fmaf_rn(s[j][i], iv, sum[a]);
            }
        // ---- P V
        uint4 pa[kTerms][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            pa[0][u] = make_uint4(h2(s[2 * u][0], s[2 * u][1]), h2(s[2 * u][2], s[2 * u][3]),
                                  h2(s[2 * u + 1][0], s[2 * u + 1][1]), h2(s[2 * u + 1][2], s[2 * u + 1][3]));
            if (kTerms == 2) {
                const uint4 a = pa[0][u];
                pa[kTerms - 1][u] =
                    make_uint4(h2(s[2 * u][0] - h_lo(a.x), s[2 * u][1] - h_hi(a.x)),
                               h2(s[2 * u][2] - h_lo(a.y), s[2 * u][3] - h_hi(a.y)),
                               h2(s[2 * u + 1][0] - h_lo(a.z), s[2 * u + 1][1] - h_hi(a.z)),
                               h2(s[2 * u + 1][2] - h_lo(a.w), s[2 * u + 1][3] - h_hi(a.w)));
            }
        }
        const int8_t *src = p.c.v + (bv * (bs / 16) + (tv % bs) / 16) * (DV * 16) + g * 16;
#pragma unroll
        for (int t = 0; t < DV / 8; ++t) {
            const uint4 vc = bv >= 0 ? *reinterpret_cast<const uint4 *>(src + t * 128) : make_uint4(0, 0, 0, 0);
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t word = u == 0 ? vc.x : u == 1 ? vc.y : u == 2 ? vc.z : vc.w;
                uint32_t b0, b1;
                codes_to_half(word, b0, b1);
                mma_f16(o, pa[0][u], b0, b1);
                if (kTerms == 2) mma_f16(o, pa[kTerms - 1][u], b0, b1);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = __fmaf_rn(acc[t][i], fix[i >> 1], o[i]);
        }
    }

    // ---- join the warps
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 1);
        sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 2);
        if (c == 0) {
            S.m[warp][g + 8 * a] = mx[a];
            S.l[warp][g + 8 * a] = sum[a];
        }
    }
#pragma unroll
    for (int t = 0; t < DV / 8; ++t) {
        *reinterpret_cast<float2 *>(&S.o[warp][g][8 * t + 2 * c]) = make_float2(acc[t][0], acc[t][1]);
        *reinterpret_cast<float2 *>(&S.o[warp][g + 8][8 * t + 2 * c]) = make_float2(acc[t][2], acc[t][3]);
    }
    __syncthreads();
    for (int row = warp; row < 16; row += kWarps) {
        const int i = row / gq, gg = row - i * gq;
        if (i >= w.tokens || gg >= heads_here) continue;
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
                const int64_t at = (t * p.heads + head) * p.splits + split;
                float *ml = p.ws + at * 2;
                if (d == lane && lane == 0) {
                    ml[0] = m;
                    ml[1] = l;
                }
                p.ws[p.T * p.heads * p.splits * 2 + at * DV + d] = o;
            }
        }
    }
}

// Joins the pieces: one warp per (token, head).
template <int DV, bool BF16>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendParams p) {
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t t = w / p.heads;
    if (t >= p.T || t >= p.q_start[p.R]) return;
    const float *ml = p.ws + w * p.splits * 2;
    const float *part = p.ws + p.T * p.heads * p.splits * 2 + w * p.splits * DV;
    float m = neg_inf();
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * s]);
    float l = 0.0f, o[DV / 32];
#pragma unroll
    for (int j = 0; j < DV / 32; ++j) o[j] = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float f = m == neg_inf() ? 1.0f : ex2(ml[2 * s] - m);
        l = __fmaf_rn(ml[2 * s + 1], f, l);
#pragma unroll
        for (int j = 0; j < DV / 32; ++j) o[j] = __fmaf_rn(part[(int64_t)s * DV + 32 * j + lane], f, o[j]);
    }
    const int64_t at = t * p.ldo + (w - t * p.heads) * DV + lane;
#pragma unroll
    for (int j = 0; j < DV / 32; ++j) {
        const float y = l == 0.0f ? 0.0f : __fdiv_rn(o[j], l);
        if (BF16) reinterpret_cast<__nv_bfloat16 *>(p.out)[at + 32 * j] = __float2bfloat16_rn(y);
        else reinterpret_cast<float *>(p.out)[at + 32 * j] = y;
    }
}

// Rows of a CTA: gq heads of a kv head by tq tokens.
void row_shape(int G, int &gq, int &tq, int &hgroups) {
    gq = G < 16 ? G : 16;
    tq = 16 / gq;
    hgroups = (G + 15) / 16;
}

template <int DK, int DV, bool BF16>
cudaError_t launch_dims(const AttendParams &p, cudaStream_t s) {
    int gq, tq, hgroups;
    row_shape(p.heads / p.c.heads, gq, tq, hgroups);
    const size_t smem = sizeof(Shared<DK, DV, BF16>);
    auto kernel = attend_kernel<DK, DV, BF16>;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(kernel, dim3((unsigned)(p.T / tq + p.R), (unsigned)(p.c.heads * hgroups), (unsigned)p.splits),
                   dim3(kThreads), smem, s, p, tq, gq, hgroups);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_pdl(attend_join_kernel<DV, BF16>, dim3((unsigned)((p.T * p.heads + 7) / 8)), dim3(256), 0, s, p);
}

}  // namespace

int attend_splits(int64_t T, int64_t R, int heads, int kv_heads, int64_t max_kv) {
    int gq, tq, hgroups;
    row_shape(heads / kv_heads, gq, tq, hgroups);
    const int64_t rows = (T + tq - 1) / tq > R ? (T + tq - 1) / tq : R;
    const int64_t ctas = (rows < 1 ? 1 : rows) * kv_heads * hgroups;
    const int64_t tiles = (max_kv + 63) / 64;
    int64_t s = (4 * (int64_t)device_sm_count() + ctas - 1) / ctas;
    const int64_t most = (tiles + kWarps - 1) / kWarps;
    if (s > most) s = most;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}

size_t attend_workspace_floats(int64_t T, int heads, int v_dim, int splits) {
    return splits <= 1 ? 0 : (size_t)T * heads * splits * (v_dim + 2);
}

cudaError_t launch_attend(const AttendParams &p, cudaStream_t s) {
    if (p.T == 0 || p.R == 0) return cudaSuccess;
    const bool bf = p.dtype != 0;
    if (p.c.k_dim == 64 && p.c.v_dim == 64) return bf ? launch_dims<64, 64, true>(p, s) : launch_dims<64, 64, false>(p, s);
    if (p.c.k_dim == 128 && p.c.v_dim == 128)
        return bf ? launch_dims<128, 128, true>(p, s) : launch_dims<128, 128, false>(p, s);
    return bf ? launch_dims<192, 128, true>(p, s) : launch_dims<192, 128, false>(p, s);
}

}  // namespace qmoe
