// kv.cu -- the paged cache of keys and values in 8 bits: its plan (block table
// and slot map from request lengths) and the append of new tokens.
#include "code8.cuh"
#include "kernels.h"

namespace qmoe {
namespace {

// ---- plan --------------------------------------------------------------------
//
// Request r has cached[r] tokens in the cache and gets fresh[r] more.  In
// order, each takes the blocks it lacks from the free list; one that the list,
// the table's width or the token capacity has no room for is denied (kv_len 0,
// its tokens without a slot).  Needs are summed over the requests that only
// the list could deny, so the granted ones take a prefix of it.
//
// One launch, bound by latency.  Every CTA sums up all requests for itself (a
// thread a run of them, 8 bytes a request from L2) and keeps the sums before
// each run; a token finds its run by bisection and its request by walking the
// run.  CTA 0 writes the requests' results.  A new block's first position
// belongs to exactly one new token, which writes the table's entry.

constexpr int kPlanThreads = 1024;

struct Need {
    int64_t fresh;   // rows in the token buffer
    int blocks;      // blocks wanted of the free list
    bool ok;         // fits the table and the token buffer
};

QMOE_DEV Need need_of(const KvPlanParams &p, int64_t r, int64_t row) {
    const int c = p.cached[r], f = p.fresh[r];
    Need n;
    n.fresh = f > 0 ? f : 0;
    n.ok = c >= 0 && f >= 0 && (int64_t)c + f <= p.max_blocks * p.block && row + n.fresh <= p.capacity;
    n.blocks = n.ok ? (c + f + p.block - 1) / p.block - (c + p.block - 1) / p.block : 0;
    return n;
}

QMOE_DEV bool granted(const KvPlanParams &p, const Need &n, int64_t before) {
    return n.ok && (n.blocks == 0 || before + n.blocks <= p.n_free);
}

// Exclusive sum over the CTA; `total` the sum of all.
QMOE_DEV int64_t block_scan(int64_t v, int64_t *part, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 31) part[warp] = s;
    __syncthreads();
    int64_t w = part[lane];                        // kPlanThreads / 32 = 32 warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int64_t before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    return (warp > 0 ? before : 0) + s - v;
}

QMOE_DEV int clamp32(int64_t v) { return (int)(v < INT32_MAX ? v : INT32_MAX); }

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const KvPlanParams p) {
    __shared__ int64_t part[32], rows[kPlanThreads], lacks[kPlanThreads];   // sums before each thread's run
    __shared__ int taken;
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int tid = threadIdx.x;
    const int64_t per = (p.R + kPlanThreads - 1) / kPlanThreads;
    const int64_t lo = tid * per < p.R ? tid * per : p.R, hi = lo + per < p.R ? lo + per : p.R;
    int64_t sum = 0, total, all;
    for (int64_t r = lo; r < hi; ++r) sum += p.fresh[r] > 0 ? p.fresh[r] : 0;
    const int64_t row0 = block_scan(sum, part, total);
    int64_t row = row0;
    sum = 0;
    for (int64_t r = lo; r < hi; ++r) {
        const Need n = need_of(p, r, row);
        sum += n.blocks;
        row += n.fresh;
    }
    const int64_t lack0 = block_scan(sum, part, all);
    rows[tid] = row0;
    lacks[tid] = lack0;
    if (tid == 0) taken = 0;
    __syncthreads();
    if (blockIdx.x == 0) {
        int64_t lack = lack0;
        int most = 0;
        row = row0;
        for (int64_t r = lo; r < hi; ++r) {
            const Need n = need_of(p, r, row);
            const bool ok = granted(p, n, lack);
            p.q_start[r] = clamp32(row);
            p.kv_lens[r] = ok ? p.cached[r] + p.fresh[r] : 0;
            lack += n.blocks;
            if (ok && n.blocks) most = (int)lack;
            row += n.fresh;
        }
        if (most > 0) atomicMax(&taken, most);
        __syncthreads();
        if (tid == 0) {
            p.q_start[p.R] = clamp32(total);
            p.taken[0] = taken;
        }
    }
    for (int64_t t = (int64_t)blockIdx.x * kPlanThreads + tid; t < p.capacity; t += (int64_t)gridDim.x * kPlanThreads) {
        int slot = -1, pos = -1;
        if (t < total) {
            int c = 0;                             // the last run that starts at or before t
#pragma unroll
            for (int step = kPlanThreads / 2; step > 0; step >>= 1)
                if (rows[c + step] <= t) c += step;
            int64_t r = c * per, lack = lacks[c];
            row = rows[c];
            Need n = need_of(p, r, row);
            while (row + n.fresh <= t) {
                row += n.fresh;
                lack += n.blocks;
                n = need_of(p, ++r, row);
            }
            if (granted(p, n, lack)) {
                const int cached = p.cached[r], have = (cached + p.block - 1) / p.block;
                pos = cached + (int)(t - row);
                const int b = pos / p.block, off = pos - b * p.block;
                int32_t *entry = p.table + r * p.max_blocks + b;
                int id;
                if (b >= have) {
                    id = p.free_blocks[lack + b - have];
                    if (off == 0) *entry = id;
                } else {
                    id = *entry;
                }
                if (id >= 0 && id < p.num_blocks) slot = id * p.block + off;
            }
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
    }
}

// ---- append --------------------------------------------------------------------
//
// A run is a sequence of rows with consecutive slots of one block; offsets
// before it are the block's earlier tokens.  The range grows to the new tokens'
// largest magnitude, the earlier codes are rounded to the new range (left alone
// when it did not grow), the new ones written.
//
// One warp a run, head and side (K or V).  It reads its rows twice, the second
// time from L1 or L2: bound by HBM for prompts (two prompts of up to 4099
// tokens, 16 heads of 192 and 128, f32: 146 MB) and by the latency of that chain of loads
// for single tokens.  Four CTAs an SM with four loads in flight a lane hide them
// best (those prompts, 5720 rows of them, take 49 us, 64 single tokens 3.5; three
// CTAs with eight loads 51 and 3.9, two 55 and 3.8).  A warp looks for runs that start among `span` rows, one
// row where rows are few.

constexpr int kAppendWarps = 8;
constexpr int kAhead = 4;                          // loads in flight a lane

template <bool BF16>
QMOE_DEV float4 load4(const void *x, int64_t i, bool vec) {
    if (vec) return load_act4(x, BF16 ? 1 : 0, i);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v[j] = BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(x)[i + j])
                    : reinterpret_cast<const float *>(x)[i + j];
    return make_float4(v[0], v[1], v[2], v[3]);
}

template <bool BF16>
QMOE_DEV float load1(const void *x, int64_t i) {
    return BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(x)[i])
                : __ldg(reinterpret_cast<const float *>(x) + i);
}

// The largest magnitude of `n` rows of DIM elements from x[at], ld apart; bad:
// an element is not finite.
template <bool BF16, int DIM>
QMOE_DEV float rows_max(const void *x, int64_t at, int64_t ld, int n, bool vec, bool &bad) {
    constexpr int kPer = DIM / 4;                  // groups of four elements in a row
    const int lane = threadIdx.x & 31;
    float m = 0.0f;
    bool odd = false;
    for (int e0 = 0; e0 < n * kPer; e0 += 32 * kAhead) {
        float4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int e = e0 + 32 * k + lane, i = e / kPer;
            v[k] = e < n * kPer ? load4<BF16>(x, at + i * ld + (e - i * kPer) * 4, vec) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            m = max_abs(max_abs(max_abs(max_abs(m, v[k].x), v[k].y), v[k].z), v[k].w);
            const float inf = __int_as_float(0x7f800000);
            odd |= !(fabsf(v[k].x) < inf && fabsf(v[k].y) < inf && fabsf(v[k].z) < inf && fabsf(v[k].w) < inf);
        }
    }
    bad = __any_sync(0xffffffffu, odd);
    return warp_max(m);
}

// Byte j of four codes, the value c in its place.
QMOE_DEV uint32_t put_byte(uint32_t w, int j, int c) {
    const int sh = 8 * j;
    return (w & ~(255u << sh)) | (uint32_t)(c & 255) << sh;
}
QMOE_DEV int get_byte(uint32_t w, int j) { return (int)(int8_t)(w >> (8 * j)); }

// Rows t .. t + n - 1 to offsets off .. of a block, one head.
template <bool BF16, int DIM>
QMOE_DEV void append_k(const KvAppendParams &p, int8_t *codes, float *range, int64_t at, int n, int off) {
    constexpr int kPer = DIM / 4;
    const int lane = threadIdx.x & 31, bs = p.c.block;
    const float old = off > 0 ? *range : 0.0f;
    bool bad;
    const float m = rows_max<BF16, DIM>(p.k, at, p.ldk, n, p.vec_k, bad);
    bad |= !(fabsf(old) < __int_as_float(0x7f800000));
    const float r = range8(fmaxf(m, old), !bad), mi = __fdiv_rn(127.0f, r);
    __syncwarp();
    if (lane == 0) *range = r;
    auto place = [&](int tok, int d) { return reinterpret_cast<uint32_t *>(codes + ((d >> 6) * bs + tok) * 64 + (d & 63)); };
    if (off > 0 && !(r == old)) {
        const float oi = __fdiv_rn(old, r);
        for (int e0 = 0; e0 < off * kPer; e0 += 32 * kAhead) {
            uint32_t w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int e = e0 + 32 * k + lane, i = e / kPer;
                w[k] = e < off * kPer ? *place(i, (e - i * kPer) * 4) : 0;
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int e = e0 + 32 * k + lane, i = e / kPer;
                if (e >= off * kPer) continue;
                *place(i, (e - i * kPer) * 4) =
                    codes4((float)get_byte(w[k], 0), (float)get_byte(w[k], 1), (float)get_byte(w[k], 2),
                           (float)get_byte(w[k], 3), old, r, oi);
            }
        }
    }
    for (int e0 = 0; e0 < n * kPer; e0 += 32 * kAhead) {
        float4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int e = e0 + 32 * k + lane, i = e / kPer;
            v[k] = e < n * kPer ? load4<BF16>(p.k, at + i * p.ldk + (e - i * kPer) * 4, p.vec_k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int e = e0 + 32 * k + lane, i = e / kPer;
            if (e < n * kPer)
                *place(off + i, (e - i * kPer) * 4) = codes4(v[k].x, v[k].y, v[k].z, v[k].w, 127.0f, r, mi);
        }
    }
}

// V holds 16 tokens of a dim in 16 bytes: a lane has whole dims of a full
// group, 16 loads (each a row's 128 bytes over the warp) and one 16-byte store;
// the tokens of other groups go byte by byte.
template <bool BF16, int DIM>
QMOE_DEV void append_v(const KvAppendParams &p, int8_t *codes, float *range, int64_t at, int n, int off) {
    const int lane = threadIdx.x & 31;
    const float old = off > 0 ? *range : 0.0f;
    bool bad;
    const float m = rows_max<BF16, DIM>(p.v, at, p.ldv, n, p.vec_v, bad);
    bad |= !(fabsf(old) < __int_as_float(0x7f800000));
    const float r = range8(fmaxf(m, old), !bad), mi = __fdiv_rn(127.0f, r);
    __syncwarp();
    if (lane == 0) *range = r;
    const bool moved = off > 0 && !(r == old);
    const float oi = moved ? __fdiv_rn(old, r) : 0.0f;
    constexpr int kPer = DIM / 4, kQ = DIM / 32;
    if (moved)
        for (int g = 0; 16 * g < off; ++g) {
            uint4 w[kQ];
#pragma unroll
            for (int q = 0; q < kQ; ++q) w[q] = *reinterpret_cast<const uint4 *>(codes + (g * DIM + 32 * q + lane) * 16);
#pragma unroll
            for (int q = 0; q < kQ; ++q) {
                uint32_t *words = reinterpret_cast<uint32_t *>(&w[q]);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (16 * g + i < off)
                        words[i >> 2] = put_byte(words[i >> 2], i & 3, code8((float)get_byte(words[i >> 2], i & 3), old, r, oi));
                *reinterpret_cast<uint4 *>(codes + (g * DIM + 32 * q + lane) * 16) = w[q];
            }
        }
    __syncwarp();
    for (int i0 = 0; i0 < n;) {                    // tokens of one group at a time
        const int tok = off + i0, g = tok >> 4, cnt = 16 - (tok & 15) < n - i0 ? 16 - (tok & 15) : n - i0;
        if (cnt == 16) {
#pragma unroll
            for (int q = 0; q < kQ; ++q) {
                const int d = 32 * q + lane;
                float x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = load1<BF16>(p.v, at + (i0 + i) * p.ldv + d);
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = codes4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], 127.0f, r, mi);
                *reinterpret_cast<uint4 *>(codes + (g * DIM + d) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            for (int e = lane; e < cnt * kPer; e += 32) {
                const int i = e / kPer, d = (e - i * kPer) * 4;
                const float4 v = load4<BF16>(p.v, at + (i0 + i) * p.ldv + d, p.vec_v);
                int8_t *c = codes + (g * DIM + d) * 16 + ((tok + i) & 15);
                c[0] = (int8_t)code8(v.x, 127.0f, r, mi);
                c[16] = (int8_t)code8(v.y, 127.0f, r, mi);
                c[32] = (int8_t)code8(v.z, 127.0f, r, mi);
                c[48] = (int8_t)code8(v.w, 127.0f, r, mi);
            }
        }
        i0 += cnt;
    }
}

template <bool BF16, int DK, int DV>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) kv_append_kernel(const KvAppendParams p, int span) {
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int side = (int)(w % (2 * p.c.heads)), h = side >> 1;
    const int64_t t0 = w / (2 * p.c.heads) * span;
    if (t0 >= p.T) return;
    const int64_t total = p.c.num_blocks * p.c.block;
    const int bs = p.c.block;
    // lane i: does a run start at row t0 + i?
    const int64_t mine = t0 + lane;
    int slot = -1;
    bool starts = false;
    if (lane < span && mine < p.T) {
        slot = p.slots[mine];
        starts = slot >= 0 && slot < total && !(slot % bs > 0 && mine > 0 && p.slots[mine - 1] == slot - 1);
    }
    for (unsigned left = __ballot_sync(0xffffffffu, starts); left; left &= left - 1) {
        const int f = __ffs(left) - 1;
        const int64_t t = t0 + f;
        const int s = __shfl_sync(0xffffffffu, slot, f), off = s % bs;
        const int64_t bh = (int64_t)(s / bs) * p.c.heads + h;
        int n = 0;
        for (int base = 0; base < bs - off; base += 32) {
            const int i = base + lane;
            const bool in = off + i < bs && t + i < p.T && p.slots[t + i] == s + i;
            const unsigned miss = ~__ballot_sync(0xffffffffu, in);
            n += miss ? __ffs(miss) - 1 : 32;
            if (miss) break;
        }
        if (side & 1)
            append_v<BF16, DV>(p, p.c.v + bh * bs * DV, p.c.v_range + bh, t * p.ldv + (int64_t)h * DV, n, off);
        else
            append_k<BF16, DK>(p, p.c.k + bh * bs * DK, p.c.k_range + bh, t * p.ldk + (int64_t)h * DK, n, off);
    }
}

template <int DK, int DV>
cudaError_t launch_append(const KvAppendParams &p, cudaStream_t s) {
    // rows a warp looks at: one while that gives the device a few thousand warps
    const int64_t sides = 2 * (int64_t)p.c.heads;
    const int span = p.T * sides <= 64 * (int64_t)device_sm_count() ? 1 : p.T < 32 ? (int)p.T : p.c.block < 32 ? p.c.block : 32;
    const int64_t warps = (p.T + span - 1) / span * sides;
    return launch_pdl(p.dtype ? kv_append_kernel<true, DK, DV> : kv_append_kernel<false, DK, DV>,
                      dim3((unsigned)((warps + kAppendWarps - 1) / kAppendWarps)), dim3(kAppendWarps * 32), 0, s, p, span);
}

}  // namespace

cudaError_t launch_kv_plan(const KvPlanParams &p, cudaStream_t s) {
    int64_t ctas = (p.capacity + kPlanThreads - 1) / kPlanThreads;
    const int64_t most = 2 * (int64_t)device_sm_count();
    ctas = ctas < 1 ? 1 : ctas < most ? ctas : most;
    return launch_pdl(kv_plan_kernel, dim3((unsigned)ctas), dim3(kPlanThreads), 0, s, p);
}

cudaError_t launch_kv_append(const KvAppendParams &p, cudaStream_t s) {
    if (p.T == 0) return cudaSuccess;
    if (p.c.k_dim == 64) return launch_append<64, 64>(p, s);
    if (p.c.k_dim == 128) return launch_append<128, 128>(p, s);
    return launch_append<192, 128>(p, s);
}

}  // namespace qmoe
