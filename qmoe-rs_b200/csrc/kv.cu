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
// Two launches.  The scan (one CTA, each thread a run of requests) writes
// q_start, kv_lens and each request's first place in the free list; the fill
// gives every token its request by bisection of q_start.  A new block's first
// position belongs to exactly one new token, which writes the table entry.

constexpr int kScanThreads = 1024;

struct Need {
    int64_t fresh;   // rows in the token buffer
    int64_t blocks;  // blocks wanted of the free list
    bool ok;         // fits the table and the token buffer
};

QMOE_DEV Need need_of(const KvPlanParams &p, int64_t r, int64_t end) {
    const int64_t c = p.cached[r], f = p.fresh[r];
    Need n;
    n.fresh = f > 0 ? f : 0;
    n.ok = c >= 0 && f >= 0 && c + f <= p.max_blocks * p.block && end + n.fresh <= p.capacity;
    n.blocks = n.ok ? (c + f + p.block - 1) / p.block - (c + p.block - 1) / p.block : 0;
    return n;
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
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < kScanThreads / 32; ++w) {
        if (w < warp) before += part[w];
        total += part[w];
    }
    return before + s - v;
}

__global__ void __launch_bounds__(kScanThreads) kv_scan_kernel(const KvPlanParams p) {
    __shared__ int64_t part[kScanThreads / 32];
    __shared__ int taken;
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int tid = threadIdx.x;
    const int64_t free_count = p.n_free;
    const int64_t per = (p.R + kScanThreads - 1) / kScanThreads;
    const int64_t lo = tid * per < p.R ? tid * per : p.R, hi = lo + per < p.R ? lo + per : p.R;
    if (tid == 0) taken = 0;
    int64_t sum = 0, total;
    for (int64_t r = lo; r < hi; ++r) sum += p.fresh[r] > 0 ? p.fresh[r] : 0;
    const int64_t row0 = block_scan(sum, part, total);
    int64_t row = row0;
    sum = 0;
    for (int64_t r = lo; r < hi; ++r) {
        const Need n = need_of(p, r, row);
        sum += n.blocks;
        row += n.fresh;
    }
    int64_t all;
    int64_t blk = block_scan(sum, part, all);
    int most = 0;
    row = row0;
    for (int64_t r = lo; r < hi; ++r) {
        const Need n = need_of(p, r, row);
        const bool ok = n.ok && (n.blocks == 0 || blk + n.blocks <= free_count);
        p.q_start[r] = (int32_t)(row < INT32_MAX ? row : INT32_MAX);
        p.kv_lens[r] = ok ? p.cached[r] + p.fresh[r] : 0;
        p.first[r] = (int32_t)(blk < INT32_MAX ? blk : INT32_MAX);
        blk += n.blocks;
        if (ok && n.blocks) most = (int)blk;
        row += n.fresh;
    }
    atomicMax(&taken, most);
    __syncthreads();
    if (tid == 0) {
        p.q_start[p.R] = (int32_t)(total < INT32_MAX ? total : INT32_MAX);
        p.taken[0] = taken;
    }
}

constexpr int kFillThreads = 256;

__global__ void __launch_bounds__(kFillThreads) kv_fill_kernel(const KvPlanParams p) {
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int64_t t = (int64_t)blockIdx.x * kFillThreads + threadIdx.x;
    if (t >= p.capacity) return;
    int slot = -1, pos = -1;
    if (t < p.q_start[p.R]) {
        int64_t lo = 0, hi = p.R;                 // q_start[lo] <= t < q_start[hi]
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (p.q_start[mid] <= t) lo = mid;
            else hi = mid;
        }
        if (p.kv_lens[lo] > 0) {
            const int c = p.cached[lo], have = (c + p.block - 1) / p.block;
            pos = c + (int)(t - p.q_start[lo]);
            const int b = pos / p.block, off = pos - b * p.block;
            int32_t *entry = p.table + lo * p.max_blocks + b;
            int id;
            if (b >= have) {
                id = p.free_blocks[p.first[lo] + b - have];
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

// ---- append --------------------------------------------------------------------
//
// One warp per (token, head) whose token starts a run: consecutive slots of
// one block.  Offsets before the run are the block's earlier tokens.  The
// range grows to the new tokens' largest magnitude, the earlier codes are
// rounded to the new range (kept when it did not grow), the new ones written.

constexpr int kAppendWarps = 8;

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

// Place of (token, dim) among the codes of one block and head, from the first
// of four dims; V steps 16 bytes a dim, K one.
template <bool IS_V>
QMOE_DEV int code_at(int tok, int d, int dim, int block) {
    return IS_V ? ((tok >> 4) * dim + d) * 16 + (tok & 15) : ((d >> 6) * block + tok) * 64 + (d & 63);
}

template <bool BF16, bool IS_V>
QMOE_DEV void append_run(const void *x, int64_t ld, int dim, bool vec, int8_t *codes, float *range, int head,
                         int64_t t, int n, int off, int block) {
    const int lane = threadIdx.x & 31;
    float m = 0.0f;
    bool bad = false;
    const int per = dim / 4;                       // groups of four dims in a row
    for (int e = lane; e < n * per; e += 32) {
        const int i = e / per, d = (e - i * per) * 4;
        const float4 v = load4<BF16>(x, (t + i) * ld + (int64_t)head * dim + d, vec);
        m = max_abs(max_abs(max_abs(max_abs(m, v.x), v.y), v.z), v.w);
        const float inf = __int_as_float(0x7f800000);
        bad |= !(fabsf(v.x) < inf && fabsf(v.y) < inf && fabsf(v.z) < inf && fabsf(v.w) < inf);
    }
    m = warp_max(m);
    bad = __any_sync(0xffffffffu, bad);
    const float old = off > 0 ? *range : 0.0f;
    bad |= !(fabsf(old) < __int_as_float(0x7f800000));
    const float r = range8(fmaxf(m, old), !bad), mi = __fdiv_rn(127.0f, r);
    __syncwarp();
    if (lane == 0) *range = r;
    if (off > 0 && !(r == old)) {
        const float oi = __fdiv_rn(old, r);
        for (int e = lane; e < off * per; e += 32) {
            const int i = e / per, d = (e - i * per) * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int8_t *c = codes + code_at<IS_V>(i, d + j, dim, block);
                *c = (int8_t)code8((float)*c, old, r, oi);
            }
        }
    }
    for (int e = lane; e < n * per; e += 32) {
        const int i = e / per, d = (e - i * per) * 4;
        const float4 v = load4<BF16>(x, (t + i) * ld + (int64_t)head * dim + d, vec);
        const int c0 = code8(v.x, 127.0f, r, mi), c1 = code8(v.y, 127.0f, r, mi);
        const int c2 = code8(v.z, 127.0f, r, mi), c3 = code8(v.w, 127.0f, r, mi);
        int8_t *c = codes + code_at<IS_V>(off + i, d, dim, block);
        if (IS_V) {
            c[0] = (int8_t)c0;
            c[16] = (int8_t)c1;
            c[32] = (int8_t)c2;
            c[48] = (int8_t)c3;
        } else {
            *reinterpret_cast<uint32_t *>(c) = pack4(c0, c1, c2, c3);
        }
    }
}

template <bool BF16>
__global__ void __launch_bounds__(kAppendWarps * 32) kv_append_kernel(const KvAppendParams p) {
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int64_t t = w / p.c.heads;
    const int h = (int)(w - t * p.c.heads);
    if (t >= p.T) return;
    const int64_t total = p.c.num_blocks * p.c.block;
    const int slot = p.slots[t];
    if (slot < 0 || slot >= total) return;
    const int off = slot % p.c.block;
    const int64_t blk = slot / p.c.block;
    if (off > 0 && t > 0 && p.slots[t - 1] == slot - 1) return;   // inside another token's run
    int n = 0;
    for (int base = 0; base < p.c.block - off; base += 32) {
        const int i = base + lane;
        const bool in = off + i < p.c.block && t + i < p.T && p.slots[t + i] == slot + i;
        const unsigned miss = ~__ballot_sync(0xffffffffu, in);
        n += miss ? __ffs(miss) - 1 : 32;
        if (miss) break;
    }
    const int64_t bh = blk * p.c.heads + h;
    append_run<BF16, false>(p.k, p.ldk, p.c.k_dim, p.vec_k, p.c.k + bh * p.c.block * p.c.k_dim, p.c.k_range + bh, h,
                            t, n, off, p.c.block);
    append_run<BF16, true>(p.v, p.ldv, p.c.v_dim, p.vec_v, p.c.v + bh * p.c.block * p.c.v_dim, p.c.v_range + bh, h,
                           t, n, off, p.c.block);
}

}  // namespace

cudaError_t launch_kv_plan(const KvPlanParams &p, cudaStream_t s) {
    cudaError_t e = launch_pdl(kv_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, p);
    if (e != cudaSuccess || p.capacity == 0) return e;
    return launch_pdl(kv_fill_kernel, dim3((unsigned)((p.capacity + kFillThreads - 1) / kFillThreads)),
                      dim3(kFillThreads), 0, s, p);
}

cudaError_t launch_kv_append(const KvAppendParams &p, cudaStream_t s) {
    if (p.T == 0) return cudaSuccess;
    const int64_t warps = p.T * p.c.heads;
    return launch_pdl(p.dtype ? kv_append_kernel<true> : kv_append_kernel<false>,
                      dim3((unsigned)((warps + kAppendWarps - 1) / kAppendWarps)), dim3(kAppendWarps * 32), 0, s, p);
}

}  // namespace qmoe
