// int8.cu -- the matrix product in 8-bit integers with a scale for each token
// and each output channel, and the row quantiser in front of it.
//
//   y[t, n] = (sum_k cx[t, k] * cw[n, k]) * sx[t] * sw[n]  (+ residual[t, n])
//
// cx, sx: the codes and scale of row t of x (code8.cuh); cw, sw: the weight's.
// The sum is a 32-bit integer and exact (K <= 131072: 127^2 K < 2^31), so
// neither tile shape nor order changes a result; the rest is f32, rounded
// once to x's type.  A row of x with a non-finite element has the scale NaN.
#include "code8.cuh"
#include "kernels.h"
#include "mma_warp.cuh"

namespace qmoe {
namespace {

using namespace sm100;

// ---- rows to codes ---------------------------------------------------------

template <bool BF16>
QMOE_DEV float load1(const void *x, int64_t i) {
    return BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(x)[i])
                : reinterpret_cast<const float *>(x)[i];
}

// Eight elements from a 16-byte aligned address.
template <bool BF16>
QMOE_DEV void load8(const void *x, int64_t i, float (&v)[8]) {
    const float4 a = load_act4(x, BF16 ? 1 : 0, i), b = load_act4(x, BF16 ? 1 : 0, i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// THREADS per row, each 8 * GROUPS elements of it in registers (GROUPS 0: any
// length or alignment, read twice).  A row is one load latency and one
// reduction, so short rows share a CTA (a warp each) and longer ones take as many
// threads as leave each one or two groups (2624 bf16 on 256 threads instead of
// 512: 4096 rows and their product to 64 channels 34 -> 25 us; four groups a
// thread are faster at 4096 rows of 7168, 49 -> 42, and slower at 400 of 8192,
// 13.5 -> 15.0).
template <bool BF16, int THREADS, int GROUPS>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS)
quant_rows_kernel(const Int8RowsParams p) {
    constexpr int kRows = THREADS < 128 ? 128 / THREADS : 1;
    constexpr int kW = THREADS / 32;              // warps of a row
    __shared__ float wmax[kW];
    __shared__ int wbad[kW];
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int tid = threadIdx.x % THREADS;
    const int64_t t = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
    if (t >= p.T) return;                         // kRows > 1: whole warps, no CTA barrier follows
    const int64_t base = t * p.ldx;
    float v[GROUPS ? GROUPS : 1][8];
    float m = 0.0f;
    bool bad = false;
    if constexpr (GROUPS > 0) {
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            const int k = (q * THREADS + tid) * 8;
            if (k < p.K) {
                load8<BF16>(p.x, base + k, v[q]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[q][j] = 0.0f;
            }
        }
#pragma unroll
        for (int q = 0; q < GROUPS; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m = max_abs(m, v[q][j]);
                bad |= !(fabsf(v[q][j]) < __int_as_float(0x7f800000));
            }
    } else {
        for (int k = tid; k < p.K; k += THREADS) {
            const float x = load1<BF16>(p.x, base + k);
            m = max_abs(m, x);
            bad |= !(fabsf(x) < __int_as_float(0x7f800000));
        }
    }
    m = warp_max(m);
    bad = __any_sync(0xffffffffu, bad);
    if constexpr (kW > 1) {
        if ((tid & 31) == 0) {
            wmax[tid >> 5] = m;
            wbad[tid >> 5] = bad;
        }
        __syncthreads();
        const int i = tid & 31;
        m = warp_max(i < kW ? wmax[i] : 0.0f);
        bad = __any_sync(0xffffffffu, i < kW && wbad[i]);
    }
    const float r = range8(m, !bad), mi = __fdiv_rn(127.0f, r);
    int8_t *o = p.codes + t * p.ldc;
    if constexpr (GROUPS > 0) {
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            const int k = (q * THREADS + tid) * 8;
            if (k >= p.ldc) continue;
            *reinterpret_cast<uint2 *>(o + k) = make_uint2(codes4(v[q][0], v[q][1], v[q][2], v[q][3], 127.0f, r, mi),
                                                           codes4(v[q][4], v[q][5], v[q][6], v[q][7], 127.0f, r, mi));
        }
    } else {
        for (int k = tid; k < p.ldc; k += THREADS)
            o[k] = (int8_t)(k < p.K ? code8(load1<BF16>(p.x, base + k), 127.0f, r, mi) : 0);
    }
    if (tid == 0) p.scales[t] = __fdiv_rn(r, 127.0f);
}

template <int THREADS, int GROUPS>
cudaError_t launch_rows(const Int8RowsParams &p, cudaStream_t s) {
    constexpr int kRows = THREADS < 128 ? 128 / THREADS : 1;
    return launch_pdl(p.dtype ? quant_rows_kernel<true, THREADS, GROUPS> : quant_rows_kernel<false, THREADS, GROUPS>,
                      dim3((unsigned)((p.T + kRows - 1) / kRows)), dim3(THREADS < 128 ? 128 : THREADS), 0, s, p);
}

// ---- the product -------------------------------------------------------------
//
// Output channels are the MMA's M (128 a tile, one TMEM lane each) and tokens
// its N (up to BN a tile), so one kernel serves one token and a long prompt:
// the weights always stream through the wide operand.  Both operands come by
// TMA in 128-byte K blocks (128-byte swizzle), rows and K past the end filled
// with zeros, and the accumulator is double-buffered in tensor memory.
//
// Eight warps: 0 TMA producer, 1 MMA issuer, 2 TMEM owner, 4-7 epilogue (one
// TMEM lane quarter each).  With tiles enough for the device the grid is
// persistent and a tile's epilogue runs under the next one's MMAs.  With fewer,
// a cluster of CTAs takes the K blocks of one tile in parts: each leaves its
// 32-bit sums in its shared memory, and after a cluster barrier each adds its
// share of the tokens from all of them (integers, so the parts' order does not
// matter).  The first weight blocks are asked for before the row quantiser in
// front has finished.
//
// Every wait is bounded; on a time-out the kernel flags the device error word,
// drains its copies and MMAs (again bounded), frees TMEM and returns.

constexpr int kABytes = 128 * 128;

// Up to 64 tokens two CTAs share an SM, so that one streams while the other
// starts or ends (four with half the stages: 32 tokens by 16384 to 7168 29.3 us,
// with two 27.3).  Wider tiles have eight warps for the epilogue: at K = 1024 it
// is what bounds the product (4096 tokens to 4096 channels, a residual added:
// 95 us with four warps and the residual loaded as it was needed, 50 us with
// eight that load a chunk ahead; 61 -> 30 without a residual).
template <int BN>
struct Tile {
    static constexpr int stage = kABytes + BN * 128;
    static constexpr int stages = (BN <= 64 ? 100 : 200) * 1024 / stage;
    static constexpr int ctas = BN <= 64 ? 2 : 1;
    static constexpr int epilogue = BN <= 64 ? 4 : 8;                 // warps
    static constexpr int threads = 128 + epilogue * 32;
    static constexpr uint32_t cols = 2 * BN < 32 ? 32 : 2 * BN;
    static_assert(stages * stage >= BN * 512, "the sums of a tile do not fit the ring");
    static_assert(ctas * cols <= 512, "tensor memory");
};

constexpr int kMaxStages = 8;

struct Smem {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t dfull[2], dempty[2], drain;
    uint32_t tmem_base;
    int abort;
    alignas(16) float sx[8][256];                             // each epilogue warp's copy of a tile's token scales
};

// The factors of a row and a channel, 2^-24 of the one and 2^24 of the other: a
// sum (below 2^31) times a row's scale (below 2^121) is then in f32's range, the
// result the same to the bit.
QMOE_DEV float row_factor(float sx) { return sx * 5.9604644775390625e-08f; }
QMOE_DEV float channel_factor(float sw) { return sw * 16777216.0f; }
// Without a residual res is -0: adding it changes no value.
QMOE_DEV float finish(int sum, float sx, float sw, float res) {
    return __fadd_rn(__fmul_rn(__fmul_rn((float)sum, sx), sw), res);
}
template <bool BF16>
QMOE_DEV void store1(void *out, int64_t at, float y) {
    if (BF16) reinterpret_cast<__nv_bfloat16 *>(out)[at] = __float2bfloat16_rn(y);
    else reinterpret_cast<float *>(out)[at] = y;
}

// A lane's channel of rows row .. row + CH - 1 (up to `count`) of the residual
// at `at`, all in flight at once.
template <bool BF16, int CH>
QMOE_DEV void load_rows(const void *residual, int64_t at, int N, int row, int count, float (&res)[CH]) {
    if (row + CH <= count) {
        at += (int64_t)row * N;
#pragma unroll
        for (int j = 0; j < CH; ++j) res[j] = load1<BF16>(residual, at + (int64_t)j * N);
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (row + j < count) res[j] = load1<BF16>(residual, at + (int64_t)(row + j) * N);
    }
}

QMOE_DEV void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}

// The int at this CTA's shared address, in CTA `rank` of the cluster.
QMOE_DEV int load_cluster(const int *at, int rank) {
    uint32_t remote;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(at)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    return v;
}

template <int BN, bool BF16>
__global__ void __launch_bounds__(Tile<BN>::threads, Tile<BN>::ctas)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                 const Int8GemmParams p, const int parts) {
    using Cfg = Tile<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Smem *S = reinterpret_cast<Smem *>(ring + Cfg::stages * Cfg::stage);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    QMOE_PDL_TRIGGER();
    const int tiles_t = (int)((p.T + BN - 1) / BN), tiles_n = (int)((p.N + 127) / 128);
    const int total = tiles_t * tiles_n;
    const int nkb = (p.K + 127) / 128;
    // the tiles of this CTA (parts > 1: one), and its K blocks of them
    const int rank = parts > 1 ? blockIdx.x % parts : 0;
    const int tile0 = parts > 1 ? blockIdx.x / parts : blockIdx.x, step = parts > 1 ? total : gridDim.x;
    const int kb0 = nkb * rank / parts, kb1 = nkb * (rank + 1) / parts;

    if (tid == 0) {
        for (int i = 0; i < Cfg::stages; ++i) {
            mbar_init(&S->full[i], 1);
            mbar_init(&S->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S->dfull[i], 1);
            mbar_init(&S->dempty[i], Cfg::epilogue);
        }
        mbar_init(&S->drain, 1);
        S->abort = 0;
        fence_mbar_init();
    }
    if (warp == 2) {
        tmem_alloc(&S->tmem_base, Cfg::cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = S->tmem_base;
    volatile int *abort = &S->abort;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t u = 0, early = 0;
            bool ok = true;
            {   // weights of the first blocks: nothing in front of this kernel writes them
                const int n0 = (tile0 / tiles_t) * 128;
                for (; (int)early < kb1 - kb0 && early < Cfg::stages; ++early) {
                    mbar_arrive_expect_tx(&S->full[early], Cfg::stage);
                    tma_load_2d(ring + early * Cfg::stage, &tm_w, &S->full[early], (kb0 + (int)early) * 128, n0);
                }
            }
            QMOE_PDL_WAIT();
            for (int tile = tile0; ok && tile < total; tile += step) {
                const int t0 = (tile % tiles_t) * BN, n0 = (tile / tiles_t) * 128;
                for (int kb = kb0; kb < kb1; ++kb, ++u) {
                    const uint32_t s = u % Cfg::stages;
                    if (u >= early) {
                        if (!(ok = mbar_wait(&S->empty[s], ((u / Cfg::stages) & 1) ^ 1, abort, p.err))) break;
                        mbar_arrive_expect_tx(&S->full[s], Cfg::stage);
                        tma_load_2d(ring + s * Cfg::stage, &tm_w, &S->full[s], kb * 128, n0);
                    }
                    tma_load_2d(ring + s * Cfg::stage + kABytes, &tm_x, &S->full[s], kb * 128, t0);
                }
            }
            if (!ok)  // let the copies already issued land before the CTA exits
                for (uint32_t v = u > Cfg::stages ? u - Cfg::stages : 0; v < u; ++v)
                    for (uint32_t n = 0; n < kMaxWaitProbes; ++n)
                        if (mbar_try_wait(&S->full[v % Cfg::stages], (v / Cfg::stages) & 1)) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        uint32_t u = 0, i = 0;
        bool ok = true, issued = false;
        const uint64_t d0 = smem_desc(smem_u32(ring), 16, 1024, 2);
        const uint32_t lo = (uint32_t)d0, hi = (uint32_t)(d0 >> 32);
        for (int tile = tile0; ok && tile < total; tile += step, ++i) {
            const int64_t left = p.T - (int64_t)(tile % tiles_t) * BN;
            const int N = left >= BN ? BN : (int)(left + 15) / 16 * 16;
            const uint32_t idesc = idesc_i8(128, N, true, true);
            const uint32_t d = tmem + (i & 1) * BN;
            if (!(ok = mbar_wait_warp(&S->dempty[i & 1], ((i >> 1) & 1) ^ 1, abort, p.err))) break;
            tc_fence_after();
            for (int kb = kb0; kb < kb1; ++kb, ++u) {
                const uint32_t s = u % Cfg::stages;
                if (!(ok = mbar_wait_warp(&S->full[s], (u / Cfg::stages) & 1, abort, p.err))) break;
                tc_fence_after();
                const uint32_t a = lo + ((s * Cfg::stage) >> 4), b = a + (kABytes >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    warp_mma_i8_ss(d, a + 2 * kk, b + 2 * kk, hi, idesc, (kb != kb0) | (kk != 0));
                issued = true;
                warp_commit(&S->empty[s]);
            }
            if (!ok) break;
            warp_commit(&S->dfull[i & 1]);
        }
        // every MMA issued so far completes before TMEM is freed
        if (issued) {
            warp_commit(&S->drain);
            for (uint32_t n = 0; n < kMaxWaitProbes; ++n)
                if (__all_sync(0xffffffffu, mbar_try_wait(&S->drain, 0))) break;
        }
        __syncwarp();
    } else if (warp >= 4) {
        // chunks of tokens, dealt to the warps of a quarter of tensor memory
        constexpr int CH = BN < 32 ? 16 : 32, kStep = CH * (Cfg::epilogue / 4);
        const int q = warp & 3, c0 = CH * ((warp - 4) >> 2);
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        const bool adds = parts == 1 && p.residual;
        const int N = (int)p.N;
        float *sx = S->sx[warp - 4];
        uint32_t i = 0;
        bool ok = true;
        QMOE_PDL_WAIT();
        for (int tile = tile0; ok && tile < total; tile += step, ++i) {
            const int64_t t0 = (int64_t)(tile % tiles_t) * BN;
            const int n = (tile / tiles_t) * 128 + q * 32 + lane, nn = n < p.N ? n : p.N - 1;
            const int count = (int)(p.T - t0 < BN ? p.T - t0 : BN);
            const int64_t at = t0 * p.N + nn;
            const float sw = channel_factor(__ldg(p.sw + nn));
            float next[CH];                       // residual of the chunk to come
#pragma unroll
            for (int j = 0; j < CH; ++j) next[j] = -0.0f;
            if (adds) load_rows<BF16>(p.residual, at, N, c0, count, next);
            __syncwarp();
            for (int j = lane; j < count; j += 32) sx[j] = row_factor(p.sx[t0 + j]);
            __syncwarp();
            if (!(ok = mbar_wait_warp(&S->dfull[i & 1], (i >> 1) & 1, abort, p.err))) break;
            tc_fence_after();
            // rolled: a tile's code stays small beside the other warps'
#pragma unroll 1
            for (int c = c0; c < count; c += kStep) {
                uint32_t v[CH];
                if constexpr (CH == 32) tmem_ld_x32(tmem + lane_addr + (i & 1) * BN + c, v);
                else tmem_ld_x16(tmem + lane_addr + (i & 1) * BN + c, v);
                float res[CH];
#pragma unroll
                for (int j = 0; j < CH; ++j) res[j] = next[j];
                if (adds) load_rows<BF16>(p.residual, at, N, c + kStep, count, next);
                tmem_wait_ld();
                if (parts > 1) {                  // every MMA has read its operands: the ring is free
                    int *sums = reinterpret_cast<int *>(ring);
#pragma unroll
                    for (int j = 0; j < CH; ++j) sums[(c + j) * 128 + q * 32 + lane] = (int)v[j];
                } else {
                    float y[CH];
#pragma unroll
                    for (int j = 0; j < CH; j += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(sx + c + j);
                        y[j] = finish((int)v[j], f.x, sw, res[j]);
                        y[j + 1] = finish((int)v[j + 1], f.y, sw, res[j + 1]);
                        y[j + 2] = finish((int)v[j + 2], f.z, sw, res[j + 2]);
                        y[j + 3] = finish((int)v[j + 3], f.w, sw, res[j + 3]);
                    }
                    const int64_t first = at + (int64_t)c * N;
                    if (n < p.N && c + CH <= count) {
#pragma unroll
                        for (int j = 0; j < CH; ++j) store1<BF16>(p.y, first + (int64_t)j * N, y[j]);
                    } else if (n < p.N) {
#pragma unroll
                        for (int j = 0; j < CH; ++j)
                            if (c + j < count) store1<BF16>(p.y, first + (int64_t)j * N, y[j]);
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S->dempty[i & 1]);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::cols);
        __syncwarp();
    }
    if (parts > 1) {
        QMOE_PDL_WAIT();
        cluster_barrier();
        const int64_t t0 = (int64_t)(tile0 % tiles_t) * BN;
        const int n = (tile0 / tiles_t) * 128 + (tid & 127);
        const int count = (int)(p.T - t0 < BN ? p.T - t0 : BN);
        const int *sums = reinterpret_cast<const int *>(ring);
        const float sw = n < p.N ? channel_factor(__ldg(p.sw + n)) : 0.0f;
        for (int j = rank + parts * (tid >> 7); j < count; j += Cfg::threads / 128 * parts) {
            int sum = 0;
            for (int r = 0; r < parts; ++r) sum += load_cluster(sums + j * 128 + (tid & 127), r);
            if (n < p.N)
                store1<BF16>(p.y, (t0 + j) * p.N + n,
                             finish(sum, row_factor(p.sx[t0 + j]), sw,
                                    p.residual ? load1<BF16>(p.residual, (t0 + j) * p.N + n) : -0.0f));
        }
        cluster_barrier();                        // the others may still read this CTA's sums
    }
}

// How a product is cut.  Up to 64 tokens one tile holds them all (the weights
// are read once); above, the widest tile of 256, 128 or 64 tokens that gives
// every SM one.  Where the tiles are still too few, clusters of 2, 4 or 8 CTAs
// share a tile's K, with two K blocks each at least (other sizes do not fill
// the device: 56 tiles of 32 tokens by 16384 take 27.7 us in fours, 30.1 in
// threes, 40 in fives).
struct Cut {
    int bn, parts;
};
Cut cut_of(int64_t T, int64_t N, int K) {
    const int64_t sms = device_sm_count(), tn = (N + 127) / 128, nkb = (K + 127) / 128;
    Cut c;
    c.bn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256;
    while (T > 64 && c.bn > 64 && tn * ((T + c.bn - 1) / c.bn) < sms) c.bn /= 2;
    const int64_t tiles = tn * ((T + c.bn - 1) / c.bn), room = sms * (c.bn <= 64 ? 2 : 1);
    int64_t parts = room / tiles;
    if (parts > nkb / 2) parts = nkb / 2;
    c.parts = parts < 2 ? 1 : parts < 4 ? 2 : parts < 8 ? 4 : 8;
    return c;
}

template <int BN>
cudaError_t launch_bn(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const Int8GemmParams &p, int parts,
                      cudaStream_t s) {
    using Cfg = Tile<BN>;
    const size_t smem = 1024 + (size_t)Cfg::stages * Cfg::stage + sizeof(Smem);
    auto kernel = p.dtype ? int8_gemm_kernel<BN, true> : int8_gemm_kernel<BN, false>;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    const int64_t total = ((p.T + BN - 1) / BN) * ((p.N + 127) / 128), room = (int64_t)device_sm_count() * Cfg::ctas;
    const int64_t grid = parts > 1 ? total * parts : total < room ? total : room;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(Cfg::threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, tm_w, tm_x, p, parts);
}

}  // namespace

int int8_token_tile(int64_t T, int64_t N, int K) { return cut_of(T, N, K).bn; }

cudaError_t launch_quant_rows(const Int8RowsParams &p, cudaStream_t s) {
    if (p.T == 0) return cudaSuccess;
    // whole groups of eight elements and codes, aligned
    const uintptr_t es = p.dtype ? 2 : 4;
    const bool vec = p.K % 8 == 0 && p.ldc % 8 == 0 && p.ldx % (16 / es) == 0 &&
                     reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.codes) % 8 == 0;
    if (!vec) return p.ldc <= 1024 ? launch_rows<32, 0>(p, s) : launch_rows<256, 0>(p, s);
    if (p.ldc <= 512) return launch_rows<32, 2>(p, s);
    if (p.ldc <= 2048) return launch_rows<128, 2>(p, s);
    if (p.ldc <= 4096) return launch_rows<256, 2>(p, s);
    if (p.ldc <= 8192) return launch_rows<512, 2>(p, s);
    if (p.ldc <= 16384) return launch_rows<1024, 2>(p, s);
    return launch_rows<1024, 0>(p, s);
}

cudaError_t launch_int8_gemm(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const Int8GemmParams &p,
                             cudaStream_t s) {
    const Cut c = cut_of(p.T, p.N, p.K);
    switch (c.bn) {
        case 16: return launch_bn<16>(tm_w, tm_x, p, c.parts, s);
        case 32: return launch_bn<32>(tm_w, tm_x, p, c.parts, s);
        case 64: return launch_bn<64>(tm_w, tm_x, p, c.parts, s);
        case 128: return launch_bn<128>(tm_w, tm_x, p, c.parts, s);
        default: return launch_bn<256>(tm_w, tm_x, p, c.parts, s);
    }
}

}  // namespace qmoe
