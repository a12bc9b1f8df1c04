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
#include "sm100.cuh"

namespace qmoe {
namespace {

using namespace sm100;

// ---- rows to codes ---------------------------------------------------------

constexpr int kRowThreads = 256;

template <bool BF16>
QMOE_DEV float load1(const void *x, int64_t i) {
    return BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(x)[i])
                : reinterpret_cast<const float *>(x)[i];
}

// One CTA per row: its largest magnitude, then its codes (the row comes from
// L1 / L2 the second time).
template <bool BF16>
__global__ void __launch_bounds__(kRowThreads)
quant_rows_kernel(const Int8RowsParams p) {
    __shared__ float wmax[kRowThreads / 32];
    __shared__ int wbad[kRowThreads / 32];
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int64_t t = blockIdx.x;
    const int64_t base = t * p.ldx;
    const int tid = threadIdx.x;
    float m = 0.0f;
    bool bad = false;
    for (int k = tid; k < p.K; k += kRowThreads) {
        const float v = load1<BF16>(p.x, base + k);
        m = max_abs(m, v);
        bad |= !(fabsf(v) < __int_as_float(0x7f800000));
    }
    m = warp_max(m);
    bad = __any_sync(0xffffffffu, bad);
    if ((tid & 31) == 0) {
        wmax[tid >> 5] = m;
        wbad[tid >> 5] = bad;
    }
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) {
        m = fmaxf(m, wmax[w]);
        any |= wbad[w];
    }
    const float r = range8(m, !any), mi = __fdiv_rn(127.0f, r);
    int8_t *o = p.codes + t * p.ldc;
    for (int k = tid; k < p.ldc; k += kRowThreads)
        o[k] = (int8_t)(k < p.K ? code8(load1<BF16>(p.x, base + k), 127.0f, r, mi) : 0);
    if (tid == 0) p.scales[t] = __fdiv_rn(r, 127.0f);
}

// ---- the product -------------------------------------------------------------
//
// Output channels are the MMA's M (128 a tile, one TMEM lane each) and tokens
// its N (up to BN a tile), so one kernel serves one token and a long prompt:
// the weights always stream through the wide operand.  Both operands come by
// TMA in 128-byte K blocks (128-byte swizzle), rows and K past the end filled
// with zeros, and the accumulator is double-buffered in tensor memory.
//
// Persistent grid, eight warps: 0 TMA producer, 1 MMA issuer, 2 TMEM owner,
// 4-7 epilogue (one TMEM lane quarter each).  Every wait is bounded; on a
// time-out the kernel flags the device error word, drains its copies and MMAs
// (again bounded), frees TMEM and returns.

constexpr int kThreads = 256;
constexpr int kABytes = 128 * 128;

template <int BN>
struct Tile {
    static constexpr int stage = kABytes + BN * 128;
    static constexpr int stages = 200 * 1024 / stage > 8 ? 8 : 200 * 1024 / stage;
    static constexpr uint32_t cols = 2 * BN < 32 ? 32 : 2 * BN;
};

constexpr int kMaxStages = 8;

struct Smem {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t dfull[2], dempty[2], drain;
    uint32_t tmem_base;
    int abort;
};

QMOE_DEV void mma_i8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}

template <int BN, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                 const Int8GemmParams p) {
    using Cfg = Tile<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Smem *S = reinterpret_cast<Smem *>(ring + Cfg::stages * Cfg::stage);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    QMOE_PDL_WAIT();
    QMOE_PDL_TRIGGER();
    const int tiles_t = (int)((p.T + BN - 1) / BN), tiles_n = (int)((p.N + 127) / 128);
    const int total = tiles_t * tiles_n;            // at least the grid
    const int nkb = (p.K + 127) / 128;

    if (tid == 0) {
        for (int i = 0; i < Cfg::stages; ++i) {
            mbar_init(&S->full[i], 1);
            mbar_init(&S->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S->dfull[i], 1);
            mbar_init(&S->dempty[i], 4);
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
            uint32_t u = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
                const int t0 = (tile % tiles_t) * BN, n0 = (tile / tiles_t) * 128;
                for (int kb = 0; kb < nkb; ++kb, ++u) {
                    const uint32_t s = u % Cfg::stages;
                    if (!(ok = mbar_wait(&S->empty[s], ((u / Cfg::stages) & 1) ^ 1, abort, p.err))) break;
                    mbar_arrive_expect_tx(&S->full[s], Cfg::stage);
                    tma_load_2d(ring + s * Cfg::stage, &tm_w, &S->full[s], kb * 128, n0);
                    tma_load_2d(ring + s * Cfg::stage + kABytes, &tm_x, &S->full[s], kb * 128, t0);
                }
            }
            if (!ok)  // let the copies already issued land before the CTA exits
                for (uint32_t v = u > Cfg::stages ? u - Cfg::stages : 0; v < u; ++v)
                    for (uint32_t n = 0; n < kMaxWaitProbes; ++n)
                        if (mbar_try_wait(&S->full[v % Cfg::stages], (v / Cfg::stages) & 1)) break;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t u = 0, i = 0;
            bool ok = true, issued = false;
            const uint64_t d0 = smem_desc(smem_u32(ring), 16, 1024, 2);
            for (int tile = blockIdx.x; ok && tile < total; tile += gridDim.x, ++i) {
                const int64_t left = p.T - (int64_t)(tile % tiles_t) * BN;
                const int N = left >= BN ? BN : (int)(left + 15) / 16 * 16;
                const uint32_t idesc = idesc_i8(128, N, true, true);
                const uint32_t d = tmem + (i & 1) * BN;
                if (!(ok = mbar_wait(&S->dempty[i & 1], ((i >> 1) & 1) ^ 1, abort, p.err))) break;
                tc_fence_after();
                for (int kb = 0; kb < nkb; ++kb, ++u) {
                    const uint32_t s = u % Cfg::stages;
                    if (!(ok = mbar_wait(&S->full[s], (u / Cfg::stages) & 1, abort, p.err))) break;
                    tc_fence_after();
                    const uint64_t a = d0 + ((s * Cfg::stage) >> 4), b = a + (kABytes >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) mma_i8_ss(d, a + 2 * kk, b + 2 * kk, idesc, (kb | kk) != 0);
                    issued = true;
                    mma_commit(&S->empty[s]);
                }
                if (!ok) break;
                mma_commit(&S->dfull[i & 1]);
            }
            // every MMA issued so far completes before TMEM is freed
            if (issued) {
                mma_commit(&S->drain);
                for (uint32_t n = 0; n < kMaxWaitProbes; ++n)
                    if (mbar_try_wait(&S->drain, 0)) break;
            }
        }
    } else if (warp >= 4) {
        constexpr int CH = BN < 32 ? 16 : 32;
        const int q = warp & 3;
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        uint32_t i = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < total; tile += gridDim.x, ++i) {
            const int64_t t0 = (int64_t)(tile % tiles_t) * BN;
            const int n = (tile / tiles_t) * 128 + q * 32 + lane;
            const float sw = n < p.N ? __ldg(p.sw + n) : 0.0f;
            const int count = (int)(p.T - t0 < BN ? p.T - t0 : BN);
            if (!(ok = mbar_wait_warp(&S->dfull[i & 1], (i >> 1) & 1, abort, p.err))) break;
            tc_fence_after();
            for (int c = 0; c < count; c += CH) {
                uint32_t v[CH];
                if constexpr (CH == 32) tmem_ld_x32(tmem + lane_addr + (i & 1) * BN + c, v);
                else tmem_ld_x16(tmem + lane_addr + (i & 1) * BN + c, v);
                tmem_wait_ld();
                if (c + CH >= count) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S->dempty[i & 1]);
                }
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    if (c + j >= count || n >= p.N) continue;
                    const int64_t t = t0 + c + j, at = t * p.N + n;
                    float y = __fmul_rn(__fmul_rn((float)(int)v[j], __ldg(p.sx + t)), sw);
                    if (p.residual) y = __fadd_rn(y, load1<BF16>(p.residual, at));
                    if (BF16) reinterpret_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(y);
                    else reinterpret_cast<float *>(p.y)[at] = y;
                }
                __syncwarp();
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::cols);
    }
}

template <int BN>
cudaError_t launch_bn(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const Int8GemmParams &p, cudaStream_t s) {
    using Cfg = Tile<BN>;
    const size_t smem = 1024 + (size_t)Cfg::stages * Cfg::stage + sizeof(Smem);
    auto kernel = p.dtype ? int8_gemm_kernel<BN, true> : int8_gemm_kernel<BN, false>;
    cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem);
    if (e != cudaSuccess) return e;
    const int64_t total = ((p.T + BN - 1) / BN) * ((p.N + 127) / 128);
    const int64_t sms = device_sm_count();
    return launch_pdl(kernel, dim3((unsigned)(total < sms ? total : sms)), dim3(kThreads), smem, s, tm_w, tm_x, p);
}

}  // namespace

int int8_token_tile(int64_t T) { return T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256; }

cudaError_t launch_quant_rows(const Int8RowsParams &p, cudaStream_t s) {
    if (p.T == 0) return cudaSuccess;
    return launch_pdl(p.dtype ? quant_rows_kernel<true> : quant_rows_kernel<false>, dim3((unsigned)p.T),
                      dim3(kRowThreads), 0, s, p);
}

cudaError_t launch_int8_gemm(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const Int8GemmParams &p,
                             cudaStream_t s) {
    switch (int8_token_tile(p.T)) {
        case 16: return launch_bn<16>(tm_w, tm_x, p, s);
        case 32: return launch_bn<32>(tm_w, tm_x, p, s);
        case 64: return launch_bn<64>(tm_w, tm_x, p, s);
        case 128: return launch_bn<128>(tm_w, tm_x, p, s);
        default: return launch_bn<256>(tm_w, tm_x, p, s);
    }
}

}  // namespace qmoe
