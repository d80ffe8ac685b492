// 8-bit products on the tensor cores (tcgen05 kind::i8, 32-bit integer sums in TMEM):
// 256 x 256 tiles by CTA pairs for large products, 128 channels x up to 128 tokens by
// single CTAs for small ones; several of either may split K.  Both are launched as
// dependents of the kernel before them: they set themselves up while it ends, and wait
// for its end before they read its results.
#include <algorithm>
#include <atomic>
#include <climits>
#include <mutex>

#include "int8_common.cuh"

namespace hb {
namespace {

using namespace ptx;
constexpr unsigned FULL = 0xffffffffu;

// HB_DEV_* bits of the launches on this device (read by hb_int8_status).
__device__ int32_t g_int8_status;

struct GemmParams {
    CUtensorMap tmap_x;    // int8 [M][K], boxes of 128 bytes
    CUtensorMap tmap_w;    // int8 [N][K]
    CUtensorMap tmap_out;  // 16-bit [M][N], box 32 x 128 bytes (pair kernel, tma_out)
    const float* x_scales;
    const float* w_scales;
    const uint16_t* bias;  // [N] or null
    uint16_t* out;
    int64_t out_rs;
    int M, N, K, act;
    int tma_out;  // out rows start on 16 bytes: TMA stores
    int tiles_m, tiles_n;
    int tile0, tiles;  // pair kernel: of these tiles [tile0, tiles)
    int turn;          // pair kernel: 1 or 2 of two launches that share the tiles, else 0
    int early_weights;  // the first weights are fetched before grid_wait
    // Cycles that a barrier wait may take (0: the products give up half-way), and that
    // copies and products under way may take to end after a wait ran out.
    long long timeout, drain;
};

// Until what arrives on `bar` has ended, whoever has given up.
__device__ __forceinline__ void bar_drain(uint64_t* bar, uint32_t parity, long long limit) {
    const long long t0 = clock64();
    while (!mbar_try_wait_cluster(bar, parity) && clock64() - t0 <= limit) {
    }
}

// Up to 128 tokens x 128 channels per CTA, the weights as the product's first
// operand: its 128 rows are then always full, the tokens' side is as narrow as there
// are tokens (BT), and the weights' bytes, which bound it, pass shared memory once.
// The CTAs of a cluster split K and exchange their 32-bit sums through distributed
// shared memory.  A thread holds one channel and half of the tokens, so a warp's
// stores of a token are 64 contiguous bytes.
template <int BT>
struct TileCfg {
    static constexpr int BC = 128, BK = 128;
    static constexpr int W_BYTES = BC * BK, X_BYTES = BT * BK, STAGE = W_BYTES + X_BYTES;
    // Copies take over a microsecond: a CTA that has an SM to itself keeps twice the
    // bytes in flight of one that shares it.
    static constexpr int STAGES = 104 * 1024 / STAGE, STAGES_ALONE = 208 * 1024 / STAGE;
    static constexpr int PITCH = BC;                   // words between tokens' partial sums
    static constexpr int HALF = BT / 2;                // tokens per warp in the epilogue: two warps share a channel
    static constexpr int TMEM_COLS = BT < 64 ? 64 : BT;  // loads of 32 columns from the second half on stay inside
    struct Ctl {
        uint64_t full[STAGES_ALONE], empty[STAGES_ALONE], done, drained;
        uint32_t tmem_base;
        int abort;   // a wait of this CTA ran out
        int failed;  // a CTA of the cluster has no sums to give
        float scales[BT + 8];  // factors of the tokens, read eight at a time
    };
    static constexpr int smem(int stages) { return stages * STAGE + (int)((sizeof(Ctl) + 15) / 16 * 16); }
    static_assert((BT + 8) * PITCH * 4 <= STAGES * STAGE, "partial sums reuse the stages");
    static_assert(STAGES_ALONE * STAGE + (int)sizeof(Ctl) + 16 <= 227 * 1024, "shared memory of one CTA");
};

template <bool BF16, int BT>
__global__ void __launch_bounds__(256, 2) k_int8_tile(const __grid_constant__ GemmParams p, int split, int stages) {
    using C = TileCfg<BT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    auto* ctl = reinterpret_cast<typename C::Ctl*>(smem + stages * C::STAGE);
    constexpr int U = 8;  // tokens finished together
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % split;
    const int n0 = blockIdx.x / split * C::BC, m0 = blockIdx.y * BT;
    const int nkb = (p.K + C::BK - 1) / C::BK;
    const int kb0 = (int)((int64_t)nkb * rank / split), kb1 = (int)((int64_t)nkb * (rank + 1) / split);

    if (smem_u32(smem) & 1023) {  // uniform over the cluster
        if (threadIdx.x == 0) atomicOr(&g_int8_status, HB_DEV_SMEM_ALIGN);
        return;
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&p.tmap_x);
        prefetch_tmap(&p.tmap_w);
        for (int i = 0; i < stages; i++) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 1);
        }
        mbar_init(&ctl->done, 1);
        mbar_init(&ctl->drained, 1);
        ctl->abort = ctl->failed = 0;
        fence_barrier_init();
        if (p.early_weights) {
            for (int s = 0; s < min(stages, kb1 - kb0); s++) {
                mbar_arrive_expect_tx(&ctl->full[s], C::STAGE);
                tma_load_2d(smem + s * C::STAGE, &p.tmap_w, &ctl->full[s], (kb0 + s) * C::BK, n0);
            }
        }
    }
    if (warp == 2) {
        tmem_alloc(&ctl->tmem_base, C::TMEM_COLS);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncwarp();
    grid_wait();
    const int channel = threadIdx.x & 127, n = n0 + channel;  // this thread's channel
    const int t0 = (warp >> 2) * C::HALF;                     // and the first of its tokens
    const float sw = n < p.N ? w_factor(p.w_scales[n]) : 0.f, bias = n < p.N && p.bias ? load16<BF16>(p.bias + n) : 0.f;
    if (threadIdx.x < BT) ctl->scales[threadIdx.x] = m0 + (int)threadIdx.x < p.M ? x_factor(p.x_scales[m0 + threadIdx.x]) : 0.f;
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    int issued = 0;  // stages filled by the first thread
    if (warp == 0 && lane == 0) {
        int s = 0, round = 0;
        for (int kb = kb0; kb < kb1; kb++, issued++) {
            if (round > 0 && !mbar_wait(&ctl->empty[s], (round - 1) & 1, abort_flag, p.timeout)) break;
            uint8_t* st = smem + s * C::STAGE;
            if (round > 0 || !p.early_weights) {
                mbar_arrive_expect_tx(&ctl->full[s], C::STAGE);
                tma_load_2d(st, &p.tmap_w, &ctl->full[s], kb * C::BK, n0);
            }
            tma_load_2d(st + C::W_BYTES, &p.tmap_x, &ctl->full[s], kb * C::BK, m0);
            if (++s == stages) s = 0, round++;
        }
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = idesc_i8(C::BC, BT);
        const int end = p.timeout > 0 ? kb1 : (kb0 + kb1) / 2;
        bool ok = end == kb1;
        if (!ok) *abort_flag = 1;
        int s = 0, round = 0;
        for (int kb = kb0; kb < end; kb++) {
            if (!mbar_wait(&ctl->full[s], round & 1, abort_flag, p.timeout)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t w = smem_u32(smem + s * C::STAGE), x = w + C::W_BYTES;
#pragma unroll
            for (int k = 0; k < C::BK; k += 32)
                mma_i8_ss(tmem, desc_sw128(w + k, 16, 1024), desc_sw128(x + k, 16, 1024), idesc, kb > kb0 || k > 0);
            tc_commit(&ctl->empty[s]);
            if (++s == stages) s = 0, round++;
        }
        if (ok) tc_commit(&ctl->done);
    }
    __syncwarp();
    // done: every product has been formed, so every copy has landed.
    bool ok = __all_sync(FULL, mbar_wait(&ctl->done, 0, abort_flag, p.timeout));
    if (!ok) {  // whichever wait ran out: nothing may be under way when the CTA gives up its memory
        if (lane == 0) atomicOr(&g_int8_status, HB_DEV_TIMEOUT);
        if (threadIdx.x == 0) {
            for (int j = max(0, issued - stages); j < issued; j++) bar_drain(&ctl->full[j % stages], (j / stages) & 1, p.drain);
        } else if (threadIdx.x == 32) {
            tc_commit(&ctl->drained);
            bar_drain(&ctl->drained, 0, p.drain);
        }
        __syncwarp();
    }
    // Finishes U tokens from j on: straight-line code, so that their latencies overlap.
    auto finish_tokens = [&](int j, int end, const int (&acc)[U]) {
        float y[U];
#pragma unroll
        for (int i = 0; i < U; i++) y[i] = finish<0>(acc[i], ctl->scales[j + i], sw, bias);
        if (p.act) {
#pragma unroll
            for (int i = 0; i < U; i++) y[i] = gelu_tanh(y[i]);
        }
        if (n >= p.N) return;
        uint16_t* dst = p.out + (int64_t)(m0 + j) * p.out_rs + n;
#pragma unroll
        for (int i = 0; i < U; i++)
            if (j + i < end) dst[i * p.out_rs] = (uint16_t)pack2<BF16>(y[i], 0.f);
    };
    const int tokens = min(BT, p.M - m0);
    const uint32_t acc0 = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + t0;
    if (split == 1) {
        if (ok) {
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < C::HALF; c += 32) {
                uint32_t r[32];
                tmem_ld32(acc0 + c, r);
#pragma unroll
                for (int i = 0; i < (C::HALF < 32 ? C::HALF : 32); i += U) {
                    int acc[U];
#pragma unroll
                    for (int e = 0; e < U; e++) acc[e] = (int)r[i + e];
                    if (t0 + c + i < tokens) finish_tokens(t0 + c + i, tokens, acc);
                }
            }
            tc_fence_before();
        }
        __syncthreads();
        if (warp == 2) {
            tc_fence_after();
            tmem_dealloc(tmem, C::TMEM_COLS);
        }
        return;
    }
    // Every CTA of the cluster sends each peer the sums of that peer's share of the
    // tokens ([source][token][channel], in the stages, which every MMA has read by
    // the first barrier) and adds up its own share.
    const int log_share = __ffs(BT) - __ffs(split), share = 1 << log_share;  // both powers of two
    int* part = reinterpret_cast<int*>(smem);
    const uint32_t mine = smem_u32(part + rank * share * C::PITCH + channel);
    ok = __syncthreads_and(ok);
    cluster_sync();  // every CTA arrives at both barriers, whatever happened before
    if (!ok && threadIdx.x < split) st_cluster_s32(cluster_map(smem_u32(&ctl->failed), threadIdx.x), 1);
    if (ok) {
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::HALF; c += 32) {
            uint32_t r[32];
            tmem_ld32(acc0 + c, r);
#pragma unroll
            for (int i = 0; i < (C::HALF < 32 ? C::HALF : 32); i++) {
                const int j = t0 + c + i;
                const uint32_t at = mine + (j & (share - 1)) * (C::PITCH * 4);
                st_cluster_s32(cluster_map(at, j >> log_share), (int)r[i]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
    if (*static_cast<volatile int*>(&ctl->failed)) return;  // a share of the sums is missing
    for (int j = U * (warp >> 2); j < share && rank * share + j < tokens; j += 2 * U) {
        int acc[U] = {};
        for (int q = 0; q < split; q++) {
#pragma unroll
            for (int i = 0; i < U; i++)
                if (j + i < share) acc[i] += part[(q * share + j + i) * C::PITCH + channel];
        }
        finish_tokens(rank * share + j, min(tokens, (rank + 1) * share), acc);
    }
}

// 256 x 256 output tiles by CTA pairs, persistent.  One MMA of a pair covers 256
// x 256 x 32: each CTA stages 128 rows of both operands, so a CTA reads half of
// the weight tile's bytes that it would need alone, and both keep 128 rows of the
// accumulator.  Two accumulators fill the TMEM: the epilogue of a tile runs under
// the products of the next.  With SPLIT 2 or 4 that many pairs, one cluster, share the K
// of one tile and exchange their sums (one tile each, for products of few tiles).
struct PairCfg {
    static constexpr int BM = 256, BN = 256, BK = 128;
    static constexpr int A_BYTES = 128 * BK, B_BYTES = 128 * BK, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 6;
    static constexpr int EPI_WARPS = 8;         // two per TMEM lane quarter, half of the columns each
    static constexpr int STAGING = 32 * 128;    // per warp: 32 rows x 64 columns of the output
    static constexpr int THREADS = 128 + 32 * EPI_WARPS;
    struct Ctl {
        uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drained;
        uint32_t tmem_base;
        int abort;      // a wait of this CTA ran out
        int failed;     // some CTA of the cluster did not see all of its sums
        int issued[2];  // in the pair's first CTA: stages that each of the two filled before it gave up
        alignas(16) float col_scale[BN];  // factors of the tile's columns
        alignas(16) float col_bias[BN];
    };
    static constexpr int STG_OFF = STAGES * STAGE;
    static constexpr int CTL_OFF = STG_OFF + EPI_WARPS * STAGING;
    static constexpr int SMEM = CTL_OFF + (int)((sizeof(Ctl) + 15) / 16 * 16);
    static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
    static_assert(3 * EPI_WARPS * 32 * 64 * 4 <= STAGES * STAGE, "sums of three other pairs reuse the stages");
    // Tiles are walked down columns of GROUP row tiles, so the tiles in flight at
    // one time share few rows of both operands (both stay in L2).
    static constexpr int GROUP = 8;
};

__device__ __forceinline__ void pair_tile(const GemmParams& p, int t, int& m0, int& n0) {
    const int per = PairCfg::GROUP * p.tiles_n;
    const int g = t / per, r = t - g * per;
    const int gm = min(PairCfg::GROUP, p.tiles_m - g * PairCfg::GROUP);
    m0 = (g * PairCfg::GROUP + r % gm) * PairCfg::BM;
    n0 = r / gm * PairCfg::BN;
}

template <bool BF16, int ACT, int SPLIT>
__global__ void __cluster_dims__(2 * SPLIT, 1, 1) __launch_bounds__(PairCfg::THREADS, 1)
    k_int8_pair(const __grid_constant__ GemmParams p) {
    using C = PairCfg;
    extern __shared__ __align__(1024) uint8_t smem[];
    auto* ctl = reinterpret_cast<C::Ctl*>(smem + C::CTL_OFF);
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = (int)cluster_rank(), rank = cta & 1, lead = cta & ~1;  // in the cluster, in the pair, the pair's first
    const int part = cta >> 1;                                            // of K
    const int first = p.tile0 + blockIdx.x / (2 * SPLIT), step = gridDim.x / (2 * SPLIT), tiles = p.tiles;
    const int blocks = (p.K + C::BK - 1) / C::BK;
    const int kb0 = blocks * part / SPLIT, nkb = blocks * (part + 1) / SPLIT - kb0;

    if (smem_u32(smem) & 1023) {  // the same in both CTAs
        if (threadIdx.x == 0) atomicOr(&g_int8_status, HB_DEV_SMEM_ALIGN);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&ctl->acc_full[i], 1);
            mbar_init(&ctl->acc_empty[i], 2 * C::EPI_WARPS);
        }
        mbar_init(&ctl->drained, 1);
        ctl->abort = ctl->failed = 0;
        ctl->issued[0] = ctl->issued[1] = INT_MAX;
        fence_barrier_init();
        prefetch_tmap(&p.tmap_x);
        prefetch_tmap(&p.tmap_w);
        if (p.tma_out) prefetch_tmap(&p.tmap_out);
    }
    if (warp == 2) {
        tmem_alloc_pair(&ctl->tmem_base, 512);
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int early = 0;
            if (p.early_weights) {
                int m0, n0;
                pair_tile(p, first, m0, n0);
                early = min(C::STAGES, nkb);  // blocks of the first tile
                for (int s = 0; s < early; s++) {
                    if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], 2 * C::STAGE);
                    tma_load_2d_pair(smem + s * C::STAGE + C::A_BYTES, &p.tmap_w, cluster_map(smem_u32(&ctl->full[s]), lead),
                                     (kb0 + s) * C::BK, n0 + 128 * rank);
                }
            }
            // The second launch reads what the first has waited for, and starts on every
            // SM that the first has left; its other warps wait for all of the first.
            if (p.turn != 2) grid_wait();
            if (p.turn == 1) grid_launch_dependents();
            int it = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                int m0, n0;
                pair_tile(p, t, m0, n0);
                for (int kb = 0; kb < nkb; kb++, it++) {
                    const int s = it % C::STAGES;
                    if (it >= C::STAGES &&
                        !mbar_wait_cluster(&ctl->empty[s], (it / C::STAGES - 1) & 1, abort_flag, p.timeout)) {
                        ok = false;
                        break;
                    }
                    uint8_t* st = smem + s * C::STAGE;
                    if (rank == 0 && it >= early) mbar_arrive_expect_tx(&ctl->full[s], 2 * C::STAGE);
                    const uint32_t bar = cluster_map(smem_u32(&ctl->full[s]), lead);
                    const int k = (kb0 + kb) * C::BK;
                    tma_load_2d_pair(st, &p.tmap_x, bar, k, m0 + 128 * rank);
                    if (it >= early) tma_load_2d_pair(st + C::A_BYTES, &p.tmap_w, bar, k, n0 + 128 * rank);
                }
            }
            if (!ok) st_cluster_s32(cluster_map(smem_u32(&ctl->issued[rank]), lead), it);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = idesc_i8(C::BM, C::BN);
            if (p.turn != 2) grid_wait();  // the clock of the waits starts when the copies can
            const int end = p.timeout > 0 ? nkb : nkb / 2;
            if (end < nkb) *abort_flag = 1;
            int it = 0, i = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step, i++) {
                const uint32_t d = tmem + (i & 1) * C::BN;
                if (i >= 2 && !mbar_wait_cluster(&ctl->acc_empty[i & 1], (i / 2 - 1) & 1, abort_flag, p.timeout)) break;
                tc_fence_after();
                for (int kb = 0; kb < end; kb++, it++) {
                    const int s = it % C::STAGES;
                    if (!mbar_wait_cluster(&ctl->full[s], (it / C::STAGES) & 1, abort_flag, p.timeout)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + C::A_BYTES;
#pragma unroll
                    for (int k = 0; k < C::BK; k += 32)
                        mma_i8_ss_pair(d, desc_sw128(a + k, 16, 1024), desc_sw128(b + k, 16, 1024), idesc, kb > 0 || k > 0);
                    tc_commit_pair(&ctl->empty[s], 3 << lead);
                }
                ok = ok && end == nkb;
                if (ok) tc_commit_pair(&ctl->acc_full[i & 1], 3 << lead);
            }
        }
    } else if (warp >= 4) {
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;
        uint8_t* stg = smem + C::STG_OFF + ew * C::STAGING;
        grid_wait();
        float *col_scale = ctl->col_scale + 128 * half, *col_bias = ctl->col_bias + 128 * half;
        int i = 0;
        bool dead = false;  // a wait ran out: only the barriers of the remaining tiles are kept, so that no warp is left at one
        for (int t = first; t < tiles; t += step, i++) {
            int m0, n0;
            pair_tile(p, t, m0, n0);
            const int row0 = m0 + 128 * rank + 32 * quarter, col0 = n0 + 128 * half;
            {  // this half's column scales and biases (its four warps only)
                const int c = threadIdx.x & 127;
                float scale = 0.f, bias = 0.f;
                if (col0 + c < p.N) {
                    scale = w_factor(p.w_scales[col0 + c]);
                    if (p.bias) bias = load16<BF16>(p.bias + col0 + c);
                }
                asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
                col_scale[c] = scale;
                col_bias[c] = bias;
                asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
            }
            if (dead) continue;
            const float row_scale = row0 + lane < p.M ? x_factor(p.x_scales[row0 + lane]) : 0.f;
            const uint64_t sx = f2_pack(row_scale, row_scale);
            // 64 columns of the warp's 32 rows from column c of its half: finished, staged, stored.
            auto finish_columns = [&](int c, const uint32_t (&lo)[32], const uint32_t (&hi)[32]) {
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {  // four columns
                        const int x = 8 * j + 2 * e;
                        const ulonglong2 sw = *reinterpret_cast<const ulonglong2*>(col_scale + c + x);
                        const ulonglong2 sb = *reinterpret_cast<const ulonglong2*>(col_bias + c + x);
                        const uint32_t(&r)[32] = x < 32 ? lo : hi;
                        o[e] = finish2<BF16, ACT>((int)r[x & 31], (int)r[(x + 1) & 31], sx, sw.x, sb.x);
                        o[e + 1] = finish2<BF16, ACT>((int)r[(x + 2) & 31], (int)r[(x + 3) & 31], sx, sw.y, sb.y);
                    }
                    // 128-byte rows with the map's swizzle: conflict-free 16-byte stores
                    *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
                if (p.tma_out) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0 && row0 < p.M && col0 + c < p.N) {
                        tma_store_2d(&p.tmap_out, stg, col0 + c, row0);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    // a lane per column and the next but 31, eight rows' values at a time
                    uint16_t* dst = p.out + (int64_t)row0 * p.out_rs + col0 + c + lane;
                    const bool in0 = col0 + c + lane < p.N, in1 = col0 + c + lane + 32 < p.N;
                    for (int r = 0; r < 32 && row0 + r < p.M; r += 8, dst += 8 * p.out_rs) {
                        uint16_t v[16];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint8_t* line = stg + (r + e) * 128 + (lane & 7) * 2;
                            v[2 * e] = *reinterpret_cast<const uint16_t*>(line + (((lane >> 3) ^ e) << 4));
                            v[2 * e + 1] = *reinterpret_cast<const uint16_t*>(line + ((((lane >> 3) + 4) ^ e) << 4));
                        }
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            if (row0 + r + e < p.M) {
                                if (in0) dst[e * p.out_rs] = v[2 * e];
                                if (in1) dst[e * p.out_rs + 32] = v[2 * e + 1];
                            }
                        }
                    }
                    __syncwarp();
                }
            };
            const bool ok = __all_sync(FULL, mbar_wait_cluster(&ctl->acc_full[i & 1], (i >> 1) & 1, abort_flag, p.timeout));
            if (!ok) {
                if (lane == 0) atomicOr(&g_int8_status, HB_DEV_TIMEOUT);
                if (lane < 2 * SPLIT) st_cluster_s32(cluster_map(smem_u32(&ctl->failed), lane), 1);
                dead = true;
            }
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(32 * quarter) << 16) + (i & 1) * C::BN + 128 * half;
            uint32_t lo[32], hi[32];
            auto read = [&](int c) {
                tmem_ld32_async(acc + c, lo);
                tmem_ld32_async(acc + c + 32, hi);
                tmem_wait_ld(lo);
                tmem_wait_ld(hi);
            };
            if constexpr (SPLIT == 1) {
                if (dead) continue;
#pragma unroll
                for (int c = 0; c < 128; c += 64) {
                    read(c);
                    if (c == 64) {  // the accumulator is in registers: the next tile but one may take its place
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(cluster_map(smem_u32(&ctl->acc_empty[i & 1]), lead));
                    }
                    finish_columns(c, lo, hi);
                }
            } else {
                // Every 64 columns have an owner among the pairs, to whom the others send
                // their sums ([source][warp][column / 4][row][4], in the stages, which every
                // MMA has read by the first barrier).  Every thread of the cluster arrives at
                // both barriers, whatever happened before.
                const uint32_t at = smem_u32(smem) + (ew * 16 * 32 + lane) * 16;
                __syncwarp();
                cluster_sync();
                if (*static_cast<volatile int*>(&ctl->failed)) dead = true;  // sums will be missing
#pragma unroll
                for (int c = 0; c < 128; c += 64) {
                    const int owner = (2 * half + c / 64) & (SPLIT - 1);
                    if (dead || owner == part) continue;
                    read(c);
                    const uint32_t slot = (part - owner - 1) & (SPLIT - 1);
                    const uint32_t to = cluster_map(at + slot * (C::EPI_WARPS * 16 * 32 * 16), 2 * owner + rank);
#pragma unroll
                    for (int v = 0; v < 32; v += 4) {
                        st_cluster_v4(to + v / 4 * 512, lo[v], lo[v + 1], lo[v + 2], lo[v + 3]);
                        st_cluster_v4(to + (v / 4 + 8) * 512, hi[v], hi[v + 1], hi[v + 2], hi[v + 3]);
                    }
                }
                __syncwarp();
                cluster_sync();
                if (!dead && (SPLIT == 2 || half == part >> 1)) {  // this warp's columns of the owned ones
                    const int c = 64 * (part & 1);
                    read(c);
                    for (int slot = 0; slot < SPLIT - 1; slot++) {
                        const uint4* from = reinterpret_cast<const uint4*>(smem) + (slot * C::EPI_WARPS + ew) * 16 * 32 + lane;
#pragma unroll
                        for (int v = 0; v < 32; v += 4) {
                            const uint4 a = from[v / 4 * 32], b = from[(v / 4 + 8) * 32];
                            lo[v] += a.x, lo[v + 1] += a.y, lo[v + 2] += a.z, lo[v + 3] += a.w;
                            hi[v] += b.x, hi[v + 1] += b.y, hi[v + 2] += b.z, hi[v + 3] += b.w;
                        }
                    }
                    finish_columns(c, lo, hi);
                }
            }
        }
        if (lane == 0) bulk_wait<0>();
    }
    __syncwarp();
    if (SPLIT > 1 && warp < 4) {  // the two barriers of the exchange
        cluster_sync();
        cluster_sync();
    }
    __syncthreads();
    cluster_sync();  // no CTA leaves while the other's MMAs read its memory or arrivals are on the way
    if (*static_cast<volatile int*>(&ctl->failed)) {  // the same in all CTAs: copies and MMAs may be under way
        if (rank == 0 && threadIdx.x == 0) {
            // Both CTAs' copies arrive here, STAGE bytes each.  The two may have given up a
            // few stages apart: what only one has filled is completed for the other.
            const int all = (tiles - first + step - 1) / step * nkb;
            const int mine = min(ctl->issued[0], all), other = min(ctl->issued[1], all), most = max(mine, other);
            for (int j = max(0, most - C::STAGES); j < most; j++) {
                uint64_t* bar = &ctl->full[j % C::STAGES];
                if (j >= mine) mbar_arrive_expect_tx(bar, C::STAGE);
                if (j >= other) mbar_complete_tx(bar, C::STAGE);
                bar_drain(bar, (j / C::STAGES) & 1, p.drain);
            }
        } else if (rank == 0 && threadIdx.x == 32) {
            tc_commit_pair(&ctl->drained, 1 << lead);
            bar_drain(&ctl->drained, 0, p.drain);
        }
        __syncwarp();
        cluster_sync();
    }
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    });
    return fn;
}

// [rows][cols] matrix of `type` (elements of `size` bytes, row stride rs bytes)
// as a 2-D map with 128-byte swizzle and a box of 128 bytes x box_rows.
int make_tmap_2d(CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, int64_t rows, int64_t cols,
                 int64_t rs, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return HB_ERR_CUDA;
    if (rows == 1) rs = (cols * size + 15) / 16 * 16;  // never used for addressing
    cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t gstride[1] = {(cuuint64_t)rs};
    cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, estride[2] = {1, 1};
    const CUresult r = enc(map, type, 2, const_cast<void*>(base), gdim, gstride, box, estride,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? HB_OK : HB_ERR_TMA;
}

constexpr int kWaitMs = 2000;
std::atomic<int> g_wait_ms{kWaitMs};  // hb_int8_set_wait_limit

std::mutex g_mu;
unsigned g_configured[64];  // per device: kernels whose shared-memory limit is set

template <class Kernel>
int configure(Kernel kern, int dev, int slot, int smem) {
    std::lock_guard<std::mutex> lk(g_mu);
    if (!(g_configured[dev] >> slot & 1u)) {
        HB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        g_configured[dev] |= 1u << slot;
    }
    return HB_OK;
}

// Clusters of 1, 2, 4 and 8 CTAs, one CTA per SM, that can be resident at once: not all
// SMs' worth, since a cluster lies within one of the device's groups of SMs, and those
// differ in size.
struct Fit {
    int clusters[4];
};

template <class Kernel>
int max_clusters(Kernel kern, int size, int* n) {
    HB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(PairCfg::THREADS);
    cfg.dynamicSmemBytes = PairCfg::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HB_CUDA_TRY(cudaOccupancyMaxActiveClusters(n, kern, &cfg));
    return HB_OK;
}
int cluster_fit(int dev, int sms, Fit* fit) {
    static Fit known[64];
    static bool asked[64];
    std::lock_guard<std::mutex> lk(g_mu);
    if (!asked[dev]) {
        int rc;
        int* n = known[dev].clusters;
        n[0] = sms;
        if ((rc = max_clusters(k_int8_pair<true, 0, 1>, 2, n + 1))) return rc;
        if ((rc = max_clusters(k_int8_pair<true, 0, 2>, 4, n + 2))) return rc;
        if ((rc = max_clusters(k_int8_pair<true, 0, 4>, 8, n + 3))) return rc;
        asked[dev] = true;
    }
    *fit = known[dev];
    return HB_OK;
}

// CTAs that split K: doubled while one round of their clusters holds every tile, with
// two blocks of K at least; a second round of a few clusters costs as much as the first
// (96 x 2048, K 8192: 10.5 us with 4 CTAs for K, 18.3 us with 8 on 128 SMs).
int tile_split(const GemmParams& p, int bt, const Fit& fit) {
    const int64_t tiles = ceil_div(p.N, 128) * ceil_div(p.M, bt), nkb = ceil_div(p.K, 128);
    int log = 0;
    while (log < 3 && tiles <= fit.clusters[log + 1] && nkb >= 4 << log) log++;
    return 1 << log;
}

template <bool BF16, int BT>
int launch_tile(const Int8Problem& q, GemmParams& p, const Fit& fit, int dev, cudaStream_t st) {
    using C = TileCfg<BT>;
    auto kern = k_int8_tile<BF16, BT>;
    constexpr int slot = 16 + BF16 * 4 + (BT == 16 ? 0 : BT == 32 ? 1 : BT == 64 ? 2 : 3);
    int rc;
    if ((rc = configure(kern, dev, slot, C::smem(C::STAGES_ALONE)))) return rc;
    if ((rc = make_tmap_2d(&p.tmap_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.x, p.M, p.K, q.x_rs, BT))) return rc;
    if ((rc = make_tmap_2d(&p.tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w, p.N, p.K, q.w_rs, C::BC))) return rc;
    const int64_t tn = ceil_div(p.N, C::BC), tm = ceil_div(p.M, BT);
    const int split = tile_split(p, BT, fit);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tn * split), (unsigned)tm);
    cfg.blockDim = dim3(256);
    const int stages = tn * tm * split <= fit.clusters[0] ? C::STAGES_ALONE : C::STAGES;
    cfg.dynamicSmemBytes = C::smem(stages);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 2 : 1;
    HB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, split, stages));
    return HB_OK;
}

// Tiles [p.tile0, p.tiles) by SPLIT pairs each.
template <bool BF16, int ACT, int SPLIT>
int launch_pair(GemmParams& p, const Fit& fit, int dev, cudaStream_t st) {
    using C = PairCfg;
    auto kern = k_int8_pair<BF16, ACT, SPLIT>;
    const int clusters = fit.clusters[SPLIT == 4 ? 3 : SPLIT], tiles = p.tiles - p.tile0;
    if (clusters <= 0) return HB_ERR_UNSUPPORTED;
    int rc;
    if ((rc = configure(kern, dev, (SPLIT / 2 * 2 + BF16) * 2 + ACT, C::SMEM))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * SPLIT * (unsigned)(SPLIT > 1 ? tiles : std::min(tiles, clusters)));  // split: one tile each
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return HB_OK;
}
template <bool BF16>
int launch_pair(GemmParams& p, int split, const Fit& fit, int dev, cudaStream_t st) {
    if (split == 4) return p.act ? launch_pair<BF16, 1, 4>(p, fit, dev, st) : launch_pair<BF16, 0, 4>(p, fit, dev, st);
    if (split == 2) return p.act ? launch_pair<BF16, 1, 2>(p, fit, dev, st) : launch_pair<BF16, 0, 2>(p, fit, dev, st);
    return p.act ? launch_pair<BF16, 1, 1>(p, fit, dev, st) : launch_pair<BF16, 0, 1>(p, fit, dev, st);
}
// All tiles: the first `whole` by a pair each, the others by `split`.
template <bool BF16>
int launch_pairs(const Int8Problem& q, GemmParams& p, int whole, int split, const Fit& fit, int dev, cudaStream_t st) {
    int rc;
    if ((rc = make_tmap_2d(&p.tmap_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.x, p.M, p.K, q.x_rs, 128))) return rc;
    if ((rc = make_tmap_2d(&p.tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w, p.N, p.K, q.w_rs, 128))) return rc;
    if (p.tma_out &&
        (rc = make_tmap_2d(&p.tmap_out, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p.out,
                           p.M, p.N, p.out_rs * 2, 32)))
        return rc;
    const int tiles = p.tiles_m * p.tiles_n;
    p.tile0 = 0;
    p.tiles = whole;
    p.turn = whole > 0 && whole < tiles;
    if (whole > 0 && (rc = launch_pair<BF16>(p, 1, fit, dev, st))) return rc;
    p.tile0 = whole;
    p.tiles = tiles;
    if (p.turn) p.turn = 2, p.early_weights = 0;
    return whole < tiles ? launch_pair<BF16>(p, split, fit, dev, st) : HB_OK;
}

// Expected times in hundredths of a microsecond, from 70 shapes (65 to 4096 tokens, 640
// to 12288 channels, K 256 to 12288) timed with every kernel.  A k-block of 128 bytes
// takes a CTA (or a pair) about 0.28 us, two CTAs of an SM together 0.47 us; the fixed
// parts are the launch, the first copies and a tile's way out.  At the crossings: 768 x
// 3072, K 3072 12.5 us in tiles of 128 tokens and 13.7 us in pairs, 1024 tokens 15.5
// and 14.2 us; 512 x 3072 12.6 us in tiles of 64 and 12.2 us of 128, 192 tokens 9.1
// and 10.6 us.
int64_t tile_cost(const GemmParams& p, int bt, const Fit& fit) {
    const int64_t split = tile_split(p, bt, fit), sms = fit.clusters[0];
    const int64_t waves = ceil_div(ceil_div(p.N, 128) * ceil_div(p.M, bt) * split, sms), kb = ceil_div(ceil_div(p.K, 128), split);
    return (bt == 128 ? 550 : 430) + (split > 1 ? 100 : 0) + (waves - 1) * 130 + kb * (waves == 1 ? 28 : waves * 47 / 2);
}
// Pairs: whole rounds of tiles first, and what is left (or everything, if that is less
// than a round) with as many pairs for each tile's K as their clusters fit, if that pays:
// 512 x 4096, K 14336: 26.4 us with 2 pairs for K, 38.9 us with 1; 256 x 3072, K 12288:
// 17.6 us with 4, 22.4 us with 2, 34.1 us with 1; 1280 x 4096 (74 tiles and 6), K 14336:
// 58.7 us with 4 for the 6, 74.1 us with 1; K 4096: 28.6 and 26.8 us.
struct PairPlan {
    int64_t cost;
    int whole, split;
};
PairPlan plan_pairs(const GemmParams& p, const Fit& fit) {
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, nkb = ceil_div(p.K, 128), pairs = fit.clusters[1];
    const int64_t by_value = p.tma_out ? 0 : 250, round = nkb * 29 + by_value, left = tiles % pairs;
    PairPlan best = {700 + ceil_div(tiles, pairs) * round, (int)tiles, 1};
    for (int log = 1; log < 3 && nkb >= 4 << (log - 1); log++) {
        if (left > fit.clusters[log + 1]) break;
        const int64_t start = tiles < pairs ? 200 : log == 1 ? 700 : 880;  // the exchange, and of a second launch
        const int64_t cost = 700 + tiles / pairs * round + start + ceil_div(nkb, 1 << log) * 29 + by_value;
        if (left && cost < best.cost) best = {cost, (int)(tiles - left), 1 << log};
    }
    return best;
}

template <bool BF16>
int launch_gemm(const Int8Problem& q, GemmParams& p, const Fit& fit, int dev, cudaStream_t st) {
    if (p.M <= 16) return launch_tile<BF16, 16>(q, p, fit, dev, st);
    if (p.M <= 32) return launch_tile<BF16, 32>(q, p, fit, dev, st);
    const int64_t narrow = tile_cost(p, 64, fit), wide = tile_cost(p, 128, fit);
    if (p.M > 64 && fit.clusters[1] > 0) {
        const PairPlan plan = plan_pairs(p, fit);
        if (plan.cost < std::min(narrow, wide) || ceil_div(p.M, 64) > 65535)  // 65535: grid rows
            return launch_pairs<BF16>(q, p, plan.whole, plan.split, fit, dev, st);
    }
    if (p.M <= 64 || narrow <= wide) return launch_tile<BF16, 64>(q, p, fit, dev, st);
    return launch_tile<BF16, 128>(q, p, fit, dev, st);
}

}  // namespace

int launch_int8_gemm(const Int8Problem& q, int dev, const DeviceInfo& di, bool early_weights, cudaStream_t st) {
    GemmParams p;
    p.x_scales = q.x_scales;
    p.w_scales = q.w_scales;
    p.bias = q.bias;
    p.out = q.out;
    p.out_rs = q.out_rs;
    p.M = q.M;
    p.N = q.N;
    p.K = q.K;
    p.act = q.act;
    p.tiles_m = (int)ceil_div(p.M, PairCfg::BM);
    p.tiles_n = (int)ceil_div(p.N, PairCfg::BN);
    p.tma_out = aligned(p.out, 16) && (p.M == 1 || p.out_rs % 8 == 0);
    p.early_weights = early_weights;
    p.timeout = (long long)g_wait_ms.load(std::memory_order_relaxed) * di.clock_khz;
    p.drain = (long long)kWaitMs * di.clock_khz;
    Fit fit;
    if (const int rc = cluster_fit(dev, di.sms, &fit)) return rc;
    return q.dtype == 1 ? launch_gemm<true>(q, p, fit, dev, st) : launch_gemm<false>(q, p, fit, dev, st);
}

}  // namespace hb

using namespace hb;

extern "C" int hb_int8_set_wait_limit(int milliseconds) {
    if (milliseconds < 0) return HB_ERR_ARG;
    g_wait_ms.store(milliseconds, std::memory_order_relaxed);
    return HB_OK;
}

extern "C" int hb_int8_status(int clear, int32_t* bits, void* stream) {
    if (!bits) return HB_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    HB_CUDA_TRY(cudaMemcpyFromSymbolAsync(bits, g_int8_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, st));
    HB_CUDA_TRY(cudaStreamSynchronize(st));
    if (clear && *bits) {
        static const int32_t zero = 0;
        HB_CUDA_TRY(cudaMemcpyToSymbolAsync(g_int8_status, &zero, sizeof(int32_t), 0, cudaMemcpyHostToDevice, st));
        HB_CUDA_TRY(cudaStreamSynchronize(st));
    }
    return HB_OK;
}
