// Linear layers in 8-bit integers: rows of 16-bit values quantised with one scale
// a row, and the product of two such matrices with scales, bias and activation.
//
//   scale_m = max_k |x_mk| / 127            code_mk = rint(x_mk * (127 / max_k |x_mk|))
//   y_mn = act((sum_k xcode_mk * wcode_nk) * (xscale_m * wscale_n) + bias_n)
//
// The sum is exact in 32-bit integers (K <= 131072: 127^2 * K < 2^31), so the
// order in which it is taken, and how K is split over CTAs, cannot change a
// result; the rest is fp32, rounded once to the 16-bit output type.
//
// No counterpart in the reference (it runs the model's bf16 layers as they are);
// these serve the FLUX blocks' projections and MLPs (hilberta/flux_adapter.py:
// 280-340 calls the projections around the attention).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <mutex>

#include "common.cuh"
#include "int8_codes.cuh"
#include "sm100_ptx.cuh"

namespace hb {
namespace {

using namespace ptx;
constexpr unsigned FULL = 0xffffffffu;

// HB_DEV_* bits of the launches on this device (read by hb_int8_status).
__device__ int32_t g_int8_status;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
    if constexpr (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <bool BF16>
__device__ __forceinline__ float load16(const uint16_t* p) {
    return unpack2<BF16>(*p).x;
}

// Largest magnitude of a pair of 16-bit values as magnitude bits (NaN sorts
// above infinity above every number, so non-finite values are never lost).
__device__ __forceinline__ uint32_t max_mag(uint32_t m, uint32_t u) { return __vmaxu2(m, u & 0x7fff7fffu); }
template <bool BF16>
__device__ __forceinline__ float mag_value(uint32_t m) {
    const uint32_t v = max(m & 0xffffu, m >> 16);
    if constexpr (BF16) return __uint_as_float(v << 16);
    return load16<false>(reinterpret_cast<const uint16_t*>(&v));
}

// Codes of four 16-bit values, in order from the low byte.
template <bool BF16>
__device__ __forceinline__ uint32_t codes4(uint32_t u0, uint32_t u1, float inv) {
    const float2 f = unpack2<BF16>(u0), g = unpack2<BF16>(u1);
    return pack_codes(code_bits(f.x, inv), code_bits(f.y, inv), code_bits(g.x, inv), code_bits(g.y, inv));
}

// ---- row quantisation ---------------------------------------------------------

struct QuantParams {
    const uint16_t* a;  // [rows][ka], row stride a_rs (elements)
    const uint16_t* b;  // [rows][kb] or null: columns ka .. ka + kb of the row
    int64_t a_rs, b_rs;
    int ka, k;  // k = ka + kb
    int rows;
    int8_t* codes;  // [rows][k], row stride c_rs (bytes)
    int64_t c_rs;
    float* scales;  // [rows]
};

// Thread t of T's share i of a row: eight values, and where their codes go.  VEC
// (rows start on 16 bytes, ka and k are multiples of 8): neighbours, in one 16-byte
// load and one 8-byte store.  Otherwise every T-th value, so that a warp's 2-byte
// loads and 1-byte stores are contiguous.  Zeros past the end of the row.
template <bool VEC, int T>
__device__ __forceinline__ uint4 load8(const QuantParams& p, int64_t row, int t, int i) {
    if constexpr (VEC) {
        const int c = 8 * (t + i * T);
        if (c >= p.k || row >= p.rows) return make_uint4(0, 0, 0, 0);
        const uint16_t* src = c < p.ka ? p.a + row * p.a_rs + c : p.b + row * p.b_rs + (c - p.ka);
        return *reinterpret_cast<const uint4*>(src);
    } else {
        uint32_t w[8];
        const uint16_t *a = p.a + row * p.a_rs, *b = p.b + row * p.b_rs;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = 8 * i * T + e * T + t;
            const uint16_t* src = c < p.ka ? a + c : b + (c - p.ka);
            w[e] = 0;
            if (c < p.k && row < p.rows) w[e] = __ldg(src);
        }
        return make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
}
template <bool VEC, int T>
__device__ __forceinline__ void store8(const QuantParams& p, int64_t row, int t, int i, uint2 codes) {
    int8_t* out = p.codes + row * p.c_rs;
    if constexpr (VEC) {
        const int c = 8 * (t + i * T);
        if (c < p.k) *reinterpret_cast<uint2*>(out + c) = codes;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = 8 * i * T + e * T + t;
            if (c < p.k) out[c] = (int8_t)((e < 4 ? codes.x : codes.y) >> (8 * (e & 3)));
        }
    }
}

__device__ __forceinline__ uint32_t max_mag(uint32_t m, const uint4& v) {
    return max_mag(max_mag(max_mag(max_mag(m, v.x), v.y), v.z), v.w);
}
template <bool BF16>
__device__ __forceinline__ uint2 codes8(const uint4& v, const RowScale& s) {
    if (!s.live) return make_uint2(0, 0);
    return make_uint2(codes4<BF16>(v.x, v.y, s.inv), codes4<BF16>(v.z, v.w, s.inv));
}

// T threads per row (a warp, or the whole CTA), up to kQuantVec vectors of 8
// values each: the row is read once and stays in registers between its maximum
// and its codes.  Memory-bound (2 K bytes read, K written per row): CTAs are
// persistent and each thread fetches its part of the next row before it works on
// this one, so loads are in flight through the reduction and the stores.
constexpr int kQuantVec = 4;

template <bool BF16, bool VEC, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T) k_quantize_rows(const __grid_constant__ QuantParams p) {
    constexpr int CTA = T < 128 ? 128 : T;
    constexpr int RPC = CTA / T;
    constexpr int NV = kQuantVec;
    __shared__ uint32_t s_max[2][CTA / 32];
    const int t = threadIdx.x % T;
    const int64_t step = (int64_t)gridDim.x * RPC;
    int64_t row = (int64_t)blockIdx.x * RPC + threadIdx.x / T;
    uint4 next[NV];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < NV; i++) next[i] = load8<VEC, T>(p, r, t, i);
    };
    fetch(row);
    for (int parity = 0; row < p.rows; row += step, parity ^= 1) {  // the same for all threads of a row
        uint4 v[NV];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = next[i];
        fetch(row + step);
#pragma unroll
        for (int i = 0; i < NV; i++) m = max_mag(m, v[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(FULL, m, o));
        if constexpr (T > 32) {  // two sets of words: a row's are read while the next row's are written
            if ((threadIdx.x & 31) == 0) s_max[parity][threadIdx.x / 32] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < T / 32; w++) m = __vmaxu2(m, s_max[parity][w]);
        }
        const RowScale s = row_scale(mag_value<BF16>(m));
        if (t == 0) p.scales[row] = s.scale;
#pragma unroll
        for (int i = 0; i < NV; i++) store8<VEC, T>(p, row, t, i, codes8<BF16>(v[i], s));
    }
}

// Rows too long for a CTA's registers: one CTA per row, read twice.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(512) k_quantize_long(const __grid_constant__ QuantParams p) {
    __shared__ uint32_t s_max[16];
    const int64_t row = blockIdx.x;
    const int n = (p.k + 8 * 512 - 1) / (8 * 512);
    uint32_t m = 0;
#pragma unroll 4
    for (int i = 0; i < n; i++) m = max_mag(m, load8<VEC, 512>(p, row, threadIdx.x, i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(FULL, m, o));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; w++) m = __vmaxu2(m, s_max[w]);
    const RowScale s = row_scale(mag_value<BF16>(m));
    if (threadIdx.x == 0) p.scales[row] = s.scale;
#pragma unroll 4
    for (int i = 0; i < n; i++)
        store8<VEC, 512>(p, row, threadIdx.x, i, codes8<BF16>(load8<VEC, 512>(p, row, threadIdx.x, i), s));
}

template <bool BF16, bool VEC>
int launch_quantize(const QuantParams& p, int sms, cudaStream_t st) {
    // Threads per row: the fewest whose registers hold it (a warp up to 1024
    // columns); persistent CTAs, as many as fill the SMs' 2048 threads.
    const int64_t groups = p.k <= 8 * kQuantVec * 32 ? ceil_div(p.rows, 4) : p.rows;
    auto grid = [&](int cta) { return (unsigned)std::min<int64_t>(groups, (int64_t)sms * (2048 / cta)); };
    if (p.k <= 8 * kQuantVec * 32)
        k_quantize_rows<BF16, VEC, 32><<<grid(128), 128, 0, st>>>(p);
    else if (p.k <= 8 * kQuantVec * 128)
        k_quantize_rows<BF16, VEC, 128><<<grid(128), 128, 0, st>>>(p);
    else if (p.k <= 8 * kQuantVec * 256)
        k_quantize_rows<BF16, VEC, 256><<<grid(256), 256, 0, st>>>(p);
    else if (p.k <= 8 * kQuantVec * 512)
        k_quantize_rows<BF16, VEC, 512><<<grid(512), 512, 0, st>>>(p);
    else
        k_quantize_long<BF16, VEC><<<p.rows, 512, 0, st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}

// ---- product ------------------------------------------------------------------

struct LinearParams {
    CUtensorMap tmap_x;    // int8 [M][K], box 128 x 128 bytes
    CUtensorMap tmap_w;    // int8 [N][K]
    CUtensorMap tmap_out;  // 16-bit [M][N], box 32 x 128 bytes (pair kernel, tma_out)
    const float* x_scales;
    const float* w_scales;
    const uint16_t* bias;  // [N] or null
    uint16_t* out;
    int64_t out_rs;
    int M, N, K;
    int vec_out;  // 8-byte stores allowed
    int tma_out;  // out rows start on 16 bytes: TMA stores
    int tiles_m, tiles_n;
    long long timeout;
};

// tanh-GELU(v) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3), the
// exponential taken in base 2.
__device__ __forceinline__ float gelu_tanh(float v) {
    const float k0 = -2.f * 1.4426950408889634f * 0.7978845608028654f;
    const float e = ex2(v * fmaf(k0 * 0.044715f, v * v, k0));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return v * r;
}
template <int ACT>
__device__ __forceinline__ float finish(int acc, float sx, float sw, float b) {
    const float v = fmaf(__int2float_rn(acc) * sx, sw, b);
    return ACT ? gelu_tanh(v) : v;
}

// A few tokens: every weight is read once and takes part in M products, so the
// bytes of the weights bound it.  A warp forms R output channels at a time, each
// lane 16 bytes of every channel's row, with 4-way 8-bit dot products; the tokens'
// codes lie in shared memory, quantised there from 16 bits by each CTA (they are a
// few KB; the first weights are on their way meanwhile).  Sums and results are
// those of the tensor-core kernels, bit for bit.
struct FewParams {
    const void* x;  // 16-bit [M][K] (x_scales null) or int8 codes
    int64_t x_rs;   // elements
    const float* x_scales;
    const int8_t* w;
    int64_t w_rs;
    const float* w_scales;
    const uint16_t* bias;
    uint16_t* out;
    int64_t out_rs;
    int M, N, K, act;
};
constexpr int kFewRows = 8;
constexpr int kFewSmem = 64 * 1024;  // codes of the tokens, at most
inline int64_t few_bytes(int64_t M, int64_t K) { return M * ((K + 15) / 16 * 16); }
inline bool is_few(int64_t M, int64_t K) { return M <= kFewRows && few_bytes(M, K) <= kFewSmem; }

// 16 bytes of a row of codes, of which `left` (at least 1) are inside it.
__device__ __forceinline__ int4 load_codes(const int8_t* p, int left) {
    if (left >= 16) return __ldg(reinterpret_cast<const int4*>(p));
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < left; i++) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
    return make_int4(w[0], w[1], w[2], w[3]);
}

// M: the tokens rounded up to a power of two; rows from p.M on do not exist.
template <bool BF16, bool CODES, int M, int R>
__global__ void __launch_bounds__(256) k_int8_few(const __grid_constant__ FewParams p) {
    extern __shared__ __align__(16) int8_t s_codes[];  // [M][pitch]
    __shared__ uint32_t s_mag[M][8];
    __shared__ float s_scale[M];
    constexpr int U = R == 4 ? 2 : 4;  // 16-byte chunks of each channel in flight
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = (blockIdx.x * 8 + warp) * R;
    const int chunks = (p.K + 15) / 16, pitch = 16 * chunks;
    int4 w[U][R];
    auto fetch = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = c0 + 32 * u + lane;
#pragma unroll
            for (int r = 0; r < R; r++)
                w[u][r] = c < chunks && n0 + r < p.N ? load_codes(p.w + (n0 + r) * p.w_rs + 16 * c, p.K - 16 * c) : make_int4(0, 0, 0, 0);
        }
    };
    fetch(0);

    if constexpr (CODES) {
        for (int i = threadIdx.x; i < p.M * chunks; i += 256) {
            const int m = i / chunks, c = i - m * chunks;
            *reinterpret_cast<int4*>(s_codes + m * pitch + 16 * c) =
                load_codes(static_cast<const int8_t*>(p.x) + m * p.x_rs + 16 * c, p.K - 16 * c);
        }
        if (threadIdx.x < p.M) s_scale[threadIdx.x] = p.x_scales[threadIdx.x];
        __syncthreads();
    } else {
        const uint16_t* x = static_cast<const uint16_t*>(p.x);
        const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && p.x_rs % 8 == 0;
        // eight values of row m from column c, zeros past the end
        auto load8 = [&](int m, int c) {
            const uint16_t* src = x + m * p.x_rs + c;
            if (vec && c + 8 <= p.K) return *reinterpret_cast<const uint4*>(src);
            uint32_t e[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < p.K) e[i / 2] |= (uint32_t)src[i] << (16 * (i & 1));
            return make_uint4(e[0], e[1], e[2], e[3]);
        };
        uint32_t mag[M];
#pragma unroll
        for (int m = 0; m < M; m++) {
            mag[m] = 0;
            for (int c = 8 * threadIdx.x; c < p.K && m < p.M; c += 8 * 256) {
                const uint4 v = load8(m, c);
                mag[m] = max_mag(mag[m], v);
            }
        }
#pragma unroll
        for (int m = 0; m < M; m++) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mag[m] = __vmaxu2(mag[m], __shfl_xor_sync(FULL, mag[m], o));
            if (lane == 0) s_mag[m][warp] = mag[m];
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < M; m++) {
            uint32_t g = s_mag[m][0];
#pragma unroll
            for (int i = 1; i < 8; i++) g = __vmaxu2(g, s_mag[m][i]);
            const RowScale s = row_scale(mag_value<BF16>(g));
            if (threadIdx.x == 0) s_scale[m] = s.scale;
            for (int c = 8 * threadIdx.x; c < pitch && m < p.M; c += 8 * 256) {
                const uint4 v = load8(m, c);
                *reinterpret_cast<uint2*>(s_codes + m * pitch + c) = codes8<BF16>(v, s);
            }
        }
        __syncthreads();
    }

    int acc[R][M] = {};
    for (int c0 = 0; c0 < chunks; c0 += 32 * U) {
        if (c0 > 0) fetch(c0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = c0 + 32 * u + lane;
            if (c < chunks) {
#pragma unroll
                for (int m = 0; m < M; m++) {
                    if (m >= p.M) break;
                    const int4 x = *reinterpret_cast<const int4*>(s_codes + m * pitch + 16 * c);
#pragma unroll
                    for (int r = 0; r < R; r++)
                        acc[r][m] = __dp4a(w[u][r].w, x.w, __dp4a(w[u][r].z, x.z, __dp4a(w[u][r].y, x.y, __dp4a(w[u][r].x, x.x, acc[r][m]))));
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
        for (int m = 0; m < M; m++) {
            const int sum = __reduce_add_sync(FULL, acc[r][m]);
            if (lane == r * M + m && n0 + r < p.N && m < p.M) {
                const float ws = p.w_scales[n0 + r], b = p.bias ? load16<BF16>(p.bias + n0 + r) : 0.f;
                const float y = p.act ? finish<1>(sum, s_scale[m], ws, b) : finish<0>(sum, s_scale[m], ws, b);
                p.out[m * p.out_rs + n0 + r] = (uint16_t)pack2<BF16>(y, 0.f);
            }
        }
    }
}

// One 128 x 128 output tile per CTA; the CTAs of a cluster split K and add their
// 32-bit sums through distributed shared memory.
struct TileCfg {
    static constexpr int BM = 128, BN = 128, BK = 128;
    static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
    static constexpr int STAGES = 6;
    static constexpr int PITCH = BN + 4;  // 32-bit words: row writes of 16 bytes hit all banks
    struct Ctl {
        uint64_t full[STAGES], empty[STAGES], done;
        uint32_t tmem_base;
        int abort;
        float rows[BM];  // row scales of the tile
    };
    static constexpr int CTL_OFF = STAGES * (A_BYTES + B_BYTES);
    static constexpr int SMEM = CTL_OFF + (int)((sizeof(Ctl) + 15) / 16 * 16);
    static_assert(BM * PITCH * 4 <= CTL_OFF, "partial sums reuse the stages");
};

template <bool BF16, int ACT>
__global__ void __launch_bounds__(128) k_int8_tile(const __grid_constant__ LinearParams p, int split) {
    using C = TileCfg;
    extern __shared__ __align__(1024) uint8_t smem[];
    auto* ctl = reinterpret_cast<C::Ctl*>(smem + C::CTL_OFF);
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % split;
    const int n0 = (blockIdx.x / split) * C::BN, m0 = blockIdx.y * C::BM;
    const int nkb = (p.K + C::BK - 1) / C::BK;
    const int kb0 = (int)((int64_t)nkb * rank / split), kb1 = (int)((int64_t)nkb * (rank + 1) / split);

    if (smem_u32(smem) & 1023) {  // uniform over the cluster
        if (threadIdx.x == 0) atomicOr(&g_int8_status, HB_DEV_SMEM_ALIGN);
        return;
    }
    if (warp == 0 && lane == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 1);
        }
        mbar_init(&ctl->done, 1);
        ctl->abort = 0;
        fence_barrier_init();
        prefetch_tmap(&p.tmap_x);
        prefetch_tmap(&p.tmap_w);
    }
    ctl->rows[threadIdx.x] = m0 + (int)threadIdx.x < p.M ? p.x_scales[m0 + threadIdx.x] : 0.f;
    const int col = n0 + 4 * lane;  // this lane's output columns
    float sw[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool in = col + i < p.N;
        sw[i] = in ? p.w_scales[col + i] : 0.f;
        b[i] = in && p.bias ? load16<BF16>(p.bias + col + i) : 0.f;
    }
    if (warp == 2) {
        tmem_alloc(&ctl->tmem_base, C::BN);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0 && lane == 0) {
        int it = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; kb++, it++) {
            const int s = it % C::STAGES;
            if (it >= C::STAGES && !mbar_wait(&ctl->empty[s], (it / C::STAGES - 1) & 1, abort_flag, p.timeout)) {
                ok = false;
                break;
            }
            uint8_t* st = smem + s * (C::A_BYTES + C::B_BYTES);
            mbar_arrive_expect_tx(&ctl->full[s], C::A_BYTES + C::B_BYTES);
            tma_load_2d(st, &p.tmap_x, &ctl->full[s], kb * C::BK, m0);
            tma_load_2d(st + C::A_BYTES, &p.tmap_w, &ctl->full[s], kb * C::BK, n0);
        }
        if (!ok) {  // let the copies in flight land before the CTA gives up its memory
            volatile int ignore = 0;
            for (int j = max(0, it - C::STAGES); j < it; j++)
                mbar_wait(&ctl->full[j % C::STAGES], (j / C::STAGES) & 1, &ignore, p.timeout);
        }
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = idesc_i8(C::BM, C::BN);
        bool ok = true;
        int it = 0;
        for (int kb = kb0; kb < kb1; kb++, it++) {
            const int s = it % C::STAGES;
            if (!mbar_wait(&ctl->full[s], (it / C::STAGES) & 1, abort_flag, p.timeout)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t a = smem_u32(smem + s * (C::A_BYTES + C::B_BYTES)), b = a + C::A_BYTES;
#pragma unroll
            for (int k = 0; k < C::BK; k += 32)
                mma_i8_ss(tmem, desc_sw128(a + k, 16, 1024), desc_sw128(b + k, 16, 1024), idesc, it > 0 || k > 0);
            tc_commit(&ctl->empty[s]);
        }
        if (ok) tc_commit(&ctl->done);
    }
    __syncwarp();
    bool ok = mbar_wait(&ctl->done, 0, abort_flag, p.timeout);
    ok = __all_sync(FULL, ok);
    if (!ok && lane == 0) atomicOr(&g_int8_status, HB_DEV_TIMEOUT);
    int* part = reinterpret_cast<int*>(smem);
    if (ok) {  // every MMA has read its stage: the tiles' memory is free
        tc_fence_after();
        int* dst = part + threadIdx.x * C::PITCH;
#pragma unroll
        for (int c = 0; c < C::BN; c += 32) {
            uint32_t r[32];
            tmem_ld32(tmem + ((uint32_t)(warp * 32) << 16) + c, r);
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
        tc_fence_before();
    }
    ok = __syncthreads_and(ok);
    if (split > 1) cluster_sync();  // every CTA of the cluster arrives here, whatever happened before
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, C::BN);
    }
    // this CTA's share of the rows, one warp per row, four columns a lane
    const int r0 = C::BM * rank / split, r1 = C::BM * (rank + 1) / split;
    if (ok && col < p.N) {
#pragma unroll 4
        for (int r = r0 + warp; r < min(r1, p.M - m0); r += 4) {
            const int* src = part + r * C::PITCH + 4 * lane;
            int4 acc = *reinterpret_cast<const int4*>(src);
            for (int q = 1; q < split; q++) {
                const int4 v = ld_cluster_v4(cluster_map(smem_u32(src), (rank + q) % split));
                acc.x += v.x;
                acc.y += v.y;
                acc.z += v.z;
                acc.w += v.w;
            }
            const float sx = ctl->rows[r];
            const uint2 o = make_uint2(pack2<BF16>(finish<ACT>(acc.x, sx, sw[0], b[0]), finish<ACT>(acc.y, sx, sw[1], b[1])),
                                       pack2<BF16>(finish<ACT>(acc.z, sx, sw[2], b[2]), finish<ACT>(acc.w, sx, sw[3], b[3])));
            uint16_t* dst = p.out + (int64_t)(m0 + r) * p.out_rs + col;
            if (p.vec_out && col + 4 <= p.N) {
                *reinterpret_cast<uint2*>(dst) = o;
            } else {
                const uint16_t e[4] = {(uint16_t)o.x, (uint16_t)(o.x >> 16), (uint16_t)o.y, (uint16_t)(o.y >> 16)};
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (col + i < p.N) dst[i] = e[i];
            }
        }
    }
    __syncwarp();
    if (split > 1) cluster_sync();  // peers may still read this CTA's sums
}

// 256 x 256 output tiles by CTA pairs, persistent.  One MMA of a pair covers 256
// x 256 x 32: each CTA stages 128 rows of both operands, so a CTA reads half of
// the weight tile's bytes that it would need alone, and both keep 128 rows of the
// accumulator.  Two accumulators fill the TMEM: the epilogue of a tile runs under
// the products of the next.
struct PairCfg {
    static constexpr int BM = 256, BN = 256, BK = 128;
    static constexpr int A_BYTES = 128 * BK, B_BYTES = 128 * BK, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 6;
    static constexpr int EPI_WARPS = 8;         // two per TMEM lane quarter, half of the columns each
    static constexpr int STAGING = 32 * 128;    // per warp: 32 rows x 64 columns of the output
    static constexpr int THREADS = 128 + 32 * EPI_WARPS;
    struct Ctl {
        uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
        uint32_t tmem_base;
        int abort;
        alignas(16) float2 cols[BN];  // weight scale and bias of the tile's columns, read two at a time
    };
    static constexpr int STG_OFF = STAGES * STAGE;
    static constexpr int CTL_OFF = STG_OFF + EPI_WARPS * STAGING;
    static constexpr int SMEM = CTL_OFF + (int)((sizeof(Ctl) + 15) / 16 * 16);
    static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
    // Tiles are walked down columns of GROUP row tiles, so the tiles in flight at
    // one time share few rows of both operands (both stay in L2).
    static constexpr int GROUP = 8;
};

__device__ __forceinline__ void pair_tile(const LinearParams& p, int t, int& m0, int& n0) {
    const int per = PairCfg::GROUP * p.tiles_n;
    const int g = t / per, r = t - g * per;
    const int gm = min(PairCfg::GROUP, p.tiles_m - g * PairCfg::GROUP);
    m0 = (g * PairCfg::GROUP + r % gm) * PairCfg::BM;
    n0 = r / gm * PairCfg::BN;
}

template <bool BF16, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::THREADS, 1)
    k_int8_pair(const __grid_constant__ LinearParams p) {
    using C = PairCfg;
    extern __shared__ __align__(1024) uint8_t smem[];
    auto* ctl = reinterpret_cast<C::Ctl*>(smem + C::CTL_OFF);
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1, tiles = p.tiles_m * p.tiles_n;
    const int nkb = (p.K + C::BK - 1) / C::BK;

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
        ctl->abort = 0;
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
                    if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], 2 * C::STAGE);
                    const uint32_t bar = cluster_map(smem_u32(&ctl->full[s]), 0);
                    tma_load_2d_pair(st, &p.tmap_x, bar, kb * C::BK, m0 + 128 * rank);
                    tma_load_2d_pair(st + C::A_BYTES, &p.tmap_w, bar, kb * C::BK, n0 + 128 * rank);
                }
            }
            if (!ok) {  // gave up: time for the copies and MMAs in flight to end before the memory is given back
                const long long t0 = clock64();
                while (clock64() - t0 < p.timeout / 1000) {
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = idesc_i8(C::BM, C::BN);
            int it = 0, i = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step, i++) {
                const uint32_t d = tmem + (i & 1) * C::BN;
                if (i >= 2 && !mbar_wait_cluster(&ctl->acc_empty[i & 1], (i / 2 - 1) & 1, abort_flag, p.timeout)) break;
                tc_fence_after();
                for (int kb = 0; kb < nkb; kb++, it++) {
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
                    tc_commit_pair(&ctl->empty[s], 3);
                }
                if (ok) tc_commit_pair(&ctl->acc_full[i & 1], 3);
            }
        }
    } else if (warp >= 4) {
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;
        uint8_t* stg = smem + C::STG_OFF + ew * C::STAGING;
        float2* cols = ctl->cols + 128 * half;
        int i = 0;
        bool dead = false;  // a wait ran out: only the barriers of the remaining tiles are kept, so that no warp is left at one
        for (int t = first; t < tiles; t += step, i++) {
            int m0, n0;
            pair_tile(p, t, m0, n0);
            const int row0 = m0 + 128 * rank + 32 * quarter, col0 = n0 + 128 * half;
            {  // this half's column scales and biases (its four warps only)
                const int c = threadIdx.x & 127;
                float2 v = make_float2(0.f, 0.f);
                if (col0 + c < p.N) {
                    v.x = p.w_scales[col0 + c];
                    if (p.bias) v.y = load16<BF16>(p.bias + col0 + c);
                }
                asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
                cols[c] = v;
                asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
            }
            if (dead) continue;
            const float sx = row0 + lane < p.M ? p.x_scales[row0 + lane] : 0.f;
            const bool ok = mbar_wait_cluster(&ctl->acc_full[i & 1], (i >> 1) & 1, abort_flag, p.timeout);
            if (!__all_sync(FULL, ok)) {
                if (lane == 0) atomicOr(&g_int8_status, HB_DEV_TIMEOUT);
                dead = true;
                continue;
            }
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(32 * quarter) << 16) + (i & 1) * C::BN + 128 * half;
#pragma unroll
            for (int c = 0; c < 128; c += 64) {
                uint32_t lo[32], hi[32];
                tmem_ld32_async(acc + c, lo);
                tmem_ld32_async(acc + c + 32, hi);
                tmem_wait_ld(lo);
                tmem_wait_ld(hi);
                if (c == 64) {  // the accumulator is in registers: the next tile but one may take its place
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(cluster_map(smem_u32(&ctl->acc_empty[i & 1]), 0));
                }
                if (lane == 0) bulk_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int x = 8 * j + 2 * e;
                        const float4 sb = *reinterpret_cast<const float4*>(cols + c + x);
                        const int u = (int)(x < 32 ? lo[x & 31] : hi[x & 31]);
                        const int v = (int)(x < 32 ? lo[(x + 1) & 31] : hi[(x + 1) & 31]);
                        o[e] = pack2<BF16>(finish<ACT>(u, sx, sb.x, sb.y), finish<ACT>(v, sx, sb.z, sb.w));
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
                    for (int r = 0; r < 32 && row0 + r < p.M; r++)
#pragma unroll
                        for (int k = 0; k < 64; k += 32) {
                            const int x = k + lane;
                            if (col0 + c + x < p.N)
                                p.out[(int64_t)(row0 + r) * p.out_rs + col0 + c + x] = *reinterpret_cast<const uint16_t*>(
                                    stg + r * 128 + (((x >> 3) ^ (r & 7)) << 4) + (x & 7) * 2);
                        }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) bulk_wait<0>();
    }
    __syncwarp();
    __syncthreads();
    cluster_sync();  // no CTA leaves while the other's MMAs read its memory or arrivals are on the way
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

struct DeviceInfo {
    int sms = 0;
    int clock_khz = 0;
    unsigned configured = 0;  // kernels whose shared-memory limit is set
};
std::mutex g_mu;
DeviceInfo g_dev[64];

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int current_device(int* dev) {
    HB_CUDA_TRY(cudaGetDevice(dev));
    return *dev < 64 ? HB_OK : HB_ERR_UNSUPPORTED;
}

int device_info(int dev, DeviceInfo* info) {
    std::lock_guard<std::mutex> lk(g_mu);
    DeviceInfo& di = g_dev[dev];
    if (!di.sms) {
        HB_CUDA_TRY(cudaDeviceGetAttribute(&di.clock_khz, cudaDevAttrClockRate, dev));
        HB_CUDA_TRY(cudaDeviceGetAttribute(&di.sms, cudaDevAttrMultiProcessorCount, dev));
    }
    *info = di;
    return HB_OK;
}

template <class Kernel>
int configure(Kernel kern, int dev, int slot, int smem, DeviceInfo* info) {
    if (const int rc = device_info(dev, info)) return rc;
    std::lock_guard<std::mutex> lk(g_mu);
    DeviceInfo& di = g_dev[dev];
    if (!(di.configured >> slot & 1u)) {
        HB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        di.configured |= 1u << slot;
    }
    return HB_OK;
}

template <bool BF16, bool CODES, int M, int R>
int launch_few(const FewParams& p, cudaStream_t st) {
    const int smem = (int)few_bytes(p.M, p.K);
    auto kern = k_int8_few<BF16, CODES, M, R>;
    if (smem > 46 * 1024)  // near the default limit and above it: rare, so the limit is set each time
        HB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem));
    kern<<<(unsigned)ceil_div(p.N, 8 * R), 256, smem, st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}

template <bool BF16, bool CODES>
int launch_few(const FewParams& p, int dev, cudaStream_t st) {
    DeviceInfo di;
    if (const int rc = device_info(dev, &di)) return rc;
    // Channels per warp: four where that still leaves two CTAs per SM, so that a
    // token's codes are read from shared memory once for four channels.
    const bool wide = p.N >= 64 * di.sms;
    if (p.M == 1) return wide ? launch_few<BF16, CODES, 1, 4>(p, st) : launch_few<BF16, CODES, 1, 1>(p, st);
    if (p.M == 2) return wide ? launch_few<BF16, CODES, 2, 4>(p, st) : launch_few<BF16, CODES, 2, 1>(p, st);
    if (p.M <= 4) return wide ? launch_few<BF16, CODES, 4, 4>(p, st) : launch_few<BF16, CODES, 4, 1>(p, st);
    return wide ? launch_few<BF16, CODES, 8, 4>(p, st) : launch_few<BF16, CODES, 8, 1>(p, st);
}

template <bool CODES>
int launch_few(const FewParams& p, int dtype, int dev, cudaStream_t st) {
    return dtype == 1 ? launch_few<true, CODES>(p, dev, st) : launch_few<false, CODES>(p, dev, st);
}

template <bool BF16, int ACT>
int launch_tile(LinearParams& p, int dev, cudaStream_t st) {
    DeviceInfo di;
    auto kern = k_int8_tile<BF16, ACT>;
    if (const int rc = configure(kern, dev, BF16 * 2 + ACT, TileCfg::SMEM, &di)) return rc;
    p.timeout = 2000LL * di.clock_khz;
    const int64_t tn = ceil_div(p.N, TileCfg::BN), tm = ceil_div(p.M, TileCfg::BM);
    const int nkb = (int)ceil_div(p.K, TileCfg::BK);
    int split = 1;  // fill the SMs: double while a tile per CTA leaves half of them idle
    while (split < 8 && tn * tm * split * 2 <= di.sms && nkb >= 4 * split) split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tn * split), (unsigned)tm);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = TileCfg::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, split));
    return HB_OK;
}

// CTA pairs that can be resident at once (every SM, unless pairs do not fit some).
template <class Kernel>
int max_pairs(Kernel kern, int dev, int slot, int* pairs) {
    static int known[64][8];
    std::lock_guard<std::mutex> lk(g_mu);
    int& n = known[dev][slot];
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(PairCfg::THREADS);
        cfg.dynamicSmemBytes = PairCfg::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        HB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
        if (n <= 0) {
            n = 0;
            return HB_ERR_UNSUPPORTED;
        }
    }
    *pairs = n;
    return HB_OK;
}

template <bool BF16, int ACT>
int launch_pair(LinearParams& p, int dev, cudaStream_t st) {
    DeviceInfo di;
    auto kern = k_int8_pair<BF16, ACT>;
    const int slot = 4 + BF16 * 2 + ACT;
    int pairs = 0, rc;
    if ((rc = configure(kern, dev, slot, PairCfg::SMEM, &di))) return rc;
    if ((rc = max_pairs(kern, dev, slot, &pairs))) return rc;
    p.timeout = 2000LL * di.clock_khz;
    p.tiles_m = (int)ceil_div(p.M, PairCfg::BM);
    p.tiles_n = (int)ceil_div(p.N, PairCfg::BN);
    p.tma_out = aligned(p.out, 16) && (p.M == 1 || p.out_rs % 8 == 0);
    if (p.tma_out &&
        (rc = make_tmap_2d(&p.tmap_out, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p.out,
                           p.M, p.N, p.out_rs * 2, 32)))
        return rc;
    const int tiles = p.tiles_m * p.tiles_n;
    k_int8_pair<BF16, ACT><<<2 * std::min(tiles, pairs), PairCfg::THREADS, PairCfg::SMEM, st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}

template <bool BF16, int ACT>
int launch_linear(LinearParams& p, int dev, cudaStream_t st) {
    // Pairs once their tiles would occupy half of the SMs; below that the smaller
    // tiles and the split of K spread the work further.
    if (ceil_div(p.M, PairCfg::BM) * ceil_div(p.N, PairCfg::BN) >= 37) return launch_pair<BF16, ACT>(p, dev, st);
    return launch_tile<BF16, ACT>(p, dev, st);
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int hb_quantize_rows(const void* a, int64_t a_rs, int ka, const void* b, int64_t b_rs, int kb, int rows,
                                int8_t* codes, int64_t codes_rs, float* scales, int dtype, void* stream) {
    if (rows < 0 || ka <= 0 || kb < 0 || (kb > 0 && !b) || (int64_t)ka + kb > HB_INT8_MAX_K) return HB_ERR_ARG;
    if (dtype != 0 && dtype != 1) return HB_ERR_UNSUPPORTED;
    if (rows == 0) return HB_OK;
    if (!a || !codes || !scales) return HB_ERR_ARG;
    const int k = ka + kb;
    if (rows > 1 && codes_rs < k) return HB_ERR_ARG;
    if (!aligned(a, 2) || !aligned(b, 2) || !aligned(scales, 4) || !aligned(codes, 16) || codes_rs % 16) return HB_ERR_ALIGN;
    QuantParams p{static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), a_rs, b_rs, ka, k, rows, codes, codes_rs, scales};
    const bool vec = aligned(a, 16) && a_rs % 8 == 0 && ka % 8 == 0 && (!kb || (aligned(b, 16) && b_rs % 8 == 0 && kb % 8 == 0));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int dev = 0, rc;
    DeviceInfo di;
    if ((rc = current_device(&dev)) || (rc = device_info(dev, &di))) return rc;
    if (dtype == 1) return vec ? launch_quantize<true, true>(p, di.sms, st) : launch_quantize<true, false>(p, di.sms, st);
    return vec ? launch_quantize<false, true>(p, di.sms, st) : launch_quantize<false, false>(p, di.sms, st);
}

namespace hb {
namespace {
// Checks shared by the two linear entries; 1: nothing to do.
int check_linear(const void* x, const int8_t* w, int64_t w_rs, const float* w_scales, const void* bias, const void* out,
                 int64_t out_rs, int M, int N, int K, int act, int dtype) {
    if (M < 0 || N < 0 || K <= 0 || K > HB_INT8_MAX_K || act < 0 || act > 1) return HB_ERR_ARG;
    if (dtype != 0 && dtype != 1) return HB_ERR_UNSUPPORTED;
    if (M == 0 || N == 0) return 1;
    if (!x || !w || !w_scales || !out) return HB_ERR_ARG;
    if ((M > 1 && out_rs < N) || (N > 1 && w_rs < K)) return HB_ERR_ARG;
    if (!aligned(w, 16) || (N > 1 && w_rs % 16) || !aligned(w_scales, 4) || !aligned(bias, 2) || !aligned(out, 2))
        return HB_ERR_ALIGN;
    if (ceil_div(M, 128) > 65535 || ceil_div(M, 128) * ceil_div(N, 128) > INT32_MAX / 8) return HB_ERR_UNSUPPORTED;
    return HB_OK;
}

int linear_codes(const int8_t* x, int64_t x_rs, const float* x_scales, const int8_t* w, int64_t w_rs, const float* w_scales,
                 const void* bias, void* out, int64_t out_rs, int M, int N, int K, int act, int dtype, int dev,
                 cudaStream_t st) {
    LinearParams p;
    int rc;
    if ((rc = make_tmap_2d(&p.tmap_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, M, K, x_rs, 128))) return rc;
    if ((rc = make_tmap_2d(&p.tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, N, K, w_rs, 128))) return rc;
    p.x_scales = x_scales;
    p.w_scales = w_scales;
    p.bias = static_cast<const uint16_t*>(bias);
    p.out = static_cast<uint16_t*>(out);
    p.out_rs = out_rs;
    p.M = M;
    p.N = N;
    p.K = K;
    p.vec_out = aligned(out, 8) && out_rs % 4 == 0;
    if (dtype == 1) return act ? launch_linear<true, 1>(p, dev, st) : launch_linear<true, 0>(p, dev, st);
    return act ? launch_linear<false, 1>(p, dev, st) : launch_linear<false, 0>(p, dev, st);
}
}  // namespace
}  // namespace hb

extern "C" int hb_int8_linear(const int8_t* x, int64_t x_rs, const float* x_scales, const int8_t* w, int64_t w_rs,
                              const float* w_scales, const void* bias, void* out, int64_t out_rs, int M, int N, int K,
                              int act, int dtype, void* stream) {
    int rc = check_linear(x, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype), dev = 0;
    if (rc) return rc > 0 ? HB_OK : rc;
    if (!x_scales || (M > 1 && x_rs < K)) return HB_ERR_ARG;
    if (!aligned(x, 16) || (M > 1 && x_rs % 16) || !aligned(x_scales, 4)) return HB_ERR_ALIGN;
    if ((rc = current_device(&dev))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (is_few(M, K)) {
        const FewParams p{x, x_rs, x_scales, w, w_rs, w_scales, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out), out_rs, M, N, K, act};
        return launch_few<true>(p, dtype, dev, st);
    }
    return linear_codes(x, x_rs, x_scales, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype, dev, st);
}

extern "C" size_t hb_int8_linear16_workspace_bytes(int M, int K) {
    if (M <= 0 || K <= 0 || K > HB_INT8_MAX_K || is_few(M, K)) return 0;
    return (size_t)(few_bytes(M, K) + 4 * (int64_t)M);
}

extern "C" int hb_int8_linear16(const void* x, int64_t x_rs, const int8_t* w, int64_t w_rs, const float* w_scales,
                                const void* bias, void* out, int64_t out_rs, int M, int N, int K, int act, int dtype,
                                void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_linear(x, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype), dev = 0;
    if (rc) return rc > 0 ? HB_OK : rc;
    if (!aligned(x, 2)) return HB_ERR_ALIGN;
    const size_t need = hb_int8_linear16_workspace_bytes(M, K);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return HB_ERR_WORKSPACE;
    if ((rc = current_device(&dev))) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!need) {
        const FewParams p{x, x_rs, nullptr, w, w_rs, w_scales, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out), out_rs, M, N, K, act};
        return launch_few<false>(p, dtype, dev, st);
    }
    int8_t* codes = static_cast<int8_t*>(workspace);
    const int64_t pitch = few_bytes(1, K);
    float* scales = reinterpret_cast<float*>(codes + pitch * M);
    if ((rc = hb_quantize_rows(x, x_rs, K, nullptr, 0, 0, M, codes, pitch, scales, dtype, stream))) return rc;
    return linear_codes(codes, pitch, scales, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype, dev, st);
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
