// 8-bit products of one to four tokens: every weight is read once, and the bytes of
// the weights bound it.  A warp forms R output channels at a time, each lane 16
// bytes of every channel's row, with 4-way 8-bit dot products; the tokens' codes lie
// in shared memory, quantised there from 16 bits by each CTA (they are a few KB; the
// first weights are on their way meanwhile).  Sums and results are those of the
// tensor-core kernels, bit for bit.  1 x 18432 with K 3072: 11.2 us (5.1 TB/s) from
// DRAM, 2.5 us of it the launch and the token, with four CTAs per SM (all 576 at once),
// 14.3 us with three; two tokens 12.7 us, 16.0 us with two CTAs per SM.  Rings of
// asynchronous copies per warp, 192 KB on their way per SM, took 11.6 us for one token
// and 0.5 us more for small products.  Three and four tokens: while the weights are few
// (int8_few_takes), past that the dot products weigh more than the weights' bytes.
#include <climits>

#include "int8_common.cuh"

namespace hb {
namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int kRows = 4;
constexpr int kSmem = 40 * 1024;  // codes of the tokens, at most
constexpr int resident(int tokens) { return tokens <= 2 ? 4 : 3; }  // CTAs per SM

// 16 bytes of a row of codes, of which `left` (at least 1) are inside it.
__device__ __forceinline__ int4 load_codes(const int8_t* p, int left) {
    if (left >= 16) return __ldg(reinterpret_cast<const int4*>(p));
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < left; i++) w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
    return make_int4(w[0], w[1], w[2], w[3]);
}

template <bool BF16, bool CODES, int M, int R>
__global__ void __launch_bounds__(256, resident(M)) k_int8_few(const __grid_constant__ Int8Problem p) {
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
    const int mine = lane < R * M ? n0 + lane / M : INT_MAX;  // the channel this lane finishes
    float ws = 0.f, bias = 0.f;
    if (mine < p.N) {
        ws = w_factor(p.w_scales[mine]);
        if (p.bias) bias = load16<BF16>(p.bias + mine);
    }

    if constexpr (CODES) {
        for (int i = threadIdx.x; i < M * chunks; i += 256) {
            const int m = i / chunks, c = i - m * chunks;
            *reinterpret_cast<int4*>(s_codes + m * pitch + 16 * c) =
                load_codes(static_cast<const int8_t*>(p.x) + m * p.x_rs + 16 * c, p.K - 16 * c);
        }
        if (threadIdx.x < M) s_scale[threadIdx.x] = x_factor(p.x_scales[threadIdx.x]);
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
            for (int c = 8 * threadIdx.x; c < p.K; c += 8 * 256) {
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
            if (threadIdx.x == 0) s_scale[m] = x_factor(s.scale);
            for (int c = 8 * threadIdx.x; c < pitch; c += 8 * 256) {
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
                    const int4 x = *reinterpret_cast<const int4*>(s_codes + m * pitch + 16 * c);
#pragma unroll
                    for (int r = 0; r < R; r++)
                        acc[r][m] = __dp4a(w[u][r].w, x.w, __dp4a(w[u][r].z, x.z, __dp4a(w[u][r].y, x.y, __dp4a(w[u][r].x, x.x, acc[r][m]))));
                }
            }
        }
    }
    int sum = 0;  // lane r * M + m finishes channel r of token m
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
        for (int m = 0; m < M; m++) {
            const int v = __reduce_add_sync(FULL, acc[r][m]);
            if (lane == r * M + m) sum = v;
        }
    }
    const int m = lane % M;
    if (mine < p.N) {
        const float y = p.act ? finish<1>(sum, s_scale[m], ws, bias) : finish<0>(sum, s_scale[m], ws, bias);
        p.out[m * p.out_rs + mine] = (uint16_t)pack2<BF16>(y, 0.f);
    }
}

template <bool BF16, bool CODES, int M, int R>
int launch(const Int8Problem& p, cudaStream_t st) {
    k_int8_few<BF16, CODES, M, R><<<(unsigned)ceil_div(p.N, 8 * R), 256, (size_t)(code_pitch(p.K) * p.M), st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}

template <bool BF16, bool CODES, int M>
int launch(const Int8Problem& p, int sms, cudaStream_t st) {
    // Channels per warp: the fewest of 1, 2 and 4 for which all CTAs run at once, since
    // each begins with the tokens' codes; and 4 past that.  One token: 8192 x 8192 14.5 us
    // with 2, 16.8 with 4, 17.5 with 1; 9216 x 3072 7.4 with 2, 8.3 with 4, 9.7 with 1; 4096
    // x 14336 15.0 with 1, 20.9 with 4; 12288 x 3072 9.4 with 4, 10.8 with 2.
    const int64_t warps = 8LL * sms * resident(M);
    if (p.N <= warps) return launch<BF16, CODES, M, 1>(p, st);
    return p.N <= 2 * warps ? launch<BF16, CODES, M, 2>(p, st) : launch<BF16, CODES, M, 4>(p, st);
}
template <bool BF16, bool CODES>
int launch(const Int8Problem& p, int sms, cudaStream_t st) {
    switch (p.M) {
        case 1: return launch<BF16, CODES, 1>(p, sms, st);
        case 2: return launch<BF16, CODES, 2>(p, sms, st);
        case 3: return launch<BF16, CODES, 3>(p, sms, st);
        default: return launch<BF16, CODES, 4>(p, sms, st);
    }
}

}  // namespace

// From 16 bits, against the quantisation and the tensor cores: 3 x 4096, K 4096 8.3 us
// and 9.8, 3 x 9216, K 3072 9.8 and 11.9, 4 x 2048, K 2048 5.4 and 6.8; 4 x 5120, K 5120
// 13.5 and 12.6, 3 x 3000, K 12288 16.4 and 14.1, 4 x 18432, K 3072 20.2 and 14.4.
bool int8_few_takes(int M, int64_t N, int K) {
    if (M > kRows || code_pitch(K) * M > kSmem) return false;
    return M <= 2 || M * N * K <= 96000000;
}

int launch_int8_few(const Int8Problem& p, const DeviceInfo& di, cudaStream_t st) {
    if (p.x_scales) return p.dtype == 1 ? launch<true, true>(p, di.sms, st) : launch<false, true>(p, di.sms, st);
    return p.dtype == 1 ? launch<true, false>(p, di.sms, st) : launch<false, false>(p, di.sms, st);
}

}  // namespace hb
