// Adaptive-LayerNorm modulation and gated residuals of the FLUX transformer
// blocks around the attention (the adaLN-Zero steps of diffusers'
// FluxTransformerBlock / FluxSingleTransformerBlock, which wrap the processor of
// hilberta/flux_adapter.py:259-340):
//
//   x' = x + gate[b] * y                         (gated residual, optional)
//   h  = LayerNorm(x') * (1 + scale[b]) + shift[b]   (LayerNorm without affine, optional)
//
// As tensor ops these are five to seven read+write passes over the [tokens,
// hidden] stream (the LayerNorm, the broadcast multiply and add of the
// modulation, the gate multiply and the residual add).  Here one warp owns one
// row: the row is read once (plus y when the residual is taken), kept in
// registers, and x' and h are each written once.
//
// Arithmetic: fp32 throughout; x' is rounded to the 16-bit type before the
// LayerNorm reads it (it is the stored residual stream); mean and variance by
// two passes over the register-held row, 1/sqrt(var + eps) by rsqrtf, and h
// rounded once.  Memory-bound: 16-byte accesses, C a multiple of 256 (8
// elements per lane per vector) up to 4096.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "common.cuh"
#include "int8_codes.cuh"
#include "sm100_ptx.cuh"

namespace hb {
namespace {

constexpr int kMaxVec = 16;  // vectors of 8 elements per lane: C <= 32 * 8 * 16 = 4096

struct AdaParams {
    const void* x;  // [rows][C], row stride x_rs (elements)
    const void* y;  // [rows][C] or null, row stride y_rs
    const void* gate;   // [B][C] (batch stride mod_bs) when y is given
    const void* shift;  // [B][C] when h is written
    const void* scale;
    void* x_out;  // [rows][C] (may alias x) when y is given
    void* h_out;  // [rows][C] or null
    int64_t x_rs, y_rs, xo_rs, h_rs, mod_bs;
    int rows, rows_per_batch, C;
    float eps;
};

template <bool BF16>
struct Vec8 {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    static __device__ __forceinline__ void load(const void* p, float (&f)[8]) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
                const float2 t = __half22float2(h);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            } else {
                const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One warp per row; lane l owns elements [8 (l + 32 i), 8 (l + 32 i) + 8) for
// i < C / 256, so each 16-byte vector access of a warp covers 512 contiguous bytes.
template <bool BF16, bool RESIDUAL, bool NORM>
__global__ void __launch_bounds__(256) k_adaln(AdaParams p) {
    using V = Vec8<BF16>;
    using T = typename V::T;
    const int lane = threadIdx.x & 31;
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;  // whole warps leave together
    const int b = row / p.rows_per_batch;
    const int nv = p.C >> 8;
    const T* x = static_cast<const T*>(p.x) + row * p.x_rs;
    uint4 xv[kMaxVec];
#pragma unroll
    for (int i = 0; i < kMaxVec; ++i)
        if (i < nv) xv[i] = *reinterpret_cast<const uint4*>(x + 8 * (lane + 32 * i));
    if constexpr (RESIDUAL) {
        const T* y = static_cast<const T*>(p.y) + row * p.y_rs;
        const T* g = static_cast<const T*>(p.gate) + b * p.mod_bs;
        T* xo = static_cast<T*>(p.x_out) + row * p.xo_rs;
#pragma unroll
        for (int i = 0; i < kMaxVec; ++i) {
            if (i < nv) {
                const int c = 8 * (lane + 32 * i);
                float fx[8], fy[8], fg[8];
                V::load(&xv[i], fx);
                V::load(y + c, fy);
                V::load(g + c, fg);
#pragma unroll
                for (int e = 0; e < 8; ++e) fx[e] = fmaf(fg[e], fy[e], fx[e]);
                xv[i] = V::pack(fx);  // the stored residual stream, rounded
                *reinterpret_cast<uint4*>(xo + c) = xv[i];
            }
        }
    }
    if constexpr (NORM) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxVec; ++i) {
            if (i < nv) {
                float f[8];
                V::load(&xv[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) s += f[e];
            }
        }
        const float inv_c = 1.f / static_cast<float>(p.C);
        const float mean = warp_sum(s) * inv_c;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxVec; ++i) {
            if (i < nv) {
                float f[8];
                V::load(&xv[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float d = f[e] - mean;
                    q = fmaf(d, d, q);
                }
            }
        }
        const float rstd = rsqrtf(warp_sum(q) * inv_c + p.eps);
        const T* sh = static_cast<const T*>(p.shift) + b * p.mod_bs;
        const T* sc = static_cast<const T*>(p.scale) + b * p.mod_bs;
        T* h = static_cast<T*>(p.h_out) + row * p.h_rs;
#pragma unroll
        for (int i = 0; i < kMaxVec; ++i) {
            if (i < nv) {
                const int c = 8 * (lane + 32 * i);
                float f[8], fs[8], fc[8];
                V::load(&xv[i], f);
                V::load(sh + c, fs);
                V::load(sc + c, fc);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = fmaf((f[e] - mean) * rstd, 1.f + fc[e], fs[e]);
                *reinterpret_cast<uint4*>(h + c) = V::pack(f);
            }
        }
    }
}

struct AdaInt8Params {
    AdaParams a;  // h_out unused
    int8_t* codes;  // [rows][C], row stride c_rs (bytes)
    int64_t c_rs;
    float* scales;  // [rows]
};

// Pairs of fp32 values in one register pair (two operations per instruction).
template <bool BF16>
struct Pairs {
    static __device__ __forceinline__ void unpack(const uint4& u, uint64_t (&f)[4]) {
        float v[8];
        Vec8<BF16>::load(&u, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = ptx::f2_pack(v[2 * i], v[2 * i + 1]);
    }
    static __device__ __forceinline__ uint4 pack(const uint64_t (&f)[4]) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) ptx::f2_unpack(f[i], v[2 * i], v[2 * i + 1]);
        return Vec8<BF16>::pack(v);
    }
};
// max(|a|, |b|, m); NaN when any of them is (so a NaN in a row is never lost).
__device__ __forceinline__ float max_abs(uint64_t pair, float m) {
    float a, b, d;
    ptx::f2_unpack(pair, a, b);
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(m));
    return d;
}
__device__ __forceinline__ float sum_of(int n, float v) {  // over n lanes, a power of two
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
        if (o < n) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The same pass with h quantised instead of rounded to 16 bits, so that the int8
// product reads half the bytes and no separate pass over h exists.  One CTA of
// C / (8 NV) threads per row, NV vectors of 8 elements each: row, modulation and h
// stay in registers.  Memory-bound by its bytes (2 C, 4 C with the residual, read
// and C, 3 C written per row), but only just: what it costs beyond them is
// instructions, so two fp32 operations go in one, a lane holds as many elements as C
// divides into (the reductions' instructions are per lane), every lane equally many
// (no tests), and mean and variance share one barrier.  The CTAs are persistent, keep
// the modulation of their batch entry and fetch a row ahead; the register limits
// keep 12 to 16 warps on an SM (16384 x 3072 with the residual: 55.8 us at 128
// registers, 60.9 at 156).  16384 x 3072, bf16, from DRAM: 55.8 us (6.3 TB/s) with the
// residual, 31.9 (4.7 TB/s) without, 32.7 with two rows ahead; 33975 x 1280: 58.2 and
// 43.8 (one vector per lane, so the reductions weigh most).
//
// Mean and variance: from the means m and the sums d of squared deviations of sets of
// n elements each, mean = sum m / sets and d = sum (d + n (m - mean)^2), first over a
// warp's lanes, then over the warps; large sums are never subtracted.
template <bool BF16, bool RESIDUAL, int NV>
__global__ void __launch_bounds__(NV == 1 ? 512 : NV == 4 ? 128 : 256, NV == 4 ? 3 : 2)
    k_adaln_int8(const __grid_constant__ AdaInt8Params q) {
    using namespace ptx;
    using P = Pairs<BF16>;
    using E = typename Vec8<BF16>::T;
    __shared__ float2 s_stat[16];  // a word per warp, zeros past the last
    __shared__ uint32_t s_mag[16];
    const AdaParams& p = q.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int c0 = 8 * threadIdx.x, cs = 8 * blockDim.x;  // first column, columns between vectors
    const int step = gridDim.x;
    const int span = 1 << (32 - __clz(warps - 1)), part = lane & (span - 1);  // warps to a power of two
    const float inv_c = 1.f / static_cast<float>(p.C), inv_w = 1.f / static_cast<float>(warps);
    if (threadIdx.x < 16) {
        s_stat[threadIdx.x] = make_float2(0.f, 0.f);
        s_mag[threadIdx.x] = 0;
    }
    __syncthreads();
    uint4 x[NV], y[NV];
    auto fetch = [&](int row) {
        if (row >= p.rows) return;
        const E* px = static_cast<const E*>(p.x) + row * p.x_rs + c0;
        const E* py = static_cast<const E*>(p.y) + row * p.y_rs + c0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = *reinterpret_cast<const uint4*>(px + i * cs);
            if constexpr (RESIDUAL) y[i] = *reinterpret_cast<const uint4*>(py + i * cs);
        }
    };
    uint64_t shift[NV][4], scale[NV][4];
    uint4 gate[NV];
    int batch_end = 0;  // modulation of rows [.., batch_end)
    const uint64_t one = f2_pack(1.f, 1.f), magic = f2_pack(12582912.f, 12582912.f);
    grid_launch_dependents();  // the product's CTAs may set themselves up meanwhile
    fetch(blockIdx.x);
    for (int row = blockIdx.x; row < p.rows; row += step) {  // the same for the whole CTA
        if (row >= batch_end) {
            const int batch = row / p.rows_per_batch;
            batch_end = (batch + 1) * p.rows_per_batch;
            const int64_t at = batch * p.mod_bs + c0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                P::unpack(*reinterpret_cast<const uint4*>(static_cast<const E*>(p.shift) + at + i * cs), shift[i]);
                P::unpack(*reinterpret_cast<const uint4*>(static_cast<const E*>(p.scale) + at + i * cs), scale[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) scale[i][e] = f2_add(scale[i][e], one);
                if constexpr (RESIDUAL) gate[i] = *reinterpret_cast<const uint4*>(static_cast<const E*>(p.gate) + at + i * cs);
            }
        }
        uint64_t f[NV][4], sum = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            P::unpack(x[i], f[i]);
            if constexpr (RESIDUAL) {
                uint64_t fy[4], fg[4];
                P::unpack(y[i], fy);
                P::unpack(gate[i], fg);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[i][e] = f2_fma(fg[e], fy[e], f[i][e]);
                const uint4 stream = P::pack(f[i]);  // the stored residual stream, rounded
                *reinterpret_cast<uint4*>(static_cast<E*>(p.x_out) + row * p.xo_rs + c0 + i * cs) = stream;
                P::unpack(stream, f[i]);
            }
            sum = f2_add(sum, f2_add(f2_add(f[i][0], f[i][1]), f2_add(f[i][2], f[i][3])));
        }
        fetch(row + step);
        constexpr float n = 8.f * NV;
        float a, b;
        f2_unpack(sum, a, b);
        const float m = (a + b) * (1.f / n);
        uint64_t dev = 0;
        const uint64_t minus = f2_pack(-m, -m);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t d = f2_add(f[i][e], minus);
                dev = f2_fma(d, d, dev);
            }
        }
        f2_unpack(dev, a, b);
        float mean = warp_sum(m) * (1.f / 32.f), t = m - mean;
        float d = warp_sum(fmaf(t * t, n, a + b));
        if (warps > 1) {  // the same for the CTA
            if (lane == 0) s_stat[warp] = make_float2(mean, d);
            __syncthreads();
            const float2 w = s_stat[part];
            mean = sum_of(span, w.x) * inv_w;
            t = w.x - mean;
            d = sum_of(span, part < warps ? fmaf(t * t, 32.f * n, w.y) : 0.f);
        }
        const float rstd = rsqrtf(fmaf(d, inv_c, p.eps));
        const uint64_t r2 = f2_pack(rstd, rstd), m2 = f2_pack(-mean, -mean);
        float mag = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[i][e] = f2_fma(f2_mul(f2_add(f[i][e], m2), r2), scale[i][e], shift[i][e]);
                mag = max_abs(f[i][e], mag);
            }
        }
        uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(mag));  // NaN sorts above infinity
        if (warps > 1) {
            if (lane == 0) s_mag[warp] = bits;
            __syncthreads();
            bits = __reduce_max_sync(0xffffffffu, s_mag[part]);
        }
        const RowScale rs = row_scale(__uint_as_float(bits));
        if (threadIdx.x == 0) q.scales[row] = rs.scale;
        const uint64_t inv2 = f2_pack(rs.inv, rs.inv);
        int8_t* out = q.codes + row * q.c_rs + c0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint32_t c[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // code_bits, two at a time
                f2_unpack(f2_add(f2_mul(f[i][e], inv2), magic), a, b);
                c[2 * e] = __float_as_uint(a);
                c[2 * e + 1] = __float_as_uint(b);
            }
            uint2 o = make_uint2(pack_codes(c[0], c[1], c[2], c[3]), pack_codes(c[4], c[5], c[6], c[7]));
            if (!rs.live) o = make_uint2(0, 0);
            *reinterpret_cast<uint2*>(out + i * cs) = o;
        }
    }
}

// CTAs of a k_adaln_int8 that fit an SM, asked once per variant and size.
template <class Kernel>
int resident_ctas(Kernel kern, int variant, int threads, int* n) {
    static std::atomic<int> known[16][17];
    std::atomic<int>& k = known[variant][threads / 32];
    if (!(*n = k.load(std::memory_order_relaxed))) {
        HB_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kern, threads, 0));
        if (*n <= 0) return HB_ERR_UNSUPPORTED;
        k.store(*n, std::memory_order_relaxed);
    }
    return HB_OK;
}

template <bool BF16, bool RESIDUAL, int NV>
int launch_adaln_int8(const AdaInt8Params& p, int sms, cudaStream_t st) {
    auto kern = k_adaln_int8<BF16, RESIDUAL, NV>;
    const int threads = p.a.C / (8 * NV);
    int per_sm = 0;
    if (const int rc = resident_ctas(kern, (BF16 * 2 + RESIDUAL) * 4 + NV - 1, threads, &per_sm)) return rc;
    kern<<<(unsigned)std::min<int64_t>(p.a.rows, (int64_t)per_sm * sms), threads, 0, st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}

template <bool BF16, bool RESIDUAL>
int launch_adaln_int8(const AdaInt8Params& p, cudaStream_t st) {
    int dev = 0, sms = 0;
    HB_CUDA_TRY(cudaGetDevice(&dev));
    HB_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // Vectors per lane: three or four if they divide the row into whole warps, else two
    // or one.  With and without the residual, 16384 x 3072: three 55.7 and 31.9 us, four
    // 56.6 and 31.6, two 68.8 and 46.2; 3590 x 2048: four 9.1 and 6.3, two 9.6 and 7.1.
    const int groups = p.a.C / 256;
    if (groups % 3 == 0) return launch_adaln_int8<BF16, RESIDUAL, 3>(p, sms, st);
    if (groups % 4 == 0) return launch_adaln_int8<BF16, RESIDUAL, 4>(p, sms, st);
    if (groups % 2 == 0) return launch_adaln_int8<BF16, RESIDUAL, 2>(p, sms, st);
    return launch_adaln_int8<BF16, RESIDUAL, 1>(p, sms, st);
}

template <bool BF16>
int launch_adaln(const AdaParams& p, cudaStream_t st) {
    const dim3 grid((p.rows + 7) / 8), block(256);
    const bool res = p.y != nullptr, norm = p.h_out != nullptr;
    if (res && norm)
        k_adaln<BF16, true, true><<<grid, block, 0, st>>>(p);
    else if (res)
        k_adaln<BF16, true, false><<<grid, block, 0, st>>>(p);
    else
        k_adaln<BF16, false, true><<<grid, block, 0, st>>>(p);
    HB_CUDA_TRY(cudaGetLastError());
    return HB_OK;
}

}  // namespace
}  // namespace hb

extern "C" int hb_adaln_residual(const void* x, int64_t x_rs, const void* y, int64_t y_rs, const void* gate,
                                 const void* shift, const void* scale, int64_t mod_bs, void* x_out, int64_t xo_rs,
                                 void* h_out, int64_t h_rs, int rows, int rows_per_batch, int C, float eps, int dtype,
                                 void* stream) {
    using namespace hb;
    if (!x || rows < 0 || rows_per_batch <= 0 || C <= 0 || !(eps >= 0.f)) return HB_ERR_ARG;
    if (!y && !h_out) return HB_ERR_ARG;                 // nothing to do
    if (y && (!gate || !x_out)) return HB_ERR_ARG;       // residual needs its gate and destination
    if (h_out && (!shift || !scale)) return HB_ERR_ARG;  // modulation needs shift and scale
    if (dtype != 0 && dtype != 1) return HB_ERR_UNSUPPORTED;
    if (C % 256 || C > 256 * kMaxVec) return HB_ERR_UNSUPPORTED;
    auto a16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
    auto s8 = [](int64_t st) { return st % 8 == 0; };
    if (!a16(x) || (y && (!a16(y) || !a16(gate) || !a16(x_out))) || (h_out && (!a16(h_out) || !a16(shift) || !a16(scale))))
        return HB_ERR_ALIGN;
    if (!s8(x_rs) || !s8(y_rs) || !s8(xo_rs) || !s8(h_rs) || !s8(mod_bs)) return HB_ERR_ALIGN;
    if (rows == 0) return HB_OK;
    AdaParams p{x, y, gate, shift, scale, x_out, h_out, x_rs, y_rs, xo_rs, h_rs, mod_bs, rows, rows_per_batch, C, eps};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == 1 ? launch_adaln<true>(p, st) : launch_adaln<false>(p, st);
}

extern "C" int hb_adaln_residual_int8(const void* x, int64_t x_rs, const void* y, int64_t y_rs, const void* gate,
                                      const void* shift, const void* scale, int64_t mod_bs, void* x_out,
                                      int64_t xo_rs, int8_t* codes, int64_t codes_rs, float* scales, int rows,
                                      int rows_per_batch, int C, float eps, int dtype, void* stream) {
    using namespace hb;
    if (rows < 0 || rows_per_batch <= 0 || C <= 0 || !(eps >= 0.f)) return HB_ERR_ARG;
    if (dtype != 0 && dtype != 1) return HB_ERR_UNSUPPORTED;
    if (C % 256 || C > 256 * kMaxVec) return HB_ERR_UNSUPPORTED;
    if (rows == 0) return HB_OK;
    if (!x || !codes || !scales || !shift || !scale) return HB_ERR_ARG;
    if (y && (!gate || !x_out)) return HB_ERR_ARG;  // residual needs its gate and destination
    if (rows > 1 && codes_rs < C) return HB_ERR_ARG;
    auto a16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
    auto s8 = [](int64_t st) { return st % 8 == 0; };
    if (!a16(x) || !a16(shift) || !a16(scale) || !a16(codes) || (y && (!a16(y) || !a16(gate) || !a16(x_out))) ||
        (reinterpret_cast<uintptr_t>(scales) & 3))
        return HB_ERR_ALIGN;
    if (!s8(x_rs) || !s8(y_rs) || !s8(xo_rs) || !s8(mod_bs) || codes_rs % 16) return HB_ERR_ALIGN;
    const AdaInt8Params p{{x, y, gate, shift, scale, x_out, nullptr, x_rs, y_rs, xo_rs, 0, mod_bs, rows, rows_per_batch, C, eps},
                          codes, codes_rs, scales};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == 1) return y ? launch_adaln_int8<true, true>(p, st) : launch_adaln_int8<true, false>(p, st);
    return y ? launch_adaln_int8<false, true>(p, st) : launch_adaln_int8<false, false>(p, st);
}
