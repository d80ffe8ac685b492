// Shared parts of the 8-bit linear layers: the arithmetic around the integer sums,
// launch parameters and the per-device facts the launchers use.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "int8_codes.cuh"
#include "sm100_ptx.cuh"

namespace hb {

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

__device__ __forceinline__ uint32_t max_mag(uint32_t m, const uint4& v) {
    return max_mag(max_mag(max_mag(max_mag(m, v.x), v.y), v.z), v.w);
}
template <bool BF16>
__device__ __forceinline__ uint2 codes8(const uint4& v, const RowScale& s) {
    if (!s.live) return make_uint2(0, 0);
    return make_uint2(codes4<BF16>(v.x, v.y, s.inv), codes4<BF16>(v.z, v.w, s.inv));
}

// tanh-GELU(v) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3), the
// exponential taken in base 2.
constexpr float kGelu0 = -2.f * 1.4426950408889634f * 0.7978845608028654f, kGelu1 = kGelu0 * 0.044715f;
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float gelu_tanh(float v) {
    return v * rcp(1.f + ptx::ex2(v * fmaf(kGelu1, v * v, kGelu0)));
}
// (sum * x_scale) * w_scale + bias.  A sum below 2^31 times the scale of bf16 rows near
// their type's end (up to 2^121) would pass fp32's range although w_scale brings the
// product back, so the kernels take 2^-24 x_scale and 2^24 w_scale: exact for
// x_scale >= 2^-102 (smaller ones lose up to 5 of 24 bits) and w_scale < 2^104.
__device__ __forceinline__ float x_factor(float scale) { return scale * 0x1p-24f; }
__device__ __forceinline__ float w_factor(float scale) { return scale * 0x1p24f; }
// sx, sw: the factors above.
template <int ACT>
__device__ __forceinline__ float finish(int acc, float sx, float sw, float b) {
    const float v = fmaf(__int2float_rn(acc) * sx, sw, b);
    return ACT ? gelu_tanh(v) : v;
}
// Two neighbouring columns at once, the same operations in packed fp32: sx the row's
// factor twice, sw and b the columns' factors and biases; packed to 16 bits.
template <bool BF16, int ACT>
__device__ __forceinline__ uint32_t finish2(int acc0, int acc1, uint64_t sx, uint64_t sw, uint64_t b) {
    using namespace ptx;
    uint64_t v = f2_fma(f2_mul(f2_pack(__int2float_rn(acc0), __int2float_rn(acc1)), sx), sw, b);
    float lo, hi;
    if constexpr (ACT) {
        const uint64_t k0 = f2_pack(kGelu0, kGelu0), k1 = f2_pack(kGelu1, kGelu1), one = f2_pack(1.f, 1.f);
        f2_unpack(f2_mul(v, f2_fma(k1, f2_mul(v, v), k0)), lo, hi);
        f2_unpack(f2_add(f2_pack(ex2(lo), ex2(hi)), one), lo, hi);
        v = f2_mul(v, f2_pack(rcp(lo), rcp(hi)));
    }
    f2_unpack(v, lo, hi);
    return pack2<BF16>(lo, hi);
}

struct DeviceInfo {
    int sms = 0;
    int clock_khz = 0;
};
// SM count and SM clock of a device, queried once.
int device_info(int dev, DeviceInfo* info);
int current_device(int* dev);
inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int64_t code_pitch(int K) { return (K + 15) / 16 * 16; }

// One product: x (codes and scales, or for a few tokens 16-bit rows with x_scales
// null) times w, see hb_int8_linear.
struct Int8Problem {
    const void* x;
    int64_t x_rs;
    const float* x_scales;
    const int8_t* w;
    int64_t w_rs;
    const float* w_scales;
    const uint16_t* bias;
    uint16_t* out;
    int64_t out_rs;
    int M, N, K, act, dtype;
};
bool int8_few_takes(int M, int64_t N, int K);  // int8_few.cu: products it serves
int launch_int8_few(const Int8Problem& p, const DeviceInfo& di, cudaStream_t st);
// int8_gemm.cu; early_weights: the weights are not written by the kernel before this
// launch, so they may be fetched before it has ended.
int launch_int8_gemm(const Int8Problem& p, int dev, const DeviceInfo& di, bool early_weights, cudaStream_t st);

}  // namespace hb
