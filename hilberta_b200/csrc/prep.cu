// Q/K/V preparation for the attention kernel: per-head RMSNorm, rotary embedding
// and the text + image concatenation in one pass over HBM.
//
// The FLUX processor (hilberta/flux_adapter.py:280-298) splits each projection
// into heads, RMS-normalises query and key rows over the head dimension with a
// learned weight (separate weights for the text and the image stream), puts the
// text tokens first, rotates query and key by the rotary embedding and hands
// [B, H, S, D] views of [B, S, H, D] storage to the attention.  As separate
// tensor ops that is four to five read+write passes per tensor; here every
// (token, head) row is read once and written once, straight into the [B, S, H, D]
// layout the attention kernel reads in place.
//
// Arithmetic follows those ops step by step (diffusers 0.36 RMSNorm and
// apply_rotary_emb with real cos/sin, the processor's dependency):
//   v   = mean over D of x^2 in fp32,     r = 1/sqrt(v + eps)
//   y   = round16(x * r)                  (the normalised row in the input dtype)
//   y   = round16(y * weight)             (weight in the input dtype)
//   out = round16(y[2i] * cos - y[2i+1] * sin),  round16(y[2i+1] * cos + y[2i] * sin)
// with each fp32 product and sum rounded separately (no fused multiply-add), as
// separate elementwise ops would (the sum of squares itself is accumulated in
// its own order).  Memory-bound: 16-byte accesses, four lanes per row, rows
// ordered head-fastest so one token's cos/sin serve all its heads from L1.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace hb {
namespace {

struct PrepParams {
    const void* txt;  // [B][T][H*D] (token stride txt_sn, batch stride txt_sb, elements)
    const void* img;  // [B][n][H*D]
    int64_t txt_sb, txt_sn, img_sb, img_sn;
    int B, T, n, H;
    const void* w_txt;  // [D] or null: no normalisation
    const void* w_img;
    float eps;
    const float* cos;  // [T + n][D] in output token order, or null: no rotation
    const float* sin;
    const int32_t* image_rows;  // [n] or null: image token i -> output token T + image_rows[i]
    void* out;                  // [B][S][H][D] with strides (o_sb, o_sn, o_sh)
    int64_t o_sb, o_sn, o_sh;
    int32_t* status;            // optional: bit HB_DEV_BAD_BLOCK for an out-of-range image row
};

// 16-bit pairs <-> fp32 (round to nearest even), two elements per instruction,
// and the product of two 16-bit pairs rounded once to 16 bits (the exact
// product of two 16-bit values fits in fp32, so this equals rounding the fp32
// product, as a 16-bit elementwise multiply does).
template <bool BF16>
struct Half16;
template <>
struct Half16<true> {
    static __device__ __forceinline__ void unpack(uint32_t u, float& a, float& b) {
        a = __uint_as_float(u << 16);
        b = __uint_as_float(u & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
    static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
        __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
};
template <>
struct Half16<false> {
    static __device__ __forceinline__ void unpack(uint32_t u, float& a, float& b) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        a = f.x;
        b = f.y;
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
    static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
        __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
};

// LPR lanes per (batch, token, head) row: lane l of the group owns the 16-byte
// chunks l, l+LPR, l+2*LPR, ... of the row, so each load instruction covers
// 16*LPR contiguous bytes of every row, while the row's sum of squares needs
// log2(LPR) shuffles and the 1/sqrt runs once per D/(8*LPR) chunks.  The row
// loop bound is the same for the whole block, so the shuffles always see a
// full warp.
template <int D, bool BF16, int LPR>
__global__ void __launch_bounds__(256) k_norm_rope_pack(const __grid_constant__ PrepParams p) {
    using H16 = Half16<BF16>;
    constexpr int CPL = D / (8 * LPR);  // 16-byte chunks per lane
    constexpr int RPB = 256 / LPR;      // rows per block iteration
    const int S = p.T + p.n;
    const int rows = p.B * S * p.H;
    const int half = threadIdx.x % LPR;  // lane within the row group
    const float inv_d = 1.f / D;  // a power of two: the product equals the division
    for (int row0 = blockIdx.x * RPB; row0 < rows; row0 += gridDim.x * RPB) {
        const int row = row0 + (threadIdx.x / LPR);
        const bool valid = row < rows;
        const int rr = valid ? row : 0;
        const int tok = rr / p.H;
        const int h = rr - tok * p.H;
        const int b = tok / S;
        const int s = tok - b * S;  // input token: text [0, T), then image
        const bool text = s < p.T;
        const uint16_t* src = (text ? static_cast<const uint16_t*>(p.txt) + (int64_t)b * p.txt_sb + (int64_t)s * p.txt_sn
                                    : static_cast<const uint16_t*>(p.img) + (int64_t)b * p.img_sb +
                                          (int64_t)(s - p.T) * p.img_sn) +
                              h * D + 8 * half;
        uint4 raw[CPL];
#pragma unroll
        for (int k = 0; k < CPL; k++)
            raw[k] = valid ? *reinterpret_cast<const uint4*>(src + 8 * LPR * k) : make_uint4(0, 0, 0, 0);
        float r = 1.f;
        const uint16_t* w = static_cast<const uint16_t*>(text ? p.w_txt : p.w_img);
        if (p.w_txt) {  // both weights or neither (checked on the host): uniform
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < CPL; k++) {
                const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float a, c;
                    H16::unpack(u[i], a, c);
                    ss = fmaf(a, a, ss);
                    ss = fmaf(c, c, ss);
                }
            }
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            r = 1.f / sqrtf(__fmul_rn(ss, inv_d) + p.eps);
        }
        if (!valid) continue;
        int so = s;  // output token
        if (!text && p.image_rows) {
            const int32_t m = p.image_rows[s - p.T];
            if (m < 0 || m >= p.n) {
                if (h == 0 && half == 0 && p.status) atomicOr(p.status, HB_DEV_BAD_BLOCK);
                continue;
            }
            so = p.T + m;
        }
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (int64_t)b * p.o_sb + (int64_t)so * p.o_sn +
                        (int64_t)h * p.o_sh + 8 * half;
#pragma unroll
        for (int k = 0; k < CPL; k++) {
            const int col = 8 * LPR * k + 8 * half;  // first column of this chunk
            uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
            if (p.w_txt) {
                const uint4 wr = *reinterpret_cast<const uint4*>(w + col);
                const uint32_t wu[4] = {wr.x, wr.y, wr.z, wr.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float a, c;
                    H16::unpack(u[i], a, c);
                    u[i] = H16::mul(H16::pack(__fmul_rn(a, r), __fmul_rn(c, r)), wu[i]);
                }
            }
            if (p.cos) {
                const float4* c4 = reinterpret_cast<const float4*>(p.cos + (int64_t)so * D + col);
                const float4* s4 = reinterpret_cast<const float4*>(p.sin + (int64_t)so * D + col);
                const float4 ca = c4[0], cb = c4[1], sa = s4[0], sb = s4[1];
                const float cs[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
                const float sn[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float a, c;
                    H16::unpack(u[i], a, c);
                    u[i] = H16::pack(__fadd_rn(__fmul_rn(a, cs[2 * i]), __fmul_rn(-c, sn[2 * i])),
                                     __fadd_rn(__fmul_rn(c, cs[2 * i + 1]), __fmul_rn(a, sn[2 * i + 1])));
                }
            }
            *reinterpret_cast<uint4*>(dst + 8 * LPR * k) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
}

// Query and key heads of one token block together (hb_norm_rope_qk):
//   r = rsqrt(mean over D of x^2 + eps),  z = x * r * w,
//   (z[2i], z[2i+1]) -> (z[2i] cos[2i] - z[2i+1] sin[2i], z[2i+1] cos[2i+1] + z[2i] sin[2i+1])
// in fp32 with one rounding at the end.  Memory-bound: every row is read and
// written once.  One warp per (token, run of heads): D / 8 lanes hold a row; the
// token's cos/sin times the head weights are formed once per run and stay in
// registers over its heads,
//   out[2i] = (x r)[2i] w cos[2i] + (x r)[2i+1] (-w[2i+1] sin[2i]),  out[2i+1] likewise,
// three packed fp32 operations a pair.  What bounds it is the bytes on their way:
// four rows per lane group, four CTAs per SM (16896 tokens x 48 heads x 128: 68 us, 6.1 TB/s; with
// three CTAs 78 us, eight rows 92 us).
struct QkParams {
    const void* x[2];  // query, key: [B][S][H][D]
    void* out[2];      // may equal x
    int64_t x_sb[2], x_sn[2], x_sh[2], o_sb[2], o_sn[2], o_sh[2];
    int H[2];
    const void* w[2];      // [D] of the rows from token T on
    const void* w_txt[2];  // [D] of the rows before token T, or null (T == 0)
    const float* cos;      // [S][D]
    const float* sin;
    int B, S, T;
    int runs, run;  // head runs per token, heads per run (a run never mixes query and key heads)
    int q_runs;     // runs of the query heads
    float eps;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(256, 4) k_norm_rope_qk(const __grid_constant__ QkParams p) {
    using namespace ptx;
    using H16 = Half16<BF16>;
    constexpr int LPR = D / 8;    // lanes per row
    constexpr int RPW = 32 / LPR; // rows (heads) a warp handles at once
    constexpr int U = 4;          // row groups in flight
    const int lane = threadIdx.x & 31;
    const int col = 8 * (lane % LPR), sub = lane / LPR;
    const int64_t items = (int64_t)p.B * p.S * p.runs;
    const int64_t warps = (int64_t)gridDim.x * 8;
    for (int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); item < items; item += warps) {
        const int64_t tok = item / p.runs;
        const int run = (int)(item - tok * p.runs);
        const int b = (int)(tok / p.S), s = (int)(tok - (int64_t)b * p.S);
        const int which = run >= p.q_runs;
        const int h0 = (run - (which ? p.q_runs : 0)) * p.run;
        const int h1 = min(h0 + p.run, p.H[which]);
        const uint16_t* src = static_cast<const uint16_t*>(p.x[which]) + b * p.x_sb[which] + s * p.x_sn[which] + col;
        uint16_t* dst = static_cast<uint16_t*>(p.out[which]) + b * p.o_sb[which] + s * p.o_sn[which] + col;
        uint64_t straight[4], crossed[4];  // factors of (x[2i], x[2i+1]) and of (x[2i+1], x[2i])
        {
            const float4* c4 = reinterpret_cast<const float4*>(p.cos + (int64_t)s * D + col);
            const float4* s4 = reinterpret_cast<const float4*>(p.sin + (int64_t)s * D + col);
            const float4 ca = c4[0], cb = c4[1], sa = s4[0], sb = s4[1];
            const uint4 wr = *reinterpret_cast<const uint4*>(
                static_cast<const uint16_t*>(s < p.T ? p.w_txt[which] : p.w[which]) + col);
            const uint32_t wu[4] = {wr.x, wr.y, wr.z, wr.w};
            const float cs[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
            const float sn[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float w0, w1;
                H16::unpack(wu[i], w0, w1);
                straight[i] = f2_pack(w0 * cs[2 * i], w1 * cs[2 * i + 1]);
                crossed[i] = f2_pack(-w1 * sn[2 * i], w0 * sn[2 * i + 1]);
            }
        }
        for (int h = h0; h < h1; h += U * RPW) {  // uniform over the warp
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int hh = h + u * RPW + sub;
                raw[u] = hh < h1 ? *reinterpret_cast<const uint4*>(src + hh * p.x_sh[which]) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int hh = h + u * RPW + sub;
                const uint32_t in[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                float f[8];
                uint64_t sq = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    H16::unpack(in[i], f[2 * i], f[2 * i + 1]);
                    const uint64_t v = f2_pack(f[2 * i], f[2 * i + 1]);
                    sq = f2_fma(v, v, sq);
                }
                float ss, odd;
                f2_unpack(sq, ss, odd);
                ss += odd;
#pragma unroll
                for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float r = rsqrtf(ss * (1.f / D) + p.eps);
                const uint64_t r2 = f2_pack(r, r);
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float a, c;
                    const uint64_t t = f2_mul(f2_pack(f[2 * i], f[2 * i + 1]), r2);
                    f2_unpack(t, a, c);
                    f2_unpack(f2_fma(f2_pack(c, a), crossed[i], f2_mul(t, straight[i])), a, c);
                    o[i] = H16::pack(a, c);
                }
                if (hh < h1) *reinterpret_cast<uint4*>(dst + hh * p.o_sh[which]) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

template <bool BF16>
int launch_norm_rope_qk(const QkParams& p, int D, int grid, cudaStream_t st) {
    if (D == 32)
        k_norm_rope_qk<32, BF16><<<grid, 256, 0, st>>>(p);
    else if (D == 64)
        k_norm_rope_qk<64, BF16><<<grid, 256, 0, st>>>(p);
    else if (D == 128)
        k_norm_rope_qk<128, BF16><<<grid, 256, 0, st>>>(p);
    else
        k_norm_rope_qk<256, BF16><<<grid, 256, 0, st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" int hb_norm_rope_qk(const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, int B, int S,
                               int T, int Hq, int Hk, int D, const void* w_q, const void* w_k, const void* w_txt_q,
                               const void* w_txt_k, float eps, const float* cos, const float* sin, int dtype, void* stream) {
    if (B < 0 || S < 0 || Hq <= 0 || Hk <= 0 || T < 0 || T > S || !(eps >= 0.f)) return HB_ERR_ARG;
    if (D != 32 && D != 64 && D != 128 && D != 256) return HB_ERR_UNSUPPORTED;
    if (dtype != 0 && dtype != 1) return HB_ERR_UNSUPPORTED;
    if (B == 0 || S == 0) return HB_OK;
    if (!q || !k || !q_out || !k_out || !strides || !w_q || !w_k || !cos || !sin || (T > 0 && (!w_txt_q || !w_txt_k)))
        return HB_ERR_ARG;
    // 16-byte vector accesses: every row start and stride must keep them aligned
    for (const void* ptr : {q, k, (const void*)q_out, (const void*)k_out, w_q, w_k, T > 0 ? w_txt_q : w_q,
                            T > 0 ? w_txt_k : w_k, (const void*)cos, (const void*)sin})
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return HB_ERR_ALIGN;
    for (int i = 0; i < 12; i++)
        if (strides[i] % 8) return HB_ERR_ALIGN;
    QkParams p;
    const void* in[2] = {q, k};
    void* out[2] = {q_out, k_out};
    for (int i = 0; i < 2; i++) {
        p.x[i] = in[i];
        p.out[i] = out[i];
        const int64_t *x = strides + 3 * i, *o = strides + 6 + 3 * i;
        p.x_sb[i] = x[0], p.x_sn[i] = x[1], p.x_sh[i] = x[2];
        p.o_sb[i] = o[0], p.o_sn[i] = o[1], p.o_sh[i] = o[2];
    }
    p.H[0] = Hq, p.H[1] = Hk;
    p.w[0] = w_q, p.w[1] = w_k;
    p.w_txt[0] = w_txt_q, p.w_txt[1] = w_txt_k;
    p.cos = cos;
    p.sin = sin;
    p.B = B, p.S = S, p.T = T;
    p.eps = eps;
    int dev = 0, sms = 0;
    HB_CUDA_TRY(cudaGetDevice(&dev));
    HB_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // Heads per run: as many as leave a warp's worth of work per resident warp
    // (the run shares its cos/sin and weights), at least one group of rows.
    const int rpw = 256 / D, most = std::max(Hq, Hk);
    const int64_t warps = (int64_t)sms * 32, tokens = (int64_t)B * S;
    int run = (most + rpw - 1) / rpw * rpw;
    while (run > rpw && tokens * (((int64_t)Hq + run - 1) / run + ((int64_t)Hk + run - 1) / run) < warps)
        run = (run / 2 + rpw - 1) / rpw * rpw;
    p.run = run;
    p.q_runs = (Hq + run - 1) / run;
    p.runs = p.q_runs + (Hk + run - 1) / run;
    const int64_t want = (tokens * p.runs + 7) / 8;
    const int grid = (int)std::min<int64_t>(want, (int64_t)sms * 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == 1 ? launch_norm_rope_qk<true>(p, D, grid, st) : launch_norm_rope_qk<false>(p, D, grid, st);
}

extern "C" int hb_norm_rope_pack(const void* txt, int64_t txt_sb, int64_t txt_sn, const void* img, int64_t img_sb,
                                 int64_t img_sn, int B, int T, int n, int H, int D, const void* w_txt,
                                 const void* w_img, float eps, const float* cos, const float* sin,
                                 const int32_t* image_rows, void* out, int64_t o_sb, int64_t o_sn, int64_t o_sh,
                                 int dtype, int32_t* status, void* stream) {
    if (!out || B <= 0 || H <= 0 || T < 0 || n < 0 || T + n <= 0) return HB_ERR_ARG;
    if ((T > 0 && !txt) || (n > 0 && !img) || ((cos == nullptr) != (sin == nullptr))) return HB_ERR_ARG;
    if ((w_txt == nullptr) != (w_img == nullptr) || !(eps >= 0.f)) return HB_ERR_ARG;
    if (D != 64 && D != 128) return HB_ERR_UNSUPPORTED;
    if (dtype != 0 && dtype != 1) return HB_ERR_UNSUPPORTED;
    // 16-byte vector accesses: every row start and stride must keep them aligned
    auto a16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
    auto s8 = [](int64_t st) { return st % 8 == 0; };  // strides in 16-bit elements
    if ((txt && !a16(txt)) || (img && !a16(img)) || !a16(out) || (w_txt && (!a16(w_txt) || !a16(w_img))) ||
        (cos && (!a16(cos) || !a16(sin))) || (image_rows && (reinterpret_cast<uintptr_t>(image_rows) & 3)))
        return HB_ERR_ALIGN;
    if (!s8(txt_sb) || !s8(txt_sn) || !s8(img_sb) || !s8(img_sn) || !s8(o_sb) || !s8(o_sn) || !s8(o_sh))
        return HB_ERR_ALIGN;
    PrepParams p;
    p.txt = txt;
    p.img = img;
    p.txt_sb = txt_sb;
    p.txt_sn = txt_sn;
    p.img_sb = img_sb;
    p.img_sn = img_sn;
    p.B = B;
    p.T = T;
    p.n = n;
    p.H = H;
    p.w_txt = w_txt;
    p.w_img = w_img;
    p.eps = eps;
    p.cos = cos;
    p.sin = sin;
    p.image_rows = image_rows;
    p.out = out;
    p.o_sb = o_sb;
    p.o_sn = o_sn;
    p.o_sh = o_sh;
    p.status = status;
    int dev = 0, sms = 0;
    HB_CUDA_TRY(cudaGetDevice(&dev));
    HB_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const int64_t rows = (int64_t)B * (T + n) * H;
    if (rows > INT32_MAX / 2) return HB_ERR_UNSUPPORTED;
    constexpr int LPR = 4;  // lanes per row (measured at 2048^2: 2 -> 0.168 ms, 4 -> 0.151, 8 -> 0.167 for Q+K+V)
    const int64_t want = (rows + 256 / LPR - 1) / (256 / LPR);
    const int grid = (int)(want < (int64_t)sms * 8 ? want : (int64_t)sms * 8);
    cudaStream_t st = (cudaStream_t)stream;
    if (D == 128) {
        if (dtype == 1)
            k_norm_rope_pack<128, true, LPR><<<grid, 256, 0, st>>>(p);
        else
            k_norm_rope_pack<128, false, LPR><<<grid, 256, 0, st>>>(p);
    } else {
        if (dtype == 1)
            k_norm_rope_pack<64, true, LPR><<<grid, 256, 0, st>>>(p);
        else
            k_norm_rope_pack<64, false, LPR><<<grid, 256, 0, st>>>(p);
    }
    HB_LAUNCH_CHECK();
    return HB_OK;
}
