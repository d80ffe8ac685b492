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
#include <algorithm>
#include <climits>
#include <cstdint>
#include <mutex>

#include "int8_common.cuh"

namespace hb {

namespace {
std::mutex g_mu;
DeviceInfo g_dev[64];
}  // namespace

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

int current_device(int* dev) {
    HB_CUDA_TRY(cudaGetDevice(dev));
    return *dev < 64 ? HB_OK : HB_ERR_UNSUPPORTED;
}

namespace {

constexpr unsigned FULL = 0xffffffffu;

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
    ptx::grid_launch_dependents();  // the product's CTAs may set themselves up meanwhile
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
    ptx::grid_launch_dependents();
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
    if (M > 1 << 30 || N > 1 << 30 || ceil_div(M, 128) * ceil_div(N, 128) > INT32_MAX / 8) return HB_ERR_UNSUPPORTED;
    return HB_OK;
}

int linear(const Int8Problem& p, bool few, bool early_weights, cudaStream_t st) {
    int dev = 0, rc;
    DeviceInfo di;
    if ((rc = current_device(&dev)) || (rc = device_info(dev, &di))) return rc;
    return few ? launch_int8_few(p, di, st) : launch_int8_gemm(p, dev, di, early_weights, st);
}
}  // namespace
}  // namespace hb

extern "C" int hb_int8_linear(const int8_t* x, int64_t x_rs, const float* x_scales, const int8_t* w, int64_t w_rs,
                              const float* w_scales, const void* bias, void* out, int64_t out_rs, int M, int N, int K,
                              int act, int dtype, void* stream) {
    const int rc = check_linear(x, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype);
    if (rc) return rc > 0 ? HB_OK : rc;
    if (!x_scales || (M > 1 && x_rs < K)) return HB_ERR_ARG;
    if (!aligned(x, 16) || (M > 1 && x_rs % 16) || !aligned(x_scales, 4)) return HB_ERR_ALIGN;
    const Int8Problem p{x, x_rs, x_scales, w, w_rs, w_scales, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out),
                        out_rs, M, N, K, act, dtype};
    return linear(p, int8_few_takes(M, K), false, static_cast<cudaStream_t>(stream));
}

extern "C" size_t hb_int8_linear16_workspace_bytes(int M, int K) {
    if (M <= 0 || K <= 0 || K > HB_INT8_MAX_K || int8_few_takes(M, K)) return 0;
    return (size_t)(code_pitch(K) * M + 4 * (int64_t)M);
}

extern "C" int hb_int8_linear16(const void* x, int64_t x_rs, const int8_t* w, int64_t w_rs, const float* w_scales,
                                const void* bias, void* out, int64_t out_rs, int M, int N, int K, int act, int dtype,
                                void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_linear(x, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype);
    if (rc) return rc > 0 ? HB_OK : rc;
    if (!aligned(x, 2)) return HB_ERR_ALIGN;
    const size_t need = hb_int8_linear16_workspace_bytes(M, K);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return HB_ERR_WORKSPACE;
    Int8Problem p{x, x_rs, nullptr, w, w_rs, w_scales, static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out),
                  out_rs, M, N, K, act, dtype};
    if (need) {
        int8_t* codes = static_cast<int8_t*>(workspace);
        float* scales = reinterpret_cast<float*>(codes + code_pitch(K) * M);
        if ((rc = hb_quantize_rows(x, x_rs, K, nullptr, 0, 0, M, codes, code_pitch(K), scales, dtype, stream))) return rc;
        p.x = codes;
        p.x_rs = code_pitch(K);
        p.x_scales = scales;
    }
    // The kernel before the product is the quantisation, an ordinary launch that does
    // not write the weights: they are final when it starts.
    return linear(p, !need, need != 0, static_cast<cudaStream_t>(stream));
}
