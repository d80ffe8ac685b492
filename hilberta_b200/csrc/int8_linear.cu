// Linear layers in 8-bit integers: rows of 16-bit values quantised with one scale
// a row, and the product of two such matrices with scales, bias and activation.
//
//   scale_m = max_k |x_mk| / 127            code_mk = rint(x_mk * (127 / max_k |x_mk|))
//   y_mn = act(((sum_k xcode_mk * wcode_nk) * xscale_m) * wscale_n + bias_n)
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

// Thread t of T's share i of a row: eight values in 8 / W loads of W neighbours, and
// where their codes go.  W is the widest load that the rows' starts, ka and k allow
// (8: 16 bytes, its codes one 8-byte store); a warp's loads and stores are contiguous
// for every W.  Zeros past the end of the row.  8000 rows of 14308:
// W = 4 56.7 us, W = 1 163.6; of 1802: W = 2 19.0, W = 1 31.7.
template <int W, int T>
__device__ __forceinline__ int column(int t, int i, int e) { return W * ((i * (8 / W) + e) * T + t); }

template <int W, int T>
__device__ __forceinline__ uint4 load8(const QuantParams& p, int64_t row, int t, int i) {
    const uint16_t *a = p.a + row * p.a_rs, *b = p.b + row * p.b_rs;
    uint32_t w[8] = {};  // W = 1: a value each, else pairs
#pragma unroll
    for (int e = 0; e < 8 / W; e++) {
        const int c = column<W, T>(t, i, e);
        const uint16_t* src = c < p.ka ? a + c : b + (c - p.ka);
        if (c < p.k && row < p.rows) {
            if constexpr (W == 8) return *reinterpret_cast<const uint4*>(src);
            if constexpr (W == 4) reinterpret_cast<uint2*>(w)[e] = *reinterpret_cast<const uint2*>(src);
            if constexpr (W == 2) w[e] = *reinterpret_cast<const uint32_t*>(src);
            if constexpr (W == 1) w[e] = __ldg(src);
        }
    }
    if constexpr (W == 1) return make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int W, int T>
__device__ __forceinline__ void store8(const QuantParams& p, int64_t row, int t, int i, uint2 codes) {
    int8_t* out = p.codes + row * p.c_rs;
#pragma unroll
    for (int e = 0; e < 8 / W; e++) {
        const int c = column<W, T>(t, i, e);
        const uint32_t word = e * W < 4 ? codes.x : codes.y;
        if (c < p.k) {
            if constexpr (W == 8) *reinterpret_cast<uint2*>(out + c) = codes;
            if constexpr (W == 4) *reinterpret_cast<uint32_t*>(out + c) = word;
            if constexpr (W == 2) *reinterpret_cast<uint16_t*>(out + c) = (uint16_t)(word >> (16 * (e & 1)));
            if constexpr (W == 1) out[c] = (int8_t)(word >> (8 * (e & 3)));
        }
    }
}

// T threads per row (a warp of four, or the whole CTA), up to kQuantVec vectors of 8
// values each: the row is read once and stays in registers between its maximum
// and its codes.  Memory-bound (2 K bytes read, K written per row): a CTA goes over
// several rows, and each thread fetches its part of the next row before it works on
// this one, so loads are in flight through the reduction and the stores.
constexpr int kQuantVec = 4;

template <bool BF16, int W, int T>
__global__ void __launch_bounds__(T == 32 ? 128 : T) k_quantize_rows(const __grid_constant__ QuantParams p) {
    constexpr int CTA = T == 32 ? 128 : T;
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
        for (int i = 0; i < NV; i++) next[i] = load8<W, T>(p, r, t, i);
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
        for (int i = 0; i < NV; i++) store8<W, T>(p, row, t, i, codes8<BF16>(v[i], s));
    }
}

// Rows too long for a CTA's registers: one CTA per row, read twice.
template <bool BF16, int W>
__global__ void __launch_bounds__(512) k_quantize_long(const __grid_constant__ QuantParams p) {
    __shared__ uint32_t s_max[16];
    const int64_t row = blockIdx.x;
    ptx::grid_launch_dependents();
    const int n = (p.k + 8 * 512 - 1) / (8 * 512);
    uint32_t m = 0;
#pragma unroll 4
    for (int i = 0; i < n; i++) m = max_mag(m, load8<W, 512>(p, row, threadIdx.x, i));
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
        store8<W, 512>(p, row, threadIdx.x, i, codes8<BF16>(load8<W, 512>(p, row, threadIdx.x, i), s));
}

template <bool BF16, int W>
int launch_quantize(const QuantParams& p, int sms, cudaStream_t st) {
    // Threads per row: the fewest of these whose registers hold it (8192 x 2048: 8.7 us
    // with 64, 13.5 with 128; 16384 x 3072: 23.8 us with 96, 25.4 with 128; 8192 x 5120:
    // 20.6 us with 160, 21.9 with 192; 8192 x 14336: the same with 448 and 512; a number only
    // known at run time costs a quarter more than any).  CTAs: as many as fill the SMs' 2048
    // threads, which is more than their registers let be resident (56 to 64 a thread for
    // W = 8: about half, 80 to 97 for W = 1: a third or a quarter), so they come in that
    // many rounds, and a dependent launch starts with the last of them.
    const int64_t warps = ceil_div(p.k, 8 * kQuantVec * 32);
    auto start = [&](auto kern, int cta, int rows) {
        kern<<<(unsigned)std::min<int64_t>(ceil_div(p.rows, rows), (int64_t)sms * (2048 / cta)), cta, 0, st>>>(p);
    };
    if (warps <= 1)
        start(k_quantize_rows<BF16, W, 32>, 128, 4);
    else if (warps <= 2)
        start(k_quantize_rows<BF16, W, 64>, 64, 1);
    else if (warps <= 3)
        start(k_quantize_rows<BF16, W, 96>, 96, 1);
    else if (warps <= 4)
        start(k_quantize_rows<BF16, W, 128>, 128, 1);
    else if (warps <= 5)
        start(k_quantize_rows<BF16, W, 160>, 160, 1);
    else if (warps <= 6)
        start(k_quantize_rows<BF16, W, 192>, 192, 1);
    else if (warps <= 8)
        start(k_quantize_rows<BF16, W, 256>, 256, 1);
    else if (warps <= 10)
        start(k_quantize_rows<BF16, W, 320>, 320, 1);
    else if (warps <= 12)
        start(k_quantize_rows<BF16, W, 384>, 384, 1);
    else if (warps <= 16)
        start(k_quantize_rows<BF16, W, 512>, 512, 1);
    else
        k_quantize_long<BF16, W><<<p.rows, 512, 0, st>>>(p);
    HB_LAUNCH_CHECK();
    return HB_OK;
}
template <bool BF16>
int launch_quantize(const QuantParams& p, uint64_t at, int sms, cudaStream_t st) {
    if (at % 8 == 0) return launch_quantize<BF16, 8>(p, sms, st);
    if (at % 4 == 0) return launch_quantize<BF16, 4>(p, sms, st);
    if (at % 2 == 0) return launch_quantize<BF16, 2>(p, sms, st);
    return launch_quantize<BF16, 1>(p, sms, st);
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
    // Elements that every load may take at once: a power of two dividing where rows and parts start.
    uint64_t at = reinterpret_cast<uintptr_t>(a) / 2 | (uint64_t)ka | (rows > 1 ? (uint64_t)a_rs : 0);
    if (kb) at |= reinterpret_cast<uintptr_t>(b) / 2 | (uint64_t)kb | (rows > 1 ? (uint64_t)b_rs : 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int dev = 0, rc;
    DeviceInfo di;
    if ((rc = current_device(&dev)) || (rc = device_info(dev, &di))) return rc;
    return dtype == 1 ? launch_quantize<true>(p, at, di.sms, st) : launch_quantize<false>(p, at, di.sms, st);
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
    return linear(p, int8_few_takes(M, N, K), false, static_cast<cudaStream_t>(stream));
}

extern "C" size_t hb_int8_linear16_workspace_bytes(int M, int K) {
    if (M <= 0 || K <= 0 || K > HB_INT8_MAX_K || int8_few_takes(M, INT32_MAX, K)) return 0;
    return (size_t)(code_pitch(K) * M + 4 * (int64_t)M);
}

extern "C" int hb_int8_linear16(const void* x, int64_t x_rs, const int8_t* w, int64_t w_rs, const float* w_scales,
                                const void* bias, void* out, int64_t out_rs, int M, int N, int K, int act, int dtype,
                                void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_linear(x, w, w_rs, w_scales, bias, out, out_rs, M, N, K, act, dtype);
    if (rc) return rc > 0 ? HB_OK : rc;
    if (!aligned(x, 2)) return HB_ERR_ALIGN;
    const size_t need = int8_few_takes(M, N, K) ? 0 : hb_int8_linear16_workspace_bytes(M, K);
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
