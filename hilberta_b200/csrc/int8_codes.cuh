// Quantisation of a row of values to 8-bit codes with one scale:
//   scale = max|x| / 127,   code = rint(x * (127 / max|x|))   (ties to even).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace hb {

// A row's scale and the factor its values are multiplied with.  A row holding an
// infinity or NaN gets the scale NaN (every output of the row becomes NaN) and
// codes 0; a row below 2^-100 counts as zeros (127 / max would overflow).
struct RowScale {
    float scale, inv;
    bool live;  // codes are not all 0 by the rules above
};
__device__ __forceinline__ RowScale row_scale(float amax) {
    RowScale r;
    r.live = amax >= 0x1p-100f && amax <= 3.402823466e38f;
    r.scale = r.live ? __fdiv_rn(amax, 127.f) : (amax < 0x1p-100f ? 0.f : __uint_as_float(0x7fc00000u));
    r.inv = r.live ? __fdiv_rn(127.f, amax) : 0.f;
    return r;
}

// The code of x in the low byte: x * inv rounded to fp32, then to the nearest
// integer by adding 1.5 * 2^23, whose low byte is the integer's two's complement.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) {
    return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f));
}
__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace hb
