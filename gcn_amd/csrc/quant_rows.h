// 8-bit rows with a scale each: element (r, c) of the matrix is scales[r] * e4m3(q[r * ldq + c]).  The pitch is a
// multiple of 16 bytes and the bytes from f to the next multiple of 16 are zero, so that a product reads rows in whole
// 16-byte pieces.  e4m3 (4 exponent bits, 3 mantissa bits, bias 7, no infinity, largest value 448) is the form whose
// conversions the hardware has: two values an instruction in either direction, rounded to nearest even.
#pragma once

#include "common.h"

namespace gcn {

constexpr float kE4m3Max = 448.0f;
// the smallest scale (2^-120): its inverse is finite, and an all-zero row needs no case of its own
constexpr float kQuantScaleMin = 7.52316384526264e-37f;

// Row pitch in bytes: a power of two up to 128 (rows never straddle a 128-byte line), then a multiple of 64.
static inline int64_t quant_pitch(int64_t f) {
    int64_t p = 16;
    while (p < f && p < 128) p *= 2;
    return f <= p ? p : (f + 63) / 64 * 64;
}

// four values as e4m3 bytes, the first `kept` of them (the others 0).  The caller's values are at most 448 in magnitude
// up to a rounding, which the conversion takes back to 448; NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d, int kept) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return kept >= 4 ? (uint32_t)r : kept <= 0 ? 0u : (uint32_t)r & ((1u << (8 * kept)) - 1u);
}

}  // namespace gcn
