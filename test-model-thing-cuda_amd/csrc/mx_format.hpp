// mx_format.hpp -- microscaled (MX) numbers on gfx950: blocks of 32 values
// that share one e8m0 scale byte s, 2^(s - 127), s = 255 being NaN.
#pragma once
#include "device_util.hpp"

namespace tmt {

enum MxFormat { MX_FP4 = 0, MX_FP8 = 1 };  // e2m1 codes, two a byte; e4m3 codes

// 2^(s - 127) in fp32; s = 0 is the subnormal 2^-127.
__device__ __forceinline__ float e8m0_value(uint32_t s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23);
}

// The scale operand of the scaled conversions, which read its exponent field
// as an e8m0 byte: 0 is 2^-127 there and 255 NaN.
__device__ __forceinline__ float e8m0_operand(uint32_t s) { return __uint_as_float(s << 23); }

// Scale byte of a block whose largest |value| has the fp32 bits `amax` (an
// integer maximum of the bits without the sign, so inf and NaN come out on
// top). Blocks of zeros take 127; a block with an inf or NaN takes 255.
//   MXFP4: exponent floor(log2 amax) - 2, the largest value in [4, 8), which
//          saturates at 6 (the format of the expert weights);
//   MXFP8: the smallest exponent with amax <= 448 * 2^e, so that nothing
//          saturates and every rounding is at most half a step.
// Exponents are at least -127; fp32 subnormals are below 2^-126 and get that.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax) {
    const int be = (int)(amax >> 23);
    if (be == 255) return 255;
    if (amax == 0) return 127;
    const int s = FMT == MX_FP4 ? be - 2 : be - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(s, 0);
}
// 1 / 2^(s - 127) for the scales that mx_scale gives a finite block (0 .. 252).
__device__ __forceinline__ float mx_inverse(uint32_t s) { return __uint_as_float((254 - s) << 23); }

// Eight scaled values to e2m1 codes, element i in bits 4i .. 4i + 3.
__device__ __forceinline__ uint32_t to_e2m1(const float* v) {
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], 1.0f, 3);
    return q;
}
// Four scaled values to e4m3 codes, one a byte.
__device__ __forceinline__ uint32_t to_e4m3(const float* v) {
    int q = 0;
    q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], q, false);
    q = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
    return (uint32_t)q;
}

// The values of codes at scale 1, in fp32.
__device__ __forceinline__ void from_e2m1(uint32_t q, float* v) {
    const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
    const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2);
    const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}
__device__ __forceinline__ void from_e4m3(uint32_t q, float* v) {
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false);
    const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
}

}  // namespace tmt
