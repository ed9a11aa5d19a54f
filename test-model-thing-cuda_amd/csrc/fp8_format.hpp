// fp8_format.hpp -- blocks of e4m3 codes with one fp32 scale.
//
// With m the block's largest magnitude, and at least 2^-100 (so that a block of
// zeros and one of fp32 subnormals have a scale and its inverse in fp32's normal
// range): code = e4m3(x * (448 / m)), scale = m / 448. Both quotients and the
// product are rounded to fp32 once; the code is at most half a step of e4m3 off.
#pragma once
#include "device_util.hpp"
#include "mx_format.hpp"

namespace tmt {

struct Fp8Scale {
    float scale, inv;
};
// From the fp32 bits of the largest |value| (an integer maximum of the bits
// without the sign, so an infinity or NaN comes out on top: the scale is NaN
// and the codes are zeros).
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t amax) {
    const float m = __uint_as_float(max(amax, 0x0d800000u));  // 2^-100
    const bool bad = amax >= 0x7f800000u;
    return {bad ? __uint_as_float(0x7fc00000u) : m / 448.0f, bad ? 0.0f : 448.0f / m};
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// How a kernel passes memory: kCached; kStoreOnce, whose stores are non-temporal; or
// kOnce, whose loads of its large inputs are as well.
enum { kCached, kStoreOnce, kOnce };
template <int PASS, class T>
__device__ __forceinline__ void put(void* p, T v) {
    if constexpr (PASS != kCached) __builtin_nontemporal_store(v, static_cast<T*>(p));
    else *static_cast<T*>(p) = v;
}
template <int PASS, class T>
__device__ __forceinline__ T get(const void* p) {
    if constexpr (PASS == kOnce) return __builtin_nontemporal_load(static_cast<const T*>(p));
    else return *static_cast<const T*>(p);
}
__device__ __forceinline__ float fp8_scaled(float v, float inv) {
    return inv == 0.0f ? 0.0f : v * inv;  // inv is 0 for a block that is NaN
}
// Codes of four values, one a byte.
__device__ __forceinline__ uint32_t fp8_codes(const float* v, float inv) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = fp8_scaled(v[i], inv);
    return to_e4m3(q);
}

}  // namespace tmt
