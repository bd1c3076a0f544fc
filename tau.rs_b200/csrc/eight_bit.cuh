// What the kernels of weights and caches in 8 bits share: the rule of scales and the conversions from and to e4m3.
//
// A block of values (128 x 128 of a weight, 128 of a row of activations, 64 positions of a head in the cache) is held as codes `x / s`
// rounded to e4m3 (nearest, ties to even) with s = 2^e the least power of two from 2^-120 on with max |x| <= 448 s, 448 being the
// greatest e4m3 number.  e4m3 has a sign, 4 bits of exponent and 3 of mantissa, so a scale that is no power of two would not make a
// code more exact; with a power of two the division is exact and the only rounding is that of the code itself, the same in 32 and in 64
// bits.  What is not finite takes no part in the scale and becomes e4m3's NaN.
#pragma once
#include "common.cuh"

namespace {

constexpr int kScaleBlock = 128;      // rows and columns of a weight, columns of an activation row, to a scale
constexpr int kLeastExponent = -120;
constexpr float kLeastScale = 7.52316384526264e-37f;      // 2^-120

// The exponent of the scale of a block whose greatest finite magnitude is `greatest`: 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float greatest) {
    const unsigned bits = __float_as_uint(greatest);
    const int exponent = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(exponent, kLeastExponent);      // zero and what is subnormal in 32 bits as well
}
// 2^exponent, for exponents from -126 to 127.
__device__ __forceinline__ float power_of_two(int exponent) { return __uint_as_float(static_cast<unsigned>(exponent + 127) << 23); }

__device__ __forceinline__ float finite_magnitude(float value) {
    const float magnitude = fabsf(value);
    return magnitude <= 3.402823466e38f ? magnitude : 0.0f;      // NaN compares false as well
}

// Two values times a power of two as e4m3 codes, the first in the low byte.  (The conversion saturates, so infinities are made NaN first.)
__device__ __forceinline__ unsigned encode_pair(float low, float high, float inverse) {
    low = fabsf(low) <= 3.402823466e38f ? low * inverse : __uint_as_float(0x7fffffffu);
    high = fabsf(high) <= 3.402823466e38f ? high * inverse : __uint_as_float(0x7fffffffu);
    unsigned short codes;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(codes) : "f"(high), "f"(low));
    return codes;
}
__device__ __forceinline__ unsigned encode_four(float a, float b, float c, float d, float inverse) {
    return encode_pair(a, b, inverse) | (encode_pair(c, d, inverse) << 16);
}

// Two codes (the low 16 bits) as two 16-bit floats: exact, e4m3's numbers are numbers of that type.
__device__ __forceinline__ unsigned decode_half2(unsigned codes) {
    unsigned halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(static_cast<unsigned short>(codes)));
    return halves;
}
__device__ __forceinline__ float half_to_float(unsigned short half) {
    float value;
    asm("cvt.f32.f16 %0, %1;" : "=f"(value) : "h"(half));
    return value;
}
// The four codes of a word as 32-bit floats.
__device__ __forceinline__ void decode_four(unsigned word, float (&out)[4]) {
    const unsigned low = decode_half2(word), high = decode_half2(word >> 16);
    out[0] = half_to_float(static_cast<unsigned short>(low));
    out[1] = half_to_float(static_cast<unsigned short>(low >> 16));
    out[2] = half_to_float(static_cast<unsigned short>(high));
    out[3] = half_to_float(static_cast<unsigned short>(high >> 16));
}

__device__ __forceinline__ unsigned pack_bf16_pair(float low, float high) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const unsigned*>(&pair);
}

}  // namespace
