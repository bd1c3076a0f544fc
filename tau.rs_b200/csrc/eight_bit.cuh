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

// One warp: norm and rotation of one head, in place (shared memory).
__device__ __forceinline__ void prepare_row(bf16* row, const float* __restrict__ weight, float eps, const float* __restrict__ cosines, const float* __restrict__ sines, int rotary_dim, int D,
                                            int lane) {
    if (weight) {
        float squares = 0.0f;
        // In the order of the 16-bit cache's prepare kernel, so that a key is the same before it is rounded to 8 bits: neighbours to a lane in heads of 64, 128 and 256 that are rotated
        // whole or not at all, else strides of 32.
        const bool neighbours = (D == 64 || D == 128 || D == 256) && (rotary_dim == 0 || rotary_dim == D);
        const int per = neighbours ? D / 32 : 1, begin = per > 1 ? lane * per : lane, end = per > 1 ? begin + per : D, by = per > 1 ? 1 : 32;
        for (int e = begin; e < end; e += by) {
            const float value = to_float(row[e]);
            squares += value * value;
        }
        const float inverse = rsqrtf(warp_sum(squares) / static_cast<float>(D) + eps);
        for (int e = lane; e < D; e += 32) row[e] = __float2bfloat16_rn(to_float(row[e]) * inverse * weight[e]);
        __syncwarp();
    }
    const int half = rotary_dim / 2;
    for (int j = lane; j < half; j += 32) {      // a pair is one lane's
        const float first = to_float(row[j]), second = to_float(row[j + half]), c = cosines[j], s = sines[j];
        // Which product is rounded before the sum is fixed, so that every kernel that prepares a row leaves the same bits.
        row[j] = __float2bfloat16_rn(__fmaf_rn(first, c, -__fmul_rn(second, s)));
        row[j + half] = __float2bfloat16_rn(__fmaf_rn(second, c, __fmul_rn(first, s)));
    }
    __syncwarp();
}

// The same of a head of 32 PER elements that is rotated whole (`rotated`) or not at all, in registers: a lane holds PER neighbours, `weight` theirs, `cosines` and `sines` those of
// elements PER (lane % 16) + i of the half-wide tables.
template <int PER>
struct alignas(2 * PER) Neighbours {
    bf16 v[PER];
};
template <int PER>
__device__ __forceinline__ Neighbours<PER> prepare_neighbours(const Neighbours<PER>& raw, bool normed, const float* weight, float eps, bool rotated, const float* cosines, const float* sines,
                                                              int lane) {
    float value[PER], squares = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        value[i] = to_float(raw.v[i]);
        squares += value[i] * value[i];
    }
    if (normed) {
        const float inverse = rsqrtf(warp_sum(squares) / static_cast<float>(32 * PER) + eps);
#pragma unroll
        for (int i = 0; i < PER; ++i) value[i] = round_through<bf16>(value[i] * inverse * weight[i]);
    }
    Neighbours<PER> result;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        // First half of the head: x cos - partner sin; second half: x cos + partner sin.
        const float partner = __shfl_xor_sync(0xffffffffu, value[i], 16), turned = __fmul_rn(partner, sines[i]);
        result.v[i] = from_float<bf16>(rotated ? __fmaf_rn(value[i], cosines[i], lane < 16 ? -turned : turned) : value[i]);
    }
    return result;
}

// `Threads` threads of a block (its first ones, or, with 0, all of it) bring `count` rows of D elements in shared memory into a page of one head, behind the `older`
// positions that it holds: the scale is the page's own (none for a page that starts here) or what the new rows need, whichever is greater, and codes that are there are rounded to
// one that grew.  Returns the page's scale, which one thread then writes to `scale_at`; every thread has read the old one by then.  `greatest_of`: a float for each warp.
template <int Threads = 0>
__device__ __forceinline__ float store_in_page(const bf16* rows, int count, int D, int older, uint8_t* page, const float* scale_at, float* greatest_of) {
    const int threads = Threads == 0 ? static_cast<int>(blockDim.x) : Threads;
    auto meet = [&]() {
        if constexpr (Threads == 0) __syncthreads();
        else asm volatile("bar.sync 1, %0;" ::"n"(Threads) : "memory");
    };
    float greatest = 0.0f;
    for (int piece = threadIdx.x; piece < count * D / 8; piece += threads) {
        const uint4 raw = reinterpret_cast<const uint4*>(rows)[piece];
        const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) greatest = fmaxf(greatest, fmaxf(finite_magnitude(__uint_as_float(words[i] << 16)), finite_magnitude(__uint_as_float(words[i] & 0xffff0000u))));
    }
    const float kept = older > 0 ? fmaxf(*scale_at, kLeastScale) : 0.0f;
    greatest = warp_max(greatest);
    if ((threadIdx.x & 31) == 0) greatest_of[threadIdx.x >> 5] = greatest;
    meet();
    for (int w = 0; w < threads / 32; ++w) greatest = fmaxf(greatest, greatest_of[w]);
    float scale = power_of_two(scale_exponent(greatest));
    if (kept >= scale) {
        scale = kept;
    } else if (older > 0) {
        const float ratio = kept / scale;      // powers of two
        for (int piece = threadIdx.x; piece < older * D / 4; piece += threads) {
            unsigned* word = reinterpret_cast<unsigned*>(page) + piece;
            float v[4];
            decode_four(*word, v);
            *word = encode_four(v[0], v[1], v[2], v[3], ratio);
        }
    }
    const float inverse = 1.0f / scale;
    for (int piece = threadIdx.x; piece < count * D / 8; piece += threads) {
        const uint4 raw = reinterpret_cast<const uint4*>(rows)[piece];
        const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
        uint2 codes;
        codes.x = encode_four(__uint_as_float(words[0] << 16), __uint_as_float(words[0] & 0xffff0000u), __uint_as_float(words[1] << 16), __uint_as_float(words[1] & 0xffff0000u), inverse);
        codes.y = encode_four(__uint_as_float(words[2] << 16), __uint_as_float(words[2] & 0xffff0000u), __uint_as_float(words[3] << 16), __uint_as_float(words[3] & 0xffff0000u), inverse);
        *reinterpret_cast<uint2*>(page + static_cast<size_t>(older) * D + piece * 8) = codes;
    }
    return scale;
}

}  // namespace
