// Activations brought to e4m3 codes with a scale for each row and 128 columns: the kernel and its launch, for the products that quantise within their call.
#pragma once
#include "eight_bit.cuh"

#include <type_traits>

namespace {

// Half a warp to 128 columns of a row, eight values to a lane, kAhead such blocks one after another with all their loads on their way first.  scales[block of columns][row].
// Bound by memory: 2,048 x 4,096 bfloat16 values 7.8 us at four, 11 at one; where there are few blocks one at a time gives more SMs work.
template <typename T, int kAhead>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ values, long long stride, uint8_t* __restrict__ codes, float* __restrict__ scales, int rows, int columns, int across) {
    grid_dependents_launch();
    grid_dependency_wait();
    typedef typename std::conditional<sizeof(T) == 2, uint4, float4>::type Vector;
    constexpr int kVectors = sizeof(T) * 8 / 16;
    const int place = threadIdx.x & 15;
    const long long items = static_cast<long long>(rows) * across, first = static_cast<long long>(blockIdx.x) * (16 * kAhead) + (threadIdx.x >> 4);
    Vector held[kAhead][kVectors];
    bool live[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const long long item = first + 16 * a;
        const int row = static_cast<int>(item / across), column = static_cast<int>(item % across) * kScaleBlock + place * 8;
        live[a] = item < items && column < columns;      // columns are a multiple of 16: a group of eight is whole or absent
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
            held[a][v] = live[a] ? __ldg(reinterpret_cast<const Vector*>(values + static_cast<size_t>(row) * stride + column) + v) : Vector{};
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const long long item = first + 16 * a;
        float x[8];
        if constexpr (sizeof(T) == 2) {
            const unsigned* words = reinterpret_cast<const unsigned*>(held[a]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(words[i] << 16);
                x[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const float*>(held[a])[i];
        }
        float greatest = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) greatest = fmaxf(greatest, finite_magnitude(x[i]));
#pragma unroll
        for (int offset = 8; offset > 0; offset >>= 1) greatest = fmaxf(greatest, __shfl_xor_sync(0xffffffffu, greatest, offset));
        if (item >= items) continue;      // the shuffles above stay within halves of the warp
        const int row = static_cast<int>(item / across), block = static_cast<int>(item % across);
        const int exponent = scale_exponent(greatest);
        const float inverse = power_of_two(-exponent);
        if (place == 0) scales[static_cast<size_t>(block) * rows + row] = power_of_two(exponent);
        if (live[a])
            *reinterpret_cast<uint2*>(codes + static_cast<size_t>(row) * columns + block * kScaleBlock + place * 8) =
                make_uint2(encode_four(x[0], x[1], x[2], x[3], inverse), encode_four(x[4], x[5], x[6], x[7], inverse));
    }
}

// Codes [rows, columns] (contiguous) and scales [blocks of columns, rows]; columns a multiple of 16, rows of values on 16-byte borders.
inline int launch_quantize_rows(int dtype, const void* values, long long stride, void* codes, float* scales, int rows, int columns, cudaStream_t s) {
    if (rows <= 0 || columns <= 0) return 0;
    const int across = (columns + kScaleBlock - 1) / kScaleBlock;
    const long long items = static_cast<long long>(rows) * across;
    const int ahead = items <= 32768 ? 1 : 4;
    const long long blocks = (items + 16 * ahead - 1) / (16 * ahead);
    if (!values || !codes || !scales || (columns & 15) || (stride & 7) || (reinterpret_cast<uintptr_t>(values) & 15) || (dtype != TAU_BF16 && dtype != TAU_F32) || blocks > 0x7fffffffll)
        return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks));
    uint8_t* bytes = static_cast<uint8_t*>(codes);
    if (dtype == TAU_BF16) {
        const bf16* from = static_cast<const bf16*>(values);
        if (ahead == 1) tau_launch(quantize_rows_kernel<bf16, 1>, grid, dim3(256), 0, s, from, stride, bytes, scales, rows, columns, across);
        else tau_launch(quantize_rows_kernel<bf16, 4>, grid, dim3(256), 0, s, from, stride, bytes, scales, rows, columns, across);
    } else {
        const float* from = static_cast<const float*>(values);
        if (ahead == 1) tau_launch(quantize_rows_kernel<float, 1>, grid, dim3(256), 0, s, from, stride, bytes, scales, rows, columns, across);
        else tau_launch(quantize_rows_kernel<float, 4>, grid, dim3(256), 0, s, from, stride, bytes, scales, rows, columns, across);
    }
    return tau_launch_status();
}

// `held`, 16-byte aligned: rows * columns codes and, behind them, a float for each row and block of columns.
inline float* scales_behind(void* held, int rows, int columns) { return reinterpret_cast<float*>(static_cast<uint8_t*>(held) + static_cast<size_t>(rows) * columns); }

}  // namespace
