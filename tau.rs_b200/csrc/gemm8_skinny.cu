// Product for a few rows of activations with the weight in 8 bits: out[M, N] = x[M, K] * w[N, K]^T + bias, M <= 32, bound by reading `w` once.
//
// Weight codes are e4m3 with a 32-bit scale for each 128 x 128 block, activations e4m3 with a scale for each row and 128 columns, so
//     out[m, n] = sum over blocks b of 128 columns: x_scale[b][m] * w_scale[n / 128][b] * (sum over the block of codes),
// and a chunk of 128 columns is a warp's unit: four mma.sync m16n8k32 on e4m3 operands with 32-bit sums, the weight's rows as A and the
// activations as B, then one multiplication of the chunk's sums by both scales.
//
// A block owns 16 output features; its 8 warps take interleaved chunks and keep up to 4 of them (2 KB each) on their way by cp.async in whole
// lines, 64 KB to a block and three blocks to an SM.  Up to 8 rows the activations come in bfloat16 and each warp quantises the chunk that it
// needs itself: a launch of its own for so few values would take longer than the whole product of a small layer.  (The lanes of a row hold a chunk
// between them, so its greatest magnitude is two shuffles away.)  More rows come quantised.
//
// Needs K % 16 == 0 and contiguous codes on a 16-byte border.
#include "eight_bit.cuh"

namespace {

constexpr int kRows = 16;        // output features to a block
constexpr int kWarps = 8;
constexpr int kDepth = 4;        // chunks on their way per warp
constexpr int kChunk = kScaleBlock;

__device__ __forceinline__ void mma_e4m3(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy_async_16(void* destination, const void* source, bool real) {
    const unsigned address = static_cast<unsigned>(__cvta_generic_to_shared(destination));
    const int bytes = real ? 16 : 0;   // 0 source bytes: the 16 destination bytes become zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(address), "l"(source), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The 32 values that a lane holds of a row's chunk (two pieces of 16 columns), quantised with the four lanes of the row: 8 words of codes; returns the scale.
__device__ __forceinline__ float quantize_chunk(const uint4 (&raw)[4], unsigned (&codes)[8]) {
    const unsigned* words = reinterpret_cast<const unsigned*>(raw);
    unsigned greatest = 0;      // bit patterns of magnitudes order as the magnitudes do
#pragma unroll
    for (int i = 0; i < 16; ++i) greatest = __vmaxu2(greatest, words[i] & 0x7fff7fffu);
    greatest = max(greatest >> 16, greatest & 0xffffu);
    greatest = max(greatest, __shfl_xor_sync(0xffffffffu, greatest, 1));
    greatest = max(greatest, __shfl_xor_sync(0xffffffffu, greatest, 2));
    const bool odd = greatest >= 0x7f80u;      // an infinity or a NaN is among them
    if (__any_sync(0xffffffffu, odd)) {
        float finite = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) finite = fmaxf(finite, fmaxf(finite_magnitude(__uint_as_float(words[i] << 16)), finite_magnitude(__uint_as_float(words[i] & 0xffff0000u))));
        finite = fmaxf(finite, __shfl_xor_sync(0xffffffffu, finite, 1));
        finite = fmaxf(finite, __shfl_xor_sync(0xffffffffu, finite, 2));
        const int exponent = scale_exponent(finite);
        const float inverse = power_of_two(-exponent);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            codes[i] = encode_four(__uint_as_float(words[2 * i] << 16), __uint_as_float(words[2 * i] & 0xffff0000u), __uint_as_float(words[2 * i + 1] << 16),
                                   __uint_as_float(words[2 * i + 1] & 0xffff0000u), inverse);
        return power_of_two(exponent);
    }
    const int exponent = scale_exponent(__uint_as_float(greatest << 16));
    const float inverse = power_of_two(-exponent);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        unsigned short low, high;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(low) : "f"(__uint_as_float(words[2 * i] & 0xffff0000u) * inverse), "f"(__uint_as_float(words[2 * i] << 16) * inverse));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(high) : "f"(__uint_as_float(words[2 * i + 1] & 0xffff0000u) * inverse), "f"(__uint_as_float(words[2 * i + 1] << 16) * inverse));
        codes[i] = low | (static_cast<unsigned>(high) << 16);
    }
    return power_of_two(exponent);
}

// `Gated`: a block's 16 rows are 8 gate rows followed by their 8 up rows; it writes silu(gate) * up (or, with `gate_limit` > 0, the clamped form).
// `Codes`: x is e4m3 codes [M, K] with scales [blocks][M]; else bfloat16 rows (NB == 1).
template <int NB, typename TOut, bool Gated, bool Codes>
__global__ void __launch_bounds__(kWarps * 32)
gemm8_skinny_kernel(const void* __restrict__ x_any, long long x_stride, const float* __restrict__ x_scales, const uint8_t* __restrict__ w, const float* __restrict__ w_scales,
                    const float* __restrict__ bias, TOut* __restrict__ out, int M, int N, int K, long long out_stride, float gate_limit) {
    static_assert(Codes || NB == 1, "bfloat16 rows are quantised eight at a time");
    grid_dependents_launch();
    extern __shared__ __align__(16) uint8_t ring_raw[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.x * kRows;
    const int across = (K + kChunk - 1) / kChunk;
    const int n_chunks = across > warp ? (across - warp + kWarps - 1) / kWarps : 0;
    const float* w_scale_row = w_scales + static_cast<size_t>(row0 / kScaleBlock) * across;      // 16 divides a block of 128 rows
    uint4* ring = reinterpret_cast<uint4*>(ring_raw) + warp * kDepth * 128;      // [depth][row][piece of 16 columns]
    // A chunk is 16 lines of 128 bytes, a row's by eight lanes; odd rows' halves change places so that eight lanes read 128 different bytes below.
    auto issue = [&](int index) {
        if (index < n_chunks) {
            const int column = (warp + index * kWarps) * kChunk + (lane & 7) * 16;
            uint4* slot = ring + (index % kDepth) * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * 4 + (lane >> 3);
                copy_async_16(slot + row * 8 + ((lane & 7) ^ ((row & 1) << 2)), w + static_cast<size_t>(min(row0 + row, N - 1)) * K + (column < K ? column : 0), column < K);
            }
        }
        copy_async_commit();
    };
#pragma unroll
    for (int index = 0; index < kDepth - 1; ++index) issue(index);
    float w_scale = n_chunks > 0 ? w_scale_row[warp] : 0.0f;
    float acc[NB][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    grid_dependency_wait();      // the weight does not depend on the previous kernel; the activations do
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 held[4] = {zero, zero, zero, zero};      // bfloat16 rows: the next chunk's values are on their way while this one's are used
    auto fetch = [&](int index) {
        const int column = (warp + index * kWarps) * kChunk + t * 16;
        const bf16* row = static_cast<const bf16*>(x_any) + static_cast<size_t>(g < M ? g : 0) * x_stride;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const bool live = g < M && index < n_chunks && column + 64 * p < K;
            held[2 * p] = live ? __ldg(reinterpret_cast<const uint4*>(row + column + 64 * p)) : zero;
            held[2 * p + 1] = live ? __ldg(reinterpret_cast<const uint4*>(row + column + 64 * p) + 1) : zero;
        }
    };
    // Quantised rows: the next chunk's codes and scales likewise.
    uint4 code_next[NB][2];
    float factor_next[NB][2];
    auto fetch_codes = [&](int index) {
        const uint8_t* x = static_cast<const uint8_t*>(x_any);
        const int block = warp + index * kWarps;
        const bool there = index < n_chunks;
        const float w_scale = there ? __ldg(w_scale_row + block) : 0.0f;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int token = j * 8 + g;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int column = block * kChunk + 64 * p + t * 16;
                code_next[j][p] = there && token < M && column < K ? __ldg(reinterpret_cast<const uint4*>(x + static_cast<size_t>(token) * K + column)) : zero;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) factor_next[j][h] = there && j * 8 + 2 * t + h < M ? __ldg(x_scales + static_cast<size_t>(block) * M + j * 8 + 2 * t + h) * w_scale : 0.0f;
        }
    };
    if constexpr (Codes) fetch_codes(0);
    else fetch(0);
    for (int index = 0; index < n_chunks; ++index) {
        copy_async_wait<kDepth - 2>();      // chunk `index` has landed, and every lane is done with the slot that is written next
        __syncwarp();
        issue(index + kDepth - 1);
        unsigned codes[NB][8];
        float factor[NB][2];      // of tokens 2t and 2t + 1
        if constexpr (Codes) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    codes[j][4 * p] = code_next[j][p].x;
                    codes[j][4 * p + 1] = code_next[j][p].y;
                    codes[j][4 * p + 2] = code_next[j][p].z;
                    codes[j][4 * p + 3] = code_next[j][p].w;
                }
                factor[j][0] = factor_next[j][0];
                factor[j][1] = factor_next[j][1];
            }
            fetch_codes(index + 1);
        } else {
            const float w_scale_here = w_scale;
            if (index + 1 < n_chunks) w_scale = w_scale_row[warp + (index + 1) * kWarps];
            const float scale = quantize_chunk(held, codes[0]);
            fetch(index + 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) factor[0][h] = __shfl_sync(0xffffffffu, scale, (2 * t + h) * 4) * w_scale_here;
        }
        const uint4* slot = ring + (index % kDepth) * 128 + g * 8;
        const int first = t ^ ((g & 1) << 2), second = first ^ 4;
        const uint4 lo[2] = {slot[first], slot[second]}, hi[2] = {slot[64 + first], slot[64 + second]};
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f}, other[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // two chains
            mma_e4m3(part, lo[0].x, hi[0].x, lo[0].y, hi[0].y, codes[j][0], codes[j][1]);
            mma_e4m3(other, lo[1].x, hi[1].x, lo[1].y, hi[1].y, codes[j][4], codes[j][5]);
            mma_e4m3(part, lo[0].z, hi[0].z, lo[0].w, hi[0].w, codes[j][2], codes[j][3]);
            mma_e4m3(other, lo[1].z, hi[1].z, lo[1].w, hi[1].w, codes[j][6], codes[j][7]);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(part[i] + other[i], factor[j][i & 1], acc[j][i]);
        }
    }
    copy_async_wait<0>();
    __syncthreads();      // the ring is done with; its memory now holds the warps' sums
    float (*partial)[NB * 8][kRows + 1] = reinterpret_cast<float (*)[NB * 8][kRows + 1]>(ring_raw);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        partial[warp][j * 8 + 2 * t][g] = acc[j][0];
        partial[warp][j * 8 + 2 * t + 1][g] = acc[j][1];
        partial[warp][j * 8 + 2 * t][g + 8] = acc[j][2];
        partial[warp][j * 8 + 2 * t + 1][g + 8] = acc[j][3];
    }
    __syncthreads();
    for (int index = threadIdx.x; index < NB * 8 * kRows; index += kWarps * 32) {
        const int token = index / kRows, r = index % kRows;
        const int feature = row0 + r;
        float sum = 0.0f;
#pragma unroll
        for (int wi = 0; wi < kWarps; ++wi) sum += partial[wi][token][r];
        if (bias && feature < N) sum += bias[feature];
        if (Gated) {
            // Threads r and r ^ 8 of the same 16 hold a gate and its up value; both are rounded as the unfused product would store them.
            const float mine = round_through<bf16>(sum);
            const float other = __shfl_xor_sync(__activemask(), mine, 8);
            if (r < 8 && token < M && feature < N) out[static_cast<size_t>(token) * out_stride + (row0 >> 1) + r] = from_float<TOut>(gated_value(mine, other, gate_limit));
        } else if (token < M && feature < N) {
            out[static_cast<size_t>(token) * out_stride + feature] = from_float<TOut>(sum);
        }
    }
}

constexpr int kRingBytes = kWarps * kDepth * 2048;
static_assert(kWarps * 4 * 8 * (kRows + 1) * 4 <= kRingBytes, "the warps' sums must fit the ring");

template <int NB, typename TOut, bool Gated, bool Codes>
int launch(const void* x, long long x_stride, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride,
           float gate_limit, cudaStream_t stream) {
    static bool ready[64] = {};
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess) return static_cast<int>(status);
    if (device >= 64 || !ready[device]) {
        status = cudaFuncSetAttribute(gemm8_skinny_kernel<NB, TOut, Gated, Codes>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
        if (status != cudaSuccess) return static_cast<int>(status);
        if (device < 64) ready[device] = true;
    }
    const int code = tau_launch(gemm8_skinny_kernel<NB, TOut, Gated, Codes>, dim3((N + kRows - 1) / kRows), dim3(kWarps * 32), kRingBytes, stream, x, x_stride, x_scales,
                                static_cast<const uint8_t*>(w), w_scales, bias, static_cast<TOut*>(out), M, N, K, out_stride, gate_limit);
    return code ? code : tau_launch_status();
}

template <int NB, bool Codes>
int launch_typed(int out_dtype, int gated, const void* x, long long x_stride, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K,
                 long long out_stride, float gate_limit, cudaStream_t s) {
    if (gated) return launch<NB, bf16, true, Codes>(x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    if (out_dtype == TAU_BF16) return launch<NB, bf16, false, Codes>(x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    return launch<NB, float, false, Codes>(x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
}

}  // namespace

// `x_scales` == nullptr: x is bfloat16 rows `x_stride` elements apart on 16-byte borders, M <= 8; else codes [M, K] and scales [blocks][M], M <= 32.
TAU_EXPORT int tau_gemm8_skinny(int out_dtype, const void* x, long long x_stride, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K,
                                long long out_stride, int gated, float gate_limit, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !w || !w_scales || !out || K <= 0 || (K & 15) || M > (x_scales ? 32 : 8) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) ||
        (!x_scales && (x_stride & 7)) || (out_dtype != TAU_BF16 && out_dtype != TAU_F32) || (gated && ((N & 15) || out_dtype != TAU_BF16)))
        return cudaErrorInvalidValue;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!x_scales) return launch_typed<1, false>(out_dtype, gated, x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    if (M <= 8) return launch_typed<1, true>(out_dtype, gated, x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    if (M <= 16) return launch_typed<2, true>(out_dtype, gated, x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    return launch_typed<4, true>(out_dtype, gated, x, x_stride, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
}
