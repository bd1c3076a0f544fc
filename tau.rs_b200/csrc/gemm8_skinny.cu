// Products for a few rows of activations with the weight in 8 bits: out[M, N] = x[M, K] * w[N, K]^T + bias, bound by reading `w` once.
//
// Weight codes are e4m3 with a 32-bit scale for each 128 x 128 block, activations e4m3 with a scale for each row and 128 columns, so
//     out[m, n] = sum over blocks b of 128 columns: x_scale[b][m] * w_scale[n / 128][b] * (sum over the block of codes),
// and a chunk of 128 columns of 16 features (2 KB) is a warp's unit: four mma.sync m16n8k32 on e4m3 operands with 32-bit sums, the weight's rows as A and the
// activations as B, then one multiplication of the chunk's sums by both scales.  (With at most 16 rows tcgen05's tiles of 128 would be empty for the most part.)  Chunks come by
// cp.async in whole lines.  Two forms: up to 8 bfloat16 rows, quantised here, a block to an SM; and up to 16 quantised rows, a block to 16 features.
//
// Needs K % 16 == 0 and contiguous codes on a 16-byte border.
#include "quantize_rows.cuh"

namespace {

constexpr int kRows = 16;        // output features to a block
constexpr int kWarps = 8;
constexpr int kDepth = 4;        // chunks on their way per warp: 64 KB to a block, three blocks to an SM
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
// x is e4m3 codes [M, K] with scales [blocks][M].
template <int NB, typename TOut, bool Gated>
__global__ void __launch_bounds__(kWarps * 32)
gemm8_skinny_kernel(const uint8_t* __restrict__ x, const float* __restrict__ x_scales, const uint8_t* __restrict__ w, const float* __restrict__ w_scales,
                    const float* __restrict__ bias, TOut* __restrict__ out, int M, int N, int K, long long out_stride, float gate_limit) {
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
    float acc[NB][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    grid_dependency_wait();      // the weight does not depend on the previous kernel; the activations do
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    // The next chunk's codes and scales are on their way while this one's are used.
    uint4 code_next[NB][2];
    float factor_next[NB][2];
    auto fetch_codes = [&](int index) {
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
    fetch_codes(0);
    for (int index = 0; index < n_chunks; ++index) {
        copy_async_wait<kDepth - 2>();      // chunk `index` has landed, and every lane is done with the slot that is written next
        __syncwarp();
        issue(index + kDepth - 1);
        unsigned codes[NB][8];
        float factor[NB][2];      // of tokens 2t and 2t + 1
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

// ---- up to 8 bfloat16 rows -------------------------------------------------------------------------------------------------------
// One block of 16 warps to an SM walks over groups of 16 features.  A warp's chunks of K are the same for every group, so it quantises its part of the activations
// once, keeps the codes in shared memory where each lane wrote its own, and from then on only streams: the ring runs on from one group into the next, and what is on its way never
// drains.  (us, against the other form and the launch that quantises for it: 8 x 4,096 x 24,576 20.3 and
// 23.2, 8 x 12,288 x 4,096 14.1 and 15.5, 1 x 1,024 x 4,096 2.6 and 3.7; 100 MB of codes at 5.0 TB/s.  Every block that has 16 features for itself quantising its
// rows: 27.0.)
constexpr int kStreamWarps = 16;

template <int Depth>
constexpr size_t stream_bytes(int across) {
    const int per_warp = (across + kStreamWarps - 1) / kStreamWarps;
    return static_cast<size_t>(kStreamWarps) * (per_warp * (1024 + 32) + Depth * 2048) + 2 * kStreamWarps * 8 * (kRows + 1) * 4;
}

template <typename TOut, bool Gated, int Depth>
__global__ void __launch_bounds__(kStreamWarps * 32, 1)
gemm8_stream_kernel(const bf16* __restrict__ x, long long x_stride, const uint8_t* __restrict__ w, const float* __restrict__ w_scales, const float* __restrict__ bias, TOut* __restrict__ out,
                    int M, int N, int K, long long out_stride, float gate_limit) {
    grid_dependents_launch();
    extern __shared__ __align__(16) uint8_t memory[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int across = (K + kChunk - 1) / kChunk, per_warp = (across + kStreamWarps - 1) / kStreamWarps;
    const int n_groups = (N + kRows - 1) / kRows;
    const int my_groups = (n_groups - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const int chunks = across > warp ? (across - warp + kStreamWarps - 1) / kStreamWarps : 0;      // of a group
    const int total = chunks * my_groups;
    uint4* held = reinterpret_cast<uint4*>(memory) + static_cast<size_t>(warp) * per_warp * 64;      // [chunk][piece][lane]
    float* held_scales = reinterpret_cast<float*>(memory + static_cast<size_t>(kStreamWarps) * per_warp * 1024) + warp * per_warp * 8;      // [chunk][token]
    uint8_t* behind = memory + static_cast<size_t>(kStreamWarps) * per_warp * (1024 + 32);
    uint4* ring = reinterpret_cast<uint4*>(behind) + warp * Depth * 128;
    float (*partial)[kStreamWarps][8][kRows + 1] = reinterpret_cast<float (*)[kStreamWarps][8][kRows + 1]>(behind + kStreamWarps * Depth * 2048);
    // The next chunk to ask for: which group of this block's, which chunk of it, which slot of the ring.
    int ask_group = blockIdx.x, ask_chunk = 0, ask_slot = 0, asked = 0;
    auto issue = [&]() {
        if (asked < total) {
            const int column = (warp + ask_chunk * kStreamWarps) * kChunk + (lane & 7) * 16, row0 = ask_group * kRows;
            uint4* slot = ring + ask_slot * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * 4 + (lane >> 3);
                copy_async_16(slot + row * 8 + ((lane & 7) ^ ((row & 1) << 2)), w + static_cast<size_t>(min(row0 + row, N - 1)) * K + (column < K ? column : 0), column < K);
            }
            if (++ask_chunk == chunks) {
                ask_chunk = 0;
                ask_group += gridDim.x;
            }
            if (++ask_slot == Depth) ask_slot = 0;
        }
        ++asked;
        copy_async_commit();
    };
#pragma unroll
    for (int i = 0; i < Depth - 1; ++i) issue();
    auto scale_of = [&](int group, int chunk) { return __ldg(w_scales + static_cast<size_t>(group * kRows / kScaleBlock) * across + warp + chunk * kStreamWarps); };
    float w_scale = total > 0 ? scale_of(blockIdx.x, 0) : 0.0f;
    grid_dependency_wait();      // the weight does not depend on the previous kernel; the activations do
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int column = (warp + chunk * kStreamWarps) * kChunk + t * 16;
        uint4 raw[4];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const bool live = g < M && column + 64 * p < K;
            const uint4* from = reinterpret_cast<const uint4*>(x + static_cast<size_t>(live ? g : 0) * x_stride + (live ? column + 64 * p : 0));
            raw[2 * p] = live ? __ldg(from) : zero;
            raw[2 * p + 1] = live ? __ldg(from + 1) : zero;
        }
        unsigned codes[8];
        const float scale = quantize_chunk(raw, codes);
        held[chunk * 64 + lane] = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        held[chunk * 64 + 32 + lane] = make_uint4(codes[4], codes[5], codes[6], codes[7]);
        if (t == 0) held_scales[chunk * 8 + g] = scale;
    }
    __syncwarp();
    int slot_number = 0, done = 0;
    for (int turn = 0, group = blockIdx.x; turn < my_groups; ++turn, group += gridDim.x) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int chunk = 0; chunk < chunks; ++chunk, ++done) {
            copy_async_wait<Depth - 2>();      // this chunk has landed, and every lane is done with the slot that is written next
            __syncwarp();
            issue();
            const float w_scale_here = w_scale;
            if (done + 1 < total) w_scale = chunk + 1 < chunks ? scale_of(group, chunk + 1) : scale_of(group + gridDim.x, 0);
            const uint4 first_codes = held[chunk * 64 + lane], second_codes = held[chunk * 64 + 32 + lane];
            const uint4* slot = ring + slot_number * 128 + g * 8;
            if (++slot_number == Depth) slot_number = 0;
            const int first = t ^ ((g & 1) << 2), second = first ^ 4;
            const uint4 lo[2] = {slot[first], slot[second]}, hi[2] = {slot[64 + first], slot[64 + second]};
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f}, other[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_e4m3(part, lo[0].x, hi[0].x, lo[0].y, hi[0].y, first_codes.x, first_codes.y);
            mma_e4m3(other, lo[1].x, hi[1].x, lo[1].y, hi[1].y, second_codes.x, second_codes.y);
            mma_e4m3(part, lo[0].z, hi[0].z, lo[0].w, hi[0].w, first_codes.z, first_codes.w);
            mma_e4m3(other, lo[1].z, hi[1].z, lo[1].w, hi[1].w, second_codes.z, second_codes.w);
            const float2 scales = *reinterpret_cast<const float2*>(held_scales + chunk * 8 + 2 * t);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(part[i] + other[i], ((i & 1) ? scales.y : scales.x) * w_scale_here, acc[i]);
        }
        float (*mine)[kRows + 1] = partial[turn & 1][warp];      // the other half is still read by the turn before
        mine[2 * t][g] = acc[0];
        mine[2 * t + 1][g] = acc[1];
        mine[2 * t][g + 8] = acc[2];
        mine[2 * t + 1][g + 8] = acc[3];
        __syncthreads();
        if (threadIdx.x < 8 * kRows) {      // four whole warps
            const int token = threadIdx.x / kRows, r = threadIdx.x % kRows, feature = group * kRows + r;
            float sum = 0.0f;
#pragma unroll
            for (int wi = 0; wi < kStreamWarps; ++wi) sum += partial[turn & 1][wi][token][r];
            if (bias && feature < N) sum += bias[feature];
            if (Gated) {
                const float value = round_through<bf16>(sum);
                const float up = __shfl_xor_sync(0xffffffffu, value, 8);
                if (r < 8 && token < M && feature < N) out[static_cast<size_t>(token) * out_stride + group * 8 + r] = from_float<TOut>(gated_value(value, up, gate_limit));
            } else if (token < M && feature < N) {
                out[static_cast<size_t>(token) * out_stride + feature] = from_float<TOut>(sum);
            }
        }
    }
    copy_async_wait<0>();
}

constexpr int kMostShared = 227 * 1024 - 256;
constexpr int kRingBytes = kWarps * kDepth * 2048;
static_assert(kWarps * 4 * 8 * (kRows + 1) * 4 <= kRingBytes, "the warps' sums must fit the ring");

template <int NB, typename TOut, bool Gated>
int launch(const void* x, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride, float gate_limit,
           cudaStream_t stream) {
    static bool ready[64] = {};
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess) return static_cast<int>(status);
    if (device >= 64 || !ready[device]) {
        status = cudaFuncSetAttribute(gemm8_skinny_kernel<NB, TOut, Gated>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
        if (status != cudaSuccess) return static_cast<int>(status);
        if (device < 64) ready[device] = true;
    }
    const int code = tau_launch(gemm8_skinny_kernel<NB, TOut, Gated>, dim3((N + kRows - 1) / kRows), dim3(kWarps * 32), kRingBytes, stream, static_cast<const uint8_t*>(x), x_scales,
                                static_cast<const uint8_t*>(w), w_scales, bias, static_cast<TOut*>(out), M, N, K, out_stride, gate_limit);
    return code ? code : tau_launch_status();
}

template <typename TOut, bool Gated, int Depth>
int launch_stream(const void* x, long long x_stride, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride, float gate_limit,
                  cudaStream_t stream) {
    static int sms[64] = {};
    int device = 0, count = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess) return static_cast<int>(status);
    if (device < 64) count = sms[device];
    if (!count) {
        status = cudaFuncSetAttribute(gemm8_stream_kernel<TOut, Gated, Depth>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
        if (status == cudaSuccess) status = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
        if (status != cudaSuccess) return static_cast<int>(status);
        if (device < 64) sms[device] = count;
    }
    const int groups = (N + kRows - 1) / kRows;
    const int code = tau_launch(gemm8_stream_kernel<TOut, Gated, Depth>, dim3(groups < count ? groups : count), dim3(kStreamWarps * 32), stream_bytes<Depth>((K + kChunk - 1) / kChunk), stream,
                                static_cast<const bf16*>(x), x_stride, static_cast<const uint8_t*>(w), w_scales, bias, static_cast<TOut*>(out), M, N, K, out_stride, gate_limit);
    return code ? code : tau_launch_status();
}

template <int Depth>
int stream_typed(int out_dtype, int gated, const void* x, long long x_stride, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride,
                 float gate_limit, cudaStream_t s) {
    if (gated) return launch_stream<bf16, true, Depth>(x, x_stride, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    if (out_dtype == TAU_BF16) return launch_stream<bf16, false, Depth>(x, x_stride, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    return launch_stream<float, false, Depth>(x, x_stride, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
}

template <int NB>
int launch_typed(int out_dtype, int gated, const void* x, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride,
                 float gate_limit, cudaStream_t s) {
    if (gated) return launch<NB, bf16, true>(x, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    if (out_dtype == TAU_BF16) return launch<NB, bf16, false>(x, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    return launch<NB, float, false>(x, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
}

}  // namespace

// The widest K that the streaming form serves (its activations' codes lie in shared memory).
TAU_EXPORT int tau_gemm8_stream_most_depth() {
    int across = 1;
    while (stream_bytes<3>(across + 1) <= kMostShared) ++across;
    return across * kChunk;
}

// bfloat16 rows `x_stride` elements apart on 16-byte borders, M <= 8, one block to an SM over the whole weight.
TAU_EXPORT int tau_gemm8_stream(int out_dtype, const void* x, long long x_stride, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride,
                                int gated, float gate_limit, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !w || !w_scales || !out || K <= 0 || (K & 15) || M > 8 || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) || (x_stride & 7) ||
        (out_dtype != TAU_BF16 && out_dtype != TAU_F32) || (gated && ((N & 15) || out_dtype != TAU_BF16)) || K > tau_gemm8_stream_most_depth())
        return cudaErrorInvalidValue;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (stream_bytes<5>((K + kChunk - 1) / kChunk) <= kMostShared) return stream_typed<5>(out_dtype, gated, x, x_stride, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    return stream_typed<3>(out_dtype, gated, x, x_stride, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
}

// x codes [M, K] with scales [blocks][M], M <= 16.
TAU_EXPORT int tau_gemm8_skinny(int out_dtype, const void* x, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K,
                                long long out_stride, int gated, float gate_limit, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !x_scales || !w || !w_scales || !out || K <= 0 || (K & 15) || M > 16 || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) ||
        (out_dtype != TAU_BF16 && out_dtype != TAU_F32) || (gated && ((N & 15) || out_dtype != TAU_BF16)))
        return cudaErrorInvalidValue;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M <= 8) return launch_typed<1>(out_dtype, gated, x, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
    return launch_typed<2>(out_dtype, gated, x, x_scales, w, w_scales, bias, out, M, N, K, out_stride, gate_limit, s);
}

// The same of bfloat16 or float32 rows `x_stride` elements apart on 16-byte borders, which are quantised into `held` first: M * K codes, then M floats for each 128 columns.
TAU_EXPORT int tau_linear8_skinny(int x_dtype, const void* x, long long x_stride, void* held, int out_dtype, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K,
                                  long long out_stride, int gated, float gate_limit, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!held || K <= 0 || M > 16) return cudaErrorInvalidValue;
    float* scales = scales_behind(held, M, K);
    const int code = launch_quantize_rows(x_dtype, x, x_stride, held, scales, M, K, static_cast<cudaStream_t>(stream));
    return code ? code : tau_gemm8_skinny(out_dtype, held, scales, w, w_scales, bias, out, M, N, K, out_stride, gated, gate_limit, stream);
}
