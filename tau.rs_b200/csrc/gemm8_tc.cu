// Tensor-core product of operands in 8 bits for sm_100a: out[M, N] = x[M, K] * w[N, K]^T + bias, both e4m3 codes with 32-bit scales.
//
//     out[m, n] = sum over blocks b of 128 columns: x_scale[b][m] * w_scale[n / 128][b] * (sum over the block of codes)
//
// The scales change every 128 columns of K, so the accumulator in tensor memory holds one such block at a time (four tcgen05.mma of kind f8f6f4, 32 columns each)
// and the sums over blocks are kept in registers: four warps for each 64 features read a block's sums with tcgen05.ld and add them times both scales, while
// the next blocks' products fill the other accumulators (two of 256 or 192 features, four of 128).  Rows (tokens) are the lanes of tensor memory and features its columns, so a thread's factor
// is one number for each 128 features: 64 multiply-adds a thread and block, 256 on each quarter of an SM, against the 512 clocks that the products of a 128 x 256 block take.
//
// Operands come by TMA (128-byte swizzle, no multicast): a stage is 128 bytes of K of 128 rows of x and BN of w.  One warp asks for tiles, one issues products,
// the others add.  It is persistent over tiles of 128 tokens x BN features, or, where there are few tiles, works on one of up to eight ranges of K
// of a tile: the ranges of a tile are a thread-block cluster, leave their sums in shared memory and each adds and stores a slice of the tokens, in the order of the ranges.
// Every wait is bounded as in the 16-bit product.
//
// Needs K % 16 == 0, contiguous codes on 16-byte borders.
#include "tcgen05.cuh"
#include "quantize_rows.cuh"

namespace {

constexpr int BM = 128;            // tokens to a tile
constexpr int BK = kScaleBlock;    // bytes, and columns, of K to a stage: one swizzled row, one scale
constexpr int kMmaK = 32;
constexpr int kPart = 64;          // features to a warp that adds: its sums are 64 registers a thread
constexpr int adders(int bn) { return 4 * bn / kPart; }      // for each 64 features a warp to each 32 lanes of tensor memory
constexpr int threads(int bn) { return 32 * (2 + adders(bn)); }
constexpr int kMostRanges = 8;

struct Shared {
    uint64_t full[8];
    uint64_t empty[8];
    uint64_t sums_full[4];
    uint64_t sums_empty[4];
    uint32_t tensor_memory_base;
    int abort_flag;
};

// Instruction descriptor: float sums, e4m3 A and B, both K-major, M = m, N = n.
__device__ __forceinline__ uint32_t descriptor_e4m3(int m, int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

__device__ __forceinline__ void mma_issue_e4m3(uint32_t sums, uint64_t a, uint64_t b, uint32_t descriptor, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(sums),
        "l"(a), "l"(b), "r"(descriptor), "r"(accumulate)
        : "memory");
}

constexpr int stage_bytes(int bn) { return (BM + bn) * BK; }
constexpr int stages_of(int bn) { return bn == 256 ? 4 : bn == 192 ? 5 : 6; }
constexpr int shared_bytes(int bn) { return static_cast<int>(sizeof(Shared)) + 1024 + stages_of(bn) * stage_bytes(bn); }

// Adds a block's sums of this warp's 32 tokens and 64 features, times the token's factor; `Step` columns of tensor memory at a time: 32, or 16 where 18 warps leave a thread 100
// registers.  The accumulator is free before the last of them are added.
template <int Step, typename Release>
__device__ __forceinline__ void add_block(uint32_t address, float factor, float (&sums)[kPart], Release release) {
#pragma unroll
    for (int c = 0; c < kPart; c += Step) {
        uint32_t v[Step];
        if constexpr (Step == 32) {
            tensor_load_32(address + c, v);
            tensor_load_wait();
        } else {
            tensor_load_16(address + c, v);
        }
        if (c + Step == kPart) {
            tensor_fence_before_sync();
            __syncwarp();
            release();
        }
#pragma unroll
        for (int j = 0; j < Step; ++j) sums[c + j] = fmaf(__uint_as_float(v[j]), factor, sums[c + j]);
    }
}

// Stores eight neighbouring results of a row, those below `left` of them; `border`: rows (and every eighth result) begin on so many bytes, up to 16.
template <typename TOut>
__device__ __forceinline__ void store_eight(TOut* target, const float (&v)[8], int left, int border) {
    if constexpr (sizeof(TOut) == 2) {
        const unsigned words[4] = {pack_bf16_pair(v[0], v[1]), pack_bf16_pair(v[2], v[3]), pack_bf16_pair(v[4], v[5]), pack_bf16_pair(v[6], v[7])};
        if (left >= 8 && border >= 4) {
            if (border == 16) {
                *reinterpret_cast<uint4*>(target) = make_uint4(words[0], words[1], words[2], words[3]);
            } else if (border == 8) {
                reinterpret_cast<uint2*>(target)[0] = make_uint2(words[0], words[1]);
                reinterpret_cast<uint2*>(target)[1] = make_uint2(words[2], words[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) reinterpret_cast<unsigned*>(target)[i] = words[i];
            }
            return;
        }
    } else if (left >= 8 && border >= 8) {
        if (border == 16) {
            reinterpret_cast<float4*>(target)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(target)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<float2*>(target)[i] = make_float2(v[2 * i], v[2 * i + 1]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) target[i] = from_float<TOut>(v[i]);
}

// Eight or, gated, sixteen sums of a row from feature `feature` on, finished and stored.
template <typename TOut, bool Gated>
__device__ __forceinline__ void finish_row(const float* v, int feature, int N, const float* __restrict__ bias, TOut* row, int border, float gate_limit) {
    if constexpr (Gated) {      // 8 gate columns, their 8 up columns; both rounded as a product that is not gated would store them
        float result[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) result[i] = gated_value(round_through<bf16>(v[i]), round_through<bf16>(v[8 + i]), gate_limit);
        store_eight(row + (feature >> 1), result, N - feature > 0 ? 8 : 0, border);      // N is a multiple of 16
    } else {
        float result[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) result[i] = v[i] + ((bias != nullptr && feature + i < N) ? bias[feature + i] : 0.0f);
        store_eight(row + feature, result, N - feature, border);
    }
}

template <int BN, typename TOut, bool Gated>
__global__ void __launch_bounds__(threads(BN), 1)
gemm8_tc_kernel(const __grid_constant__ CUtensorMap input_map, const __grid_constant__ CUtensorMap weight_map, const float* __restrict__ x_scales, const float* __restrict__ w_scales,
                const float* __restrict__ bias, TOut* __restrict__ out, int M, int N, int K, long long out_stride, int ranges, int border, float gate_limit) {
    extern __shared__ uint8_t shared_raw[];
    Shared* shared = reinterpret_cast<Shared*>(shared_raw);
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(shared_raw) + sizeof(Shared) + 1023) & ~uintptr_t(1023));
    constexpr uint32_t kStages = stages_of(BN), kInputBytes = BM * BK, kStageBytes = stage_bytes(BN);
    constexpr uint32_t kSlots = 512 / BN, kColumns = 512;      // all of tensor memory: two or four accumulators
    constexpr int kAdders = adders(BN), kThreads = threads(BN);
    constexpr int kPartialStride = BN + 4;                        // floats to a row of the sums that a cluster shares: 16-byte loads of neighbouring rows fall on different banks
    static_assert(BM * kPartialStride * 4 <= static_cast<int>(kStages * kStageBytes), "the shared sums must fit the stages");
    static_assert(alone_on_an_sm(shared_bytes(BN)), "two blocks of an SM could wait for each other's tensor memory");
    float* const partial = reinterpret_cast<float*>(tiles);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int feature_tiles = (N + BN - 1) / BN, token_tiles = (M + BM - 1) / BM;
    const int n_items = feature_tiles * token_tiles * ranges;      // item = tile * ranges + range; neighbouring tiles share their features
    const int k_blocks = (K + BK - 1) / BK;
    volatile int* abort_flag = &shared->abort_flag;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            barrier_init(&shared->full[s], 1);
            barrier_init(&shared->empty[s], 1);
        }
        for (uint32_t a = 0; a < kSlots; ++a) {
            barrier_init(&shared->sums_full[a], 1);
            barrier_init(&shared->sums_empty[a], kAdders);
        }
        shared->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(&shared->tensor_memory_base)), "r"(kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tensor_fence_before_sync();
    __syncthreads();
    tensor_fence_after_sync();
    const uint32_t tensor_base = shared->tensor_memory_base;
    grid_dependents_launch();      // only now: a block that took tensor memory before this one would keep it waiting

    if (warp == 0) {
        // ---- the tiles, by TMA.  The weight never depends on the previous kernel: until every stage is in use only its tiles are asked for.
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true, waited = false;
            int held = 0, held_k[8], held_token[8];
            uint32_t asked = 0;      // stages handed to copies so far
            auto release = [&]() {
                grid_dependency_wait();
                waited = true;
                for (int h = 0; h < held; ++h) tma_load_2d(tiles + h * kStageBytes, &input_map, held_k[h], held_token[h], &shared->full[h]);
            };
            for (int item = blockIdx.x; item < n_items && alive; item += gridDim.x) {
                const int tile = item / ranges, range = item - tile * ranges;
                const int feature0 = (tile / token_tiles) * BN, token0 = (tile % token_tiles) * BM;
                const int first = k_blocks * range / ranges, last = k_blocks * (range + 1) / ranges;
                for (int kb = first; kb < last; ++kb) {
                    if (!waited && held == static_cast<int>(kStages)) release();
                    if (!barrier_wait(&shared->empty[stage], phase ^ 1u, abort_flag)) { alive = false; break; }
                    uint8_t* input_tile = tiles + stage * kStageBytes;
                    barrier_expect_bytes(&shared->full[stage], kStageBytes);
                    tma_load_2d(input_tile + kInputBytes, &weight_map, kb * BK, feature0, &shared->full[stage]);
                    if (waited) {
                        tma_load_2d(input_tile, &input_map, kb * BK, token0, &shared->full[stage]);
                    } else {   // the first stages: stage == held
                        held_k[held] = kb * BK;
                        held_token[held] = token0;
                        ++held;
                    }
                    ++asked;
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
            if (!waited) release();
            // Nothing leaves, and no sums are shared through this memory, before the copies have landed.
            for (uint32_t n = asked > kStages ? asked - kStages : 0; n < asked; ++n) barrier_outlast(&shared->full[n % kStages], (n / kStages) & 1u);
        }
    } else if (warp == 1) {
        // ---- products: the whole warp, one lane issues
        const bool leader = elect_one();
        const uint32_t base = __shfl_sync(0xffffffffu, tensor_base, 0), first_tile = __shfl_sync(0xffffffffu, smem_address(tiles), 0);
        auto warp_wait = [&](uint64_t* barrier, uint32_t parity) { return __all_sync(0xffffffffu, barrier_wait(barrier, parity, abort_flag)) != 0; };
        const uint32_t descriptor = descriptor_e4m3(BM, BN);
        uint32_t stage = 0, phase = 0, number = 0;      // number: blocks of 128 columns so far
        bool alive = true;
        for (int item = blockIdx.x; item < n_items && alive; item += gridDim.x) {
            const int range = item % ranges;
            const int count = k_blocks * (range + 1) / ranges - k_blocks * range / ranges;
            for (int i = 0; i < count; ++i, ++number) {
                const uint32_t slot = number % kSlots, use = number / kSlots;
                if (use > 0 && !warp_wait(&shared->sums_empty[slot], (use - 1) & 1u)) { alive = false; break; }
                if (!warp_wait(&shared->full[stage], phase)) { alive = false; break; }
                tensor_fence_after_sync();
                const uint32_t input_address = first_tile + stage * kStageBytes, weight_address = input_address + kInputBytes;
                if (leader) {
#pragma unroll
                    for (int k = 0; k < BK / kMmaK; ++k)
                        mma_issue_e4m3(base + slot * BN, tile_descriptor(input_address + k * kMmaK), tile_descriptor(weight_address + k * kMmaK), descriptor, k > 0 ? 1u : 0u);
                    mma_commit(&shared->empty[stage]);
                    mma_commit(&shared->sums_full[slot]);
                }
                __syncwarp();
                if (++stage == kStages) { stage = 0; phase ^= 1u; }
            }
        }
    } else {
        // ---- adders: a warp owns 32 tokens (those lanes of tensor memory that its number allows) and 64 of the features
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        uint32_t number = 0;
        bool alive = true;
        grid_dependency_wait();      // the scales come from the previous kernel, and it may still read what is written here
        for (int item = blockIdx.x; item < n_items && alive; item += gridDim.x) {
            const int tile = item / ranges, range = item - tile * ranges;
            const int feature0 = (tile / token_tiles) * BN + part * kPart, token = (tile % token_tiles) * BM + quarter * 32 + lane;
            const int first = k_blocks * range / ranges, count = k_blocks * (range + 1) / ranges - first;
            const float* x_scale = x_scales + static_cast<size_t>(first) * M + min(token, M - 1);
            const float* w_scale = w_scales + static_cast<size_t>(min(feature0, N - 1) / kScaleBlock) * k_blocks + first;      // 64 divides 128: one scale to a warp
            float sums[kPart];
#pragma unroll
            for (int c = 0; c < kPart; ++c) sums[c] = 0.0f;
            // Factors of the next two blocks are on their way: a load takes about as long as a block's products.
            float x_next[2], w_next[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                x_next[a] = a < count ? x_scale[static_cast<size_t>(a) * M] : 0.0f;
                w_next[a] = a < count ? w_scale[a] : 0.0f;
            }
            for (int i = 0; i < count; ++i, ++number) {
                const uint32_t slot = number % kSlots, use = number / kSlots;
                const float factor = x_next[0] * w_next[0];
                x_next[0] = x_next[1];
                w_next[0] = w_next[1];
                if (i + 2 < count) {
                    x_next[1] = x_scale[static_cast<size_t>(i + 2) * M];
                    w_next[1] = w_scale[i + 2];
                }
                if (!__all_sync(0xffffffffu, barrier_wait(&shared->sums_full[slot], use & 1u, abort_flag))) { alive = false; break; }
                tensor_fence_after_sync();
                const uint32_t address = tensor_base + (static_cast<uint32_t>(quarter * 32) << 16) + slot * BN + part * kPart;
                auto release = [&]() {
                    if (lane == 0) barrier_arrive(&shared->sums_empty[slot]);
                };
                if (token - lane < M) add_block<(BN > 192 ? 16 : 32)>(address, factor, sums, release);      // some of these 32 tokens are there
                else release();
            }
            if (!alive) break;
            if (ranges == 1) {
                if (token < M) {
                    TOut* row = out + static_cast<size_t>(token) * out_stride;
                    constexpr int kStep = Gated ? 16 : 8;
#pragma unroll
                    for (int c = 0; c < kPart; c += kStep)
                        if (feature0 + c < N) finish_row<TOut, Gated>(sums + c, feature0 + c, N, bias, row, border, gate_limit);
                }
            } else {
                // One item to a block here.  The stages are free: every product has read them (the sums are complete) and no copy is left.
                float* mine = partial + static_cast<size_t>(quarter * 32 + lane) * kPartialStride + part * kPart;
#pragma unroll
                for (int c = 0; c < kPart; c += 4) *reinterpret_cast<float4*>(mine + c) = make_float4(sums[c], sums[c + 1], sums[c + 2], sums[c + 3]);
            }
        }
    }

    tensor_fence_before_sync();
    __syncthreads();
    if (ranges > 1) {
        // The cluster's blocks hold the ranges of one tile.  Every thread of every block comes here, also after a wait that ran out.
        cluster_share_abort(&shared->abort_flag, ranges);
        cluster_sync_all();
        if (*abort_flag == 0) {
            grid_dependency_wait();
            const int tile = blockIdx.x / ranges, rank = static_cast<int>(cluster_rank());
            const int feature0 = (tile / token_tiles) * BN, token0 = (tile % token_tiles) * BM;
            const int live = min(BM, M - token0), per = (live + ranges - 1) / ranges;
            constexpr int kStep = Gated ? 16 : 8, kPieces = BN / kStep;
            const int begin = rank * per, rows = max(0, min(per, live - begin));
            for (int index = threadIdx.x; index < rows * kPieces; index += kThreads) {
                const int row = begin + index / kPieces, c = index % kPieces * kStep;
                if (feature0 + c >= N) continue;
                const uint32_t own = smem_address(partial + static_cast<size_t>(row) * kPartialStride + c);
                float sum[kStep];
#pragma unroll
                for (int i = 0; i < kStep; ++i) sum[i] = 0.0f;
#pragma unroll
                for (int r = 0; r < kMostRanges; ++r) {
                    if (r >= ranges) continue;
                    const uint32_t from = cluster_address_of(own, r);
#pragma unroll
                    for (int i = 0; i < kStep; i += 4) {
                        const float4 part = cluster_load_4(from + i * 4);
                        sum[i] += part.x; sum[i + 1] += part.y; sum[i + 2] += part.z; sum[i + 3] += part.w;
                    }
                }
                finish_row<TOut, Gated>(sum, feature0 + c, N, bias, out + static_cast<size_t>(token0 + row) * out_stride, border, gate_limit);
            }
        }
        cluster_sync_all();      // nobody leaves while another still reads its sums
    }
    if (warp == 1) {
        tensor_fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tensor_base), "r"(kColumns) : "memory");
    }
}

int code_map(CUtensorMap* map, const void* codes, long long rows, int K, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t extents[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(K)};
    const cuuint32_t box[2] = {BK, static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
    const CUresult result = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), extents, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return result == CUDA_SUCCESS ? 0 : cudaErrorInvalidValue;
}

struct Call {
    const void* x;
    const float* x_scales;
    const void* w;
    const float *w_scales, *bias;
    void* out;
    int M, N, K;
    long long out_stride;
    int ranges, sms;
    float gate_limit;
};

template <int BN, typename TOut, bool Gated>
int launch(const Call& c, cudaStream_t stream) {
    static bool ready[64] = {};
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess) return static_cast<int>(status);
    if (device >= 64 || !ready[device]) {
        status = cudaFuncSetAttribute(gemm8_tc_kernel<BN, TOut, Gated>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes(BN));
        if (status != cudaSuccess) return static_cast<int>(status);
        if (device < 64) ready[device] = true;
    }
    CUtensorMap input_map, weight_map;
    int code = code_map(&input_map, c.x, c.M, c.K, BM);
    if (!code) code = code_map(&weight_map, c.w, c.N, c.K, BN);
    if (code) return code;
    const long long tiles = static_cast<long long>((c.N + BN - 1) / BN) * ((c.M + BM - 1) / BM);
    if (tiles * c.ranges > 0x7fffffffll) return cudaErrorInvalidValue;
    const unsigned long long bits = static_cast<unsigned long long>(c.out_stride) * sizeof(TOut) | reinterpret_cast<uintptr_t>(c.out) | 16u;
    const int border = static_cast<int>(bits & (~bits + 1));
    if (c.ranges > 1)
        code = tau_launch_clusters(c.ranges, gemm8_tc_kernel<BN, TOut, Gated>, dim3(static_cast<unsigned>(tiles * c.ranges)), dim3(threads(BN)), shared_bytes(BN), stream, input_map, weight_map,
                                   c.x_scales, c.w_scales, c.bias, static_cast<TOut*>(c.out), c.M, c.N, c.K, c.out_stride, c.ranges, border, c.gate_limit);
    else
        code = tau_launch(gemm8_tc_kernel<BN, TOut, Gated>, dim3(static_cast<unsigned>(tiles < c.sms ? tiles : c.sms)), dim3(threads(BN)), shared_bytes(BN), stream, input_map, weight_map, c.x_scales,
                          c.w_scales, c.bias, static_cast<TOut*>(c.out), c.M, c.N, c.K, c.out_stride, 1, border, c.gate_limit);
    return code ? code : tau_launch_status();
}

template <int BN>
int launch_typed(int out_dtype, int gated, const Call& c, cudaStream_t stream) {
    if (gated) return launch<BN, bf16, true>(c, stream);
    if (out_dtype == TAU_BF16) return launch<BN, bf16, false>(c, stream);
    return launch<BN, float, false>(c, stream);
}

}  // namespace

TAU_EXPORT int tau_gemm8_tc_status() {
    int flag = 0;
    cudaDeviceSynchronize();
    if (cudaMemcpyFromSymbol(&flag, wait_error, sizeof(flag)) != cudaSuccess) return -1;
    return flag;
}

// x codes [M, K] with scales [blocks][M]; w codes [N, K] with scales [blocks of N][blocks].  `features`: 128, 192 or 256 to a tile of 128 tokens; `ranges`: 1 to 8 ranges of K to a
// tile.  0: chosen.
TAU_EXPORT int tau_gemm8_tc(int out_dtype, const void* x, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K, long long out_stride,
                            int gated, float gate_limit, int features, int ranges, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !x_scales || !w || !w_scales || !out || K <= 0 || (K & 15) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) ||
        (out_dtype != TAU_BF16 && out_dtype != TAU_F32) || (gated && ((N & 15) || out_dtype != TAU_BF16)) || (features != 0 && features != 128 && features != 192 && features != 256) ||
        ranges < 0 || ranges > kMostRanges)
        return cudaErrorInvalidValue;
    int device = 0, sms = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return cudaErrorInvalidValue;
    const int k_blocks = (K + BK - 1) / BK, token_tiles = (M + BM - 1) / BM;
    // What is not given is chosen by what a round of tiles costs: a block of K takes a tile about as long as 192 features and its own (some 1.1 ns a feature; 4,096 columns: 15 us at
    // 128 features, 18 at 192, 21 at 256), and the join of two, four or eight ranges as long as 1,500, 3,500 and 6,000 such steps of a feature.  Clusters have to fit the machine at
    // once, whose groups of SMs hold about 72 of two, 32 of four and 12 of eight.  (us at 128, 192 and 256 features: 16 x 4,096 x 24,576 31, 23 and 28; 512 x 4,096 x 6,144
    // 30, 19 and 22; 2,048 x 4,096 x 6,144 85, 68 and 61; 64 x 12,288 x 4,096 in one, two and four ranges 38, 23 and 16; 64 x 1,024 x 6,144 in one and two 5.7 and 7.0.)
    long long least = 0;
    int best_features = 0, best_ranges = 0;
    for (int bn = 256; bn >= 128; bn -= 64) {
        if (features != 0 && features != bn) continue;
        const long long n = static_cast<long long>((N + bn - 1) / bn) * token_tiles;
        for (int r = 1; r <= kMostRanges; r *= 2) {
            if (ranges != 0 ? r > 1 : r > 1 && (n > (r == 2 ? 72 : r == 4 ? 32 : 12) || k_blocks < 4 * r)) break;
            const long long cost = (n + sms - 1) / sms * ((k_blocks + r - 1) / r) * (bn + 192) + (r == 1 ? 0 : r == 2 ? 1500 : r == 4 ? 3500 : 6000);
            if (best_features == 0 || cost < least) {
                least = cost;
                best_features = bn;
                best_ranges = r;
            }
        }
    }
    features = best_features;
    if (ranges == 0) ranges = best_ranges;
    if (ranges > k_blocks) ranges = k_blocks;
    const Call call = {x, x_scales, w, w_scales, bias, out, M, N, K, out_stride, ranges, sms, gate_limit};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (features == 256) return launch_typed<256>(out_dtype, gated, call, s);
    if (features == 192) return launch_typed<192>(out_dtype, gated, call, s);
    return launch_typed<128>(out_dtype, gated, call, s);
}

// The same of bfloat16 or float32 rows `x_stride` elements apart on 16-byte borders, which are quantised into `held` first: M * K codes, then M floats for each 128 columns.
TAU_EXPORT int tau_linear8_tc(int x_dtype, const void* x, long long x_stride, void* held, int out_dtype, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K,
                              long long out_stride, int gated, float gate_limit, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!held || K <= 0) return cudaErrorInvalidValue;
    float* scales = scales_behind(held, M, K);
    const int code = launch_quantize_rows(x_dtype, x, x_stride, held, scales, M, K, static_cast<cudaStream_t>(stream));
    return code ? code : tau_gemm8_tc(out_dtype, held, scales, w, w_scales, bias, out, M, N, K, out_stride, gated, gate_limit, 0, 0, stream);
}
