// Decode attention over pages held in 8 bits: one new token per sequence over its cached context, split along the context.
//
// Compiled for one head size (-DTAU_HEAD_DIM=...).  With codes c and a scale for each page (64 positions) and head,
//     o = sum_j w_j s_V[page j] c_V[j] / sum_j w_j,   w_j = exp(scale * s_K[page j] * (q . c_K[j]) - max),
// so a page's scales are factors outside its sums: the score's is multiplied into the softmax scale, the value's into the page's part of the
// accumulator.  e4m3's numbers are numbers of 16-bit floats (the conversion is exact), so both products run on f16 operands with 32-bit sums:
// queries are brought to [1, 2) per head by a power of two (exact for a bfloat16 within 2^-14 of the head's greatest element, and off by at most
// 2^-25 of that below), weights are at most one and are rounded to 11 bits.
//
// What bounds it: 2 D bytes of codes for each cached position and key/value head, read once for the head's whole group of query heads.
// A block serves up to 8 (or 16) query heads of one key/value head and a range of the sequence's pages; one warp asks for pages by TMA (a page of
// a head is a box of 64 rows in 128-byte swizzled rows, several pages ahead), four warps take 16 positions each of every page.  Scores are
// computed transposed (rows are keys, columns the group's query heads, mma.sync m16n8k16: with at most 16 columns there is nothing for
// tcgen05's 128 rows to do), probabilities cross over by movmatrix, and values meet them as O^T = V^T P.  The order of elements inside a head is free
// as long as both operands share it, so a lane's 16-byte load of a key serves four products.
// Up to 8 ranges of a sequence form a cluster and are joined through shared memory, in the order of the ranges; more leave records for a second kernel.
#include "tcgen05.cuh"
#include "eight_bit.cuh"

#ifndef TAU_HEAD_DIM
#error "compile with -DTAU_HEAD_DIM=<multiple of 16 up to 256>"
#endif

namespace {

constexpr int D = TAU_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head_dim must be a multiple of 16 between 16 and 256");
constexpr int kPage = 64;
constexpr int kGroupWarps = 4;                    // consumers of a page; one more warp asks for pages
constexpr int kHalves = (D + 127) / 128;          // boxes of 128 bytes to a row
constexpr int kBoxBytes = kPage * 128;
constexpr int kTileBytes = kHalves * kBoxBytes;   // a page of a head's keys, or of its values
constexpr int kStageBytes = 2 * kTileBytes;
// Two pages ahead and four blocks to an SM where a page is 16 KB; three of 32 KB and two blocks for wider heads (64 sequences of 2,048 positions, 32 heads of 128 over 8: 54 us so,
// 60 with four pages and three blocks, 61 with six and two).
template <int Groups>
constexpr int kStagesOf = kHalves == 1 ? 2 * Groups : 3;
constexpr int kMostStages = kHalves == 1 ? 4 : 3;
constexpr int kKeySteps = D / 16;                 // products of 16 head elements
constexpr int kMostClustered = 8;
constexpr float kFailed = -1.0f;                  // in the place of a range's sum of weights (never negative): a wait ran out there
constexpr int kMostOrdered = 1024;                // sequences that a block puts in order
constexpr float kLog2e = 1.4426950408889634f;
// Weights are kept times 2^14: what f16 holds with all its bits then reaches down to 2^-28 of the greatest, and a long tail of small weights keeps its sum.
constexpr float kWeightBits = 14.0f;
constexpr float kLeastShare = 0.00390625f;      // 2^-8: a page whose value scale is smaller than this share of the accumulators' is added in 32 bits

struct Shared {
    uint64_t full[kMostStages];
    uint64_t empty[kMostStages];
    float key_scale[kMostStages], share[kMostStages], older[kMostStages];
    float unit[2];
    uint64_t stored;                              // the newest position is in its page
    float new_key_scale, new_value_scale;         // that page's scales
    int abort_flag;
};

// What the kernel needs to prepare single tokens itself: queries, and where `store` is set keys and values, come as a stacked projection left them, [sequences,
// (n_heads + 2 n_kv_heads) D]; they are normalised per head, rotated, and the newest key and value enter their pages.  `projected` == nullptr: queries are ready, the cache complete.
struct Prepare {
    const bf16* projected;
    long long stride;
    const float* q_weight;
    const float* k_weight;
    float eps;
    const float* cos_table;
    const float* sin_table;
    int rotary_dim;
    int store;
    int vectors;      // heads of 64, 128 or 256 that are rotated whole or not at all, in rows on 16-byte borders
};

__device__ __forceinline__ void tma_load_3d(void* destination, const CUtensorMap* map, int x, int y, int z, uint64_t* barrier) {
    if (operands_lost()) return;
#ifdef TAU_LOST_RANGE      // the test of a wait that runs out where ranges meet through memory
    if (blockIdx.x == TAU_LOST_RANGE) return;
#endif
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_address(destination)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_address(barrier))
                 : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack_half2(float low, float high) {
    unsigned packed;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(packed) : "f"(high), "f"(low));
    return packed;
}

// 16 bytes of a page in shared memory: chunk `chunk` of row `row` (of 128-byte rows whose chunks the copy permuted by the row's number).
__device__ __forceinline__ uint4 page_chunk(const uint8_t* tile, int row, int chunk) {
    return *reinterpret_cast<const uint4*>(tile + (chunk >> 3) * kBoxBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ unsigned page_word(const uint8_t* tile, int row, int byte) {
    return *reinterpret_cast<const unsigned*>(tile + (byte >> 7) * kBoxBytes + row * 128 + ((((byte >> 4) & 7) ^ (row & 7)) << 4) + (byte & 15));
}

// The element of a head that lane t holds as number `i` (0..3) of product `step`: whole groups of 64 elements give each lane 16 neighbours, what is left
// behind them four for each 16 elements.
__device__ __forceinline__ int key_element(int step, int t, int i) {
    const int group = step >> 2;
    return group < D / 64 ? group * 64 + t * 16 + (step & 3) * 4 + i : step * 16 + t * 4 + i;
}

// Sequence number `place` of `n` when longer ones come first: lengths are told apart by quarters of a power of two (of pages), within such a class the order is that of the
// sequences.  Every thread of the block calls it.
__device__ __forceinline__ int by_length(const int* __restrict__ seq_len, int n, int place) {
    const int threads = blockDim.x;
    constexpr int kClasses = 64;
    __shared__ unsigned char class_of[kMostOrdered];
    __shared__ int members[kClasses];
    __shared__ int chosen;
    for (int i = threadIdx.x; i < kClasses; i += threads) members[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += threads) {
        const int pages = max(1, (seq_len[i] + kPage - 1) / kPage);
        const int of = kClasses - 1 - min(kClasses - 1, (__float_as_int(static_cast<float>(pages)) >> 21) - (127 << 2));      // the two leading bits behind the first
        class_of[i] = static_cast<unsigned char>(of);
        atomicAdd(&members[of], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, mine = members[2 * lane] + members[2 * lane + 1];
        int up_to = mine;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, up_to, offset);
            if (lane >= offset) up_to += other;
        }
        const int owner = __ffs(__ballot_sync(0xffffffffu, up_to > place)) - 1;      // place < n: some lane's
        int left = place - __shfl_sync(0xffffffffu, up_to - mine, owner), of = 2 * owner;
        if (left >= members[of]) left -= members[of++];
        for (int first = 0; first < n; first += 32) {
            const unsigned here = __ballot_sync(0xffffffffu, first + lane < n && class_of[min(first + lane, n - 1)] == of);
            const int count = __popc(here);
            if (left < count) {
                if ((here >> lane & 1u) && __popc(here & ((1u << lane) - 1u)) == left) chosen = first + lane;
                break;
            }
            left -= count;
        }
    }
    __syncthreads();
    return chosen;
}

constexpr int kValueRounds = (D + 127) / 128;      // rounds of 128 columns: a lane holds 16 columns, 8 tiles of 16 rows

// Groups of four warps share the pages of a block's range out, every other page to each of two, and a block's warps are joined in shared memory; accumulators stand in a unit of their own.
template <int NT, bool Runs, int Groups>
__global__ void __launch_bounds__((4 * Groups + 1) * 32, NT == 1 && kHalves == 1 && !Runs && Groups == 1 ? 4 : 2)
decode8_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, const bf16* __restrict__ queries, bf16* __restrict__ out,
               uint8_t* __restrict__ key_pages, uint8_t* __restrict__ value_pages, float* __restrict__ key_scales, float* __restrict__ value_scales, float* __restrict__ partial_o, float* __restrict__ partial_ml,
               const int* __restrict__ seq_len, const int* __restrict__ cu_seqlens, const int* __restrict__ page_rows, int page_stride, int n_heads, int n_kv_heads, int passes, float scale,
               int window, int splits, int clustered, int longest_first, Prepare prepare) {
    constexpr int kHeads = 8 * NT, kWarps = kGroupWarps * Groups, kThreads = (kWarps + 1) * 32, kStages = kStagesOf<Groups>;
    static_assert(Groups == 1 || kHalves == 1, "a group has two stages of its own");
    extern __shared__ uint8_t shared_raw[];
    Shared* shared = reinterpret_cast<Shared*>(shared_raw);
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(shared_raw) + sizeof(Shared) + 1023) & ~uintptr_t(1023));
    // Once every page has been read the stages hold what the warps bring to the join.
    float (*merge_o)[kHeads][D] = reinterpret_cast<float (*)[kHeads][D]>(stages);
    static_assert(kWarps * kHeads * D * 4 <= kStages * kStageBytes, "the join must fit the stages");
    __shared__ float merge_ml[kWarps][kHeads][2];
    __shared__ float block_ml[kHeads][2];
    __shared__ __align__(16) bf16 own[Runs ? 1 : kHeads + 2][D];      // prepared here: queries, then the newest key and value
    __shared__ float greatest_of[2 * kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x;
    const int kv_head = blockIdx.y / passes, pass = blockIdx.y % passes;
    const int group = n_heads / n_kv_heads;
    volatile int* abort_flag = &shared->abort_flag;
    int seq = blockIdx.z;
    if constexpr (!Runs) {
        if (longest_first) seq = by_length(seq_len, gridDim.z, seq);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            barrier_init(&shared->full[s], 2);      // the copies', and the scales'
            barrier_init(&shared->empty[s], kGroupWarps);
        }
        barrier_init(&shared->stored, kWarps);
        shared->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // Heads that are rotated whole (or not at all): a lane holds kNear neighbours of a row, and what it multiplies them with is here before the rows are.  (A step's lengths and the tables are
    // there before its first kernel begins.)
    constexpr bool kVectors = !Runs && (D == 64 || D == 128 || D == 256);
    constexpr int kNear = kVectors ? D / 32 : 1;
    __shared__ float rotation[2][kVectors ? D / 2 : 1];
    const bool near = kVectors && prepare.vectors != 0;
    float q_weights[kNear], k_weights[kNear];
    if constexpr (kVectors) {
        if (near) {
            const size_t row = static_cast<size_t>(max(0, seq_len[seq] - 1)) * (D / 2);
            for (int j = threadIdx.x; j < D / 2; j += kThreads) {
                rotation[0][j] = prepare.rotary_dim ? prepare.cos_table[row + j] : 1.0f;
                rotation[1][j] = prepare.rotary_dim ? prepare.sin_table[row + j] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kNear; ++i) {
                q_weights[i] = prepare.q_weight ? prepare.q_weight[kNear * lane + i] : 1.0f;
                k_weights[i] = prepare.k_weight ? prepare.k_weight[kNear * lane + i] : 1.0f;
            }
            __syncthreads();
        }
    }
    grid_dependency_wait();
    // The block's columns: query heads of the group, or, with `Runs`, pairs of a new token and a head, tokens first.  Column j belongs to row `place(j)` of queries and results.
    const int row0 = Runs ? cu_seqlens[seq] : seq, news = Runs ? cu_seqlens[seq + 1] - row0 : 1;
    const int column0 = pass * kHeads, heads_here = min(kHeads, news * group - column0);
    if (Runs && heads_here <= 0) return;      // the whole cluster: a run shorter than the longest
    auto place = [&](int j) {
        const int column = column0 + j, token = Runs ? column / group : 0;
        return static_cast<size_t>(row0 + token) * n_heads + kv_head * group + (Runs ? column - token * group : column);
    };
    const int start = seq_len[seq] - news, token_lo = Runs ? column0 / group : 0, token_hi = Runs ? (column0 + heads_here - 1) / group : 0;
    // What any of the columns sees.
    const int length = start + token_hi + 1, first = window > 0 ? max(0, start + token_lo + 1 - window) : 0;
    const int first_page = first / kPage, pages_end = (length + kPage - 1) / kPage;
    const int per_split = (max(0, pages_end - first_page) + splits - 1) / splits;
    const int page_lo = first_page + split * per_split, page_hi = min(pages_end, page_lo + per_split);
    const int count = max(0, page_hi - page_lo);
    // The range with the newest position: nobody else reads that page of that head.
    const bool stores = !Runs && prepare.projected != nullptr && prepare.store && count > 0 && page_hi == pages_end;
    float running_max[NT][2], running_sum[NT][2];      // log2 units; the sums and accumulators belong to weights exp2(score - max + 14)
    float unit[2] = {0.0f, 0.0f};      // producer: what one in a group's accumulators stands for, the greatest value scale of its pages so far
    float acc[NT][kValueRounds][8][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        running_max[n][0] = running_max[n][1] = -INFINITY;
        running_sum[n][0] = running_sum[n][1] = 0.0f;
#pragma unroll
        for (int r = 0; r < kValueRounds; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[n][r][i][j] = 0.0f;
    }

    if (warp == kWarps) {
        // ---- the pages, in order: the numbers and scales of 32 at a time, a lane each
        const int* pages = page_rows + static_cast<size_t>(seq) * page_stride;
        bool alive = true;
        int asked = 0;
        for (int base = 0; base < count && alive; base += 32) {
            const bool mine = base + lane < count;
            const int place = mine ? pages[page_lo + base + lane] * n_kv_heads + kv_head : 0;
            const float k_scale = mine ? key_scales[place] : 0.0f, v_scale = mine ? value_scales[place] : 0.0f;
            for (int i = 0; i < min(32, count - base); ++i) {
                const int number = base + i, stage = number % kStages;
                const int box = __shfl_sync(0xffffffffu, place, i);
                bool ready = true;
                if (number >= kStages) ready = barrier_wait(&shared->empty[stage], (number / kStages - 1) & 1, abort_flag);
                if (!__all_sync(0xffffffffu, ready)) {
                    alive = false;
                    break;
                }
                if (stores && number == count - 1 && !__all_sync(0xffffffffu, barrier_wait(&shared->stored, 0, abort_flag))) {
                    alive = false;
                    break;
                }
                if (lane == 0) {
                    barrier_expect_bytes(&shared->full[stage], kStageBytes);
                    uint8_t* tile = stages + stage * kStageBytes;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) tma_load_3d(tile + h * kBoxBytes, &key_map, h * 128, 0, box, &shared->full[stage]);
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) tma_load_3d(tile + kTileBytes + h * kBoxBytes, &value_map, h * 128, 0, box, &shared->full[stage]);
                }
                asked = number + 1;
                // The scales of the stages that were free from the start follow once all their copies are on their way.
                if (number < kStages - 1 && number + 1 < count) continue;
                for (int n = number < kStages ? 0 : number; n <= number; ++n) {
                    float k_of = __shfl_sync(0xffffffffu, k_scale, n - base), v_of = __shfl_sync(0xffffffffu, v_scale, n - base);
                    if (stores && n == count - 1) {
                        k_of = shared->new_key_scale;
                        v_of = shared->new_value_scale;
                    }
                    // A page's value scale joins the weights as its share of the accumulators' unit (powers of two: exact), so a unit that grows rescales them.
                    const bool other = Groups == 2 && (n & 1);
                    const float before = other ? unit[1] : unit[0], grown = fmaxf(before, v_of);
                    if (lane == 0) {
                        shared->key_scale[n % kStages] = k_of;
                        shared->share[n % kStages] = v_of / grown;
                        shared->older[n % kStages] = before / grown;
                        barrier_arrive(&shared->full[n % kStages]);
                    }
                    if (other) unit[1] = grown;
                    else unit[0] = grown;
                }
                __syncwarp();
            }
        }
        if (lane == 0) {
            shared->unit[0] = unit[0];
            shared->unit[1] = unit[1];
            // Whoever gives up, this warp or one that adds: the copies in flight own their stages until they have landed.
            for (int number = max(0, asked - kStages); number < asked; ++number) barrier_outlast(&shared->full[number % kStages], (number / kStages) & 1);
        }
    } else {
        if (!Runs && prepare.projected != nullptr && count > 0) {
            // ---- the token's own rows, one to a warp at a time
            const int position = length - 1;
            const bf16* from = prepare.projected + static_cast<size_t>(seq) * prepare.stride;
            const float* cosines = prepare.cos_table + static_cast<size_t>(position) * (prepare.rotary_dim / 2);
            const float* sines = prepare.sin_table + static_cast<size_t>(position) * (prepare.rotary_dim / 2);
            const int tasks = heads_here + (stores ? 2 : 0);
            if constexpr (kVectors) {
                if (near) {
                    // All of the warp's rows are on their way together; the arithmetic is that of the 16-bit cache's prepare kernel for such heads.
                    typedef Neighbours<kNear> Near;
                    constexpr int kMost = (kHeads + 2 + kWarps - 1) / kWarps;
                    Near raw[kMost];
#pragma unroll
                    for (int a = 0; a < kMost; ++a) {
                        const int task = warp + kWarps * a;
                        const int head = task == heads_here ? n_heads + kv_head : task == heads_here + 1 ? n_heads + n_kv_heads + kv_head : kv_head * group + task;
                        if (task < tasks) raw[a] = *reinterpret_cast<const Near*>(from + static_cast<size_t>(head) * D + kNear * lane);
                    }
#pragma unroll
                    for (int a = 0; a < kMost; ++a) {
                        const int task = warp + kWarps * a;
                        if (task >= tasks) break;
                        const bool is_key = task == heads_here, is_value = task == heads_here + 1;
                        Near* row = reinterpret_cast<Near*>(own[is_key ? kHeads : is_value ? kHeads + 1 : task]) + lane;
                        if (is_value) {
                            *row = raw[a];
                            continue;
                        }
                        *row = prepare_neighbours<kNear>(raw[a], is_key ? prepare.k_weight != nullptr : prepare.q_weight != nullptr, is_key ? k_weights : q_weights, prepare.eps,
                                                         prepare.rotary_dim != 0, &rotation[0][kNear * (lane & 15)], &rotation[1][kNear * (lane & 15)], lane);
                    }
                }
            }
            for (int task = near ? tasks : warp; task < tasks; task += kWarps) {
                const bool is_key = task == heads_here, is_value = task == heads_here + 1;
                const int head = is_key ? n_heads + kv_head : is_value ? n_heads + n_kv_heads + kv_head : kv_head * group + task;
                bf16* row = own[is_key ? kHeads : is_value ? kHeads + 1 : task];
                for (int e = lane; e < D; e += 32) row[e] = from[static_cast<size_t>(head) * D + e];
                __syncwarp();
                prepare_row(row, is_value ? nullptr : is_key ? prepare.k_weight : prepare.q_weight, prepare.eps, cosines, sines, is_value ? 0 : prepare.rotary_dim, D, lane);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");      // every consumer warp comes here before any of its waits
            if (stores) {
                const size_t place_of = static_cast<size_t>(page_rows[static_cast<size_t>(seq) * page_stride + position / kPage]) * n_kv_heads + kv_head;
                const int older = position % kPage;
                const float k_of = store_in_page<kWarps * 32>(own[Runs ? 0 : kHeads], 1, D, older, key_pages + place_of * kPage * D, key_scales + place_of, greatest_of);
                const float v_of = store_in_page<kWarps * 32>(own[Runs ? 0 : kHeads + 1], 1, D, older, value_pages + place_of * kPage * D, value_scales + place_of, greatest_of + kWarps);
                if (threadIdx.x == 0) {
                    key_scales[place_of] = shared->new_key_scale = k_of;
                    value_scales[place_of] = shared->new_value_scale = v_of;
                }
                asm volatile("fence.proxy.async;" ::: "memory");      // the page is read back by a copy
                __syncwarp();
                if (lane == 0) barrier_arrive(&shared->stored);
            }
        }
        // ---- queries: this lane's elements of heads g (and g + 8), brought to [1, 2) per head
        unsigned q_frag[NT][kKeySteps][2];
        float q_power[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int head = n * 8 + g;
            const bool live = head < heads_here && count > 0;
            const bf16* row = !Runs && prepare.projected != nullptr ? own[live ? head : 0] : queries + place(live ? head : 0) * D;
            float greatest = 0.0f;
#pragma unroll
            for (int step = 0; step < kKeySteps; ++step) {
                const uint2 raw = live ? *reinterpret_cast<const uint2*>(row + key_element(step, t, 0)) : make_uint2(0u, 0u);
                q_frag[n][step][0] = raw.x;
                q_frag[n][step][1] = raw.y;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    greatest = fmaxf(greatest, finite_magnitude(__uint_as_float(q_frag[n][step][i] << 16)));
                    greatest = fmaxf(greatest, finite_magnitude(__uint_as_float(q_frag[n][step][i] & 0xffff0000u)));
                }
            }
            greatest = fmaxf(greatest, __shfl_xor_sync(0xffffffffu, greatest, 1));
            greatest = fmaxf(greatest, __shfl_xor_sync(0xffffffffu, greatest, 2));
            const int exponent = min(max(static_cast<int>(__float_as_uint(greatest) >> 23) - 127, -100), 126);
            const float inverse = power_of_two(-exponent);
            q_power[n] = power_of_two(exponent);
#pragma unroll
            for (int step = 0; step < kKeySteps; ++step)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    q_frag[n][step][i] = pack_half2(__uint_as_float(q_frag[n][step][i] << 16) * inverse, __uint_as_float(q_frag[n][step][i] & 0xffff0000u) * inverse);
        }
        // The factor of the scores of heads 2t and 2t + 1, but for the page's scale (log2 units).
        float factor[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) factor[n][h] = __shfl_sync(0xffffffffu, q_power[n], (2 * t + h) * 4) * scale * kLog2e;

        // With `Runs` each column sees up to its token's own position, and from its own window's begin on.
        int column_end[NT][2], column_first[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                column_end[n][h] = Runs ? start + (column0 + n * 8 + 2 * t + h) / group + 1 : length;
                column_first[n][h] = Runs && window > 0 ? max(0, column_end[n][h] - window) : first;
            }
        const int page_part = (warp & (kGroupWarps - 1)) * 16;      // this warp's positions of a page
        bool alive = true;
        for (int number = Groups == 1 ? 0 : warp / kGroupWarps; number < count; number += Groups) {
            const int stage = number % kStages;
            alive = __all_sync(0xffffffffu, barrier_wait(&shared->full[stage], (number / kStages) & 1, abort_flag));
            if (!alive) break;
            const int base = (page_lo + number) * kPage + page_part;      // position of this warp's first key
            if (base < length && base + 16 > first) {
                const uint8_t* key_tile = stages + stage * kStageBytes;
                const uint8_t* value_tile = key_tile + kTileBytes;
                const float k_scale = shared->key_scale[stage], share = shared->share[stage], older = shared->older[stage];
                const bool whole = base >= first && base + 16 <= length;
                // Scores of 16 keys and 8 heads: rows g and g + 8 are keys base + g and base + g + 8.
                float score[NT][4], score_odd[NT][4];      // two chains, so that consecutive products do not wait for each other
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) score[n][j] = score_odd[n][j] = 0.0f;
                const int row_lo = page_part + g, row_hi = row_lo + 8;
                constexpr int kGroups = D / 64;
#pragma unroll
                for (int c = 0; c < kGroups; ++c) {
                    // Odd rows take the groups of a pair in the other order, so that eight lanes read 128 different bytes.
                    const int swapped = (c ^ 1) < kGroups && (g & 1) ? c ^ 1 : c;
                    uint4 lo = page_chunk(key_tile, row_lo, swapped * 4 + t), hi = page_chunk(key_tile, row_hi, swapped * 4 + t);
                    if ((c ^ 1) < kGroups) {
                        if (c & 1) continue;
                        uint4 lo2 = page_chunk(key_tile, row_lo, (swapped ^ 1) * 4 + t), hi2 = page_chunk(key_tile, row_hi, (swapped ^ 1) * 4 + t);
                        const bool turn = (g & 1) != 0;
                        const uint4 lo_first = turn ? lo2 : lo, lo_second = turn ? lo : lo2, hi_first = turn ? hi2 : hi, hi_second = turn ? hi : hi2;
                        const unsigned low[8] = {lo_first.x, lo_first.y, lo_first.z, lo_first.w, lo_second.x, lo_second.y, lo_second.z, lo_second.w};
                        const unsigned high[8] = {hi_first.x, hi_first.y, hi_first.z, hi_first.w, hi_second.x, hi_second.y, hi_second.z, hi_second.w};
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const unsigned a0 = decode_half2(low[j]), a2 = decode_half2(low[j] >> 16), a1 = decode_half2(high[j]), a3 = decode_half2(high[j] >> 16);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(j & 1 ? score_odd[n] : score[n], a0, a1, a2, a3, q_frag[n][c * 4 + j][0], q_frag[n][c * 4 + j][1]);
                        }
                    } else {
                        const unsigned low[4] = {lo.x, lo.y, lo.z, lo.w}, high[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const unsigned a0 = decode_half2(low[j]), a2 = decode_half2(low[j] >> 16), a1 = decode_half2(high[j]), a3 = decode_half2(high[j] >> 16);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(j & 1 ? score_odd[n] : score[n], a0, a1, a2, a3, q_frag[n][c * 4 + j][0], q_frag[n][c * 4 + j][1]);
                        }
                    }
                }
#pragma unroll
                for (int step = kGroups * 4; step < kKeySteps; ++step) {
                    const unsigned low = page_word(key_tile, row_lo, step * 16 + t * 4), high = page_word(key_tile, row_hi, step * 16 + t * 4);
                    const unsigned a0 = decode_half2(low), a2 = decode_half2(low >> 16), a1 = decode_half2(high), a3 = decode_half2(high >> 16);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(step & 1 ? score_odd[n] : score[n], a0, a1, a2, a3, q_frag[n][step][0], q_frag[n][step][1]);
                }
                // Keys whose values are not finite, where some columns see a key that others do not: they count as zeros below, and as NaN in the scores of the columns that see them.
                unsigned odd_keys = 0;
                if constexpr (Runs) {
                    if (base + 16 > start + token_lo + 1 || (window > 0 && base < length - window)) {
                        const int slots[4] = {2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9};
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            unsigned odd = 0;
#pragma unroll
                            for (int r = 0; r < kValueRounds; ++r) {
                                if ((8 * r + g) * 16 >= D) continue;
                                const uint4 v = page_chunk(value_tile, page_part + slots[s], 8 * r + g);
                                odd |= __vcmpeq4(v.x & 0x7f7f7f7fu, 0x7f7f7f7fu) | __vcmpeq4(v.y & 0x7f7f7f7fu, 0x7f7f7f7fu) | __vcmpeq4(v.z & 0x7f7f7f7fu, 0x7f7f7f7fu) |
                                       __vcmpeq4(v.w & 0x7f7f7f7fu, 0x7f7f7f7fu);
                            }
                            const unsigned who = __ballot_sync(0xffffffffu, odd != 0u);
#pragma unroll
                            for (int other = 0; other < 4; ++other)
                                if (who & (0x11111111u << other)) odd_keys |= 1u << (2 * other + (s & 1) + 8 * (s >> 1));
                        }
                    }
                }
                const bool apart = share < kLeastShare;      // a 16-bit weight would lose bits: the page's sums are taken apart and added in 32 bits
                const float by_share = apart ? 1.0f : share;
                bool moved = older != 1.0f;
                float correction[NT][2];
                unsigned pb0[NT], pb1[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float p[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float by = factor[n][h] * k_scale;
                        const bool live_lo = base + g >= column_first[n][h] && base + g < column_end[n][h], live_hi = base + g + 8 >= column_first[n][h] && base + g + 8 < column_end[n][h];
                        const float nan = __uint_as_float(0x7fffffffu);
                        const float low = !live_lo ? -INFINITY : Runs && (odd_keys >> g & 1u) ? nan : (score[n][h] + score_odd[n][h]) * by;
                        const float high = !live_hi ? -INFINITY : Runs && (odd_keys >> (g + 8) & 1u) ? nan : (score[n][2 + h] + score_odd[n][2 + h]) * by;
                        float most = fmaxf(low, high);
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                        const float new_max = fmaxf(running_max[n][h], most);      // finite where one of the 16 keys is visible: always, but for columns of a run
                        moved |= new_max != running_max[n][h];
                        const float from = Runs && new_max == -INFINITY ? 0.0f : new_max;
                        correction[n][h] = exp2f(running_max[n][h] - from);
                        running_max[n][h] = new_max;
                        p[h] = exp2f(low - from + kWeightBits);
                        p[2 + h] = exp2f(high - from + kWeightBits);
                        running_sum[n][h] = running_sum[n][h] * correction[n][h] + p[h] + p[2 + h];
                    }
                    pb0[n] = pack_half2(p[0] * by_share, p[1] * by_share);
                    pb1[n] = pack_half2(p[2] * by_share, p[3] * by_share);
                    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb0[n]) : "r"(pb0[n]));
                    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb1[n]) : "r"(pb1[n]));
                }
                if (__any_sync(0xffffffffu, moved)) {      // in a long context almost never
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int r = 0; r < kValueRounds; ++r)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
#pragma unroll
                                for (int j = 0; j < 4; ++j) acc[n][r][i][j] *= correction[n][j & 1] * older;
                }
                // Values of keys 2t, 2t + 1, 2t + 8, 2t + 9, columns 128 r + 16 g .. + 16.
#pragma unroll
                for (int r = 0; r < kValueRounds; ++r) {
                    const int chunk = 8 * r + g;
                    uint4 v[4];
                    const int slots[4] = {2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9};
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        v[s] = chunk * 16 < D ? page_chunk(value_tile, page_part + slots[s], chunk) : make_uint4(0u, 0u, 0u, 0u);
                        // What nobody sees may be NaN, and a weight of zero would not hide that.
                        if ((!whole && (base + slots[s] < first || base + slots[s] >= length)) || (Runs && (odd_keys >> slots[s] & 1u))) v[s] = make_uint4(0u, 0u, 0u, 0u);
                    }
                    const unsigned w0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, w1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
                    const unsigned w8[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, w9[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
                    auto tile = [&](int i, unsigned (&a)[4]) {      // columns 2 i (row g) and 2 i + 1 (row g + 8) of this lane's 16
                        const unsigned pick = (i & 1) ? 0x7362u : 0x5140u;
                        const unsigned near = __byte_perm(w0[i >> 1], w1[i >> 1], pick), far = __byte_perm(w8[i >> 1], w9[i >> 1], pick);
                        a[0] = decode_half2(near);
                        a[1] = decode_half2(near >> 16);
                        a[2] = decode_half2(far);
                        a[3] = decode_half2(far >> 16);
                    };
                    if (!apart) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            unsigned a[4];
                            tile(i, a);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(acc[n][r][i], a[0], a[1], a[2], a[3], pb0[n], pb1[n]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            unsigned a[4];
                            tile(i, a);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma_f16(part, a[0], a[1], a[2], a[3], pb0[n], pb1[n]);
#pragma unroll
                                for (int j = 0; j < 4; ++j) acc[n][r][i][j] = fmaf(part[j], share, acc[n][r][i][j]);
                            }
                        }
                    }
                }
            } else if (shared->older[stage] != 1.0f) {      // nothing of the page is this warp's, but its unit is
                const float older = shared->older[stage];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < kValueRounds; ++r)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[n][r][i][j] *= older;
            }
            __syncwarp();
            if (lane == 0) barrier_arrive(&shared->empty[stage]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                running_sum[n][h] += __shfl_xor_sync(0xffffffffu, running_sum[n][h], 4);
                running_sum[n][h] += __shfl_xor_sync(0xffffffffu, running_sum[n][h], 8);
                running_sum[n][h] += __shfl_xor_sync(0xffffffffu, running_sum[n][h], 16);
            }
    }
    __syncthreads();      // the stages are done with
    grid_dependents_launch();      // only now: what starts beside this kernel takes room that its own later blocks, or clusters, wait for
    if (warp < kWarps) {
        const float one = shared->unit[Groups == 1 ? 0 : warp / kGroupWarps];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int head = n * 8 + 2 * t + h;
#pragma unroll
                for (int r = 0; r < kValueRounds; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int column = 128 * r + 16 * g + 2 * i;
                        if (column < D) *reinterpret_cast<float2*>(&merge_o[warp][head][column]) = make_float2(acc[n][r][i][h] * one, acc[n][r][i][2 + h] * one);
                    }
                if (g == 0) {
                    merge_ml[warp][head][0] = running_max[n][h];
                    merge_ml[warp][head][1] = running_sum[n][h];
                }
            }
    }
    __syncthreads();
    const bool failed = *abort_flag != 0;
    for (int index = threadIdx.x; index < heads_here * D; index += kThreads) {
        const int h = index / D, c = index % D;
        float total_max = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) total_max = fmaxf(total_max, merge_ml[w][h][0]);
        float o = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (merge_ml[w][h][1] == 0.0f) continue;      // saw no key
            const float by = exp2f(merge_ml[w][h][0] - total_max);
            o += merge_o[w][h][c] * by;
            sum += merge_ml[w][h][1] * by;
        }
        if (splits == 1) {
            if (!failed) out[place(h) * D + c] = __float2bfloat16_rn(sum != 0.0f ? o / sum : 0.0f);      // a sequence without positions: zeros
        } else if (clustered) {
            merge_o[0][h][c] = o;      // this thread alone reads and writes (h, c) of the first warp's part
            if (c == 0) {
                block_ml[h][0] = total_max;
                block_ml[h][1] = sum;
            }
        } else {
            const size_t slot = place(h) * splits + split;
            if (sum != 0.0f && !failed) partial_o[slot * D + c] = o;
            if (c == 0) {
                partial_ml[slot * 2] = total_max;
                partial_ml[slot * 2 + 1] = failed ? kFailed : sum;
            }
        }
    }
    if (splits == 1 || !clustered) return;
    cluster_share_abort(&shared->abort_flag, splits);
    cluster_sync_all();
    if (*abort_flag == 0) {
        const int rank = blockIdx.x;      // the cluster spans the grid's x
        for (int index = rank * kThreads + threadIdx.x; index < heads_here * D; index += splits * kThreads) {
            const int h = index / D, c = index % D;
            const uint32_t o_address = smem_address(&merge_o[0][h][c]), ml_address = smem_address(&block_ml[h][0]);
            float split_max[kMostClustered], split_sum[kMostClustered], split_o[kMostClustered];
#pragma unroll
            for (int s = 0; s < kMostClustered; ++s) {
                split_max[s] = -INFINITY;
                split_sum[s] = split_o[s] = 0.0f;
                if (s < splits) {
                    const uint32_t remote = cluster_address_of(ml_address, s);
                    split_max[s] = cluster_load(remote);
                    split_sum[s] = cluster_load(remote + 4);
                    split_o[s] = cluster_load(cluster_address_of(o_address, s));
                }
            }
            float total_max = -INFINITY;
#pragma unroll
            for (int s = 0; s < kMostClustered; ++s) total_max = fmaxf(total_max, split_max[s]);
            float o = 0.0f, sum = 0.0f;
#pragma unroll
            for (int s = 0; s < kMostClustered; ++s) {
                if (split_sum[s] == 0.0f) continue;      // a range without a position
                const float by = exp2f(split_max[s] - total_max);
                o += split_o[s] * by;
                sum += split_sum[s] * by;
            }
            out[place(h) * D + c] = __float2bfloat16_rn(sum != 0.0f ? o / sum : 0.0f);
        }
    }
    cluster_sync_all();      // nobody leaves while its results are read
}

// Joins the records of a sequence's ranges in their order: a block (of whole warps) to a head, a thread to a column.  A head of which a range failed is left as it was, and
// so are rows behind the last run (`cu_seqlens`), of which there are no records.
__global__ void join_kernel(const float* __restrict__ partial_o, const float* __restrict__ partial_ml, bf16* __restrict__ out, const int* __restrict__ cu_seqlens, int n_seqs, int n_heads,
                            int splits) {
    grid_dependents_launch();
    grid_dependency_wait();
    if (cu_seqlens && static_cast<int>(blockIdx.y) >= cu_seqlens[n_seqs]) return;
    __shared__ float factor[256];
    __shared__ float inverse;
    __shared__ bool failed;
    const int head = blockIdx.x, seq = blockIdx.y;
    const size_t base = (static_cast<size_t>(seq) * n_heads + head) * splits;
    if (threadIdx.x < 32) {
        float total_max = -INFINITY, sum = 0.0f;
        bool lost = false;
        for (int s = threadIdx.x; s < splits; s += 32) {
            const float own = partial_ml[(base + s) * 2 + 1];
            if (own != 0.0f) total_max = fmaxf(total_max, partial_ml[(base + s) * 2]);
            lost |= own == kFailed;
        }
        total_max = warp_max(total_max);
        lost = __any_sync(0xffffffffu, lost);
        for (int s = threadIdx.x; s < splits; s += 32) {
            const float own = partial_ml[(base + s) * 2 + 1];
            factor[s] = own != 0.0f ? exp2f(partial_ml[(base + s) * 2] - total_max) : 0.0f;
            sum += own != 0.0f ? own * factor[s] : 0.0f;
        }
        sum = warp_sum(sum);
        if (threadIdx.x == 0) {
            inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
            failed = lost;
        }
    }
    __syncthreads();
    if (failed) return;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
        float o = 0.0f;
#pragma unroll 8
        for (int s = 0; s < splits; ++s) {
            const float by = factor[s];
            const float value = by != 0.0f ? partial_o[(base + s) * D + c] : 0.0f;      // a range without a position left no context
            o += value * by;
        }
        out[(static_cast<size_t>(seq) * n_heads + head) * D + c] = __float2bfloat16_rn(o * inverse);
    }
}

int page_map(CUtensorMap* map, const void* pages, long long boxes) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t extents[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(kPage), static_cast<cuuint64_t>(boxes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(D) * kPage};
    const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(kPage), 1};      // rows shorter than a box are filled with zeros
    const cuuint32_t steps[3] = {1, 1, 1};
    const CUresult result = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pages), extents, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return result == CUDA_SUCCESS ? 0 : cudaErrorInvalidValue;
}

template <int Groups>
constexpr int shared_bytes() { return static_cast<int>(sizeof(Shared)) + 1024 + kStagesOf<Groups> * kStageBytes; }

// Multiprocessors of the current device, asked for once.
int multiprocessors() {
    static int counts[64] = {};
    int device = 0, count = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 1;
    if (device < 64 && counts[device]) return counts[device];
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || count < 1) return 1;
    if (device < 64) counts[device] = count;
    return count;
}

struct Call {
    const bf16* queries;
    bf16* out;
    uint8_t *key_pages, *value_pages;
    float *key_scales, *value_scales, *partial_o, *partial_ml;
    const int *seq_len, *cu_seqlens, *page_rows;
    int page_stride, n_seqs, n_tokens, n_heads, n_kv_heads, passes;
    float scale;
    int window, splits;
    Prepare prepare;
};

template <int NT, bool Runs, int Groups>
int launch_groups(const CUtensorMap& key_map, const CUtensorMap& value_map, const Call& c, cudaStream_t stream) {
    static bool ready[64] = {};
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess) return static_cast<int>(status);
    if (device >= 64 || !ready[device]) {
        status = cudaFuncSetAttribute(decode8_kernel<NT, Runs, Groups>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes<Groups>());
        if (status != cudaSuccess) return static_cast<int>(status);
        if (device < 64) ready[device] = true;
    }
    const dim3 grid(c.splits, c.n_kv_heads * c.passes, c.n_seqs);
    const bool clustered = c.splits > 1 && c.splits <= kMostClustered;
    // Long sequences start first, so that the SMs share them out and short ones fill what is left at the end, up to three times as many blocks as there are places: 40 of 64 to 6,000
    // positions 74 -> 59 us, 64 of up to 2,048 46 -> 36, 200 of up to 1,000 58 -> 52, 8 of 2,048 no slower; beyond that putting them in order costs a block more than it gives
    // (256 of up to 300: 36 -> 38).
    const long long places = static_cast<long long>(multiprocessors()) * (NT == 1 && kHalves == 1 && !Runs && Groups == 1 ? 4 : 2), blocks = static_cast<long long>(grid.x) * grid.y * grid.z;
    const int longest_first = !Runs && c.n_seqs > 1 && c.n_seqs <= kMostOrdered && blocks <= 3 * places;
    // Beside the kernel before it only where all blocks find room at once (8 sequences of 2,048 positions 14.4 -> 13.9 us; 640 blocks of 40 sequences 73 -> 78).
    const bool early = blocks <= places;
    int code;
    if (clustered)
        code = tau_launch_clusters_as(early, c.splits, decode8_kernel<NT, Runs, Groups>, grid, dim3((kGroupWarps * Groups + 1) * 32), shared_bytes<Groups>(), stream, key_map, value_map, c.queries, c.out, c.key_pages, c.value_pages, c.key_scales, c.value_scales,
                                      c.partial_o, c.partial_ml, c.seq_len, c.cu_seqlens, c.page_rows, c.page_stride, c.n_heads, c.n_kv_heads, c.passes, c.scale, c.window, c.splits, 1, longest_first, c.prepare);
    else
        code = tau_launch_as(early, decode8_kernel<NT, Runs, Groups>, grid, dim3((kGroupWarps * Groups + 1) * 32), shared_bytes<Groups>(), stream, key_map, value_map, c.queries, c.out, c.key_pages, c.value_pages, c.key_scales, c.value_scales, c.partial_o,
                             c.partial_ml, c.seq_len, c.cu_seqlens, c.page_rows, c.page_stride, c.n_heads, c.n_kv_heads, c.passes, c.scale, c.window, c.splits, 0, longest_first, c.prepare);
    if (code == 0 && c.splits > kMostClustered)
        code = tau_launch(join_kernel, dim3(c.n_heads, c.n_tokens), dim3(D < 128 ? (D + 31) / 32 * 32 : 128), 0, stream, c.partial_o, c.partial_ml, c.out, c.cu_seqlens, c.n_seqs, c.n_heads, c.splits);
    return code ? code : tau_launch_status();
}

template <int NT, bool Runs>
int launch(const CUtensorMap& key_map, const CUtensorMap& value_map, const Call& c, cudaStream_t stream) {
    // Two groups of warps where all their blocks, two to an SM, fit at once, one to an SM in clusters of more than four, which find room less easily (a decode step of 8 layers, ms in one
    // group and two: one sequence of 300 positions 0.556 and 0.541, of 16,000 0.72 and 0.68; 8 of 2,000 in two ranges 0.683 and 0.641; 4 of 1,000 in four ranges 0.630 and 0.601, in
    // eight 0.608 and 0.646).
    if constexpr (NT == 1 && kHalves == 1 && !Runs) {
        const bool crowded = c.splits > 4 && c.splits <= kMostClustered;
        if (static_cast<long long>(c.splits) * c.n_kv_heads * c.passes * c.n_seqs <= (crowded ? 1 : 2) * multiprocessors()) return launch_groups<NT, Runs, 2>(key_map, value_map, c, stream);
    }
    return launch_groups<NT, Runs, 1>(key_map, value_map, c, stream);
}

}  // namespace

// Columns to a block: 16 where there are more than 8 and a head's accumulators leave room for them.
static int columns_to_a_block(long long columns) { return columns > 8 && D <= 128 ? 16 : 8; }

TAU_EXPORT int tau_decode8_status() {
    int flag = 0;
    cudaDeviceSynchronize();
    if (cudaMemcpyFromSymbol(&flag, wait_error, sizeof(flag)) != cudaSuccess) return -1;
    return flag;
}

// bfloat16 queries and output [tokens, n_heads D]; pages [boxes / n_kv_heads, n_kv_heads, 64, D] of e4m3 codes with scales [boxes].  `cu_seqlens` == nullptr: one token to
// a sequence; else the runs' bounds, none longer than `max_new`.  `projected` != nullptr (single tokens, a group of query heads that one block serves):
// `queries` is not read, see `Prepare`.  More than 8 splits need scratch of n_tokens * n_heads * splits * (D + 2) floats.
TAU_EXPORT int tau_decode8(const void* queries, void* key_pages, void* value_pages, float* key_scales, float* value_scales, void* out, const int* seq_len,
                           const int* cu_seqlens, const int* page_rows, int page_stride, long long boxes, int n_seqs, int n_tokens, int max_new, int n_heads, int n_kv_heads, float scale,
                           int window, int splits, float* scratch, long long scratch_floats, const void* projected, long long projected_stride, const float* q_weight, const float* k_weight,
                           float eps, const float* cos_table, const float* sin_table, int rotary_dim, int store, void* stream) {
    if (n_seqs <= 0 || n_tokens <= 0) return 0;
    if ((!queries && !projected) || !key_pages || !value_pages || !key_scales || !value_scales || !out || !seq_len || !page_rows || page_stride <= 0 || boxes <= 0 || n_heads <= 0 || n_kv_heads <= 0 ||
        n_heads % n_kv_heads != 0 || window < 0 || splits < 1 || splits > 256 || n_seqs > 65535 || n_tokens > 65535 || max_new < 1 || (!cu_seqlens && (max_new != 1 || n_tokens != n_seqs)) ||
        boxes > 0x7fffffffll || (reinterpret_cast<uintptr_t>(queries) & 7) ||
        (projected && (cu_seqlens || rotary_dim < 0 || rotary_dim > D || (rotary_dim & 1) || (rotary_dim > 0 && (!cos_table || !sin_table)))) ||
        (splits > kMostClustered && (!scratch || scratch_floats < static_cast<long long>(n_tokens) * n_heads * splits * (D + 2))))
        return cudaErrorInvalidValue;
    const long long columns = static_cast<long long>(n_heads / n_kv_heads) * max_new;
    const int to_a_block = columns_to_a_block(columns);
    if (n_kv_heads * ((columns + to_a_block - 1) / to_a_block) > 65535 || (projected && columns > to_a_block)) return cudaErrorInvalidValue;      // a page is stored by one block alone
    CUtensorMap key_map, value_map;
    int status = page_map(&key_map, key_pages, boxes);
    if (!status) status = page_map(&value_map, value_pages, boxes);
    if (status) return status;
    const Call call = {static_cast<const bf16*>(queries), static_cast<bf16*>(out), static_cast<uint8_t*>(key_pages), static_cast<uint8_t*>(value_pages), key_scales, value_scales, scratch,
                       scratch ? scratch + static_cast<size_t>(n_tokens) * n_heads * splits * D : nullptr, seq_len, cu_seqlens, page_rows, page_stride, n_seqs, n_tokens, n_heads, n_kv_heads,
                       static_cast<int>((columns + to_a_block - 1) / to_a_block), scale, window, splits,
                       {static_cast<const bf16*>(projected), projected_stride, q_weight, k_weight, eps, cos_table, sin_table, rotary_dim, store,
                        projected && (D == 64 || D == 128 || D == 256) && (rotary_dim == 0 || rotary_dim == D) && (projected_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(projected) & 15) == 0}};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if constexpr (D <= 128)
        if (to_a_block == 16) return cu_seqlens ? launch<2, true>(key_map, value_map, call, s) : launch<2, false>(key_map, value_map, call, s);
    return cu_seqlens ? launch<1, true>(key_map, value_map, call, s) : launch<1, false>(key_map, value_map, call, s);
}
