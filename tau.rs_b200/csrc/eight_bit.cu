// Weights, activations and caches held in 8 bits (e4m3): quantising, the plain product over such operands, the store into cache pages
// and the pages read back.  The rule of scales is in eight_bit.cuh.
//
// The reference keeps weights and caches in 16 and 32 bits (crates/models/src/components/gated_attention/kv_cache.rs:12-24); this is
// the library's own.
#include "quantize_rows.cuh"

namespace {

// ---- quantising ---------------------------------------------------------------------------------------------------------------------
// One block to 128 x 128 values of a weight; a thread holds 64 of them between the maximum and the codes, so the weight is read once.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_blocks_kernel(const T* __restrict__ values, long long stride, uint8_t* __restrict__ codes, float* __restrict__ scales, int rows, int columns) {
    grid_dependency_wait();      // and nothing starts beside this kernel: products ask for their weight before what is in front of them has ended
    __shared__ float greatest_of[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = blockIdx.y * kScaleBlock, column = blockIdx.x * kScaleBlock + lane * 4;
    float held[16][4];
    float greatest = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = row0 + warp + 8 * i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            held[i][j] = (row < rows && column + j < columns) ? to_float(values[static_cast<size_t>(row) * stride + column + j]) : 0.0f;
            greatest = fmaxf(greatest, finite_magnitude(held[i][j]));
        }
    }
    greatest = warp_max(greatest);
    if (lane == 0) greatest_of[warp] = greatest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) greatest = fmaxf(greatest, greatest_of[w]);
    const int exponent = scale_exponent(greatest);
    const float inverse = power_of_two(-exponent);
    if (threadIdx.x == 0) scales[static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x] = power_of_two(exponent);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = row0 + warp + 8 * i;
        if (row >= rows || column >= columns) continue;      // columns are a multiple of 16: a group of four is whole or absent
        *reinterpret_cast<unsigned*>(codes + static_cast<size_t>(row) * columns + column) = encode_four(held[i][0], held[i][1], held[i][2], held[i][3], inverse);
    }
}

// ---- the plain product ----------------------------------------------------------------------------------------------------------------
// 32 rows x 32 features to a block of 256 threads, four results to a thread; 32 columns at a time in shared memory, decoded.  The sum
// over a block of 128 columns is kept apart and joins times both scales.  The kernel that the fast ones are checked against.
template <typename TOut>
__global__ void __launch_bounds__(256)
gemm8_simt_kernel(const uint8_t* __restrict__ x, const float* __restrict__ x_scales, const uint8_t* __restrict__ w, const float* __restrict__ w_scales,
                  const float* __restrict__ bias, TOut* __restrict__ out, int M, int N, int K, long long out_stride) {
    grid_dependents_launch();
    grid_dependency_wait();
    __shared__ float x_tile[32][33], w_tile[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int feature = blockIdx.x * 32 + tx, across = (K + kScaleBlock - 1) / kScaleBlock;
    const int row0 = blockIdx.y * 32;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < K; k0 += 32) {
        __syncthreads();
        {   // 32 x 8 words of four codes from each operand, one to a thread
            const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4;
            float values[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row0 + r < M && k0 + c < K) decode_four(*reinterpret_cast<const unsigned*>(x + static_cast<size_t>(row0 + r) * K + k0 + c), values);
#pragma unroll
            for (int j = 0; j < 4; ++j) x_tile[r][c + j] = values[j];
            float weights[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (static_cast<int>(blockIdx.x) * 32 + r < N && k0 + c < K)
                decode_four(*reinterpret_cast<const unsigned*>(w + static_cast<size_t>(blockIdx.x * 32 + r) * K + k0 + c), weights);
#pragma unroll
            for (int j = 0; j < 4; ++j) w_tile[r][c + j] = weights[j];
        }
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < 32; ++k) {
            const float weight = w_tile[tx][k];
#pragma unroll
            for (int i = 0; i < 4; ++i) part[i] = fmaf(x_tile[ty + 8 * i][k], weight, part[i]);
        }
        if ((k0 + 32) % kScaleBlock == 0 || k0 + 32 >= K) {
            const int block = k0 / kScaleBlock;
            const float w_scale = feature < N ? w_scales[static_cast<size_t>(feature / kScaleBlock) * across + block] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row0 + ty + 8 * i;
                if (row < M) sum[i] = fmaf(part[i], x_scales[static_cast<size_t>(block) * M + row] * w_scale, sum[i]);
                part[i] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + ty + 8 * i;
        if (row < M && feature < N) out[static_cast<size_t>(row) * out_stride + feature] = from_float<TOut>(sum[i] + (bias ? bias[feature] : 0.0f));
    }
}

// What a gated product makes of the rows that an ungated one left: groups of 8 gate columns and their 8 up columns.
__global__ void gate_groups_kernel(const bf16* __restrict__ stacked, bf16* __restrict__ out, long long count, int inner, long long out_stride, float limit) {
    grid_dependents_launch();
    grid_dependency_wait();
    const long long index = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (index >= count) return;
    const long long row = index / inner;
    const int column = static_cast<int>(index % inner);
    const bf16* source = stacked + row * 2 * inner + (column >> 3) * 16 + (column & 7);
    out[row * out_stride + column] = __float2bfloat16_rn(gated_value(to_float(source[0]), to_float(source[8]), limit));
}

// ---- the cache ------------------------------------------------------------------------------------------------------------------------
constexpr int kPage = 64;

// How keys, values and queries of new tokens come: as they are to be kept (`prepared` false), or as a stacked projection left them: then
// queries and keys are normalised per head (rounded to bfloat16), rotated in 32 bits (rounded again), and queries written out.
struct StoreSource {
    const bf16* keys;             // head h of token i at keys + i * key_stride + h * D
    const bf16* values;
    long long key_stride, value_stride;
    const bf16* query_rows;       // or nullptr: no queries
    long long query_stride;
    bf16* queries;                // [tokens, n_heads * D]
    const float* q_weight;        // or nullptr: no norm
    const float* k_weight;
    float eps;
    const float* cos_table;       // [positions, rotary_dim / 2]
    const float* sin_table;
    int rotary_dim;
    int n_heads;
};
constexpr int kQueryHeads = 4;      // query heads to a block

// A lane's norm weights, and its share of the rotation's tables at a position.
template <int PER>
struct Prepared {
    float weight[PER];
    __device__ __forceinline__ Prepared(const float* __restrict__ from, int lane) {
#pragma unroll
        for (int i = 0; i < PER; ++i) weight[i] = from ? __ldg(from + PER * lane + i) : 1.0f;
    }
};
template <int PER>
__device__ __forceinline__ void angles(const StoreSource& source, int position, int lane, float (&cosines)[PER], float (&sines)[PER]) {
    const size_t table = static_cast<size_t>(position) * (16 * PER) + PER * (lane & 15);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        cosines[i] = source.rotary_dim ? __ldg(source.cos_table + table + i) : 1.0f;
        sines[i] = source.rotary_dim ? __ldg(source.sin_table + table + i) : 0.0f;
    }
}

// All threads: `count` rows of D elements, `stride` apart, one behind the other in shared memory; 16 bytes at a time and four such loads on their way where the rows allow it.
__device__ __forceinline__ void stage_rows(const bf16* __restrict__ source, long long stride, int count, int D, bf16* staged) {
    if (((reinterpret_cast<uintptr_t>(source) | static_cast<uintptr_t>(stride * 2)) & 15) == 0) {
        const int per_row = D / 8, pieces = count * per_row;
        for (int base = threadIdx.x; base < pieces; base += 4 * 256) {
            uint4 raw[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int piece = base + 256 * a, row = piece / per_row;
                if (piece < pieces) raw[a] = __ldg(reinterpret_cast<const uint4*>(source + row * stride) + (piece - row * per_row));
            }
#pragma unroll
            for (int a = 0; a < 4; ++a)
                if (base + 256 * a < pieces) reinterpret_cast<uint4*>(staged)[base + 256 * a] = raw[a];
        }
    } else {
        for (int index = threadIdx.x; index < count * D; index += 256) staged[index] = source[index / D * stride + index % D];
    }
    __syncthreads();
}

// grid (pages touched, key heads + value heads + groups of query heads).  A block serves the new tokens of one sequence in one page: it
// alone reads and writes that page of that head, so a scale that has to grow and the older codes that are rounded to it need no meeting.
// PER > 0: heads of 32 PER elements that are rotated whole or not at all, in rows on 16-byte borders, are prepared in registers, several rows to a warp at once, and queries go
// through no shared memory (1,000 tokens of 32 query and 8 key heads of 128: 18 us, row by row in shared memory 46; four rows
// to a warp at once instead of two: 20, and 14 for 15 with 300 tokens).
template <int PER>
__global__ void __launch_bounds__(256)
store_kernel(StoreSource source, uint8_t* __restrict__ key_pages, uint8_t* __restrict__ value_pages, float* __restrict__ key_scales, float* __restrict__ value_scales,
             const int* __restrict__ cu_seqlens, const int* __restrict__ seq_start, const int* __restrict__ page_rows, int page_stride, int n_seqs, int n_kv_heads, int D, int most) {
    grid_dependents_launch();
    grid_dependency_wait();
    extern __shared__ __align__(16) bf16 staged[];      // [tokens here][D]
    __shared__ float greatest_of[8];
    __shared__ int found[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // Which sequence and page: the first warp adds up the pages that 32 sequences at a time touch.
    if (most == 1) {      // one token to a sequence: the block's number is the sequence's
        if (threadIdx.x == 0) {
            found[0] = blockIdx.x;
            found[1] = cu_seqlens[blockIdx.x];
            found[2] = seq_start[blockIdx.x];
            found[3] = 1;
        }
    } else if (warp == 0) {
        int before = 0, seq = -1, page = 0, start = 0, first = 0, count = 0;
        const int item = blockIdx.x;
        for (int base = 0; base < n_seqs; base += 32) {
            const int s = base + lane;
            int s_first = 0, s_count = 0, s_start = 0, touched = 0;
            if (s < n_seqs) {
                s_first = cu_seqlens[s];
                s_count = cu_seqlens[s + 1] - s_first;
                s_start = seq_start[s];
                touched = s_count > 0 ? (s_start + s_count - 1) / kPage - s_start / kPage + 1 : 0;
            }
            int through = touched;
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, through, offset);
                if (lane >= offset) through += other;
            }
            const bool mine = item >= before + through - touched && item < before + through;
            const unsigned who = __ballot_sync(0xffffffffu, mine);
            if (who != 0u) {
                const int owner = __ffs(who) - 1;
                seq = base + owner;
                start = __shfl_sync(0xffffffffu, s_start, owner);
                first = __shfl_sync(0xffffffffu, s_first, owner);
                count = __shfl_sync(0xffffffffu, s_count, owner);
                page = start / kPage + item - before - __shfl_sync(0xffffffffu, through - touched, owner);
                break;
            }
            before += __shfl_sync(0xffffffffu, through, 31);
        }
        if (lane == 0) {
            const int low = max(start, page * kPage), high = min(start + count, (page + 1) * kPage);
            found[0] = seq;
            found[1] = first + low - start;      // first packed row
            found[2] = low;
            found[3] = min(high - low, most);      // what the staging holds
        }
    }
    __syncthreads();
    const int seq = found[0], row0 = found[1], position0 = found[2], count = found[3];
    if (seq < 0) return;      // the host counts pages from above
    const int half = source.rotary_dim / 2;
    if (static_cast<int>(blockIdx.y) >= 2 * n_kv_heads) {      // queries: one head after another
        const int head0 = (blockIdx.y - 2 * n_kv_heads) * kQueryHeads, heads = min(kQueryHeads, source.n_heads - head0);
        if constexpr (PER > 0) {
            constexpr int kRowsAhead = PER <= 4 ? 2 : 1;
            Prepared<PER> with(source.q_weight, lane);
            for (int begin = warp; begin < count; begin += 8 * kRowsAhead) {
                Neighbours<PER> raw[kRowsAhead][kQueryHeads];
                float cosines[kRowsAhead][PER], sines[kRowsAhead][PER];
#pragma unroll
                for (int a = 0; a < kRowsAhead; ++a) {
                    const int token = min(begin + 8 * a, count - 1);
                    const bf16* row = source.query_rows + static_cast<size_t>(row0 + token) * source.query_stride + static_cast<size_t>(head0) * D + PER * lane;
#pragma unroll
                    for (int h = 0; h < kQueryHeads; ++h) raw[a][h] = *reinterpret_cast<const Neighbours<PER>*>(row + min(h, heads - 1) * D);
                    angles<PER>(source, position0 + token, lane, cosines[a], sines[a]);
                }
#pragma unroll
                for (int a = 0; a < kRowsAhead; ++a) {
                    const int token = begin + 8 * a;
                    if (token >= count) break;
                    Neighbours<PER>* target = reinterpret_cast<Neighbours<PER>*>(source.queries + (static_cast<size_t>(row0 + token) * source.n_heads + head0) * D) + lane;
#pragma unroll
                    for (int h = 0; h < kQueryHeads; ++h) {
                        const Neighbours<PER> result = prepare_neighbours<PER>(raw[a][h], source.q_weight != nullptr, with.weight, source.eps, half > 0, cosines[a], sines[a], lane);
                        if (h < heads) target[h * 32] = result;
                    }
                }
            }
        } else {
            for (int head = head0; head < head0 + heads; ++head) {
                stage_rows(source.query_rows + static_cast<size_t>(row0) * source.query_stride + static_cast<size_t>(head) * D, source.query_stride, count, D, staged);
                for (int token = warp; token < count; token += 8) {
                    const size_t table = static_cast<size_t>(position0 + token) * half;
                    prepare_row(staged + token * D, source.q_weight, source.eps, source.cos_table + table, source.sin_table + table, source.rotary_dim, D, lane);
                }
                __syncthreads();
                for (int piece = threadIdx.x; piece < count * D / 8; piece += 256) {
                    const int token = piece / (D / 8), part = piece - token * (D / 8);
                    reinterpret_cast<uint4*>(source.queries + (static_cast<size_t>(row0 + token) * source.n_heads + head) * D)[part] = reinterpret_cast<const uint4*>(staged)[piece];
                }
                __syncthreads();
            }
        }
        return;
    }
    const bool is_key = static_cast<int>(blockIdx.y) < n_kv_heads;
    const int head = is_key ? blockIdx.y : blockIdx.y - n_kv_heads;
    const size_t place = static_cast<size_t>(page_rows[static_cast<size_t>(seq) * page_stride + position0 / kPage]) * n_kv_heads + head;
    uint8_t* page = (is_key ? key_pages : value_pages) + place * kPage * D;
    float* scale_at = (is_key ? key_scales : value_scales) + place;
    const int older = position0 % kPage;
    const long long stride = is_key ? source.key_stride : source.value_stride;
    stage_rows((is_key ? source.keys : source.values) + static_cast<long long>(row0) * stride + static_cast<long long>(head) * D, stride, count, D, staged);
    if (PER > 0 && is_key && (source.k_weight != nullptr || half > 0)) {
        if constexpr (PER > 0) {
            constexpr int kRowsAhead = PER <= 4 ? 2 : 1;
            Prepared<PER> with(source.k_weight, lane);
            for (int begin = warp; begin < count; begin += 8 * kRowsAhead) {
                float cosines[kRowsAhead][PER], sines[kRowsAhead][PER];
#pragma unroll
                for (int a = 0; a < kRowsAhead; ++a) angles<PER>(source, position0 + min(begin + 8 * a, count - 1), lane, cosines[a], sines[a]);
#pragma unroll
                for (int a = 0; a < kRowsAhead; ++a) {
                    const int token = begin + 8 * a;
                    if (token >= count) break;
                    Neighbours<PER>* row = reinterpret_cast<Neighbours<PER>*>(staged + token * D) + lane;
                    *row = prepare_neighbours<PER>(*row, source.k_weight != nullptr, with.weight, source.eps, half > 0, cosines[a], sines[a], lane);
                }
            }
        }
        __syncthreads();
    } else if (is_key && (source.k_weight != nullptr || half > 0)) {
        for (int token = warp; token < count; token += 8) {
            const size_t table = static_cast<size_t>(position0 + token) * half;
            prepare_row(staged + token * D, source.k_weight, source.eps, source.cos_table + table, source.sin_table + table, source.rotary_dim, D, lane);
        }
        __syncthreads();
    }
    const float scale = store_in_page(staged, count, D, older, page, scale_at, greatest_of);
    if (threadIdx.x == 0) *scale_at = scale;
}

constexpr int kReadHeads = 16;      // at most so many heads to a block
// All ones in each byte that is a NaN code.
__device__ __forceinline__ unsigned nan_codes(unsigned word) { return __vcmpeq4(word & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// Pages of the step's sequences as the bfloat16 values that they stand for (exact: 4 significant bits times a power of two).
// grid (`span` pages of a sequence, sequence, groups of `heads` heads), from the first page of a sequence on or, with `sparse`, from the first that a query sees.  Positions that a sequence does
// not have are zeros; with `sparse` only pages that a query sees are written at all (and `places` gets the numbers that the pages have in the result; those of other pages are numbers that it has
// too), and positions that none sees are zeros: what a window left behind may be NaN, and a weight of
// zero would not hide that.  Bound by memory: a page's heads lie one behind the other, so where there are pages enough a block takes several and pays for its page's number and
// scale once (64 sequences of up to 200 positions, 8 heads of 128: 14 us for 17 MB of codes read and 34 MB of values written).
template <bool Windowed>
__global__ void __launch_bounds__(256)
read_kernel(const uint8_t* __restrict__ key_pages, const uint8_t* __restrict__ value_pages, const float* __restrict__ key_scales, const float* __restrict__ value_scales,
            bf16* __restrict__ keys, bf16* __restrict__ values, int* __restrict__ places, const int* __restrict__ seq_start, const int* __restrict__ seq_len, const int* __restrict__ page_rows,
            int page_stride, int span, int page_heads, int n_kv_heads, int heads, int D, int window, int sparse) {
    __shared__ unsigned char odd[kReadHeads * kPage];      // positions with a value that is not finite
    grid_dependents_launch();
    grid_dependency_wait();
    const int seq = blockIdx.y, head0 = blockIdx.z * heads, here = min(heads, n_kv_heads - head0);
    const int first_seen = Windowed ? max(0, seq_start[seq] + 1 - window) : 0, first_page = first_seen / kPage, page = first_page + blockIdx.x;
    if constexpr (Windowed) {
        if (blockIdx.x == 0 && blockIdx.z == 0)
            for (int p = threadIdx.x; p < page_stride; p += 256) places[static_cast<size_t>(seq) * page_stride + p] = seq * span + min(max(p - first_page, 0), span - 1);
    } else {
        if (places != nullptr && blockIdx.z == 0 && threadIdx.x == 0) places[static_cast<size_t>(seq) * page_stride + page] = seq * span + page;
    }
    const int live = min(kPage, seq_len[seq] - page * kPage);      // positions that the sequence has in this page
    const int first = max(0, first_seen - page * kPage);      // the first position of this page that a query sees
    if (sparse && live <= 0) return;
    const size_t place = live > 0 ? static_cast<size_t>(page_rows[static_cast<size_t>(seq) * page_stride + page]) * page_heads + head0 : 0;
    const int per_head = kPage * D / 16, begin = first * D / 16, end = live * D / 16;      // pieces of 16 elements
    // For attention (`sparse`), where some queries see a position and others do not: a value that is not finite would reach those that do not, through a weight of zero.  It becomes zero
    // and its position's key NaN, which a mask does hide.
    const bool guarded = sparse && (Windowed || (page + 1) * kPage > seq_start[seq]);
    if (guarded) {
        for (int index = threadIdx.x; index < here * kPage; index += 256) odd[index] = 0;
        __syncthreads();
    }
    constexpr int kAhead = 4;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {      // values, then keys
        const uint4* codes = reinterpret_cast<const uint4*>((pass == 0 ? value_pages : key_pages) + place * kPage * D);
        const float* scales = (pass == 0 ? value_scales : key_scales) + place;
        uint4* target = reinterpret_cast<uint4*>((pass == 0 ? values : keys) + ((static_cast<size_t>(seq) * span + blockIdx.x) * n_kv_heads + head0) * kPage * D);
        for (int base = threadIdx.x; base < here * per_head; base += 256 * kAhead) {
            uint4 raw[kAhead];
            float scale[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int piece = base + 256 * a, head = piece / per_head, place_in = piece - head * per_head;
                const bool held = head < here && place_in >= begin && place_in < end;
                raw[a] = held ? __ldg(codes + piece) : make_uint4(0u, 0u, 0u, 0u);
                scale[a] = held ? __ldg(scales + head) : 0.0f;
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int piece = base + 256 * a;
                if (piece >= here * per_head) break;
                unsigned words[4] = {raw[a].x, raw[a].y, raw[a].z, raw[a].w};
                if (guarded) {
                    const int position = piece / per_head * kPage + piece % per_head * 16 / D;
                    if (pass == 0) {
                        if (nan_codes(words[0]) | nan_codes(words[1]) | nan_codes(words[2]) | nan_codes(words[3])) {
                            odd[position] = 1;
#pragma unroll
                            for (int i = 0; i < 4; ++i) words[i] &= ~nan_codes(words[i]);
                        }
                    } else if (odd[position]) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) words[i] = 0x7f7f7f7fu;
                    }
                }
                uint4 wide[2];
                unsigned* out = reinterpret_cast<unsigned*>(wide);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v[4];
                    decode_four(words[i], v);
                    out[2 * i] = pack_bf16_pair(v[0] * scale[a], v[1] * scale[a]);
                    out[2 * i + 1] = pack_bf16_pair(v[2] * scale[a], v[3] * scale[a]);
                }
                target[2 * piece] = wide[0];
                target[2 * piece + 1] = wide[1];
            }
        }
        if (guarded && pass == 0) __syncthreads();
    }
}

}  // namespace

// Codes [rows, columns] (contiguous) and scales [blocks of rows, blocks of columns] of a matrix whose columns are a multiple of 16.
TAU_EXPORT int tau_quantize_blocks(int dtype, const void* values, long long stride, void* codes, float* scales, int rows, int columns, void* stream) {
    if (rows <= 0 || columns <= 0) return 0;
    if (!values || !codes || !scales || (columns & 15) || (dtype != TAU_BF16 && dtype != TAU_F32) || (rows + kScaleBlock - 1) / kScaleBlock > 65535) return cudaErrorInvalidValue;
    const dim3 grid((columns + kScaleBlock - 1) / kScaleBlock, (rows + kScaleBlock - 1) / kScaleBlock);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == TAU_BF16)
        tau_launch(quantize_blocks_kernel<bf16>, grid, dim3(256), 0, s, static_cast<const bf16*>(values), stride, static_cast<uint8_t*>(codes), scales, rows, columns);
    else
        tau_launch(quantize_blocks_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(values), stride, static_cast<uint8_t*>(codes), scales, rows, columns);
    return tau_launch_status();
}

// Codes [rows, columns] (contiguous) and scales [blocks of columns, rows]; columns a multiple of 16, rows of values on 16-byte borders.
TAU_EXPORT int tau_quantize_rows(int dtype, const void* values, long long stride, void* codes, float* scales, int rows, int columns, void* stream) {
    return launch_quantize_rows(dtype, values, stride, codes, scales, rows, columns, static_cast<cudaStream_t>(stream));
}

// x codes [M, K] with scales [blocks, M]; w codes [N, K] with scales [blocks of N, blocks]; both contiguous on 16-byte borders, K a multiple of 16.
TAU_EXPORT int tau_gemm8_simt(int out_dtype, const void* x, const float* x_scales, const void* w, const float* w_scales, const float* bias, void* out, int M, int N, int K,
                              long long out_stride, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !x_scales || !w || !w_scales || !out || K <= 0 || (K & 15) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(w) & 15) ||
        (out_dtype != TAU_BF16 && out_dtype != TAU_F32))
        return cudaErrorInvalidValue;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M > 65535 * 32) return cudaErrorInvalidValue;
    const dim3 grid((N + 31) / 32, (M + 31) / 32);
    if (out_dtype == TAU_BF16)
        tau_launch(gemm8_simt_kernel<bf16>, grid, dim3(256), 0, s, static_cast<const uint8_t*>(x), x_scales, static_cast<const uint8_t*>(w), w_scales, bias, static_cast<bf16*>(out), M, N, K, out_stride);
    else
        tau_launch(gemm8_simt_kernel<float>, grid, dim3(256), 0, s, static_cast<const uint8_t*>(x), x_scales, static_cast<const uint8_t*>(w), w_scales, bias, static_cast<float*>(out), M, N, K, out_stride);
    return tau_launch_status();
}

TAU_EXPORT int tau_gate_groups(const void* stacked, void* out, long long rows, int inner, long long out_stride, float limit, void* stream) {
    if (rows <= 0 || inner <= 0) return 0;
    if (!stacked || !out || (inner & 7) || (rows * inner + 255) / 256 > 0x7fffffffll) return cudaErrorInvalidValue;
    tau_launch(gate_groups_kernel, dim3(static_cast<unsigned>((rows * inner + 255) / 256)), dim3(256), 0, static_cast<cudaStream_t>(stream), static_cast<const bf16*>(stacked),
               static_cast<bf16*>(out), rows * inner, inner, out_stride, limit);
    return tau_launch_status();
}

// Stores the keys and values of `tokens` new tokens; with `query_rows` the queries are prepared beside them.  `cos_table` == nullptr needs rotary_dim 0.
TAU_EXPORT int tau_cache8_store(const void* keys, long long key_stride, const void* values, long long value_stride, void* key_pages, void* value_pages, float* key_scales,
                                float* value_scales, const int* cu_seqlens, const int* seq_start, const int* page_rows, int page_stride, int n_seqs, int tokens, int single,
                                int n_kv_heads, int D, const void* query_rows, long long query_stride, void* queries, int n_heads, const float* q_weight, const float* k_weight,
                                float eps, const float* cos_table, const float* sin_table, int rotary_dim, void* stream) {
    if (tokens <= 0 || n_seqs <= 0) return 0;
    if (!keys || !values || !key_pages || !value_pages || ((reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages)) & 15) || !key_scales || !value_scales || !cu_seqlens || !seq_start || !page_rows || page_stride <= 0 || n_kv_heads <= 0 || D < 16 ||
        D > 256 || (D & 15) || rotary_dim < 0 || rotary_dim > D || (rotary_dim & 1) || (rotary_dim > 0 && (!cos_table || !sin_table)) || (query_rows && (!queries || (reinterpret_cast<uintptr_t>(queries) & 15) || n_heads <= 0)))
        return cudaErrorInvalidValue;
    const StoreSource source = {static_cast<const bf16*>(keys), static_cast<const bf16*>(values), key_stride, value_stride, static_cast<const bf16*>(query_rows), query_stride,
                                static_cast<bf16*>(queries), q_weight, k_weight, eps, cos_table, sin_table, rotary_dim, n_heads};
    // A run of n tokens touches at most (n + 62) / 64 + 1 pages, and no more pages than it has tokens.
    const long long bound = static_cast<long long>(tokens) / kPage + 2ll * n_seqs;
    const unsigned items = single ? static_cast<unsigned>(n_seqs) : static_cast<unsigned>(bound < tokens ? bound : tokens);
    const unsigned parts = 2u * n_kv_heads + (query_rows ? (n_heads + kQueryHeads - 1) / kQueryHeads : 0);
    if (parts > 65535u) return cudaErrorInvalidValue;
    const int rows = single ? 1 : kPage;      // staged rows
    const bool neighbours = (query_rows || k_weight || rotary_dim) && (rotary_dim == 0 || rotary_dim == D) && (!query_rows || ((query_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(query_rows) & 15) == 0));
    auto run = [&](auto kernel) {
        tau_launch(kernel, dim3(items, parts), dim3(256), static_cast<size_t>(rows) * D * sizeof(bf16), static_cast<cudaStream_t>(stream), source, static_cast<uint8_t*>(key_pages),
                   static_cast<uint8_t*>(value_pages), key_scales, value_scales, cu_seqlens, seq_start, page_rows, page_stride, n_seqs, n_kv_heads, D, rows);
    };
    if (neighbours && D == 64) run(store_kernel<2>);
    else if (neighbours && D == 128) run(store_kernel<4>);
    else if (neighbours && D == 256) run(store_kernel<8>);
    else run(store_kernel<0>);
    return tau_launch_status();
}

// `span`: pages laid out for each sequence: all that the page rows list, or, with `sparse` and a window, as many as the queries of its run can see.  `n_kv_heads` heads from `first_head` on are read
// of pages of `page_heads`.
TAU_EXPORT int tau_cache8_read(const void* key_pages, const void* value_pages, const float* key_scales, const float* value_scales, void* keys, void* values, int* places, const int* seq_start,
                               const int* seq_len, const int* page_rows, int page_stride, int span, int n_seqs, int page_heads, int first_head, int n_kv_heads, int D, int window, int sparse, void* stream) {
    if (n_seqs <= 0) return 0;
    if (!key_pages || !value_pages || ((reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages)) & 15) || !key_scales || !value_scales || !keys || !values || !seq_start || !seq_len ||
        !page_rows || page_stride <= 0 || span <= 0 || (sparse ? !places : span != page_stride) || (window <= 0 && span != page_stride) || n_kv_heads <= 0 || first_head < 0 || first_head + n_kv_heads > page_heads || D < 16 || D > 256 ||
        (D & 15) || n_seqs > 65535 || n_kv_heads > 65535)
        return cudaErrorInvalidValue;
    static int counts[64] = {};      // multiprocessors of each device, asked for once
    int device = 0, sms = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return cudaErrorInvalidDevice;
    if (device < 64) sms = counts[device];
    if (!sms) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return cudaErrorInvalidDevice;
        if (device < 64) counts[device] = sms;
    }
    const long long blocks = static_cast<long long>(n_kv_heads) * n_seqs * span, wanted = 8ll * sms;      // one head to a block as long as all fit the machine at once
    const int most = n_kv_heads < kReadHeads ? n_kv_heads : kReadHeads;
    const int heads = blocks <= wanted ? 1 : static_cast<int>(blocks / wanted < most ? blocks / wanted : most);
    const size_t before = static_cast<size_t>(first_head) * kPage * D;
    auto run = [&](auto kernel) {
        tau_launch(kernel, dim3(span, n_seqs, (n_kv_heads + heads - 1) / heads), dim3(256), 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(key_pages) + before,
                   static_cast<const uint8_t*>(value_pages) + before, key_scales + first_head, value_scales + first_head, static_cast<bf16*>(keys), static_cast<bf16*>(values), places, seq_start, seq_len,
                   page_rows, page_stride, span, page_heads, n_kv_heads, heads, D, window, sparse);
    };
    if (sparse && window > 0) run(read_kernel<true>);
    else run(read_kernel<false>);
    return tau_launch_status();
}
