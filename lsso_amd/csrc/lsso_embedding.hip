// Token embedding y[t] = scale * W[token[t]] and the gradient of its table,
//   dW[v] = scale * sum over the counted tokens t with token[t] = v of dy[t].
//
// Forward: a copy with an index, bound by HBM (the rows that are named, once,
// and y).  A workgroup takes whole rows, a thread 8 elements of one row at a
// time, with its rows' steps unrolled so that several id -> row -> store chains
// are in flight: 262,144 tokens of 256 features in 27 us, 4.9 TB/s.
//
// Gradient: floats added by atomics would make the sums' order, and so their
// rounding, change from call to call, and rows that many tokens share (six
// symbols in 262,144 tokens) would queue at one address.  Instead the tokens
// are sorted by id (stable, so a row's tokens keep their order), and each row
// is summed once, in FP32, in an order that depends on the sizes alone:
//   1. radix sort of (id, index) in passes of up to 10 bits of the id (one for
//      tables of up to 1,023 rows, two up to 2^20 - 1, three up to 2^30 - 1): a
//      histogram per tile of tokens, then a stable scatter that ranks equal
//      digits of 64 lanes by ballots and takes its bases from the histograms;
//      Workgroups beside the sort's few write zeros over dW, which most rows of a
//      large table keep;
//   2. the sorted order is cut into chunks, and lanes that cover a row (whole
//      waves from 512 features on) go through one chunk each: the rows of dy are
//      gathered 8 ahead whatever the runs' lengths, a run that ends is stored, and
//      one that crosses the chunk's ends leaves a partial sum.  A wave per table
//      row instead had to search its run, gathered a row at a time, and left
//      the frequent words of a text to few waves;
//   3. the partials of each run that crosses are added, by a wave or a workgroup.
// Tokens that count nowhere (excluded, padding, out of range) get the id
// `vocabulary` and sort behind every row.
//
// Bound: reading dy (gathered whole rows) and writing dW, plus the latency of two
// launches per pass, the sums' and, with more than one chunk, the join's.

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kLookupThreads = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kDigitBits = 10;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSumThreads = 256;
constexpr int kSumWaves = kSumThreads / 64;
constexpr int kJoinThreads = 1024;
constexpr int kJoinWaves = kJoinThreads / 64;
constexpr int kWaveChunks = 16;  // longest run, in chunks, that one wave joins

__device__ __forceinline__ int64_t read_token(const EmbeddingArgs& a, int64_t t) {
    return a.wide_tokens ? static_cast<const int64_t*>(a.tokens)[t]
                         : static_cast<int64_t>(static_cast<const int32_t*>(a.tokens)[t]);
}

// Pieces of 8 elements of a row of `dim` >= 8: the last one starts early
// enough to end within the row, and writes again what its neighbour wrote.
__device__ __forceinline__ int piece_at(int piece, int dim) {
    return 8 * piece + 8 <= dim ? 8 * piece : dim - 8;
}

template <int W, int Y>
__global__ __launch_bounds__(kLookupThreads) void lookup_kernel(EmbeddingArgs a) {
    const auto* weight = static_cast<const typename Values<W>::Element*>(a.weight);
    auto* y = static_cast<typename Values<Y>::Element*>(a.y);
    const int dim = static_cast<int>(a.dim);
    const int per_row = dim >= 8 ? (dim + 7) / 8 : dim;   // short rows go element by element
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
    const int rows = static_cast<int>(a.count - row0 < a.block_rows ? a.count - row0 : a.block_rows);
    const int items = rows * per_row;
#pragma unroll 4
    for (int i = threadIdx.x; i < items; i += kLookupThreads) {
        const int r = i / per_row;
        const int piece = i - r * per_row;
        const int64_t t = row0 + r;
        const int64_t token = read_token(a, t);
        const bool named = token >= 0 && token < a.vocabulary;
        const bool kept = a.row_mask == nullptr || a.row_mask[t] != 0;
        // An id outside the table is the caller's error: its row is NaN.
        const float other = kept ? __builtin_nanf("") : 0.0f;
        const int64_t row = named && kept ? token : 0;
        if (dim >= 8) {
            const int k = piece_at(piece, dim);
            float v[8];
            Values<W>::load8(weight + row * a.weight_stride + k, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = named && kept ? a.scale * v[e] : other;
            }
            Values<Y>::store8(y + t * a.dim + k, v);
        } else {
            const float v = Values<W>::load(weight + row * a.weight_stride + piece);
            Values<Y>::store(y + t * a.dim + piece, named && kept ? a.scale * v : other);
        }
    }
}

// Sort key of token t: its id, or `vocabulary` where it counts nowhere.
__device__ __forceinline__ uint32_t token_key(const EmbeddingArgs& a, int64_t t) {
    const int64_t token = read_token(a, t);
    const bool counted = token >= 0 && token < a.vocabulary && token != a.padding_index &&
                         (a.row_mask == nullptr || a.row_mask[t] != 0);
    return static_cast<uint32_t>(counted ? token : a.vocabulary);
}

__device__ __forceinline__ uint32_t sort_key(const EmbeddingArgs& a, const SortPass& p, int64_t i) {
    return p.keys_in == nullptr ? token_key(a, i) : p.keys_in[i];
}

// Zeros over the pass' part of the gradient by the workgroups behind the tiles';
// the sums that follow write the rows that tokens name.
__device__ __forceinline__ void clear_part(const EmbeddingArgs& a, const SortPass& p, int64_t part) {
    char* to = static_cast<char*>(a.grad_weight);
    const int64_t bytes = a.vocabulary * a.dim * (a.weight_type == LSSO_HIP_F32 ? 4 : 2);
    const int64_t begin = bytes / 16 * part / p.parts;
    const int64_t end = bytes / 16 * (part + 1) / p.parts;
    const int64_t step = static_cast<int64_t>(gridDim.x - a.tiles) * kSortThreads;
#pragma unroll 4
    for (int64_t i = begin + (blockIdx.x - a.tiles) * kSortThreads + threadIdx.x; i < end; i += step) {
        store16_unaligned(to + 16 * i, (u32x4){0, 0, 0, 0});
    }
    const int64_t rest = bytes / 16 * 16 + 2 * static_cast<int64_t>(threadIdx.x);
    if (part == 0 && blockIdx.x == a.tiles && rest < bytes) {
        *reinterpret_cast<uint16_t*>(to + rest) = 0;
    }
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(EmbeddingArgs a, SortPass p) {
    __shared__ uint32_t histogram[kDigits];
    if (blockIdx.x >= a.tiles) {
        clear_part(a, p, p.part);
        return;
    }
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        histogram[d] = 0;
    }
    __syncthreads();
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.tile_tokens;
    const int64_t end = begin + a.tile_tokens < a.count ? begin + a.tile_tokens : a.count;
    for (int64_t i = begin + threadIdx.x; i < end; i += kSortThreads) {
        atomicAdd(&histogram[(sort_key(a, p, i) >> p.shift) & (digits - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        a.histograms[static_cast<int64_t>(blockIdx.x) * digits + d] = histogram[d];
    }
}

// Lanes of the wave whose digit equals this lane's, among `active` lanes.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool active) {
    uint64_t lanes = __ballot(active);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1);
        lanes &= (digit >> b) & 1 ? set : ~set;
    }
    return lanes;
}

__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(EmbeddingArgs a, SortPass p) {
    __shared__ uint32_t at[kSortWaves][kDigits];   // per wave: counts, then the next place of each digit
    __shared__ uint32_t wave_total[kSortWaves];
    if (blockIdx.x >= a.tiles) {
        clear_part(a, p, p.part + 1);
        return;
    }
    const int digits = 1 << p.bits;
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) {
        at[i / kDigits][i % kDigits] = 0;
    }
    // Tokens of each digit in the tiles before this one, and in all: every digit
    // has 1024 / digits threads, which take the tiles in turn.
    const int my_digit = static_cast<int>(threadIdx.x) & (digits - 1);
    uint32_t before = 0;
    uint32_t all = 0;
#pragma unroll 8
    for (int64_t tile = threadIdx.x >> p.bits; tile < a.tiles; tile += kSortThreads >> p.bits) {
        const uint32_t n = a.histograms[tile * digits + my_digit];
        before += tile < static_cast<int64_t>(blockIdx.x) ? n : 0;
        all += n;
    }
    __syncthreads();
    if (digits < kSortThreads) {
        // Integers: the order of these additions changes nothing.
        atomicAdd(&at[0][my_digit], before);
        atomicAdd(&at[1][my_digit], all);
        __syncthreads();
        before = at[0][my_digit];
        all = static_cast<int>(threadIdx.x) < digits ? at[1][my_digit] : 0;
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kDigits; i += kSortThreads) {
            at[i / kDigits][i % kDigits] = 0;
        }
        __syncthreads();
    }
    // The tile's tokens in order: each wave takes a contiguous part of them.
    const int64_t part = a.tile_tokens / kSortWaves;
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.tile_tokens + wave * part;
    const int64_t end = begin + part < a.count ? begin + part : a.count;
    for (int64_t i = begin + lane; i - lane < end; i += 64) {
        const bool active = i < end;
        const uint32_t digit = active ? (sort_key(a, p, i) >> p.shift) & (digits - 1) : 0;
        const uint64_t same = same_digit(digit, p.bits, active);
        if (active && lane == __ffsll(static_cast<unsigned long long>(same)) - 1) {
            at[wave][digit] += __popcll(same);
        }
        wave_lds_order();
    }
    // Exclusive sum of `all` over the digits.
    uint32_t sum = all;
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t other = __shfl_up(sum, s);
        sum += lane >= s ? other : 0;
    }
    if (lane == 63) {
        wave_total[wave] = sum;
    }
    __syncthreads();
    uint32_t place = sum - all + before;
    for (int w = 0; w < wave; ++w) {
        place += wave_total[w];
    }
    if (static_cast<int>(threadIdx.x) < digits) {
        for (int w = 0; w < kSortWaves; ++w) {
            const uint32_t n = at[w][threadIdx.x];
            at[w][threadIdx.x] = place;
            place += n;
        }
    }
    __syncthreads();
    for (int64_t i = begin + lane; i - lane < end; i += 64) {
        const bool active = i < end;
        const uint32_t key = active ? sort_key(a, p, i) : 0;
        const uint32_t digit = (key >> p.shift) & (digits - 1);
        const uint64_t same = same_digit(digit, p.bits, active);
        const uint32_t first = active ? at[wave][digit] : 0;
        wave_lds_order();   // every lane reads before the leader moves the place on
        if (active) {
            const int rank = __popcll(same & ((1ull << lane) - 1));
            p.keys_out[first + rank] = key;
            p.index_out[first + rank] = p.index_in == nullptr ? static_cast<uint32_t>(i) : p.index_in[i];
            if (rank == 0) {
                at[wave][digit] = first + __popcll(same);
            }
        }
        wave_lds_order();
    }
}

// First sorted position whose id is at least `key`, found by the whole wave:
// each step probes 64 evenly spaced positions of the range that is left.
__device__ __forceinline__ int64_t first_at_least(const uint32_t* keys, int64_t count, uint32_t key, int lane) {
    int64_t low = 0;
    int64_t left = count;   // the answer lies in [low, low + left]
    while (left > 0) {
        const int64_t step = (left + 63) / 64;
        const int64_t probe = low + step * lane;
        const bool less = probe < low + left && keys[probe] < key;
        const int n = __popcll(__ballot(less));   // keys ascend: the lanes before the answer
        if (n == 0) {
            return low;
        }
        const int64_t end = low + left;
        low += step * (n - 1) + 1;                // behind the last probe that was less
        left = step - 1 < end - low ? step - 1 : end - low;
    }
    return low;
}

template <int W>
__device__ __forceinline__ void store_row(const EmbeddingArgs& a, int64_t row, int k, const float (&sum)[8]) {
    auto* at = static_cast<typename Values<W>::Element*>(a.grad_weight) + row * a.dim;
    if (a.dim >= 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = a.scale * sum[e];
        }
        Values<W>::store8(at + k, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e < a.dim) {
                Values<W>::store(at + e, a.scale * sum[e]);
            }
        }
    }
}

__device__ __forceinline__ void store_row(const EmbeddingArgs& a, int64_t row, int k, const float (&sum)[8]) {
    if (a.weight_type == LSSO_HIP_F32) {
        store_row<LSSO_HIP_F32>(a, row, k, sum);
    } else if (a.weight_type == LSSO_HIP_BF16) {
        store_row<LSSO_HIP_BF16>(a, row, k, sum);
    } else {
        store_row<LSSO_HIP_F16>(a, row, k, sum);
    }
}

// Lanes that share a row: the power of two that covers its pieces, at most `most`.
__device__ __forceinline__ int row_lanes(int64_t dim, int most) {
    int width = 1;
    while (width < most && 8 * width < dim) {
        width *= 2;
    }
    return width;
}

// Lanes of a row in the join: 128 features a workgroup, more where that would cut a
// row into more than four.  A long run's partials come as fast as the CUs that read
// them (262,144 tokens of 256 features, a table of 6: 22 us on one, 13 on two),
// but short ones cost each of them a search.
__host__ __device__ inline int join_lanes(int64_t dim) { return dim <= 512 ? 16 : dim <= 1024 ? 32 : 64; }

// Features of this lane: piece `piece` of its row.
__device__ __forceinline__ int lane_feature(const EmbeddingArgs& a, int piece, bool& inside) {
    const int dim = static_cast<int>(a.dim);
    inside = 8 * piece < dim;
    return dim < 8 || !inside ? 0 : piece_at(piece, dim);
}

// N sorted positions from a multiple of N on: their ids and tokens.
template <int N>
struct Positions {
    uint32_t key[N];
    uint32_t index[N];
    __device__ __forceinline__ Positions(const EmbeddingArgs& a, int64_t at) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {   // the arrays end at a multiple of 64
            const u32x4 keys = *reinterpret_cast<const u32x4*>(a.keys + at + i);
            const u32x4 tokens = *reinterpret_cast<const u32x4*>(a.index + at + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                key[i + e] = keys[e];
                index[i + e] = tokens[e];
            }
        }
    }
};

// Their rows of dy, 8 features each, as they were loaded.
template <int G, int N>
struct Gathered {
    static constexpr int kPieces = G == LSSO_HIP_F32 ? 2 : 1;
    u32x4 raw[N][kPieces];
    // Of the first `here` positions; behind them any row that is there.
    __device__ __forceinline__ Gathered(const EmbeddingArgs& a, const Positions<N>& p, int here, int k) {
        const auto* dy = static_cast<const typename Values<G>::Element*>(a.grad_y);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const auto* row = dy + static_cast<int64_t>(p.index[j < here ? j : 0]) * a.grad_stride;
            if (a.dim >= 8) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    raw[j][i] = load16_unaligned(row + k + 4 * i);
                }
            } else {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = e < a.dim ? Values<G>::load(row + e) : 0.0f;
                }
                put(raw[j], v);
            }
        }
    }
    __device__ __forceinline__ static void put(u32x4 (&to)[kPieces], const float (&v)[8]) {
        if constexpr (G == LSSO_HIP_F32) {
            to[0] = __builtin_bit_cast(u32x4, (f32x4){v[0], v[1], v[2], v[3]});
            to[1] = __builtin_bit_cast(u32x4, (f32x4){v[4], v[5], v[6], v[7]});
        } else {
            to[0] = Values<G>::pack8(v);
        }
    }
    __device__ __forceinline__ void add(int j, float (&sum)[8]) const {
        float v[8];
        if constexpr (G == LSSO_HIP_F32) {
            const f32x4 low = __builtin_bit_cast(f32x4, raw[j][0]);
            const f32x4 high = __builtin_bit_cast(f32x4, raw[j][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = low[e];
                v[4 + e] = high[e];
            }
        } else {
            Values<G>::unpack8(raw[j][0], v);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum[e] += v[e];
        }
    }
};

// The runs of one chunk, by the lanes of a row.  A run that lies inside the chunk
// is stored, one that begins before it or goes on behind it leaves a partial sum,
// in slot 0 if it holds the chunk's first position, else in 1.  Bound by the latency
// of ids -> tokens -> rows of dy, so the next batch of each is in flight while one
// is added: 32,800 tokens of 768 features and 32,000 table rows 18 us (23 without
// the second batch, 50 by table rows), 262,144 of 256 and 6 rows 25 us, 5.3 TB/s
// of dy (47; 29).
template <int G, int W>
__global__ __launch_bounds__(kSumThreads) void sum_kernel(EmbeddingArgs a) {
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int width = row_lanes(a.dim, 64);
    bool inside;
    const int k = lane_feature(a, 64 * blockIdx.y + (lane & (width - 1)), inside);
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * kSumWaves + wave) * (64 / width) + lane / width;
    if (c >= a.chunks) {
        return;
    }
    const int64_t c0 = c * a.chunk_tokens;
    const int64_t c1 = c0 + a.chunk_tokens < a.count ? c0 + a.chunk_tokens : a.count;
    const uint32_t before = c0 > 0 ? a.keys[c0 - 1] : ~0u;   // no id
    const uint32_t behind = c1 < a.count ? a.keys[c1] : ~0u;
    const uint32_t vocabulary = static_cast<uint32_t>(a.vocabulary);
    constexpr int N = G == LSSO_HIP_F32 ? 4 : 8;   // rows of a batch; a second one is in flight
    const auto at_most = [&](int64_t base) { return static_cast<int>(c1 - base < N ? c1 - base : N); };
    const auto within = [&](int64_t base) { return base < c1 ? base : c0; };
    float sum[8] = {};
    bool first_run = true;
    Positions<N> now(a, c0);
    Positions<N> next(a, within(c0 + N));
    Gathered<G, N> rows(a, now, at_most(c0), k);
    for (int64_t base = c0; base < c1 && now.key[0] < vocabulary; base += N) {
        const Positions<N> later(a, within(base + 2 * N));
        const Gathered<G, N> following(a, next, at_most(within(base + N)), k);
        const int here = at_most(base);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t key = now.key[j];
            if (j >= here || key >= vocabulary) {
                continue;
            }
            rows.add(j, sum);
            const bool last = base + j + 1 == c1;
            const uint32_t after = last ? behind : j + 1 < N ? now.key[(j + 1) % N] : next.key[0];
            if (after == key && !last) {
                continue;
            }
            if (inside && (first_run && before == key || after == key)) {
                float* at = a.partials + (2 * c + (first_run ? 0 : 1)) * a.dim;
                if (a.dim >= 8) {
                    Values<LSSO_HIP_F32>::store8(at + k, sum);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (e < a.dim) {
                            at[e] = sum[e];
                        }
                    }
                }
            } else if (inside) {
                store_row<W>(a, key, k, sum);
            }
            first_run = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum[e] = 0.0f;
            }
        }
        now = next;
        next = later;
        rows = following;
    }
}

// Adds the partials of chunks [from, to) of a run that begins in chunk c at
// position i0.
__device__ __forceinline__ void add_partials(const EmbeddingArgs& a, int64_t from, int64_t to, int64_t c, int64_t i0,
                                             int k, float (&sum)[8]) {
#pragma unroll 4
    for (int64_t p = from; p < to; ++p) {
        const float* at = a.partials + (2 * p + (p == c && i0 > c * a.chunk_tokens ? 1 : 0)) * a.dim + k;
        float v[8];
        if (a.dim >= 8) {
            Values<LSSO_HIP_F32>::load8(at, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = e < a.dim ? at[e] : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum[e] += v[e];
        }
    }
}

// The runs that begin in a chunk and go on behind it (at most one per chunk; it
// holds the chunk's last position).  A wave takes one chunk; a run of few chunks
// is joined by it, a longer one afterwards by the whole workgroup.
__global__ __launch_bounds__(kJoinThreads) void join_kernel(EmbeddingArgs a) {
    __shared__ float parts[kJoinWaves][64][8];
    __shared__ int64_t begins[kJoinWaves];   // position of a wave's run, or -1
    __shared__ int64_t ends[kJoinWaves];
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int width = row_lanes(a.dim, join_lanes(a.dim));
    const int lane_groups = 64 / width;
    bool inside;
    const int k = lane_feature(a, join_lanes(a.dim) * blockIdx.y + (lane & (width - 1)), inside);
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kJoinWaves + wave;
    const int64_t c0 = c * a.chunk_tokens;
    const int64_t c1 = c0 + a.chunk_tokens;
    int64_t found = -1;
    int64_t found_end = 0;
    if (c1 < a.count) {   // all conditions are the same for the whole wave
        const uint32_t key = a.keys[c1 - 1];
        const bool here = c0 == 0 || a.keys[c0 - 1] != key;
        if (key < a.vocabulary && here && a.keys[c1] == key) {
            const int64_t i0 = c0 + first_at_least(a.keys + c0, a.chunk_tokens, key, lane);
            const int64_t i1 = i0 + first_at_least(a.keys + i0, a.count - i0, key + 1, lane);
            const int64_t last = (i1 - 1) / a.chunk_tokens;
            if (last - c < kWaveChunks) {
                if (inside && lane < width) {
                    float sum[8] = {};
                    add_partials(a, c, last + 1, c, i0, k, sum);
                    store_row(a, key, k, sum);
                }
            } else {
                found = i0;
                found_end = i1;
            }
        }
    }
    if (lane == 0) {
        begins[wave] = found;
        ends[wave] = found_end;
    }
    __syncthreads();
    const int groups = lane_groups * kJoinWaves;
    const int group = wave * lane_groups + lane / width;
    for (int w = 0; w < kJoinWaves; ++w) {
        const int64_t i0 = begins[w];
        if (i0 < 0) {   // the same for the whole workgroup
            continue;
        }
        const int64_t first = static_cast<int64_t>(blockIdx.x) * kJoinWaves + w;
        const int64_t last = (ends[w] - 1) / a.chunk_tokens;
        float sum[8] = {};
        // Consecutive chunks to each group of lanes, in order.
        const int64_t share = (last - first + groups) / groups;
        const int64_t from = first + group * share;
        const int64_t to = from + share < last + 1 ? from + share : last + 1;
        if (inside) {
            add_partials(a, from, to, first, i0, k, sum);
        }
        for (int s = width; s < 64; s <<= 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum[e] += __shfl_xor(sum[e], s);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            parts[wave][lane][e] = sum[e];
        }
        __syncthreads();
        if (wave == 0 && inside && lane < width) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum[e] = 0.0f;
                for (int v = 0; v < kJoinWaves; ++v) {
                    sum[e] += parts[v][lane][e];
                }
            }
            store_row(a, a.keys[i0], k, sum);
        }
        __syncthreads();
    }
}

template <int W>
hipError_t launch_lookup(const EmbeddingArgs& a, int y_type, dim3 grid, hipStream_t stream) {
    switch (y_type) {
        case LSSO_HIP_F16: lookup_kernel<W, LSSO_HIP_F16><<<grid, kLookupThreads, 0, stream>>>(a); break;
        case LSSO_HIP_BF16: lookup_kernel<W, LSSO_HIP_BF16><<<grid, kLookupThreads, 0, stream>>>(a); break;
        default: lookup_kernel<W, LSSO_HIP_F32><<<grid, kLookupThreads, 0, stream>>>(a); break;
    }
    return hipGetLastError();
}

template <int G>
void launch_sum(const EmbeddingArgs& a, dim3 grid, hipStream_t stream) {
    switch (a.weight_type) {
        case LSSO_HIP_F16: sum_kernel<G, LSSO_HIP_F16><<<grid, kSumThreads, 0, stream>>>(a); break;
        case LSSO_HIP_BF16: sum_kernel<G, LSSO_HIP_BF16><<<grid, kSumThreads, 0, stream>>>(a); break;
        default: sum_kernel<G, LSSO_HIP_F32><<<grid, kSumThreads, 0, stream>>>(a); break;
    }
}

}  // namespace

hipError_t launch_embedding(const EmbeddingArgs& args, int y_type, hipStream_t stream) {
    if (args.count == 0) {
        return hipSuccess;
    }
    EmbeddingArgs a = args;
    // About eight steps of a thread per workgroup, fewer where that would
    // leave compute units without one.
    const int64_t per_row = a.dim >= 8 ? (a.dim + 7) / 8 : a.dim;
    int64_t rows = (8 * kLookupThreads + per_row - 1) / per_row;
    const int64_t spread = (a.count + 1023) / 1024;
    rows = rows < spread ? rows : spread;
    const int64_t least = (a.count + 0x3fffff) / 0x400000;   // a launch holds fewer than 2^32 threads
    a.block_rows = rows > least ? rows : least;
    const dim3 grid(static_cast<unsigned>((a.count + a.block_rows - 1) / a.block_rows));
    switch (a.weight_type) {
        case LSSO_HIP_F16: return launch_lookup<LSSO_HIP_F16>(a, y_type, grid, stream);
        case LSSO_HIP_BF16: return launch_lookup<LSSO_HIP_BF16>(a, y_type, grid, stream);
        default: return launch_lookup<LSSO_HIP_F32>(a, y_type, grid, stream);
    }
}

// Sizes of the gradient's steps.  Tiles of 1,024 tokens (64 per wave), more where
// that would make over 128 tiles, whose histograms every tile reads.  Chunks of
// 16 to 128 tokens: short ones keep a wave's chain of gathers short, long ones
// keep the partials few.  Sums and join together, us, 256 features (a table of 6, and
// one of 32,000) and 768:
//   16,384 tokens: chunks of 16 13.7, 15.2, 19.7; of 32 15.3, 19.4, 20.6
//   32,768: of 16 14.6, 15.8, 29.6; of 32 15.8, 19.7, 23.8
//   65,536: of 16 22.3, 25.3, 49.5; of 32 17.4, 21.9, 42.3; of 64 21.7, 29.3, 35.8
//   98,304: of 32 27.8, 28.2, 67.0; of 64 22.3, 29.0, 63.5
//   262,144: of 32 49.5, 62.6, 171; of 64 36.9, 51.6, 159; of 128 34.4, 53.1, 160
//   524,288: of 64 103, 116; of 128 93, 105
void plan_embedding_grad(EmbeddingArgs* a, size_t* bytes) {
    int64_t tile = 1024;
    while ((a->count + tile - 1) / tile > 128) {
        tile *= 2;
    }
    a->tile_tokens = tile;
    a->tiles = (a->count + tile - 1) / tile;
    a->chunk_tokens = a->count >= (1 << 19) ? 128 : a->count >= (3 << 15) ? 64 : a->count >= (1 << 15) ? 32 : 16;
    a->chunks = (a->count + a->chunk_tokens - 1) / a->chunk_tokens;
    a->key_bits = 1;
    while ((a->vocabulary >> a->key_bits) != 0) {
        ++a->key_bits;
    }
    a->passes = (a->key_bits + kDigitBits - 1) / kDigitBits;
    const size_t words = static_cast<size_t>((a->count + 63) / 64 * 64);
    const int arrays = a->passes > 1 ? 4 : 2;   // ids and indices, in two copies where passes alternate
    size_t at = 0;
    for (int i = 0; i < 4; ++i) {
        a->off_sorted[i] = at;
        at += i < arrays ? 4 * words : 0;
    }
    a->off_histograms = at;
    at += 4 * static_cast<size_t>(a->tiles) * kDigits;
    a->off_partials = at;
    at += 4 * 2 * static_cast<size_t>(a->chunks) * static_cast<size_t>(a->dim);
    *bytes = (at + 255) / 256 * 256;
}

hipError_t launch_embedding_grad(const EmbeddingArgs& args, void* workspace, int grad_type, hipStream_t stream) {
    EmbeddingArgs a = args;
    size_t bytes;
    plan_embedding_grad(&a, &bytes);
    char* base = static_cast<char*>(workspace);
    a.histograms = reinterpret_cast<uint32_t*>(base + a.off_histograms);
    a.partials = reinterpret_cast<float*>(base + a.off_partials);
    uint32_t* sorted[4];
    for (int i = 0; i < 4; ++i) {
        sorted[i] = reinterpret_cast<uint32_t*>(base + a.off_sorted[i]);
    }
    // Workgroups that write zeros: 64 KiB each and launch, at most two rounds.
    const int64_t bytes_out = a.vocabulary * a.dim * (a.weight_type == LSSO_HIP_F32 ? 4 : 2);
    const int launches = a.count > 0 ? 2 * a.passes : 1;
    const int64_t clear = (bytes_out / launches + 65535) / 65536;
    const dim3 blocks(static_cast<unsigned>(a.tiles + (clear < 512 ? clear : 512)));
    const int each = (a.key_bits + a.passes - 1) / a.passes;
    int copy = 0;
    for (int pass = 0; pass < (a.count > 0 ? a.passes : 1); ++pass) {
        SortPass p{};
        p.shift = pass * each;
        p.bits = a.key_bits - p.shift < each ? a.key_bits - p.shift : each;
        p.part = 2 * pass;
        p.parts = launches;
        if (pass > 0) {
            p.keys_in = sorted[2 * copy];
            p.index_in = sorted[2 * copy + 1];
            copy ^= 1;
        }
        p.keys_out = sorted[2 * copy];
        p.index_out = sorted[2 * copy + 1];
        sort_count_kernel<<<blocks, kSortThreads, 0, stream>>>(a, p);
        if (a.count > 0) {
            sort_scatter_kernel<<<blocks, kSortThreads, 0, stream>>>(a, p);
        }
    }
    a.keys = sorted[2 * copy];
    a.index = sorted[2 * copy + 1];
    const unsigned feature_blocks = static_cast<unsigned>((a.dim + 511) / 512);
    int64_t lanes = 8;   // of a row, eight features each, to the power of two
    while (lanes < 512 && lanes < a.dim) {
        lanes *= 2;
    }
    const int64_t per_block = kSumWaves * (512 / lanes);
    if (a.count > 0) {
        const dim3 sums(static_cast<unsigned>((a.chunks + per_block - 1) / per_block), feature_blocks);
        switch (grad_type) {
            case LSSO_HIP_F16: launch_sum<LSSO_HIP_F16>(a, sums, stream); break;
            case LSSO_HIP_BF16: launch_sum<LSSO_HIP_BF16>(a, sums, stream); break;
            default: launch_sum<LSSO_HIP_F32>(a, sums, stream); break;
        }
    }
    if (a.chunks > 1) {   // else no run goes on behind its chunk
        const dim3 joins(static_cast<unsigned>((a.chunks + kJoinWaves - 1) / kJoinWaves),
                         static_cast<unsigned>((a.dim + 8 * join_lanes(a.dim) - 1) / (8 * join_lanes(a.dim))));
        join_kernel<<<joins, kJoinThreads, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
