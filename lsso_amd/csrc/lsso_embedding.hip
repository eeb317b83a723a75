// Token embedding y[t] = scale * W[token[t]] and the gradient of its table,
//   dW[v] = scale * sum over the counted tokens t with token[t] = v of dy[t].
//
// Forward: a copy with an index, bound by HBM (the rows that are named, once,
// and y).  A workgroup takes whole rows, a thread 8 elements of one row at a
// time, with its rows' steps unrolled so that several id -> row -> store chains
// are in flight.
//
// Gradient: floats added by atomics would make the sums' order, and so their
// rounding, change from call to call, and rows that many tokens share (six
// symbols in 262,144 tokens) would queue at one address.  Instead the tokens
// are sorted by id (stable, so a row's tokens keep their order), and each row
// is summed once, in FP32, in an order that depends on the sizes alone:
//   1. radix sort of (id, index) in one or two passes of up to 10 bits: a
//      histogram per tile of tokens, then a stable scatter that ranks equal
//      digits of 64 lanes by ballots and takes its bases from the histograms;
//   2. a wave finds the runs of up to 8 table rows by a 64-ary search (three probes
//      of the sorted ids for 262,144 tokens) and adds up those of at most 8 tokens;
//      rows that no token names are written as zeros here;
//   3. beside it, in the same launch, a wave per chunk of the sorted order adds up
//      the longer runs, and leaves partial sums of those that cross its ends: the
//      frequent words of a text lie side by side, and by rows a few waves had
//      nearly all tokens (365 us instead of about 30 at 32,800 tokens of 768);
//   4. the partials of each such run are added, by a wave or a workgroup.
// Tokens that count nowhere (excluded, padding, out of range) get the id
// `vocabulary` and sort behind every row.
//
// Bound: reading dy (gathered whole rows) and writing dW, plus the latency of
// four or six launches.

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
constexpr int kFewTokens = 8;    // longest run that the wave of its row sums
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

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(EmbeddingArgs a, SortPass p) {
    __shared__ uint32_t histogram[kDigits];
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

// Sum of dy rows index[i0 .. i1) over 8 features of this lane, taken by the
// groups of `width` lanes in turn and then joined, the same in every group.
template <int G>
__device__ __forceinline__ void sum_rows(const EmbeddingArgs& a, int64_t i0, int64_t i1, int k, int lane, int width,
                                         float (&sum)[8]) {
    const auto* dy = static_cast<const typename Values<G>::Element*>(a.grad_y);
    const int groups = 64 / width;
    const int dim = static_cast<int>(a.dim);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        sum[e] = 0.0f;
    }
    for (int64_t base = i0; base < i1; base += 64) {
        // One load brings the next 64 indices, a shuffle hands them out.
        const int mine = static_cast<int>(a.index[base + lane < i1 ? base + lane : base]);
        const int here = static_cast<int>(i1 - base < 64 ? i1 - base : 64);
#pragma unroll 8
        for (int i = 0; i < here; i += groups) {
            const int at = i + lane / width;
            const int64_t token = __shfl(mine, at < 64 ? at : 0);
            const auto* row = dy + token * a.grad_stride;
            float v[8];
            if (dim >= 8) {
                Values<G>::load8(row + k, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = e < dim ? Values<G>::load(row + e) : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // Not 0 * v: what a lane reads past the run may be anything.
                sum[e] += at < here ? v[e] : 0.0f;
            }
        }
    }
    for (int s = width; s < 64; s <<= 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum[e] += __shfl_xor(sum[e], s);
        }
    }
}

__device__ __forceinline__ void store_row(const EmbeddingArgs& a, int64_t row, int k, const float (&sum)[8]) {
    const auto put = [&](auto values) {
        using V = decltype(values);
        auto* at = static_cast<typename V::Element*>(a.grad_weight) + row * a.dim;
        if (a.dim >= 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = a.scale * sum[e];
            }
            V::store8(at + k, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (e < a.dim) {
                    V::store(at + e, a.scale * sum[e]);
                }
            }
        }
    };
    if (a.weight_type == LSSO_HIP_F32) {
        put(Values<LSSO_HIP_F32>());
    } else if (a.weight_type == LSSO_HIP_BF16) {
        put(Values<LSSO_HIP_BF16>());
    } else {
        put(Values<LSSO_HIP_F16>());
    }
}

// Lanes that share a row: the power of two that covers its pieces, at most 64.
__device__ __forceinline__ int row_lanes(int64_t dim) {
    int width = 1;
    while (width < 64 && 8 * width < dim) {
        width *= 2;
    }
    return width;
}

// Features of this lane in feature block `block` (64 lanes x 8 features).
__device__ __forceinline__ int lane_feature(const EmbeddingArgs& a, int block, int lane, int width, bool& inside) {
    const int piece = 64 * block + (lane & (width - 1));
    const int dim = static_cast<int>(a.dim);
    inside = 8 * piece < dim;
    return dim < 8 || !inside ? 0 : piece_at(piece, dim);
}

// Bound by the latency of ids -> index -> gathered rows of dy; a wave keeps up to 8
// of the rows in flight.  32,800 tokens of 768 features, a third of them excluded,
// and 32,000 table rows: 50 us; 262,144 tokens of 256 features and 6 rows: 29 us,
// 4.6 TB/s of dy.
// Workgroups past row_blocks take the chunks of long runs.
template <int G>
__global__ __launch_bounds__(kSumThreads) void row_sum_kernel(EmbeddingArgs a) {
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int width = row_lanes(a.dim);
    const int blocks = static_cast<int>((a.dim + 511) / 512);
    float sum[8];
    if (blockIdx.x < a.row_blocks) {
        // wave_rows consecutive rows: one search for the first one's run, then the
        // others' borders from the next 64 ids, where those reach far enough.
        const int64_t first = (static_cast<int64_t>(blockIdx.x) * kSumWaves + wave) * a.wave_rows;
        const int64_t end = first + a.wave_rows < a.vocabulary ? first + a.wave_rows : a.vocabulary;
        if (first >= end) {
            return;
        }
        int64_t i0 = first_at_least(a.keys, a.count, static_cast<uint32_t>(first), lane);
        int64_t window = i0;   // position of the ids in `ahead`
        uint32_t ahead = window + lane < a.count ? a.keys[window + lane] : ~0u;
        for (int64_t row = first; row < end; ++row) {
            const int inside = __popcll(__ballot(ahead <= static_cast<uint32_t>(row)));
            int64_t i1 = window + inside;
            if (inside == 64) {   // the run may go on behind the window
                i1 = i0 + first_at_least(a.keys + i0, a.count - i0, static_cast<uint32_t>(row) + 1, lane);
                window = i1;
                ahead = window + lane < a.count ? a.keys[window + lane] : ~0u;
            }
            if (i1 - i0 <= kFewTokens) {   // a longer one goes by chunks
                for (int block = 0; block < blocks; ++block) {
                    bool inside_row;
                    const int k = lane_feature(a, block, lane, width, inside_row);
                    sum_rows<G>(a, i0, i1, k, lane, width, sum);
                    if (inside_row && lane < width) {
                        store_row(a, row, k, sum);
                    }
                }
            }
            i0 = i1;
        }
        return;
    }
    // The runs of more than kFewTokens that chunk c meets: one that lies inside it
    // is summed here, one that begins before it or goes on behind it leaves a
    // partial sum, in slot 0 if it holds the chunk's first position, else in 1.
    const int64_t c = static_cast<int64_t>(blockIdx.x - a.row_blocks) * kSumWaves + wave;
    if (c >= a.chunks) {
        return;
    }
    const int64_t c0 = c * a.chunk_tokens;
    const int64_t c1 = c0 + a.chunk_tokens < a.count ? c0 + a.chunk_tokens : a.count;
    const uint32_t before = c0 > 0 ? a.keys[c0 - 1] : ~0u;
    const uint32_t behind = c1 < a.count ? a.keys[c1] : ~0u;
    for (int64_t base = c0; base < c1;) {
        // One run a turn: its end among the next 64 ids, or the chunk's.
        const uint32_t ahead = base + lane < c1 ? a.keys[base + lane] : ~0u;
        const uint32_t key = __shfl(ahead, 0);
        int64_t end = base + __popcll(__ballot(ahead == key));
        while (end < c1 && a.keys[end] == key) {   // a chunk may be longer than a wave
            end = base + first_at_least(a.keys + base, c1 - base, key + 1, lane);
        }
        if (key >= a.vocabulary) {
            break;
        }
        const bool crosses = (base == c0 && before == key) || (end == c1 && behind == key);
        int64_t length = end - base;
        if (crosses && length <= kFewTokens) {
            const int64_t i0 = base == c0 ? first_at_least(a.keys, a.count, key, lane) : base;
            length = first_at_least(a.keys + i0, a.count - i0, key + 1, lane);
        }
        if (length > kFewTokens) {
            for (int block = 0; block < blocks; ++block) {
                bool inside;
                const int k = lane_feature(a, block, lane, width, inside);
                sum_rows<G>(a, base, end, k, lane, width, sum);
                if (inside && lane < width) {
                    if (!crosses) {
                        store_row(a, key, k, sum);
                    } else {
                        float* at = a.partials + (2 * c + (base == c0 ? 0 : 1)) * a.dim;
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
                    }
                }
            }
        }
        base = end;
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
    const int width = row_lanes(a.dim);
    const int lane_groups = 64 / width;
    bool inside;
    const int k = lane_feature(a, blockIdx.y, lane, width, inside);
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
            if (i1 - i0 > kFewTokens && last - c < kWaveChunks) {
                if (inside && lane < width) {
                    float sum[8] = {};
                    add_partials(a, c, last + 1, c, i0, k, sum);
                    store_row(a, key, k, sum);
                }
            } else if (i1 - i0 > kFewTokens) {
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
// 32 to 128 tokens: short ones keep a wave's chain of gathers short, long ones
// keep the partials few.  Rows per wave: up to 8, so that a large table's empty
// rows share a search (2, 4, 8: 24, 22, 20 us for 8,192 tokens of a table of 32,000
// x 256; 53, 48, 55 for 32,800 of 768), while a small table still has 2,048 waves;
// more where a launch would otherwise pass 2^32 threads.
void plan_embedding_grad(EmbeddingArgs* a, size_t* bytes) {
    int64_t tile = 1024;
    while ((a->count + tile - 1) / tile > 128) {
        tile *= 2;
    }
    const int64_t least = (a->vocabulary + (1 << 24) - 1) >> 24;
    a->wave_rows = a->vocabulary >= 8 * 2048 ? 8 : a->vocabulary / 2048 > 1 ? a->vocabulary / 2048 : 1;
    a->wave_rows = a->wave_rows > least ? a->wave_rows : least;
    a->tile_tokens = tile;
    a->tiles = (a->count + tile - 1) / tile;
    a->chunk_tokens = a->count >= (1 << 19) ? 128 : a->count >= (1 << 17) ? 64 : 32;
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
    const dim3 tiles(static_cast<unsigned>(a.tiles));
    const int each = (a.key_bits + a.passes - 1) / (a.passes > 0 ? a.passes : 1);
    int copy = 0;
    if (a.count > 0) {
        for (int pass = 0; pass < a.passes; ++pass) {
            SortPass p{};
            p.shift = pass * each;
            p.bits = a.key_bits - p.shift < each ? a.key_bits - p.shift : each;
            if (pass > 0) {
                p.keys_in = sorted[2 * copy];
                p.index_in = sorted[2 * copy + 1];
                copy ^= 1;
            }
            p.keys_out = sorted[2 * copy];
            p.index_out = sorted[2 * copy + 1];
            sort_count_kernel<<<tiles, kSortThreads, 0, stream>>>(a, p);
            sort_scatter_kernel<<<tiles, kSortThreads, 0, stream>>>(a, p);
        }
    }
    a.keys = sorted[2 * copy];
    a.index = sorted[2 * copy + 1];
    const unsigned feature_blocks = static_cast<unsigned>((a.dim + 511) / 512);
    a.row_blocks = (a.vocabulary + kSumWaves * a.wave_rows - 1) / (kSumWaves * a.wave_rows);
    const int64_t chunk_blocks = a.count > kFewTokens ? (a.chunks + kSumWaves - 1) / kSumWaves : 0;
    const dim3 sums(static_cast<unsigned>(a.row_blocks + chunk_blocks));
    switch (grad_type) {
        case LSSO_HIP_F16: row_sum_kernel<LSSO_HIP_F16><<<sums, kSumThreads, 0, stream>>>(a); break;
        case LSSO_HIP_BF16: row_sum_kernel<LSSO_HIP_BF16><<<sums, kSumThreads, 0, stream>>>(a); break;
        default: row_sum_kernel<LSSO_HIP_F32><<<sums, kSumThreads, 0, stream>>>(a); break;
    }
    if (a.chunks > 1) {   // else no run goes on behind its chunk
        join_kernel<<<dim3(static_cast<unsigned>((a.chunks + kJoinWaves - 1) / kJoinWaves), feature_blocks), kJoinThreads,
                      0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
