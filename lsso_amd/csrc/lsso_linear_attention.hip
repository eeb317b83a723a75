// Linear attention with a decay for each head, l = exp(log_decay):
//   S_t = l S_{t-1} + k_t (x) v_t,   y_t = scale q_t S_t.
// A token that the mask excludes leaves S as it is, so the exponents below count
// the tokens that are kept.
//
// One walk does the forward and the three products of its gradient:
//   out_t = sum over s <= t of l^(t-s) (a_t . b_s) c_s.
// y is the walk of (q, k, v); dq of (dy, v, k); dv of (k, q, dy) and dk of (v,
// dy, q), both from the last token to the first, which negative token strides
// make of the same kernel.  The state of the backward walk is the gradient of S.
//
// A walk takes 64 tokens at a time.  Within them the products run against each
// other, P = (a b^T) l^(t-s) below the diagonal and P c; what came before
// reaches them through the state, l^t a S; and S becomes l^n S + sum of
// l^(n-s) b_s (x) c_s.  All four are MFMAs.  S stays in the accumulators of the
// workgroup's waves, a slice of its columns in each, from the first token of
// the walk to the last, so q, k, v and y pass through HBM once and S not at all.
// The accumulators of S (row d in register and lane group, column e in the lane)
// are the operand of a S with d as the summed index, in an order of d that a is
// laid out to share in LDS; c is read transposed out of LDS once for both of its
// products.
//
// Few heads leave the device empty, so a sequence is cut into segments: a first
// launch walks pieces of all but the last of them for their states alone (b and c), a
// second makes every segment's first state of them, and the third is the walk.  A
// walk that repeats another's states (dq the forward's, dk those of dv, transposed)
// starts with the third.
//
// What is rounded: the MFMAs take 16-bit operands, and P, S and l^(n-s) c are
// FP32 values.  Each goes in as parts, every next one what is left of those before
// it: three of BF16, which hold it whole, or two of FP16 (22 bits), so that S is an
// FP32 state and outputs are rounded once.  (Two rounded parts of BF16 left S 2.4e-6
// off, and of y and the gradients enough last bits for 1.1e-4 of their norm.  They
// took 74 us a walk at 64 x 2,048 tokens of 4 heads of 64, three truncated ones 84,
// three rounded ones 86.)  FP16:
// values are brought to 2^13 and more by powers of two before they are split, and the
// sums freed of them: the decayed c of each column and each row of P (of a small
// gradient, their terms are far below FP16's normal range, and a product may pass
// 65,504), and each column of S (of many tokens, it passes 65,504 too, in one feature
// of v and not in another).
//
// What is not finite stays causal: a zero of P above the diagonal times an infinite c
// would be a NaN, so a chunk whose S shows one takes P c without it and makes its
// column NaN from its token on.
//
// Bound: what a chunk's barriers and its waves' own chains of products leave open.  64 x
// 2,048 tokens of 4 heads of 64 in BF16 (268 MB a walk, 41 us at the rate of a large
// copy): a walk takes 82 to 86 us; its waves issue 29% of their time and wait 52%, the
// MFMAs are busy 20%.  Chunks are loaded one ahead.  On the same case with two parts of
// P, S and c (74 us), slower: one barrier a chunk and LDS twice (82 us); eight waves that
// share the rows of S (79 to 104); four workgroups to a compute unit, whose registers
// spill (88).  Two chunks ahead changed nothing.

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_product.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kChunk = 64;
constexpr int kTiles = kChunk / 16;
constexpr int kPairs = 6;   // tiles of t by pairs of tiles of s, on and below the diagonal
// Where in P the pair of tiles with tile s is, of tile t >= s.
__device__ __forceinline__ constexpr int pair_of(int t, int s) { return t + (t == 3 ? 1 : 0) + (s >> 1); }
constexpr double kLog2e = 1.4426950408889634;

// log2 of the decay; a head that forgets at once (-inf) keeps l^0 = 1.
__device__ __forceinline__ float decay_rate(float log_decay) {
    const float rate = static_cast<float>(log_decay * kLog2e);
    return rate < -1.0e30f ? -1.0e30f : rate;
}

// Parts that an FP32 value goes into the matrix instructions in.
template <int T>
constexpr int kParts = T == LSSO_HIP_BF16 ? 3 : 2;

// Four FP32 values as 16-bit parts each.  BF16: upper bits, three times, which hold
// all 24 (rounded parts take a third more instructions); FP16: rounded, then what that
// left.  Of a value that is or rounds to infinity the second part is held finite: the
// opposite infinity or a NaN would make a NaN of the product.
template <int T>
__device__ __forceinline__ void split(f32x4 v, u32x2 (&part)[kParts<T>]) {
    constexpr float kMost = T == LSSO_HIP_F16 ? 64.0f : 1.0e38f;   // past any remainder
#pragma unroll
    for (int p = 0; p < kParts<T>; ++p) {
        f32x4 taken;
        if constexpr (T == LSSO_HIP_BF16) {
            uint32_t bits[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bits[i] = __float_as_uint(v[i]);
                taken[i] = __uint_as_float(bits[i] & 0xffff0000u);
            }
            part[p] = (u32x2){__builtin_amdgcn_perm(bits[1], bits[0], 0x07060302u),
                              __builtin_amdgcn_perm(bits[3], bits[2], 0x07060302u)};
        } else {
            part[p] = (u32x2){Values<T>::pack(v[0], v[1]), Values<T>::pack(v[2], v[3])};
            taken = (f32x4){Values<T>::low(part[p][0]), Values<T>::high(part[p][0]), Values<T>::low(part[p][1]),
                            Values<T>::high(part[p][1])};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] -= taken[i];
            if (p == 0) {
                v[i] = __builtin_amdgcn_fmed3f(v[i], -kMost, kMost);
            }
        }
    }
}

__device__ __forceinline__ u32x4 join(const u32x2& low, const u32x2& high) {
    return (u32x4){low[0], low[1], high[0], high[1]};
}

// Where the rows of a chunk are.  A walk goes on by one addition to a pointer: what
// a chunk costs in scalar instructions, each wave pays.  Rows in the order of the
// walk; `low` is the lowest address of a whole chunk.
struct ChunkRows {
    const char* low;
    int64_t advance;      // bytes from chunk to chunk
    int64_t stride;       // bytes from row to row
    uint32_t step;        // its size
    int records;          // bytes of a whole chunk

    // data: of token 0; the chunk that begins with `token` first.
    __device__ __forceinline__ ChunkRows(const void* data, int64_t token_stride, int bytes, int columns, int token)
        : stride(token_stride * bytes) {
        step = static_cast<uint32_t>(stride < 0 ? -stride : stride);
        low = static_cast<const char*>(data) + (stride < 0 ? token + kChunk - 1 : token) * stride;
        advance = kChunk * stride;
        const int64_t all = static_cast<int64_t>(kChunk - 1) * step + bytes * columns;
        records = all > 0x7fffffff ? 0x7fffffff : static_cast<int>(all);
    }
    __device__ __forceinline__ bool turned() const { return stride < 0; }
    // The buffer of the first `rows` rows.  Rows past them are behind its end: in a
    // turned chunk, whose last rows are its lowest, before its base, from where their
    // offsets wrap round.
    __device__ __forceinline__ BufferRsrc buffer(int rows) const {
        const int missing = kChunk - rows;
        return make_buffer(low - (turned() ? missing * stride : 0), records - static_cast<int>(missing * step));
    }
    // Offset of row 0's bytes `at` in that buffer.
    __device__ __forceinline__ uint32_t offset(int row, int rows, uint32_t at) const {
        return static_cast<uint32_t>(turned() ? rows - 1 - row : row) * step + at;
    }
    __device__ __forceinline__ uint32_t round(int count) const { return count * (turned() ? 0u - step : step); }
};

// The larger of v and of another lane's: a move within a row of 16 lanes.
template <int CONTROL>
__device__ __forceinline__ uint32_t larger_of(uint32_t v) {
    const uint32_t other = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CONTROL, 0xf, 0xf, true);
    return v > other ? v : other;
}

// The largest value of a wave's lanes, all of them not negative, as bits.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = larger_of<0x121>(v);   // row_ror:1
    v = larger_of<0x122>(v);
    v = larger_of<0x124>(v);
    v = larger_of<0x128>(v);
    const uint32_t r0 = __builtin_amdgcn_readlane(static_cast<int>(v), 0);
    const uint32_t r1 = __builtin_amdgcn_readlane(static_cast<int>(v), 16);
    const uint32_t r2 = __builtin_amdgcn_readlane(static_cast<int>(v), 32);
    const uint32_t r3 = __builtin_amdgcn_readlane(static_cast<int>(v), 48);
    return larger(larger(r0, r1), larger(r2, r3));
}

// A chunk of one tensor on its way to LDS: 64 rows of `features` 16-bit values,
// in 16-byte pieces.  WHOLE: whole pieces, and 64 rows within a buffer's 2^31
// bytes, so that a piece's address is the chunk's and a lane's own offset; rows
// and pieces that do not exist are zeros or, within the buffer, another row's.
template <int WIDTH, int THREADS, bool WHOLE>
struct ChunkLoads {
    static constexpr int kPieces = WIDTH / 8;                       // of a row
    static constexpr int kEach = kChunk * kPieces / THREADS;        // of a thread
    static_assert(kChunk * kPieces % THREADS == 0, "whole rounds");
    static_assert(THREADS % kPieces == 0, "a thread's pieces are of one column");
    u32x4 raw[kEach];
    ChunkRows rows_at;
    int features;

    __device__ __forceinline__ static int row(int i) { return (static_cast<int>(threadIdx.x) + i * THREADS) / kPieces; }
    __device__ __forceinline__ static int column(int i) {
        return 8 * ((static_cast<int>(threadIdx.x) + i * THREADS) % kPieces);
    }
    __device__ __forceinline__ ChunkLoads(const uint16_t* data, int64_t token_stride, int features_, int token)
        : rows_at(data, token_stride, 2, features_, token), features(features_) {}
    // The next chunk, of `rows` rows.
    __device__ __forceinline__ void issue(int rows) {
        if constexpr (WHOLE) {
            const BufferRsrc buffer = rows_at.buffer(rows);
            const uint32_t at = rows_at.offset(row(0), rows, 2 * column(0));
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                raw[i] = buffer_load16(buffer, at + i * rows_at.round(THREADS / kPieces));
            }
        } else {
            const char* first = rows_at.low - (rows_at.turned() ? (kChunk - 1) * rows_at.stride : 0);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint16_t* at = reinterpret_cast<const uint16_t*>(
                    first + (row(i) < rows ? row(i) : rows - 1) * rows_at.stride);
                if (features >= 8) {
                    raw[i] = load16_unaligned(at + piece_start<8>(column(i), features));
                } else {
                    raw[i] = load_short_piece(at, column(i), features);
                }
            }
        }
        rows_at.low += rows_at.advance;
    }
    // With zeros past the features, and for rows that do not count.
    __device__ __forceinline__ u32x4 piece(int i, uint64_t kept) const {
        u32x4 v = raw[i];
        if constexpr (!WHOLE) {
            if (features >= 8) {
                v = align_piece16(v, column(i), features);
            }
        }
        const bool in = column(i) < features && ((kept >> row(i)) & 1) != 0;
        return in ? v : (u32x4){0u, 0u, 0u, 0u};
    }
    // The largest bits without a sign of a row, in all lanes that have a piece of it.
    __device__ __forceinline__ static uint32_t row_most(const u32x4& v) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 pair = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
        }
        uint32_t most = pair[0] > pair[1] ? pair[0] : pair[1];
        most = larger_of<0xb1>(most);        // quad_perm 1, 0, 3, 2
        most = larger_of<0x4e>(most);        // quad_perm 2, 3, 0, 1
        if constexpr (kPieces >= 8) {
            most = larger_of<0x141>(most);   // row_half_mirror
        }
        if constexpr (kPieces >= 16) {
            most = larger_of<0x140>(most);   // row_mirror
        }
        return most;
    }
};

// The exponent of the power of two that brings the largest of some values to 2^13 ..
// 2^14, where FP16 parts hold their 22 bits; none of next to nothing, of an infinity
// or a NaN.
__device__ __forceinline__ int power_of(float most) {
    const int exponent = static_cast<int>((__float_as_uint(most) & 0x7fffffffu) >> 23) - 127;
    return exponent > -100 && exponent < 128 ? 13 - exponent : 0;
}
__device__ __forceinline__ float two_to(int exponent) {   // of -126 .. 127
    return __uint_as_float(static_cast<uint32_t>(127 + exponent) << 23);
}

// The largest of lanes i, i + 16, i + 32 and i + 48, in all of them.
__device__ __forceinline__ float column_max(float v) {
    const uint32_t bits = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    const uint32_t some = __float_as_uint(fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1])));
    const auto halves = __builtin_amdgcn_permlane32_swap(some, some, false, false);
    return fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// Zeros in place of the infinities and NaNs among read_columns' 8 values of the tokens
// s0 .. s0 + 3 and s0 + 16 .. s0 + 19; how far the chunk's end is from the first of them.
template <int T>
__device__ __forceinline__ float drop_wild(u32x4& v, int s0) {
    constexpr uint32_t kExponent = T == LSSO_HIP_F16 ? 0x7c00u : 0x7f80u;
    float reach = 0.0f;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const uint32_t exponent = kExponent << (16 * (i & 1));
        if ((v[i / 2] & exponent) == exponent) {
            v[i / 2] &= (i & 1) != 0 ? 0x0000ffffu : 0xffff0000u;
            reach = static_cast<float>(kChunk - (s0 + 16 * (i >> 2) + (i & 3)));
        }
    }
    return reach;
}

// 8 values of k (or s) for one lane: rows at `at` and 16 rows on, read
// transposed; lane i of 16 receives column i.
__device__ __forceinline__ u32x4 read_columns(const uint16_t* at, int pitch) {
    const u32x2 low = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at)));
    const u32x2 high =
        __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at + 16 * pitch)));
    return (u32x4){low[0], low[1], high[0], high[1]};
}

// xcd_local_block in 32 bits.
__device__ __forceinline__ uint32_t xcd_local_block32(uint32_t physical, uint32_t blocks) {
    const uint32_t per_xcd = blocks / 8;
    return physical >= per_xcd * 8 ? physical : (physical % 8) * per_xcd + physical / 8;
}

__device__ __forceinline__ void buffer_store8(u32x2 value, BufferRsrc buffer, uint32_t offset) {
    typedef __attribute__((ext_vector_type(2))) unsigned int Pair;
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(Pair, value), buffer, offset, 0, 0);
}

__device__ __forceinline__ int64_t offset_of(const WalkTensor& t, int64_t batch, int head) {
    return batch * t.batch + (head / t.heads_per) * t.head;
}

// T: type; KT: 32-feature steps of a and b; NW: waves; WE: 16-column blocks of c
// and S in a wave; WHOLE: rows are whole 16-byte pieces; STATES: the state alone
// that a piece of the sequence adds to.  Three waves of a SIMD where the registers
// of a form allow it.
template <int T, int KT, int NW, int WE, bool WHOLE, bool STATES>
__global__ __launch_bounds__(64 * NW, NW == 4 && KT * WE <= 2 && WE == 1 ? 3 : (NW == 2 && KT == 4 ? 1 : 2)) void walk_kernel(WalkArgs a) {
    constexpr int kThreads = 64 * NW;
    constexpr int kFeatures = 32 * KT;
    constexpr int kColumns = 16 * NW * WE;
    constexpr int kPitch = kFeatures + 8;        // rows 16 bytes apart modulo the banks
    constexpr int kColumnPitch = kColumns + 8;
    constexpr int PARTS = kParts<T>;
    constexpr int kPart = kPairs * 64 * 8;       // values of one part of P
    __shared__ __attribute__((aligned(16))) uint16_t lds_a[STATES ? 8 : kChunk * kPitch];
    // The state alone leaves room for two chunks, and needs a barrier less for it.
    constexpr int kBuffers = STATES ? 2 : 1;
    __shared__ __attribute__((aligned(16))) uint16_t lds_bs[kBuffers][kChunk * kPitch];
    __shared__ __attribute__((aligned(16))) uint16_t lds_cs[kBuffers][kChunk * kColumnPitch];
    // P in operand order: [part][pair][lane][8 s].
    __shared__ __attribute__((aligned(16))) uint16_t lds_p[STATES ? 8 : PARTS * kPart];
    // Of each token of the chunk: the kept ones up to it; l to the power of the kept
    // ones behind it, times scale_update; of those from it to the end of its 16; of
    // those up to it, times scale_across.
    __shared__ __attribute__((aligned(16))) float rank[kChunk];
    __shared__ __attribute__((aligned(16))) float to_ends[kBuffers][kChunk];
    __shared__ __attribute__((aligned(16))) float to_tile[kChunk];
    __shared__ __attribute__((aligned(16))) float from_start[kChunk];
    // FP16: the largest bits of each row of a and of b.
    constexpr bool kScaled = T == LSSO_HIP_F16 && !STATES;
    __shared__ uint32_t most_a[kScaled ? kChunk : 1];
    __shared__ uint32_t most_b[kScaled ? kChunk : 1];
    __shared__ __attribute__((aligned(16))) float unscale[kScaled ? kColumns : 4];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int in = lane & 15;
    const int group = lane >> 4;

    // Heads of a token next to each other, on one XCD: they share lines.
    // (In 32 bits: a division of 64 takes longer than a chunk's products.)
    const uint32_t blocks_across = static_cast<uint32_t>((a.out_features + kColumns - 1) / kColumns);
    const uint32_t parts = static_cast<uint32_t>(STATES ? a.pieces : a.segments);
    const uint32_t index = static_cast<uint32_t>(xcd_local_block32(blockIdx.x, gridDim.x));
    const uint32_t row_of_blocks = index / blocks_across;
    const int column0 = static_cast<int>(index - row_of_blocks * blocks_across) * kColumns;
    const uint32_t row_of_heads = row_of_blocks / static_cast<uint32_t>(a.heads);
    const int head = static_cast<int>(row_of_blocks - row_of_heads * static_cast<uint32_t>(a.heads));
    const uint32_t batch = row_of_heads / parts;
    const uint32_t part = row_of_heads - batch * parts;
    const int64_t system = static_cast<int64_t>(batch) * a.heads + head;
    const int size = a.features * a.out_features;

    const uint16_t* from_a = static_cast<const uint16_t*>(a.a.data) + offset_of(a.a, batch, head);
    const uint16_t* from_b = static_cast<const uint16_t*>(a.b.data) + offset_of(a.b, batch, head);
    const uint16_t* from_c = static_cast<const uint16_t*>(a.c.data) + offset_of(a.c, batch, head);
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + batch * a.mask_batch;
    const float rate = decay_rate(a.log_decay[head]);

    const int length = static_cast<int>(a.length);
    const int chunks = (length + kChunk - 1) / kChunk;
    const int segment_chunks = static_cast<int>(a.segment_chunks);
    const int piece_chunks = static_cast<int>(a.piece_chunks);
    const int segment = static_cast<int>(STATES ? part / static_cast<uint32_t>(a.segment_pieces) : part);
    const int piece = STATES ? static_cast<int>(part) - segment * static_cast<int>(a.segment_pieces) : 0;
    const int begin = segment * segment_chunks + piece * piece_chunks;
    const int behind = STATES && (piece + 1) * piece_chunks < segment_chunks ? begin + piece_chunks
                                                                             : (segment + 1) * segment_chunks;
    const int end = behind < chunks ? behind : chunks;

    ChunkLoads<kFeatures, kThreads, WHOLE> loads_a(from_a, a.a.token, a.features, begin * kChunk);
    ChunkLoads<kFeatures, kThreads, WHOLE> loads_b(from_b, a.b.token, a.features, begin * kChunk);
    ChunkLoads<kColumns, kThreads, WHOLE> loads_c(from_c + column0, a.c.token, a.out_features - column0,
                                                  begin * kChunk);
    uint8_t kept_byte = 0;
    const auto rows_of = [&](int chunk) {
        const int left = length - chunk * kChunk;
        return left < kChunk ? left : kChunk;
    };
    const auto issue = [&](int chunk) {
        const int rows = rows_of(chunk);
        if constexpr (!STATES) {
            loads_a.issue(rows);
        }
        loads_b.issue(rows);
        loads_c.issue(rows);
        kept_byte = lane >= rows ? 0 : (mask == nullptr ? 1 : mask[(chunk * kChunk + lane) * a.mask_token]);
    };
    if (begin < end) {
        issue(begin);
    }

    // S: rows 16 dt + 4 group + r, column column0 + 16 (wave WE + we) + in.
    f32x4 state[2 * KT][WE];
    const auto state_row = [](int lane_, int dt, int r) { return 16 * dt + 4 * (lane_ >> 4) + r; };
    const auto state_column = [&](int lane_, int we) { return column0 + 16 * (wave * WE + we) + (lane_ & 15); };
    const float* first = nullptr;
    int row_stride = a.out_features;
    int column_stride = 1;
    // 1 as long as the exponents of the first state are one less than those of the tokens.
    int pending = 0;
    if constexpr (!STATES) {
        if (a.segments > 1) {
            first = a.states + (system * a.segments + part) * size;
            row_stride = static_cast<int>(a.states_row);
            column_stride = static_cast<int>(a.states_column);
        } else if (a.first != nullptr) {
            first = a.first + system * size;
            row_stride = static_cast<int>(a.first_row);
            column_stride = static_cast<int>(a.first_column);
        }
        pending = a.shift;
        for (int64_t i = 0; i < part * a.segment_pieces && pending != 0; ++i) {
            pending = a.counts[batch * a.pieces + i] == 0 ? 1 : 0;
        }
    }
    // Of a transposed state a lane's rows are neighbours in memory: four to a load (34
    // us instead of 36 a walk at 2 x 4,096 tokens of 6 heads of 128 in FP16, before its
    // powers of two).  Four
    // columns to a load of the other order, exchanged among four lanes, were no faster.
    if (!STATES && first != nullptr && row_stride == 1 && a.features % 4 == 0) {   // uniform
#pragma unroll
        for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                const int d = state_row(lane, dt, 0);
                const int e = state_column(lane, we);
                const bool in_state = d < a.features && e < a.out_features;
                float v[4];
                load_values<LSSO_HIP_F32, 4>(first + (in_state ? d + e * column_stride : 0), v);
                state[dt][we] = in_state ? (f32x4){v[0], v[1], v[2], v[3]} : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
    } else {
#pragma unroll
        for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
            for (int we = 0; we < WE; ++we) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = state_row(lane, dt, r);
                    const int e = state_column(lane, we);
                    float v = 0.0f;
                    if (!STATES && first != nullptr) {   // uniform
                        const bool in_state = d < a.features && e < a.out_features;
                        v = first[in_state ? d * row_stride + e * column_stride : 0];
                        v = in_state ? v : 0.0f;
                    }
                    state[dt][we][r] = v;
                }
            }
        }
    }
    if constexpr (!STATES) {
        // Of a short tile the other half of its 32 s: zeros, and never written again.
#pragma unroll
        for (int i = 0; i < kTiles; i += 2) {
            if (wave == i % NW) {
                uint16_t* to = lds_p + (pair_of(i, i) * 64 + lane) * 8 + 4;
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    *reinterpret_cast<u32x2*>(to + p * kPart) = (u32x2){0u, 0u};
                }
            }
        }
    }
    const bool exact = a.features == kFeatures && column0 + kColumns <= a.out_features;
    int counted = 0;
    // 2 to the power of it is past features * scale_within * l^(t-s).
    const float widest = static_cast<float>(a.features) * fabsf(a.scale_within) *
                         __builtin_amdgcn_exp2f(static_cast<float>(kChunk) * fmaxf(rate, 0.0f));
    const int past_scale =
        __builtin_amdgcn_readfirstlane(static_cast<int>(__float_as_uint(widest) >> 23)) - 126;

    const int out_bytes = a.wide_out != 0 ? 4 : 2;
    ChunkRows rows_out(static_cast<const char*>(a.out.data) + out_bytes * (offset_of(a.out, batch, head) + column0),
                       a.out.token, out_bytes, a.out_features - column0, begin * kChunk);
    const auto write = [&](int chunk, uint64_t keep, f32x4 (&out)[kTiles][WE]) {
        const int rows = rows_of(chunk);
        if (keep != ~uint64_t{0}) {   // uniform
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    out[tile][we] =
                        ((keep >> (16 * tile + in)) & 1) != 0 ? out[tile][we] : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
        }
        if constexpr (WHOLE) {
            const BufferRsrc buffer = rows_out.buffer(rows);
            const int e = 16 * wave * WE + 4 * group;
            const uint32_t at = rows_out.offset(in, rows, out_bytes * e);
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                const bool some = e + 16 * we < a.out_features - column0;
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    const f32x4 v = out[tile][we];
                    const uint32_t to = some ? at + tile * rows_out.round(16) + 16 * out_bytes * we : kOutOfRange;
                    if (a.wide_out != 0) {
                        buffer_store16(__builtin_bit_cast(u32x4, v), buffer, to);
                    } else {
                        buffer_store8((u32x2){Values<T>::pack(v[0], v[1]), Values<T>::pack(v[2], v[3])}, buffer, to);
                    }
                }
            }
            rows_out.low += rows_out.advance;
        } else {
            const int own = opaque_int(lane);   // nothing of this path is held across the loop
            const int e0 = column0 + 16 * wave * WE + 4 * (own >> 4);
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                const int t = 16 * tile + (own & 15);
                const int64_t at = offset_of(a.out, batch, head) + (chunk * kChunk + t) * a.out.token + e0;
#pragma unroll
                for (int we = 0; we < WE; ++we) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int c = 16 * we + r;
                        if (t < rows && e0 + c < a.out_features) {
                            if (a.wide_out != 0) {
                                static_cast<float*>(const_cast<void*>(a.out.data))[at + c] = out[tile][we][r];
                            } else {
                                Values<T>::store(static_cast<uint16_t*>(const_cast<void*>(a.out.data)) + at + c,
                                                 out[tile][we][r]);
                            }
                        }
                    }
                }
            }
        }
    };

    for (int chunk = begin; chunk < end; ++chunk) {
        uint16_t* lds_b = lds_bs[STATES ? chunk & 1 : 0];
        uint16_t* lds_c = lds_cs[STATES ? chunk & 1 : 0];
        float* to_end = to_ends[STATES ? chunk & 1 : 0];
        const uint64_t kept = __ballot(kept_byte != 0);
        const int total = __popcll(kept);
        const int less = total > 0 ? pending : 0;
        const bool full = exact && total == kChunk;
        {
            const int count = __popcll(kept & (~uint64_t{0} >> (63 - lane)));
            if (wave == 0) {
                rank[lane] = static_cast<float>(count);
                from_start[lane] = a.scale_across * __builtin_amdgcn_exp2f(rate * static_cast<float>(count - less));
            }
            if (wave == NW - 1) {
                const int tile_end = __popcll(kept & (~uint64_t{0} >> (63 - (lane | 15))));
                to_end[lane] = a.scale_update * __builtin_amdgcn_exp2f(rate * static_cast<float>(total - count));
                to_tile[lane] = a.scale_within * __builtin_amdgcn_exp2f(rate * static_cast<float>(tile_end - count));
            }
        }
        const auto stage = [&](bool whole) {
            if constexpr (!STATES) {
#pragma unroll
                for (int i = 0; i < loads_a.kEach; ++i) {
                    // Within 32 features the order 8 g + 4 h + r of feature 16 h + 4 g
                    // + r, which is the order of S's rows in a lane group's registers.
                    const u32x4 v = whole ? loads_a.raw[i] : loads_a.piece(i, kept);
                    const int column = loads_a.column(i);
                    uint16_t* to =
                        lds_a + loads_a.row(i) * kPitch + (column & ~31) + 2 * (column & 8) + ((column & 16) >> 2);
                    *reinterpret_cast<u32x2*>(to) = (u32x2){v[0], v[1]};
                    *reinterpret_cast<u32x2*>(to + 8) = (u32x2){v[2], v[3]};
                    if constexpr (kScaled) {
                        const uint32_t most = loads_a.row_most(v);
                        if (column == 0) {
                            most_a[loads_a.row(i)] = most;
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < loads_b.kEach; ++i) {
                const u32x4 v = whole ? loads_b.raw[i] : loads_b.piece(i, kept);
                *reinterpret_cast<u32x4*>(lds_b + loads_b.row(i) * kPitch + loads_b.column(i)) = v;
                if constexpr (kScaled) {
                    const uint32_t most = loads_b.row_most(v);
                    if (loads_b.column(i) == 0) {
                        most_b[loads_b.row(i)] = most;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < loads_c.kEach; ++i) {
                *reinterpret_cast<u32x4*>(lds_c + loads_c.row(i) * kColumnPitch + loads_c.column(i)) =
                    whole ? loads_c.raw[i] : loads_c.piece(i, kept);
            }
        };
        if (WHOLE && full) {
            stage(true);
        } else {
            stage(false);
        }
        __syncthreads();
        if (chunk + 1 < end) {
            issue(chunk + 1);
        }
        f32x4 out[kTiles][WE];
        // FP16: the exponent of the power of two of the row of P that the lane has of a
        // tile.  |a_t . b_s| is below features * 2^(of a_t's largest + of the chunk's
        // largest b + 2): P comes to 2^15 at most, and a value of 2^-17 of that bound
        // still has its 22 bits.  (No power is above 2^60, so that what came before, which
        // is multiplied by it too, stays finite.)
        int most_key = 0;
        if constexpr (kScaled) {
            const uint32_t key = most_b[lane];   // P is no number, scaled or not, where b is none
            most_key = static_cast<int>(wave_max(key < 0x7c00u ? key : 0u) >> 10);
        }
        const auto row_power = [&](int tile) {
            int query = 0;
            if constexpr (kScaled) {
                query = static_cast<int>(most_a[16 * tile + in] >> 10);
            }
            const int past = (query > 1 ? query : 1) + (most_key > 1 ? most_key : 1) - 28 + past_scale;
            const int power = 15 - past;
            return power > 60 ? 60 : (power < -100 ? -100 : power);
        };
        // FP16: the exponent of the power of two for each column of S.
        int held[WE];
#pragma unroll
        for (int we = 0; we < WE; ++we) {
            held[we] = 0;
            if constexpr (T == LSSO_HIP_F16) {
                float most = 0.0f;
#pragma unroll
                for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        most = fmaxf(most, fabsf(state[dt][we][r]));
                    }
                }
                held[we] = power_of(column_max(most));
            }
        }
        if constexpr (!STATES) {
            // P: its tiles of 16 s by 16 t, lane column t, rows s; those below the
            // diagonal and then those on it dealt to the waves.
            const auto product = [&](int tile, int s) {
                f32x4 score = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    const u32x4 query =
                        *reinterpret_cast<const u32x4*>(lds_a + (16 * tile + in) * kPitch + 32 * k + 8 * group);
                    const uint16_t* row = lds_b + (16 * s + in) * kPitch + 32 * k + 4 * group;
                    score = mfma_small<T>(
                        join(*reinterpret_cast<const u32x2*>(row), *reinterpret_cast<const u32x2*>(row + 16)), query,
                        score);
                }
                return score;
            };
            const auto put = [&](int tile, int s, f32x4 score) {
                if constexpr (kScaled) {
                    score *= ldexpf(1.0f, row_power(tile));
                }
                u32x2 parts_of[PARTS];
                split<T>(score, parts_of);
                uint16_t* to = lds_p + (pair_of(tile, s) * 64 + lane) * 8 + 4 * (s & 1);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    *reinterpret_cast<u32x2*>(to + p * kPart) = parts_of[p];
                }
            };
            constexpr int kBelow = kTiles * (kTiles - 1) / 2;
#pragma unroll
            for (int round = (kBelow - 1) / NW; round >= 0; --round) {
                const int index = round * NW + wave;   // 0: (1, 0); 1, 2: (2, s); 3 .. 5: (3, s)
                if (index < kBelow) {
                    const int tile = index >= 3 ? 3 : (index >= 1 ? 2 : 1);
                    const int s = index - tile * (tile - 1) / 2;
                    // l^(t - s) by the end of the tile of s, between the two: neither factor is above 1.
                    const float after =
                        __builtin_amdgcn_exp2f(rate * (rank[16 * tile + in] - rank[16 * s + 15]));
                    put(tile, s, product(tile, s) * *reinterpret_cast<const f32x4*>(to_tile + 16 * s + 4 * group) * after);
                }
            }
#pragma unroll
            for (int tile = wave; tile < kTiles; tile += NW) {
                f32x4 score = product(tile, tile);
                const float rank_t = rank[16 * tile + in];
                const f32x4 rank_s = *reinterpret_cast<const f32x4*>(rank + 16 * tile + 4 * group);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float weight = a.scale_within * __builtin_amdgcn_exp2f(rate * (rank_t - rank_s[r]));
                    score[r] = 4 * group + r <= in ? score[r] * weight : 0.0f;
                }
                put(tile, tile, score);
            }
            // a S, before the chunk's own tokens reach S.  FP16: each column of S times a power
            // of two, which y's rows e are freed of.
            const int own = opaque_int(lane);   // no address of these is held across the loop
            float factor[WE];
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                factor[we] = two_to(held[we]);
                if (kScaled && own < 16) {
                    unscale[16 * (wave * WE + we) + own] = two_to(-held[we]);
                }
            }
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    out[tile][we] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                u32x4 from_state[WE][PARTS];
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    u32x2 upper[PARTS];
                    u32x2 lower[PARTS];
                    split<T>(state[2 * k][we] * factor[we], upper);
                    split<T>(state[2 * k + 1][we] * factor[we], lower);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        from_state[we][p] = join(upper[p], lower[p]);
                    }
                }
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    const u32x4 query =
                        *reinterpret_cast<const u32x4*>(lds_a + (16 * tile + in) * kPitch + 32 * k + 8 * group);
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) {
                            out[tile][we] = mfma_small<T>(from_state[we][p], query, out[tile][we]);
                        }
                    }
                }
            }
            if constexpr (kScaled) {
                wave_lds_order();   // unscale: this wave's own columns
            }
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                float weight = from_start[16 * tile + in];
                if constexpr (kScaled) {
                    weight = ldexpf(weight, row_power(tile));
                }
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    out[tile][we] *= weight;
                    if constexpr (kScaled) {
                        out[tile][we] *= *reinterpret_cast<const f32x4*>(unscale + 16 * (wave * WE + we) + 4 * (own >> 4));
                    }
                }
            }
        }
        pending -= less;
        counted += total;
        // The tiles' powers, a byte each: behind the barrier most_a is the next chunk's.
        uint32_t powers = 0;
        if constexpr (kScaled) {
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                powers |= static_cast<uint32_t>(row_power(tile) & 0xff) << (8 * tile);
            }
        }
        // c of the lane's column e, and S decayed.  FP16: a power of two brings l^(n-s) c of
        // each column to its range; S is multiplied by it too, which must not pass 2^100,
        // and freed of it at the end.
        const float decay = __builtin_amdgcn_exp2f(rate * static_cast<float>(total - less));
        u32x4 value[2][WE];
        float power[WE];
        const auto weighted = [&](int j, int we, int h) {   // of 4 tokens
            const u32x4& raw = value[j][we];
            const f32x4 c = {Values<T>::low(raw[2 * h]), Values<T>::high(raw[2 * h]), Values<T>::low(raw[2 * h + 1]),
                             Values<T>::high(raw[2 * h + 1])};
            return c * *reinterpret_cast<const f32x4*>(to_end + 32 * j + 16 * h + 4 * group);
        };
        const auto read_value = [&](int j, int we) {
            value[j][we] = read_columns(
                lds_c + (32 * j + 4 * group + (in >> 2)) * kColumnPitch + 16 * (wave * WE + we) + 4 * (in & 3), kColumnPitch);
        };
#pragma unroll
        for (int we = 0; we < WE; ++we) {
            power[we] = 1.0f;
            if constexpr (T == LSSO_HIP_F16) {
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    read_value(j, we);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const f32x4 v = weighted(j, we, h);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            most = fmaxf(most, fabsf(v[i]));
                        }
                    }
                }
                const int room = held[we] + 87;   // to 2^100
                const int wanted = power_of(column_max(most));
                const int exponent = wanted < room ? wanted : room;
                power[we] = two_to(exponent);
                // The weighted values are made again: held, they cost 16 registers more.
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    asm volatile("" : "+v"(value[j][we]) : : "memory");
                }
            }
#pragma unroll
            for (int dt = 0; dt < 2 * KT; ++dt) {
                state[dt][we] *= decay * power[we];
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {   // 32 tokens s
            u32x4 decayed[WE][PARTS];
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                if constexpr (T != LSSO_HIP_F16) {
                    read_value(j, we);
                }
                u32x2 upper[PARTS];
                u32x2 lower[PARTS];
                split<T>(weighted(j, we, 0) * power[we], upper);
                split<T>(weighted(j, we, 1) * power[we], lower);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    decayed[we][p] = join(upper[p], lower[p]);
                }
            }
            const uint16_t* keys = lds_b + (32 * j + 4 * group + (in >> 2)) * kPitch + 4 * (in & 3);
#pragma unroll
            for (int dt = 0; dt < 2 * KT; ++dt) {
                const u32x4 key = read_columns(keys + 16 * dt, kPitch);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
                        state[dt][we] = mfma_small<T>(key, decayed[we][p], state[dt][we]);
                    }
                }
            }
        }
        if constexpr (T == LSSO_HIP_F16) {
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                const float back = __uint_as_float((254u << 23) - __float_as_uint(power[we]));
#pragma unroll
                for (int dt = 0; dt < 2 * KT; ++dt) {
                    state[dt][we] *= back;
                }
            }
        }
        if constexpr (!STATES) {
            // P is whole, and nobody reads the chunk any more: the next one may be staged.
            __syncthreads();
            // A c that is not finite made S so.  P's zeros for earlier tokens must not meet
            // it: from its token on the column is a NaN, and the product takes a zero.
            bool broken = false;
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                broken = broken || !finite(state[0][we][0]);
            }
            if (__any(broken)) {
                const int own = opaque_int(lane);   // nothing of this path is held across the loop
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    float reach = 0.0f;   // from the first such token of the column to the chunk's end
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        reach = fmaxf(reach, drop_wild<T>(value[j][we], 32 * j + 4 * (own >> 4)));
                    }
                    reach = column_max(reach);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int clean = kChunk - static_cast<int>(__shfl(reach, 4 * (own >> 4) + r)) - (own & 15);
#pragma unroll
                        for (int tile = 0; tile < kTiles; ++tile) {
                            out[tile][we][r] = 16 * tile < clean ? out[tile][we][r] : __builtin_nanf("");
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int tile = 2 * j; tile < kTiles; ++tile) {
                    const uint16_t* from = lds_p + (pair_of(tile, 2 * j) * 64 + lane) * 8;
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        const u32x4 score = *reinterpret_cast<const u32x4*>(from + p * kPart);
#pragma unroll
                        for (int we = 0; we < WE; ++we) {
                            out[tile][we] = mfma_small<T>(value[j][we], score, out[tile][we]);
                        }
                    }
                }
            }
            if constexpr (kScaled) {
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    const float back = ldexpf(1.0f, -static_cast<int8_t>(powers >> (8 * tile)));
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
                        out[tile][we] *= back;
                    }
                }
            }
            if (a.out.data != nullptr) {
                write(chunk, kept, out);
            }
        }
    }

    float* to = nullptr;
    float multiplier = 1.0f;
    if constexpr (STATES) {
        to = a.updates + (system * a.pieces + part) * size;
        if (head == 0 && column0 == 0 && tid == 0) {
            a.counts[batch * a.pieces + part] = counted;
        }
    } else if (a.last != nullptr && part == a.segments - 1) {
        to = a.last + system * size;
        // The walk's own exponents are one less than those of a state before its
        // last token, which a walk to the front ends with.
        multiplier = a.shift != 0 && pending == 0 ? __builtin_amdgcn_exp2f(rate) : 1.0f;
    }
    if (to != nullptr) {
        const int own = opaque_int(lane);
#pragma unroll
        for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
            for (int we = 0; we < WE; ++we) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = state_row(own, dt, r);
                    const int e = state_column(own, we);
                    if (d < a.features && e < a.out_features) {
                        to[d * a.out_features + e] = state[dt][we][r] * multiplier;
                    }
                }
            }
        }
    }
}

// The state before the first token of each segment, from what the pieces add; V
// elements of it to a thread, AHEAD pieces in flight.
constexpr int kCarryThreads = 256;
template <int V, int AHEAD>
__global__ __launch_bounds__(kCarryThreads) void carry_kernel(WalkArgs a) {
    const int size = a.features * a.out_features;
    const uint32_t blocks = static_cast<uint32_t>((size + V * kCarryThreads - 1) / (V * kCarryThreads));
    const uint32_t system = blockIdx.x / blocks;   // batch, head
    const int i = static_cast<int>((blockIdx.x - system * blocks) * kCarryThreads + threadIdx.x) * V;
    const uint32_t batch = system / static_cast<uint32_t>(a.heads);
    const float rate = decay_rate(a.log_decay[system - batch * static_cast<uint32_t>(a.heads)]);
    const bool mine = i < size;
    float state[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        state[v] = 0.0f;
        if (a.first != nullptr && mine) {
            const int d = (i + v) / a.out_features;
            state[v] = a.first[static_cast<int64_t>(system) * size + d * a.first_row +
                               (i + v - d * a.out_features) * a.first_column];
        }
    }
    int pending = a.shift;
    const int each = static_cast<int>(a.segment_pieces);
    int left = 0;   // pieces of the segment
    const float* from = a.updates + system * a.pieces * size + (mine ? i : 0);
    const int* counts = a.counts + batch * a.pieces;
    float* to = a.states + system * a.segments * size + i;
    const int pieces = static_cast<int>(a.pieces);
    const int lane = static_cast<int>(threadIdx.x) & (AHEAD - 1);
    const auto store = [&]() {
        if (mine) {
            store_values<LSSO_HIP_F32, V>(to, state);
        }
        to += size;
    };
    for (int s0 = 0; s0 < pieces; s0 += AHEAD) {
        const int some = pieces - s0 < AHEAD ? pieces - s0 : AHEAD;
        // One load of all the counts: a scalar load of each would be waited for.
        const int these = counts[s0 + (lane < some ? lane : 0)];
        float update[AHEAD][V];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {   // the last one again where there are fewer
            load_values<LSSO_HIP_F32, V>(from + static_cast<int64_t>(s0 + (j < some ? j : some - 1)) * size, update[j]);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (j < some) {   // uniform
                if (left == 0) {
                    store();
                    left = each;
                }
                --left;
                const int count = __builtin_amdgcn_readlane(these, j);
                const int less = count > 0 ? pending : 0;
                pending -= less;
                const float decay = __builtin_amdgcn_exp2f(rate * static_cast<float>(count - less));
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    state[v] = state[v] * decay + update[j][v];
                }
            }
        }
    }
    store();   // of the last segment
}

template <int T, int KT, int NW, int WE, bool WHOLE>
void launch_form(const WalkArgs& a, hipStream_t stream) {
    constexpr int kColumns = 16 * NW * WE;
    const int64_t across = (a.out_features + kColumns - 1) / kColumns;
    const int64_t systems = a.batch * a.heads;
    if (a.segments > 1 && a.reuse == 0) {
        walk_kernel<T, KT, NW, WE, WHOLE, true>
            <<<static_cast<unsigned>(systems * a.pieces * across), 64 * NW, 0, stream>>>(a);
        // Four elements to a thread where that leaves a workgroup to each compute unit.
        const int64_t elements = a.features * a.out_features;
        const int64_t blocks = (elements + 4 * kCarryThreads - 1) / (4 * kCarryThreads);
        if (elements % 4 != 0 || systems * blocks < 256) {
            carry_kernel<1, 32><<<static_cast<unsigned>(systems * ((elements + kCarryThreads - 1) / kCarryThreads)),
                                  kCarryThreads, 0, stream>>>(a);
        } else if (a.pieces > 4) {
            carry_kernel<4, 16><<<static_cast<unsigned>(systems * blocks), kCarryThreads, 0, stream>>>(a);
        } else {
            carry_kernel<4, 4><<<static_cast<unsigned>(systems * blocks), kCarryThreads, 0, stream>>>(a);
        }
    }
    walk_kernel<T, KT, NW, WE, WHOLE, false>
        <<<static_cast<unsigned>(systems * a.segments * across), 64 * NW, 0, stream>>>(a);
}

template <int T, int KT, bool WHOLE>
void launch_columns(const WalkArgs& a, hipStream_t stream) {
    if (a.out_features <= 32) {
        launch_form<T, KT, 2, 1, WHOLE>(a, stream);
    } else if (KT == 4 || a.out_features <= 64) {   // two column blocks a wave do not fit beside 128 rows of S
        launch_form<T, KT, 4, 1, WHOLE>(a, stream);
    } else {
        launch_form<T, KT, 4, KT == 4 ? 1 : 2, WHOLE>(a, stream);
    }
}

template <int T, bool WHOLE>
void launch_features(const WalkArgs& a, hipStream_t stream) {
    if (a.features <= 32) {
        launch_columns<T, 1, WHOLE>(a, stream);
    } else if (a.features <= 64) {
        launch_columns<T, 2, WHOLE>(a, stream);
    } else {
        launch_columns<T, 4, WHOLE>(a, stream);
    }
}

template <int T>
__global__ __launch_bounds__(256) void head_sum_kernel(HeadSumArgs a, int64_t count) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += stride) {
        const int64_t head = i / a.features;
        const float* at = a.partial + (head * a.shared) * a.features + (i - head * a.features);
        float total = 0.0f;
        for (int s = 0; s < a.shared; ++s) {
            total += at[static_cast<int64_t>(s) * a.features];
        }
        Values<T>::store(static_cast<typename Values<T>::Element*>(a.out) + i, total);
    }
}

// One token: a workgroup for each sequence and head.  S is read and written
// once, four columns to a thread, and everything is FP32.  Bound: HBM, 34 us for 128
// sequences of 12 heads of 128 x 128, 8% of them masked (186 MB, 5.8 TB/s).
constexpr int kStepThreads = 256;
constexpr int kStepRows = 4;   // rows of S of a thread in flight
template <int T, bool WHOLE>
__global__ __launch_bounds__(kStepThreads) void attention_step_kernel(AttentionStepArgs a) {
    using Element = typename Values<T>::Element;
    __shared__ float query[kWalkFeatures];
    __shared__ float key[kWalkFeatures];
    __shared__ float value[kWalkFeatures];
    __shared__ f32x4 parts[kStepThreads];
    const int tid = threadIdx.x;
    const int64_t batch = blockIdx.x / a.heads;
    const int head = static_cast<int>(blockIdx.x - batch * a.heads);
    Element* y = static_cast<Element*>(a.y) + (batch * a.heads + head) * static_cast<int64_t>(a.value_features);
    if (a.mask != nullptr && a.mask[batch] == 0) {
        if (tid < a.value_features) {
            Values<T>::store(y + tid, 0.0f);
        }
        return;   // the whole workgroup
    }
    if (tid < a.features) {
        query[tid] = Values<T>::load(static_cast<const Element*>(a.q.data) + offset_of(a.q, batch, head) + tid);
        key[tid] = Values<T>::load(static_cast<const Element*>(a.k.data) + offset_of(a.k, batch, head) + tid);
    }
    if (tid < a.value_features) {
        value[tid] = Values<T>::load(static_cast<const Element*>(a.v.data) + offset_of(a.v, batch, head) + tid);
    }
    const float decay = __builtin_amdgcn_exp2f(decay_rate(a.log_decay[head]));
    __syncthreads();
    const int across = (a.value_features + 3) / 4;
    int lanes = 1;
    while (lanes < across) {
        lanes *= 2;   // at most 32
    }
    const int rows = kStepThreads / lanes;
    const int e = 4 * (tid % lanes);
    float* state = a.state + batch * a.state_batch + static_cast<int64_t>(head) * a.features * a.value_features;
    f32x4 total = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e < a.value_features) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = WHOLE || e + i < a.value_features ? value[e + i] : 0.0f;
        }
        for (int d0 = tid / lanes; d0 < a.features; d0 += kStepRows * rows) {
            f32x4 s[kStepRows];
#pragma unroll
            for (int r = 0; r < kStepRows; ++r) {
                const int d = d0 + r * rows;
                if (d < a.features) {
                    const float* at = state + d * a.value_features + e;
                    if constexpr (WHOLE) {
                        s[r] = *reinterpret_cast<const f32x4*>(at);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[r][i] = e + i < a.value_features ? at[i] : 0.0f;
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < kStepRows; ++r) {
                const int d = d0 + r * rows;
                if (d < a.features) {
                    float* at = state + d * a.value_features + e;
                    s[r] = s[r] * decay + v * key[d];
                    total += s[r] * query[d];
                    if constexpr (WHOLE) {
                        *reinterpret_cast<f32x4*>(at) = s[r];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (e + i < a.value_features) {
                                at[i] = s[r][i];
                            }
                        }
                    }
                }
            }
        }
    }
    parts[tid] = total;
    __syncthreads();
    if (tid < a.value_features) {
        float sum = 0.0f;
        for (int r = 0; r < rows; ++r) {
            sum += parts[r * lanes + tid / 4][tid % 4];
        }
        Values<T>::store(y + tid, a.scale * sum);
    }
}

}  // namespace

void plan_walk(WalkArgs* a) {
    const int64_t chunks = (a->length + kChunk - 1) / kChunk;
    const int64_t systems = a->batch * a->heads;
    // As many segments as the device holds at once (three workgroups to a compute unit,
    // of more than 64 features two: a round more costs its whole time), but none
    // shorter than two chunks; pieces of them until there are 1,024 workgroups.
    const bool wide = a->features > 64 || a->out_features > 64;
    const int64_t blocks = systems * (a->features > 64 && a->out_features > 64 ? 2 : 1);
    const auto parts = [&](int64_t held, int64_t whole) {   // of `whole` chunks
        const int64_t count = blocks > 0 ? held / blocks : 1;
        const int64_t most = (whole + 1) / 2;
        return count > most ? most : (count > 1 ? count : int64_t{1});
    };
    const int64_t segments = chunks > 0 ? parts(wide ? 512 : 768, chunks) : 1;
    a->segment_chunks = chunks > 0 ? (chunks + segments - 1) / segments : 1;
    a->segments = chunks > 0 ? (chunks + a->segment_chunks - 1) / a->segment_chunks : 1;
    a->segment_pieces = a->segments > 1 ? parts(1024 / (a->segments - 1), a->segment_chunks) : 1;
    a->piece_chunks = (a->segment_chunks + a->segment_pieces - 1) / a->segment_pieces;
    a->segment_pieces = (a->segment_chunks + a->piece_chunks - 1) / a->piece_chunks;
    a->pieces = (a->segments - 1) * a->segment_pieces;
}

hipError_t launch_walk(const WalkArgs& a, int dtype, hipStream_t stream) {
    const auto near = [](const WalkTensor& t) { return t.token < (1 << 23) && t.token > -(1 << 23); };
    const bool whole = a.features % 8 == 0 && a.out_features % 8 == 0 && near(a.a) && near(a.b) && near(a.c);
    if (dtype == LSSO_HIP_F16) {
        whole ? launch_features<LSSO_HIP_F16, true>(a, stream) : launch_features<LSSO_HIP_F16, false>(a, stream);
    } else {
        whole ? launch_features<LSSO_HIP_BF16, true>(a, stream) : launch_features<LSSO_HIP_BF16, false>(a, stream);
    }
    return hipGetLastError();
}

hipError_t launch_head_sum(const HeadSumArgs& a, int dtype, hipStream_t stream) {
    const int64_t count = a.rows * a.kv_heads * a.features;
    const int64_t blocks = (count + 255) / 256;
    const unsigned grid = static_cast<unsigned>(blocks < 65536 ? blocks : 65536);
    if (dtype == LSSO_HIP_F16) {
        head_sum_kernel<LSSO_HIP_F16><<<grid, 256, 0, stream>>>(a, count);
    } else {
        head_sum_kernel<LSSO_HIP_BF16><<<grid, 256, 0, stream>>>(a, count);
    }
    return hipGetLastError();
}

hipError_t launch_attention_step(const AttentionStepArgs& a, int dtype, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.batch * a.heads);
    const bool whole = a.value_features % 4 == 0 && a.state_batch % 4 == 0 &&
                       reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
    if (dtype == LSSO_HIP_F16) {
        whole ? attention_step_kernel<LSSO_HIP_F16, true><<<grid, kStepThreads, 0, stream>>>(a)
              : attention_step_kernel<LSSO_HIP_F16, false><<<grid, kStepThreads, 0, stream>>>(a);
    } else {
        whole ? attention_step_kernel<LSSO_HIP_BF16, true><<<grid, kStepThreads, 0, stream>>>(a)
              : attention_step_kernel<LSSO_HIP_BF16, false><<<grid, kStepThreads, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
