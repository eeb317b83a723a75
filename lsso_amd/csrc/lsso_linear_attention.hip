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
// launch walks all but the last of them for their states alone (b and c), a
// second makes every segment's first state of them, and the third is the walk.
//
// What is rounded: the MFMAs take 16-bit operands, and P, S and l^(n-s) c are
// FP32 values.  P and S go in as two 16-bit parts, the second what rounding left
// of the first, so that outputs are off by one rounding of their own; one part
// would leave sqrt(2) to sqrt(3).  l^(n-s) c, which makes the FP32 state, goes in
// as two parts of FP16 and three of BF16 (two leave a state 2.4e-6 off).
// FP16: S is scaled by a power of two that brings its largest value in a wave to
// 2^14 before it is split (the state of many tokens passes 65,504); P must stay
// below 65,504.

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_product.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kChunk = 64;
constexpr int kTiles = kChunk / 16;
constexpr double kLog2e = 1.4426950408889634;

// log2 of the decay; a head that forgets at once (-inf) keeps l^0 = 1.
__device__ __forceinline__ float decay_rate(float log_decay) {
    const float rate = static_cast<float>(log_decay * kLog2e);
    return rate < -1.0e30f ? -1.0e30f : rate;
}

// Four FP32 values as PARTS 16-bit ones each: rounded, then what that left.  Of
// a value that rounds to infinity the second part is held finite: the opposite
// infinity or a NaN would make a NaN of the product.
template <int T, int PARTS>
__device__ __forceinline__ void split(f32x4 v, u32x2 (&part)[PARTS]) {
    constexpr float kMost = T == LSSO_HIP_F16 ? 64.0f : 1.0e38f;   // past any rounding error
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        part[p] = (u32x2){Values<T>::pack(v[0], v[1]), Values<T>::pack(v[2], v[3])};
        if (p + 1 < PARTS) {
            const f32x4 rounded = {Values<T>::low(part[p][0]), Values<T>::high(part[p][0]),
                                   Values<T>::low(part[p][1]), Values<T>::high(part[p][1])};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __builtin_amdgcn_fmed3f(v[i] - rounded[i], -kMost, kMost);
            }
        }
    }
}

__device__ __forceinline__ u32x4 join(const u32x2& low, const u32x2& high) {
    return (u32x4){low[0], low[1], high[0], high[1]};
}

// A chunk of one tensor on its way to LDS: 64 rows of `features` 16-bit values,
// in 16-byte pieces, zeros past the features.
template <int WIDTH, int THREADS, bool WHOLE>
struct ChunkLoads {
    static constexpr int kPieces = WIDTH / 8;                       // of a row
    static constexpr int kEach = kChunk * kPieces / THREADS;        // of a thread
    static_assert(kChunk * kPieces % THREADS == 0, "whole rounds");
    u32x4 raw[kEach];

    __device__ __forceinline__ static int row(int i) { return (static_cast<int>(threadIdx.x) + i * THREADS) / kPieces; }
    __device__ __forceinline__ static int column(int i) {
        return 8 * ((static_cast<int>(threadIdx.x) + i * THREADS) % kPieces);
    }
    // rows: how many of the chunk exist; those past it read the last one.
    __device__ __forceinline__ void issue(const uint16_t* from, int64_t stride, int rows, int features, int column0) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = row(i) < rows ? row(i) : rows - 1;
            const uint16_t* at = from + r * stride;
            const int k = column0 + column(i);
            if constexpr (WHOLE) {
                raw[i] = load16_unaligned(at + (k < features ? k : 0));
            } else if (features >= 8) {
                raw[i] = load16_unaligned(at + piece_start<8>(k, features));
            } else {
                raw[i] = load_short_piece(at, k, features);
            }
        }
    }
    __device__ __forceinline__ u32x4 piece(int i, uint64_t kept, int features, int column0) const {
        const int k = column0 + column(i);
        u32x4 v = raw[i];
        if constexpr (!WHOLE) {
            if (features >= 8) {
                v = align_piece16(v, k, features);
            }
        }
        const bool in = k < features && ((kept >> row(i)) & 1) != 0;
        return in ? v : (u32x4){0u, 0u, 0u, 0u};
    }
};

// 8 values of k (or s) for one lane: rows at `at` and 16 rows on, read
// transposed; lane i of 16 receives column i.
__device__ __forceinline__ u32x4 read_columns(const uint16_t* at, int pitch) {
    const u32x2 low = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at)));
    const u32x2 high =
        __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at + 16 * pitch)));
    return (u32x4){low[0], low[1], high[0], high[1]};
}

__device__ __forceinline__ int64_t offset_of(const WalkTensor& t, int64_t batch, int head) {
    return batch * t.batch + (head / t.heads_per) * t.head;
}

// T: type; KT: 32-feature steps of a and b; NW: waves; WE: 16-column blocks of c
// and S in a wave; WHOLE: rows are whole 16-byte pieces; STATES: the segment's
// state alone.
template <int T, int KT, int NW, int WE, bool WHOLE, bool STATES>
__global__ __launch_bounds__(64 * NW) void walk_kernel(WalkArgs a) {
    constexpr int kThreads = 64 * NW;
    constexpr int kFeatures = 32 * KT;
    constexpr int kColumns = 16 * NW * WE;
    constexpr int kPitch = kFeatures + 8;        // rows 16 bytes apart modulo the banks
    constexpr int kColumnPitch = kColumns + 8;
    constexpr int kParts = T == LSSO_HIP_BF16 ? 3 : 2;   // of the decayed c
    __shared__ __attribute__((aligned(16))) uint16_t lds_a[STATES ? 8 : kChunk * kPitch];
    __shared__ __attribute__((aligned(16))) uint16_t lds_b[kChunk * kPitch];
    __shared__ __attribute__((aligned(16))) uint16_t lds_c[kChunk * kColumnPitch];
    // P in operand order: [part][tile of t][32 s][lane][8 s].
    __shared__ __attribute__((aligned(16))) uint16_t lds_p[STATES ? 8 : 2 * kTiles * 2 * 64 * 8];
    __shared__ __attribute__((aligned(16))) float rank[kChunk];   // kept tokens of the chunk up to each

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = tid >> 6;
    const int in = lane & 15;
    const int group = lane >> 4;

    // Heads of a token next to each other, on one XCD: they share lines.
    const int blocks_across = (a.out_features + kColumns - 1) / kColumns;
    int64_t block = xcd_local_block(blockIdx.x, gridDim.x);
    const int column0 = static_cast<int>(block % blocks_across) * kColumns;
    block /= blocks_across;
    const int head = static_cast<int>(block % a.heads);
    block /= a.heads;
    const int64_t segments = STATES ? a.segments - 1 : a.segments;   // the last one's state is the walk's own
    const int64_t segment = block % segments;
    const int64_t batch = block / segments;

    const uint16_t* from_a = static_cast<const uint16_t*>(a.a.data) + offset_of(a.a, batch, head);
    const uint16_t* from_b = static_cast<const uint16_t*>(a.b.data) + offset_of(a.b, batch, head);
    const uint16_t* from_c = static_cast<const uint16_t*>(a.c.data) + offset_of(a.c, batch, head);
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + batch * a.mask_batch;
    const float rate = decay_rate(a.log_decay[head]);
    const int64_t slot = (batch * a.heads + head) * static_cast<int64_t>(a.features) * a.out_features;

    const int64_t chunks = (a.length + kChunk - 1) / kChunk;
    const int64_t begin = segment * a.segment_chunks;
    const int64_t end = begin + a.segment_chunks < chunks ? begin + a.segment_chunks : chunks;

    // S: rows 16 dt + 4 group + r, column column0 + 16 (wave WE + we) + in.
    f32x4 state[2 * KT][WE];
#pragma unroll
    for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
        for (int we = 0; we < WE; ++we) {
            state[dt][we] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    const auto state_row = [&](int dt, int r) { return 16 * dt + 4 * group + r; };
    const auto state_column = [&](int we) { return column0 + 16 * (wave * WE + we) + in; };
    // 1 as long as the exponents of the first state are one less than those of the tokens.
    int pending = 0;
    if constexpr (!STATES) {
        const float* first = nullptr;
        int64_t row_stride = a.out_features;
        int64_t column_stride = 1;
        if (a.segments > 1) {
            first = a.states + ((batch * a.heads + head) * a.segments + segment) *
                                   (static_cast<int64_t>(a.features) * a.out_features);
        } else if (a.first != nullptr) {
            first = a.first + slot;
            row_stride = a.first_row;
            column_stride = a.first_column;
        }
        if (first != nullptr) {
#pragma unroll
            for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
                for (int we = 0; we < WE; ++we) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = state_row(dt, r);
                        const int e = state_column(we);
                        if (d < a.features && e < a.out_features) {
                            state[dt][we][r] = first[d * row_stride + e * column_stride];
                        }
                    }
                }
            }
        }
        pending = a.shift;
        for (int64_t i = 0; i < segment && pending != 0; ++i) {
            pending = a.counts[batch * a.segments + i] == 0 ? 1 : 0;
        }
    }
    int64_t counted = 0;

    ChunkLoads<kFeatures, kThreads, WHOLE> loads_a;
    ChunkLoads<kFeatures, kThreads, WHOLE> loads_b;
    ChunkLoads<kColumns, kThreads, WHOLE> loads_c;
    uint8_t kept_byte = 0;
    const auto issue = [&](int64_t chunk) {
        const int64_t token = chunk * kChunk;
        const int rows = static_cast<int>(a.length - token < kChunk ? a.length - token : kChunk);
        if constexpr (!STATES) {
            loads_a.issue(from_a + token * a.a.token, a.a.token, rows, a.features, 0);
        }
        loads_b.issue(from_b + token * a.b.token, a.b.token, rows, a.features, 0);
        loads_c.issue(from_c + token * a.c.token, a.c.token, rows, a.out_features, column0);
        kept_byte = lane >= rows ? 0 : (mask == nullptr ? 1 : mask[(token + lane) * a.mask_token]);
    };
    if (begin < end) {
        issue(begin);
    }
    for (int64_t chunk = begin; chunk < end; ++chunk) {
        const uint64_t kept = __ballot(kept_byte != 0);
        const int total = __popcll(kept);
        if (tid < kChunk) {
            rank[tid] = static_cast<float>(__popcll(kept & (~uint64_t{0} >> (63 - tid))));
        }
        if constexpr (!STATES) {
#pragma unroll
            for (int i = 0; i < loads_a.kEach; ++i) {
                // Within 32 features the order 8 g + 4 h + r of feature 16 h + 4 g
                // + r, which is the order of S's rows in a lane group's registers.
                const u32x4 v = loads_a.piece(i, kept, a.features, 0);
                const int column = loads_a.column(i);
                uint16_t* to = lds_a + loads_a.row(i) * kPitch + (column & ~31) + 2 * (column & 8) + ((column & 16) >> 2);
                *reinterpret_cast<u32x2*>(to) = (u32x2){v[0], v[1]};
                *reinterpret_cast<u32x2*>(to + 8) = (u32x2){v[2], v[3]};
            }
        }
#pragma unroll
        for (int i = 0; i < loads_b.kEach; ++i) {
            *reinterpret_cast<u32x4*>(lds_b + loads_b.row(i) * kPitch + loads_b.column(i)) =
                loads_b.piece(i, kept, a.features, 0);
        }
#pragma unroll
        for (int i = 0; i < loads_c.kEach; ++i) {
            *reinterpret_cast<u32x4*>(lds_c + loads_c.row(i) * kColumnPitch + loads_c.column(i)) =
                loads_c.piece(i, kept, a.out_features, column0);
        }
        __syncthreads();
        if (chunk + 1 < end) {
            issue(chunk + 1);
        }
        const int less = total > 0 ? pending : 0;
        f32x4 out[kTiles][WE];
        if constexpr (!STATES) {
            // P, a tile of 16 t in a wave: lane column t, rows s.
#pragma unroll
            for (int round = 0; round < kTiles / NW; ++round) {
                // Two tiles of a wave: one short, one long.
                const int tile = round % 2 == 0 ? wave : kTiles - 1 - wave;
                u32x4 query[KT];
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    query[k] = *reinterpret_cast<const u32x4*>(lds_a + (16 * tile + in) * kPitch + 32 * k + 8 * group);
                }
                const float rank_t = rank[16 * tile + in];
                for (int s = 0; s <= (tile | 1); ++s) {
                    f32x4 score = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (s <= tile) {
#pragma unroll
                        for (int k = 0; k < KT; ++k) {
                            const uint16_t* row = lds_b + (16 * s + in) * kPitch + 32 * k + 4 * group;
                            const u32x2 low = *reinterpret_cast<const u32x2*>(row);
                            const u32x2 high = *reinterpret_cast<const u32x2*>(row + 16);
                            score = mfma_small<T>((u32x4){low[0], low[1], high[0], high[1]}, query[k], score);
                        }
                        const f32x4 rank_s = *reinterpret_cast<const f32x4*>(rank + 16 * s + 4 * group);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float weight = a.scale_within * __builtin_amdgcn_exp2f(rate * (rank_t - rank_s[r]));
                            score[r] = s < tile || 4 * group + r <= in ? score[r] * weight : 0.0f;
                        }
                    }
                    u32x2 part[2];
                    split<T>(score, part);
                    uint16_t* to = lds_p + (((tile * 2) + (s >> 1)) * 64 + lane) * 8 + 4 * (s & 1);
                    *reinterpret_cast<u32x2*>(to) = part[0];
                    *reinterpret_cast<u32x2*>(to + kTiles * 2 * 64 * 8) = part[1];
                }
            }
            // a S, before the chunk's own tokens reach S.
            float factor = 1.0f;
            float unfactor = 1.0f;
            if constexpr (T == LSSO_HIP_F16) {
                float most = 0.0f;
#pragma unroll
                for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            most = fmaxf(most, fabsf(state[dt][we][r]));
                        }
                    }
                }
#pragma unroll
                for (int offset = 1; offset < 64; offset *= 2) {
                    most = fmaxf(most, __shfl_xor(most, offset));
                }
                const int exponent = static_cast<int>(__float_as_uint(most) >> 23) - 127;
                if (exponent > -100 && exponent < 128) {   // neither next to nothing nor infinite
                    factor = __uint_as_float(static_cast<uint32_t>(127 + 14 - exponent) << 23);
                    unfactor = __uint_as_float(static_cast<uint32_t>(127 - 14 + exponent) << 23);
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
                u32x4 high[WE];
                u32x4 low[WE];
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    u32x2 first[2];
                    u32x2 second[2];
                    split<T>(state[2 * k][we] * factor, first);
                    split<T>(state[2 * k + 1][we] * factor, second);
                    high[we] = join(first[0], second[0]);
                    low[we] = join(first[1], second[1]);
                }
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
                    const u32x4 query =
                        *reinterpret_cast<const u32x4*>(lds_a + (16 * tile + in) * kPitch + 32 * k + 8 * group);
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
                        out[tile][we] = mfma_small<T>(high[we], query, out[tile][we]);
                        out[tile][we] = mfma_small<T>(low[we], query, out[tile][we]);
                    }
                }
            }
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                const float weight = a.scale_across * unfactor *
                                     __builtin_amdgcn_exp2f(rate * (rank[16 * tile + in] - static_cast<float>(less)));
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    out[tile][we] *= weight;
                }
            }
            __syncthreads();   // P is whole
        }
        const float decay = __builtin_amdgcn_exp2f(rate * static_cast<float>(total - less));
#pragma unroll
        for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                state[dt][we] *= decay;
            }
        }
        pending -= less;
        counted += total;
#pragma unroll
        for (int j = 0; j < 2; ++j) {   // 32 tokens s
            u32x4 value[WE];
            const uint16_t* transposed =
                lds_c + (32 * j + 4 * group + (in >> 2)) * kColumnPitch + 16 * wave * WE + 4 * (in & 3);
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                value[we] = read_columns(transposed + 16 * we, kColumnPitch);
            }
            if constexpr (!STATES) {
#pragma unroll
                for (int tile = 2 * j; tile < kTiles; ++tile) {
                    const uint16_t* from = lds_p + ((tile * 2 + j) * 64 + lane) * 8;
                    const u32x4 high = *reinterpret_cast<const u32x4*>(from);
                    const u32x4 low = *reinterpret_cast<const u32x4*>(from + kTiles * 2 * 64 * 8);
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
                        out[tile][we] = mfma_small<T>(value[we], high, out[tile][we]);
                        out[tile][we] = mfma_small<T>(value[we], low, out[tile][we]);
                    }
                }
            }
            float weight[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 rank_s = *reinterpret_cast<const f32x4*>(rank + 32 * j + 16 * h + 4 * group);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    weight[4 * h + r] =
                        a.scale_update * __builtin_amdgcn_exp2f(rate * (static_cast<float>(total) - rank_s[r]));
                }
            }
            u32x4 parts[WE][kParts];
#pragma unroll
            for (int we = 0; we < WE; ++we) {
                float v[8];
                Values<T>::unpack8(value[we], v);
                u32x2 first[kParts];
                u32x2 second[kParts];
                split<T>((f32x4){v[0] * weight[0], v[1] * weight[1], v[2] * weight[2], v[3] * weight[3]}, first);
                split<T>((f32x4){v[4] * weight[4], v[5] * weight[5], v[6] * weight[6], v[7] * weight[7]}, second);
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    parts[we][p] = join(first[p], second[p]);
                }
            }
            const uint16_t* keys = lds_b + (32 * j + 4 * group + (in >> 2)) * kPitch + 4 * (in & 3);
#pragma unroll
            for (int dt = 0; dt < 2 * KT; ++dt) {
                const u32x4 key = read_columns(keys + 16 * dt, kPitch);
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
#pragma unroll
                    for (int we = 0; we < WE; ++we) {
                        state[dt][we] = mfma_small<T>(key, parts[we][p], state[dt][we]);
                    }
                }
            }
        }
        if constexpr (!STATES) {
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                const int64_t token = chunk * kChunk + 16 * tile + in;
                if (token >= a.length || a.out.data == nullptr) {
                    continue;
                }
                const bool keep = ((kept >> (16 * tile + in)) & 1) != 0;
                const int64_t row = offset_of(a.out, batch, head) + token * a.out.token;
#pragma unroll
                for (int we = 0; we < WE; ++we) {
                    const int e = column0 + 16 * (wave * WE + we) + 4 * group;
                    const f32x4 v = keep ? out[tile][we] : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                    if (a.wide_out != 0) {
                        float* to = static_cast<float*>(const_cast<void*>(a.out.data)) + row + e;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (e + r < a.out_features) {
                                to[r] = v[r];
                            }
                        }
                    } else {
                        uint16_t* to = static_cast<uint16_t*>(const_cast<void*>(a.out.data)) + row + e;
                        if (e + 4 <= a.out_features) {
                            const u32x2 packed = {Values<T>::pack(v[0], v[1]), Values<T>::pack(v[2], v[3])};
                            __builtin_memcpy(to, &packed, sizeof(packed));
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                if (e + r < a.out_features) {
                                    Values<T>::store(to + r, v[r]);
                                }
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();   // the chunk's readers are done
    }

    float* to = nullptr;
    float multiplier = 1.0f;
    if constexpr (STATES) {
        to = a.states + ((batch * a.heads + head) * a.segments + segment) *
                            (static_cast<int64_t>(a.features) * a.out_features);
        if (head == 0 && column0 == 0 && tid == 0) {
            a.counts[batch * a.segments + segment] = static_cast<int>(counted);
        }
    } else if (a.last != nullptr && segment == a.segments - 1) {
        to = a.last + slot;
        // The walk's own exponents are one less than those of a state before its
        // last token, which a walk to the front ends with.
        multiplier = a.shift != 0 && pending == 0 ? __builtin_amdgcn_exp2f(rate) : 1.0f;
    }
    if (to != nullptr) {
#pragma unroll
        for (int dt = 0; dt < 2 * KT; ++dt) {
#pragma unroll
            for (int we = 0; we < WE; ++we) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = state_row(dt, r);
                    const int e = state_column(we);
                    if (d < a.features && e < a.out_features) {
                        to[d * a.out_features + e] = state[dt][we][r] * multiplier;
                    }
                }
            }
        }
    }
}

// states: each segment's update becomes the state before its first token.
constexpr int kCarryThreads = 256;
__global__ __launch_bounds__(kCarryThreads) void carry_kernel(WalkArgs a) {
    const int size = a.features * a.out_features;
    const int blocks = (size + kCarryThreads - 1) / kCarryThreads;
    const int64_t system = blockIdx.x / blocks;   // batch, head
    const int i = static_cast<int>(blockIdx.x - system * blocks) * kCarryThreads + static_cast<int>(threadIdx.x);
    if (i >= size) {
        return;
    }
    const int64_t batch = system / a.heads;
    const int head = static_cast<int>(system - batch * a.heads);
    const float rate = decay_rate(a.log_decay[head]);
    float state = 0.0f;
    if (a.first != nullptr) {
        const int d = i / a.out_features;
        state = a.first[system * size + d * a.first_row + (i - d * a.out_features) * a.first_column];
    }
    int pending = a.shift;
    float* at = a.states + system * a.segments * size + i;
    float update = at[0];
    for (int64_t s = 0; s < a.segments; ++s) {
        const float next = s + 2 < a.segments ? at[(s + 1) * size] : 0.0f;   // in flight behind the store
        at[s * size] = state;
        if (s + 1 < a.segments) {
            const int count = a.counts[batch * a.segments + s];
            const int less = count > 0 ? pending : 0;
            pending -= less;
            state = state * __builtin_amdgcn_exp2f(rate * static_cast<float>(count - less)) + update;
        }
        update = next;
    }
}

template <int T, int KT, int NW, int WE, bool WHOLE>
void launch_form(const WalkArgs& a, hipStream_t stream) {
    constexpr int kColumns = 16 * NW * WE;
    const int64_t across = (a.out_features + kColumns - 1) / kColumns;
    const int64_t systems = a.batch * a.heads;
    if (a.segments > 1) {
        walk_kernel<T, KT, NW, WE, WHOLE, true>
            <<<static_cast<unsigned>(systems * (a.segments - 1) * across), 64 * NW, 0, stream>>>(a);
        const int64_t blocks = (a.features * a.out_features + kCarryThreads - 1) / kCarryThreads;
        carry_kernel<<<static_cast<unsigned>(systems * blocks), kCarryThreads, 0, stream>>>(a);
    }
    walk_kernel<T, KT, NW, WE, WHOLE, false>
        <<<static_cast<unsigned>(systems * a.segments * across), 64 * NW, 0, stream>>>(a);
}

template <int T, int KT, bool WHOLE>
void launch_columns(const WalkArgs& a, hipStream_t stream) {
    if (a.out_features <= 32) {
        launch_form<T, KT, 2, 1, WHOLE>(a, stream);
    } else if (a.out_features <= 64) {
        launch_form<T, KT, 4, 1, WHOLE>(a, stream);
    } else {
        launch_form<T, KT, 4, 2, WHOLE>(a, stream);
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
// once, four columns to a thread, and everything is FP32.
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
    // Segments until every compute unit has two workgroups, but none shorter than
    // four chunks: a segment costs its state's write and two reads, and a second
    // read of b and c.
    int64_t segments = systems > 0 ? (512 + systems - 1) / systems : 1;
    const int64_t most = (chunks + 3) / 4;
    segments = segments < most ? segments : most;
    segments = segments > 1 ? segments : 1;
    a->segment_chunks = (chunks + segments - 1) / segments;
    a->segment_chunks = a->segment_chunks > 0 ? a->segment_chunks : 1;
    a->segments = chunks > 0 ? (chunks + a->segment_chunks - 1) / a->segment_chunks : 1;
}

hipError_t launch_walk(const WalkArgs& a, int dtype, hipStream_t stream) {
    const bool whole = a.features % 8 == 0 && a.out_features % 8 == 0;
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
