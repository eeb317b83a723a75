// Gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its
// gradients.  All products are the tiled loop of lsso_product.h:
//
//   gate_kernel    g, u = x Wg^T, x Wu^T in one pass over x; h = act(g) * u
//                  from the FP32 accumulators.  Training also keeps g and u.
//   product_kernel y = h Wd^T, and in the backward dx = dg Wg + du Wu
//   grad_kernel    dh = dy Wd, and from it dg = dh u act'(g), du = dh act(g)
//   weight_kernel  dWg = dg^T x, dWu = du^T x, dWd = dy^T h in one launch,
//                  over row ranges whose FP32 partials join_kernel adds in order
//
// Operands are 16-bit values of x's type: x, the weights (FP32 weights are
// rounded once per call, as the projections round theirs) and g, u, h, dg, du,
// which are rounded once when they are stored, because the products that take
// them run on 16-bit matrix instructions.  g and u keep [rows, 2, Fp] and h
// [rows, Fp], Fp the hidden width rounded up to 8 with zeros behind it, so
// every row is whole 16-byte pieces.  Operands whose own rows are not (odd
// widths or strides) are copied into such rows first: element loads in the
// product's loop cost more than one more pass over x.
//
// Rows that a mask excludes: their h, dg and du are stored as zeros, their y
// and dx too, and the loads of x and dy that would carry them into a weight
// gradient are suppressed, so what they hold (NaN included) reaches nothing.

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_product.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

// act(g) and act'(g), FP32.
__device__ __forceinline__ void activation(int kind, float g, float& value, float& slope) {
    if (kind == LSSO_HIP_SILU) {
        // g far below zero: exp overflows to infinity and the sigmoid is 0.
        const float s = 1.0f / (1.0f + __expf(-g));
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        value = g * cdf;
        slope = cdf + g * 0.39894228040143268f * __expf(-0.5f * g * g);
    }
}

__device__ __forceinline__ void activation(int kind, float g, float& value) {
    if (kind == LSSO_HIP_SILU) {
        value = g * (1.0f / (1.0f + __expf(-g)));
    } else {
        value = g * (0.5f * (1.0f + erff(g * 0.70710678118654752f)));
    }
}

// Tile of this workgroup: columns fastest, so that the tiles that share P's
// rows follow each other on one XCD.
struct Tile {
    int64_t p0;
    int64_t q0;
};
__device__ __forceinline__ Tile tile_of(int64_t q_tiles, int64_t tiles, int bp, int bq) {
    const int64_t block = xcd_local_block(blockIdx.x, tiles);
    const int64_t p = block / q_tiles;
    return {p * bp, (block - p * q_tiles) * bq};
}

// Loads of one operand in rows: stage s of [k0, k1) of the rows from `base`.
template <typename Layout>
struct RowLoads {
    BufferRsrc buffer;
    uint32_t offset;       // this lane's line and element, bytes
    uint32_t step;         // bytes between the lines of consecutive loads
    int64_t element;       // this lane's element of stage 0
    int64_t elements;

    __device__ __forceinline__ RowLoads(const Operand& o, int wave, int lane, int64_t most_lines)
        : buffer(lines(o, most_lines)),
          offset(static_cast<uint32_t>(2 * (Layout::load_line(wave, lane, 0) * o.stride +
                                            Layout::load_element(wave, lane)))),
          step(static_cast<uint32_t>(2 * 64 * o.stride)),
          element(Layout::load_element(wave, lane)),
          elements(o.elements) {}
    // The same lines of another matrix of this stride.
    __device__ __forceinline__ static BufferRsrc lines(const Operand& o, int64_t most_lines) {
        return make_buffer(o.base, 2 * (o.lines < most_lines ? o.lines : most_lines) * o.stride);
    }
    __device__ __forceinline__ void issue(char* lds, int wave, int64_t k, int j) const { issue(buffer, lds, wave, k, j); }
    __device__ __forceinline__ void issue(BufferRsrc buffer, char* lds, int wave, int64_t k, int j) const {
        const uint32_t at = k + element < elements ? offset + j * step + static_cast<uint32_t>(2 * k) : kOutOfRange;
        load_to_lds(buffer, lds + 1024 * (4 * j + wave), at);
    }
};

// Loads of one operand in columns: lines are k.
template <typename Layout>
struct ColumnLoads {
    const uint16_t* base;
    int64_t stride;
    uint32_t offset;       // kOutOfRange for a lane past the columns
    uint32_t step;

    __device__ __forceinline__ ColumnLoads(const Operand& o, int wave, int lane)
        : base(o.base), stride(o.stride) {
        const int element = Layout::load_element(wave, lane);
        offset = element < o.elements
                     ? static_cast<uint32_t>(2 * (Layout::load_line(wave, lane, 0) * o.stride + element))
                     : kOutOfRange;
        step = static_cast<uint32_t>(2 * 4 * Layout::kRowsPerLoad * o.stride);
    }
    // Lines [k, min(k + kStageK, end)).
    __device__ __forceinline__ BufferRsrc stage(int64_t k, int64_t end) const {
        const int64_t lines = end - k < kStageK ? end - k : kStageK;
        return make_buffer(base + (lines > 0 ? k : 0) * stride, 2 * lines * stride);
    }
    __device__ __forceinline__ void issue(BufferRsrc buffer, char* lds, int wave, int j, bool keep = true) const {
        load_to_lds(buffer, lds + 1024 * (4 * j + wave), keep && offset != kOutOfRange ? offset + j * step : kOutOfRange);
    }
};

// ---------------------------------------------------------------- h, g and u
// Q is [gate rows | up rows] of the tile's 32 NB columns of h: wave column w
// takes gate columns 32 w .. and the same up columns, so a lane holds both
// factors of its products.
template <int T, int MB, bool KEEP>
__global__ __launch_bounds__(kProductThreads, 2) void gate_kernel(FeedForwardArgs a) {
    using S = ProductShape<T, true, true, MB, 2>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    constexpr int kColumns = S::BQ / 2;
    const Tile tile = tile_of(a.q_tiles, a.tiles, S::BP, kColumns);
    const RowLoads<typename S::PLayout> x({a.x + tile.p0 * a.x_stride, a.x_stride, a.rows - tile.p0, a.in_pitch}, wave,
                                          lane, S::BP);
    // Load 0 of Q is rows 0 .. 63 of its stage, load 1 rows 64 .. 127.
    const RowLoads<typename S::QLayout> gate({a.gate + tile.q0 * a.in_pitch, a.in_pitch, a.hidden - tile.q0,
                                              a.in_pitch}, wave, lane, kColumns);
    const RowLoads<typename S::QLayout> up({a.up + tile.q0 * a.in_pitch, a.in_pitch, a.hidden - tile.q0, a.in_pitch},
                                           wave, lane, kColumns);
    static_assert(S::QLayout::kLoads == 2 && kColumns == 64, "one load of each weight");
    f32x16 acc[2][MB];
    run_product<S>(
        lds, a.stages, acc,
        [&](char* stage, int s) {
            const int64_t k = static_cast<int64_t>(s) * kStageK;
#pragma unroll
            for (int j = 0; j < S::PLayout::kLoads; ++j) {
                x.issue(stage, wave, k, j);
            }
            char* q = stage + S::PLayout::kBytes;
            gate.issue(q, wave, k, 0);
            up.issue(q + 4096, wave, k, 0);
        },
        [&](int n) { return kColumns * n + 32 * (wave >> 1); });

    const int half = lane >> 5;
    const int64_t column = tile.q0 + 32 * (wave >> 1) + 8 * half;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row = tile.p0 + 32 * (MB * (wave & 1) + m) + (lane & 31);
        float g[2][8];
        float u[2][8];
        row_pieces(acc[0][m], g);
        row_pieces(acc[1][m], u);
        const bool inside = row < a.rows;
        const bool kept = inside && (a.row_mask == nullptr || a.row_mask[row] != 0);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (!inside || column + 16 * c >= a.pitch) {
                continue;
            }
            float h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float act;
                activation(a.activation, g[c][e], act);
                h[e] = kept ? act * u[c][e] : 0.0f;
            }
            store16_unaligned(a.h + row * a.pitch + column + 16 * c, Values<T>::pack8(h));
            if (KEEP) {
                uint16_t* at = a.gates + 2 * row * a.pitch + column + 16 * c;
                store16_unaligned(at, Values<T>::pack8(g[c]));
                store16_unaligned(at + a.pitch, Values<T>::pack8(u[c]));
            }
        }
    }
}

// ------------------------------------------------------------------ y and dx
// out = P Q^T over one or two K segments: y = h Wd^T (Q in rows, one segment)
// or dx = dg Wg + du Wu (Q in columns, two).  With `splits` > 1 the stages are
// divided and FP32 partials left for join_kernel.
template <int T, bool Q_ROWS, int MB, int NB>
__global__ __launch_bounds__(kProductThreads, 2) void product_kernel(FeedForwardProduct a) {
    using S = ProductShape<T, true, Q_ROWS, MB, NB>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const Tile tile = tile_of(a.q_tiles, a.tiles, S::BP, S::BQ);
    const int split = blockIdx.y;
    const int first = split * a.split_stages;
    const int last = first + a.split_stages < a.stages ? first + a.split_stages : a.stages;
    const Operand rows{a.p + tile.p0 * a.p_stride, a.p_stride, a.rows - tile.p0, a.k};
    const RowLoads<typename S::PLayout> p(rows, wave, lane, S::BP);
    f32x16 acc[NB][MB];
    const auto q_start = [&](int n) { return 32 * (NB * (wave >> 1) + n); };
    if constexpr (Q_ROWS) {
        const RowLoads<typename S::QLayout> q({a.q + tile.q0 * a.q_stride, a.q_stride, a.columns - tile.q0, a.k}, wave,
                                              lane, S::BQ);
        run_product<S>(
            lds, last - first, acc,
            [&](char* stage, int s) {
                const int64_t k = first + s < last ? static_cast<int64_t>(first + s) * kStageK : a.k;
#pragma unroll
                for (int j = 0; j < S::PLayout::kLoads; ++j) {
                    p.issue(stage, wave, k, j);
                }
#pragma unroll
                for (int j = 0; j < S::QLayout::kLoads; ++j) {
                    q.issue(stage + S::PLayout::kBytes, wave, k, j);
                }
            },
            q_start);
    } else {
        ColumnLoads<typename S::QLayout> q({a.q + tile.q0, a.q_stride, a.k, a.q_pitch - tile.q0}, wave, lane);
        const uint16_t* const second_q = a.q_second + tile.q0;
        const uint16_t* const first_q = q.base;
        run_product<S>(
            lds, last - first, acc,
            [&](char* stage, int s) {
                const int at = first + s;
                const bool second = at >= a.segment_stages;
                const int64_t k = at < last ? static_cast<int64_t>(at - (second ? a.segment_stages : 0)) * kStageK : a.k;
                Operand of = rows;
                of.base += second ? a.p_second : 0;
                const BufferRsrc pb = RowLoads<typename S::PLayout>::lines(of, S::BP);
#pragma unroll
                for (int j = 0; j < S::PLayout::kLoads; ++j) {
                    p.issue(pb, stage, wave, k, j);
                }
                q.base = second ? second_q : first_q;
                const BufferRsrc qb = q.stage(k, a.q_lines);
#pragma unroll
                for (int j = 0; j < S::QLayout::kLoads; ++j) {
                    q.issue(qb, stage + S::PLayout::kBytes, wave, j);
                }
            },
            q_start);
    }

    const int half = lane >> 5;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row = tile.p0 + 32 * (MB * (wave & 1) + m) + (lane & 31);
        const bool inside = row < a.rows;
        const bool kept = inside && (a.row_mask == nullptr || a.row_mask[row] != 0);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float v[2][8];
            row_pieces(acc[n][m], v);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int64_t column = tile.q0 + q_start(n) + 16 * c + 8 * half;
                if (!inside || column >= a.columns) {
                    continue;
                }
                if (a.partials != nullptr) {
                    float* at = a.partials + (split * a.rows + row) * a.partial_pitch + column;
                    Values<LSSO_HIP_F32>::store8(at, v[c]);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[c][e] = kept ? v[c][e] : 0.0f;
                }
                uint16_t* at = a.out + row * a.columns + column;
                if (column + 8 <= a.columns) {
                    Values<T>::store8(at, v[c]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (column + e < a.columns) {
                            Values<T>::store(at + e, v[c][e]);
                        }
                    }
                }
            }
        }
    }
}

// ----------------------------------------------------------------- dg and du
template <int T, int MB, int NB>
__global__ __launch_bounds__(kProductThreads, 2) void grad_kernel(FeedForwardArgs a) {
    using S = ProductShape<T, true, false, MB, NB>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const Tile tile = tile_of(a.q_tiles, a.tiles, S::BP, S::BQ);
    const RowLoads<typename S::PLayout> dy({a.dy + tile.p0 * a.dy_stride, a.dy_stride, a.rows - tile.p0, a.out_pitch},
                                           wave, lane, S::BP);
    const ColumnLoads<typename S::QLayout> down({a.down + tile.q0, a.down_pitch, a.out_features,
                                                 a.down_pitch - tile.q0}, wave, lane);
    f32x16 acc[NB][MB];
    const auto q_start = [&](int n) { return 32 * (NB * (wave >> 1) + n); };
    run_product<S>(
        lds, a.stages, acc,
        [&](char* stage, int s) {
            const int64_t k = static_cast<int64_t>(s) * kStageK;
#pragma unroll
            for (int j = 0; j < S::PLayout::kLoads; ++j) {
                dy.issue(stage, wave, k, j);
            }
            const BufferRsrc buffer = down.stage(k, a.out_features);
#pragma unroll
            for (int j = 0; j < S::QLayout::kLoads; ++j) {
                down.issue(buffer, stage + S::PLayout::kBytes, wave, j);
            }
        },
        q_start);

    const int half = lane >> 5;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row = tile.p0 + 32 * (MB * (wave & 1) + m) + (lane & 31);
        const bool inside = row < a.rows;
        const bool kept = inside && (a.row_mask == nullptr || a.row_mask[row] != 0);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float dh[2][8];
            row_pieces(acc[n][m], dh);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int64_t column = tile.q0 + q_start(n) + 16 * c + 8 * half;
                if (!inside || column >= a.pitch) {
                    continue;
                }
                const int64_t at = 2 * row * a.pitch + column;
                float g[8];
                float u[8];
                Values<T>::load8(a.gates + at, g);
                Values<T>::load8(a.gates + at + a.pitch, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float act, slope;
                    activation(a.activation, g[e], act, slope);
                    g[e] = kept ? dh[c][e] * u[e] * slope : 0.0f;
                    u[e] = kept ? dh[c][e] * act : 0.0f;
                }
                store16_unaligned(a.grads + at, Values<T>::pack8(g));
                store16_unaligned(a.grads + at + a.pitch, Values<T>::pack8(u));
            }
        }
    }
}

// ----------------------------------------------------------- weight gradients
// One of up to three products P^T Q over a range of rows, P and Q in columns.
template <int T, int MB, int NB, bool MASKED>
__global__ __launch_bounds__(kProductThreads, 2) void weight_kernel(FeedForwardWeights a) {
    using S = ProductShape<T, false, false, MB, NB>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    __shared__ uint32_t kept[MASKED ? kWeightSplitRows / 32 + kRing : 1];   // rows of each stage
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    int64_t block = xcd_local_block(blockIdx.x, gridDim.x);
    const int64_t split = block / a.tiles;
    block -= split * a.tiles;
    int which = 0;
    while (which < a.count - 1 && block >= a.products[which].tiles) {
        block -= a.products[which].tiles;
        ++which;
    }
    const WeightProduct w = a.products[which];
    const int64_t p_tile = block / w.q_tiles;
    const int64_t p0 = p_tile * S::BP;
    const int64_t q0 = (block - p_tile * w.q_tiles) * S::BQ;
    const int64_t r0 = split * a.split_rows;
    const int64_t r1 = r0 + a.split_rows < a.rows ? r0 + a.split_rows : a.rows;
    if constexpr (MASKED) {
        for (int64_t i = 64 * wave; i < a.split_rows + kRing * kStageK; i += kProductThreads) {
            const int64_t r = r0 + i + lane;
            const uint64_t rows = __ballot(r < r1 && a.row_mask[r < r1 ? r : r0] != 0);
            if (lane < 2) {
                const int word = static_cast<int>(i / 32) + lane;
                if (word < kWeightSplitRows / 32 + kRing) {
                    kept[word] = static_cast<uint32_t>(rows >> (32 * lane));
                }
            }
        }
        __syncthreads();
    }
    const ColumnLoads<typename S::PLayout> p({w.p + p0, w.p_stride, 0, w.p_columns - p0}, wave, lane);
    const ColumnLoads<typename S::QLayout> q({w.q + q0, w.q_stride, 0, w.q_columns - q0}, wave, lane);
    f32x16 acc[NB][MB];
    const auto q_start = [&](int n) { return 32 * (NB * (wave >> 1) + n); };
    run_product<S>(
        lds, static_cast<int>((r1 - r0 + kStageK - 1) / kStageK), acc,
        [&](char* stage, int s) {
            const int64_t k = r0 + static_cast<int64_t>(s) * kStageK;
            const BufferRsrc pb = p.stage(k, r1);
            const BufferRsrc qb = q.stage(k, r1);
            const uint32_t rows = MASKED ? __builtin_amdgcn_readfirstlane(kept[s]) : ~0u;
#pragma unroll
            for (int j = 0; j < S::PLayout::kLoads; ++j) {
                p.issue(pb, stage, wave, j, !MASKED || (rows >> S::PLayout::load_line(wave, lane, j)) & 1);
            }
#pragma unroll
            for (int j = 0; j < S::QLayout::kLoads; ++j) {
                q.issue(qb, stage + S::PLayout::kBytes, wave, j,
                        !MASKED || (rows >> S::QLayout::load_line(wave, lane, j)) & 1);
            }
        },
        q_start);

    const int half = lane >> 5;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row = p0 + 32 * (MB * (wave & 1) + m) + (lane & 31);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float v[2][8];
            row_pieces(acc[n][m], v);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int64_t column = q0 + q_start(n) + 16 * c + 8 * half;
                if (row < w.out_rows && column < w.partial_pitch) {
                    float* at = a.partials + split * a.partial_floats + w.partial_offset + row * w.partial_pitch + column;
                    Values<LSSO_HIP_F32>::store8(at, v[c]);
                }
            }
        }
    }
}

// Sum of `splits` partials [rows, pitch] in order, rounded once into out [rows,
// columns]; up to three such sums in one launch (blockIdx.y).
__global__ __launch_bounds__(256) void join_kernel(FeedForwardJoin a) {
    const JoinOutput o = a.outputs[blockIdx.y];
    const int64_t pieces = (o.columns + 3) / 4;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= o.rows * pieces) {
        return;
    }
    const int64_t row = i / pieces;
    const int64_t column = 4 * (i - row * pieces);
    const float* at = a.partials + o.offset + row * o.pitch + column;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int64_t s = 0; s < a.splits; ++s) {
        sum += *reinterpret_cast<const f32x4*>(at + s * a.split_floats);
    }
    if (a.row_mask != nullptr && a.row_mask[row] == 0) {
        sum = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    const auto put = [&](auto values) {
        using V = decltype(values);
        auto* out = static_cast<typename V::Element*>(o.out) + row * o.columns + column;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (column + e < o.columns) {
                V::store(out + e, sum[e]);
            }
        }
    };
    if (a.type == LSSO_HIP_F32) {
        put(Values<LSSO_HIP_F32>());
    } else if (a.type == LSSO_HIP_BF16) {
        put(Values<LSSO_HIP_BF16>());
    } else {
        put(Values<LSSO_HIP_F16>());
    }
}

// Copies of up to five matrices as 16-bit rows of `pitch` columns with zeros
// behind the last one: FP32 weights, and operands with odd rows.
template <int T>
__global__ __launch_bounds__(256) void pack_kernel(FeedForwardPack a) {
    int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    int which = 0;
    while (which < a.count && i >= a.matrices[which].pieces) {
        i -= a.matrices[which].pieces;
        ++which;
    }
    if (which == a.count) {
        return;
    }
    const PackMatrix& m = a.matrices[which];
    const int64_t per_row = m.pitch / 8;
    const int64_t row = i / per_row;
    const int64_t column = 8 * (i - row * per_row);
    float v[8];
    const auto get = [&](auto values) {
        using V = decltype(values);
        const auto* from = static_cast<const typename V::Element*>(m.from) + row * m.stride + column;
        if (column + 8 <= m.columns) {
            V::load8(from, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = column + e < m.columns ? V::load(from + e) : 0.0f;
            }
        }
    };
    if (m.wide) {
        get(Values<LSSO_HIP_F32>());
    } else {
        get(Values<T>());
    }
    store16_unaligned(m.to + row * m.pitch + column, Values<T>::pack8(v));
}

// Tile edges of a product, in 64s: P and Q.
struct Edges {
    int mb;
    int nb;
};

int64_t tiles_of(int64_t p, int64_t q, int64_t bp, int64_t bq) { return ((p + bp - 1) / bp) * ((q + bq - 1) / bq); }

// The largest tile that still gives every CU its two workgroups; the larger
// the tile, the fewer bytes a product moves between L2, LDS and registers.
constexpr int64_t kSlots = 512;

Edges choose_edges(int64_t p, int64_t q) {
    if (tiles_of(p, q, 256, 128) >= kSlots) {
        return {4, 2};
    }
    return tiles_of(p, q, 128, 128) >= kSlots / 2 ? Edges{2, 2} : Edges{1, 1};
}

int choose_gate(int64_t rows, int64_t pitch) {
    if (tiles_of(rows, pitch, 256, 64) >= kSlots) {
        return 4;
    }
    return tiles_of(rows, pitch, 128, 64) >= kSlots / 2 ? 2 : 1;
}

template <int T, bool KEEP>
void launch_gate(const FeedForwardArgs& a, int mb, dim3 grid, hipStream_t stream) {
    switch (mb) {
        case 4: gate_kernel<T, 4, KEEP><<<grid, kProductThreads, 0, stream>>>(a); break;
        case 2: gate_kernel<T, 2, KEEP><<<grid, kProductThreads, 0, stream>>>(a); break;
        default: gate_kernel<T, 1, KEEP><<<grid, kProductThreads, 0, stream>>>(a); break;
    }
}

template <int T>
hipError_t launch_gate(const FeedForwardArgs& args, hipStream_t stream) {
    FeedForwardArgs a = args;
    const int mb = choose_gate(a.rows, a.pitch);
    a.stages = static_cast<int>((a.in_pitch + kStageK - 1) / kStageK);
    a.q_tiles = (a.pitch + 63) / 64;
    a.tiles = a.q_tiles * ((a.rows + 64 * mb - 1) / (64 * mb));
    const dim3 grid(static_cast<unsigned>(a.tiles));
    a.gates != nullptr ? launch_gate<T, true>(a, mb, grid, stream) : launch_gate<T, false>(a, mb, grid, stream);
    return hipGetLastError();
}

template <int T, bool Q_ROWS>
hipError_t launch_product(const FeedForwardProduct& args, hipStream_t stream) {
    FeedForwardProduct a = args;
    const Edges e{a.mb, a.nb};
    a.q_tiles = (a.columns + 64 * e.nb - 1) / (64 * e.nb);
    a.tiles = a.q_tiles * ((a.rows + 64 * e.mb - 1) / (64 * e.mb));
    const dim3 grid(static_cast<unsigned>(a.tiles), static_cast<unsigned>(a.splits));
    if (a.splits == 1) {
        a.partials = nullptr;
    }
    switch (e.mb) {
        case 4: product_kernel<T, Q_ROWS, 4, 2><<<grid, kProductThreads, 0, stream>>>(a); break;
        case 2: product_kernel<T, Q_ROWS, 2, 2><<<grid, kProductThreads, 0, stream>>>(a); break;
        default: product_kernel<T, Q_ROWS, 1, 1><<<grid, kProductThreads, 0, stream>>>(a); break;
    }
    const hipError_t error = hipGetLastError();
    if (a.splits == 1 || error != hipSuccess) {
        return error;
    }
    FeedForwardJoin join{};
    join.partials = a.partials;
    join.splits = a.splits;
    join.split_floats = a.rows * a.partial_pitch;
    join.row_mask = a.row_mask;
    join.type = T;
    join.outputs[0] = {0, a.partial_pitch, a.rows, a.columns, a.out};
    join_kernel<<<dim3(static_cast<unsigned>((a.rows * ((a.columns + 3) / 4) + 255) / 256), 1), 256, 0, stream>>>(join);
    return hipGetLastError();
}

template <int T>
hipError_t launch_grad(const FeedForwardArgs& args, hipStream_t stream) {
    FeedForwardArgs a = args;
    const Edges e = choose_edges(a.rows, a.pitch);
    a.stages = static_cast<int>((a.out_pitch + kStageK - 1) / kStageK);
    a.q_tiles = (a.pitch + 64 * e.nb - 1) / (64 * e.nb);
    a.tiles = a.q_tiles * ((a.rows + 64 * e.mb - 1) / (64 * e.mb));
    const dim3 grid(static_cast<unsigned>(a.tiles));
    switch (e.mb) {
        case 4: grad_kernel<T, 4, 2><<<grid, kProductThreads, 0, stream>>>(a); break;
        case 2: grad_kernel<T, 2, 2><<<grid, kProductThreads, 0, stream>>>(a); break;
        default: grad_kernel<T, 1, 1><<<grid, kProductThreads, 0, stream>>>(a); break;
    }
    return hipGetLastError();
}

template <int T, bool MASKED>
void launch_weights(const FeedForwardWeights& a, int mb, dim3 grid, hipStream_t stream) {
    if (mb == 4) {
        weight_kernel<T, 4, 2, MASKED><<<grid, kProductThreads, 0, stream>>>(a);
    } else {
        weight_kernel<T, 2, 2, MASKED><<<grid, kProductThreads, 0, stream>>>(a);
    }
}

template <int T>
hipError_t launch_weights(const FeedForwardWeights& args, hipStream_t stream) {
    FeedForwardWeights a = args;
    const dim3 grid(static_cast<unsigned>(a.tiles * a.splits));
    a.row_mask != nullptr ? launch_weights<T, true>(a, a.mb, grid, stream)
                          : launch_weights<T, false>(a, a.mb, grid, stream);
    return hipGetLastError();
}

}  // namespace

void plan_product(int64_t rows, int64_t columns, int64_t stages, FeedForwardProduct* a) {
    const Edges e = choose_edges(rows, columns);
    a->mb = e.mb;
    a->nb = e.nb;
    a->stages = static_cast<int>(stages);
    const int64_t tiles = tiles_of(rows, columns, 64 * e.mb, 64 * e.nb);
    // A long K over few tiles: split so that the CUs fill, at least 8 stages each.
    int64_t splits = tiles > 0 ? kSlots / tiles : 1;
    splits = splits < stages / 8 ? splits : stages / 8;
    splits = splits < 1 ? 1 : splits;
    a->split_stages = static_cast<int>((stages + splits - 1) / splits);
    a->splits = static_cast<int>((stages + a->split_stages - 1) / a->split_stages);
    a->partial_pitch = (columns + 7) / 8 * 8;
}

void plan_weights(FeedForwardWeights* a) {
    a->mb = 2;
    const auto count = [&](int64_t bp, int64_t bq) {
        int64_t tiles = 0;
        for (int i = 0; i < a->count; ++i) {
            tiles += tiles_of(a->products[i].out_rows, a->products[i].partial_pitch, bp, bq);
        }
        return tiles;
    };
    // The large tile where its workgroups still have 512 rows each.
    if (count(256, 128) * a->rows >= 512 * kSlots * 1) {
        a->mb = 4;
    }
    const int64_t bp = 64 * a->mb;
    a->tiles = count(bp, 128);
    a->partial_floats = 0;
    for (int i = 0; i < a->count; ++i) {
        WeightProduct& w = a->products[i];
        w.q_tiles = (w.partial_pitch + 127) / 128;
        w.tiles = w.q_tiles * ((w.out_rows + bp - 1) / bp);
        w.partial_offset = a->partial_floats;
        a->partial_floats += w.out_rows * w.partial_pitch;
    }
    int64_t splits = a->tiles > 0 ? kSlots / a->tiles : 1;
    const int64_t most = (a->rows + 127) / 128;
    splits = splits < most ? splits : most;
    const int64_t least = (a->rows + kWeightSplitRows - 1) / kWeightSplitRows;
    splits = splits > least ? splits : least;
    splits = splits < 1 ? 1 : splits;
    const int64_t per = (a->rows + splits - 1) / splits;
    a->split_rows = (per + kStageK - 1) / kStageK * kStageK;
    a->splits = a->rows > 0 ? (a->rows + a->split_rows - 1) / a->split_rows : 1;
}

hipError_t launch_feed_forward_gate(const FeedForwardArgs& a, hipStream_t stream) {
    return a.type == LSSO_HIP_BF16 ? launch_gate<LSSO_HIP_BF16>(a, stream) : launch_gate<LSSO_HIP_F16>(a, stream);
}
hipError_t launch_feed_forward_product(const FeedForwardProduct& a, bool q_rows, hipStream_t stream) {
    if (a.type == LSSO_HIP_BF16) {
        return q_rows ? launch_product<LSSO_HIP_BF16, true>(a, stream) : launch_product<LSSO_HIP_BF16, false>(a, stream);
    }
    return q_rows ? launch_product<LSSO_HIP_F16, true>(a, stream) : launch_product<LSSO_HIP_F16, false>(a, stream);
}
hipError_t launch_feed_forward_grad(const FeedForwardArgs& a, hipStream_t stream) {
    return a.type == LSSO_HIP_BF16 ? launch_grad<LSSO_HIP_BF16>(a, stream) : launch_grad<LSSO_HIP_F16>(a, stream);
}
hipError_t launch_feed_forward_weights(const FeedForwardWeights& a, hipStream_t stream) {
    return a.type == LSSO_HIP_BF16 ? launch_weights<LSSO_HIP_BF16>(a, stream) : launch_weights<LSSO_HIP_F16>(a, stream);
}
hipError_t launch_feed_forward_join(const FeedForwardJoin& a, int outputs, hipStream_t stream) {
    int64_t most = 0;
    for (int i = 0; i < outputs; ++i) {
        const int64_t items = a.outputs[i].rows * ((a.outputs[i].columns + 3) / 4);
        most = items > most ? items : most;
    }
    join_kernel<<<dim3(static_cast<unsigned>((most + 255) / 256), static_cast<unsigned>(outputs)), 256, 0, stream>>>(a);
    return hipGetLastError();
}
hipError_t launch_feed_forward_pack(const FeedForwardPack& a, int type, hipStream_t stream) {
    int64_t pieces = 0;
    for (int i = 0; i < a.count; ++i) {
        pieces += a.matrices[i].pieces;
    }
    if (pieces == 0) {
        return hipSuccess;
    }
    const dim3 grid(static_cast<unsigned>((pieces + 255) / 256));
    if (type == LSSO_HIP_BF16) {
        pack_kernel<LSSO_HIP_BF16><<<grid, 256, 0, stream>>>(a);
    } else {
        pack_kernel<LSSO_HIP_F16><<<grid, 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
