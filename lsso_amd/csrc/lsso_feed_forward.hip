// Gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its
// gradients.  All products are the tiled loop of lsso_product.h:
//
//   gate_kernel    g, u = x Wg^T, x Wu^T in one pass over x; h = act(g) u from
//                  the FP32 accumulators.  Training also keeps the two factors
//                  of the backward, u act'(g) and act(g): rounded once, where
//                  kept g and u would be rounded before them (gradients off by
//                  sqrt(3) instead of 1.85 output roundings), and the backward
//                  evaluates no activation.
//   product_kernel y = h Wd^T, and in the backward dx = dg Wg + du Wu
//   grad_kernel    dh = dy Wd, and from it dg = dh (u act'(g)), du = dh act(g)
//   weight_kernel  dWg = dg^T x, dWu = du^T x, dWd = dy^T h in one launch,
//                  over row ranges whose FP32 partials join_kernel adds in order
//
// Operands are 16-bit values of x's type: x, the weights (FP32 weights are
// rounded once per call, as the projections round theirs) and h, dg and du,
// which are rounded once when they are stored, because the products that take
// them run on 16-bit matrix instructions.  The kept factors lie as [rows, 2, Fp],
// as do dg and du, and h as [rows, Fp], Fp the hidden width rounded up to 8 with zeros behind it, so
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

// act(g), and with SLOPE act'(g), FP32.  SiLU: g / (1 + exp(-g)); an exponential
// that overflows leaves a sigmoid of 0.  GELU: g Phi(g), with Phi's tail
// Phi(-|g|) = t (a1 + t (a2 + ...)) exp(-g^2 / 2) / 2, t = 1 / (1 + p |g| /
// sqrt(2)), from Abramowitz and Stegun 7.1.26 (off by at most 7.5e-8 of Phi);
// the exponential is also that of the derivative's normal density.  The error
// function of the device library in its place took about twice the epilogue's
// vector instructions.
template <bool SLOPE>
__device__ __forceinline__ void activation(int kind, float g, float& value, float& slope) {
    if (kind == LSSO_HIP_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
        value = g * s;
        slope = SLOPE ? s * (1.0f + g * (1.0f - s)) : 0.0f;
    } else {
        const float x = fabsf(g);
        const float t = __builtin_amdgcn_rcpf(1.0f + (0.3275911f * 0.70710678f) * x);
        const float e = __expf(-0.5f * g * g);
        const float poly =
            t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
        const float tail = 0.5f * poly * e;
        const float cdf = g < 0.0f ? tail : 1.0f - tail;
        value = g * cdf;
        slope = SLOPE ? cdf + 0.39894228f * g * e : 0.0f;
    }
}

// Q's loads in rows: lines are the tile's columns.
template <typename Stage>
struct QRowLoads {
    uint32_t offset;       // this lane's line and element, bytes
    uint32_t step;         // bytes between the lines of consecutive loads
    int element;           // this lane's element of stage 0
    int elements;

    __device__ __forceinline__ QRowLoads(int64_t stride, int64_t k_elements, int wave, int lane)
        : step(static_cast<uint32_t>(2 * 32 * stride)),
          elements(static_cast<int>(k_elements)) {
        element = Stage::load_element(wave, lane);
        offset = static_cast<uint32_t>(2 * (Stage::load_row(wave, lane, 0) * stride + element));
    }
    __device__ __forceinline__ static BufferRsrc lines(const uint16_t* base, int64_t stride, int64_t rows, int most) {
        return make_buffer(base, 2 * (rows < most ? rows : most) * stride);
    }
    __device__ __forceinline__ void issue(BufferRsrc buffer, char* lds, int wave, int k, int j, int line_step) const {
        load_to_lds(buffer, lds + 1024 * (4 * j + wave),
                    k + element < elements ? offset + line_step * step + static_cast<uint32_t>(2 * k) : kOutOfRange);
    }
};

// P's fragments: MB blocks of 16 rows, 8 k per lane.
template <int MB>
struct PRowLoads {
    uint32_t offset;
    uint32_t step;         // bytes between blocks
    int element;
    int elements;

    __device__ __forceinline__ PRowLoads(int64_t stride, int64_t k_elements, int wave, int lane)
        : offset(static_cast<uint32_t>(2 * ((16 * MB * wave + (lane & 15)) * stride + 8 * (lane >> 4)))),
          step(static_cast<uint32_t>(2 * 16 * stride)),
          element(8 * (lane >> 4)),
          elements(static_cast<int>(k_elements)) {}
    __device__ __forceinline__ static BufferRsrc lines(const uint16_t* base, int64_t stride, int64_t rows) {
        return make_buffer(base, 2 * (rows < 64 * MB ? rows : 64 * MB) * stride);
    }
    __device__ __forceinline__ void load(BufferRsrc buffer, int k, u32x4 (&fragments)[MB]) const {
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            fragments[m] = buffer_load16(
                buffer, k + element < elements ? offset + m * step + static_cast<uint32_t>(2 * k) : kOutOfRange);
        }
    }
};

// Both operands' loads of consecutive tiles, stages [first, last) of each: P
// [rows, k] and Q [columns, k].
template <typename S>
struct RowStream {
    using Q = typename S::QStage;
    const uint16_t* p_base;
    int64_t p_stride;
    int64_t rows;
    const uint16_t* q_base;
    int64_t q_stride;
    int64_t columns;
    int first;
    int last;
    int wave;
    PRowLoads<S::MB> p;
    QRowLoads<Q> q;
    TileWalk p_walk;
    TileWalk q_walk;
    int slot;
    int stage;
    BufferRsrc p_rows;
    BufferRsrc q_rows;

    __device__ __forceinline__ RowStream(const uint16_t* p_base_, int64_t p_stride_, int64_t rows_,
                                         const uint16_t* q_base_, int64_t q_stride_, int64_t columns_, int64_t k,
                                         int first_, int last_, const TileWalk& walk, int wave_, int lane)
        : p_base(p_base_), p_stride(p_stride_), rows(rows_), q_base(q_base_), q_stride(q_stride_), columns(columns_),
          first(first_), last(last_), wave(wave_), p(p_stride_, k, wave_, lane), q(q_stride_, k, wave_, lane),
          p_walk(walk), q_walk(walk), slot(2 * first_), stage(first_) {
        aim_p();
        aim_q();
    }
    __device__ __forceinline__ void aim_p() {
        const int64_t p0 = static_cast<int64_t>(p_walk.p) * S::BP;
        p_rows = PRowLoads<S::MB>::lines(p_base + p0 * p_stride, p_stride, p_walk.left > 0 ? rows - p0 : 0);
    }
    __device__ __forceinline__ void aim_q() {
        const int64_t q0 = static_cast<int64_t>(q_walk.q) * S::BQ;
        q_rows = QRowLoads<Q>::lines(q_base + q0 * q_stride, q_stride, q_walk.left > 0 ? columns - q0 : 0, S::BQ);
    }
    __device__ __forceinline__ void load_p(u32x4 (&fragments)[S::MB]) {
        p.load(p_rows, slot * kSlotK, fragments);
        if (++slot == 2 * last) {
            slot = 2 * first;
            p_walk.next();
            aim_p();
        }
    }
    __device__ __forceinline__ void issue_q(char* lds) {
#pragma unroll
        for (int j = 0; j < Q::kLoads; ++j) {
            q.issue(q_rows, lds, wave, stage * kRowsStageK, j, j);
        }
        if (++stage == last) {
            stage = first;
            q_walk.next();
            aim_q();
        }
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

// FP32 rows of a wave's blocks into partials [rows, pitch] from row p0 and
// column q0 on.  Blocks: 32 x 32 (lane & 31 the row, entry 4 q + e column 8 q + 4
// half + e).
template <typename S>
__device__ __forceinline__ void store_partials(char* mine, int lane, const f32x16 (&acc)[S::NB][S::MB],
                                               float* partials, int64_t pitch, int64_t p0, int64_t rows, int64_t q0) {
    using Exchange = RowExchange<32, 128>;
    static_assert(Exchange::kSize <= S::kWaveBytes, "the exchange fits the wave's LDS");
#pragma unroll
    for (int m = 0; m < S::MB; ++m) {
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = {acc[n][m][4 * q], acc[n][m][4 * q + 1], acc[n][m][4 * q + 2], acc[n][m][4 * q + 3]};
                Exchange::put(mine, lane, 32 * q + 16 * (lane >> 5), v);
            }
            wave_lds_order();
            const int64_t column = q0 + 32 * n + Exchange::byte(lane) / 4;
#pragma unroll
            for (int i = 0; i < Exchange::kSteps; ++i) {
                const u32x4 value = Exchange::get(mine, lane, i);
                const int64_t row = p0 + 32 * m + Exchange::row(lane, i);
                if (row < rows && column < pitch) {
                    *reinterpret_cast<u32x4*>(partials + row * pitch + column) = value;
                }
            }
            wave_lds_order();
        }
    }
}

// ------------------------------------------------------- h and its two factors
// Q is [gate rows | up rows] of the tile's 64 columns of h, so a lane holds both
// factors of its products: block n < 4 the gate's, n + 4 the up's.
template <int T, int MB, bool KEEP>
__device__ __forceinline__ void gate_epilogue(const FeedForwardArgs& a, char* mine, int lane, int64_t p0, int64_t q0,
                                              const f32x4 (&acc)[8][MB]) {
    // 16 rows at a time: 16-bit rows of 64 columns through the exchange, h, then
    // the factors.
    using Exchange = RowExchange<16, 128>;
    constexpr int kOutputs = KEEP ? 3 : 1;
    const int64_t column = q0 + Exchange::byte(lane) / 2;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row0 = p0 + 16 * m;
        const int64_t row = row0 + (lane & 15);
        const bool kept = row < a.rows && (a.row_mask == nullptr || a.row_mask[row] != 0);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            float h[4];
            float first[4];
            float second[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float act, slope;
                activation<KEEP>(a.activation, acc[n][m][e], act, slope);
                const float u = acc[n + 4][m][e];
                h[e] = kept ? act * u : 0.0f;
                first[e] = slope * u;
                second[e] = act;
            }
            const int byte = 32 * n + 8 * (lane >> 4);
            Exchange::put(mine, lane, byte, (u32x2){Values<T>::pack(h[0], h[1]), Values<T>::pack(h[2], h[3])});
            if (KEEP) {
                Exchange::put(mine + Exchange::kSize, lane, byte,
                              (u32x2){Values<T>::pack(first[0], first[1]), Values<T>::pack(first[2], first[3])});
                Exchange::put(mine + 2 * Exchange::kSize, lane, byte,
                              (u32x2){Values<T>::pack(second[0], second[1]), Values<T>::pack(second[2], second[3])});
            }
        }
        wave_lds_order();
#pragma unroll
        for (int o = 0; o < kOutputs; ++o) {
            uint16_t* const out = o == 0 ? a.h : a.gates + (o - 1) * a.pitch;
            const int64_t pitch = o == 0 ? a.pitch : 2 * a.pitch;
#pragma unroll
            for (int i = 0; i < Exchange::kSteps; ++i) {
                const u32x4 value = Exchange::get(mine + o * Exchange::kSize, lane, i);
                const int64_t to = row0 + Exchange::row(lane, i);
                if (to < a.rows && column < a.pitch) {
                    store16_unaligned(out + to * pitch + column, value);
                }
            }
        }
        wave_lds_order();
    }
}

template <int T, int MB, bool KEEP>
using GateShape = RowsShape<T, MB, 8, (KEEP ? 3 : 1) * RowExchange<16, 128>::kSize>;

template <int T, int MB, bool KEEP>
__global__ __launch_bounds__(kProductThreads, 2) void gate_kernel(FeedForwardArgs a) {
    using S = GateShape<T, MB, KEEP>;
    using Q = typename S::QStage;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    constexpr int kColumns = 64;
    TileWalk walk(a.tiles, a.q_tiles);
    if (walk.left == 0) {
        return;
    }
    const PRowLoads<MB> p(a.x_stride, a.in_pitch, wave, lane);
    const QRowLoads<Q> q(a.in_pitch, a.in_pitch, wave, lane);
    static_assert(Q::kLoads == 4, "two loads of each weight");
    TileWalk p_walk = walk;
    int p_slot = 0;
    const auto x_rows = [&] {
        const int64_t p0 = static_cast<int64_t>(p_walk.p) * S::BP;
        return PRowLoads<MB>::lines(a.x + p0 * a.x_stride, a.x_stride, p_walk.left > 0 ? a.rows - p0 : 0);
    };
    BufferRsrc x = x_rows();
    TileWalk q_walk = walk;
    int q_stage = 0;
    const auto weight_rows = [&](const uint16_t* weight) {
        const int64_t q0 = static_cast<int64_t>(q_walk.q) * kColumns;
        return QRowLoads<Q>::lines(weight + q0 * a.in_pitch, a.in_pitch, q_walk.left > 0 ? a.hidden - q0 : 0, kColumns);
    };
    BufferRsrc gate = weight_rows(a.gate);
    BufferRsrc up = weight_rows(a.up);
    const auto load_p = [&](u32x4 (&fragments)[MB]) {
        p.load(x, p_slot * kSlotK, fragments);
        if (++p_slot == 2 * a.stages) {
            p_slot = 0;
            p_walk.next();
            x = x_rows();
        }
    };
    const auto issue_q = [&](char* stage) {
        // Loads 0 and 1 of Q are rows 0 .. 63 of its stage, 2 and 3 the rest.
        const int k = q_stage * kRowsStageK;
        q.issue(gate, stage, wave, k, 0, 0);
        q.issue(gate, stage, wave, k, 1, 1);
        q.issue(up, stage, wave, k, 2, 0);
        q.issue(up, stage, wave, k, 3, 1);
        if (++q_stage == a.stages) {
            q_stage = 0;
            q_walk.next();
            gate = weight_rows(a.gate);
            up = weight_rows(a.up);
        }
    };
    run_rows_tiles<S>(lds, walk.left, a.stages, load_p, issue_q, [&](const f32x4 (&acc)[8][MB]) {
        gate_epilogue<T, MB, KEEP>(a, lds + S::kRingBytes + S::kWaveBytes * wave, lane,
                                   static_cast<int64_t>(walk.p) * S::BP + 16 * MB * wave,
                                   static_cast<int64_t>(walk.q) * kColumns, acc);
        walk.next();
    });
}

// ------------------------------------------------------------------ y and dx
// out = P Q^T: y = h Wd^T, or dx = [dg | du] [Wg^T | Wu^T]^T with both weights
// transposed side by side, as dg and du lie.  With `splits` > 1 the stages are
// divided and FP32 partials left for join_kernel.
template <int T, int MB, int NB>
using ProductRows = RowsShape<T, MB, NB, RowExchange<16, 32 * NB>::kSize>;

template <int T, int MB, int NB>
__device__ __forceinline__ void product_epilogue(const FeedForwardProduct& a, char* mine, int lane, int split,
                                                 int64_t p0, int64_t q0, const f32x4 (&acc)[NB][MB]) {
    if (a.partials != nullptr) {   // uniform
        using Exchange = RowExchange<16, 32 * NB>;   // half the columns at a time
        float* const out = a.partials + split * a.rows * a.partial_pitch;
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int64_t row0 = p0 + 16 * m;
#pragma unroll
            for (int n0 = 0; n0 < NB; n0 += NB / 2) {
#pragma unroll
                for (int n = 0; n < NB / 2; ++n) {
                    Exchange::put(mine, lane, 64 * n + 16 * (lane >> 4), acc[n0 + n][m]);
                }
                wave_lds_order();
                const int64_t column = q0 + 16 * n0 + Exchange::byte(lane) / 4;
#pragma unroll
                for (int i = 0; i < Exchange::kSteps; ++i) {
                    const u32x4 value = Exchange::get(mine, lane, i);
                    const int64_t to = row0 + Exchange::row(lane, i);
                    if (to < a.rows && column < a.partial_pitch) {
                        *reinterpret_cast<u32x4*>(out + to * a.partial_pitch + column) = value;
                    }
                }
                wave_lds_order();
            }
        }
        return;
    }
    using Exchange = RowExchange<16, 32 * NB>;
    const int64_t column = q0 + Exchange::byte(lane) / 2;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row0 = p0 + 16 * m;
        const int64_t row = row0 + (lane & 15);
        const bool kept = row < a.rows && (a.row_mask == nullptr || a.row_mask[row] != 0);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            f32x4 v = acc[n][m];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = kept ? v[e] : 0.0f;
            }
            Exchange::put(mine, lane, 32 * n + 8 * (lane >> 4),
                          (u32x2){Values<T>::pack(v[0], v[1]), Values<T>::pack(v[2], v[3])});
        }
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < Exchange::kSteps; ++i) {
            const u32x4 value = Exchange::get(mine, lane, i);
            const int64_t to = row0 + Exchange::row(lane, i);
            uint16_t* at = a.out + to * a.columns + column;
            if (to < a.rows && column + 8 <= a.columns) {
                store16_unaligned(at, value);
            } else if (to < a.rows) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (column + e < a.columns) {
                        at[e] = static_cast<uint16_t>(value[e / 2] >> (16 * (e & 1)));
                    }
                }
            }
        }
        wave_lds_order();
    }
}

template <int T, int MB, int NB>
__global__ __launch_bounds__(kProductThreads, 2) void product_kernel(FeedForwardProduct a) {
    using S = ProductRows<T, MB, NB>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    TileWalk walk(a.tiles, a.q_tiles);
    if (walk.left == 0) {
        return;
    }
    const int split = blockIdx.y;
    const int first = split * a.split_stages;
    const int last = first + a.split_stages < a.stages ? first + a.split_stages : a.stages;
    RowStream<S> stream(a.p, a.p_stride, a.rows, a.q, a.q_stride, a.columns, a.k, first, last, walk, wave, lane);
    run_rows_tiles<S>(
        lds, walk.left, last - first, [&](u32x4 (&fragments)[MB]) { stream.load_p(fragments); },
        [&](char* stage) { stream.issue_q(stage); },
        [&](const f32x4 (&acc)[NB][MB]) {
            product_epilogue<T, MB, NB>(a, lds + S::kRingBytes + S::kWaveBytes * wave, lane, split,
                                        static_cast<int64_t>(walk.p) * S::BP + 16 * MB * wave,
                                        static_cast<int64_t>(walk.q) * S::BQ, acc);
            walk.next();
        });
}

// ----------------------------------------------------------------- dg and du
template <int T, int MB, int NB>
using GradShape = RowsShape<T, MB, NB, RowExchange<16, 256>::kSize>;

template <int T, int MB, int NB>
__device__ __forceinline__ void grad_epilogue(const FeedForwardArgs& a, char* mine, int lane, int64_t p0, int64_t q0,
                                              const f32x4 (&acc)[NB][MB]) {
    // dh goes through the exchange in FP32, 16 rows x 64 columns at a time: in
    // its rows the factors are read and dg, du written whole pieces at a time.
    using Exchange = RowExchange<16, 256>;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row0 = p0 + 16 * m;
#pragma unroll
        for (int n0 = 0; n0 < NB; n0 += 4) {
            const int64_t column = q0 + 16 * n0 + 8 * (lane & 7);
            u32x4 raw[2][2];
            bool kept[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t row = row0 + 8 * i + (lane >> 3);
                if (row < a.rows && column < a.pitch) {
                    const uint16_t* at = a.gates + 2 * row * a.pitch + column;
                    raw[i][0] = load16_unaligned(at);
                    raw[i][1] = load16_unaligned(at + a.pitch);
                    kept[i] = a.row_mask == nullptr || a.row_mask[row] != 0;
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                Exchange::put(mine, lane, 64 * n + 16 * (lane >> 4), acc[n0 + n][m]);
            }
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * i + (lane >> 3);
                const int64_t row = row0 + r;
                const char* from = mine + r * Exchange::kPitch + 32 * (lane & 7);
                const f32x4 low = *reinterpret_cast<const f32x4*>(from);
                const f32x4 high = *reinterpret_cast<const f32x4*>(from + 16);
                if (row < a.rows && column < a.pitch) {
                    float dg[8];
                    float du[8];
                    Values<T>::unpack8(raw[i][0], dg);
                    Values<T>::unpack8(raw[i][1], du);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float dh = e < 4 ? low[e & 3] : high[e & 3];
                        dg[e] = kept[i] ? dh * dg[e] : 0.0f;
                        du[e] = kept[i] ? dh * du[e] : 0.0f;
                    }
                    uint16_t* at = a.grads + 2 * row * a.pitch + column;
                    store16_unaligned(at, Values<T>::pack8(dg));
                    store16_unaligned(at + a.pitch, Values<T>::pack8(du));
                }
            }
            wave_lds_order();
        }
    }
}

template <int T, int MB, int NB>
__global__ __launch_bounds__(kProductThreads, 2) void grad_kernel(FeedForwardArgs a) {
    using S = GradShape<T, MB, NB>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    TileWalk walk(a.tiles, a.q_tiles);
    if (walk.left == 0) {
        return;
    }
    RowStream<S> stream(a.dy, a.dy_stride, a.rows, a.down_columns, a.out_pitch, a.hidden, a.out_pitch, 0, a.stages, walk,
                        wave, lane);
    run_rows_tiles<S>(
        lds, walk.left, a.stages, [&](u32x4 (&fragments)[MB]) { stream.load_p(fragments); },
        [&](char* stage) { stream.issue_q(stage); },
        [&](const f32x4 (&acc)[NB][MB]) {
            grad_epilogue<T, MB, NB>(a, lds + S::kRingBytes + S::kWaveBytes * wave, lane,
                                     static_cast<int64_t>(walk.p) * S::BP + 16 * MB * wave,
                                     static_cast<int64_t>(walk.q) * S::BQ, acc);
            walk.next();
        });
}

// ----------------------------------------------------------- weight gradients
// One of up to three products P^T Q over a range of rows, P and Q in columns.
template <int T, int MB, int NB, int WP, bool MASKED>
__global__ __launch_bounds__(kProductThreads, 2) void weight_kernel(FeedForwardWeights a) {
    using S = ProductShape<T, false, false, MB, NB, WP>;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    __shared__ uint32_t kept[MASKED ? kWeightSplitRows / 32 + kRing : 1];   // rows of each stage
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
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
    const auto q_start = [&](int n) { return S::wave_q(wave) + 32 * n; };
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

    store_partials<S>(lds + S::kWaveBytes * wave, lane, acc,
                      a.partials + split * a.partial_floats + w.partial_offset, w.partial_pitch,
                      p0 + S::wave_p(wave), w.out_rows, q0 + q_start(0));
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
// behind the last one (FP32 weights, operands with odd rows), or of their
// transposes.  A workgroup takes 64 x 64 of a matrix, a thread 2 pieces of 8.
constexpr int kPackEdge = 64;

template <int T>
__global__ __launch_bounds__(256) void pack_kernel(FeedForwardPack a) {
    __shared__ uint16_t square[kPackEdge][kPackEdge + 8];
    int block = static_cast<int>(blockIdx.x);
    int which = 0;
    while (block >= a.matrices[which].tiles) {   // the grid is the sum of all tiles
        block -= a.matrices[which].tiles;
        ++which;
    }
    const PackMatrix& m = a.matrices[which];
    const int across = static_cast<int>((m.columns + kPackEdge - 1) / kPackEdge);
    const int64_t r0 = static_cast<int64_t>(block / across) * kPackEdge;
    const int64_t c0 = static_cast<int64_t>(block % across) * kPackEdge;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 32 * i + static_cast<int>(threadIdx.x >> 3);
        const int c = 8 * static_cast<int>(threadIdx.x & 7);
        float v[8] = {};
        const auto get = [&](auto values) {
            using V = decltype(values);
            const auto* from = static_cast<const typename V::Element*>(m.from) + (r0 + r) * m.stride + c0 + c;
            if (r0 + r < m.rows && c0 + c + 8 <= m.columns) {
                V::load8(from, v);
            } else if (r0 + r < m.rows) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = c0 + c + e < m.columns ? V::load(from + e) : 0.0f;
                }
            }
        };
        if (m.wide) {
            get(Values<LSSO_HIP_F32>());
        } else {
            get(Values<T>());
        }
        const u32x4 packed = Values<T>::pack8(v);
        if (!m.transposed) {
            if (r0 + r < m.rows && c0 + c < m.pitch) {
                store16_unaligned(m.to + (r0 + r) * m.pitch + c0 + c, packed);
            }
        } else {
            *reinterpret_cast<u32x4*>(&square[r][c]) = packed;
        }
    }
    if (!m.transposed) {   // the same for the whole workgroup
        return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = 32 * i + static_cast<int>(threadIdx.x >> 3);   // a row of the transpose
        const int r = 8 * static_cast<int>(threadIdx.x & 7);
        if (c0 + c < m.columns && r0 + r < m.rows) {
            u32x4 out;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                out[e] = static_cast<uint32_t>(square[r + 2 * e][c]) | static_cast<uint32_t>(square[r + 2 * e + 1][c]) << 16;
            }
            store16_unaligned(m.to + (c0 + c) * m.pitch + r0 + r, out);
        }
    }
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

// A multiple of eight workgroups (one share per XCD), at most what is resident.
dim3 tile_grid(int tiles, int slots, int splits = 1) {
    const int per_xcd = (tiles + 7) / 8;
    return dim3(static_cast<unsigned>(8 * (per_xcd < slots ? per_xcd : slots)), static_cast<unsigned>(splits));
}

template <int T, int MB, bool KEEP>
hipError_t launch_gate(FeedForwardArgs a, hipStream_t stream) {
    using S = GateShape<T, MB, KEEP>;
    a.stages = static_cast<int>((a.in_pitch + kRowsStageK - 1) / kRowsStageK);
    a.q_tiles = static_cast<int>((a.pitch + 63) / 64);
    a.tiles = a.q_tiles * static_cast<int>((a.rows + S::BP - 1) / S::BP);
    gate_kernel<T, MB, KEEP><<<tile_grid(a.tiles, S::kSlots), kProductThreads, 0, stream>>>(a);
    return hipGetLastError();
}

template <int T, bool KEEP>
hipError_t launch_gate(const FeedForwardArgs& a, hipStream_t stream) {
    switch (choose_gate(a.rows, a.pitch)) {
        case 4: return launch_gate<T, 4, KEEP>(a, stream);
        case 2: return launch_gate<T, 2, KEEP>(a, stream);
        default: return launch_gate<T, 1, KEEP>(a, stream);
    }
}

template <int T>
hipError_t launch_gate(const FeedForwardArgs& a, hipStream_t stream) {
    return a.gates != nullptr ? launch_gate<T, true>(a, stream) : launch_gate<T, false>(a, stream);
}

template <int T, int MB, int NB>
hipError_t launch_product(FeedForwardProduct a, hipStream_t stream) {
    using S = ProductRows<T, MB, NB>;
    a.q_tiles = static_cast<int>((a.columns + S::BQ - 1) / S::BQ);
    a.tiles = a.q_tiles * static_cast<int>((a.rows + S::BP - 1) / S::BP);
    product_kernel<T, MB, NB><<<tile_grid(a.tiles, S::kSlots, a.splits), kProductThreads, 0, stream>>>(a);
    return hipGetLastError();
}

template <int T>
hipError_t launch_product(const FeedForwardProduct& args, hipStream_t stream) {
    FeedForwardProduct a = args;
    if (a.splits == 1) {
        a.partials = nullptr;
    }
    const hipError_t error = a.mb == 4   ? launch_product<T, 4, 8>(a, stream)
                             : a.mb == 2 ? launch_product<T, 2, 8>(a, stream)
                                         : launch_product<T, 1, 4>(a, stream);
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

template <int T, int MB, int NB>
hipError_t launch_grad(FeedForwardArgs a, hipStream_t stream) {
    using S = GradShape<T, MB, NB>;
    a.stages = static_cast<int>((a.out_pitch + kRowsStageK - 1) / kRowsStageK);
    a.q_tiles = static_cast<int>((a.pitch + S::BQ - 1) / S::BQ);
    a.tiles = a.q_tiles * static_cast<int>((a.rows + S::BP - 1) / S::BP);
    grad_kernel<T, MB, NB><<<tile_grid(a.tiles, S::kSlots), kProductThreads, 0, stream>>>(a);
    return hipGetLastError();
}

template <int T>
hipError_t launch_grad(const FeedForwardArgs& a, hipStream_t stream) {
    switch (choose_edges(a.rows, a.pitch).mb) {
        case 4: return launch_grad<T, 4, 8>(a, stream);
        case 2: return launch_grad<T, 2, 8>(a, stream);
        default: return launch_grad<T, 1, 4>(a, stream);
    }
}

template <int T, bool MASKED>
void launch_weights(const FeedForwardWeights& a, int mb, dim3 grid, hipStream_t stream) {
    if (mb == 4) {
        weight_kernel<T, 2, 4, 4, MASKED><<<grid, kProductThreads, 0, stream>>>(a);
    } else {
        weight_kernel<T, 2, 2, 2, MASKED><<<grid, kProductThreads, 0, stream>>>(a);
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
    // A long K over few tiles: split so that the CUs fill, at least 4 stages each.
    int64_t splits = tiles > 0 ? kSlots / tiles : 1;
    splits = splits < stages / 4 ? splits : stages / 4;
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
hipError_t launch_feed_forward_product(const FeedForwardProduct& a, hipStream_t stream) {
    return a.type == LSSO_HIP_BF16 ? launch_product<LSSO_HIP_BF16>(a, stream) : launch_product<LSSO_HIP_F16>(a, stream);
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
hipError_t launch_feed_forward_pack(const FeedForwardPack& args, int type, hipStream_t stream) {
    FeedForwardPack a = args;
    int64_t tiles = 0;
    for (int i = 0; i < a.count; ++i) {
        PackMatrix& m = a.matrices[i];
        const int64_t n = ((m.rows + kPackEdge - 1) / kPackEdge) * ((m.columns + kPackEdge - 1) / kPackEdge);
        tiles += n;
        m.tiles = static_cast<int>(n);
    }
    if (tiles == 0) {
        return hipSuccess;
    }
    const dim3 grid(static_cast<unsigned>(tiles));
    if (type == LSSO_HIP_BF16) {
        pack_kernel<LSSO_HIP_BF16><<<grid, 256, 0, stream>>>(a);
    } else {
        pack_kernel<LSSO_HIP_F16><<<grid, 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
