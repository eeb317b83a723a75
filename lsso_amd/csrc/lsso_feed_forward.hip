// Gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wd^T, and its
// gradients.  All products are the tiled loop of lsso_product.h:
//
//   gate_kernel    g, u = x Wg^T, x Wu^T in one pass over x; h = act(g) u from
//                  the FP32 accumulators.  Training also keeps the two factors
//                  of the backward, u act'(g) and act(g), fine or rounded to
//                  16 bits, so that the backward evaluates no activation.  From
//                  fine ones gradients are off by sqrt(2) output roundings (dg
//                  or du, and the output), from 16-bit ones by sqrt(3), and
//                  from kept 16-bit g and u they would be by 1.85.
//   product_kernel y = h Wd^T, and in the backward dx = dg Wg + du Wu
//   grad_kernel    dh = dy Wd, and from it dg = dh (u act'(g)), du = dh act(g)
//   weight_kernel  dWg = dg^T x, dWu = du^T x, dWd = dy^T h in one launch,
//                  over row ranges whose FP32 partials join_kernel adds in order
//
// Operands are 16-bit values of x's type: x, the weights (FP32 weights are
// rounded once per call, as the projections round theirs) and h, dg and du,
// which are rounded once when they are stored, because the products that take
// them run on 16-bit matrix instructions.  The kept factors lie as [rows, 2, Fp],
// as do dg and du, and h as [rows, Fp], Fp the hidden width rounded up to 8 with
// zeros behind it, so every row is whole 16-byte pieces.  Fine factors are the
// upper bits of the FP32 value, so with its range: 20 beside BF16, 24 beside FP16, whose
// roundings are then at most a sixteenth of the type's.  Their first 16 bits lie where
// 16-bit factors do, the rest behind all of them: per column a byte of four bits of
// either, or by 8 columns 8 bytes of either.  131,072 x 256 -> 688: gate kernel 234 us
// instead of 199, gradient kernel 265 instead of 226; 8,192 x 768 -> 2,048: 71 instead of
// 64, 64 instead of 57.  Operands whose own rows are not (odd
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

// Fine factors: FP32 values rounded to their upper bits (round), of which the first 16 of
// two are `upper`, and the rest of four columns' first and second factors `lower`.
template <int T>
struct Fine {
    static constexpr int kLowerBytes = T == LSSO_HIP_BF16 ? 1 : 2;   // per column, of both factors
    __device__ static __forceinline__ float round(float v) {
        return __uint_as_float(__float_as_uint(v) + (T == LSSO_HIP_BF16 ? 0x800u : 0x80u));
    }
    __device__ static __forceinline__ uint32_t upper(float a, float b) {
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    // The third bytes of four values.
    __device__ static __forceinline__ uint32_t third(const float (&v)[4]) {
        return __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0c0c0501u) |
               __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x05010c0cu);
    }
    // BF16: of both factors of four columns in one word.
    __device__ static __forceinline__ uint32_t lower(const float (&first)[4], const float (&second)[4]) {
        return (third(first) >> 4 & 0x0f0f0f0fu) | (third(second) & 0xf0f0f0f0u);
    }
    // Eight columns of one factor from their upper and third bytes.
    __device__ static __forceinline__ void join(const u32x4& upper, uint32_t third0, uint32_t third1, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t select = ((e & 1) != 0 ? 0x0706000cu : 0x0504000cu) | static_cast<uint32_t>(e & 3) << 8;
            v[e] = __uint_as_float(__builtin_amdgcn_perm(upper[e / 2], e < 4 ? third0 : third1, select));
        }
    }
    // Of eight columns: both factors from their upper bits and what `lower` points to.
    struct Lower {
        uint32_t word[T == LSSO_HIP_BF16 ? 2 : 4];
        __device__ __forceinline__ void load(const char* at) {
            if constexpr (T == LSSO_HIP_BF16) {
                const u32x2 v = *reinterpret_cast<const u32x2*>(at);
                word[0] = v[0];
                word[1] = v[1];
            } else {
                const u32x4 v = load16_unaligned(at);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    word[i] = v[i];
                }
            }
        }
        __device__ __forceinline__ void join(const u32x4& upper0, const u32x4& upper1, float (&first)[8],
                                             float (&second)[8]) const {
            if constexpr (T == LSSO_HIP_BF16) {
                Fine::join(upper0, word[0] << 4 & 0xf0f0f0f0u, word[1] << 4 & 0xf0f0f0f0u, first);
                Fine::join(upper1, word[0] & 0xf0f0f0f0u, word[1] & 0xf0f0f0f0u, second);
            } else {
                Fine::join(upper0, word[0], word[1], first);
                Fine::join(upper1, word[2], word[3], second);
            }
        }
    };
};

// What is kept for the backward.
enum class Keep { kNothing, kRounded, kFine };

// act(g), and with SLOPE act'(g), FP32.  SiLU: g / (1 + exp(-g)); an exponential
// that overflows leaves a sigmoid of 0.  GELU: g Phi(g), Phi(-|g|) = tail =
// exp(-g^2 / 2) P(|g|) / Q(|g|); the exponential is also that of the derivative's
// normal density.  P / Q is a fit to Mills' ratio over sqrt(2 pi), of degrees 3 and 4,
// from linear programs that minimize the largest weighted error over [0, 13.4]: off
// by at most 1.6e-8 of Phi and 1.3e-6 of the tail, in FP32 with the exponential's
// rounded argument by 1.5e-7 and, down to g = -13, 8e-6 of the tail.  (Abramowitz and
// Stegun 7.1.26, five terms bounded in Phi alone, leaves 3% of the tail at -12, more
// than a 16-bit rounding from -6 on; with it the gate kernel takes 467 us instead of
// 491 at 262,144 rows of 256 -> 1,024, whose tiles cost these instructions more than
// MFMAs, and with the device library's error function about 80 more.)  Behind 13.2 the
// exponential is below FP32's range and the tail 0.  Of an infinite g both activations
// are what their formulas are: inf at inf, NaN at -inf.
template <bool SLOPE>
__device__ __forceinline__ void activation(int kind, float g, float& value, float& slope) {
    constexpr float kLog2e = 1.44269504f;
    if (kind == LSSO_HIP_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
        value = g * s;
        slope = SLOPE ? s + value * (1.0f - s) : 0.0f;
    } else {
        const float x = fminf(fabsf(g), 14.0f);   // the powers stay finite
        const float p = 0.49999997f + x * (0.344746023f + x * (0.109477423f + x * 0.0146328295f));
        const float q = 1.0f + x * (1.48737419f + x * (0.905736148f + x * (0.274088085f + x * 0.0366882086f)));
        const float e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * g * g);
        const float tail = e * (p * __builtin_amdgcn_rcpf(q));
        const float phi = g < 0.0f ? tail : 1.0f - tail;
        value = g * phi;
        slope = SLOPE ? phi + 0.39894228f * g * e : 0.0f;
    }
}

// One operand's loads: rows of a tile.
template <typename Stage>
struct RowLoads {
    uint32_t offset;       // this lane's row and element, bytes
    uint32_t step;         // bytes between the rows of consecutive loads
    int element;           // this lane's element of stage 0
    int elements;

    __device__ __forceinline__ RowLoads(int64_t stride, int64_t k_elements, int wave, int lane)
        : step(static_cast<uint32_t>(2 * Stage::kRowsPerRound * stride)),
          element(Stage::load_element(wave, lane)),
          elements(static_cast<int>(k_elements)) {
        offset = static_cast<uint32_t>(2 * (Stage::load_row(wave, lane) * stride + element));
    }
    // The `rows` rows from `base` on (none where that is negative), at most `most`.
    __device__ __forceinline__ static BufferRsrc aim(const uint16_t* base, int64_t stride, int64_t rows, int most) {
        return make_buffer(base, 2 * (rows < most ? rows : most) * stride);
    }
    // Load j of a stage, of the rows of round `round` of the buffer.
    __device__ __forceinline__ void issue(BufferRsrc buffer, char* lds, int waves, int wave, int k, int j,
                                          int round) const {
        load_to_lds(buffer, lds + 1024 * (waves * j + wave),
                    k + element < elements ? offset + round * step + static_cast<uint32_t>(2 * k) : kOutOfRange);
    }
};

// Both operands' loads of consecutive tiles, stages [first, last) of each: P
// [rows, k] and Q [columns, k].
template <typename S>
struct RowStream {
    using P = typename S::PStage;
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
    RowLoads<P> p;
    RowLoads<Q> q;
    TileWalk walk;
    int stage;
    BufferRsrc p_rows;
    BufferRsrc q_rows;

    __device__ __forceinline__ RowStream(const uint16_t* p_base_, int64_t p_stride_, int64_t rows_,
                                         const uint16_t* q_base_, int64_t q_stride_, int64_t columns_, int64_t k,
                                         int first_, int last_, const TileWalk& walk_, int wave_, int lane)
        : p_base(p_base_), p_stride(p_stride_), rows(rows_), q_base(q_base_), q_stride(q_stride_), columns(columns_),
          first(first_), last(last_), wave(wave_), p(p_stride_, k, wave_, lane), q(q_stride_, k, wave_, lane),
          walk(walk_), stage(first_) {
        aim();
    }
    __device__ __forceinline__ void aim() {
        const int64_t p0 = static_cast<int64_t>(walk.p) * S::BP;
        const int64_t q0 = static_cast<int64_t>(walk.q) * S::BQ;
        p_rows = RowLoads<P>::aim(p_base + p0 * p_stride, p_stride, walk.left > 0 ? rows - p0 : 0, S::BP);
        q_rows = RowLoads<Q>::aim(q_base + q0 * q_stride, q_stride, walk.left > 0 ? columns - q0 : 0, S::BQ);
    }
    __device__ __forceinline__ void issue(char* lds, int j) {
        const int k = stage * kRowsStageK;
        if (j < P::kLoads) {
            p.issue(p_rows, lds, S::kWaves, wave, k, j, j);
        } else {
            q.issue(q_rows, lds + P::kBytes, S::kWaves, wave, k, j - P::kLoads, j - P::kLoads);
        }
        if (j == S::kLoads - 1 && ++stage == last) {
            stage = first;
            walk.next();
            aim();
        }
    }
};

// One operand's loads in columns: lines are k.
template <typename Stage>
struct ColumnLoads {
    const uint16_t* base;
    int64_t stride;
    int line;
    uint32_t offset;       // kOutOfRange for a lane past the columns
    uint32_t step;

    // Of the columns from `base_` on, of which there are `columns`.
    __device__ __forceinline__ ColumnLoads(const uint16_t* base_, int64_t stride_, int64_t columns, int wave, int lane)
        : base(base_), stride(stride_), line(Stage::load_line(wave, lane)) {
        const int element = Stage::load_element(wave, lane);
        offset = element < columns ? static_cast<uint32_t>(2 * (line * stride + element)) : kOutOfRange;
        step = static_cast<uint32_t>(2 * Stage::kLinesPerRound * stride);
    }
    // Load j of lines [k, min(k + kColumnsStageK, end)), of those whose bit in `kept` is set.
    __device__ __forceinline__ void issue(char* lds, int waves, int wave, int64_t k, int64_t end, int j,
                                          uint32_t kept) const {
        const int64_t lines = end - k < kColumnsStageK ? end - k : kColumnsStageK;
        const BufferRsrc buffer = make_buffer(base + (lines > 0 ? k : 0) * stride, 2 * lines * stride);
        const bool load = offset != kOutOfRange && (kept >> (line + j * Stage::kLinesPerRound) & 1) != 0;
        load_to_lds(buffer, lds + 1024 * (waves * j + wave), load ? offset + j * step : kOutOfRange);
    }
};

// FP32 rows of a wave's blocks of 32 x 32 into partials [rows, pitch] from row
// p0 and column q0 on.
template <int MB, int NB>
__device__ __forceinline__ void store_partials(char* mine, int lane, const f32x16 (&acc)[NB][MB], float* partials,
                                               int64_t pitch, int64_t p0, int64_t rows, int64_t q0) {
    using Exchange = RowExchange<128>;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16& c = acc[n][m];
                Exchange::put(mine, lane, 32 * q + 16 * (lane >> 5),
                              (f32x4){c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]});
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
// Q is [gate rows | up rows] of the tile's columns of h, and a wave takes the
// same columns of both, so that a lane holds both factors of its products: block
// n < NB / 2 the gate's, n + NB / 2 the up's.  A wave's 32 rows at a time go
// through the exchange as rows of its columns: h, the factors' 16 bits one after the
// other, then what more of both is kept.  The factors wait for their turn in the
// accumulators that they come from.

// A pass of the exchange to memory: rows of BYTES from byte `first` of `to`'s on,
// `pitch` bytes apart, up to byte `end`.
template <int BYTES>
__device__ __forceinline__ void store_exchange(const char* mine, int lane, char* to, int64_t pitch, int64_t row0,
                                               int64_t rows, int64_t first, int64_t end) {
    using Exchange = RowExchange<BYTES>;
    wave_lds_order();
    const int64_t piece = first + Exchange::byte(lane);
#pragma unroll
    for (int i = 0; i < Exchange::kSteps; ++i) {
        const u32x4 value = Exchange::get(mine, lane, i);
        const int64_t row = row0 + Exchange::row(lane, i);
        if (row < rows && piece < end) {
            store16_unaligned(to + row * pitch + piece, value);
        }
    }
    wave_lds_order();
}

template <int T, int MB, int NB, Keep KEEP>
__device__ __forceinline__ void gate_epilogue(const FeedForwardArgs& a, char* mine, int lane, int64_t p0, int64_t q0,
                                              f32x16 (&acc)[NB][MB]) {
    using Exchange = RowExchange<32 * NB>;
    constexpr bool kFine = KEEP == Keep::kFine;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row0 = p0 + 32 * m;
        const int64_t row = row0 + (lane & 31);
        const bool kept = row < a.rows && (a.row_mask == nullptr || a.row_mask[row] != 0);
        // Opaque where there are more passes: else the addresses of all are held at once.
        int here = KEEP == Keep::kNothing ? lane : opaque_int(lane);
#pragma unroll
        for (int n = 0; n < NB / 2; ++n) {
            f32x16& gate = acc[n][m];
            f32x16& up = acc[n + NB / 2][m];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float act, slope;
                    activation<KEEP != Keep::kNothing>(a.activation, gate[4 * q + e], act, slope);
                    h[e] = act * up[4 * q + e];
                    if (KEEP != Keep::kNothing) {
                        slope *= up[4 * q + e];
                        gate[4 * q + e] = kFine ? Fine<T>::round(slope) : slope;
                        up[4 * q + e] = kFine ? Fine<T>::round(act) : act;
                    }
                }
                Exchange::put(mine, here, 64 * n + 16 * q + 8 * (here >> 5),
                              (u32x2){kept ? Values<T>::pack(h[0], h[1]) : 0u, kept ? Values<T>::pack(h[2], h[3]) : 0u});
            }
        }
        store_exchange<32 * NB>(mine, here, reinterpret_cast<char*>(a.h), 2 * a.pitch, row0, a.rows, 2 * q0, 2 * a.pitch);
#pragma unroll
        for (int o = 0; o < (KEEP != Keep::kNothing ? 2 : 0); ++o) {
            here = opaque_int(lane);
#pragma unroll
            for (int n = 0; n < NB / 2; ++n) {
                const f32x16& v = acc[n + o * (NB / 2)][m];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    Exchange::put(mine, here, 64 * n + 16 * q + 8 * (here >> 5),
                                  kFine ? (u32x2){Fine<T>::upper(v[4 * q], v[4 * q + 1]),
                                                  Fine<T>::upper(v[4 * q + 2], v[4 * q + 3])}
                                        : (u32x2){Values<T>::pack(v[4 * q], v[4 * q + 1]),
                                                  Values<T>::pack(v[4 * q + 2], v[4 * q + 3])});
                }
            }
            store_exchange<32 * NB>(mine, here, reinterpret_cast<char*>(a.gates + o * a.pitch), 4 * a.pitch, row0,
                                    a.rows, 2 * q0, 2 * a.pitch);
        }
        if constexpr (kFine) {
            constexpr int kBytes = Fine<T>::kLowerBytes;
            using LowerExchange = RowExchange<16 * NB * kBytes>;
            here = opaque_int(lane);
#pragma unroll
            for (int n = 0; n < NB / 2; ++n) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float first[4];
                    float second[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        first[e] = acc[n][m][4 * q + e];
                        second[e] = acc[n + NB / 2][m][4 * q + e];
                    }
                    const int byte = kBytes * (32 * n + 8 * q) + 4 * (here >> 5);
                    if constexpr (T == LSSO_HIP_BF16) {
                        LowerExchange::put(mine, here, byte, Fine<T>::lower(first, second));
                    } else {
                        LowerExchange::put(mine, here, byte, Fine<T>::third(first));
                        LowerExchange::put(mine, here, byte + 8, Fine<T>::third(second));
                    }
                }
            }
            store_exchange<16 * NB * kBytes>(mine, here, a.gates_lower, a.lower_pitch, row0, a.rows, kBytes * q0,
                                             a.lower_pitch);
        }
    }
}

//
// 262,144 x 256 -> 2 x 1,024 FP16 GELU: 491 us, 560 TFLOP/s, with 4 stages a tile
// bound by the epilogue's VALU work between the tiles' MFMAs (the eight waves of the
// one workgroup run in step); 8,192 x 768 -> 2 x 2,048: 52 us, 990 TFLOP/s, by LDS and
// L2 requests (a plain 8,192^3 product of the vendor's library reaches 1,436).
template <int T, int MB, int NB, int WP, int WQ>
using GateShape = RowsShape<T, MB, NB, WP, WQ, RowExchange<32 * NB>::kSize>;

template <int T, int MB, int NB, int WP, int WQ, Keep KEEP>
__global__ __launch_bounds__(64 * WP * WQ, 2) void gate_kernel(FeedForwardArgs a) {
    using S = GateShape<T, MB, NB, WP, WQ>;
    using P = typename S::PStage;
    using Q = typename S::QStage;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    constexpr int kColumns = S::BQ / 2;
    TileWalk walk(a.tiles, a.q_tiles);
    if (walk.left == 0) {
        return;
    }
    const RowLoads<P> p(a.x_stride, a.in_pitch, wave, lane);
    const RowLoads<Q> q(a.in_pitch, a.in_pitch, wave, lane);
    static_assert(Q::kLoads % 2 == 0, "whole loads of each weight");
    TileWalk ahead = walk;
    int stage = 0;
    BufferRsrc x, gate, up;
    const auto aim = [&] {
        const int64_t p0 = static_cast<int64_t>(ahead.p) * S::BP;
        const int64_t q0 = static_cast<int64_t>(ahead.q) * kColumns;
        const int64_t rows = ahead.left > 0 ? a.rows - p0 : 0;
        const int64_t columns = ahead.left > 0 ? a.hidden - q0 : 0;
        x = RowLoads<P>::aim(a.x + p0 * a.x_stride, a.x_stride, rows, S::BP);
        gate = RowLoads<Q>::aim(a.gate + q0 * a.in_pitch, a.in_pitch, columns, kColumns);
        up = RowLoads<Q>::aim(a.up + q0 * a.in_pitch, a.in_pitch, columns, kColumns);
    };
    aim();
    const int wave_column = S::wave_q(wave) / 2;
    run_rows_tiles<S>(
        lds, walk.left, a.stages,
        [&](char* to, int j) {
            const int k = stage * kRowsStageK;
            if (j < P::kLoads) {
                p.issue(x, to, S::kWaves, wave, k, j, j);
            } else {
                // The first half of Q's loads are the gate's rows, the second the up's.
                constexpr int kEach = Q::kLoads / 2;
                const int i = j - P::kLoads;
                q.issue(i < kEach ? gate : up, to + P::kBytes, S::kWaves, wave, k, i, i % kEach);
            }
            if (j == S::kLoads - 1 && ++stage == a.stages) {
                stage = 0;
                ahead.next();
                aim();
            }
        },
        [&](int n) { return n < NB / 2 ? wave_column + 32 * n : kColumns + wave_column + 32 * (n - NB / 2); },
        [&](f32x16 (&acc)[NB][MB]) {
            gate_epilogue<T, MB, NB, KEEP>(a, lds + S::kRingBytes + S::kWaveBytes * wave, lane,
                                           static_cast<int64_t>(walk.p) * S::BP + S::wave_p(wave),
                                           static_cast<int64_t>(walk.q) * kColumns + wave_column, acc);
            walk.next();
        });
}

// ------------------------------------------------------------------ y and dx
// out = P Q^T: y = h Wd^T, or dx = [dg | du] [Wg^T | Wu^T]^T with both weights
// transposed side by side, as dg and du lie.  With `splits` > 1 the stages are
// divided and FP32 partials left for join_kernel.
template <int T, int MB, int NB>
__device__ __forceinline__ void product_epilogue(const FeedForwardProduct& a, char* mine, int lane, int split,
                                                 int64_t p0, int64_t q0, const f32x16 (&acc)[NB][MB]) {
    if (a.partials != nullptr) {   // uniform
        store_partials<MB, NB>(mine, lane, acc, a.partials + split * a.rows * a.partial_pitch, a.partial_pitch, p0,
                               a.rows, q0);
        return;
    }
    constexpr int kGroup = NB < 2 ? 1 : 2;   // blocks of 32 columns at a time
    using Exchange = RowExchange<64 * kGroup>;
    const int half = lane >> 5;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row0 = p0 + 32 * m;
        const int64_t row = row0 + (lane & 31);
        const bool kept = row < a.rows && (a.row_mask == nullptr || a.row_mask[row] != 0);
#pragma unroll
        for (int n0 = 0; n0 < NB; n0 += kGroup) {
#pragma unroll
            for (int n = 0; n < kGroup; ++n) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x16& c = acc[n0 + n][m];
                    Exchange::put(mine, lane, 64 * n + 16 * q + 8 * half,
                                  (u32x2){kept ? Values<T>::pack(c[4 * q], c[4 * q + 1]) : 0u,
                                          kept ? Values<T>::pack(c[4 * q + 2], c[4 * q + 3]) : 0u});
                }
            }
            wave_lds_order();
            const int64_t column = q0 + 32 * n0 + Exchange::byte(lane) / 2;
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
}

template <int T, int MB, int NB, int WP, int WQ>
using ProductRows = RowsShape<T, MB, NB, WP, WQ, RowExchange<128>::kSize>;

template <int T, int MB, int NB, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ, 2) void product_kernel(FeedForwardProduct a) {
    using S = ProductRows<T, MB, NB, WP, WQ>;
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
        lds, walk.left, last - first, [&](char* to, int j) { stream.issue(to, j); },
        [&](int n) { return S::wave_q(wave) + 32 * n; },
        [&](const f32x16 (&acc)[NB][MB]) {
            product_epilogue<T, MB, NB>(a, lds + S::kRingBytes + S::kWaveBytes * wave, lane, split,
                                        static_cast<int64_t>(walk.p) * S::BP + S::wave_p(wave),
                                        static_cast<int64_t>(walk.q) * S::BQ + S::wave_q(wave), acc);
            walk.next();
        });
}

// ------------------------------------------------------------------ few rows
// Up to 32 rows (a decoding step): the time is the weights' bytes and the
// launches, not the MFMAs.  A workgroup takes 16 columns of h (16 rows of both
// weights) or of y, its eight waves share K, and a wave multiplies fragments on
// v_mfma_f32_16x16x32 as its loads bring them, four steps ahead and nothing
// staged; the waves' sums meet in LDS, in order.  h is carried as two 16-bit values
// (rounded, and what rounding left, nothing of a value past the type's range): its
// bytes are few here, and y is then rounded once, not after h.  A token of 256 -> 1,024 -> 256 takes 4.1 + 3.8 us; with the
// tiles' kernels 40 workgroups went through up to 16 stages and a third launch
// joined K's splits, 11 us.  A token of 4,096 -> 11,008 -> 4,096 with weights from
// HBM: 37 + 24 us, 4.9 and 3.8 TB/s (loads as the compiler places them: 36 + 40).
constexpr int kFewWaves = 8;
constexpr int kFewSteps = 4;   // of 32 k per wave, in flight together

// Rows of 8 k per lane: lane & 15 the row, lane >> 4 the piece.
struct FewLoads {
    BufferRsrc buffer;
    uint32_t offset;
    int element;
    int elements;
    __device__ __forceinline__ FewLoads(const uint16_t* base, int64_t stride, int64_t rows, int64_t k, int lane)
        : buffer(make_buffer(base, 2 * (rows < 16 ? rows : 16) * stride)),
          offset(static_cast<uint32_t>(2 * ((lane & 15) * stride + 8 * (lane >> 4)))),
          element(8 * (lane >> 4)),
          elements(static_cast<int>(k)) {}
    __device__ __forceinline__ u32x4 load(int k) const {
        return buffer_load16(buffer, k + element < elements ? offset + static_cast<uint32_t>(2 * k) : kOutOfRange);
    }
};

// sums[n][t]: of Q's operand n and P's row tile t, complete in the waves t < RT:
// lane & 15 the row, 4 (lane >> 4) + e the column.
// PARTS: 16-bit parts of P, which are added up.
template <int T, int NQ, int RT, int PARTS>
__device__ __forceinline__ void few_rows_product(const FewLoads (&q)[NQ], const FewLoads (&p)[PARTS][RT], int k_end,
                                                 f32x4 (&total)[NQ]) {
    __shared__ f32x4 parts[kFewWaves][NQ][RT][64];
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    f32x4 acc[NQ][RT] = {};
    for (int k = 32 * wave; k < k_end; k += 32 * kFewWaves * kFewSteps) {
        u32x4 qf[kFewSteps][NQ];
        u32x4 pf[kFewSteps][PARTS * RT];
#pragma unroll
        for (int s = 0; s < kFewSteps; ++s) {   // zeros behind k_end
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                qf[s][n] = q[n].load(k + 32 * kFewWaves * s);
            }
#pragma unroll
            for (int i = 0; i < PARTS * RT; ++i) {
                pf[s][i] = p[i / RT][i % RT].load(k + 32 * kFewWaves * s);
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // else the compiler moves each load down to its use
#pragma unroll
        for (int s = 0; s < kFewSteps; ++s) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int i = 0; i < PARTS * RT; ++i) {
                    acc[n][i % RT] = mfma_small<T>(qf[s][n], pf[s][i], acc[n][i % RT]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            parts[wave][n][t][lane] = acc[n][t];
        }
    }
    __syncthreads();
    if (wave < RT) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            f32x4 sum = parts[0][n][wave][lane];
#pragma unroll
            for (int w = 1; w < kFewWaves; ++w) {
                sum += parts[w][n][wave][lane];
            }
            total[n] = sum;
        }
    }
}

template <int T, int RT, Keep KEEP>
__global__ __launch_bounds__(64 * kFewWaves) void few_gate_kernel(FeedForwardArgs a) {
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    const int64_t q0 = 16 * static_cast<int64_t>(blockIdx.x);
    const FewLoads q[2] = {FewLoads(a.gate + q0 * a.in_pitch, a.in_pitch, a.hidden - q0, a.in_pitch, lane),
                           FewLoads(a.up + q0 * a.in_pitch, a.in_pitch, a.hidden - q0, a.in_pitch, lane)};
    f32x4 total[2];
    if constexpr (RT == 1) {
        const FewLoads p[1][1] = {{FewLoads(a.x, a.x_stride, a.rows, a.in_pitch, lane)}};
        few_rows_product<T, 2, 1, 1>(q, p, static_cast<int>(a.in_pitch), total);
    } else {
        const FewLoads p[1][2] = {{FewLoads(a.x, a.x_stride, a.rows, a.in_pitch, lane),
                                   FewLoads(a.x + 16 * a.x_stride, a.x_stride, a.rows - 16, a.in_pitch, lane)}};
        few_rows_product<T, 2, 2, 1>(q, p, static_cast<int>(a.in_pitch), total);
    }
    const int64_t row = 16 * wave + (lane & 15);
    const int64_t column = q0 + 4 * (lane >> 4);
    if (wave >= RT || row >= a.rows || column >= a.pitch) {
        return;
    }
    const bool kept = a.row_mask == nullptr || a.row_mask[row] != 0;
    float h[4];
    float first[4];
    float second[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float act, slope;
        activation<KEEP != Keep::kNothing>(a.activation, total[0][e], act, slope);
        h[e] = kept ? act * total[1][e] : 0.0f;
        first[e] = KEEP == Keep::kFine ? Fine<T>::round(slope * total[1][e]) : slope * total[1][e];
        second[e] = KEEP == Keep::kFine ? Fine<T>::round(act) : act;
    }
    const u32x2 rounded = {Values<T>::pack(h[0], h[1]), Values<T>::pack(h[2], h[3])};
    *reinterpret_cast<u32x2*>(a.h + row * a.pitch + column) = rounded;
    // Of an infinity the difference would be the other one, or NaN, and y NaN.
    const auto left = [](float value, float part) { return __builtin_isfinite(part) ? value - part : 0.0f; };
    *reinterpret_cast<u32x2*>(a.h_low + row * a.pitch + column) =
        (u32x2){Values<T>::pack(left(h[0], Values<T>::low(rounded[0])), left(h[1], Values<T>::high(rounded[0]))),
                Values<T>::pack(left(h[2], Values<T>::low(rounded[1])), left(h[3], Values<T>::high(rounded[1])))};
    if constexpr (KEEP == Keep::kRounded) {
        uint16_t* at = a.gates + 2 * row * a.pitch + column;
        *reinterpret_cast<u32x2*>(at) = (u32x2){Values<T>::pack(first[0], first[1]), Values<T>::pack(first[2], first[3])};
        *reinterpret_cast<u32x2*>(at + a.pitch) =
            (u32x2){Values<T>::pack(second[0], second[1]), Values<T>::pack(second[2], second[3])};
    }
    if constexpr (KEEP == Keep::kFine) {
        using F = Fine<T>;
        uint16_t* at = a.gates + 2 * row * a.pitch + column;
        *reinterpret_cast<u32x2*>(at) = (u32x2){F::upper(first[0], first[1]), F::upper(first[2], first[3])};
        *reinterpret_cast<u32x2*>(at + a.pitch) = (u32x2){F::upper(second[0], second[1]), F::upper(second[2], second[3])};
        char* lower = a.gates_lower + row * a.lower_pitch + F::kLowerBytes * (column / 8 * 8) + column % 8;
        if constexpr (T == LSSO_HIP_BF16) {
            *reinterpret_cast<uint32_t*>(lower) = F::lower(first, second);
        } else {
            *reinterpret_cast<uint32_t*>(lower) = F::third(first);
            *reinterpret_cast<uint32_t*>(lower + 8) = F::third(second);
        }
    }
}

template <int T, int RT, int PARTS>
__global__ __launch_bounds__(64 * kFewWaves) void few_product_kernel(FeedForwardProduct a) {
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    const int64_t q0 = 16 * static_cast<int64_t>(blockIdx.x);
    const FewLoads q[1] = {FewLoads(a.q + q0 * a.q_stride, a.q_stride, a.columns - q0, a.k, lane)};
    const auto rows = [&](const uint16_t* base, int from) {
        return FewLoads(base + from * a.p_stride, a.p_stride, a.rows - from, a.k, lane);
    };
    const uint16_t* const low = PARTS == 2 ? a.p_low : a.p;
    f32x4 total[1];
    if constexpr (RT == 1 && PARTS == 1) {
        few_rows_product<T, 1, 1, 1>(q, {{rows(a.p, 0)}}, static_cast<int>(a.k), total);
    } else if constexpr (RT == 1) {
        few_rows_product<T, 1, 1, 2>(q, {{rows(a.p, 0)}, {rows(low, 0)}}, static_cast<int>(a.k), total);
    } else if constexpr (PARTS == 1) {
        few_rows_product<T, 1, 2, 1>(q, {{rows(a.p, 0), rows(a.p, 16)}}, static_cast<int>(a.k), total);
    } else {
        few_rows_product<T, 1, 2, 2>(q, {{rows(a.p, 0), rows(a.p, 16)}, {rows(low, 0), rows(low, 16)}},
                                     static_cast<int>(a.k), total);
    }
    const int64_t row = 16 * wave + (lane & 15);
    const int64_t column = q0 + 4 * (lane >> 4);
    if (wave >= RT || row >= a.rows) {
        return;
    }
    const bool kept = a.row_mask == nullptr || a.row_mask[row] != 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (column + e < a.columns) {
            Values<T>::store(a.out + row * a.columns + column + e, kept ? total[0][e] : 0.0f);
        }
    }
}

// ----------------------------------------------------------------- dg and du
// dh goes through the exchange in FP32, 32 rows x 32 columns at a time: in its
// rows the factors are read and dg, du written as whole pieces.
template <int T, int MB, int NB, bool FINE>
__device__ __forceinline__ void grad_epilogue(const FeedForwardArgs& a, char* mine, int lane, int64_t p0, int64_t q0,
                                              const f32x16 (&acc)[NB][MB]) {
    using Exchange = RowExchange<128>;
    constexpr int kLanes = 4;   // of a row, 8 columns each
    constexpr int kRows = 64 / kLanes;
    constexpr int kSteps = 32 / kRows;
    const int half = lane >> 5;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t row0 = p0 + 32 * m;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int64_t column = q0 + 32 * n + 8 * (lane % kLanes);
            u32x4 raw[kSteps][2];
            typename Fine<T>::Lower lower[FINE ? kSteps : 1];
            bool kept[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int64_t row = row0 + kRows * i + lane / kLanes;
                if (row < a.rows && column < a.pitch) {
                    const uint16_t* at = a.gates + 2 * row * a.pitch + column;
                    raw[i][0] = load16_unaligned(at);
                    raw[i][1] = load16_unaligned(at + a.pitch);
                    if constexpr (FINE) {
                        lower[i].load(a.gates_lower + row * a.lower_pitch + Fine<T>::kLowerBytes * column);
                    }
                    kept[i] = a.row_mask == nullptr || a.row_mask[row] != 0;
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16& c = acc[n][m];
                Exchange::put(mine, lane, 32 * q + 16 * half,
                              (f32x4){c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]});
            }
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int r = kRows * i + lane / kLanes;
                const int64_t row = row0 + r;
                const f32x4 low = __builtin_bit_cast(f32x4, Exchange::piece(mine, r, 32 * (lane % kLanes)));
                const f32x4 high = __builtin_bit_cast(f32x4, Exchange::piece(mine, r, 32 * (lane % kLanes) + 16));
                if (row < a.rows && column < a.pitch) {
                    float dg[8];
                    float du[8];
                    if constexpr (FINE) {
                        lower[i].join(raw[i][0], raw[i][1], dg, du);
                    } else {
                        Values<T>::unpack8(raw[i][0], dg);
                        Values<T>::unpack8(raw[i][1], du);
                    }
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

template <int T, int MB, int NB, int WP, int WQ>
using GradShape = RowsShape<T, MB, NB, WP, WQ, RowExchange<128>::kSize>;

template <int T, int MB, int NB, int WP, int WQ, bool FINE>
__global__ __launch_bounds__(64 * WP * WQ, 2) void grad_kernel(FeedForwardArgs a) {
    using S = GradShape<T, MB, NB, WP, WQ>;
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
        lds, walk.left, a.stages, [&](char* to, int j) { stream.issue(to, j); },
        [&](int n) { return S::wave_q(wave) + 32 * n; },
        [&](const f32x16 (&acc)[NB][MB]) {
            grad_epilogue<T, MB, NB, FINE>(a, lds + S::kRingBytes + S::kWaveBytes * wave, lane,
                                           static_cast<int64_t>(walk.p) * S::BP + S::wave_p(wave),
                                           static_cast<int64_t>(walk.q) * S::BQ + S::wave_q(wave), acc);
            walk.next();
        });
}

// ----------------------------------------------------------- weight gradients
// One of up to three products P^T Q over a range of rows, P and Q in columns.
template <int T, int MB, int NB, int WP, int WQ, bool MASKED>
__global__ __launch_bounds__(64 * WP * WQ, 2) void weight_kernel(FeedForwardWeights a) {
    using S = ColumnsShape<T, MB, NB, WP, WQ>;
    using P = typename S::PStage;
    using Q = typename S::QStage;
    __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
    __shared__ uint32_t kept[MASKED ? kWeightSplitRows / 32 + kColumnsRing : 1];   // rows of each stage
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
        for (int64_t i = 64 * wave; i < a.split_rows + kColumnsRing * kColumnsStageK; i += S::kThreads) {
            const int64_t r = r0 + i + lane;
            const uint64_t rows = __ballot(r < r1 && a.row_mask[r < r1 ? r : r0] != 0);
            const int word = static_cast<int>(i / 32) + lane;
            if (lane < 2 && word < kWeightSplitRows / 32 + kColumnsRing) {
                kept[word] = static_cast<uint32_t>(rows >> (32 * lane));
            }
        }
        __syncthreads();
    }
    const ColumnLoads<P> p(w.p + p0, w.p_stride, w.p_columns - p0, wave, lane);
    const ColumnLoads<Q> q(w.q + q0, w.q_stride, w.q_columns - q0, wave, lane);
    f32x16 acc[NB][MB];
    run_columns_product<S>(lds, static_cast<int>((r1 - r0 + kColumnsStageK - 1) / kColumnsStageK), acc,
                           [&](char* to, int s, int j) {
                               const int64_t k = r0 + static_cast<int64_t>(s) * kColumnsStageK;
                               const uint32_t rows = MASKED ? __builtin_amdgcn_readfirstlane(kept[s]) : ~0u;
                               if (j < P::kLoads) {
                                   p.issue(to, S::kWaves, wave, k, r1, j, rows);
                               } else {
                                   q.issue(to + P::kBytes, S::kWaves, wave, k, r1, j - P::kLoads, rows);
                               }
                           });
    static_assert(RowExchange<128>::kSize <= S::kWaveBytes, "the exchange fits the wave's LDS");
    store_partials<MB, NB>(lds + S::kWaveBytes * wave, lane, acc,
                           a.partials + split * a.partial_floats + w.partial_offset, w.partial_pitch,
                           p0 + S::wave_p(wave), w.out_rows, q0 + S::wave_q(wave));
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
constexpr int kPackBlocks = 1 << 22;   // in x: a launch's x holds fewer than 2^32 threads

template <int T>
__global__ __launch_bounds__(256) void pack_kernel(FeedForwardPack a) {
    __shared__ uint16_t square[kPackEdge][kPackEdge + 8];
    int block = static_cast<int>(blockIdx.y) * kPackBlocks + static_cast<int>(blockIdx.x);
    int which = 0;
    while (which < a.count && block >= a.matrices[which].tiles) {
        block -= a.matrices[which].tiles;
        ++which;
    }
    if (which == a.count) {   // the grid is at least the sum of all tiles
        return;
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

// Tiles of the row products: 256 x 256 by 8 waves, one workgroup per CU; 128 x 128
// by 4, two per CU; or small ones (64 x 64, three; the gate's 64 x 128, two) by 4.  The
// larger the tile, the fewer bytes a product moves between L2, LDS and registers, but
// what counts first is how often the workgroups that are resident go round: small
// tiles while they go round once, then the fewer of 5 per round of large tiles and 3
// per round of middle ones.  Measured with kernel and K the same on both sides:
//   small and middle, y of K = 2,048 and 768 columns: 768 and 192 tiles (one round and
//   one) 22.8 and 25.0 us, 864 and 216 (two and one) 37.0 and 26.0; gate of K = 768: 512
//   and 256 13.4 and 14.0, 544 and 272 18.6 and 14.8; dg and du of K = 768: 736 and 184 16.0
//   and 18.3, 800 and 200 23.6 and 18.5;
//   middle and large, the same y: 480 and 120 tiles (one and one) 39.9 and 47.6, 516 and
//   129 (two and one) 56.3 and 50.8, 1,020 and 255 69.7 and 60.5, 1,032 and 258 (three
//   and two) 82.0 and 93.0, 1,536 and 384 102 and 100, 1,548 and 387 (four and two) 133
//   and 130, 6,144 and 1,536 (twelve and six) 436 and 366; the gate of K = 768: 512 and
//   128 18.1 and 22.4, 544 and 136 23.8 and 22.6, 1,056 and 264 36.2 and 42.8, 1,568 and
//   392 53.7 and 44.3.  (The gate of K = 256, whose epilogue is most of it, keeps 12.4
//   against 15.3 on middle tiles up to 224 large ones, and loses 16.4 to 15.1 from 240.)
enum class Edge { kLarge, kMiddle, kSmall };

int64_t tiles_of(int64_t p, int64_t q, int64_t bp, int64_t bq) { return ((p + bp - 1) / bp) * ((q + bq - 1) / bq); }

constexpr int64_t kCus = 256;

// small_q: columns of a small tile, of which small_slots are resident at a time.
Edge choose_edge(int64_t p, int64_t q, int64_t small_q = 64, int64_t small_slots = 3 * kCus) {
    if (tiles_of(p, q, 64, small_q) <= small_slots) {
        return Edge::kSmall;
    }
    const int64_t large = (tiles_of(p, q, 256, 256) + kCus - 1) / kCus;
    const int64_t middle = (tiles_of(p, q, 128, 128) + 2 * kCus - 1) / (2 * kCus);
    return 5 * large <= 3 * middle ? Edge::kLarge : Edge::kMiddle;
}

// A multiple of eight workgroups (one share per XCD), at most what is resident.
dim3 tile_grid(int tiles, int slots, int splits = 1) {
    const int per_xcd = (tiles + 7) / 8;
    return dim3(static_cast<unsigned>(8 * (per_xcd < slots ? per_xcd : slots)), static_cast<unsigned>(splits));
}

template <int T, int MB, int NB, int WP, int WQ, Keep KEEP>
hipError_t launch_gate(FeedForwardArgs a, hipStream_t stream) {
    using S = GateShape<T, MB, NB, WP, WQ>;
    a.stages = static_cast<int>((a.in_pitch + kRowsStageK - 1) / kRowsStageK);
    a.q_tiles = static_cast<int>((a.pitch + S::BQ / 2 - 1) / (S::BQ / 2));
    a.tiles = a.q_tiles * static_cast<int>((a.rows + S::BP - 1) / S::BP);
    gate_kernel<T, MB, NB, WP, WQ, KEEP><<<tile_grid(a.tiles, S::kSlots), S::kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

template <int T, Keep KEEP>
hipError_t launch_tiles_gate(const FeedForwardArgs& a, hipStream_t stream) {
    switch (choose_edge(a.rows, 2 * a.pitch, 128, 2 * kCus)) {
        case Edge::kLarge: return launch_gate<T, 2, 4, 4, 2, KEEP>(a, stream);
        case Edge::kMiddle: return launch_gate<T, 2, 2, 2, 2, KEEP>(a, stream);
        default: return launch_gate<T, 1, 2, 2, 2, KEEP>(a, stream);
    }
}

template <int T, Keep KEEP>
hipError_t launch_few_gate(const FeedForwardArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((a.pitch + 15) / 16));
    if (a.rows <= 16) {
        few_gate_kernel<T, 1, KEEP><<<grid, 64 * kFewWaves, 0, stream>>>(a);
    } else {
        few_gate_kernel<T, 2, KEEP><<<grid, 64 * kFewWaves, 0, stream>>>(a);
    }
    return hipGetLastError();
}

template <int T, Keep KEEP>
hipError_t launch_gate(const FeedForwardArgs& a, hipStream_t stream) {
    return a.rows <= kFewRows ? launch_few_gate<T, KEEP>(a, stream) : launch_tiles_gate<T, KEEP>(a, stream);
}

template <int T>
hipError_t launch_gate(const FeedForwardArgs& a, hipStream_t stream) {
    if (a.gates == nullptr) {
        return launch_gate<T, Keep::kNothing>(a, stream);
    }
    return a.gates_lower != nullptr ? launch_gate<T, Keep::kFine>(a, stream) : launch_gate<T, Keep::kRounded>(a, stream);
}

template <int T, int MB, int NB, int WP, int WQ>
hipError_t launch_product(FeedForwardProduct a, hipStream_t stream) {
    using S = ProductRows<T, MB, NB, WP, WQ>;
    a.q_tiles = static_cast<int>((a.columns + S::BQ - 1) / S::BQ);
    a.tiles = a.q_tiles * static_cast<int>((a.rows + S::BP - 1) / S::BP);
    product_kernel<T, MB, NB, WP, WQ><<<tile_grid(a.tiles, S::kSlots, a.splits), S::kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

template <int T, int PARTS>
hipError_t launch_few_product(const FeedForwardProduct& a, dim3 grid, hipStream_t stream) {
    if (a.rows <= 16) {
        few_product_kernel<T, 1, PARTS><<<grid, 64 * kFewWaves, 0, stream>>>(a);
    } else {
        few_product_kernel<T, 2, PARTS><<<grid, 64 * kFewWaves, 0, stream>>>(a);
    }
    return hipGetLastError();
}

template <int T>
hipError_t launch_product(const FeedForwardProduct& args, hipStream_t stream) {
    FeedForwardProduct a = args;
    if (a.rows <= kFewRows) {
        const dim3 grid(static_cast<unsigned>((a.columns + 15) / 16));
        return a.p_low != nullptr ? launch_few_product<T, 2>(a, grid, stream) : launch_few_product<T, 1>(a, grid, stream);
    }
    if (a.splits == 1) {
        a.partials = nullptr;
    }
    hipError_t error;
    switch (choose_edge(a.rows, a.columns)) {
        case Edge::kLarge: error = launch_product<T, 2, 4, 4, 2>(a, stream); break;
        case Edge::kMiddle: error = launch_product<T, 2, 2, 2, 2>(a, stream); break;
        default: error = launch_product<T, 1, 1, 2, 2>(a, stream); break;
    }
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

template <int T, int MB, int NB, int WP, int WQ>
hipError_t launch_grad(FeedForwardArgs a, hipStream_t stream) {
    using S = GradShape<T, MB, NB, WP, WQ>;
    a.stages = static_cast<int>((a.out_pitch + kRowsStageK - 1) / kRowsStageK);
    a.q_tiles = static_cast<int>((a.pitch + S::BQ - 1) / S::BQ);
    a.tiles = a.q_tiles * static_cast<int>((a.rows + S::BP - 1) / S::BP);
    if (a.gates_lower != nullptr) {
        grad_kernel<T, MB, NB, WP, WQ, true><<<tile_grid(a.tiles, S::kSlots), S::kThreads, 0, stream>>>(a);
    } else {
        grad_kernel<T, MB, NB, WP, WQ, false><<<tile_grid(a.tiles, S::kSlots), S::kThreads, 0, stream>>>(a);
    }
    return hipGetLastError();
}

// With few stages a tile's time is its epilogue (the factors read, dg and du
// written), which two workgroups of a CU overlap and one large one does not: 65,536
// rows of 1,024 take 142 us on middle tiles and 181 on large ones with K = 256, 163 and
// 190 with 384, 179 and 202 with 512; 32,768 of 2,048 with 768 225 and 218, 16,384 of 2,048
// with 1,024 129 and 123.
template <int T>
hipError_t launch_grad(const FeedForwardArgs& a, hipStream_t stream) {
    Edge edge = choose_edge(a.rows, a.pitch);
    if (edge == Edge::kLarge && a.out_pitch <= 512) {
        edge = Edge::kMiddle;
    }
    switch (edge) {
        case Edge::kLarge: return launch_grad<T, 2, 4, 4, 2>(a, stream);
        case Edge::kMiddle: return launch_grad<T, 2, 2, 2, 2>(a, stream);
        default: return launch_grad<T, 1, 1, 2, 2>(a, stream);
    }
}

template <int T, bool MASKED>
void launch_weights(const FeedForwardWeights& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.tiles * a.splits));
    if (a.large) {
        weight_kernel<T, 2, 4, 4, 2, MASKED><<<grid, 512, 0, stream>>>(a);
    } else {
        weight_kernel<T, 2, 2, 2, 2, MASKED><<<grid, 256, 0, stream>>>(a);
    }
}

template <int T>
hipError_t launch_weights(const FeedForwardWeights& a, hipStream_t stream) {
    a.row_mask != nullptr ? launch_weights<T, true>(a, stream) : launch_weights<T, false>(a, stream);
    return hipGetLastError();
}

}  // namespace

void plan_product(int64_t rows, int64_t columns, int64_t stages, FeedForwardProduct* a) {
    a->stages = static_cast<int>(stages);
    int64_t splits = 1;
    if (rows > kFewRows && choose_edge(rows, columns) == Edge::kSmall) {
        // A long K over few tiles: split so that each CU has two, at least 4
        // stages each.
        const int64_t tiles = tiles_of(rows, columns, 64, 64);
        splits = tiles > 0 ? 2 * kCus / tiles : 1;
        splits = splits < stages / 4 ? splits : stages / 4;
        splits = splits < 1 ? 1 : splits;
    }
    a->split_stages = static_cast<int>((stages + splits - 1) / splits);
    a->splits = static_cast<int>((stages + a->split_stages - 1) / a->split_stages);
    a->partial_pitch = (columns + 7) / 8 * 8;
}

// Tiles of 256 x 256 (one workgroup per CU) where they are well filled and their
// splits still have 512 rows, else of 128 x 128 (three).  The splits fill the
// device's workgroups once: more of them would write and read more partials, a
// second round of workgroups would be partly empty.
void plan_weights(FeedForwardWeights* a) {
    const auto count = [&](int64_t edge) {
        int64_t tiles = 0;
        for (int i = 0; i < a->count; ++i) {
            tiles += tiles_of(a->products[i].out_rows, a->products[i].partial_pitch, edge, edge);
        }
        return tiles;
    };
    const int64_t large = count(256);
    a->large = 3 * large <= count(128) && large * a->rows >= 512 * kCus;
    const int64_t edge = a->large ? 256 : 128;
    a->tiles = count(edge);
    a->partial_floats = 0;
    for (int i = 0; i < a->count; ++i) {
        WeightProduct& w = a->products[i];
        w.q_tiles = (w.partial_pitch + edge - 1) / edge;
        w.tiles = w.q_tiles * ((w.out_rows + edge - 1) / edge);
        w.partial_offset = a->partial_floats;
        a->partial_floats += w.out_rows * w.partial_pitch;
    }
    int64_t splits = a->tiles > 0 ? (a->large ? kCus : 3 * kCus) / a->tiles : 1;
    const int64_t most = (a->rows + 127) / 128;
    splits = splits < most ? splits : most;
    splits = splits < 1 ? 1 : splits;
    // The kernel keeps a split's mask in LDS; as many splits with a mask as
    // without one, so that it only changes what is added.
    const int64_t least = (a->rows + kWeightSplitRows - 1) / kWeightSplitRows;
    splits = splits > least ? splits : least;
    const int64_t per = (a->rows + splits - 1) / splits;
    a->split_rows = (per + kColumnsStageK - 1) / kColumnsStageK * kColumnsStageK;
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
    const dim3 grid(static_cast<unsigned>(tiles < kPackBlocks ? tiles : kPackBlocks),
                    static_cast<unsigned>((tiles + kPackBlocks - 1) / kPackBlocks));
    if (type == LSSO_HIP_BF16) {
        pack_kernel<LSSO_HIP_BF16><<<grid, 256, 0, stream>>>(a);
    } else {
        pack_kernel<LSSO_HIP_F16><<<grid, 256, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
