// Tiled 16-bit matrix product of the feed-forward kernels:
//   out[p][q] = sum over k of P[p, k] Q[q, k],  FP32 accumulation,
// in two forms: for operands that lie in memory across k ([k][p], "columns": the
// weight gradients dy^T x, whose k are the rows of long activations), and for
// operands along k ([p][k], "rows": x W^T; dy W comes to it with W transposed
// once per call), further down.
//
// A workgroup of 4 waves owns a BP x BQ tile, a wave MB x NB blocks of 32 x 32
// on v_mfma_f32_32x32x16.  The operands' stages of 32 k go from memory
// to LDS without passing registers (buffer_load ... lds, 16 bytes per lane), in
// a ring of three: two stages are in flight while one is multiplied.  The
// largest tile, 256 x 128, keeps 128 accumulators and 72 KB of LDS, so two
// workgroups share a CU and one multiplies while the other waits, begins or
// stores.  Per stage a wave reads 12 KB of fragments for 16 MFMAs; a stage's
// second half is read under the first half's MFMAs and the next stage's first
// half under the second's, so the one barrier per stage finds nothing to wait
// for but the loads.
//
// LDS is written linearly by the loads (lane i at 16 i), so conflicts are
// avoided by which global piece a lane asks for:
//   rows:    64 bytes per p, piece c at slot c ^ f(p), f = ((p >> 1) & 3) ^
//            ((p >> 3) & 1): any 8 or 16 consecutive rows of one piece fall on
//            different banks;
//   columns: 2 BP bytes per k, group of 16 columns g at g ^ {0, 3, 5, 6}[k % 4]
//            (k % 4 for 4 groups): the 4 rows of a transposed read likewise.
//
// Rows past an operand's end, k past K and rows that a mask excludes are loads
// past the buffer's end, which bring zeros and touch no memory.
#pragma once

#include "lsso_device.h"
#include "lsso_values.h"

namespace lsso_hip {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void LdsVoid;

constexpr int kStageK = 32;
constexpr int kRing = 3;
constexpr int kProductThreads = 256;

template <int T>
__device__ __forceinline__ f32x16 mfma_block(const u32x4& a, const u32x4& b, const f32x16& c) {
    if constexpr (T == LSSO_HIP_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
}

// Bytes of one operand's stage, and the per-lane side of its loads and reads.
// WIDTH: rows (or columns) of the operand in the tile; IN_ROWS: [p][k] in memory.
template <int WIDTH, bool IN_ROWS>
struct StageLayout {
    static constexpr int kBytes = WIDTH * kStageK * 2;
    static constexpr int kLoads = kBytes / 1024 / 4;          // per wave
    static constexpr int kRowsPerLoad = 1024 / (2 * WIDTH);   // of k, in columns
    static_assert(kLoads >= 1, "a tile edge is at least 64");

    __device__ static __forceinline__ int row_swizzle(int p) { return ((p >> 1) & 3) ^ ((p >> 3) & 1); }
    __device__ static __forceinline__ int column_swizzle(int k) {
        if constexpr (WIDTH == 64) {
            return k & 3;
        }
        return ((k & 1) != 0 ? 3 : 0) ^ ((k & 2) != 0 ? 5 : 0);
    }
    // What lane `lane` of wave `wave` loads with load j: p (in rows) or k (in columns) ...
    __device__ static __forceinline__ int load_line(int wave, int lane, int j) {
        return IN_ROWS ? 16 * (4 * j + wave) + (lane >> 2)
                       : kRowsPerLoad * (4 * j + wave) + lane / (WIDTH / 8);
    }
    // ... and its first element along the line; the same for every j.
    __device__ static __forceinline__ int load_element(int wave, int lane) {
        const int line = load_line(wave, lane, 0);
        if constexpr (IN_ROWS) {
            return 8 * ((lane & 3) ^ row_swizzle(line));
        } else {
            const int piece = lane % (WIDTH / 8);
            return 16 * ((piece >> 1) ^ column_swizzle(line)) + 8 * (piece & 1);
        }
    }
    // Byte of this lane's fragment of the block of 32 p from p0 (a multiple of
    // 32) in a stage, of k step 0 or 1.
    __device__ static __forceinline__ int fragment(int lane, int p0, int step) {
        if constexpr (IN_ROWS) {
            const int p = lane & 31;
            return 64 * p0 + (64 * p + 16 * ((2 * step + (lane >> 5)) ^ row_swizzle(p)));
        } else {
            const int k = (lane & 15) / 4 + 8 * (lane >> 5);
            const int group = p0 / 16 + ((lane >> 4) & 1);
            return 2 * WIDTH * (k + 16 * step) + 32 * (group ^ column_swizzle(k)) + 8 * (lane & 3);
        }
    }
    __device__ static __forceinline__ u32x4 read(const char* at) {
        if constexpr (IN_ROWS) {
            return *reinterpret_cast<const u32x4*>(at);
        } else {
            const u32x2 low = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at)));
            const u32x2 high =
                __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at + 2 * WIDTH * 4)));
            return (u32x4){low[0], low[1], high[0], high[1]};
        }
    }
};

__device__ __forceinline__ void load_to_lds(BufferRsrc buffer, char* lds, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (LdsVoid*)lds, 16, offset, 0, 0, 0);
}

// This wave's LDS reads are done and all but its newest PENDING loads have
// landed, then the same of every wave of the workgroup.
template <int PENDING>
__device__ __forceinline__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PENDING) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// An operand of the product.  In rows: `base` is the tile's first row, `lines`
// the rows from there on, `elements` = K.  In columns: `base` is the tile's
// first column of k = 0, `lines` = K, `elements` the columns from there on.
// Both lines' strides and `elements` are multiples of 8 and base is 16-byte
// aligned (or a tile offset of 16-byte pieces from such).
struct Operand {
    const uint16_t* base;
    int64_t stride;
    int64_t lines;
    int64_t elements;
};

// T: type code; MB x NB blocks of 32 x 32 per wave; WP waves along P, 4 / WP
// along Q.
template <int T_, bool P_ROWS_, bool Q_ROWS_, int MB_, int NB_, int WP_>
struct ProductShape {
    static constexpr int T = T_;
    static constexpr bool P_ROWS = P_ROWS_;
    static constexpr bool Q_ROWS = Q_ROWS_;
    static constexpr int MB = MB_;
    static constexpr int NB = NB_;
    static constexpr int WP = WP_;
    static constexpr int WQ = 4 / WP;
    static constexpr int BP = 32 * MB * WP;
    static constexpr int BQ = 32 * NB * WQ;
    using PLayout = StageLayout<BP, P_ROWS>;
    using QLayout = StageLayout<BQ, Q_ROWS>;
    static constexpr int kStageBytes = PLayout::kBytes + QLayout::kBytes;
    static constexpr int kLdsBytes = kRing * kStageBytes;
    static constexpr int kWaveBytes = kLdsBytes / 4;   // of the epilogue
    static constexpr int kLoads = PLayout::kLoads + QLayout::kLoads;
    // First row and column of the tile that are this wave's.
    __device__ static __forceinline__ int wave_p(int wave) { return 32 * MB * (wave % WP); }
    __device__ static __forceinline__ int wave_q(int wave) { return 32 * NB * (wave / WP); }
};

// This wave's index, as the scalar that it is.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Runs `stages` stages (at least one): issue(buffer, s) starts the loads of
// stage s (which may lie past the last) into the LDS stage `buffer`, exactly
// kLoads per wave.  q_start(n) is the tile's first column of this wave's Q block
// n.  The order is written down with scheduling barriers: left to itself the
// compiler moves the fragments' reads down to their MFMAs, to save registers
// that nothing else needs, and every MFMA then waits for LDS.
template <typename S, typename Issue, typename QStart>
__device__ __forceinline__ void run_product(char* lds, int stages, f32x16 (&acc)[S::NB][S::MB], Issue issue,
                                            QStart q_start) {
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[n][m][e] = 0.0f;
            }
        }
    }
    u32x4 pf[2][S::MB];
    u32x4 qf[2][S::NB];
    const auto read = [&](int buffer, int step) {
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            qf[step][n] = S::QLayout::read(lds + buffer * S::kStageBytes + S::PLayout::kBytes +
                                           S::QLayout::fragment(lane, q_start(n), step));
        }
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
            pf[step][m] = S::PLayout::read(lds + buffer * S::kStageBytes +
                                           S::PLayout::fragment(lane, S::wave_p(wave) + 32 * m, step));
        }
    };
    const auto multiply = [&](int step) {
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
#pragma unroll
            for (int n = 0; n < S::NB; ++n) {
                acc[n][m] = mfma_block<S::T>(qf[step][n], pf[step][m], acc[n][m]);
            }
        }
    };
    const auto stage = [&](int buffer, int s) {
        issue(lds + (buffer + 2) % kRing * S::kStageBytes, s + 2);
        read(buffer, 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(0);
        __builtin_amdgcn_sched_barrier(0);
        stage_barrier<S::kLoads>();
        read((buffer + 1) % kRing, 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply(1);
        __builtin_amdgcn_sched_barrier(0);
    };
    issue(lds, 0);
    issue(lds + S::kStageBytes, 1);
    stage_barrier<S::kLoads>();
    read(0, 0);
    for (int s = 0;;) {
        stage(0, s);
        if (++s == stages) break;
        stage(1, s);
        if (++s == stages) break;
        stage(2, s);
        if (++s == stages) break;
    }
    // The loads past the last stage still write their zeros: neither into LDS
    // that the epilogue uses nor into what another workgroup may hold by then.
    stage_barrier<0>();
}

// The accumulators of one block hold, in lane (half, j), row p = j and columns
// q = 8 i + 4 half + e of entry 4 i + e.  row_pieces() exchanges the halves so
// that a lane holds two whole pieces of 8 columns: piece c (0, 1) the columns
// 16 c + 8 half + 0 .. 7.
__device__ __forceinline__ void row_pieces(const f32x16& acc, float (&piece)[2][8]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const auto pair = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[8 * c + e]),
                                                               __float_as_uint(acc[8 * c + 4 + e]), false, false);
            piece[c][e] = __uint_as_float(pair[0]);
            piece[c][4 + e] = __uint_as_float(pair[1]);
        }
    }
}

// ---------------------------------------------------------------------------
// The product for both operands in rows (x W^T).  A stage is 64 k, so that every
// load covers whole 128-byte lines: the L2 answers one request per channel and
// clock whatever its size, half a request per CU, and with stages of 32 k (64
// bytes of a row) the requests alone took longer than the MFMAs.  For the same
// reason the largest tile is 256 x 256 (8 waves, 64 KB a stage): 32 bytes per CU
// and clock at the matrix rate, where the L2 gives 54.  Fragments of P read
// straight from memory into the lanes that multiply them save LDS bandwidth, but
// 64 lanes on 16 rows are 64 separate accesses (16 bytes per clock).
//
// Two stages alternate: one is multiplied while the next one's loads are in
// flight.  Fragments of a step (16 k) are read under the MFMAs of the step
// before; the barrier that frees a stage and admits the next lies before the
// last step's MFMAs, whose fragments are in registers by then.
constexpr int kRowsStageK = 64;
constexpr int kRowsSteps = 4;

// Stage of WIDTH rows, loaded by WAVES waves.
template <int WIDTH, int WAVES>
struct RowsStage {
    static constexpr int kBytes = WIDTH * kRowsStageK * 2;
    static constexpr int kLoads = kBytes / 1024 / WAVES;   // per wave
    static constexpr int kRowsPerRound = 8 * WAVES;        // of one load of every wave
    static_assert(kLoads >= 1, "every wave loads");
    // Piece c of row p lies at slot c ^ swizzle(p), so that any 8 or 16 rows of
    // one piece fall on different banks.
    __device__ static __forceinline__ int swizzle(int p) { return (p & 7) ^ ((p >> 3) & 1); }
    // Row of this lane's first load (kRowsPerRound further for each one after
    // it) and its first element of that row.
    __device__ static __forceinline__ int load_row(int wave, int lane) { return 8 * wave + (lane >> 3); }
    __device__ static __forceinline__ int load_element(int wave, int lane) {
        return 8 * ((lane & 7) ^ swizzle(load_row(wave, lane)));
    }
    // This lane's fragment of rows p0 .. p0 + 31 (p0 a multiple of 32) at a step.
    __device__ static __forceinline__ u32x4 read(const char* stage, int lane, int p0, int step) {
        const int p = lane & 31;
        return *reinterpret_cast<const u32x4*>(stage + 128 * p0 +
                                               (128 * p + 16 * ((2 * step + (lane >> 5)) ^ swizzle(p))));
    }
};

// T: type code; MB x NB blocks of 32 x 32 per wave, WP x WQ waves; EXCHANGE:
// bytes of LDS per wave for the epilogue.
template <int T_, int MB_, int NB_, int WP_, int WQ_, int EXCHANGE>
struct RowsShape {
    static constexpr int T = T_;
    static constexpr int MB = MB_;
    static constexpr int NB = NB_;
    static constexpr int WP = WP_;
    static constexpr int WQ = WQ_;
    static constexpr int kWaves = WP * WQ;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int BP = 32 * MB * WP;
    static constexpr int BQ = 32 * NB * WQ;
    using PStage = RowsStage<BP, kWaves>;
    using QStage = RowsStage<BQ, kWaves>;
    static constexpr int kStageBytes = PStage::kBytes + QStage::kBytes;
    static constexpr int kRingBytes = 2 * kStageBytes;
    static constexpr int kWaveBytes = EXCHANGE;
    static constexpr int kLdsBytes = kRingBytes + kWaves * EXCHANGE;
    static constexpr int kLoads = PStage::kLoads + QStage::kLoads;
    // Workgroups that are resident on one XCD's 32 CUs: by LDS (160 KB) and by
    // registers (accumulators, two steps' fragments and 48 more of 512 for the
    // waves of a SIMD).
    static constexpr int kByLds = 160 * 1024 / kLdsBytes;
    static constexpr int kByRegisters = 512 / (16 * MB * NB + 8 * (MB + NB) + 48) * 4 / kWaves;
    static constexpr int kSlots = 32 * (kByLds < kByRegisters ? kByLds : kByRegisters);
    __device__ static __forceinline__ int wave_p(int wave) { return 32 * MB * (wave % WP); }
    __device__ static __forceinline__ int wave_q(int wave) { return 32 * NB * (wave / WP); }
};

// The tiles of one workgroup: XCD x (workgroup index mod 8) takes the x-th eighth
// of them, columns fastest, its workgroups in turn, so that the tiles that
// share P's rows are multiplied at the same time beside one L2.
struct TileWalk {
    int p;            // tile of this step
    int q;
    int left;         // tiles to go, this one included
    int step_p;
    int step_q;
    int q_tiles;

    __device__ __forceinline__ TileWalk(int tiles, int q_tiles_) : q_tiles(q_tiles_) {
        const int per_xcd = (tiles + 7) / 8;
        const int begin = static_cast<int>(blockIdx.x % 8) * per_xcd;
        const int end = begin + per_xcd < tiles ? begin + per_xcd : tiles;
        const int first = begin + static_cast<int>(blockIdx.x / 8);
        const int step = static_cast<int>(gridDim.x / 8);
        left = first < end ? (end - first + step - 1) / step : 0;
        p = first / q_tiles;
        q = first - p * q_tiles;
        step_p = step / q_tiles;
        step_q = step - step_p * q_tiles;
    }
    __device__ __forceinline__ void next() {
        --left;
        p += step_p;
        q += step_q;
        if (q >= q_tiles) {
            q -= q_tiles;
            ++p;
        }
    }
};

// Runs `tiles` tiles of `stages` stages each.  issue(lds) starts the loads of the
// next stage, kLoads per wave, in order through all tiles and asked for two past
// the last; q_start(n) is the tile's first row of Q of this wave's block n;
// epilogue(acc) takes a tile's sums.  The loads run ahead across the tiles'
// borders, so a tile's first stages arrive under the epilogue of the one
// before: a tile of 256 k has four stages, and began with a wait for memory as
// long as all its MFMAs.
template <typename S, typename Issue, typename QStart, typename Epilogue>
__device__ __forceinline__ void run_rows_tiles(char* lds, int tiles, int stages, Issue issue, QStart q_start,
                                               Epilogue epilogue) {
    const int lane = threadIdx.x & 63;
    const int wave = wave_index();
    f32x16 acc[S::NB][S::MB];
    u32x4 pf[2][S::MB];
    u32x4 qf[2][S::NB];
    const auto read = [&](const char* stage, int step) {
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            qf[step & 1][n] = S::QStage::read(stage + S::PStage::kBytes, lane, q_start(n), step);
        }
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
            pf[step & 1][m] = S::PStage::read(stage, lane, S::wave_p(wave) + 32 * m, step);
        }
    };
    const auto multiply = [&](int step) {
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
#pragma unroll
            for (int n = 0; n < S::NB; ++n) {
                acc[n][m] = mfma_block<S::T>(qf[step & 1][n], pf[step & 1][m], acc[n][m]);
            }
        }
    };
    int at = 0;   // LDS offset of this stage
    const auto stage = [&] {
        char* const here = lds + at;
        at ^= S::kStageBytes;
#pragma unroll
        for (int step = 0; step < kRowsSteps - 1; ++step) {
            read(here, step + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(step);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage_barrier<0>();   // the next stage has landed, and nobody reads this one any more
        issue(here);
        read(lds + at, 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply(kRowsSteps - 1);
        __builtin_amdgcn_sched_barrier(0);
    };
    issue(lds);
    issue(lds + S::kStageBytes);
    stage_barrier<S::kLoads>();
    read(lds, 0);
    for (int tile = 0; tile < tiles; ++tile) {
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
#pragma unroll
            for (int m = 0; m < S::MB; ++m) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    acc[n][m][e] = 0.0f;
                }
            }
        }
        for (int s = 0; s < stages; ++s) {
            stage();
        }
        epilogue(acc);
    }
    // The loads past the last stage still write their zeros: not into LDS that
    // another workgroup may hold by then.
    stage_barrier<0>();
}

// A wave's exchange of 32 rows of BYTES (64 or 128) through its own part of LDS,
// from a lane per row to BYTES / 16 consecutive lanes per row: stored from the
// accumulators' layout, an instruction covers 32 bytes of each of 32 rows, and
// partly written lines cost the memory side twice (131,072 x 688 x 3 stores at
// 2.6 TB/s); exchanged, it covers whole lines.  LDS serves a wave's accesses in
// order, so no barrier is needed; pieces are swizzled as in the stages.
template <int BYTES>
struct RowExchange {
    static constexpr int kSize = 32 * BYTES;
    static constexpr int kLanes = BYTES / 16;        // per row
    static constexpr int kRows = 64 / kLanes;        // per access
    static constexpr int kSteps = 32 / kRows;
    __device__ static __forceinline__ int swizzle(int row) {
        return BYTES == 128 ? (row & 7) ^ ((row >> 3) & 1) : ((row >> 1) & 3) ^ ((row >> 3) & 1);
    }
    // V: 8 or 16 bytes at `byte` of row lane % 32.
    template <typename V>
    __device__ static __forceinline__ void put(char* lds, int lane, int byte, const V& value) {
        const int r = lane & 31;
        *reinterpret_cast<V*>(lds + r * BYTES + (byte ^ (16 * swizzle(r)))) = value;
    }
    __device__ static __forceinline__ int row(int lane, int step) { return kRows * step + lane / kLanes; }
    __device__ static __forceinline__ int byte(int lane) { return 16 * (lane % kLanes); }
    __device__ static __forceinline__ u32x4 piece(const char* lds, int row, int byte) {
        return *reinterpret_cast<const u32x4*>(lds + row * BYTES + (byte ^ (16 * swizzle(row))));
    }
    __device__ static __forceinline__ u32x4 get(const char* lds, int lane, int step) {
        return piece(lds, row(lane, step), byte(lane));
    }
};

}  // namespace lsso_hip
