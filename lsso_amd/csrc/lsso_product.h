// Tiled 16-bit matrix products of the feed-forward kernels:
//   out[p][q] = sum over k of P[p, k] Q[q, k],  FP32 accumulation,
// in two forms: for operands that lie in memory across k ([k][p], "columns": the
// weight gradients dy^T x, whose k are the rows of long activations), and for
// operands along k ([p][k], "rows": x W^T; dy W comes to it with W transposed
// once per call), further down.
//
// A workgroup owns a BP x BQ tile, each of its waves MB x NB blocks of 32 x 32 on
// v_mfma_f32_32x32x16.  The operands' stages go from memory to LDS without
// passing registers (buffer_load ... lds, 16 bytes per lane), and a step's
// fragments are read under the MFMAs of the step before.  LDS is written
// linearly by the loads (lane i at 16 i), so bank conflicts are avoided by which
// piece of memory a lane asks for (the swizzles below: no conflict cycles in the
// columns' kernel, 0.3 to 2% in the rows', 3 to 6% where the epilogue exchanges
// most).  Rows past an operand's end, k past K and rows that a mask excludes are
// loads past the buffer's end, which bring zeros and touch no memory.
#pragma once

#include "lsso_device.h"
#include "lsso_values.h"

namespace lsso_hip {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void LdsVoid;

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

template <int T>
__device__ __forceinline__ f32x4 mfma_small(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (T == LSSO_HIP_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
}

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

// This wave's index, as the scalar that it is.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---------------------------------------------------------------------------
// The product for both operands in columns.  A stage is 32 k of whole 128-byte
// lines, in a ring of three: two are in flight while one is multiplied.
// Fragments come from transposed LDS reads (4 k x 16 columns per 16 lanes).
constexpr int kColumnsStageK = 32;
constexpr int kColumnsRing = 3;

// Stage of WIDTH columns, loaded by WAVES waves.
template <int WIDTH, int WAVES>
struct ColumnsStage {
    static constexpr int kBytes = WIDTH * kColumnsStageK * 2;
    static constexpr int kLoads = kBytes / 1024 / WAVES;       // per wave
    static constexpr int kPieces = WIDTH / 8;                  // 16-byte pieces of a line
    static constexpr int kLinesPerLoad = 64 / kPieces;
    static constexpr int kLinesPerRound = kLinesPerLoad * WAVES;
    static_assert(kLoads >= 1, "every wave loads");
    // Group g of 16 columns of line k lies at g ^ swizzle(k), so that the four
    // lines of a transposed read, and the two groups beside each other, fall on
    // different banks.
    __device__ static __forceinline__ int swizzle(int k) { return ((k & 1) != 0 ? 3 : 0) ^ ((k & 2) != 0 ? 5 : 0); }
    // Line of this lane's first load (kLinesPerRound further for each one after
    // it) and its first element of that line.
    __device__ static __forceinline__ int load_line(int wave, int lane) {
        return kLinesPerLoad * wave + lane / kPieces;
    }
    __device__ static __forceinline__ int load_element(int wave, int lane) {
        const int piece = lane % kPieces;
        return 16 * ((piece >> 1) ^ swizzle(load_line(wave, lane))) + 8 * (piece & 1);
    }
    // Byte in a stage of this lane's fragment of columns p0 .. p0 + 31 at a step.
    __device__ static __forceinline__ int fragment(int lane, int p0, int step) {
        const int k = (lane & 15) / 4 + 8 * (lane >> 5);
        const int group = p0 / 16 + ((lane >> 4) & 1);
        return 2 * WIDTH * (k + 16 * step) + 32 * (group ^ swizzle(k)) + 8 * (lane & 3);
    }
    __device__ static __forceinline__ u32x4 read(const char* at) {
        const u32x2 low = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at)));
        const u32x2 high =
            __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(at + 2 * WIDTH * 4)));
        return (u32x4){low[0], low[1], high[0], high[1]};
    }
};

// T: type code; MB x NB blocks of 32 x 32 per wave, WP x WQ waves.
template <int T_, int MB_, int NB_, int WP_, int WQ_>
struct ColumnsShape {
    static constexpr int T = T_;
    static constexpr int MB = MB_;
    static constexpr int NB = NB_;
    static constexpr int WP = WP_;
    static constexpr int WQ = WQ_;
    static constexpr int kWaves = WP * WQ;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int BP = 32 * MB * WP;
    static constexpr int BQ = 32 * NB * WQ;
    using PStage = ColumnsStage<BP, kWaves>;
    using QStage = ColumnsStage<BQ, kWaves>;
    static constexpr int kStageBytes = PStage::kBytes + QStage::kBytes;
    static constexpr int kLdsBytes = kColumnsRing * kStageBytes;
    static constexpr int kWaveBytes = kLdsBytes / kWaves;   // of the epilogue
    static constexpr int kLoads = PStage::kLoads + QStage::kLoads;
    __device__ static __forceinline__ int wave_p(int wave) { return 32 * MB * (wave % WP); }
    __device__ static __forceinline__ int wave_q(int wave) { return 32 * NB * (wave / WP); }
};

// Runs `stages` stages (at least one): issue(stage, s, j) starts load j of the
// kLoads per wave of stage s (which may lie past the last) into an LDS stage.
// The order is written down with scheduling barriers: left to itself the
// compiler moves the fragments' reads down to their MFMAs, to save registers
// that nothing else needs, and every MFMA then waits for LDS.
template <typename S, typename Issue>
__device__ __forceinline__ void run_columns_product(char* lds, int stages, f32x16 (&acc)[S::NB][S::MB], Issue issue) {
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
        const char* const stage = lds + buffer * S::kStageBytes;
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            qf[step][n] = S::QStage::read(stage + S::PStage::kBytes +
                                          S::QStage::fragment(lane, S::wave_q(wave) + 32 * n, step));
        }
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
            pf[step][m] = S::PStage::read(stage + S::PStage::fragment(lane, S::wave_p(wave) + 32 * m, step));
        }
    };
    // The MFMAs of a step; with the first one's the loads of a stage, spread out.
    const auto multiply = [&](int step, char* to, int s) {
        constexpr int kBlocks = S::MB * S::NB;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            if (step == 0) {
#pragma unroll
                for (int j = 0; j < S::kLoads; ++j) {
                    if (j * kBlocks / S::kLoads == i) {
                        issue(to, s, j);
                    }
                }
            }
            f32x16& c = acc[i % S::NB][i / S::NB];
            c = mfma_block<S::T>(qf[step][i % S::NB], pf[step][i / S::NB], c);
            if (step == 0) {
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto stage = [&](int buffer, int s) {
        read(buffer, 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(0, lds + (buffer + 2) % kColumnsRing * S::kStageBytes, s + 2);
        stage_barrier<S::kLoads>();   // the next stage has landed, this one is in registers
        read((buffer + 1) % kColumnsRing, 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply(1, nullptr, 0);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < S::kLoads; ++j) {
            issue(lds + i * S::kStageBytes, i, j);
        }
    }
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
// Steps over which a wave spreads its loads of a stage.  It issues in order, and
// all of them at once hold it until the address unit has taken them all.
// Two steps measured best of one to three (8,192 x 4,096 -> 4,096: 1,105, 1,121 and
// 1,110 TFLOP/s).
constexpr int kSpreadSteps = 2;

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

// Runs `tiles` tiles of `stages` stages each.  issue(stage, j) starts load j of the
// kLoads per wave of the next stage into an LDS stage, in order through all tiles
// and asked for two stages past the last; q_start(n) is the tile's first row of Q of this wave's block n;
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
    // The MFMAs of a step, and between them the loads whose turn it is: load j of
    // a stage goes before MFMA j * kSpread / kLoads, counted from the last step
    // of the stage before last through the first steps of the last one.
    constexpr int kBlocks = S::MB * S::NB;
    constexpr int kSpread = kSpreadSteps * kBlocks;
    const auto multiply = [&](int step, char* stage, int first) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
#pragma unroll
            for (int j = 0; j < S::kLoads; ++j) {
                if (j * kSpread / S::kLoads == first + i) {
                    issue(stage, j);
                }
            }
            f32x16& c = acc[i % S::NB][i / S::NB];
            c = mfma_block<S::T>(qf[step & 1][i % S::NB], pf[step & 1][i / S::NB], c);
            if (first < kSpread) {
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    int at = 0;   // LDS offset of this stage
    const auto stage = [&] {
        char* const here = lds + at;
        char* const other = lds + (at ^ S::kStageBytes);
        at ^= S::kStageBytes;
#pragma unroll
        for (int step = 0; step < kRowsSteps - 1; ++step) {
            read(here, step + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(step, other, (step + 1) * kBlocks);
        }
        stage_barrier<0>();   // the next stage has landed, and nobody reads this one any more
        read(other, 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply(kRowsSteps - 1, here, 0);
    };
#pragma unroll
    for (int j = 0; j < S::kLoads; ++j) {
        issue(lds, j);
    }
    // What the last step of a stage before the first would have issued.
    constexpr int kBegun = (S::kLoads + kSpreadSteps - 1) / kSpreadSteps;
#pragma unroll
    for (int j = 0; j < kBegun; ++j) {
        issue(lds + S::kStageBytes, j);
    }
    stage_barrier<kBegun>();
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

// A wave's exchange of 32 rows of BYTES (32, 64 or 128) through its own part of LDS,
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
        return BYTES == 128  ? (row & 7) ^ ((row >> 3) & 1)
               : BYTES == 64 ? ((row >> 1) & 3) ^ ((row >> 3) & 1)
                             : ((row >> 2) & 1) ^ ((row >> 3) & 1);
    }
    // V: 4, 8 or 16 bytes at `byte` of row lane % 32.
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
