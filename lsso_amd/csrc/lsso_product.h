// Tiled 16-bit matrix product of the feed-forward kernels:
//   out[p][q] = sum over k of P[p, k] Q[q, k],  FP32 accumulation,
// for operands that lie in memory either along k ([p][k], "rows") or across it
// ([k][p], "columns"), so that x W^T, dy W and dy^T x are the same loop and no
// operand is ever transposed in memory.
//
// A workgroup of 4 waves (2 x 2) owns a BP x BQ tile, a wave MB x NB blocks of
// 32 x 32 on v_mfma_f32_32x32x16.  The operands' stages of 32 k go from memory
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
    // Byte of this lane's fragment of block b (32 p from p0) in a stage, first
    // k step; the second one is second_step() further.
    __device__ static __forceinline__ int fragment(int lane, int p0) {
        if constexpr (IN_ROWS) {
            const int p = p0 + (lane & 31);
            return 64 * p + 16 * ((lane >> 5) ^ row_swizzle(p));
        } else {
            const int k = (lane & 15) / 4 + 8 * (lane >> 5);
            const int group = p0 / 16 + ((lane >> 4) & 1);
            return 2 * WIDTH * k + 32 * (group ^ column_swizzle(k)) + 8 * (lane & 3);
        }
    }
    __device__ static __forceinline__ u32x4 read(const char* stage, int fragment_at, int step) {
        if constexpr (IN_ROWS) {
            // Step 1 takes pieces 2 and 3: slot bit 1 flips.
            return *reinterpret_cast<const u32x4*>(stage + (fragment_at ^ (32 * step)));
        } else {
            const char* at = stage + fragment_at + 2 * WIDTH * 16 * step;
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

template <int T_, bool P_ROWS_, bool Q_ROWS_, int MB_, int NB_>
struct ProductShape {
    static constexpr int T = T_;
    static constexpr bool P_ROWS = P_ROWS_;
    static constexpr bool Q_ROWS = Q_ROWS_;
    static constexpr int MB = MB_;
    static constexpr int NB = NB_;
    static constexpr int BP = 64 * MB;
    static constexpr int BQ = 64 * NB;
    using PLayout = StageLayout<BP, P_ROWS>;
    using QLayout = StageLayout<BQ, Q_ROWS>;
    static constexpr int kStageBytes = PLayout::kBytes + QLayout::kBytes;
    static constexpr int kLdsBytes = kRing * kStageBytes;
    static constexpr int kLoads = PLayout::kLoads + QLayout::kLoads;
};

// Runs `stages` stages: issue(buffer, s) starts the loads of stage s (which may
// lie past the last) into the LDS stage `buffer`, exactly kLoads per wave.
// q_start(nb) is the tile's first column of this wave's Q block nb.
template <typename S, typename Issue, typename QStart>
__device__ __forceinline__ void run_product(char* lds, int stages, f32x16 (&acc)[S::NB][S::MB], Issue issue,
                                            QStart q_start) {
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    int p_at[S::MB];
    int q_at[S::NB];
#pragma unroll
    for (int m = 0; m < S::MB; ++m) {
        p_at[m] = S::PLayout::fragment(lane, 32 * (S::MB * (wave & 1) + m));
    }
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
        q_at[n] = S::PLayout::kBytes + S::QLayout::fragment(lane, q_start(n));
    }
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
    const auto read = [&](const char* stage, int step) {
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            qf[step][n] = S::QLayout::read(stage, q_at[n], step);
        }
#pragma unroll
        for (int m = 0; m < S::MB; ++m) {
            pf[step][m] = S::PLayout::read(stage, p_at[m], step);
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
    issue(lds, 0);
    issue(lds + S::kStageBytes, 1);
    stage_barrier<S::kLoads>();
    read(lds, 0);
    int at = 0;   // this stage's buffer
    for (int s = 0; s < stages; ++s) {
        const int next = at == kRing - 1 ? 0 : at + 1;
        const int after = next == kRing - 1 ? 0 : next + 1;
        issue(lds + after * S::kStageBytes, s + 2);
        read(lds + at * S::kStageBytes, 1);
        multiply(0);
        stage_barrier<S::kLoads>();
        read(lds + next * S::kStageBytes, 0);
        multiply(1);
        at = next;
    }
    // The loads past the last stage still write their zeros: not into LDS that
    // another workgroup may hold by then.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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

}  // namespace lsso_hip
