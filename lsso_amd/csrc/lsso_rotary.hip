// Rotary positions of a query and a key in one launch: the pair (x, x') of a
// token at position p becomes
//   m (x cos a - x' sin a, x sin a + x' cos a),   a = p f_j,
// with the pairs' partners next to each other or half of the rotated part
// apart; features past the rotated part are copied.  The gradient is the turn
// by -a.
//
// Angles are products in 64 bits, brought into one turn before they are rounded
// to 32: a position of a million times a frequency of 1 has no correct digit
// left of its cosine in 32 bits.  That costs a few FP64 operations and a sine
// and cosine for each token and pair, so a workgroup makes them once for a tile
// of tokens, keeps them in LDS, and turns all heads of both tensors with them.
//
// Bound: HBM, one read and one write of each tensor.

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kThreads = 256;
constexpr int kTable = 2048;      // phases of a tile: 16 KB of LDS
constexpr int kMostTokens = 16;   // of a tile
constexpr int kRows = 4;          // rows of a thread in flight
constexpr int kMostTiles = 4096;  // of a grid; each workgroup takes every gridDim.x-th tile

// i / d for i d < 2^32, by magic = ceil(2^32 / d).
__device__ __forceinline__ uint32_t divide(uint32_t i, uint32_t magic) {
    return magic == 0 ? i : __umulhi(i, magic);   // 0: d is 1
}

__device__ double position_at(const RotaryArgs& a, int64_t batch, int64_t token) {
    const int64_t at = batch * a.position_batch_stride + token * a.position_token_stride;
    switch (a.position_type) {
        case LSSO_HIP_IDS_I32: return static_cast<const int32_t*>(a.positions)[at];
        case LSSO_HIP_IDS_I64: return static_cast<double>(static_cast<const int64_t*>(a.positions)[at]);
        case LSSO_HIP_IDS_F32: return static_cast<const float*>(a.positions)[at];
        case LSSO_HIP_IDS_F64: return static_cast<const double*>(a.positions)[at];
        default: return static_cast<double>(token);
    }
}

// T: type; HALF: the partner of feature j is feature j + half, else pairs are
// neighbours; V: features of an access, which divides what a lane turns at once
// (half of the rotated part, or all of it).
template <int T, bool HALF, int V>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
    using Element = typename Values<T>::Element;
    __shared__ float2 table[kTable];
    __shared__ double position[kMostTokens];
    __shared__ int64_t base[2][kMostTokens];
    const int tid = threadIdx.x;
    const int half = a.half;
    const int turned = HALF ? half / V : 2 * half / V;                       // units that turn
    const int copied = (a.features - 2 * half + V - 1) / V;                  // units that are copied
    const int units = turned + copied;
    const int64_t tokens = a.batch * a.length;
    const int64_t tiles = (tokens + a.tile - 1) / a.tile;
    const int lanes = 1 << a.lanes_shift;
    const int rows_at_once = kThreads >> a.lanes_shift;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t first = tile * a.tile;
        const int count = static_cast<int>(tokens - first < a.tile ? tokens - first : a.tile);
        __syncthreads();   // the last tile's readers are done
        if (tid < count) {
            const int64_t batch = (first + tid) / a.length;
            const int64_t token = first + tid - batch * a.length;
            position[tid] = position_at(a, batch, token);
            for (int w = 0; w < a.count; ++w) {
                base[w][tid] = batch * a.tensors[w].batch_stride + token * a.tensors[w].token_stride;
            }
        }
        __syncthreads();
        for (int i = tid; i < count * half; i += kThreads) {
            const int t = divide(i, a.half_magic);
            // In turns, so that the whole ones can be dropped.
            const double turns = position[t] * (a.frequencies[i - t * half] * 0.15915494309189535);
            float sine;
            float cosine;
            sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
            table[i] = make_float2(a.amplitude * cosine, a.amplitude * a.sign * sine);
        }
        __syncthreads();
        for (int w = 0; w < a.count; ++w) {
            const RotaryTensor& tensor = a.tensors[w];
            const Element* x = static_cast<const Element*>(tensor.x);
            Element* y = static_cast<Element*>(tensor.y);
            const int rows = count * tensor.heads;
            for (int row0 = tid >> a.lanes_shift; row0 < rows; row0 += kRows * rows_at_once) {
                for (int u = tid & (lanes - 1); u < units; u += lanes) {
                    const bool turns = u < turned;
                    const int feature = u * V + (HALF && !turns ? half : 0);
                    const bool whole = turns || feature + V <= a.features;
                    float v[kRows][V];
                    float other[kRows][HALF ? V : 1];
#pragma unroll
                    for (int k = 0; k < kRows; ++k) {
                        const int row = row0 + k * rows_at_once;
                        if (row < rows) {
                            const int t = divide(row, tensor.head_magic);
                            const Element* at =
                                x + base[w][t] + (row - t * tensor.heads) * tensor.head_stride + feature;
                            if (whole) {
                                load_values<T, V>(at, v[k]);
                                if constexpr (HALF) {
                                    if (turns) {
                                        load_values<T, V>(at + half, other[k]);
                                    }
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < V; ++i) {
                                    v[k][i] = feature + i < a.features ? Values<T>::load(at + i) : 0.0f;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kRows; ++k) {
                        const int row = row0 + k * rows_at_once;
                        if (row >= rows) {
                            continue;
                        }
                        const int t = divide(row, tensor.head_magic);
                        Element* to = y + (first * tensor.heads + row) * a.features + feature;
                        if (!turns) {
                            if (whole) {
                                store_values<T, V>(to, v[k]);
                            } else {
#pragma unroll
                                for (int i = 0; i < V; ++i) {
                                    if (feature + i < a.features) {
                                        Values<T>::store(to + i, v[k][i]);
                                    }
                                }
                            }
                        } else if constexpr (HALF) {
                            const float2* phase = table + t * half + feature;
                            float second[V];
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                const float2 p = phase[i];
                                const float value = v[k][i] * p.x - other[k][i] * p.y;
                                second[i] = v[k][i] * p.y + other[k][i] * p.x;
                                v[k][i] = value;
                            }
                            store_values<T, V>(to, v[k]);
                            store_values<T, V>(to + half, second);
                        } else {
                            const float2* phase = table + t * half + feature / 2;
#pragma unroll
                            for (int i = 0; i < V; i += 2) {
                                const float2 p = phase[i / 2];
                                const float value = v[k][i] * p.x - v[k][i + 1] * p.y;
                                v[k][i + 1] = v[k][i] * p.y + v[k][i + 1] * p.x;
                                v[k][i] = value;
                            }
                            store_values<T, V>(to, v[k]);
                        }
                    }
                }
            }
        }
    }
}

uint32_t magic(uint32_t d) { return d == 1 ? 0 : static_cast<uint32_t>(((uint64_t{1} << 32) + d - 1) / d); }

template <int T, bool HALF, int V>
void launch(RotaryArgs a, hipStream_t stream) {
    const int units = (HALF ? a.half : 2 * a.half) / V + (a.features - 2 * a.half + V - 1) / V;
    a.lanes_shift = 0;
    while ((1 << a.lanes_shift) < units && (1 << a.lanes_shift) < kThreads) {
        ++a.lanes_shift;
    }
    const int64_t tokens = a.batch * a.length;
    // A tile as large as its phases fit, but no larger than leaves eight tiles
    // to a compute unit.
    int64_t tile = (tokens + 2047) / 2048;
    const int64_t most = a.half > 0 ? kTable / a.half : kMostTokens;
    tile = tile > most ? most : tile;
    a.tile = static_cast<int>(tile > kMostTokens ? kMostTokens : tile);
    const int64_t tiles = (tokens + a.tile - 1) / a.tile;
    const unsigned grid = static_cast<unsigned>(tiles < kMostTiles ? tiles : kMostTiles);
    rotary_kernel<T, HALF, V><<<grid, kThreads, 0, stream>>>(a);
}

template <int T, bool HALF>
void launch_vector(const RotaryArgs& a, hipStream_t stream) {
    const int length = HALF ? a.half : 2 * a.half;
    if (length % 8 == 0) {
        launch<T, HALF, 8>(a, stream);
    } else if (length % 4 == 0) {
        launch<T, HALF, 4>(a, stream);
    } else if (length % 2 == 0) {
        launch<T, HALF, 2>(a, stream);
    } else if constexpr (HALF) {
        launch<T, true, 1>(a, stream);
    }
}

template <int T>
void launch_layout(const RotaryArgs& a, int layout, hipStream_t stream) {
    if (layout == LSSO_HIP_ROTARY_HALF) {
        launch_vector<T, true>(a, stream);
    } else {
        launch_vector<T, false>(a, stream);
    }
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& args, int dtype, int layout, hipStream_t stream) {
    RotaryArgs a = args;
    if (a.batch * a.length == 0 || a.count == 0) {
        return hipSuccess;
    }
    a.half_magic = magic(static_cast<uint32_t>(a.half));
    for (int w = 0; w < a.count; ++w) {
        a.tensors[w].head_magic = magic(static_cast<uint32_t>(a.tensors[w].heads));
    }
    switch (dtype) {
        case LSSO_HIP_F16: launch_layout<LSSO_HIP_F16>(a, layout, stream); break;
        case LSSO_HIP_BF16: launch_layout<LSSO_HIP_BF16>(a, layout, stream); break;
        default: launch_layout<LSSO_HIP_F32>(a, layout, stream); break;
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
