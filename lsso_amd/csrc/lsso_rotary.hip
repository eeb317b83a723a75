// Rotary positions of a query and a key in one launch: the pair (x, x') of a
// token at position p becomes
//   m (x cos a - x' sin a, x sin a + x' cos a),   a = p f_j,
// with the pairs' partners next to each other or half of the rotated part
// apart; features past the rotated part are copied.  The gradient is the turn
// by -a.
//
// Angles are products in 64 bits, brought into one turn before they are rounded
// to 32: a position of a million times a frequency of 1 has no correct digit
// left of its cosine in 32 bits.  Of FP32 tensors the sines are taken in 64 bits too
// and rounded once (64 x 4,096 tokens of 4 + 4 heads of 64: 201 us, 5.3 TB/s, with
// either).
//
// Bound: HBM, one read and one write of each tensor.  A thread takes the same few
// features of every head of a token, so that each phase is made once, with the
// first heads' loads already on their way, and nothing passes through LDS.  (The
// phases of a tile of tokens made first, kept in LDS and read by all heads took 115
// us instead of 95 at 64 x 4,096 tokens of 4 + 4 heads of 64 in BF16: the loads
// waited for them and for two barriers.)

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;   // of a thread in flight
constexpr int64_t kMostGrid = 1 << 22;

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
// neighbours; V: features of an access, which divides what is turned (half of the
// rotated part, or all of it).
template <int T, bool HALF, int V>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
    using Element = typename Values<T>::Element;
    constexpr int kPhases = HALF ? V : V / 2;
    const int half = a.half;
    const int turned = HALF ? half / V : 2 * half / V;                             // units of a head that turn
    const int units = turned + (a.features - 2 * half + V - 1) / V;                // and that are copied
    const int64_t items = a.batch * a.length * units;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; item < items; item += step) {
        const int64_t row = quotient(item, units);
        const int unit = static_cast<int>(item - row * units);
        const int64_t batch = quotient(row, a.length);
        const int64_t token = row - batch * a.length;
        const bool turns = unit < turned;
        const int feature = unit * V + (HALF && !turns ? half : 0);
        const bool whole = turns || feature + V <= a.features;
        // The heads of both tensors in one row, of which this workgroup takes a part.
        const int heads0 = a.tensors[0].heads;
        const int heads = heads0 + (a.count > 1 ? a.tensors[1].heads : 0);
        const int first = static_cast<int>(blockIdx.y) * a.heads_each;
        const int last = first + a.heads_each < heads ? first + a.heads_each : heads;
        const auto from = [&](int head) {
            const RotaryTensor& t = a.tensors[head < heads0 ? 0 : 1];
            return static_cast<const Element*>(t.x) + batch * t.batch_stride + token * t.token_stride +
                   (head < heads0 ? head : head - heads0) * t.head_stride + feature;
        };
        const auto to = [&](int head) {
            const RotaryTensor& t = a.tensors[head < heads0 ? 0 : 1];
            return static_cast<Element*>(t.y) +
                   (row * t.heads + (head < heads0 ? head : head - heads0)) * a.features + feature;
        };
        if (!whole) {
            for (int head = first; head < last; ++head) {
                for (int i = 0; feature + i < a.features; ++i) {
                    to(head)[i] = from(head)[i];
                }
            }
            continue;
        }
        Raw<T, V> raw[kHeads];
        Raw<T, V> other[HALF ? kHeads : 1];
        const auto load = [&](int head0) {
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                if (head0 + k < last) {
                    const Element* at = from(head0 + k);
                    raw[k].load(at);
                    if constexpr (HALF) {
                        if (turns) {
                            other[k].load(at + half);
                        }
                    }
                }
            }
        };
        load(first);
        float cosine[kPhases];
        float sine[kPhases];
        if (turns) {
            const double position = position_at(a, batch, token);
            const double* frequencies = a.frequencies + (HALF ? feature : feature / 2);
#pragma unroll
            for (int i = 0; i < kPhases; ++i) {
                // In turns, so that the whole ones can be dropped.
                const double angle = position * (frequencies[i] * 0.15915494309189535);
                const double turn = 2.0 * (angle - rint(angle));
                if constexpr (T == LSSO_HIP_F32) {
                    // FP32 outputs show the rounding of the angle and of the function.
                    double s;
                    double c;
                    sincospi(turn, &s, &c);
                    cosine[i] = static_cast<float>(a.amplitude * c);
                    sine[i] = a.sign * static_cast<float>(a.amplitude * s);
                } else {
                    sincospif(static_cast<float>(turn), &sine[i], &cosine[i]);
                    cosine[i] *= a.amplitude;
                    sine[i] *= a.amplitude * a.sign;
                }
            }
        }
        for (int head0 = first; head0 < last; head0 += kHeads) {
            if (head0 != first) {
                load(head0);
            }
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                if (head0 + k >= last) {
                    break;
                }
                Element* at = to(head0 + k);
                float v[V];
                raw[k].values(v);
                if (!turns) {
                    store_values<T, V>(at, v);
                } else if constexpr (HALF) {
                    float first_half[V];
                    float second_half[V];
                    other[k].values(second_half);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        first_half[i] = v[i] * cosine[i] - second_half[i] * sine[i];
                        second_half[i] = v[i] * sine[i] + second_half[i] * cosine[i];
                    }
                    store_values<T, V>(at, first_half);
                    store_values<T, V>(at + half, second_half);
                } else {
                    float both[V];
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        both[i] = v[i] * cosine[i / 2] - v[i + 1] * sine[i / 2];
                        both[i + 1] = v[i] * sine[i / 2] + v[i + 1] * cosine[i / 2];
                    }
                    store_values<T, V>(at, both);
                }
            }
        }
    }
}

template <int T, bool HALF, int V>
void launch(RotaryArgs a, hipStream_t stream) {
    const int units = (HALF ? a.half : 2 * a.half) / V + (a.features - 2 * a.half + V - 1) / V;
    const int64_t items = a.batch * a.length * units;
    const int64_t blocks = (items + kThreads - 1) / kThreads;
    const int heads = a.tensors[0].heads + (a.count > 1 ? a.tensors[1].heads : 0);
    // All heads to a thread, unless that leaves compute units without two workgroups:
    // then fewer, whose phases are made more than once.
    int parts = 1;
    while (parts * kHeads < heads && blocks * parts < 512) {
        ++parts;
    }
    a.heads_each = (heads + parts - 1) / parts;
    parts = (heads + a.heads_each - 1) / a.heads_each;
    const dim3 grid(static_cast<unsigned>(blocks < kMostGrid ? blocks : kMostGrid), static_cast<unsigned>(parts));
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

hipError_t launch_rotary(const RotaryArgs& a, int dtype, int layout, hipStream_t stream) {
    if (a.batch * a.length == 0 || a.count == 0) {
        return hipSuccess;
    }
    switch (dtype) {
        case LSSO_HIP_F16: launch_layout<LSSO_HIP_F16>(a, layout, stream); break;
        case LSSO_HIP_BF16: launch_layout<LSSO_HIP_BF16>(a, layout, stream); break;
        default: launch_layout<LSSO_HIP_F32>(a, layout, stream); break;
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
