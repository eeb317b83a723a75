// Group norm with an activation, channels last:
//   y = act(z),  z = w_c xhat + b_c,  xhat = (x - mean) rstd,
// mean and rstd = 1 / sqrt(var + eps) over the n = tokens x channels of a group
// of one sample.  With dz = dy act'(z) and dn = w_c dz,
//   dx = rstd (dn - (sum of dn + xhat sum of dn xhat) / n),
//   dw_c = sum of dz xhat,  db_c = sum of dz.
// Rows that the mask excludes count nowhere and come out as zeros.
//
// Bound: HBM.  Two forms:
//
// Every token a sample of its own (heads of a token, or a layer norm): a group's
// channels are read once, by a team of lanes (up to a wave, or the workgroup) that
// keeps them in registers, sums them over its lanes, and writes y.  Teams of neighbouring groups sit next to
// each other, so that a wave reads whole lines.  Each lane stays with its
// channels while its workgroup walks over the rows, which leaves dw and db in
// its registers to the end.
//
// Longer samples: a channels-last row holds all groups, and a group's share of it
// may be 16 bytes, so a workgroup takes whole rows of a range of tokens and each
// thread keeps to a few channels.  One launch leaves mean and squared deviations of
// each group in each range (of each channel, where a workgroup has not all of them),
// one joins them to the groups' statistics, one applies them: x is read again, from
// the last-level cache where it fits.  The backward does the same with its two sums.
//
// 64 x 4,096 tokens of 4 groups of 64 in BF16, each token by itself: 58 us forward
// (4.6 TB/s) and 89 backward (4.5).  32 samples of 56 x 56 x 256 in FP16: 19 + 23 us
// and, backward, 34 + 33, with joins of 4 to 5 us.
//
// Variances come from deviations: of four rows at a time from their own mean,
// joined to what is known so far by the rule for two parts (Chan, Golub and
// LeVeque, 1979).  Sums of squares lose a variance that is small beside the
// mean's square, and a fixed pivot is worth as little as its outliers let it.

#include "lsso_activation.h"
#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kThreads = 256;
constexpr int kBlockRows = 4;        // rows of a thread in flight
constexpr int kTeamMost = 4;         // most pieces of a lane of a wave's team
constexpr int kLaneMost = 32;        // most values of a lane
constexpr int64_t kMostGrid = 1 << 20;

// act(z) and act'(z) of one kind.  FP32 outputs show more than the fast forms hold
// (1e-5 of the sigmoid's and the distribution function's own value).
template <int T, int KIND, bool SLOPE>
__device__ __forceinline__ void act(float z, float& value, float& slope) {
    if constexpr (KIND == 0) {
        value = z;
        slope = 1.0f;
    } else if constexpr (T != LSSO_HIP_F32) {
        activation<SLOPE>(KIND, z, value, slope);
    } else if constexpr (KIND == LSSO_HIP_SILU) {
        const float s = 1.0f / (1.0f + expf(-z));
        value = z * s;
        slope = SLOPE ? s + value * (1.0f - s) : 0.0f;
    } else {
        const float phi = normcdff(z);
        value = z * phi;
        slope = SLOPE ? phi + 0.3989422804f * z * expf(-0.5f * z * z) : 0.0f;
    }
}

template <int KIND>
struct Kind {
    static constexpr int value = KIND;
};
// f of the activation's kind: one branch for all of a row's elements.
template <typename F>
__device__ __forceinline__ void by_kind(int kind, F f) {
    if (kind == 0) {
        f(Kind<0>{});
    } else if (kind == LSSO_HIP_SILU) {
        f(Kind<LSSO_HIP_SILU>{});
    } else {
        f(Kind<LSSO_HIP_GELU>{});
    }
}

__device__ __forceinline__ float parameter(const void* values, int type, int c, float absent) {
    if (values == nullptr) {
        return absent;
    }
    switch (type) {
        case LSSO_HIP_F16: return f16_bits_to_float(static_cast<const uint16_t*>(values)[c]);
        case LSSO_HIP_BF16: return bf16_bits_to_float(static_cast<const uint16_t*>(values)[c]);
        default: return static_cast<const float*>(values)[c];
    }
}

__device__ __forceinline__ void store_parameter(void* values, int type, int c, float v) {
    switch (type) {
        case LSSO_HIP_F16: static_cast<uint16_t*>(values)[c] = to_f16_bits(v); break;
        case LSSO_HIP_BF16: static_cast<uint16_t*>(values)[c] = to_bf16_bits(v); break;
        default: static_cast<float*>(values)[c] = v; break;
    }
}

// Sum over the team's lanes, a power of two of neighbours, in all of them: up to 16
// by moves within a row of lanes, which wait for no LDS.
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
    return __builtin_bit_cast(float,
                              __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
__device__ __forceinline__ float team_sum(float v, int lanes) {
    if (lanes > 1) {
        v += moved<0xb1>(v);    // quad_perm 1, 0, 3, 2
    }
    if (lanes > 2) {
        v += moved<0x4e>(v);    // quad_perm 2, 3, 0, 1
    }
    if (lanes > 4) {
        v += moved<0x141>(v);   // row_half_mirror: of the other four lanes, which hold one value
    }
    if (lanes > 8) {
        v += moved<0x140>(v);   // row_mirror: of the other eight
    }
    if (lanes > 16) {
        v += __shfl_xor(v, 16);
    }
    if (lanes > 32) {
        v += __shfl_xor(v, 32);
    }
    return v;
}

// Teams of a workgroup: `at_once` rows of `across` groups.
struct Teams {
    int lane;       // of the team
    int group;
    int row;
    int at_once;
    int across;
    bool active;
    __device__ __forceinline__ Teams(const GroupNormArgs& a) {
        const int teams = kThreads / a.team;
        across = 1;
        while (across < a.groups && across < teams) {
            across *= 2;
        }
        at_once = teams / across;
        const int team = static_cast<int>(threadIdx.x) / a.team;
        lane = static_cast<int>(threadIdx.x) % a.team;
        group = static_cast<int>(blockIdx.y) * across + team % across;
        row = team / across;
        active = group < a.groups;
    }
};

// T: type; V: channels of a piece; K: pieces of a lane; BACKWARD: dx and the
// partials of dw and db instead of y.
template <int T, int V, int K, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void team_norm_kernel(GroupNormArgs a) {
    using Element = typename Values<T>::Element;
    const Teams t(a);
    const int size = a.channels / a.groups;
    const int pieces = size / V;
    // Of FP32 divided: the reciprocal's own rounding shows.
    const float count = static_cast<float>(size);
    const float share = 1.0f / count;
    // A team of the whole workgroup passes its waves' sums through LDS, in two places by
    // turns: whoever writes one again has met all its readers at the other's barrier.
    __shared__ float waves[2][kThreads / 64];
    int turn = 0;
    const auto mean_of = [&](float sum) {
        if (a.team <= 64) {   // uniform
            sum = team_sum(sum, a.team);
        } else {
            sum = team_sum(sum, 64);
            if ((threadIdx.x & 63) == 0) {
                waves[turn][threadIdx.x >> 6] = sum;
            }
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kThreads / 64; ++i) {
                sum += waves[turn][i];
            }
            turn ^= 1;
        }
        return T == LSSO_HIP_F32 ? sum / count : sum * share;
    };
    const int channel0 = (t.active ? t.group : 0) * size;
    float w[K][V];
    float b[K][V];
    float grad_w[BACKWARD ? K : 1][V];
    float grad_b[BACKWARD ? K : 1][V];
    bool mine[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int piece = t.lane + a.team * k;
        mine[k] = t.active && piece < pieces;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[k][i] = mine[k] ? parameter(a.weight, a.parameter_type, channel0 + piece * V + i, 1.0f) : 0.0f;
            b[k][i] = mine[k] ? parameter(a.bias, a.parameter_type, channel0 + piece * V + i, 0.0f) : 0.0f;
            if constexpr (BACKWARD) {
                grad_w[k][i] = 0.0f;
                grad_b[k][i] = 0.0f;
            }
        }
    }
    // Rows of a team in flight: as many as hold 32 values of x.
    constexpr int kFlight = K * V <= 8 ? (BACKWARD ? 2 : 4) : (K * V <= 16 ? 2 : 1);
    const int64_t step = static_cast<int64_t>(gridDim.x) * t.at_once;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * t.at_once; row0 < a.samples; row0 += kFlight * step) {
        bool inside[kFlight];
        bool kept[kFlight];
        int64_t at[kFlight];
        Raw<T, V> raw_x[kFlight][K];
        Raw<T, V> raw_dy[kFlight][BACKWARD ? K : 1];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const int64_t row = row0 + t.row + f * step;
            inside[f] = row < a.samples;
            kept[f] = inside[f] && (a.row_mask == nullptr || a.row_mask[row] != 0);
            at[f] = (inside[f] ? row : 0) * a.channels + channel0;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int piece = t.lane + a.team * k;
                raw_x[f][k].clear();
                if (mine[k] && kept[f]) {
                    raw_x[f][k].load(static_cast<const Element*>(a.x) + at[f] + piece * V);
                }
                if constexpr (BACKWARD) {
                    raw_dy[f][k].clear();
                    if (mine[k] && kept[f]) {
                        raw_dy[f][k].load(static_cast<const Element*>(a.dy) + at[f] + piece * V);
                    }
                }
            }
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            float x[K][V];
            float dy[BACKWARD ? K : 1][V];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                raw_x[f][k].values(x[k]);
                if constexpr (BACKWARD) {
                    raw_dy[f][k].values(dy[k]);
                }
            }
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sum += x[k][i];
                }
            }
            const float mean = mean_of(sum);
            float squares = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[k][i] = mine[k] ? x[k][i] - mean : 0.0f;
                    squares += x[k][i] * x[k][i];
                }
            }
            const float rstd = 1.0f / sqrtf(mean_of(squares) + a.eps);
            if constexpr (!BACKWARD) {
                by_kind(a.activation, [&](auto kind) {
#pragma unroll
                    for (int k = 0; k < K; ++k) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            float y;
                            float slope;
                            act<T, decltype(kind)::value, false>(x[k][i] * rstd * w[k][i] + b[k][i], y, slope);
                            x[k][i] = kept[f] ? y : 0.0f;
                        }
                    }
                });
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (mine[k] && inside[f]) {
                        store_values<T, V>(static_cast<Element*>(a.y) + at[f] + (t.lane + a.team * k) * V, x[k]);
                    }
                }
            } else {
                float first = 0.0f;
                float second = 0.0f;
                by_kind(a.activation, [&](auto kind) {
#pragma unroll
                    for (int k = 0; k < K; ++k) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            x[k][i] *= rstd;
                            float value;
                            float slope;
                            act<T, decltype(kind)::value, true>(x[k][i] * w[k][i] + b[k][i], value, slope);
                            // A row that is left out has no part in any sum.
                            const float dz = kept[f] ? dy[k][i] * slope : 0.0f;
                            const float normal = kept[f] ? x[k][i] : 0.0f;
                            grad_b[k][i] += dz;
                            grad_w[k][i] += dz * normal;
                            dy[k][i] = dz * w[k][i];
                            first += dy[k][i];
                            second += dy[k][i] * normal;
                        }
                    }
                });
                first = mean_of(first);
                second = mean_of(second);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    float dx[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        dx[i] = kept[f] ? rstd * (dy[k][i] - (first + x[k][i] * second)) : 0.0f;
                    }
                    if (a.dx != nullptr && mine[k] && inside[f]) {
                        store_values<T, V>(static_cast<Element*>(a.dx) + at[f] + (t.lane + a.team * k) * V, dx);
                    }
                }
            }
        }
    }
    if constexpr (BACKWARD) {
        // The rows' teams of a group, one after the other: partials [blocks][dw, db][channels].
        __shared__ float shared[kThreads][K * V + 1];
        float* out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * a.channels;
        const int stride = t.across * a.team;   // threads of one row
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    shared[threadIdx.x][k * V + i] = part == 0 ? grad_w[k][i] : grad_b[k][i];
                }
            }
            __syncthreads();
            if (t.row == 0) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float total = 0.0f;
                        for (int r = 0; r < t.at_once; ++r) {
                            total += shared[threadIdx.x + r * stride][k * V + i];
                        }
                        if (mine[k]) {
                            out[part * a.channels + channel0 + (t.lane + a.team * k) * V + i] = total;
                        }
                    }
                }
            }
        }
    }
}

// The part of a workgroup of the kernels over splits: a thread keeps to one
// piece of V channels and takes every at_once-th row of the split.
template <int V>
struct Columns {
    int wide;        // pieces of the workgroup's channels
    int at_once;
    int channel;
    int row;
    bool active;
    __device__ __forceinline__ Columns(const GroupNormArgs& a) {
        const int pieces = a.channels / V;
        const int first = static_cast<int>(blockIdx.y) * kThreads;
        wide = pieces - first < kThreads ? pieces - first : kThreads;
        at_once = kThreads / wide;
        row = static_cast<int>(threadIdx.x) / wide;
        channel = (first + static_cast<int>(threadIdx.x) % wide) * V;
        active = row < at_once;
    }
};

// A split's partials: the rows that count, two values of each group (by_group: a
// workgroup has all channels) or of each channel, and in the backward two of each
// channel in front of them.
struct Partials {
    bool by_group;
    int columns;       // of the joined values: groups or channels
    int unit;          // channels of a column
    int64_t joined;    // where they begin
    int64_t pitch;
    __host__ __device__ Partials(const GroupNormArgs& a, bool backward) {
        by_group = a.channels / a.vector <= kThreads;
        columns = by_group ? a.groups : a.channels;
        unit = by_group ? a.channels / a.groups : 1;
        joined = 1 + (backward && by_group ? 2 * static_cast<int64_t>(a.channels) : 0);
        pitch = joined + 2 * static_cast<int64_t>(columns);
    }
};

// From values of each channel, in LDS, those of each group, by a team of lanes:
// f(group, its first channel, channels, lane of the team, lanes of the team).
template <typename F>
__device__ __forceinline__ void over_groups(const GroupNormArgs& a, F f) {
    const int size = a.channels / a.groups;
    int team = 1;
    while (team < 64 && team < size) {
        team *= 2;
    }
    for (int group = static_cast<int>(threadIdx.x) / team; group < a.groups; group += kThreads / team) {
        f(group, group * size, size, static_cast<int>(threadIdx.x) & (team - 1), team);
    }
}

// Rows at, at + step, ... (kBlockRows of them) of a thread: loads, and which count.
template <int T, int V>
__device__ __forceinline__ void load_rows(const void* from, const GroupNormArgs& a, int64_t sample, int64_t at, int step,
                                          int64_t end, int channel, Raw<T, V> (&v)[kBlockRows],
                                          bool (&kept)[kBlockRows]) {
    using Element = typename Values<T>::Element;
#pragma unroll
    for (int r = 0; r < kBlockRows; ++r) {
        const int64_t row = at + static_cast<int64_t>(r) * step;
        kept[r] = row < end && (a.row_mask == nullptr || a.row_mask[sample * a.length + row] != 0);
        v[r].clear();
        if (kept[r]) {
            v[r].load(static_cast<const Element*>(from) + (sample * a.length + row) * a.channels + channel);
        }
    }
}

// Mean and squared deviations of each channel over a split's rows.
template <int T, int V>
__global__ __launch_bounds__(kThreads) void norm_statistics_kernel(GroupNormArgs a) {
    __shared__ float shared[kThreads][2 * V + 1];
    __shared__ float rows[kThreads];
    const Columns<V> c(a);
    const Partials layout(a, false);
    const int64_t items = a.samples * a.splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = quotient(item, a.splits);
        const int64_t begin = (item - sample * a.splits) * a.split_rows;
        const int64_t end = begin + a.split_rows < a.length ? begin + a.split_rows : a.length;
        float count = 0.0f;
        float mean[V];
        float squares[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            mean[i] = 0.0f;
            squares[i] = 0.0f;
        }
        if (c.active) {
            for (int64_t at = begin + c.row; at < end; at += kBlockRows * c.at_once) {
                Raw<T, V> raw[kBlockRows];
                bool kept[kBlockRows];
                load_rows<T, V>(a.x, a, sample, at, c.at_once, end, c.channel, raw, kept);
                float v[kBlockRows][V];
                float some = 0.0f;
#pragma unroll
                for (int r = 0; r < kBlockRows; ++r) {
                    raw[r].values(v[r]);
                }
#pragma unroll
                for (int r = 0; r < kBlockRows; ++r) {
                    some += kept[r] ? 1.0f : 0.0f;
                }
                if (some > 0.0f) {
                    const float share = 1.0f / some;
                    const float all = count + some;
                    const float weight = some / all;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < kBlockRows; ++r) {
                            sum += v[r][i];
                        }
                        const float middle = sum * share;
                        float deviations = 0.0f;
#pragma unroll
                        for (int r = 0; r < kBlockRows; ++r) {
                            const float d = kept[r] ? v[r][i] - middle : 0.0f;
                            deviations += d * d;
                        }
                        const float apart = middle - mean[i];
                        squares[i] += deviations + apart * apart * (count * weight);
                        mean[i] += apart * weight;
                    }
                    count = all;
                }
            }
        }
        __syncthreads();   // the last item's readers are done
#pragma unroll
        for (int i = 0; i < V; ++i) {
            shared[threadIdx.x][i] = mean[i];
            shared[threadIdx.x][V + i] = squares[i];
        }
        rows[threadIdx.x] = count;
        __syncthreads();
        float* out = a.partials + item * layout.pitch;
        float kept_rows = 0.0f;
        for (int r = 0; r < c.at_once; ++r) {
            kept_rows += rows[r * c.wide];
        }
        if (blockIdx.y == 0 && threadIdx.x == 0) {
            out[0] = kept_rows;
        }
        for (int j = threadIdx.x; j < c.wide * V; j += kThreads) {
            const int thread = j / V;
            const int i = j - thread * V;
            // Two sums that wait for nobody: a merge of two at a time is a chain of divisions.
            const float pivot = shared[thread][i];
            float apart = 0.0f;
            for (int r = 0; r < c.at_once; ++r) {
                apart += rows[r * c.wide] * (shared[thread + r * c.wide][i] - pivot);
            }
            const float m = kept_rows > 0.0f ? pivot + apart / kept_rows : 0.0f;
            float s = 0.0f;
            for (int r = 0; r < c.at_once; ++r) {
                const float off = shared[thread + r * c.wide][i] - m;
                s += shared[thread + r * c.wide][V + i] + rows[r * c.wide] * off * off;
            }
            if (layout.by_group) {
                shared[thread][i] = m;
                shared[thread][V + i] = s;
            } else {
                const int channel = (static_cast<int>(blockIdx.y) * kThreads) * V + j;
                out[layout.joined + channel] = m;
                out[layout.joined + layout.columns + channel] = s;
            }
        }
        if (layout.by_group) {   // the channels have as many rows each
            __syncthreads();
            over_groups(a, [&](int group, int channel0, int size, int lane, int team) {
                float sum = 0.0f;
                for (int k = lane; k < size; k += team) {
                    sum += shared[(channel0 + k) / V][(channel0 + k) % V];
                }
                const float middle = team_sum(sum, team) / static_cast<float>(size);
                float deviations = 0.0f;
                for (int k = lane; k < size; k += team) {
                    const float* of = &shared[(channel0 + k) / V][(channel0 + k) % V];
                    const float apart = of[0] - middle;
                    deviations += of[V] + kept_rows * apart * apart;
                }
                deviations = team_sum(deviations, team);
                if (lane == 0) {
                    out[layout.joined + group] = middle;
                    out[layout.joined + layout.columns + group] = deviations;
                }
            });
        }
    }
}

// A few workgroups join what many left, so that each has many loads to wait for.
constexpr int kJoinThreads = 1024;

// Threads of a join, about four values each: 1,024 of them join 256 values in 8.9 us,
// 64 in 4.2, since a sum waits for all waves.
int join_threads(int64_t values) {
    int threads = 64;
    while (threads < kJoinThreads && threads * 4 < values) {
        threads *= 2;
    }
    return threads;
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = team_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        scratch[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    float total = 0.0f;
    for (unsigned i = 0; i < blockDim.x / 64; ++i) {
        total += scratch[i];
    }
    return total;
}

// f(partials of the split, column) of all splits of a sample and the `size` columns
// from channel0 on, dealt to the threads.
template <typename F>
__device__ __forceinline__ void over_splits(const GroupNormArgs& a, const float* part, int64_t pitch, int channel0,
                                            int size, F f) {
    int64_t split = static_cast<int>(threadIdx.x) / size;
    int channel = static_cast<int>(threadIdx.x) % size;
    const int splits = static_cast<int>(blockDim.x) / size;
    const int channels = static_cast<int>(blockDim.x) % size;
#pragma unroll 4
    for (; split < a.splits; split += splits) {
        f(part + split * pitch, channel0 + channel);
        channel += channels;
        if (channel >= size) {
            channel -= size;
            ++split;
        }
    }
}

// A group's statistics from its splits.
__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(GroupNormArgs a) {
    __shared__ float scratch[kJoinThreads / 64];
    const Partials layout(a, false);
    const int size = layout.columns / a.groups;
    const int64_t items = a.samples * a.groups;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = quotient(item, a.groups);
        const int column0 = static_cast<int>(item - sample * a.groups) * size;
        const float* part = a.partials + sample * a.splits * layout.pitch;
        float n = 0.0f;
        float sum = 0.0f;
        over_splits(a, part, layout.pitch, column0, size, [&](const float* of, int column) {
            const float some = of[0] * static_cast<float>(layout.unit);
            n += some;
            sum += some > 0.0f ? some * of[layout.joined + column] : 0.0f;
        });
        n = block_sum(n, scratch);
        sum = block_sum(sum, scratch);
        const float mean = n > 0.0f ? sum / n : 0.0f;
        float squares = 0.0f;
        over_splits(a, part, layout.pitch, column0, size, [&](const float* of, int column) {
            const float some = of[0] * static_cast<float>(layout.unit);
            const float apart = some > 0.0f ? of[layout.joined + column] - mean : 0.0f;
            squares += some > 0.0f ? of[layout.joined + layout.columns + column] + some * apart * apart : 0.0f;
        });
        squares = block_sum(squares, scratch);
        if (threadIdx.x == 0) {
            a.statistics[2 * item] = mean;
            a.statistics[2 * item + 1] = n > 0.0f ? 1.0f / sqrtf(squares / n + a.eps) : 0.0f;
        }
    }
}

// A thread's channels: w, b, and the statistics of their groups.
template <int V>
struct ChannelValues {
    float w[V];
    float b[V];
    float mean[V];
    float rstd[V];
    __device__ __forceinline__ void parameters(const GroupNormArgs& a, int channel) {
        if (a.parameter_type == LSSO_HIP_F32 && a.weight != nullptr && a.bias != nullptr) {   // uniform
            load_values<LSSO_HIP_F32, V>(static_cast<const float*>(a.weight) + channel, w);
            load_values<LSSO_HIP_F32, V>(static_cast<const float*>(a.bias) + channel, b);
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = parameter(a.weight, a.parameter_type, channel + i, 1.0f);
            b[i] = parameter(a.bias, a.parameter_type, channel + i, 0.0f);
        }
    }
    // Two values of each group, to the channels of each.
    __device__ __forceinline__ static void spread(const GroupNormArgs& a, const float* from, int64_t sample, int channel,
                                                  float (&first)[V], float (&second)[V]) {
        const uint32_t size = static_cast<uint32_t>(a.channels) / static_cast<uint32_t>(a.groups);
        const float* groups = from + 2 * sample * a.groups;
        if (size % V == 0) {   // uniform: the channels are of one group
            const uint32_t group = static_cast<uint32_t>(channel) / size;
            const float one = groups[2 * group];
            const float two = groups[2 * group + 1];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                first[i] = one;
                second[i] = two;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t group = static_cast<uint32_t>(channel + i) / size;
            first[i] = groups[2 * group];
            second[i] = groups[2 * group + 1];
        }
    }
    __device__ __forceinline__ void of_sample(const GroupNormArgs& a, int64_t sample, int channel) {
        spread(a, a.statistics, sample, channel, mean, rstd);
    }
};

template <int T, int V>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(GroupNormArgs a) {
    using Element = typename Values<T>::Element;
    const Columns<V> c(a);
    if (!c.active) {
        return;   // no barrier follows
    }
    ChannelValues<V> channel;
    channel.parameters(a, c.channel);
    const int64_t items = a.samples * a.splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = quotient(item, a.splits);
        const int64_t begin = (item - sample * a.splits) * a.split_rows;
        const int64_t end = begin + a.split_rows < a.length ? begin + a.split_rows : a.length;
        channel.of_sample(a, sample, c.channel);
        for (int64_t at = begin + c.row; at < end; at += kBlockRows * c.at_once) {
            Raw<T, V> raw[kBlockRows];
            bool kept[kBlockRows];
            load_rows<T, V>(a.x, a, sample, at, c.at_once, end, c.channel, raw, kept);
#pragma unroll
            for (int r = 0; r < kBlockRows; ++r) {
                float v[V];
                raw[r].values(v);
                by_kind(a.activation, [&](auto kind) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float slope;
                        float y;
                        act<T, decltype(kind)::value, false>(
                            (v[i] - channel.mean[i]) * channel.rstd[i] * channel.w[i] + channel.b[i], y, slope);
                        v[i] = kept[r] ? y : 0.0f;
                    }
                });
                const int64_t row = at + static_cast<int64_t>(r) * c.at_once;
                if (row < end) {
                    store_values<T, V>(
                        static_cast<Element*>(a.y) + (sample * a.length + row) * a.channels + c.channel, v);
                }
            }
        }
    }
}

// DX: dx, from the groups' sums; else the sums of dz xhat and dz of each channel
// over a split's rows.
template <int T, int V, bool DX>
__global__ __launch_bounds__(kThreads) void norm_grad_kernel(GroupNormArgs a) {
    using Element = typename Values<T>::Element;
    __shared__ float shared[DX ? 1 : kThreads][2 * V + 1];
    __shared__ float rows[DX ? 1 : kThreads];
    const Columns<V> c(a);
    const Partials layout(a, true);
    ChannelValues<V> channel;
    if (c.active) {
        channel.parameters(a, c.channel);
    }
    const int64_t items = a.samples * a.splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = quotient(item, a.splits);
        const int64_t begin = (item - sample * a.splits) * a.split_rows;
        const int64_t end = begin + a.split_rows < a.length ? begin + a.split_rows : a.length;
        float first[V];    // DX: the group's mean of dn, else this channel's sum of dz
        float second[V];   // the same with xhat
        float count = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            first[i] = 0.0f;
            second[i] = 0.0f;
        }
        if (c.active) {
            channel.of_sample(a, sample, c.channel);
            if constexpr (DX) {
                ChannelValues<V>::spread(a, a.sums, sample, c.channel, first, second);
            }
            for (int64_t at = begin + c.row; at < end; at += kBlockRows * c.at_once) {
                Raw<T, V> raw_x[kBlockRows];
                Raw<T, V> raw_dy[kBlockRows];
                bool kept[kBlockRows];
                load_rows<T, V>(a.x, a, sample, at, c.at_once, end, c.channel, raw_x, kept);
                load_rows<T, V>(a.dy, a, sample, at, c.at_once, end, c.channel, raw_dy, kept);
#pragma unroll
                for (int r = 0; r < kBlockRows; ++r) {
                    count += kept[r] ? 1.0f : 0.0f;
                    float x[V];
                    float dy[V];
                    raw_x[r].values(x);
                    raw_dy[r].values(dy);
                    by_kind(a.activation, [&](auto kind) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float normal = kept[r] ? (x[i] - channel.mean[i]) * channel.rstd[i] : 0.0f;
                            float value;
                            float slope;
                            act<T, decltype(kind)::value, true>(normal * channel.w[i] + channel.b[i], value, slope);
                            const float dz = kept[r] ? dy[i] * slope : 0.0f;
                            if constexpr (DX) {
                                x[i] = kept[r] ? channel.rstd[i] * (dz * channel.w[i] - (first[i] + normal * second[i]))
                                               : 0.0f;
                            } else {
                                first[i] += dz;
                                second[i] += dz * normal;
                            }
                        }
                    });
                    if constexpr (DX) {
                        const int64_t row = at + static_cast<int64_t>(r) * c.at_once;
                        if (row < end) {
                            store_values<T, V>(
                                static_cast<Element*>(a.dx) + (sample * a.length + row) * a.channels + c.channel, x);
                        }
                    }
                }
            }
        }
        if constexpr (!DX) {
            __syncthreads();   // the last item's readers are done
#pragma unroll
            for (int i = 0; i < V; ++i) {
                shared[threadIdx.x][i] = second[i];
                shared[threadIdx.x][V + i] = first[i];
            }
            rows[threadIdx.x] = count;
            __syncthreads();
            // dw and db of each channel of the split, and the groups' sums of them times w.
            float* out = a.partials + item * layout.pitch;
            for (int j = threadIdx.x; j < 2 * c.wide * V; j += kThreads) {
                const int part = j >= c.wide * V ? 1 : 0;
                const int thread = (j - part * c.wide * V) / V;
                const int i = (j - part * c.wide * V) - thread * V;
                float total = 0.0f;
                for (int r = 0; r < c.at_once; ++r) {
                    total += shared[thread + r * c.wide][part * V + i];
                }
                out[1 + part * a.channels + static_cast<int>(blockIdx.y) * kThreads * V + thread * V + i] = total;
                if (layout.by_group) {
                    shared[thread][part * V + i] = total * parameter(a.weight, a.parameter_type, thread * V + i, 1.0f);
                }
            }
            if (blockIdx.y == 0 && threadIdx.x == 0) {
                float total = 0.0f;
                for (int r = 0; r < c.at_once; ++r) {
                    total += rows[r * c.wide];
                }
                out[0] = total;
            }
            if (layout.by_group) {
                __syncthreads();
                over_groups(a, [&](int group, int channel0, int size, int lane, int team) {
                    float with_normal = 0.0f;
                    float alone = 0.0f;
                    for (int k = lane; k < size; k += team) {
                        const float* of = &shared[(channel0 + k) / V][(channel0 + k) % V];
                        with_normal += of[0];
                        alone += of[V];
                    }
                    with_normal = team_sum(with_normal, team);
                    alone = team_sum(alone, team);
                    if (lane == 0) {
                        out[layout.joined + group] = with_normal;
                        out[layout.joined + layout.columns + group] = alone;
                    }
                });
            }
        }
    }
}

// The groups' means of dn and dn xhat from the channels' sums of every split.
__global__ __launch_bounds__(kJoinThreads) void norm_grad_join_kernel(GroupNormArgs a) {
    __shared__ float scratch[kJoinThreads / 64];
    const Partials layout(a, true);
    const int size = layout.columns / a.groups;
    const int64_t items = a.samples * a.groups;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = quotient(item, a.groups);
        const int column0 = static_cast<int>(item - sample * a.groups) * size;
        float n = 0.0f;
        float first = 0.0f;
        float second = 0.0f;
        over_splits(a, a.partials + sample * a.splits * layout.pitch, layout.pitch, column0, size,
                    [&](const float* of, int column) {
                        const float w = layout.by_group ? 1.0f : parameter(a.weight, a.parameter_type, column, 1.0f);
                        n += of[0] * static_cast<float>(layout.unit);
                        second += w * of[layout.joined + column];
                        first += w * of[layout.joined + layout.columns + column];
                    });
        n = block_sum(n, scratch);
        first = block_sum(first, scratch);
        second = block_sum(second, scratch);
        if (threadIdx.x == 0) {
            a.sums[2 * item] = n > 0.0f ? first / n : 0.0f;
            a.sums[2 * item + 1] = n > 0.0f ? second / n : 0.0f;
        }
    }
}

// dw and db: column sums of `rows` partials, 16 of a column's rows at a time.
constexpr int kSumColumns = 16;
__global__ __launch_bounds__(kThreads) void norm_columns_kernel(GroupNormArgs a, const float* partials, int64_t rows,
                                                              int64_t pitch) {
    __shared__ float shared[kThreads / kSumColumns][kSumColumns + 1];
    const int in = static_cast<int>(threadIdx.x) % kSumColumns;
    const int at = static_cast<int>(threadIdx.x) / kSumColumns;
    const int column = static_cast<int>(blockIdx.x) * kSumColumns + in;
    float total = 0.0f;
    if (column < 2 * a.channels) {
#pragma unroll 8
        for (int64_t r = at; r < rows; r += kThreads / kSumColumns) {
            total += partials[r * pitch + column];
        }
    }
    shared[at][in] = total;
    __syncthreads();
    if (at == 0 && column < 2 * a.channels) {
        total = 0.0f;
#pragma unroll
        for (int r = 0; r < kThreads / kSumColumns; ++r) {
            total += shared[r][in];
        }
        void* out = column < a.channels ? a.grad_weight : a.grad_bias;
        if (out != nullptr) {
            store_parameter(out, a.parameter_type, column < a.channels ? column : column - a.channels, total);
        }
    }
}

template <int T, int V, int K>
void launch_team_pieces(const GroupNormArgs& a, bool backward, hipStream_t stream) {
    int across = 1;
    while (across < a.groups && across < kThreads / a.team) {
        across *= 2;
    }
    const dim3 grid(static_cast<unsigned>(a.blocks), static_cast<unsigned>((a.groups + across - 1) / across));
    if (backward) {
        team_norm_kernel<T, V, K, true><<<grid, kThreads, 0, stream>>>(a);
    } else {
        team_norm_kernel<T, V, K, false><<<grid, kThreads, 0, stream>>>(a);
    }
}

template <int T, int V>
void launch_team(const GroupNormArgs& a, bool backward, hipStream_t stream) {
    switch (a.team_pieces) {
        case 1: launch_team_pieces<T, V, 1>(a, backward, stream); break;
        case 2: launch_team_pieces<T, V, 2>(a, backward, stream); break;
        case 3: launch_team_pieces<T, V, 3>(a, backward, stream); break;
        case 4: launch_team_pieces<T, V, 4>(a, backward, stream); break;
        default:   // of narrow pieces, up to the 32 values that four of 8 are
            if constexpr (V <= 4) {
                if (a.team_pieces == 8) {
                    launch_team_pieces<T, V, 8>(a, backward, stream);
                }
            }
            if constexpr (V <= 2) {
                if (a.team_pieces == 16) {
                    launch_team_pieces<T, V, 16>(a, backward, stream);
                }
            }
            if constexpr (V == 1) {
                if (a.team_pieces == 32) {
                    launch_team_pieces<T, V, 32>(a, backward, stream);
                }
            }
    }
}

unsigned capped(int64_t blocks) { return static_cast<unsigned>(blocks < kMostGrid ? blocks : kMostGrid); }

template <int T, int V>
void launch_forward(const GroupNormArgs& a, hipStream_t stream) {
    if (a.team != 0) {
        launch_team<T, V>(a, false, stream);
        return;
    }
    if (a.samples * a.splits == 0) {
        return;
    }
    const dim3 grid(capped(a.samples * a.splits),
                    static_cast<unsigned>((a.channels / V + kThreads - 1) / kThreads));
    norm_statistics_kernel<T, V><<<grid, kThreads, 0, stream>>>(a);
    const int threads = join_threads(a.splits * (Partials(a, false).columns / a.groups));
    norm_join_kernel<<<capped(a.samples * a.groups), threads, 0, stream>>>(a);
    norm_apply_kernel<T, V><<<grid, kThreads, 0, stream>>>(a);
}

template <int T, int V>
void launch_backward(const GroupNormArgs& a, hipStream_t stream) {
    const unsigned columns = static_cast<unsigned>((2 * a.channels + kSumColumns - 1) / kSumColumns);
    const bool parameters = a.grad_weight != nullptr || a.grad_bias != nullptr;
    if (a.team != 0) {
        launch_team<T, V>(a, true, stream);
        if (parameters) {
            norm_columns_kernel<<<columns, kThreads, 0, stream>>>(a, a.partials, a.blocks,
                                                                  2 * static_cast<int64_t>(a.channels));
        }
        return;
    }
    const bool rows = a.samples * a.splits > 0;
    const dim3 grid(capped(a.samples * a.splits),
                    static_cast<unsigned>((a.channels / V + kThreads - 1) / kThreads));
    if (rows) {
        norm_grad_kernel<T, V, false><<<grid, kThreads, 0, stream>>>(a);
    }
    if (parameters) {   // without rows they are zeros
        norm_columns_kernel<<<columns, kThreads, 0, stream>>>(a, a.partials + 1, a.samples * a.splits,
                                                              Partials(a, true).pitch);
    }
    if (rows && a.dx != nullptr) {
        const int threads = join_threads(a.splits * (Partials(a, true).columns / a.groups));
        norm_grad_join_kernel<<<capped(a.samples * a.groups), threads, 0, stream>>>(a);
        norm_grad_kernel<T, V, true><<<grid, kThreads, 0, stream>>>(a);
    }
}

template <int T>
void launch_vector(const GroupNormArgs& a, bool backward, hipStream_t stream) {
    const auto run = [&](auto forward_form, auto backward_form) {
        if (backward) {
            backward_form(a, stream);
        } else {
            forward_form(a, stream);
        }
    };
    switch (a.vector) {
        case 8: run(launch_forward<T, 8>, launch_backward<T, 8>); break;
        case 4: run(launch_forward<T, 4>, launch_backward<T, 4>); break;
        case 2: run(launch_forward<T, 2>, launch_backward<T, 2>); break;
        default: run(launch_forward<T, 1>, launch_backward<T, 1>); break;
    }
}

hipError_t launch(const GroupNormArgs& a, int dtype, bool backward, hipStream_t stream) {
    switch (dtype) {
        case LSSO_HIP_F16: launch_vector<LSSO_HIP_F16>(a, backward, stream); break;
        case LSSO_HIP_BF16: launch_vector<LSSO_HIP_BF16>(a, backward, stream); break;
        default: launch_vector<LSSO_HIP_F32>(a, backward, stream); break;
    }
    return hipGetLastError();
}

int widest(int n) { return n % 8 == 0 ? 8 : (n % 4 == 0 ? 4 : (n % 2 == 0 ? 2 : 1)); }

}  // namespace

void plan_group_norm(GroupNormArgs* a, bool backward, size_t* partial_bytes) {
    const int size = a->channels / a->groups;
    a->team = 0;
    a->vector = widest(size);
    const int pieces = size / a->vector;
    if (a->length == 1 && size <= kThreads * kLaneMost) {
        // The lanes of a wave and pieces that leave the fewest registers empty; of equals
        // the most lanes, which hold fewer registers each.  Wider: the workgroup (65,536 x 4,096
        // in FP16: 240 us forward and 606 trained; as samples of one row they left 2 GiB
        // of partials and took 2,740 and 6,910).
        a->team = kThreads;
        a->team_pieces = (pieces + kThreads - 1) / kThreads;
        if (a->team_pieces > 4) {
            a->team_pieces = a->team_pieces <= 8 ? 8 : (a->team_pieces <= 16 ? 16 : 32);
        }
        int best = 1 << 30;
        for (int k = 1; k <= kTeamMost; ++k) {
            int lanes = 1;
            while (lanes * k < pieces) {
                lanes *= 2;
            }
            if (lanes <= 64 && lanes * k < best) {
                best = lanes * k;
                a->team = lanes;
                a->team_pieces = k;
            }
        }
        int across = 1;
        while (across < a->groups && across < kThreads / a->team) {
            across *= 2;
        }
        const int64_t at_once = kThreads / a->team / across;
        const int64_t rows = (a->samples + at_once - 1) / at_once;
        // Eight workgroups to a compute unit forward; half of it backward, whose
        // partials are read again.
        const int64_t most = backward ? 1024 : 2048;
        a->blocks = rows < most ? (rows > 0 ? rows : 1) : most;
        *partial_bytes = backward ? sizeof(float) * 2 * static_cast<size_t>(a->channels) * static_cast<size_t>(a->blocks) : 0;
        return;
    }
    a->vector = widest(a->channels);
    const int64_t across = (a->channels / a->vector + kThreads - 1) / kThreads;
    const int64_t wide = a->channels / a->vector < kThreads ? a->channels / a->vector : kThreads;
    const int64_t block = kBlockRows * (kThreads / wide);   // rows of a workgroup in flight
    // About two workgroups to a compute unit, each with whole blocks of rows (twice as
    // many join twice the partials: padded 8 x 1,001 x 300 26.3 -> 27.7 us a call).
    const int64_t items = a->samples * across;
    const int64_t wanted = items > 0 && items < 512 ? 512 / items : 1;
    const int64_t rows = (a->length + wanted - 1) / wanted;
    a->split_rows = rows > 0 ? (rows + block - 1) / block * block : block;
    a->splits = (a->length + a->split_rows - 1) / a->split_rows;
    *partial_bytes = sizeof(float) * static_cast<size_t>(Partials(*a, backward).pitch) * static_cast<size_t>(a->samples) *
                     static_cast<size_t>(a->splits);
}

hipError_t launch_group_norm(const GroupNormArgs& a, int dtype, hipStream_t stream) {
    return launch(a, dtype, false, stream);
}

hipError_t launch_group_norm_backward(const GroupNormArgs& a, int dtype, hipStream_t stream) {
    return launch(a, dtype, true, stream);
}

}  // namespace lsso_hip
