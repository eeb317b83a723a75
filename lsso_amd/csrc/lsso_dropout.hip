// Residual dropout with a mask that is never stored:
//   y = residual + keep * x * scale,   scale = 65536 / (65536 - threshold).
//
// The mask is a function of the element's index alone, so the backward pass
// draws it again from the same seed instead of reading it: element i takes the
// 16-bit value i % 8 of the Philox-4x32-10 block (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) of counter
// (i / 8, offset) under the key `seed`, and is kept when it is at least
// `threshold`, the drop probability in units of 2^-16.  `scale` is the inverse
// of the keep probability that this threshold realizes, so the expectation is
// exact.  16 bits per element, not 32: one block then serves 8 elements.
//
// Bound: HBM.  Forward 3, backward 2 streams of the tensor.  A thread takes one
// block's 8 elements per step, 16 bytes of each 16-bit operand.  262,144 x 256 BF16:
// forward 73 us (5.5 TB/s), backward 44 us (6.1 TB/s), where a large copy reaches 6.6;
// the generator's 20 products of 32 x 32 bits per thread hide under the loads.

#include "lsso_device.h"
#include "lsso_internal.h"
#include "lsso_values.h"

#include "lsso_hip.h"

namespace lsso_hip {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ u32x4 philox(uint64_t group, uint64_t offset, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(group);
    uint32_t c1 = static_cast<uint32_t>(group >> 32);
    uint32_t c2 = static_cast<uint32_t>(offset);
    uint32_t c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed);
    uint32_t k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
        const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return (u32x4){c0, c1, c2, c3};
}

// T: the tensors' type code; ADD: with a residual.
template <int T, bool ADD>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs a) {
    using Element = typename Values<T>::Element;
    uint64_t seed = a.seed;
    uint64_t offset = a.offset;
    if (a.state != nullptr) {
        seed = static_cast<uint64_t>(a.state[0]);
        offset += static_cast<uint64_t>(a.state[1]);
    }
    const Element* x = static_cast<const Element*>(a.x);
    const Element* residual = static_cast<const Element*>(a.residual);
    Element* y = static_cast<Element*>(a.y);
    const int64_t group = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t first = 8 * group;
    if (first >= a.count) {
        return;
    }
    const bool whole = first + 8 <= a.count;
    float v[8];
    float r[8];
    if (whole) {
        Values<T>::load8(x + first, v);
        if (ADD) {
            Values<T>::load8(residual + first, r);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = first + i < a.count ? Values<T>::load(x + first + i) : 0.0f;
            r[i] = ADD && first + i < a.count ? Values<T>::load(residual + first + i) : 0.0f;
        }
    }
    const u32x4 words = philox(static_cast<uint64_t>(group), offset, seed);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = (words[i / 2] >> (16 * (i & 1))) & 0xffffu;
        // A dropped element is left out rather than multiplied by zero: an
        // infinity or NaN in it goes with it.
        const float kept = v[i] * a.scale;
        const float sum = ADD ? r[i] + kept : kept;
        v[i] = bits >= a.threshold ? sum : (ADD ? r[i] : 0.0f);
    }
    if (whole) {
        Values<T>::store8(y + first, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (first + i < a.count) {
                Values<T>::store(y + first + i, v[i]);
            }
        }
    }
}

template <int T>
void launch(const DropoutArgs& a, hipStream_t stream) {
    const int64_t groups = (a.count + 7) / 8;
    const dim3 grid(static_cast<unsigned>((groups + kThreads - 1) / kThreads));
    if (a.residual != nullptr) {
        dropout_kernel<T, true><<<grid, kThreads, 0, stream>>>(a);
    } else {
        dropout_kernel<T, false><<<grid, kThreads, 0, stream>>>(a);
    }
}

}  // namespace

hipError_t launch_dropout(const DropoutArgs& a, int dtype, hipStream_t stream) {
    if (a.count == 0) {
        return hipSuccess;
    }
    switch (dtype) {
        case LSSO_HIP_F16: launch<LSSO_HIP_F16>(a, stream); break;
        case LSSO_HIP_BF16: launch<LSSO_HIP_BF16>(a, stream); break;
        default: launch<LSSO_HIP_F32>(a, stream); break;
    }
    return hipGetLastError();
}

}  // namespace lsso_hip
