// The activations of the operators around the mixers.
#pragma once

#include "lsso_device.h"
#include "lsso_hip.h"

namespace lsso_hip {

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

}  // namespace lsso_hip
