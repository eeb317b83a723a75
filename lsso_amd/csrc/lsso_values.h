// Element types of the operators that take FP16, BF16 or FP32 tensors: loads
// and stores of 1 and of 8 elements, through FP32.  Addresses need no more than
// the element's own alignment (16-byte accesses of global memory do not on
// gfx950), so odd rows, strides and bases take the same path.
#pragma once

#include "lsso_device.h"
#include "lsso_hip.h"

namespace lsso_hip {

template <int T>
struct Values;

template <>
struct Values<LSSO_HIP_F32> {
    using Element = float;
    __device__ static __forceinline__ float load(const float* at) { return *at; }
    __device__ static __forceinline__ void store(float* at, float v) { *at = v; }
    __device__ static __forceinline__ void load8(const float* at, float (&v)[8]) {
        const f32x4 low = __builtin_bit_cast(f32x4, load16_unaligned(at));
        const f32x4 high = __builtin_bit_cast(f32x4, load16_unaligned(at + 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = low[i];
            v[4 + i] = high[i];
        }
    }
    __device__ static __forceinline__ void store8(float* at, const float (&v)[8]) {
        store16_unaligned(at, __builtin_bit_cast(u32x4, (f32x4){v[0], v[1], v[2], v[3]}));
        store16_unaligned(at + 4, __builtin_bit_cast(u32x4, (f32x4){v[4], v[5], v[6], v[7]}));
    }
};

template <>
struct Values<LSSO_HIP_BF16> {
    using Element = uint16_t;
    __device__ static __forceinline__ float low(uint32_t pair) { return bf16_lo(pair); }
    __device__ static __forceinline__ float high(uint32_t pair) { return bf16_hi(pair); }
    __device__ static __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
    __device__ static __forceinline__ float load(const uint16_t* at) { return bf16_bits_to_float(*at); }
    __device__ static __forceinline__ void store(uint16_t* at, float v) { *at = to_bf16_bits(v); }
    __device__ static __forceinline__ void load8(const uint16_t* at, float (&v)[8]) { unpack8(load16_unaligned(at), v); }
    __device__ static __forceinline__ void store8(uint16_t* at, const float (&v)[8]) { store16_unaligned(at, pack8(v)); }
    __device__ static __forceinline__ void unpack8(const u32x4& raw, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = low(raw[i]);
            v[2 * i + 1] = high(raw[i]);
        }
    }
    __device__ static __forceinline__ u32x4 pack8(const float (&v)[8]) {
        return (u32x4){pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7])};
    }
};

template <>
struct Values<LSSO_HIP_F16> {
    using Element = uint16_t;
    __device__ static __forceinline__ float low(uint32_t pair) { return f16_lo(pair); }
    __device__ static __forceinline__ float high(uint32_t pair) { return f16_hi(pair); }
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
    }
    __device__ static __forceinline__ float load(const uint16_t* at) { return f16_bits_to_float(*at); }
    __device__ static __forceinline__ void store(uint16_t* at, float v) { *at = to_f16_bits(v); }
    __device__ static __forceinline__ void load8(const uint16_t* at, float (&v)[8]) { unpack8(load16_unaligned(at), v); }
    __device__ static __forceinline__ void store8(uint16_t* at, const float (&v)[8]) { store16_unaligned(at, pack8(v)); }
    __device__ static __forceinline__ void unpack8(const u32x4& raw, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = low(raw[i]);
            v[2 * i + 1] = high(raw[i]);
        }
    }
    __device__ static __forceinline__ u32x4 pack8(const float (&v)[8]) {
        return (u32x4){pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7])};
    }
};

// V (1, 2, 4 or 8) elements in one access (two of 8 FP32 elements).
template <int T, int V>
__device__ __forceinline__ void load_values(const typename Values<T>::Element* at, float (&v)[V]) {
    if constexpr (V == 8) {
        Values<T>::load8(at, v);
    } else {
        typename Values<T>::Element raw[V];
        __builtin_memcpy(raw, at, sizeof(raw));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = Values<T>::load(raw + i);
        }
    }
}
template <int T, int V>
__device__ __forceinline__ void store_values(typename Values<T>::Element* at, const float (&v)[V]) {
    if constexpr (V == 8) {
        Values<T>::store8(at, v);
    } else {
        typename Values<T>::Element raw[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            Values<T>::store(raw + i, v[i]);
        }
        __builtin_memcpy(at, raw, sizeof(raw));
    }
}

}  // namespace lsso_hip
