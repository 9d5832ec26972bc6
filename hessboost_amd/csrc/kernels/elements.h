// The operators' element types and vectors of them.
#pragma once
#include "common.h"

namespace hbr {

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// To nearest, ties to even; a NaN stays one.
__device__ __forceinline__ uint16_t f32_bf16(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

struct F32 {
    using type = float;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
struct Bf16 {
    using type = uint16_t;
    static __device__ __forceinline__ float up(uint16_t v) { return bf16_f32(v); }
    static __device__ __forceinline__ uint16_t down(float v) { return f32_bf16(v); }
};

template <typename T, int V>
struct alignas(sizeof(T) * V <= 16 ? sizeof(T) * V : 16) Vec {
    T v[V];
};

// A vector from a buffer at a byte offset; zeros past its end.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> buffer_vec(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    if constexpr (sizeof(T) * V == 16) return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
    else if constexpr (sizeof(T) * V == 8) return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
    else if constexpr (sizeof(T) * V == 4) return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
    else return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
}

}  // namespace hbr
