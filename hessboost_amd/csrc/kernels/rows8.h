// Rows in 8 bits: e4m3 codes, 32 columns of a row sharing a power of two.
//
// The power is the smallest, 2^-109 at least, under which none of the 32 is
// above e4m3's largest, 448: nothing saturates, and a value is off by at most
// half of e4m3's step, 2^-4 of itself, or 2^-10 of the power where that is more.
// A power of two, so that a code times it is a bf16 exactly (four bits of 2^-118
// to 2^128) and a product of such values has no rounding but its own. An element
// that is infinite or no number is held as no number and counts nothing for the power.
#pragma once
#include "elements.h"

namespace hbr {

constexpr int kPowerBias = 127, kLeastPower = -109;

// The power's exponent for the largest magnitude of 32 values.
__device__ __forceinline__ int32_t power_of(float largest) {
    const uint32_t bits = __float_as_uint(largest);
    return max((int32_t)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u), kLeastPower);
}

// A value's part in the largest: nothing where it is infinite or no number.
__device__ __forceinline__ float magnitude(float v) {
    const float m = __builtin_fabsf(v);
    return m < INFINITY ? m : 0.0f;
}

// 2^e for the exponents of powers and their opposites.
__device__ __forceinline__ float exp2_of(int32_t e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two values, times `by` (the power's inverse), as codes in the low or high half of `into`.
template <bool High>
__device__ __forceinline__ uint32_t two_codes(float a, float b, float by, uint32_t into) {
    a = __builtin_fabsf(a) < INFINITY ? a * by : NAN;
    b = __builtin_fabsf(b) < INFINITY ? b * by : NAN;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)into, High);
}

template <int V>
__device__ __forceinline__ Vec<uint8_t, V> codes_of(const float (&v)[V], float by) {
    Vec<uint8_t, V> out;
    if constexpr (V == 1) {
        out.v[0] = (uint8_t)two_codes<false>(v[0], v[0], by, 0);
    } else if constexpr (V == 2) {
        const uint16_t both = (uint16_t)two_codes<false>(v[0], v[1], by, 0);
        __builtin_memcpy(&out, &both, 2);
    } else {
        uint32_t words[V / 4];
#pragma unroll
        for (int k = 0; k < V / 4; k++)
            words[k] = two_codes<true>(v[4 * k + 2], v[4 * k + 3], by, two_codes<false>(v[4 * k], v[4 * k + 1], by, 0));
        __builtin_memcpy(&out, words, V);
    }
    return out;
}

// What codes stand for.
template <int V>
__device__ __forceinline__ void values_of(const Vec<uint8_t, V> &c, float power, float (&v)[V]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < V; k += 4) {
        uint32_t word = 0;
        __builtin_memcpy(&word, &c.v[k], V - k < 4 ? V - k : 4);
        const f32x2 low = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false);
        v[k] = low[0] * power;
        if constexpr (V > 1) v[k + 1] = low[1] * power;
        if constexpr (V > 2) {
            const f32x2 high = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
            v[k + 2] = high[0] * power;
            v[k + 3] = high[1] * power;
        }
    }
}

}  // namespace hbr
