// Helpers of the sequence operators (gated recurrence, block norm, token scores).
#pragma once

#include "snnf_common.h"

namespace snnf {

template <typename XT> inline constexpr bool kPrecise = sizeof(XT) == 4;

// a = sigmoid(g) = 1 / (1 + e) and 1 - a = e / (1 + e) with e = exp(-g), both to full relative accuracy; a NaN stays one, and a g of
// infinity gives a = 1 and 1 - a = 0 exactly. e is kept from overflowing. v_exp_f32 works on powers of two; for float32 tensors what the
// product with log2(e) loses is put back to first order.
template <bool PRECISE>
__device__ __forceinline__ void leak(float g, float& a, float& rest) {
    constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.925963033500e-8f, kLn2 = 0.69314718055994530942f;
    float e;
    if constexpr (PRECISE) {
        const float y = __builtin_elementwise_minimum(__builtin_elementwise_maximum(g, -86.0f), 200.0f);
        const float t = y * -kLog2e;
        e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e, fmaf(y, -kLog2eLow, fmaf(y, -kLog2e, -t)) * kLn2, e);
    } else {
        e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -kLog2e, 124.0f));
    }
    a = __builtin_amdgcn_rcpf(1.0f + e);
    rest = e * a;
}

// Sum over the 64 lanes of a wave, in every lane, always in the same order.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int mask = 32; mask > 0; mask >>= 1) v += __shfl_xor(v, mask, 64);
    return v;
}

// VEC elements that lie as elements of T do and no better: rows of odd widths start anywhere. The memory unit takes wide accesses at any
// alignment; what crosses a line costs a second one.
template <typename T, int VEC> struct Words;
template <> struct Words<float, 4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Words<bf16_t, 8> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Words<f16_t, 8> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Words<float, 8> { typedef uint32_t type __attribute__((ext_vector_type(8), aligned(4))); };

template <typename T>
__device__ __forceinline__ float element(uint32_t word, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(word);
    else if constexpr (dtype_of<T>::value == SNNF_BF16) return __uint_as_float(j == 0 ? word << 16 : word & 0xffff0000u);
    else return f16_bits_to_float(j == 0 ? word & 0xffffu : word >> 16);
}
template <typename T>
__device__ __forceinline__ uint32_t pair_word(float lo, float hi) {
    if constexpr (dtype_of<T>::value == SNNF_BF16) return float_to_bf16_pair(lo, hi);
    else return float_to_f16_bits(lo) | float_to_f16_bits(hi) << 16;
}

}  // namespace snnf
