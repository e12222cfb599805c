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

// Workgroups that are as many as a long tensor has rows: a launch takes fewer than 2^32 threads along x, so that the rest goes along y. Those behind
// the last one have nothing to do.
inline dim3 grid_of(int64_t groups) {
    constexpr int64_t kAlong = 1 << 21;
    return groups <= kAlong ? dim3(static_cast<unsigned>(groups)) : dim3(kAlong, static_cast<unsigned>((groups + kAlong - 1) / kAlong));
}
__device__ __forceinline__ uint32_t group_index() { return blockIdx.y * gridDim.x + blockIdx.x; }

// The value of the lane `MASK` apart, by exchange within the register file (a shuffle through LDS takes several times as long). Which lane
// that is for 4 and 8, where rows of 8 and 16 lanes are mirrored, does not matter to a sum or maximum that has been taken over the smaller
// distances before.
template <int MASK>
__device__ __forceinline__ float across(float v) {
    const int bits = __float_as_int(v);
    if constexpr (MASK == 1) return __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, 0xB1, 0xf, 0xf, false));        // lanes 1 0 3 2
    else if constexpr (MASK == 2) return __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, 0x4E, 0xf, 0xf, false));   // lanes 2 3 0 1
    else if constexpr (MASK == 4) return __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, 0x141, 0xf, 0xf, false));  // 8 lanes mirrored
    else if constexpr (MASK == 8) return __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, 0x140, 0xf, 0xf, false));  // 16 lanes mirrored
    else return __shfl_xor(v, MASK, 64);
}
// Over groups of `lanes` (4 to 64) neighbouring lanes, in every lane, always in the same order: with the rows of 16 lanes summed, the exchange of
// rows or halves leaves one half's value in one register and the other's in the other.
template <typename Op>
__device__ __forceinline__ float over_lanes(float v, int lanes, Op op) {
    v = op(v, across<1>(v));
    v = op(v, across<2>(v));
    if (lanes >= 8) v = op(v, across<4>(v));
    if (lanes >= 16) v = op(v, across<8>(v));
    if (lanes >= 32) {
        const auto pair = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(pair[0]), __uint_as_float(pair[1]));
    }
    if (lanes >= 64) {
        const auto pair = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(pair[0]), __uint_as_float(pair[1]));
    }
    return v;
}
__device__ __forceinline__ float lane_sum(float v, int lanes = 64) {
    return over_lanes(v, lanes, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float lane_max(float v, int lanes = 64) {
    return over_lanes(v, lanes, [](float a, float b) { return fmaxf(a, b); });
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

// Elements of a 16-byte access.
template <typename T> inline constexpr int kVec = sizeof(T) == 4 ? 4 : 8;

// VEC elements of T as they lie in memory; zeros behind the end of a row.
template <typename T, int VEC> struct Raw {
    static constexpr int kWords = VEC * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ float operator[](int j) const {
        if constexpr (sizeof(T) == 4) return element<T>(w[j], 0);
        else return element<T>(w[j / 2], j % 2);
    }
    __device__ __forceinline__ void load(const void* base, int64_t at, int left) {
        const T* p = static_cast<const T*>(base) + at;
        if (left >= VEC) {
            const auto words = *reinterpret_cast<const typename Words<T, VEC>::type*>(p);
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = words[i];
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if constexpr (sizeof(T) == 4) w[i] = i < left ? __float_as_uint(p[i]) : 0u;
                else w[i] = (2 * i < left ? p[2 * i].bits : 0u) | (2 * i + 1 < left ? static_cast<uint32_t>(p[2 * i + 1].bits) << 16 : 0u);
            }
        }
    }
    // a vector of the program's, ones where it has none
    __device__ __forceinline__ void load_vector(const void* base, int at, int left) {
        if (base != nullptr) {
            load(base, at, left);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = sizeof(T) == 4 ? __float_as_uint(1.0f) : pair_word_or_zero(1.0f);
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t at, int left) const {
        T* p = static_cast<T*>(base) + at;
        if (left >= VEC) {
            typename Words<T, VEC>::type words;
#pragma unroll
            for (int i = 0; i < kWords; ++i) words[i] = w[i];
            *reinterpret_cast<typename Words<T, VEC>::type*>(p) = words;
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if constexpr (sizeof(T) == 4) {
                    if (j < left) p[j] = __uint_as_float(w[j]);
                } else {
                    if (j < left) p[j].bits = static_cast<uint16_t>(j % 2 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu);
                }
            }
        }
    }
    __device__ __forceinline__ void put(int j, float first, float second) {
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(first), w[j + 1] = __float_as_uint(second);
        else w[j / 2] = pair_word<T>(first, second);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    // The same bits, of which the compiler knows nothing: what was taken apart before is not kept for the next use.
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) asm("" : "+v"(w[i]));
    }
    __device__ __forceinline__ static uint32_t pair_word_or_zero(float v) {
        if constexpr (sizeof(T) == 4) return 0u;
        else return pair_word<T>(v, v);
    }
};
}  // namespace snnf
