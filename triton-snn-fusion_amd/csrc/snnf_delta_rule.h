// Parts of the gated delta rule's kernels: numbers as sums of bfloat16 terms for the matrix units, fragments, what forward and backward pass share.
#pragma once

#include "snnf_sequence.h"

namespace snnf {

// ------------------------------------------------------------------------------------------------------------------
// Products on the matrix units
// ------------------------------------------------------------------------------------------------------------------
// A number is the sum of up to three bfloat16 terms, each what the ones before it leave, rounded: 8 bits each, so that one holds a bfloat16, two a float16, three a
// float32 to within 2^-25. A product of two sums adds the products of terms whose ranks add up to less than `RANKS`: 3 of them are off by some 2^-24 of the
// factors' magnitudes, as a float32 product is, 2 by some 2^-17. The matrix units multiply bfloat16 at 16 times the rate of float32, and a product of
// a 16-bit tensor (one term) with the float32 state takes three passes.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2a __attribute__((ext_vector_type(2)));

template <int N> struct Terms {
    u32x4a t[N];                        // 8 elements each
};
template <typename T> inline constexpr int kTerms = sizeof(T) == 4 ? 3 : (dtype_of<T>::value == SNNF_F16 ? 2 : 1);

template <int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[N]) {
    out[0] = float_to_bf16_pair(a, b);
#pragma unroll
    for (int n = 1; n < N; ++n) {
        a -= __uint_as_float(out[n - 1] << 16);
        b -= __uint_as_float(out[n - 1] & 0xffff0000u);
        out[n] = float_to_bf16_pair(a, b);
    }
}
template <int N>
__device__ __forceinline__ Terms<N> split(const float (&x)[8]) {
    Terms<N> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t words[N];
        split_pair<N>(x[2 * i], x[2 * i + 1], words);
#pragma unroll
        for (int n = 0; n < N; ++n) r.t[n][i] = words[n];
    }
    return r;
}
template <int N>
__device__ __forceinline__ Terms<N> split(const f32x4& a, const f32x4& b) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return split<N>(x);
}

__device__ __forceinline__ f32x4 mfma(const u32x4a& a, const u32x4a& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// c + a b over 32 places, [16 x 32] x [32 x 16]: lane l has row (column) l % 16 of its operand and 8 of the places, those of its group l / 16; c has column l % 16
// and rows 4 (l / 16) + 0..3. The smallest terms first.
template <int RANKS, int NA, int NB>
__device__ __forceinline__ f32x4 product(const Terms<NA>& a, const Terms<NB>& b, f32x4 c) {
#pragma unroll
    for (int rank = RANKS - 1; rank >= 0; --rank)
#pragma unroll
        for (int i = 0; i <= rank; ++i)
            if (i < NA && rank - i < NB) c = mfma(a.t[i], b.t[rank - i], c);
    return c;
}

// Which of 32 places of a contraction group `g` holds as its element j: in order where both operands come from memory, or where one is an accumulator
// (two tiles of 16 rows, of which a group has 4g to 4g + 3) and is multiplied where it lies, without a way through LDS.
__device__ __forceinline__ constexpr int accumulated_place(int g, int j) { return j < 4 ? 4 * g + j : 12 + 4 * g + j; }

constexpr int kChunk = 64;              // steps that are taken at once
constexpr int kBlocks = 6;              // fragments [16 x 32] of a triangular matrix [64 x 64] that are not zero

// ------------------------------------------------------------------------------------------------------------------
// Operands
// ------------------------------------------------------------------------------------------------------------------
struct HeadView {                       // [T, N, heads, D], elements of a head next to each other
    const void* data;
    int64_t step, row, head;
};

struct DeltaArgs {
    HeadView q, k, v, gate, beta, out, dout, dq, dk, dv, dgate, dbeta;
    int T, N, H, HV, DK, DV, chunks;
    float scale;
    int gate_float, beta_there;         // gates in float32 beside 16-bit tensors
    const uint8_t* starts;
    int64_t starts_step, starts_row;
    const int32_t* lengths;
    const float* state;
    float* state_out;
    const float* dstate;
    float* dstate_in;
    // per chunk of a value head
    uint32_t* blocks;                   // fragments of the inverse, then of the scores
    float* vectors;                     // since, until, beta [64] each
    float* marks;                       // state before the chunk [DK][DV]
    float* deltas;                      // v - S k [64][DV]
    float* later;                       // gradient of the state behind the chunk [DK][DV]
    float* pulls;                       // gradient of beta delta's cause [64][DV]
};

__device__ __forceinline__ int length_of(const DeltaArgs& p, int n) {
    if (p.lengths == nullptr) return p.T;
    const int length = p.lengths[n];
    return length < 0 ? 0 : (length < p.T ? length : p.T);
}

// 8 elements of a row from `at` on, zeros behind its end.
template <typename T>
__device__ __forceinline__ Terms<kTerms<T>> row_terms(const T* row, int at, int width) {
    Raw<T, 8> raw;
    raw.load(row, at, width - at);
    if constexpr (dtype_of<T>::value == SNNF_BF16) {
        Terms<1> r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.t[0][i] = raw.w[i];
        return r;
    } else {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = raw[j];
        return split<kTerms<T>>(x);
    }
}
template <int N>
__device__ __forceinline__ Terms<N> no_terms() {
    Terms<N> r;
#pragma unroll
    for (int n = 0; n < N; ++n) r.t[n] = u32x4a{0, 0, 0, 0};
    return r;
}

// Fragment f = 0..5 of a lower triangular [64 x 64] matrix: rows of tile 0, 1, 2, 2, 3, 3, columns of half 0, 0, 0, 1, 0, 1. Of an upper one
// (a transposed lower one): rows of tile 0, 0, 1, 1, 2, 3, columns of half 0, 1, 0, 1, 1, 1.
__device__ __forceinline__ constexpr int lower_tile(int f) { return f < 2 ? f : (f < 4 ? 2 : 3); }
__device__ __forceinline__ constexpr int lower_half(int f) { return f == 3 || f == 5 ? 1 : 0; }
__device__ __forceinline__ constexpr int upper_tile(int f) { return f < 2 ? 0 : (f < 4 ? 1 : f - 2); }
__device__ __forceinline__ constexpr int upper_half(int f) { return f == 0 || f == 2 ? 0 : 1; }

// Words of a chunk's fragments: 3 terms of the inverse, `ranks` of the scores.
__host__ __device__ __forceinline__ constexpr int block_words(int ranks) { return kBlocks * (3 + ranks) * 256; }

// ------------------------------------------------------------------------------------------------------------------
// Keys and queries of a chunk in LDS
// ------------------------------------------------------------------------------------------------------------------
// [term][64 rows][32 KS + 8], the elements of every 32 in the order of `accumulated_place`, so that a row's 16 bytes are an operand against an accumulator over
// the head's elements, and 4 rows x 16 elements, transposed on their way by the LDS unit, one over the steps.
template <typename T, int KS> struct Rows {
    static constexpr int kStride = 32 * KS + 8, kPlane = kChunk * kStride, kSize = kTerms<T> * kPlane;      // in elements
    static constexpr int kPieces = kChunk * 4 * KS;                                                    // of 8 elements

    __device__ __forceinline__ static void put(uint16_t* lds, int piece, const Terms<kTerms<T>>& x) {
        const int row = piece / (4 * KS), at = piece % (4 * KS), s = at / 4, quad = 2 * (at % 4);
        const int place = quad < 4 ? 8 * quad : 8 * (quad - 4) + 4;                                     // the next quad lies 8 further
        uint16_t* to = lds + row * kStride + 32 * s + place;
#pragma unroll
        for (int n = 0; n < kTerms<T>; ++n) {
            *reinterpret_cast<u32x2a*>(to + n * kPlane) = u32x2a{x.t[n][0], x.t[n][1]};
            *reinterpret_cast<u32x2a*>(to + n * kPlane + 8) = u32x2a{x.t[n][2], x.t[n][3]};
        }
    }
    // rows 16 tile.., elements 32 s..
    __device__ __forceinline__ static Terms<kTerms<T>> rows(const uint16_t* lds, int tile, int s) {
        const int lane = threadIdx.x & 63;
        const uint16_t* from = lds + (16 * tile + lane % 16) * kStride + 32 * s + 8 * (lane / 16);
        Terms<kTerms<T>> r;
#pragma unroll
        for (int n = 0; n < kTerms<T>; ++n) r.t[n] = *reinterpret_cast<const u32x4a*>(from + n * kPlane);
        return r;
    }
    // elements 16 tile.. as rows, steps of half `half` as places
    __device__ __forceinline__ static Terms<kTerms<T>> columns(const uint16_t* lds, int tile, int half) {
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        const int lane = threadIdx.x & 63, l = lane % 16;
        const uint16_t* from = lds + (32 * half + 4 * (lane / 16) + l / 4) * kStride + 32 * (tile / 2) + 8 * (l % 4) + 4 * (tile % 2);
        Terms<kTerms<T>> r;
#pragma unroll
        for (int n = 0; n < kTerms<T>; ++n) {
            const u32x2a low = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(from + n * kPlane)));
            const u32x2a high = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(from + n * kPlane + 16 * kStride)));
            r.t[n] = u32x4a{low[0], low[1], high[0], high[1]};
        }
        return r;
    }
    // elements 16 tile + 4 (lane / 16) + 0..3 of a row
    __device__ __forceinline__ static f32x4 four(const uint16_t* lds, int row, int tile) {
        const int lane = threadIdx.x & 63;
        const uint16_t* from = lds + row * kStride + 32 * (tile / 2) + 8 * (lane / 16) + 4 * (tile % 2);
        f32x4 r{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = kTerms<T> - 1; n >= 0; --n) {
            const u32x2a words = *reinterpret_cast<const u32x2a*>(from + n * kPlane);
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] += element<bf16_t>(words[j / 2], j % 2);
        }
        return r;
    }
};

// Pieces of a chunk's rows on their way from memory to LDS, `COUNT` to a thread of `THREADS`.
template <typename T, int KS, int THREADS> struct Staged {
    static constexpr int kCount = Rows<T, KS>::kPieces / THREADS;
    Raw<T, 8> raw[kCount];
    __device__ __forceinline__ void load(const HeadView& x, int first, int limit, int n, int head, int width) {
        const T* base = static_cast<const T*>(x.data) + n * x.row + head * x.head;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int piece = threadIdx.x + i * THREADS, t = first + piece / (4 * KS), at = 8 * (piece % (4 * KS));
            if (t < limit && at < width) raw[i].load(base + t * x.step, at, width - at);
            else raw[i].clear();
        }
    }
    __device__ __forceinline__ void store(uint16_t* lds) const {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            Terms<kTerms<T>> r;
            if constexpr (dtype_of<T>::value == SNNF_BF16) {
#pragma unroll
                for (int w = 0; w < 4; ++w) r.t[0][w] = raw[i].w[w];
            } else {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = raw[i][j];
                r = split<kTerms<T>>(x);
            }
            Rows<T, KS>::put(lds, threadIdx.x + i * THREADS, r);
        }
    }
};

// Gates: of the activations' type or float32; none: no decay, every step learnt in full.
template <typename T>
__device__ __forceinline__ float gate_value(const HeadView& x, bool is_float, int t, int n, int head, float otherwise) {
    if (x.data == nullptr) return otherwise;
    const int64_t at = t * x.step + n * x.row + head * x.head;
    return is_float ? static_cast<const float*>(x.data)[at] : to_float(static_cast<const T*>(x.data)[at]);
}

// A gate below this leaves less than 2^-149 of the state: the state starts anew, as where a start is set.
constexpr float kForgotten = -104.0f;

// exp of a difference of logarithms in powers of two, which are summed in float64: a float32 sum of many would lose what a small difference has.
__device__ __forceinline__ float decay_of(double x) {
    if (!(x > -160.0)) return x != x ? __builtin_nanf("") : 0.0f;
    const double whole = __builtin_rint(x);
    return ldexpf(__builtin_amdgcn_exp2f(static_cast<float>(x - whole)), static_cast<int>(whole < 1000.0 ? whole : 1000.0));
}

// Row i of a factor that a vanished decay has made 0 drops what it would multiply, infinities and NaN as well.
__device__ __forceinline__ float kept(float factor, float x) { return factor == 0.0f ? 0.0f : factor * x; }

// Workgroups to heads and parts of them so that the parts of a head, which read the same keys, run on one of the 8 dies and share its cache: neighbouring workgroups go to
// different dies. False: nothing to do.
__device__ __forceinline__ bool part_of_head(int heads, int parts, int* head, int* part) {
    constexpr int kDies = 8;
    const int die = blockIdx.x % kDies, order = blockIdx.x / kDies;
    *part = order % parts;
    *head = order / parts * kDies + die;
    return *head < heads;
}
inline unsigned head_groups(int heads, int parts) { return static_cast<unsigned>((heads + 7) / 8 * 8 * parts); }

// Fragments, decays and inverses of all chunks; transposed for the backward pass.
template <typename T, int KS, bool BACKWARD> void launch_chunks(const DeltaArgs& p, hipStream_t stream);

// Terms of what the output alone depends on: scores, and the state and corrections that they multiply.
template <typename T> inline constexpr int kOutputRanks = sizeof(T) == 4 ? 3 : 2;

int check_delta(const char* name, const snnf_delta_rule_call* call);
DeltaArgs delta_args(const snnf_delta_rule_call* call);
int64_t delta_chunks(const snnf_delta_rule_call* call);
}  // namespace snnf
