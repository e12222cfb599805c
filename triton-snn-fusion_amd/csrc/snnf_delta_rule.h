// Parts of the gated delta rule's kernels: numbers as sums of bfloat16 terms for the matrix units, fragments, what forward and backward pass share.
#pragma once

#include <algorithm>
#include <type_traits>

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

// What a term leaves comes from a dot product with (-1, 0) or (0, -1), which saves taking the pair apart (7 instructions for three terms of two numbers, 11 with shifts and
// subtractions). The differences are exact.
template <int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[N]) {
    // (-1, 0) and (0, -1), from registers: as an inline constant of the instruction -1.0 does not mean the first
    uint32_t lower = 0x0000bf80u, upper = 0xbf800000u;
    asm("" : "+s"(lower), "+s"(upper));
    const snnf_bf16x2 first = __builtin_bit_cast(snnf_bf16x2, lower), second = __builtin_bit_cast(snnf_bf16x2, upper);
    out[0] = float_to_bf16_pair(a, b);
#pragma unroll
    for (int n = 1; n < N; ++n) {
        const snnf_bf16x2 term = __builtin_bit_cast(snnf_bf16x2, out[n - 1]);
        a = __builtin_amdgcn_fdot2_f32_bf16(term, first, a, false);
        b = __builtin_amdgcn_fdot2_f32_bf16(term, second, b, false);
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

// Over the four rows of 16 lanes
__device__ __forceinline__ float sum_of_rows(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Nothing is moved across by the compiler, which would put loads off until their values are needed.
__device__ __forceinline__ void now() { __builtin_amdgcn_sched_barrier(0); }

// An accumulator multiplied next lies where the second operand of a product does: a lane has a column and, of two tiles of 16 rows, 4 (l / 16) to 4 (l / 16) + 3 each, 8 places out of 32. What they are
// places of is up to the first operand. Over steps, a tile's rows are 16 steps, and the first operand takes its places in that order. Over a head's elements, the rows
// of two tiles are chosen so that the places are 32 elements in order:
__device__ __forceinline__ int head_element(int tile, int r) { return 32 * (tile / 2) + 8 * ((threadIdx.x & 63) / 16) + 4 * (tile % 2) + r; }

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
    int gate_float;                     // gates in float32 beside 16-bit tensors
    int near_keys, near_values;         // whether a chunk's rows are whole vectors within reach of 31 bits
    const uint8_t* starts;
    int64_t starts_step, starts_row;
    const int32_t* lengths;
    const float* state;
    float* state_out;
    const float* dstate;
    float* dstate_in;
    // per chunk of a value head
    uint32_t* blocks;                   // fragments of the inverse, then of the scores, then vectors
    uint16_t* marks;                    // state before the chunk, as planes (below)
    uint16_t* deltas;                   // v - S k, [rank][16 value columns][64][16], so that a wave writes whole lines
    uint16_t* later;                    // gradient of the state behind the chunk, as marks
    uint16_t* pulls;                    // Z, as deltas
    // Few heads: chunks in segments of `per`, walked side by side
    int segments, per;
    float* transfers;                   // per head and segment but the last walked: what it makes of a state (below)
    float* between;                     // per head and segment: the state before it (backward: the gradient of the state behind it, of all but the last)
};

// Of a chunk's block: 3 terms of the inverse's fragments, `ranks` of the scores', then exp(G), exp(G_64 - G), beta [64] each, whether any of the first two is 0, the steps that start anew as 64 bits, and zeros.
constexpr int kSince = 0, kUntil = kChunk, kBeta = 2 * kChunk, kBroken = 3 * kChunk, kFresh = 3 * kChunk + 2, kZeros = 3 * kChunk + 4;
__host__ __device__ __forceinline__ constexpr int block_pieces(int ranks) { return kBlocks * (3 + ranks) + 1; }      // of 256 words
__host__ __device__ __forceinline__ constexpr int block_words(int ranks) { return block_pieces(ranks) * 256; }
__host__ __device__ __forceinline__ constexpr int block_vectors(int ranks) { return kBlocks * (3 + ranks) * 256; }

// Terms of what the output alone depends on: scores, and the state and corrections that they multiply. A call whose gradients will be wanted has as many of what the gradients of queries, keys
// and gates are products of (RANKS below): 2 where all of those are rounded to 16 bits, 3 where gates are float32, whose gradients float32 are, too. In the gradient of gates those of queries and keys cancel: with
// one term of the states for bfloat16 it had been off by 1.5 to 2.8 times bfloat16's rounding (and 120 of 1590 us of a training pass of 4096 x 4 x 16 heads shorter), with two terms of everything
// float32 gates' by 1 to 4 x 10^-5 of its size (with three by 0.5 to 1.4 x 10^-6; forward and backward of 4096 x 4 x 16 heads of 128 bfloat16 take 1512 in place of 1113 us then).
template <typename T> inline constexpr int kOutputRanks = sizeof(T) == 4 ? 3 : 2;

// What the walks leave for the gradients, as the terms of which those are products. States [rank][value column][32 KS elements of a key], value columns up to what a walk's workgroups have; the 64 bytes
// of 32 elements lie at a place that depends on the column, so that columns read side by side from LDS come from different banks.
__host__ __device__ __forceinline__ constexpr int padded_values(int DV) { return DV <= 64 ? 64 : (DV + 127) / 128 * 128; }
template <int KS>
__device__ __forceinline__ int mark_place(int column, int tile) { return (tile / 2 ^ (column & (KS - 1))) * 32 + 4 * (tile % 2); }
// The terms of a wave's 16 columns from column `left` on, elements 32 s to 32 s + 31 and the 32 behind them, which lie in one line of 128 bytes: lanes swap halves so that an instruction writes whole ones.
template <int KS, int RANKS>
__device__ __forceinline__ void store_marks(uint16_t* marks, int DV, int left, int s, const u32x4a (&first)[3], const u32x4a (&second)[3]) {
    const int lane = threadIdx.x & 63, low = lane % 8;
    const bool upper = lane % 16 >= 8;
    const int column = left + low, at = mark_place<KS>(column, 2 * (s + upper)) + 8 * (lane / 16);
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
        u32x4a x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(upper ? first[r][i] : second[r][i]), 0x128, 0xf, 0xf, false));     // from 8 lanes on
            x[i] = upper ? other : first[r][i];
            y[i] = upper ? second[r][i] : other;
        }
        uint16_t* to = marks + static_cast<uint32_t>((r * padded_values(DV) + column) * 32 * KS + at);
        *reinterpret_cast<u32x4a*>(to) = x;
        *reinterpret_cast<u32x4a*>(to + 8 * 32 * KS) = y;      // column + 8, whose place is the same
    }
}
inline int64_t mark_elements(int ranks, int KS, int DV) { return static_cast<int64_t>(ranks) * padded_values(DV) * 32 * KS; }
// Of a segment: the matrix that takes the state before it to the state behind it, what it adds ([32 KS rows][value columns]), and whether the state before it is forgotten. The matrix lies as
// the products that take it load it: [32 columns][tile of rows][half of 8 columns][lane][4 columns].
__host__ __device__ __forceinline__ constexpr int transfer_matrix(int KS) { return 32 * KS * 32 * KS; }
__host__ __device__ __forceinline__ constexpr int transfer_floats(int KS, int DV) { return transfer_matrix(KS) + 32 * KS * padded_values(DV) + 4; }
template <int KS>
__device__ __forceinline__ int transfer_place(int tile, int r, int column) {      // row head_element(tile, r)
    return (((column / 32 * 2 * KS + tile) * 2 + column % 8 / 4) * 64 + column % 32 / 8 * 16 + (threadIdx.x & 63) / 16 * 4 + r) * 4 + column % 4;
}
template <int KS>
__device__ __forceinline__ void store_transfer(float* to, const f32x4 (&x)[2 * KS], bool matrix, int column, int values) {
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) to[matrix ? transfer_place<KS>(d, r, column) : transfer_matrix(KS) + head_element(d, r) * values + column] = x[d][r];
}
inline int64_t delta_elements(int ranks, int DV) { return static_cast<int64_t>(ranks) * kChunk * padded_values(DV); }

__device__ __forceinline__ int length_of(const DeltaArgs& p, int n) {
    if (p.lengths == nullptr) return p.T;
    const int length = p.lengths[n];
    return length < 0 ? 0 : (length < p.T ? length : p.T);
}

template <typename T>
__device__ __forceinline__ Terms<kTerms<T>> terms_of(const Raw<T, 8>& raw) {
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
// Fragment f = 0..5 of a lower triangular [64 x 64] matrix: rows of tile 0, 1, 2, 2, 3, 3, columns of half 0, 0, 0, 1, 0, 1. Of an upper one
// (a transposed lower one): rows of tile 0, 0, 1, 1, 2, 3, columns of half 0, 1, 0, 1, 1, 1.
__device__ __forceinline__ constexpr int lower_tile(int f) { return f < 2 ? f : (f < 4 ? 2 : 3); }
__device__ __forceinline__ constexpr int lower_half(int f) { return f == 3 || f == 5 ? 1 : 0; }
__device__ __forceinline__ constexpr int upper_tile(int f) { return f < 2 ? 0 : (f < 4 ? 1 : f - 2); }
__device__ __forceinline__ constexpr int upper_half(int f) { return f == 0 || f == 2 ? 0 : 1; }

// ------------------------------------------------------------------------------------------------------------------
// Keys and queries of a chunk in LDS
// ------------------------------------------------------------------------------------------------------------------
// [term][64 rows][32 KS], the 16 bytes of 8 elements at a place that depends on the row, so that 16 rows side by side are read from all banks and rows can
// come straight from memory, past the registers.
template <int SLOTS>                    // of 16 bytes in a row
__device__ __forceinline__ int slot_of(int row, int slot) {
    static_assert(SLOTS == 4 || SLOTS == 8 || SLOTS == 16, "rows of 64, 128 or 256 bytes");
    return slot ^ (SLOTS == 16 ? row & 15 : (SLOTS == 8 ? row >> 1 & 7 : row >> 2 & 3));
}
template <typename T, int KS> struct Rows {
    static constexpr int kSlots = 4 * KS, kStride = 32 * KS, kPlane = kChunk * kStride, kSize = kTerms<T> * kPlane;      // in elements

    __device__ __forceinline__ static void put(uint16_t* lds, int piece, const Terms<kTerms<T>>& x) {
        const int row = piece / kSlots;
        uint16_t* to = lds + row * kStride + 8 * slot_of<kSlots>(row, piece % kSlots);
#pragma unroll
        for (int n = 0; n < kTerms<T>; ++n) *reinterpret_cast<u32x4a*>(to + n * kPlane) = x.t[n];
    }
    // rows 16 tile.., elements 32 s..
    __device__ __forceinline__ static Terms<kTerms<T>> rows(const uint16_t* lds, int tile, int s) {
        const int lane = threadIdx.x & 63, row = lane % 16;
        const uint16_t* from = lds + 16 * tile * kStride + row * kStride + 8 * slot_of<kSlots>(row, 4 * s + lane / 16);
        Terms<kTerms<T>> r;
#pragma unroll
        for (int n = 0; n < kTerms<T>; ++n) r.t[n] = *reinterpret_cast<const u32x4a*>(from + n * kPlane);
        return r;
    }
    // the elements of `head_element(tile, ..)` as rows, steps of half `half` as places: four rows of 16 elements, transposed on their way by the LDS unit
    __device__ __forceinline__ static Terms<kTerms<T>> columns(const uint16_t* lds, int tile, int half) {
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        const int lane = threadIdx.x & 63, row = 4 * (lane / 16) + lane % 16 / 4;
        const uint16_t* from = lds + (32 * half + row) * kStride + 8 * slot_of<kSlots>(row, 4 * (tile / 2) + lane % 4) + 4 * (tile % 2);
        Terms<kTerms<T>> r;
#pragma unroll
        for (int n = 0; n < kTerms<T>; ++n) {
            const u32x2a low = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(from + n * kPlane)));
            const u32x2a high = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(from + n * kPlane + 16 * kStride)));
            r.t[n] = u32x4a{low[0], low[1], high[0], high[1]};
        }
        return r;
    }
    // elements head_element(tile, 0..3) of a row
    __device__ __forceinline__ static f32x4 four(const uint16_t* lds, int row, int tile) {
        const uint16_t* from = lds + row * kStride + 8 * slot_of<kSlots>(row, 4 * (tile / 2) + (threadIdx.x & 63) / 16) + 4 * (tile % 2);
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

// 16 bytes a lane from memory to LDS, a lane's behind the one before it: `lds` is the first lane's byte address. Written out, since the compiler lets every later read of LDS wait for what it
// knows to be on its way there; whoever reads waits (`arrived`) and passes a barrier first. m0 cannot be named as overwritten: the compiler keeps it from its registers and writes it
// itself only for what these kernels do not hold (registers with an index that varies, messages, other loads to LDS); its listing of them has no m0 but these.
__device__ __forceinline__ void to_lds(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(lds) : "memory");
}
__device__ __forceinline__ void to_lds(const void* base, uint32_t offset, uint32_t lds) {        // base: the same in all lanes
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(p))));
}
// A chunk's rows of 16 bytes times SLOTS to LDS in the order of `slot_of`, by WAVES waves; zeros for rows from `rows` on and behind `width` elements, from 16 bytes of them.
template <int SLOTS, int WAVES>
__device__ __forceinline__ void rows_to_lds(int wave, const uint16_t* base, int64_t step, int rows, int width, const void* zeros, uint16_t* lds) {
    constexpr int ROWS = 64 / SLOTS;    // of one instruction
    static_assert(ROWS * WAVES % 16 == 0, "a lane's place in a row is the same in all of its rows");
    const int lane = threadIdx.x & 63, row = wave * ROWS + lane / SLOTS, at = 8 * slot_of<SLOTS>(row, lane % SLOTS);
    const uint32_t to = lds_address(lds) + wave * 1024, offset = static_cast<uint32_t>(row * static_cast<int>(step) + at) * 2;
    const bool whole = rows >= kChunk && width >= 8 * SLOTS;
#pragma unroll
    for (int i = 0; i < kChunk / ROWS / WAVES; ++i) {
        const uint16_t* from = base + i * WAVES * ROWS * step;
        if (whole) {
            to_lds(from, offset, to + i * WAVES * 1024);
        } else {
            const bool there = i * WAVES * ROWS + row < rows && at < width;
            to_lds(there ? reinterpret_cast<const char*>(from) + offset : reinterpret_cast<const char*>(zeros), to + i * WAVES * 1024);
        }
    }
}

// Pieces of 8 elements of a chunk's rows on their way from memory, PER_ROW of a row, COUNT to a thread of THREADS: neighbouring threads take neighbouring pieces. Where
// rows are whole vectors within reach a thread has one offset for all of them; else, and in the last rows of a sequence, each element is looked at.
template <typename T, int PER_ROW, int THREADS> struct Staged {
    static constexpr int kCount = kChunk * PER_ROW / THREADS, kRows = THREADS / PER_ROW;      // rows from one of a thread's pieces to the next
    static_assert(THREADS % PER_ROW == 0 && kChunk % kRows == 0, "a thread's pieces lie in one column");
    Raw<T, 8> raw[kCount];
    // base: the chunk's first row; rows, width: how many rows and elements there are
    __device__ __forceinline__ void load(const T* base, int64_t step, int rows, int width, bool near) {
        const int row = threadIdx.x % THREADS / PER_ROW, at = 8 * (threadIdx.x % PER_ROW);
        if (near && rows >= kChunk) {
            const uint32_t offset = at < width ? static_cast<uint32_t>(row * static_cast<int>(step) + at) * sizeof(T) : 0u;
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                const char* from = reinterpret_cast<const char*>(base + i * kRows * step);
                const auto words = *reinterpret_cast<const typename Words<T, 8>::type*>(from + offset);
#pragma unroll
                for (int w = 0; w < Raw<T, 8>::kWords; ++w) raw[i].w[w] = words[w];
            }
            if (width < 8 * PER_ROW) {
#pragma unroll
                for (int i = 0; i < kCount; ++i)
#pragma unroll
                    for (int w = 0; w < Raw<T, 8>::kWords; ++w) raw[i].w[w] = at < width ? raw[i].w[w] : 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                if (row + i * kRows < rows && at < width) raw[i].load(base, (row + i * kRows) * step + at, width - at);
                else raw[i].clear();
            }
        }
    }
};
template <typename T, int KS, int THREADS>
__device__ __forceinline__ void put_rows(const Staged<T, 4 * KS, THREADS>& x, uint16_t* lds) {
#pragma unroll
    for (int i = 0; i < x.kCount; ++i) {
        Rows<T, KS>::put(lds, threadIdx.x % THREADS + i * THREADS, terms_of(x.raw[i]));
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Values of a chunk in LDS
// ------------------------------------------------------------------------------------------------------------------
// [64][16 WAVES], 16-bit elements as above, float32 ones with a pitch of their own. A wave reads its 16 columns in the accumulators' layout and, once it has them, uses the room to
// turn what it writes into rows.
template <typename T, int WAVES> struct Tile {
    static constexpr int kColumns = 16 * WAVES, kSlots = 2 * WAVES, kStride = sizeof(T) == 4 ? kColumns + 8 : kColumns, kSize = kChunk * kStride;
    // byte address of a column's 16-bit (32-bit: its) element within the wave's 16
    template <typename E>
    __device__ __forceinline__ static uint32_t place(int row, int column) {
        const int wave = threadIdx.x >> 6;
        if constexpr (sizeof(T) == 4) return (row * kStride + 16 * wave) * 4 + column * sizeof(E);
        else return row * kStride * 2 + 16 * slot_of<kSlots>(row, 2 * wave + column / 8) + 2 * (column % 8);
    }
    template <int THREADS>
    __device__ __forceinline__ static void put(T* lds, const Staged<T, 2 * WAVES, THREADS>& x) {
#pragma unroll
        for (int i = 0; i < x.kCount; ++i) {
            const int row = threadIdx.x % THREADS / kSlots + i * x.kRows, slot = threadIdx.x % kSlots;
            T* to = lds + row * kStride + 8 * (sizeof(T) == 4 ? slot : slot_of<kSlots>(row, slot));
#pragma unroll
            for (int w = 0; w < Raw<T, 8>::kWords; w += 4)
                reinterpret_cast<u32x4a*>(to)[w / 4] = u32x4a{x.raw[i].w[w], x.raw[i].w[w + 1], x.raw[i].w[w + 2], x.raw[i].w[w + 3]};
        }
    }
    // rows 16 i + 4 (lane / 16) + 0..3 of the lane's column
    __device__ __forceinline__ static f32x4 get(const T* lds, int i) {
        const int lane = threadIdx.x & 63, l = lane % 16, row = 4 * (lane / 16);
        f32x4 r;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(lds) + place<float>(16 * i + row + j, l));
        } else {
            typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
            const char* from = reinterpret_cast<const char*>(lds) + place<T>(row + l / 4, 4 * (l % 4)) + 16 * i * kStride * 2;
            const u32x2a words = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(from)));
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = element<T>(words[j / 2], j % 2);
        }
        return r;
    }
    // The wave's 16 columns of x as E, in the room of 16 columns of T.
    template <typename E>
    __device__ __forceinline__ static void turn(T* lds, const E (&x)[16]) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            *reinterpret_cast<E*>(reinterpret_cast<char*>(lds) + place<E>(4 * (lane / 16) + i % 4, lane % 16) + 16 * (i / 4) * kStride * sizeof(T)) = x[i];
    }
    // 16 bytes of them: piece `lane + 64 i` of row (...) / pieces a row
    template <typename E>
    __device__ __forceinline__ static u32x4a piece(const T* lds, int i, int* row, int* at) {
        constexpr int EACH = 16 / sizeof(E), PER_ROW = 16 / EACH;
        const int lane = threadIdx.x & 63, index = lane + 64 * i;
        *row = index / PER_ROW, *at = EACH * (index % PER_ROW);
        return *reinterpret_cast<const u32x4a*>(reinterpret_cast<const char*>(lds) + place<E>(*row, *at));
    }
    // The wave's 16 columns into its room...
    __device__ __forceinline__ static void turn_values(T* lds, const f32x4 (&x)[4]) {
        T y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = from_float<T>(x[i / 4][i % 4]);
        turn<T>(lds, y);
    }
    // ... and from there to rows of memory; `rows` are written, those from `live` on as zeros.
    __device__ __forceinline__ static void write(const T* lds, T* base, int64_t step, int rows, int live, int width, bool near) {
        __builtin_amdgcn_wave_barrier();
        constexpr int EACH = 16 / sizeof(T), COUNT = kChunk / 64 * 16 / EACH;
        const bool whole = near && live >= kChunk && width >= 16;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            int row, at;
            const u32x4a words = piece<T>(lds, i, &row, &at);
            if (whole) {
                *reinterpret_cast<typename Words<T, kVec<T>>::type*>(reinterpret_cast<char*>(base) + static_cast<uint32_t>(row * static_cast<int>(step) + at) * sizeof(T)) = words;
            } else if (row < rows) {
                T* to = base + row * step + at;
#pragma unroll
                for (int j = 0; j < EACH; ++j) {
                    const uint32_t word = row < live ? words[j * sizeof(T) / 4] : 0u;
                    if (at + j >= width) continue;
                    if constexpr (sizeof(T) == 4) to[j] = __uint_as_float(word);
                    else to[j].bits = static_cast<uint16_t>(j % 2 ? word >> 16 : word);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    // The terms of the wave's 16 columns to where those are in planes [rank][16 columns][64][16].
    template <int RANKS>
    __device__ __forceinline__ static void write_terms(T* lds, const f32x4 (&x)[4], uint16_t* base, int columns) {
        uint32_t words[8][RANKS];
#pragma unroll
        for (int i = 0; i < 8; ++i) split_pair<RANKS>(x[i / 2][2 * (i % 2)], x[i / 2][2 * (i % 2) + 1], words[i]);
#pragma unroll
        for (int n = 0; n < RANKS; ++n) {
            uint16_t y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = static_cast<uint16_t>(i % 2 ? words[i / 2][n] >> 16 : words[i / 2][n]);
            turn<uint16_t>(lds, y);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                int row, at;
                const u32x4a piece16 = piece<uint16_t>(lds, i, &row, &at);
                *reinterpret_cast<u32x4a*>(base + static_cast<uint32_t>(n * kChunk * columns + row * 16 + at)) = piece16;
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// A chunk's block on its way to LDS.
template <int PIECES, int WAVES, int LAST> struct StagedBlock {     // the first PIECES - 1 and piece LAST
    static constexpr int kCount = (PIECES + WAVES - 1) / WAVES;
    u32x4a words[kCount];
    __device__ __forceinline__ void load(const uint32_t* from) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            if (wave + i * WAVES < PIECES) words[i] = *reinterpret_cast<const u32x4a*>(from + (wave + i * WAVES < PIECES - 1 ? wave + i * WAVES : LAST) * 256 + lane * 4);
    }
    __device__ __forceinline__ void store(uint32_t* lds) const {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            if (wave + i * WAVES < PIECES) *reinterpret_cast<u32x4a*>(lds + (wave + i * WAVES) * 256 + lane * 4) = words[i];
    }
};
// Threads of a walk's workgroup: with one term to an element four waves more, which load.
template <typename T> __host__ __device__ __forceinline__ constexpr int walk_threads(int waves) { return 64 * (waves + (kTerms<T> == 1 ? 4 : 0)); }
// What a walk reads of a chunk: keys, queries, values (or the gradient of what is read) and the chunk's block, without queries and scores if not ALL; through registers...
template <int PIECES, bool ALL> inline constexpr int kTaken = ALL ? PIECES : kBlocks * 3 + 1;      // of a block's pieces: without the scores if not ALL
template <typename T, int KS, int WAVES, int PIECES, bool ALL> struct StagedChunk {
    Staged<T, 4 * KS, 64 * WAVES> k, q;
    Staged<T, 2 * WAVES, 64 * WAVES> v;
    StagedBlock<kTaken<PIECES, ALL>, WAVES, PIECES - 1> block;
    __device__ __forceinline__ void load(const DeltaArgs& p, const T* keys, const T* queries, const T* values, int64_t step, int rows, int width, const uint32_t* from) {
        k.load(keys, p.k.step, rows, p.DK, p.near_keys);
        if constexpr (ALL) q.load(queries, p.q.step, rows, p.DK, p.near_keys);
        v.load(values, step, rows, width, p.near_values);
        block.load(from);
    }
    __device__ __forceinline__ void store(uint16_t* keys, uint16_t* queries, T* tile, uint32_t* to) const {
        put_rows<T, KS, 64 * WAVES>(k, keys);
        if constexpr (ALL) put_rows<T, KS, 64 * WAVES>(q, queries);
        Tile<T, WAVES>::put(tile, v);
        block.store(to);
    }
};
// ... or, with one term to an element, as they are, a chunk ahead into the other buffer: past the registers where rows are whole vectors, else through them at once. Loads past the registers wait for
// room on their way, some 3000 of 13000 cycles a chunk where the waves that walk do it: four more do nothing but load.
template <typename T, int KS, int WAVES, int PIECES, bool ALL = true> struct ChunkReader {
    static constexpr bool kDirect = kTerms<T> == 1;
    static constexpr int kLoaders = kDirect ? 4 : 0, kBuffers = kDirect ? 2 : 1;
    struct Buffers {
        uint16_t keys[Rows<T, KS>::kSize], queries[Rows<T, KS>::kSize];
        T tile[Tile<T, WAVES>::kSize];
        uint32_t block[kTaken<PIECES, ALL> * 256];
    };
    struct Chunk {                      // its first row of keys, queries and values, and how many rows and values there are
        const T *keys, *queries, *values;
        int64_t step;
        int rows, width;
        const uint32_t* block;
    };
    struct Nothing {};
    std::conditional_t<kDirect, Nothing, StagedChunk<T, KS, WAVES, PIECES, ALL>> next;

    __device__ __forceinline__ void fetch(const DeltaArgs& p, const Chunk& c, Buffers& to) {
        if constexpr (!kDirect) {
            next.load(p, c.keys, c.queries, c.values, c.step, c.rows, c.width, c.block);
        } else {
            constexpr int W = kLoaders;
            const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
            const uint32_t* zeros = c.block + block_vectors((PIECES - 1) / kBlocks - 3) + kZeros;
            if (p.near_keys) {
                rows_to_lds<4 * KS, W>(wave, reinterpret_cast<const uint16_t*>(c.keys), p.k.step, c.rows, p.DK, zeros, to.keys);
                if constexpr (ALL) rows_to_lds<4 * KS, W>(wave, reinterpret_cast<const uint16_t*>(c.queries), p.q.step, c.rows, p.DK, zeros, to.queries);
            } else {
                Staged<T, 4 * KS, 64 * W> x;
                x.load(c.keys, p.k.step, c.rows, p.DK, false);
                put_rows<T, KS, 64 * W>(x, to.keys);
                if constexpr (ALL) {
                    x.load(c.queries, p.q.step, c.rows, p.DK, false);
                    put_rows<T, KS, 64 * W>(x, to.queries);
                }
            }
            if (p.near_values) {
                rows_to_lds<2 * WAVES, W>(wave, reinterpret_cast<const uint16_t*>(c.values), c.step, c.rows, c.width, zeros, reinterpret_cast<uint16_t*>(to.tile));
            } else {
                Staged<T, 2 * WAVES, 64 * W> x;
                x.load(c.values, c.step, c.rows, c.width, false);
                Tile<T, WAVES>::put(to.tile, x);
            }
            const uint32_t at = lds_address(to.block) + wave * 1024;
#pragma unroll
            for (int i = 0; i < (kTaken<PIECES, ALL> + W - 1) / W; ++i) {
                const int piece = wave + i * W;
                if (piece < kTaken<PIECES, ALL>) to_lds(c.block + (piece < kTaken<PIECES, ALL> - 1 ? piece : PIECES - 1) * 256, lane * 16u, at + i * W * 1024);
            }
        }
    }
    // Has the chunk that was fetched last in LDS, for all waves; the one before it may be overwritten from then on.
    __device__ __forceinline__ void wait(Buffers& to) {
        if constexpr (kDirect) {
            __syncthreads();
        } else {
            __syncthreads();
            next.store(to.keys, to.queries, to.tile, to.block);
            __syncthreads();
        }
    }
};
template <int N>
__device__ __forceinline__ Terms<N> block_terms(const uint32_t* lds, int fragment) {
    Terms<N> r;
#pragma unroll
    for (int n = 0; n < N; ++n) r.t[n] = *reinterpret_cast<const u32x4a*>(lds + (fragment * N + n) * 256 + (threadIdx.x & 63) * 4);
    return r;
}
// Of a vector of a chunk: rows 16 i + 4 (lane / 16) + 0..3
__device__ __forceinline__ f32x4 row_factors(const uint32_t* vectors, int which, int i) {
    return *reinterpret_cast<const f32x4*>(vectors + which + 16 * i + 4 * ((threadIdx.x & 63) / 16));
}
// What a vanished decay would multiply is dropped, infinities and NaN as well.
__device__ __forceinline__ void drop(f32x4& x, const f32x4& factor) {
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = factor[r] == 0.0f ? 0.0f : x[r];
}

// In a matrix product the zeros above the diagonal and between two parts of a chunk do not keep infinities and NaN from steps that they do not concern. Where there are any (times 0 they are
// not 0), they are taken out of x, rows in the accumulators' layout, and the rows that they are to reach, their own and those behind them in the same part, come back as bits 4 i + r.
__device__ __forceinline__ bool all_finite(const f32x4 (&x)[4]) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = fmaf(x[i / 4][i % 4], 0.0f, sum);
    return __ballot(sum != 0.0f) == 0;
}
__device__ __forceinline__ uint32_t take_out(f32x4 (&x)[4], uint64_t fresh) {
    const int first = 4 * ((threadIdx.x & 63) / 16);
    uint32_t own = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const bool finite = fabsf(x[i / 4][i % 4]) < __builtin_inff();
        own |= finite ? 0u : 1u << i;
        x[i / 4][i % 4] = finite ? x[i / 4][i % 4] : 0.0f;
    }
    // bit t: step t of the lane's column
    uint64_t rows = static_cast<uint64_t>((own & 15u) | (own & 240u) << 12 ) << first | static_cast<uint64_t>((own >> 8 & 15u) | (own >> 12) << 16) << (32 + first);
    rows |= __shfl_xor(rows, 16, 64);
    rows |= __shfl_xor(rows, 32, 64);
    uint64_t open = ~fresh;             // bit t: no start among the last d steps up to t
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        rows |= open & rows << d;
        open &= open << d;
    }
    const uint32_t low = static_cast<uint32_t>(rows >> first), high = static_cast<uint32_t>(rows >> (32 + first));
    return (low & 15u) | (low >> 12 & 240u) | (high & 15u) << 8 | (high >> 16 & 15u) << 12;
}
__device__ __forceinline__ void put_back(f32x4 (&x)[4], uint32_t rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][r] = rows >> (4 * i + r) & 1 ? __builtin_nanf("") : x[i][r];
}

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

// The same for two sums as pairs of float32, without float64: the difference of the larger parts and what its rounding lost, exactly, then the smaller parts.
struct Sum {
    float large, small;
};
__device__ __forceinline__ Sum sum_of(double x) {
    const float large = static_cast<float>(x);
    return {large, static_cast<float>(x - large)};
}
__device__ __forceinline__ float decay_between(const Sum& from, const Sum& to) {
    const float x = to.large - from.large, back = x - to.large;
    const float lost = (to.large - (x - back)) - (from.large + back);
    const float whole = __builtin_rintf(x), rest = (x - whole) + (lost + (to.small - from.small));
    return x <= -160.0f ? 0.0f : ldexpf(__builtin_amdgcn_exp2f(rest), static_cast<int>(fminf(whole, 1000.0f)));
}

// Row i of a factor that a vanished decay has made 0 drops what it would multiply, infinities and NaN as well.
__device__ __forceinline__ float kept(float factor, float x) { return factor == 0.0f ? 0.0f : factor * x; }

// Workgroups to heads and parts of them so that the parts of a head, which read the same keys, run on one of the 8 dies and share its cache: neighbouring workgroups go to
// different dies. False: nothing to do.
__device__ __forceinline__ bool part_of_head(int heads, int parts, int* head, int* part) {
    constexpr int kDies = 8;
    const int index = static_cast<int>(group_index()), die = index % kDies, order = index / kDies;
    *part = order % parts;
    *head = order / parts * kDies + die;
    return *head < heads;
}
inline dim3 head_grid(int heads, int parts) { return grid_of(static_cast<int64_t>((heads + 7) / 8 * 8) * parts); }

// Fragments, decays and inverses of all chunks; transposed for the backward pass.
template <typename T, int KS, int RANKS, bool BACKWARD> void launch_chunks(const DeltaArgs& p, hipStream_t stream);

// Workgroups to a segment on its first walk, and what joins the states (backward: from the last segment on).
inline int transfer_parts(int waves, int KS, int DV) { return (DV + 16 * waves - 1) / (16 * waves) + (2 * KS + waves - 1) / waves; }
template <int KS> void launch_join(const DeltaArgs& p, bool backward, hipStream_t stream);
int delta_segments(const snnf_delta_rule_call* call, bool backward);
size_t delta_segment_floats(const snnf_delta_rule_call* call, bool backward);
void set_segments(DeltaArgs& p, const snnf_delta_rule_call* call, bool backward, float* workspace);

int check_delta(const char* name, const snnf_delta_rule_call* call);
DeltaArgs delta_args(const snnf_delta_rule_call* call);
int64_t delta_chunks(const snnf_delta_rule_call* call);
int delta_ranks(const snnf_delta_rule_call* call, bool training);
int64_t delta_mark_elements(const snnf_delta_rule_call* call);
// Whether a chunk's rows lie within reach of 31-bit offsets, and, where they go to LDS as they are, on 16 bytes.
inline bool near_by(const HeadView& x, int dtype, bool read) {
    const bool reach = x.step >= 0 && x.step <= 0x7fffffff / (kChunk * dtype_size(dtype)) - 1024;
    return reach && (!read || dtype != SNNF_BF16 || (aligned_to(x.data, 16) && (x.step | x.row | x.head) % 8 == 0));
}
// Workgroups of 32 value columns where those of 64 leave half of the chip idle: half as much to read and write for each (4096 x 4 x 16 heads of 128 bfloat16, forward and backward: 1109 us, with 64 columns
// 1187). Of 128, with eight waves, a head's keys are read once, but no room is left for waves that load: 16, 20 and 32 x 16 heads of 1024 steps take 216, 335 and 400 us, with 64 columns 214, 268
// and 384.
inline bool two_waves(const DeltaArgs& p) { return p.DV > 32 && 2 * p.N * p.HV * p.segments * ((p.DV + 63) / 64) <= compute_units(); }
}  // namespace snnf
