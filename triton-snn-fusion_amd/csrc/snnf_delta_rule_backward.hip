// Gated delta rule, gradient. With U = diag(beta) delta, P = scale (Q K^T o D), S the state before a chunk and R the gradient of the state behind it:
//     dU = P^T dout + diag(e^(G_64 - G)) K R,   Z = (I + L^T diag(beta))^-1 dU,   dv = diag(beta) Z
//     dS = e^(G_64) R + Q^T diag(scale e^G) dout - K^T diag(e^G) dv                         (the walk back, which leaves Z and R)
//     dP_ij = scale D_ij dout_i . U_j,   dL_ij = -D_ij dv_i . U_j
//     dq = diag(scale e^G) dout S^T + dP K
//     dk = diag(e^(G_64 - G)) U R^T - diag(e^G) dv S^T + dP^T Q + (dL + dL^T) K,   dbeta = Z . delta          (chunk by chunk)
// Gates: what raises G_i raises with every query the scores and the state it reads, and lowers what keys leave. Collected by operand,
//     dG_i = q_i . dq_i - k_i . dk_i + 2 (beta_i dbeta_i - v_i . dv_i),    dgate_t = sum of dG_i for i >= t in the chunk + <S', R>
// where S' is the state behind the chunk, so that no sum runs over more than a chunk: <S', R> = e^(G_64) <S, R> + sum_i e^(G_64 - G_i) k_i . (R U_i).
#include "snnf_delta_rule.h"

namespace snnf {
namespace {

// ------------------------------------------------------------------------------------------------------------------
// The walk back
// ------------------------------------------------------------------------------------------------------------------
// As the walk forward, with R in accumulators: 4096 x 4 x 16 heads of 128 bfloat16 305 us, 4.8 a chunk.
// In segments where heads are few, as the walk forward: a segment's effect on R is A^T R + B, and a first walk (TRANSFER) takes the identity and no gradient of its outputs for A^T, the
// gradient of its outputs and no R for B.
template <typename T, int KS, int WAVES, int RANKS, bool TRANSFER>
__global__ __launch_bounds__(kTerms<T> == 1 ? 512 : 256) void delta_walk_back_kernel(DeltaArgs p) {
    constexpr int TERMS = kTerms<T>, PIPE = TERMS == 1 ? 2 : 1;
    using Lds = Rows<T, KS>;
    using Values = Tile<T, WAVES>;
    using Reader = ChunkReader<T, KS, WAVES, block_pieces(3)>;
    __shared__ alignas(16) typename Reader::Buffers lds[Reader::kBuffers];
    const int value_parts = (p.DV + Values::kColumns - 1) / Values::kColumns, segments = TRANSFER ? p.segments - 1 : p.segments;
    int item, columns;
    if (!part_of_head(p.N * p.HV * segments, TRANSFER ? value_parts + (2 * KS + WAVES - 1) / WAVES : value_parts, &item, &columns)) return;
    const int head = item / segments, segment = item % segments + TRANSFER, n = head / p.HV, hv = head % p.HV, h = hv / (p.HV / p.H), limit = length_of(p, n);
    const int chunks = (limit + kChunk - 1) / kChunk, begin = segment * p.per, last = chunks == 0 ? 0 : (chunks - 1) / p.per;
    const int live = segment < last ? begin + p.per : chunks;
    const bool matrix = TRANSFER && columns >= value_parts;
    if (segment > last || (matrix && segment == last)) return;      // what comes behind the last segment is known
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane / 16;
    const int left = (matrix ? columns - value_parts : columns) * Values::kColumns, mine = left + 16 * wave, column = mine + lane % 16;
    const bool there = column < (matrix ? 32 * KS : p.DV);
    const T* k_base = static_cast<const T*>(p.k.data) + n * p.k.row + h * p.k.head;
    const T* q_base = static_cast<const T*>(p.q.data) + n * p.q.row + h * p.q.head;
    const T* o_base = static_cast<const T*>(p.dout.data) + n * p.dout.row + hv * p.dout.head + (matrix ? 0 : left);
    T* v_base = static_cast<T*>(const_cast<void*>(p.dv.data)) + n * p.dv.row + hv * p.dv.head + mine;
    const auto place = [&](int chunk) {
        const int64_t first = static_cast<int64_t>(chunk) * kChunk;
        return typename Reader::Chunk{k_base + first * p.k.step, q_base + first * p.q.step, o_base + first * p.dout.step, p.dout.step, limit - chunk * kChunk, matrix ? 0 : p.DV - left,
                                      p.blocks + (static_cast<int64_t>(head) * p.chunks + chunk) * block_words(3)};
    };
    Reader reader;
    const auto fetch = [&](int chunk) {
        if (chunk >= begin) reader.fetch(p, place(chunk), lds[chunk % Reader::kBuffers]);
    };
    if constexpr (Reader::kDirect)
        if (wave >= WAVES) {
            fetch(live - 1);
            for (int chunk = live - 1; chunk >= begin; --chunk) {
                arrived();
                __syncthreads();
                fetch(chunk - 1);
            }
            return;
        }
    const int64_t cell = static_cast<int64_t>(head) * p.DK * p.DV + column;
    const float* behind = nullptr;
    if (segment == last) behind = p.dstate == nullptr ? nullptr : p.dstate + cell;
    else if constexpr (!TRANSFER) behind = p.between + (static_cast<int64_t>(head) * segments + segment) * p.DK * p.DV + column;
    f32x4 later[2 * KS];
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = head_element(d, r);
            later[d][r] = behind != nullptr && there && row < p.DK ? behind[static_cast<int64_t>(row) * p.DV] : (matrix && row == column ? 1.0f : 0.0f);
        }
    bool forgotten = false;
    if constexpr (!Reader::kDirect) fetch(live - 1);
    for (int chunk = live - 1; chunk >= begin; --chunk) {
        const int64_t index = static_cast<int64_t>(head) * p.chunks + chunk;
        typename Reader::Buffers& here = lds[chunk % Reader::kBuffers];
        const uint16_t *keys = here.keys, *queries = here.queries;
        T* tile = here.tile;
        const uint32_t *block = here.block, *vectors = block + block_vectors(3);
        reader.wait(here);
        if constexpr (!Reader::kDirect) fetch(chunk - 1);
        now();
        // K R
        f32x4 pull[4], dout[4], z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pull[i] = z[i] = f32x4{0, 0, 0, 0};
        Terms<TERMS> a[PIPE][4];
        Terms<3> x[2];
        const auto load = [&](int s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) a[s % PIPE][i] = Lds::rows(keys, i, s);
        };
        load(0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (PIPE == 2 && s + 1 < KS) load(s + 1);
            now();
            x[s % 2] = split<3>(later[2 * s], later[2 * s + 1]);
            if constexpr (!TRANSFER)
                if (s % 2 == 1) store_marks<KS, RANKS>(p.later + index * (RANKS * padded_values(p.DV) * 32 * KS), p.DV, mine, s - 1, x[0].t, x[1].t);
#pragma unroll
            for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                for (int j = 0; j <= rank; ++j)
                    if (j < TERMS) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) pull[i] = mfma(a[s % PIPE][i].t[j], x[s % 2].t[rank - j], pull[i]);
                    }
            if (PIPE == 1 && s + 1 < KS) load(s + 1);
        }
        const bool broken = __builtin_amdgcn_readfirstlane(vectors[kBroken]) != 0;
        const float rest = __uint_as_float(__builtin_amdgcn_readfirstlane(vectors[kSince + kChunk - 1]));
        forgotten = forgotten || rest == 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 until = row_factors(vectors, kUntil, i);
            if (broken) drop(pull[i], until);
            pull[i] *= until;
            dout[i] = Values::get(tile, i);
        }
        // dU, then Z
        if (!matrix) {
            const Terms<TERMS> x[2] = {split<TERMS>(dout[0], dout[1]), split<TERMS>(dout[2], dout[3])};
            Terms<3> scores[kBlocks];
#pragma unroll
            for (int f = 0; f < kBlocks; ++f) scores[f] = block_terms<3>(block + kBlocks * 3 * 256, f);
            now();
#pragma unroll
            for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                for (int j = 0; j <= rank; ++j)
                    if (rank - j < TERMS) {
#pragma unroll
                        for (int f = 0; f < kBlocks; ++f) pull[upper_tile(f)] = mfma(scores[f].t[j], x[upper_half(f)].t[rank - j], pull[upper_tile(f)]);
                    }
        }
        {
            Terms<3> inverse[kBlocks];
#pragma unroll
            for (int f = 0; f < kBlocks; ++f) inverse[f] = block_terms<3>(block, f);
            now();
            const Terms<3> x[2] = {split<3>(pull[0], pull[1]), split<3>(pull[2], pull[3])};
#pragma unroll
            for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                for (int j = 0; j <= rank; ++j)
#pragma unroll
                    for (int f = 0; f < kBlocks; ++f) z[upper_tile(f)] = mfma(inverse[f].t[j], x[upper_half(f)].t[rank - j], z[upper_tile(f)]);
        }
        if constexpr (!TRANSFER) Values::template write_terms<RANKS>(tile, z, p.pulls + index * (RANKS * kChunk * padded_values(p.DV)) + mine * kChunk, padded_values(p.DV));
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] *= row_factors(vectors, kBeta, i);
        if constexpr (!TRANSFER) Values::turn_values(tile, z);
        if constexpr (!TRANSFER) Values::write(tile, v_base + static_cast<int64_t>(chunk) * kChunk * p.dv.step, p.dv.step, p.T - chunk * kChunk, limit - chunk * kChunk, p.DV - mine, p.near_values);
        // R in front of the chunk
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 since = row_factors(vectors, kSince, i);
            if (broken) drop(z[i], since), drop(dout[i], since);
            z[i] *= -since;
            dout[i] *= since * p.scale;
        }
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d) {
            if (broken) drop(later[d], f32x4{rest, rest, rest, rest});
            later[d] *= rest;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                if (matrix && which == 1) continue;
                Terms<TERMS> c[2 * KS];
#pragma unroll
                for (int d = 0; d < 2 * KS; ++d) c[d] = Lds::columns(which == 0 ? keys : queries, d, half);
                now();
                const Terms<3> x = which == 0 ? split<3>(z[2 * half], z[2 * half + 1]) : split<3>(dout[2 * half], dout[2 * half + 1]);
#pragma unroll
                for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                    for (int j = 0; j <= rank; ++j)
                        if (j < TERMS) {
#pragma unroll
                            for (int d = 0; d < 2 * KS; ++d) later[d] = mfma(c[d].t[j], x.t[rank - j], later[d]);
                        }
            }
    }
    if constexpr (TRANSFER) {
        float* to = p.transfers + static_cast<int64_t>(item) * transfer_floats(KS, p.DV);
        if (there) store_transfer<KS>(to, later, matrix, column, padded_values(p.DV));
        if (matrix && columns == value_parts && threadIdx.x == 0) to[transfer_floats(KS, p.DV) - 4] = forgotten ? 1.0f : 0.0f;
        return;
    }
    if (segment == last) {
        for (int t = chunks * kChunk + wave * 4 + group; t < p.T; t += 4 * WAVES)      // padding
            for (int c = left + lane % 16; c < p.DV && c < left + Values::kColumns; c += 16) v_base[t * p.dv.step + c - mine] = from_float<T>(0.0f);
    }
    if (segment == 0) {
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = head_element(d, r);
                if (there && row < p.DK) p.dstate_in[cell + static_cast<int64_t>(row) * p.DV] = later[d][r];
            }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Gradients chunk by chunk
// ------------------------------------------------------------------------------------------------------------------
// Of queries and keys transposed, [DK x steps]: a wave owns 16 steps as columns, so that dP and dL, contracted over steps next, are multiplied as they lie in
// accumulators. Those are worked out twice, with the wave's steps as rows and as columns of the matrix.
// A row of 32 value columns in LDS: [term][64 rows][32], 16 bytes at a place that depends on the row.
__device__ __forceinline__ uint32_t value_place(int row, int slot) { return static_cast<uint32_t>(row * 32 + 8 * slot_of<4>(row, slot)); }
template <int N>
__device__ __forceinline__ Terms<N> value_rows(const uint16_t* lds, int tile) {
    const int lane = threadIdx.x & 63;
    const uint16_t* from = lds + 16 * tile * 32 + value_place(lane % 16, lane / 16);
    Terms<N> r;
#pragma unroll
    for (int n = 0; n < N; ++n) r.t[n] = *reinterpret_cast<const u32x4a*>(from + n * kChunk * 32);
    return r;
}
// Two times 16 columns of 64 steps to there, instruction `part` of four.
__device__ __forceinline__ void value_rows_to_lds(const uint16_t* from, uint16_t* lds, int part) {
    const int lane = threadIdx.x & 63, row = 16 * part + lane / 4, slot = slot_of<4>(row, lane % 4);
    to_lds(from, static_cast<uint32_t>(slot / 2 * kChunk * 16 + row * 16 + slot % 2 * 8) * 2, lds_address(lds) + part * 1024);
}
// Of a state's 32 value columns [32][32 KS]: elements of `head_element(tile, ..)` as rows, value columns as places, in order.
template <int N, int KS>
__device__ __forceinline__ Terms<N> state_columns(const uint16_t* lds, int tile) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const int lane = threadIdx.x & 63, column = 8 * (lane / 16) + lane % 16 / 4;
    const uint16_t* low = lds + column * 32 * KS + mark_place<KS>(column, tile) + 8 * (lane % 4);
    const uint16_t* high = lds + (column + 4) * 32 * KS + mark_place<KS>(column + 4, tile) + 8 * (lane % 4);
    Terms<N> r;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const u32x2a a = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(low + n * 1024 * KS)));
        const u32x2a b = __builtin_bit_cast(u32x2a, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(high + n * 1024 * KS)));
        r.t[n] = u32x4a{a[0], a[1], b[0], b[1]};
    }
    return r;
}
template <int N>
__device__ __forceinline__ float term_sum(const Terms<N>& x, int j) {
    float v = 0.0f;
#pragma unroll
    for (int n = N - 1; n >= 0; --n) v += element<bf16_t>(x.t[n][j / 2], j % 2);
    return v;
}
// Eight elements next to each other
template <typename T>
__device__ __forceinline__ void store_eight(T* to, int left, const f32x4& x, const f32x4& y) {
    Raw<T, 8> raw;
#pragma unroll
    for (int r = 0; r < 4; r += 2) raw.put(r, x[r], x[r + 1]), raw.put(4 + r, y[r], y[r + 1]);
    if (left > 0) raw.store(to, 0, left);
}
template <typename T>
__device__ __forceinline__ void store_gate(const DeltaArgs& p, const HeadView& x, int t, int n, int hv, float v) {
    if (x.data == nullptr) return;
    const int64_t at = t * x.step + n * x.row + hv * x.head;
    if (p.gate_float) static_cast<float*>(const_cast<void*>(x.data))[at] = v;
    else static_cast<T*>(const_cast<void*>(x.data))[at] = from_float<T>(v);
}

// Where all gradients are rounded to 16 bits the logarithm is rounded to float32: a decay by 2^-10 is off by 2^-21 then.
template <bool FINE>
__device__ __forceinline__ float decay_apart(const Sum& one, const Sum& other, bool ahead) {
    if constexpr (FINE) {
        return ahead ? decay_between(other, one) : decay_between(one, other);
    } else {
        const float x = (one.large - other.large) + (one.small - other.small);
        return __builtin_amdgcn_exp2f(ahead ? x : -x);
    }
}

// Two waves to 16 steps: the first works out dL, the second dP, and each has half of the head's elements of everything else; they exchange dL and dP through LDS. A workgroup takes one chunk after the
// other, each in pieces of 32 value columns and then a last one of keys and queries; with bfloat16, two terms to what the walks left, four more waves load the next piece while one is worked on.
// Bound by memory and by the phases between barriers: 4096 chunks of 128 bfloat16 elements read and write 1.2 GB in 370 us (3.2 TB/s; without waves of their own for the loads 435).
template <typename T, int KS, int RANKS> struct GradientPieces {
    static constexpr int TERMS = kTerms<T>, BUFFERS = TERMS == 1 && RANKS == 2 ? 2 : 1;     // by the room in LDS
    static constexpr int THREADS = BUFFERS == 2 ? 768 : 512;
    struct Slice {                      // 32 value columns of everything
        uint16_t marks[RANKS][1024 * KS], later[RANKS][1024 * KS], deltas[RANKS][kChunk * 32], pulls[RANKS][kChunk * 32], douts[TERMS][kChunk * 32];
    };
    struct Heads {
        uint16_t keys[Rows<T, KS>::kSize], queries[Rows<T, KS>::kSize];
        uint32_t between[2][4][2][RANKS][256];     // of 16 steps: dL and dP by rows, then dP by columns; halves of the other steps
    };
    union Piece {
        Slice slice;
        Heads heads;
    };
};

// SHARED: whether value heads share queries and keys, whose gradients are their sums then, held over the chunks of a head's members.
template <typename T, int KS, int RANKS, bool SHARED>
__global__ __launch_bounds__((GradientPieces<T, KS, RANKS>::THREADS)) void delta_gradient_kernel(DeltaArgs p) {
    using Lds = Rows<T, KS>;
    using Pieces = GradientPieces<T, KS, RANKS>;
    constexpr int TERMS = Pieces::TERMS, BUFFERS = Pieces::BUFFERS;
    constexpr bool LOADERS = BUFFERS == 2;
    __shared__ alignas(16) typename Pieces::Piece lds[BUFFERS];
    __shared__ alignas(16) Sum total[kChunk];
    __shared__ alignas(16) int part[kChunk];
    __shared__ alignas(16) float betas[kChunk], dsums[2][kChunk], tails[2][kChunk], own_sums[kChunk], dots[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = wave / 4 % 2, w = wave % 4, group = lane / 16, column = lane % 16;
    const int own = 16 * w + column, members = SHARED ? p.HV / p.H : 1, columns = padded_values(p.DV), slices = (p.DV + 31) / 32;
    const int places = p.N * p.H * p.chunks;
    struct Item {                       // a chunk of a value head
        int place, member, chunk, n, h, rows;
    };
    const auto settle = [&](Item& x) {
        const int head = x.place / p.chunks;
        x.chunk = x.place - head * p.chunks, x.n = head / p.H, x.h = head % p.H;
        x.rows = length_of(p, x.n) - x.chunk * kChunk;
    };
    // The first chunk from there on that has steps; those that have none get their zeros on the way.
    const auto find = [&](Item& x) {
        for (; x.place < places; x.place += static_cast<int>(gridDim.x)) {
            settle(x);
            if (x.rows > 0) return;
            if (wave >= 8) continue;
            const int steps = p.T - x.chunk * kChunk < kChunk ? p.T - x.chunk * kChunk : kChunk;
            T* dquery = static_cast<T*>(const_cast<void*>(p.dq.data)) + static_cast<int64_t>(x.chunk) * kChunk * p.dq.step + x.n * p.dq.row + x.h * p.dq.head;
            T* dkey = static_cast<T*>(const_cast<void*>(p.dk.data)) + static_cast<int64_t>(x.chunk) * kChunk * p.dk.step + x.n * p.dk.row + x.h * p.dk.head;
            for (int i = threadIdx.x; i < steps * p.DK; i += 512) {
                const int t = i / p.DK, e = i - t * p.DK;
                dquery[t * p.dq.step + e] = dkey[t * p.dk.step + e] = from_float<T>(0.0f);
            }
            for (int i = threadIdx.x; i < steps * members; i += 512)
                store_gate<T>(p, p.dgate, x.chunk * kChunk + i / members, x.n, x.h * members + i % members, 0.0f),
                    store_gate<T>(p, p.dbeta, x.chunk * kChunk + i / members, x.n, x.h * members + i % members, 0.0f);
        }
    };
    const auto index_of = [&](const Item& x) { return (static_cast<int64_t>(x.n) * p.HV + x.h * members + x.member) * p.chunks + x.chunk; };

    Raw<T, 8> o_next, v_next;           // a piece to each of 256 threads; the values of the lane's own step
    const auto fetch_slice = [&](const Item& x, int s, typename Pieces::Slice& to) {
        constexpr int WAVES = LOADERS ? 4 : 8;
        const int from_wave = wave % WAVES;
        const int64_t index = index_of(x);
        const uint16_t *marks = p.marks + index * (RANKS * columns * 32 * KS), *later = p.later + index * (RANKS * columns * 32 * KS);
#pragma unroll
        for (int r = 0; r < RANKS; ++r)
#pragma unroll
            for (int i = 0; i < (2 * KS + WAVES - 1) / WAVES; ++i)
                if (from_wave + WAVES * i < 2 * KS) {
                    const uint32_t from = static_cast<uint32_t>((r * columns + 32 * s) * 32 * KS + 512 * (from_wave + WAVES * i)) * 2 + lane * 16;
                    to_lds(marks, from, lds_address(to.marks[r]) + (from_wave + WAVES * i) * 1024);
                    to_lds(later, from, lds_address(to.later[r]) + (from_wave + WAVES * i) * 1024);
                }
        const int64_t rows_at = index * (RANKS * kChunk * columns) + 32 * kChunk * s;
#pragma unroll
        for (int r = 0; r < RANKS; ++r) {
            if (LOADERS || team == 0) value_rows_to_lds(p.deltas + rows_at + r * kChunk * columns, to.deltas[r], w);
            if (LOADERS || team == 1) value_rows_to_lds(p.pulls + rows_at + r * kChunk * columns, to.pulls[r], w);
        }
        o_next.clear();
        const T* douts = static_cast<const T*>(p.dout.data) + static_cast<int64_t>(x.chunk) * kChunk * p.dout.step + x.n * p.dout.row + (x.h * members + x.member) * p.dout.head;
        const int row = threadIdx.x % 256 / 4, at = 32 * s + 8 * (threadIdx.x % 4);
        if (row < x.rows && (LOADERS || team == 0) && at < p.DV) o_next.load(douts, row * p.dout.step + at, p.DV - at);
    };
    const auto put_slice = [&](typename Pieces::Slice& to) {
        if (!LOADERS && team == 1) return;
        const Terms<TERMS> o = terms_of(o_next);
#pragma unroll
        for (int r = 0; r < TERMS; ++r) *reinterpret_cast<u32x4a*>(to.douts[r] + value_place(threadIdx.x % 256 / 4, threadIdx.x % 4)) = o.t[r];
    };
    const auto fetch_values = [&](const Item& x, int s) {
        v_next.clear();
        const T* values = static_cast<const T*>(p.v.data) + static_cast<int64_t>(x.chunk) * kChunk * p.v.step + x.n * p.v.row + (x.h * members + x.member) * p.v.head;
        const int own_at = 32 * s + 8 * group;
        if (team == 0 && own < x.rows && own_at < p.DV) v_next.load(values, own * p.v.step + own_at, p.DV - own_at);
    };
    // What a chunk's steps have of their own: exp(G), exp(G_64 - G), beta and exp(G_64) of the lane's own step; gate, start and beta of the first wave's
    float since_next, until_next, beta_next, rest_next, gate_next, row_beta_next;
    bool start_next;
    const auto fetch_steps = [&](const Item& x) {
        const int hv = x.h * members + x.member;
        const float* vectors = reinterpret_cast<const float*>(p.blocks + index_of(x) * block_words(3) + block_vectors(3));
        since_next = vectors[kSince + own], until_next = vectors[kUntil + own], beta_next = vectors[kBeta + own], rest_next = vectors[kSince + kChunk - 1];
        if (wave == 0) {
            const int t = x.chunk * kChunk + (lane < x.rows ? lane : 0);
            gate_next = gate_value<T>(p.gate, p.gate_float, t, x.n, hv, 0.0f);
            start_next = p.starts != nullptr && p.starts[t * p.starts_step + x.n * p.starts_row] != 0;
            row_beta_next = vectors[kBeta + lane];
        }
    };
    const auto fetch_heads = [&](const Item& x, typename Pieces::Heads& to) {
        constexpr int THREADS = LOADERS ? 256 : 512;
        const T* keys = static_cast<const T*>(p.k.data) + static_cast<int64_t>(x.chunk) * kChunk * p.k.step + x.n * p.k.row + x.h * p.k.head;
        const T* queries = static_cast<const T*>(p.q.data) + static_cast<int64_t>(x.chunk) * kChunk * p.q.step + x.n * p.q.row + x.h * p.q.head;
        if constexpr (TERMS == 1) {
            if (p.near_keys) {
                const uint32_t* zeros = p.blocks + index_of(x) * block_words(3) + block_vectors(3) + kZeros;
                rows_to_lds<4 * KS, THREADS / 64>(LOADERS ? w : wave, reinterpret_cast<const uint16_t*>(keys), p.k.step, x.rows, p.DK, zeros, to.keys);
                rows_to_lds<4 * KS, THREADS / 64>(LOADERS ? w : wave, reinterpret_cast<const uint16_t*>(queries), p.q.step, x.rows, p.DK, zeros, to.queries);
                return;
            }
        }
        Staged<T, 4 * KS, THREADS> k_rows, q_rows;
        k_rows.load(keys, p.k.step, x.rows, p.DK, p.near_keys);
        q_rows.load(queries, p.q.step, x.rows, p.DK, p.near_keys);
        put_rows<T, KS, THREADS>(k_rows, to.keys);
        put_rows<T, KS, THREADS>(q_rows, to.queries);
    };

    Item item{static_cast<int>(blockIdx.x), 0, 0, 0, 0, 0};
    find(item);
    if (item.place >= places) return;
    int turn = 0;                       // pieces so far
    const auto after = [&](const Item& x) {
        Item next = x;
        if (++next.member == members) {
            next.member = 0;
            next.place += static_cast<int>(gridDim.x);
            find(next);
        }
        return next;
    };
    if constexpr (LOADERS)
        if (wave >= 8) {
            fetch_slice(item, 0, lds[0].slice);
            put_slice(lds[0].slice);
            for (;;) {
                for (int s = 0; s < slices; ++s) {
                    arrived();
                    __syncthreads();
                    ++turn;
                    if (s + 1 < slices) {
                        fetch_slice(item, s + 1, lds[turn % BUFFERS].slice);
                        put_slice(lds[turn % BUFFERS].slice);
                    } else {
                        fetch_heads(item, lds[turn % BUFFERS].heads);
                    }
                }
                arrived();
                __syncthreads();
                item = after(item);
                ++turn;
                if (item.place < places) {
                    fetch_slice(item, 0, lds[turn % BUFFERS].slice);
                    put_slice(lds[turn % BUFFERS].slice);
                }
                for (int i = 0; i < 4; ++i) __syncthreads();      // of the others, below
                if (item.place >= places) return;
            }
        }
    if constexpr (!LOADERS) fetch_slice(item, 0, lds[0].slice);
    fetch_values(item, 0);
    fetch_steps(item);
    f32x4 dq_all[KS], dk_all[KS];
    for (;;) {
        if (SHARED && item.member == 0) {
#pragma unroll
            for (int d = 0; d < KS; ++d) dq_all[d] = dk_all[d] = f32x4{0, 0, 0, 0};
        }
        const float since = since_next, until = until_next, beta = beta_next, rest = rest_next;
        // by_row: the wave's steps are rows of dL (dP), the others, up to them, its columns; by_column: the other way round
        f32x4 by_row[4], by_column[4], dq[KS], ds[KS], dk[KS];
#pragma unroll
        for (int j = 0; j < 4; ++j) by_row[j] = by_column[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < KS; ++d) dq[d] = ds[d] = dk[d] = f32x4{0, 0, 0, 0};
        float dbeta = 0.0f, zv = 0.0f, dot = 0.0f;
        for (int s = 0; s < slices; ++s, ++turn) {
            typename Pieces::Slice& here = lds[turn % BUFFERS].slice;
            if constexpr (!LOADERS) put_slice(here);
            const Raw<T, 8> v = v_next;
            if (s == 0 && wave == 0) {
                const bool fresh = lane < item.rows && (start_next || gate_next < kForgotten);
                double sum = fresh || lane >= item.rows ? 0.0 : static_cast<double>(gate_next) * 1.4426950408889634074;
                part[lane] = __popcll(__ballot(fresh) & (~0ull >> (63 - lane)));
#pragma unroll
                for (int d = 1; d < 64; d *= 2) {
                    const double before = __shfl_up(sum, d, 64);
                    if (lane >= d) sum += before;
                }
                total[lane] = sum_of(sum);
                betas[lane] = row_beta_next;
            }
            if constexpr (!LOADERS) arrived();
            __syncthreads();
            if (s + 1 < slices) fetch_values(item, s + 1);
            const Terms<TERMS> o_own = value_rows<TERMS>(here.douts[0], w);
            const Terms<RANKS> z_own = value_rows<RANKS>(here.pulls[0], w), delta_own = value_rows<RANKS>(here.deltas[0], w);
            if (team == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float z = term_sum(z_own, j);
                    dbeta = fmaf(z, term_sum(delta_own, j), dbeta);
                    zv = fmaf(z, v[j], zv);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j <= w) {
                    const Terms<RANKS> x = value_rows<RANKS>(here.deltas[0], j);
                    if (team == 0) by_row[j] = product<RANKS>(x, z_own, by_row[j]);
                    else by_row[j] = product<RANKS>(x, o_own, by_row[j]);
                }
                if (j >= w) {
                    if (team == 0) by_column[j] = product<RANKS>(value_rows<RANKS>(here.pulls[0], j), delta_own, by_column[j]);
                    else by_column[j] = product<RANKS>(value_rows<TERMS>(here.douts[0], j), delta_own, by_column[j]);
                }
            }
#pragma unroll
            for (int d = 0; d < KS; ++d) {
                const Terms<RANKS> x = state_columns<RANKS, KS>(here.marks[0], team * KS + d), y = state_columns<RANKS, KS>(here.later[0], team * KS + d);
                if (d == w) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) dot = fmaf(term_sum(x, j), term_sum(y, j), dot);
                }
                dq[d] = product<RANKS>(x, o_own, dq[d]);
                ds[d] = product<RANKS>(x, z_own, ds[d]);
                dk[d] = product<RANKS>(y, delta_own, dk[d]);
            }
            if constexpr (BUFFERS == 1) {
                __syncthreads();
                if (s + 1 < slices) fetch_slice(item, s + 1, lds[0].slice);
                else fetch_heads(item, lds[0].heads);
            }
        }
        typename Pieces::Heads& here = lds[turn % BUFFERS].heads;
        const uint16_t *keys = here.keys, *queries = here.queries;
        if constexpr (!LOADERS) arrived();
        __syncthreads();
        const Item next = after(item);
        ++turn;
        if (next.place < places) {
            fetch_values(next, 0);
            fetch_steps(next);
        }
        // The other steps are rows 4 group + r of the tiles
        const Sum mine_total = total[own];
        const int mine_part = part[own];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = 16 * j + 4 * group;
            typedef int i32x4 __attribute__((ext_vector_type(4)));
            const f32x4 sums[2] = {*reinterpret_cast<const f32x4*>(total + at), *reinterpret_cast<const f32x4*>(total + at + 2)};
            const i32x4 parts = *reinterpret_cast<const i32x4*>(part + at);
            const f32x4 others = *reinterpret_cast<const f32x4*>(betas + at);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int x = at + r;
                const Sum other = {sums[r / 2][r % 2 * 2], sums[r / 2][r % 2 * 2 + 1]};
                const float d = parts[r] == mine_part ? decay_apart<RANKS == 3>(mine_total, other, x <= own) : 0.0f;
                if (team == 0) {
                    by_row[j][r] = x == own ? 0.0f : kept(-d * beta * others[r], x < own ? by_row[j][r] : by_column[j][r]);
                } else {
                    by_row[j][r] = x <= own ? kept(p.scale * d * others[r], by_row[j][r]) : 0.0f;
                    by_column[j][r] = x >= own ? kept(p.scale * d * beta, by_column[j][r]) : 0.0f;
                }
            }
        }
        const auto publish = [&](int where, const f32x4 (&x)[4]) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const Terms<RANKS> y = split<RANKS>(x[2 * half], x[2 * half + 1]);
#pragma unroll
                for (int r = 0; r < RANKS; ++r) *reinterpret_cast<u32x4a*>(&here.between[where][w][half][r][lane * 4]) = y.t[r];
            }
        };
        const auto published = [&](int where, int half) {
            Terms<RANKS> x;
#pragma unroll
            for (int r = 0; r < RANKS; ++r) x.t[r] = *reinterpret_cast<const u32x4a*>(&here.between[where][w][half][r][lane * 4]);
            return x;
        };
        publish(team, by_row);
        float tail = 0.0f;
#pragma unroll
        for (int d = 0; d < KS; ++d) {
            const f32x4 k = Lds::four(keys, own, team * KS + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float behind = kept(until * beta, dk[d][r]);
                tail = fmaf(k[r], behind, tail);
                dk[d][r] = behind - kept(since * beta, ds[d][r]);
                dq[d][r] = kept(since * p.scale, dq[d][r]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const Terms<RANKS> x = published(0, half), y = published(1, half);
#pragma unroll
            for (int d = 0; d < KS; ++d) {
                const auto k = Lds::columns(keys, team * KS + d, half);
                dk[d] = product<RANKS>(k, x, dk[d]);
                dq[d] = product<RANKS>(k, y, dq[d]);
            }
        }
        __syncthreads();
        if (team == 1) publish(0, by_column);
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const Terms<RANKS> x = published(0, half);
#pragma unroll
            for (int d = 0; d < KS; ++d) dk[d] = product<RANKS>(Lds::columns(queries, team * KS + d, half), x, dk[d]);
        }
        float sum = 0.0f;
#pragma unroll
        for (int d = 0; d < KS; ++d) {
            const f32x4 k = Lds::four(keys, own, team * KS + d), q = Lds::four(queries, own, team * KS + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += q[r] * dq[d][r] - k[r] * dk[d][r];
            if constexpr (SHARED) {
                dq_all[d] += dq[d];
                dk_all[d] += dk[d];
            }
        }
        sum = sum_of_rows(sum);
        tail = sum_of_rows(tail);
        dbeta = sum_of_rows(dbeta);
        zv = sum_of_rows(zv);
        dot = lane_sum(dot);
        const int first = item.chunk * kChunk, hv = item.h * members + item.member, t_own = first + own;
        if (group == 0) {
            dsums[team][own] = sum;
            tails[team][own] = tail;
            if (team == 0) {
                own_sums[own] = 2.0f * beta * (dbeta - zv);
                if (t_own < p.T) store_gate<T>(p, p.dbeta, t_own, item.n, hv, own < item.rows ? dbeta : 0.0f);
            }
        }
        if (lane == 0) dots[wave] = dot;
        if (item.member == members - 1 && t_own < p.T) {
            T* dquery = static_cast<T*>(const_cast<void*>(p.dq.data)) + t_own * p.dq.step + item.n * p.dq.row + item.h * p.dq.head;
            T* dkey = static_cast<T*>(const_cast<void*>(p.dk.data)) + t_own * p.dk.step + item.n * p.dk.row + item.h * p.dk.head;
#pragma unroll
            for (int d = 0; d < KS; d += 2) {
                const int at = head_element(team * KS + d, 0);
                if constexpr (SHARED) {
                    store_eight<T>(dquery + at, p.DK - at, dq_all[d], dq_all[d + 1]);
                    store_eight<T>(dkey + at, p.DK - at, dk_all[d], dk_all[d + 1]);
                } else {
                    store_eight<T>(dquery + at, p.DK - at, dq[d], dq[d + 1]);
                    store_eight<T>(dkey + at, p.DK - at, dk[d], dk[d + 1]);
                }
            }
        }
        __syncthreads();
        if (wave == 0) {
            const int mine = part[lane], before = lane == 0 ? 0 : part[lane - 1], last = part[kChunk - 1], t = first + lane;
            float all = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) all += dots[i];
            const float behind = kept(rest, all) + lane_sum(tails[0][lane] + tails[1][lane]);
            float v = dsums[0][lane] + dsums[1][lane] + own_sums[lane];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const float more = __shfl_down(v, d, 64);
                const int theirs = __shfl_down(mine, d, 64);
                if (lane + d < 64 && theirs == mine) v += more;
            }
            if (mine == last) v += behind;
            if (t < p.T) store_gate<T>(p, p.dgate, t, item.n, hv, lane < item.rows && mine == before ? v : 0.0f);
        }
        if (next.place >= places) return;
        item = next;
        if constexpr (BUFFERS == 1) {
            fetch_slice(item, 0, lds[0].slice);
        }
    }
}

template <typename T, int KS, int RANKS>
void launch_backward(const DeltaArgs& p, hipStream_t stream) {
    launch_chunks<T, KS, 3, true>(p, stream);
    if (p.segments > 1) {
        delta_walk_back_kernel<T, KS, 4, 3, true><<<head_grid(p.N * p.HV * (p.segments - 1), transfer_parts(4, KS, p.DV)), dim3(walk_threads<T>(4)), 0, stream>>>(p);
        launch_join<KS>(p, true, stream);
    }
    bool narrow = false;
    if constexpr (kTerms<T> == 1) {
        narrow = two_waves(p);
        if (narrow) delta_walk_back_kernel<T, KS, 2, RANKS, false><<<head_grid(p.N * p.HV * p.segments, (p.DV + 31) / 32), dim3(walk_threads<T>(2)), 0, stream>>>(p);
    }
    if (!narrow) delta_walk_back_kernel<T, KS, 4, RANKS, false><<<head_grid(p.N * p.HV * p.segments, (p.DV + 63) / 64), dim3(walk_threads<T>(4)), 0, stream>>>(p);
    const int64_t places = static_cast<int64_t>(p.N) * p.H * p.chunks, units = compute_units();
    const dim3 grid(static_cast<unsigned>(places < units ? places : units)), block(GradientPieces<T, KS, RANKS>::THREADS);
    if (p.HV > p.H) delta_gradient_kernel<T, KS, RANKS, true><<<grid, block, 0, stream>>>(p);
    else delta_gradient_kernel<T, KS, RANKS, false><<<grid, block, 0, stream>>>(p);
}
template <typename T>
void launch_backward(const DeltaArgs& p, int ranks, hipStream_t stream) {
    const bool small = p.DK <= 64;
    if (ranks == 3) small ? launch_backward<T, 2, 3>(p, stream) : launch_backward<T, 4, 3>(p, stream);
    else if constexpr (kOutputRanks<T> == 2) small ? launch_backward<T, 2, 2>(p, stream) : launch_backward<T, 4, 2>(p, stream);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_delta_rule_backward_workspace_bytes(const snnf_delta_rule_call* call) {
    if (check_delta("snnf_delta_rule_backward_workspace_bytes", call) != SNNF_OK) return 0;
    return static_cast<size_t>(delta_chunks(call)) *
           (block_words(3) * 4 + (delta_mark_elements(call) + delta_elements(delta_ranks(call, true), call->value_size)) * sizeof(uint16_t)) +
           delta_segment_floats(call, true) * 4;
}

extern "C" int snnf_delta_rule_backward(const snnf_delta_rule_call* call, const void* marks, const snnf_heads* dout, const float* dstate, const snnf_heads* dquery,
                                        const snnf_heads* dkey, const snnf_heads* dvalue, const snnf_heads* dgate, const snnf_heads* dbeta, float* dstate_in,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_delta("snnf_delta_rule_backward", call);
    if (rc != SNNF_OK) return rc;
    if (call->T == 0 || call->N == 0) return SNNF_OK;
    const auto missing = [](const snnf_heads* x) { return x == nullptr || x->data == nullptr; };
    if (call->query.data == nullptr || call->key.data == nullptr || call->value.data == nullptr || marks == nullptr || missing(dout) || missing(dquery) || missing(dkey) ||
        missing(dvalue) || dgate == nullptr || dbeta == nullptr || dstate_in == nullptr)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_delta_rule_backward: operands, marks, dout and what gradients are written to must be non-null");
    if (!aligned_to(marks, 16)) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_delta_rule_backward: marks must lie on 16 bytes");
    const size_t need = snnf_delta_rule_backward_workspace_bytes(call);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
        return fail(SNNF_ERR_WORKSPACE, "snnf_delta_rule_backward: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    const auto view = [](const snnf_heads* x) { return HeadView{x->data, x->step, x->row, x->head}; };
    DeltaArgs p = delta_args(call);
    p.dout = view(dout), p.dq = view(dquery), p.dk = view(dkey), p.dv = view(dvalue), p.dgate = view(dgate), p.dbeta = view(dbeta);
    p.dstate = dstate, p.dstate_in = dstate_in;
    const int64_t chunks = delta_chunks(call);
    p.near_values = call->value_size % 8 == 0 && near_by(p.dout, call->dtype, true) && near_by(p.dv, call->dtype, false);
    p.marks = static_cast<uint16_t*>(const_cast<void*>(marks));
    p.deltas = p.marks + chunks * delta_mark_elements(call);
    p.blocks = static_cast<uint32_t*>(workspace);
    p.later = reinterpret_cast<uint16_t*>(p.blocks + chunks * block_words(3));
    p.pulls = p.later + chunks * delta_mark_elements(call);
    set_segments(p, call, true, reinterpret_cast<float*>(p.pulls + chunks * delta_elements(delta_ranks(call, true), call->value_size)));
    hipStream_t hs = as_stream(stream);
    const int ranks = delta_ranks(call, true);
    if (call->dtype == SNNF_F32) launch_backward<float>(p, ranks, hs);
    else if (call->dtype == SNNF_BF16) launch_backward<bf16_t>(p, ranks, hs);
    else launch_backward<f16_t>(p, ranks, hs);
    return check_launch("snnf_delta_rule_backward");
}
