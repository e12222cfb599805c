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
template <typename T, int KS>
__global__ __launch_bounds__(kTerms<T> == 1 ? 512 : 256) void delta_walk_back_kernel(DeltaArgs p) {
    constexpr int WAVES = 4, RANKS = kOutputRanks<T>, TERMS = kTerms<T>, PIPE = TERMS == 1 ? 2 : 1;
    using Lds = Rows<T, KS>;
    using Values = Tile<T, WAVES>;
    using Reader = ChunkReader<T, KS, WAVES, block_pieces(3)>;
    __shared__ alignas(16) typename Reader::Buffers lds[Reader::kBuffers];
    int head, columns;
    if (!part_of_head(p.N * p.HV, (p.DV + 63) / 64, &head, &columns)) return;
    const int n = head / p.HV, hv = head % p.HV, h = hv / (p.HV / p.H), limit = length_of(p, n), live = (limit + kChunk - 1) / kChunk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane / 16;
    const int left = columns * Values::kColumns, mine = left + 16 * wave, column = mine + lane % 16;
    const bool there = column < p.DV;
    const int64_t cell = static_cast<int64_t>(head) * p.DK * p.DV + column;
    f32x4 later[2 * KS];
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = head_element(d, r);
            later[d][r] = p.dstate != nullptr && there && row < p.DK ? p.dstate[cell + static_cast<int64_t>(row) * p.DV] : 0.0f;
        }
    const T* k_base = static_cast<const T*>(p.k.data) + n * p.k.row + h * p.k.head;
    const T* q_base = static_cast<const T*>(p.q.data) + n * p.q.row + h * p.q.head;
    const T* o_base = static_cast<const T*>(p.dout.data) + n * p.dout.row + hv * p.dout.head + left;
    T* v_base = static_cast<T*>(const_cast<void*>(p.dv.data)) + n * p.dv.row + hv * p.dv.head + mine;
    Reader reader;
    const auto fetch = [&](int chunk) {
        const int64_t first = static_cast<int64_t>(chunk) * kChunk;
        if (chunk >= 0) reader.fetch(p, k_base + first * p.k.step, q_base + first * p.q.step, o_base + first * p.dout.step, p.dout.step, limit - chunk * kChunk, p.DV - left,
                                     p.blocks + (static_cast<int64_t>(head) * p.chunks + chunk) * block_words(3), lds[chunk % Reader::kBuffers]);
    };
    fetch(live - 1);
    for (int chunk = live - 1; chunk >= 0; --chunk) {
        const int64_t index = static_cast<int64_t>(head) * p.chunks + chunk;
        typename Reader::Buffers& here = lds[chunk % Reader::kBuffers];
        const uint16_t *keys = here.keys, *queries = here.queries;
        T* tile = here.tile;
        const uint32_t *block = here.block, *vectors = block + block_vectors(3);
        reader.wait(here);
        fetch(chunk - 1);
        now();
        // K R
        f32x4 pull[4], dout[4], z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pull[i] = z[i] = f32x4{0, 0, 0, 0};
        Terms<TERMS> a[PIPE][4];
        const auto load = [&](int s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) a[s % PIPE][i] = Lds::rows(keys, i, s);
        };
        load(0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (PIPE == 2 && s + 1 < KS) load(s + 1);
            now();
            const Terms<3> x = split<3>(later[2 * s], later[2 * s + 1]);
            uint16_t* marks = p.later + index * (RANKS * padded_values(p.DV) * 32 * KS);
#pragma unroll
            for (int r = 0; r < RANKS; ++r)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    *reinterpret_cast<u32x2a*>(marks + static_cast<uint32_t>((r * padded_values(p.DV) + column) * 32 * KS + mark_place<KS>(column, 2 * s + half) + 4 * group)) =
                        u32x2a{x.t[r][2 * half], x.t[r][2 * half + 1]};
#pragma unroll
            for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                for (int j = 0; j <= rank; ++j)
                    if (j < TERMS) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) pull[i] = mfma(a[s % PIPE][i].t[j], x.t[rank - j], pull[i]);
                    }
            if (PIPE == 1 && s + 1 < KS) load(s + 1);
        }
        const bool broken = __builtin_amdgcn_readfirstlane(vectors[kBroken]) != 0;
        const float rest = __uint_as_float(__builtin_amdgcn_readfirstlane(vectors[kSince + kChunk - 1]));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 until = row_factors(vectors, kUntil, i);
            if (broken) drop(pull[i], until);
            pull[i] *= until;
            dout[i] = Values::get(tile, i);
        }
        // dU, then Z
        {
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
        Values::template write_terms<RANKS>(tile, z, p.pulls + index * (RANKS * kChunk * padded_values(p.DV)) + mine, padded_values(p.DV));
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] *= row_factors(vectors, kBeta, i);
        Values::turn_values(tile, z);
        Values::write(tile, v_base + static_cast<int64_t>(chunk) * kChunk * p.dv.step, p.dv.step, p.T - chunk * kChunk, limit - chunk * kChunk, p.DV - mine, p.near_values);
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
    for (int t = live * kChunk + wave * 4 + group; t < p.T; t += 4 * WAVES)      // padding
        for (int c = left + lane % 16; c < p.DV && c < left + Values::kColumns; c += 16) v_base[t * p.dv.step + c - mine] = from_float<T>(0.0f);
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = head_element(d, r);
            if (there && row < p.DK) p.dstate_in[cell + static_cast<int64_t>(row) * p.DV] = later[d][r];
        }
}

// ------------------------------------------------------------------------------------------------------------------
// Gradients chunk by chunk
// ------------------------------------------------------------------------------------------------------------------
// Of queries and keys transposed, [DK x steps]: a wave owns 16 steps as columns, so that dP and dL, contracted over steps next, are multiplied as they lie in
// accumulators. Those are worked out twice, with the wave's steps as rows and as columns of the matrix.
__device__ __forceinline__ float over_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
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
// Rows of a plane [64][columns] to there: four instructions, one to a wave.
__device__ __forceinline__ void value_rows_to_lds(const uint16_t* plane, int columns, uint16_t* lds) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = 16 * wave + lane / 4;
    to_lds(plane, static_cast<uint32_t>(row * columns + 8 * slot_of<4>(row, lane % 4)) * 2, lds_address(lds) + wave * 1024);
}
// Of a state's 32 value columns [32][32 KS]: elements of `head_element(tile, ..)` as rows, value columns as places, in order.
template <int N, int KS>
__device__ __forceinline__ Terms<N> state_columns(const uint16_t* lds, int tile) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const int lane = threadIdx.x & 63, column = 8 * (lane / 16) + lane % 16 / 4;
    const uint16_t* low = lds + column * 32 * KS + mark_place<KS>(column, tile) + 4 * (lane % 4);
    const uint16_t* high = lds + (column + 4) * 32 * KS + mark_place<KS>(column + 4, tile) + 4 * (lane % 4);
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
template <typename T>
__device__ __forceinline__ void store_four(T* to, int left, const f32x4& x) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < left) to[r] = from_float<T>(x[r]);
}

// GROUPED: several value heads to a key head, whose gradients are summed one after the other.
template <typename T, int KS, bool GROUPED>
__global__ __launch_bounds__(256, sizeof(T) == 4 || GROUPED ? 1 : 2) void delta_gradient_kernel(DeltaArgs p) {
    using Lds = Rows<T, KS>;
    constexpr int RANKS = kOutputRanks<T>, TERMS = kTerms<T>, TILES = 2 * KS;
    __shared__ union {
        struct {                        // 32 value columns of everything
            uint16_t marks[RANKS][1024 * KS], later[RANKS][1024 * KS], deltas[RANKS][kChunk * 32], pulls[RANKS][kChunk * 32], douts[TERMS][kChunk * 32];
        };
        struct {
            uint16_t keys[Lds::kSize], queries[Lds::kSize];
        };
    } lds;
    __shared__ double total[kChunk];
    __shared__ int part[kChunk];
    __shared__ float betas[kChunk], dsums[kChunk], tails[kChunk], dots[4];
    const uint32_t place = group_index();
    if (place >= static_cast<uint32_t>(p.N) * p.H * p.chunks) return;
    const int chunk = place % p.chunks, n = place / p.chunks / p.H, h = place / p.chunks % p.H, first = chunk * kChunk, limit = length_of(p, n);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane / 16, column = lane % 16, own = 16 * wave + column, t_own = first + own;
    const bool there = t_own < limit;
    const int members = p.HV / p.H, gate_size = p.gate_float ? 4 : static_cast<int>(sizeof(T));
    const auto store_gate = [&](const HeadView& x, int t, int hv, float v) {
        if (x.data == nullptr) return;
        const int64_t at = t * x.step + n * x.row + hv * x.head;
        if (gate_size == 4) static_cast<float*>(const_cast<void*>(x.data))[at] = v;
        else static_cast<T*>(const_cast<void*>(x.data))[at] = from_float<T>(v);
    };
    T* dquery = static_cast<T*>(const_cast<void*>(p.dq.data)) + t_own * p.dq.step + n * p.dq.row + h * p.dq.head;
    T* dkey = static_cast<T*>(const_cast<void*>(p.dk.data)) + t_own * p.dk.step + n * p.dk.row + h * p.dk.head;
    f32x4 dq_all[TILES], dk_all[TILES];
#pragma unroll
    for (int d = 0; d < TILES; ++d) dq_all[d] = dk_all[d] = f32x4{0, 0, 0, 0};
    const int columns = padded_values(p.DV);
    for (int member = 0; member < members; ++member) {
        const int hv = h * members + member;
        if (first >= limit) {
            if (group == 0 && t_own < p.T) store_gate(p.dgate, t_own, hv, 0.0f), store_gate(p.dbeta, t_own, hv, 0.0f);
            continue;
        }
        const int64_t index = (static_cast<int64_t>(n) * p.HV + hv) * p.chunks + chunk;
        const float* vectors = reinterpret_cast<const float*>(p.blocks + index * block_words(3) + block_vectors(3));
        __syncthreads();
        if (wave == 0) {
            const int t = first + lane;
            const bool inside = t < limit;
            const float g = inside ? gate_value<T>(p.gate, p.gate_float, t, n, hv, 0.0f) : 0.0f;
            const bool fresh = inside && (g < kForgotten || (p.starts != nullptr && p.starts[t * p.starts_step + n * p.starts_row] != 0));
            double sum = fresh ? 0.0 : static_cast<double>(g) * 1.4426950408889634074;
            part[lane] = __popcll(__ballot(fresh) & (~0ull >> (63 - lane)));
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const double before = __shfl_up(sum, d, 64);
                if (lane >= d) sum += before;
            }
            total[lane] = sum;
            betas[lane] = vectors[kBeta + lane];
        }
        const float since = vectors[kSince + own], until = vectors[kUntil + own], beta = vectors[kBeta + own];
        const uint16_t *marks = p.marks + index * (RANKS * columns * 32 * KS), *later = p.later + index * (RANKS * columns * 32 * KS);
        const uint16_t *deltas = p.deltas + index * (RANKS * kChunk * columns), *pulls = p.pulls + index * (RANKS * kChunk * columns);
        const T* douts = static_cast<const T*>(p.dout.data) + n * p.dout.row + hv * p.dout.head;
        const T* values = static_cast<const T*>(p.v.data) + n * p.v.row + hv * p.v.head;
        f32x4 score_row[4], score_column[4], pull_row[4], pull_column[4], dq[TILES], ds[TILES], dk[TILES];
#pragma unroll
        for (int j = 0; j < 4; ++j) score_row[j] = score_column[j] = pull_row[j] = pull_column[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < TILES; ++d) dq[d] = ds[d] = dk[d] = f32x4{0, 0, 0, 0};
        float dbeta = 0.0f, zv = 0.0f, dot = 0.0f;
        for (int s = 0; 32 * s < p.DV; ++s) {
            if (s > 0) __syncthreads();
#pragma unroll
            for (int r = 0; r < RANKS; ++r) {
#pragma unroll
                for (int i = wave; i < 2 * KS; i += 4) {
                    const uint32_t from = static_cast<uint32_t>((r * columns + 32 * s) * 32 * KS + 512 * i) * 2 + lane * 16;
                    to_lds(marks, from, lds_address(lds.marks[r]) + i * 1024);
                    to_lds(later, from, lds_address(lds.later[r]) + i * 1024);
                }
                value_rows_to_lds(deltas + r * kChunk * columns + 32 * s, columns, lds.deltas[r]);
                value_rows_to_lds(pulls + r * kChunk * columns + 32 * s, columns, lds.pulls[r]);
            }
            {
                const int row = threadIdx.x / 4, at = 32 * s + 8 * (threadIdx.x % 4);
                const auto o = first + row < limit && at < p.DV ? row_terms<T>(douts + (first + row) * p.dout.step, at, p.DV) : no_terms<TERMS>();
#pragma unroll
                for (int r = 0; r < TERMS; ++r) *reinterpret_cast<u32x4a*>(lds.douts[r] + value_place(row, threadIdx.x % 4)) = o.t[r];
            }
            Raw<T, 8> v;
            const int at = 32 * s + 8 * group;
            if (there && at < p.DV) v.load(values + t_own * p.v.step, at, p.DV - at);
            else v.clear();
            arrived();
            __syncthreads();
            const Terms<TERMS> o_own = value_rows<TERMS>(lds.douts[0], wave);
            const Terms<RANKS> z_own = value_rows<RANKS>(lds.pulls[0], wave), delta_own = value_rows<RANKS>(lds.deltas[0], wave);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float z = term_sum(z_own, j);
                dbeta = fmaf(z, term_sum(delta_own, j), dbeta);
                zv = fmaf(z, v[j], zv);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j <= wave) {
                    const Terms<RANKS> x = value_rows<RANKS>(lds.deltas[0], j);
                    score_row[j] = product<RANKS>(x, o_own, score_row[j]);
                    pull_row[j] = product<RANKS>(x, z_own, pull_row[j]);
                }
                if (j >= wave) {
                    score_column[j] = product<RANKS>(value_rows<TERMS>(lds.douts[0], j), delta_own, score_column[j]);
                    pull_column[j] = product<RANKS>(value_rows<RANKS>(lds.pulls[0], j), delta_own, pull_column[j]);
                }
            }
#pragma unroll
            for (int d = 0; d < TILES; ++d) {
                const Terms<RANKS> x = state_columns<RANKS, KS>(lds.marks[0], d), y = state_columns<RANKS, KS>(lds.later[0], d);
                if (d % 4 == wave) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) dot = fmaf(term_sum(x, j), term_sum(y, j), dot);
                }
                dq[d] = product<RANKS>(x, o_own, dq[d]);
                ds[d] = product<RANKS>(x, z_own, ds[d]);
                dk[d] = product<RANKS>(y, delta_own, dk[d]);
            }
        }
        __syncthreads();
        {
            Staged<T, 4 * KS, 256> x;
            const T* from = static_cast<const T*>(p.k.data) + static_cast<int64_t>(first) * p.k.step + n * p.k.row + h * p.k.head;
            x.load(from, p.k.step, limit - first, p.DK, p.near_keys);
            put_rows<T, KS, 256>(x, lds.keys);
            from = static_cast<const T*>(p.q.data) + static_cast<int64_t>(first) * p.q.step + n * p.q.row + h * p.q.head;
            x.load(from, p.q.step, limit - first, p.DK, p.near_keys);
            put_rows<T, KS, 256>(x, lds.queries);
        }
        __syncthreads();
        const uint16_t *keys = lds.keys, *queries = lds.queries;
        float tail = 0.0f;
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            const f32x4 k = Lds::four(keys, own, d);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float behind = kept(until * beta, dk[d][r]);
                tail = fmaf(k[r], behind, tail);
                dk[d][r] = behind - kept(since * beta, ds[d][r]);
                dq[d][r] = kept(since * p.scale, dq[d][r]);
            }
        }
        // x: the other step, row of the tile
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int x = 16 * j + 4 * group + r;
                const float d = part[x] == part[own] ? decay_of(x <= own ? total[own] - total[x] : total[x] - total[own]) : 0.0f;
                const float both = -d * beta * betas[x];
                score_row[j][r] = x <= own ? kept(p.scale * d * betas[x], score_row[j][r]) : 0.0f;
                score_column[j][r] = x >= own ? kept(p.scale * d * beta, score_column[j][r]) : 0.0f;
                pull_row[j][r] = x < own ? kept(both, pull_row[j][r]) : (x > own ? kept(both, pull_column[j][r]) : 0.0f);
            }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const Terms<RANKS> a = split<RANKS>(score_row[2 * half], score_row[2 * half + 1]), b = split<RANKS>(score_column[2 * half], score_column[2 * half + 1]);
            const Terms<RANKS> c = split<RANKS>(pull_row[2 * half], pull_row[2 * half + 1]);
#pragma unroll
            for (int d = 0; d < TILES; ++d) {
                const auto k = Lds::columns(keys, d, half), q = Lds::columns(queries, d, half);
                dq[d] = product<RANKS>(k, a, dq[d]);
                dk[d] = product<RANKS>(q, b, dk[d]);
                dk[d] = product<RANKS>(k, c, dk[d]);
            }
        }
        float sum = 0.0f;
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            const f32x4 k = Lds::four(keys, own, d), q = Lds::four(queries, own, d);
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += q[r] * dq[d][r] - k[r] * dk[d][r];
            if constexpr (GROUPED) dq_all[d] += dq[d], dk_all[d] += dk[d];
            else dq_all[d] = dq[d], dk_all[d] = dk[d];
        }
        sum = over_groups(sum);
        tail = over_groups(tail);
        dbeta = over_groups(dbeta);
        zv = over_groups(zv);
        dot = lane_sum(dot);
        if (group == 0) {
            dsums[own] = sum + 2.0f * beta * (dbeta - zv);
            tails[own] = tail;
            if (t_own < p.T) store_gate(p.dbeta, t_own, hv, there ? dbeta : 0.0f);
        }
        if (lane == 0) dots[wave] = dot;
        __syncthreads();
        if (wave == 0) {
            const int mine = part[lane], before = lane == 0 ? 0 : part[lane - 1], last = part[kChunk - 1], t = first + lane;
            const float rest = vectors[kSince + kChunk - 1];
            const float behind = kept(rest, dots[0] + dots[1] + dots[2] + dots[3]) + lane_sum(tails[lane]);
            float v = dsums[lane];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const float more = __shfl_down(v, d, 64);
                const int theirs = __shfl_down(mine, d, 64);
                if (lane + d < 64 && theirs == mine) v += more;
            }
            if (mine == last) v += behind;
            if (t < p.T) store_gate(p.dgate, t, hv, t < limit && mine == before ? v : 0.0f);
        }
    }
    if (t_own < p.T) {
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
            const int at = head_element(d, 0);
            store_four<T>(dquery + at, p.DK - at, dq_all[d]);
            store_four<T>(dkey + at, p.DK - at, dk_all[d]);
        }
    }
}

template <typename T, int KS>
void launch_backward(const DeltaArgs& p, hipStream_t stream) {
    launch_chunks<T, KS, true>(p, stream);
    delta_walk_back_kernel<T, KS><<<dim3(head_groups(p.N * p.HV, (p.DV + 63) / 64)), dim3(256), 0, stream>>>(p);
    const dim3 grid = grid_of(static_cast<int64_t>(p.N) * p.H * p.chunks);
    if (p.HV > p.H) delta_gradient_kernel<T, KS, true><<<grid, dim3(256), 0, stream>>>(p);
    else delta_gradient_kernel<T, KS, false><<<grid, dim3(256), 0, stream>>>(p);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_delta_rule_backward_workspace_bytes(const snnf_delta_rule_call* call) {
    if (check_delta("snnf_delta_rule_backward_workspace_bytes", call) != SNNF_OK) return 0;
    return static_cast<size_t>(delta_chunks(call)) *
           (block_words(3) * 4 + (delta_mark_elements(call) + delta_elements(delta_ranks(call), call->value_size)) * sizeof(uint16_t));
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
    hipStream_t hs = as_stream(stream);
    const bool small = call->key_size <= 64;
    if (call->dtype == SNNF_F32) small ? launch_backward<float, 2>(p, hs) : launch_backward<float, 4>(p, hs);
    else if (call->dtype == SNNF_BF16) small ? launch_backward<bf16_t, 2>(p, hs) : launch_backward<bf16_t, 4>(p, hs);
    else small ? launch_backward<f16_t, 2>(p, hs) : launch_backward<f16_t, 4>(p, hs);
    return check_launch("snnf_delta_rule_backward");
}
