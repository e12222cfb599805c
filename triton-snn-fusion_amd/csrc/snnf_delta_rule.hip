// Gated delta rule, forward: per value head with a state S of [DK x DV]
//     S <- exp(gate_t) S,   delta_t = v_t - S^T k_t,   S <- S + beta_t k_t delta_t^T,   out_t = scale S^T q_t
// Chunks of 64 steps at once. With G the running sum of gates inside a chunk, D_ij = exp(G_i - G_j) for j <= i and L_ij = D_ij k_i . k_j for j < i:
//     delta = (I + L diag(beta))^-1 (V - diag(e^G) K S),   out = scale (diag(e^G) Q S + (Q K^T o D) diag(beta) delta),
//     S <- e^(G_64) S + K^T diag(e^(G_64 - G)) diag(beta) delta
#include "snnf_delta_rule.h"

namespace snnf {
namespace {

// ------------------------------------------------------------------------------------------------------------------
// What chunks need that does not depend on the state
// ------------------------------------------------------------------------------------------------------------------
// The backward pass wants transposes: of the scores, and of (I + diag(beta) L)^-1, whose transpose turns a gradient of beta delta into that of the rows in front.
// A workgroup to a chunk of a value head, a wave to 16 rows. The inverse: blocks on the diagonal by substitution, those below by products in float32. Bound by the chain of loads, substitution,
// three joins of blocks and stores, of which four workgroups to a CU overlap, for which registers and LDS just do (17 KB of LDS more for a matrix of scores, and 100 bytes of spilled registers a thread with them,
// 181 us in place of 122): 8192 chunks of 128 bfloat16 elements, two thirds of them of steps that are there, 122 us. 4096 whole ones, 264 MB of heads and fragments, 78 us (3.4 TB/s).
constexpr int kPitch = 68;              // of a [64 x 64] matrix in LDS: rows start 4 banks apart

// rows 16 a.., columns 16 b + 4 (lane / 16) + 0..3 of lane % 16's row
__device__ __forceinline__ f32x4 block_row(const float* m, int a, int b) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const f32x4*>(m + (16 * a + lane % 16) * kPitch + 16 * b + 4 * (lane / 16));
}
__device__ __forceinline__ f32x4 multiply_f32(const f32x4& a, const f32x4& b, f32x4 c) {       // 16 places, place 4 (lane / 16) + s in step s
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
}

template <typename T, int KS, int RANKS, bool BACKWARD>
__global__ __launch_bounds__(256, kTerms<T> == 3 ? 2 : 4) void delta_chunk_kernel(DeltaArgs p) {
    constexpr int TERMS = kTerms<T>;
    constexpr int kMatrix = kChunk * kPitch, kFragments = 4 * KS * TERMS * 256;
    __shared__ alignas(16) uint32_t shared[kFragments > 2 * kMatrix ? kFragments : 2 * kMatrix];     // keys, then the matrices
    // L below the diagonal, the scores transposed above it, four columns to the right: score [i][c] at [c][i + 4]
    float *both = reinterpret_cast<float*>(shared), *inverse = both + kMatrix;
    __shared__ Sum total[kChunk];
    __shared__ alignas(16) int part[kChunk];
    __shared__ float beta[kChunk];
    const uint32_t index = group_index();
    if (index >= static_cast<uint32_t>(p.N) * p.HV * p.chunks) return;
    const int chunk = index % p.chunks, head = index / p.chunks, n = head / p.HV, hv = head % p.HV, h = hv / (p.HV / p.H);
    const int first = chunk * kChunk, limit = length_of(p, n);
    if (first >= limit) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane / 16, column = lane % 16;
    uint32_t* blocks = p.blocks + static_cast<int64_t>(index) * block_words(RANKS);
    float* vectors = reinterpret_cast<float*>(blocks + block_vectors(RANKS));

    // The wave's 16 rows; out of reach: the chunk's first, which is there, and zeros in their place
    const T* keys = static_cast<const T*>(p.k.data) + n * p.k.row + h * p.k.head;
    const T* queries = static_cast<const T*>(p.q.data) + n * p.q.row + h * p.q.head;
    Raw<T, 8> k_raw[KS], q_raw[KS];
    {
        const int row = first + 16 * wave + column;
        const auto rows = [&](const T* base, int64_t step, Raw<T, 8> (&x)[KS]) {
            if (p.DK % 8 == 0) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int at = 32 * s + 8 * group;
                    x[s].load(base, row < limit && at < p.DK ? row * step + at : first * step, 8);
                }
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    if (row >= limit || 32 * s + 8 * group >= p.DK) x[s].clear();
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int at = 32 * s + 8 * group;
                    if (row < limit && at < p.DK) x[s].load(base, row * step + at, p.DK - at);
                    else x[s].clear();
                }
            }
        };
        rows(keys, p.k.step, k_raw);
        rows(queries, p.q.step, q_raw);
    }
    if (wave == 0) {
        const int t = first + lane;
        const bool there = t < limit;
        float g = there ? gate_value<T>(p.gate, p.gate_float, t, n, hv, 0.0f) : 0.0f;
        const float b = there ? gate_value<T>(p.beta, p.gate_float, t, n, hv, 1.0f) : 0.0f;
        const bool fresh = there && (g < kForgotten || (p.starts != nullptr && p.starts[t * p.starts_step + n * p.starts_row] != 0));
        double sum = fresh ? 0.0 : static_cast<double>(g) * 1.4426950408889634074;
        const int mine = __popcll(__ballot(fresh) & (~0ull >> (63 - lane)));
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double before = __shfl_up(sum, d, 64);
            if (lane >= d) sum += before;
        }
        total[lane] = sum_of(sum), part[lane] = mine, beta[lane] = b;
        const double all = __shfl(sum, 63, 64);
        const int last = __shfl(mine, 63, 64);
        const float since = mine == 0 ? decay_of(sum) : 0.0f, until = mine == last ? decay_of(all - sum) : 0.0f;
        vectors[kSince + lane] = since;
        vectors[kUntil + lane] = until;
        vectors[kBeta + lane] = b;
        const bool broken = __ballot(since == 0.0f || until == 0.0f) != 0;
        const uint64_t starts = __ballot(fresh);
        const uint32_t word = lane == 0 ? __float_as_uint(broken ? 1.0f : 0.0f) : (lane == 2 ? static_cast<uint32_t>(starts) : (lane == 3 ? static_cast<uint32_t>(starts >> 32) : 0u));
        vectors[kBroken + lane] = __uint_as_float(word);
    }
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kk[j] = qk[j] = f32x4{0, 0, 0, 0};
    {
        Terms<TERMS> k[KS], q[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            k[s] = terms_of(k_raw[s]), q[s] = terms_of(q_raw[s]);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) *reinterpret_cast<u32x4a*>(shared + ((wave * KS + s) * TERMS + i) * 256 + lane * 4) = k[s].t[i];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > wave) break;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s % 2 == 0) now();
                const Terms<TERMS> other = block_terms<TERMS>(shared, j * KS + s);
                kk[j] = product<3>(k[s], other, kk[j]);
                qk[j] = product<3>(q[s], other, qk[j]);
            }
        }
    }
    __syncthreads();
    {
        const int row = 16 * wave + 4 * group;
        Sum mine[4];
        int segment[4];
        float rate[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) mine[r] = total[row + r], segment[r] = part[row + r], rate[r] = beta[row + r];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = 16 * j + column;
            if (j <= wave) {
                const Sum other = total[c];
                const int theirs = part[c];
                const float theirs_rate = beta[c];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float d = decay_between(other, mine[r]);
                    d = c <= row + r && segment[r] == theirs ? d : 0.0f;
                    const float below = d * kk[j][r] * (BACKWARD ? rate[r] : theirs_rate);
                    if (c < row + r) both[(row + r) * kPitch + c] = d != 0.0f ? below : 0.0f;
                    qk[j][r] = d != 0.0f ? d * qk[j][r] * p.scale : 0.0f;
                }
                float* score = both + c * kPitch + row + 4;
                if (j < wave) {
                    *reinterpret_cast<f32x4*>(score) = qk[j];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (c <= row + r) score[r] = qk[j][r];
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) inverse[(row + r) * kPitch + c] = 0.0f;
            now();
        }
    }
    __syncthreads();
    // Diagonal blocks by substitution, a column of the inverse to a lane (four lanes to the same).
    {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == column ? 1.0f : 0.0f;
        // four columns of the block at a time
#pragma unroll
        for (int j = 0; j < 15; ++j) {
            if (j % 4 == 0) now();
#pragma unroll
            for (int i = j + 1; i < 16; ++i) x[i] = fmaf(-both[(16 * wave + i) * kPitch + 16 * wave + j], x[j], x[i]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i / 4 == group) inverse[(16 * wave + i) * kPitch + 16 * wave + column] = x[i];
    }
    __syncthreads();
    // Blocks below: T_ij = -T_ii sum_k A_ik T_kj, one diagonal of blocks after the other.
#pragma unroll
    for (int d = 1; d < 4; ++d) {
        f32x4 corner{0, 0, 0, 0};
        const int j = wave - d;
        if (j >= 0) {
            f32x4 sum{0, 0, 0, 0};
            for (int k = j; k < wave; ++k) {
                f32x4 b;
#pragma unroll
                for (int s = 0; s < 4; ++s) b[s] = inverse[(16 * k + 4 * group + s) * kPitch + 16 * j + column];
                sum = multiply_f32(block_row(both, wave, k), b, sum);
            }
            corner = multiply_f32(block_row(inverse, wave, wave), sum, corner);
#pragma unroll
            for (int r = 0; r < 4; ++r) inverse[(16 * wave + 4 * group + r) * kPitch + 16 * j + column] = -corner[r];
        }
        __syncthreads();
    }
    // Fragments as the other kernels load them: a row of one matrix, a column of the other
    const auto place = [&](int e) { return 4 * group + (e < 4 ? e : 12 + e); };
    const auto fragment = [&](const float* m, int f, bool transposed, int shift) {
        const int line = 16 * (BACKWARD ? upper_tile(f) : lower_tile(f)) + column, from = 32 * (BACKWARD ? upper_half(f) : lower_half(f));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = transposed ? m[(from + place(e)) * kPitch + line + shift] : m[line * kPitch + from + place(e) + shift];
        if (shift > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (BACKWARD ? line <= from + place(e) : from + place(e) <= line) ? x[e] : 0.0f;
        }
        return split<3>(x);
    };
    for (int f = wave; f < kBlocks; f += 4) {
        const Terms<3> x = fragment(inverse, f, BACKWARD, 0), y = fragment(both, f, !BACKWARD, 4);
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<u32x4a*>(blocks + (f * 3 + i) * 256 + lane * 4) = x.t[i];
#pragma unroll
        for (int i = 0; i < RANKS; ++i) *reinterpret_cast<u32x4a*>(blocks + (kBlocks * 3 + f * RANKS + i) * 256 + lane * 4) = y.t[i];
    }
}

// ------------------------------------------------------------------------------------------------------------------
// The walk over the chunks
// ------------------------------------------------------------------------------------------------------------------
// A wave owns 16 columns of the state, in accumulators, and of everything that is multiplied from it on: products go over the heads' elements
// or over steps, whose place in an accumulator is a matter of the other operand's order, so that nothing but keys, queries and what crosses the kernel's edge passes through LDS.
// Bound by a wave's own instructions: some 180 matrix instructions of 16 cycles and 1100 others of 4 a chunk, of which little overlaps within a wave, and LDS, memory and stores beside them.
// A chunk takes 4.1 us (32 x 16 heads of 128 bfloat16, 64 columns to a workgroup), with what gradients will read, whose stores have to wait for room, 4.7 (4096 x 4 x 16, 32 columns: 300 us).
// Few heads leave most of the chip idle, so that their chunks are cut into segments. What a segment does to a state S is A S + B: A is where it takes the identity, with values of 0, B where it
// takes no state at all. kTransfer walks the segments for both, side by side; the states between them follow (`delta_join_kernel`), and a second walk over all segments has its states at once.
// A prompt of 8192 steps x 16 heads of 128 bfloat16, 8 segments: chunks 34, first walk 80, states 18, second walk 68 us; in one go chunks and walk took 634.
enum Walk { kOutputs, kTraining, kTransfer };

template <typename T, int KS, int WAVES, int RANKS, Walk WALK>
__global__ __launch_bounds__(kTerms<T> == 1 && walk_threads<T>(WAVES) <= 512 ? 512 : walk_threads<T>(WAVES)) void delta_walk_kernel(DeltaArgs p) {
    using Lds = Rows<T, KS>;
    using Values = Tile<T, WAVES>;
    constexpr int TERMS = kTerms<T>, PIPE = TERMS == 1 ? 2 : 1;
    constexpr bool TRAIN = WALK == kTraining, TRANSFER = WALK == kTransfer;
    using Reader = ChunkReader<T, KS, WAVES, block_pieces(RANKS), !TRANSFER>;
    __shared__ alignas(16) typename Reader::Buffers lds[Reader::kBuffers];
    const int value_parts = (p.DV + Values::kColumns - 1) / Values::kColumns, segments = TRANSFER ? p.segments - 1 : p.segments;
    int item, columns;
    if (!part_of_head(p.N * p.HV * segments, TRANSFER ? value_parts + (32 * KS + Values::kColumns - 1) / Values::kColumns : value_parts, &item, &columns)) return;
    const int head = item / segments, segment = item % segments, n = head / p.HV, hv = head % p.HV, h = hv / (p.HV / p.H), limit = length_of(p, n);
    const int chunks = (limit + kChunk - 1) / kChunk, begin = segment * p.per, last = chunks == 0 ? 0 : (chunks - 1) / p.per;
    const int live = segment < last ? begin + p.per : chunks;
    const bool matrix = TRANSFER && columns >= value_parts;
    if (segment > last || (TRANSFER && (segment == last || (matrix && segment == 0)))) return;      // the first segment's state is known
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane / 16;
    const int left = (matrix ? columns - value_parts : columns) * Values::kColumns, mine = left + 16 * wave, column = mine + lane % 16;
    const bool there = column < (matrix ? 32 * KS : p.DV);
    const T* k_base = static_cast<const T*>(p.k.data) + n * p.k.row + h * p.k.head;
    const T* q_base = static_cast<const T*>(p.q.data) + n * p.q.row + h * p.q.head;
    const T* v_base = static_cast<const T*>(p.v.data) + n * p.v.row + hv * p.v.head + (matrix ? 0 : left);
    T* out_base = static_cast<T*>(const_cast<void*>(p.out.data)) + n * p.out.row + hv * p.out.head + mine;
    const auto place = [&](int chunk) {
        const int64_t first = static_cast<int64_t>(chunk) * kChunk;
        return typename Reader::Chunk{k_base + first * p.k.step, q_base + first * p.q.step, v_base + first * p.v.step, p.v.step, limit - chunk * kChunk, matrix ? 0 : p.DV - left,
                                      p.blocks + (static_cast<int64_t>(head) * p.chunks + chunk) * block_words(RANKS)};
    };
    Reader reader;
    const auto fetch = [&](int chunk) {
        if (chunk < live) reader.fetch(p, place(chunk), lds[chunk % Reader::kBuffers]);
    };
    if constexpr (Reader::kDirect)
        if (wave >= WAVES) {
            fetch(begin);
            for (int chunk = begin; chunk < live; ++chunk) {
                arrived();
                __syncthreads();
                fetch(chunk + 1);
            }
            return;
        }
    const int64_t cell = static_cast<int64_t>(head) * p.DK * p.DV + column;
    // The first of several segments has its state from a copy: the last one's may take its place meanwhile.
    float* slot = p.segments > 1 ? p.between + (static_cast<int64_t>(head) * p.segments + segment) * p.DK * p.DV + column : nullptr;
    const float* before = nullptr;
    if (TRANSFER || last == 0) before = segment > 0 || p.state == nullptr ? nullptr : p.state + cell;
    else before = slot;
    f32x4 state[2 * KS];
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = head_element(d, r);
            state[d][r] = before != nullptr && there && row < p.DK ? before[static_cast<int64_t>(row) * p.DV] : (matrix && row == column ? 1.0f : 0.0f);
        }
    if (TRANSFER && segment == 0) {
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (there && head_element(d, r) < p.DK) slot[static_cast<int64_t>(head_element(d, r)) * p.DV] = state[d][r];
    }
    bool forgotten = false;
    if constexpr (!Reader::kDirect) fetch(begin);
    for (int chunk = begin; chunk < live; ++chunk) {
        const int64_t index = static_cast<int64_t>(head) * p.chunks + chunk;
        typename Reader::Buffers& here = lds[chunk % Reader::kBuffers];
        const uint16_t *keys = here.keys, *queries = here.queries;
        T* tile = here.tile;
        const uint32_t *block = here.block, *vectors = block + block_vectors(TRANSFER ? 0 : RANKS);
        reader.wait(here);
        if constexpr (!Reader::kDirect) fetch(chunk + 1);
        now();
        // S k and S q, the state's terms a step ahead of the products that take them
        f32x4 ks[4], out[4], right[4], delta[4], since[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ks[i] = out[i] = delta[i] = f32x4{0, 0, 0, 0};
        Terms<TERMS> a[PIPE][8];
        Terms<3> x[2] = {split<3>(state[0], state[1]), {}}, inverse[kBlocks];
        const auto load = [&](int s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[s % PIPE][i] = Lds::rows(keys, i, s);
                if constexpr (!TRANSFER) a[s % PIPE][4 + i] = Lds::rows(queries, i, s);
            }
        };
        load(0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            now();
            if (PIPE == 2 && s + 1 < KS) load(s + 1);
            if constexpr (TRAIN)
                if (s % 2 == 1) store_marks<KS, RANKS>(p.marks + index * (RANKS * padded_values(p.DV) * 32 * KS), p.DV, mine, s - 1, x[0].t, x[1].t);
            if (s + 1 < KS) x[(s + 1) % 2] = split<3>(state[2 * s + 2], state[2 * s + 3]);
            if (s + 1 == KS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) right[i] = Values::get(tile, i), since[i] = row_factors(vectors, kSince, i);
                if constexpr (PIPE == 2) {
#pragma unroll
                    for (int f = 0; f < 2; ++f) inverse[f] = block_terms<3>(block, f);
                }
            }
#pragma unroll
            for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                for (int j = 0; j <= rank; ++j)
                    if (j < TERMS) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) ks[i] = mfma(a[s % PIPE][i].t[j], x[s % 2].t[rank - j], ks[i]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!TRANSFER && rank < RANKS) out[i] = mfma(a[s % PIPE][4 + i].t[j], x[s % 2].t[rank - j], out[i]);
                    }
            if (PIPE == 1 && s + 1 < KS) load(s + 1);
        }
        const bool broken = __builtin_amdgcn_readfirstlane(vectors[kBroken]) != 0;
        const float rest = __uint_as_float(__builtin_amdgcn_readfirstlane(vectors[kSince + kChunk - 1]));
        if constexpr (TRANSFER) forgotten = forgotten || rest == 0.0f;
        if (broken) {
#pragma unroll
            for (int i = 0; i < 4; ++i) drop(ks[i], since[i]), drop(out[i], since[i]);
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) drop(state[d], f32x4{rest, rest, rest, rest});
        }
        // delta
        now();
        uint32_t infinite = 0;
        bool finite;
        Terms<RANKS> scores[kBlocks];
        f32x4 beta[4];
        {
#pragma unroll
            for (int i = 0; i < 4; ++i) right[i] -= since[i] * ks[i];
            finite = all_finite(right);
            if (!finite) infinite = take_out(right, vectors[kFresh] | static_cast<uint64_t>(vectors[kFresh + 1]) << 32);
#pragma unroll
            for (int f = PIPE == 2 ? 2 : 0; f < kBlocks; ++f) inverse[f] = block_terms<3>(block, f);
            const Terms<3> y[2] = {split<3>(right[0], right[1]), split<3>(right[2], right[3])};
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                    for (int j = 0; j <= rank; ++j)
#pragma unroll
                        for (int f = 0; f < kBlocks; ++f)
                            if (lower_half(f) == half) delta[lower_tile(f)] = mfma(inverse[f].t[j], y[half].t[rank - j], delta[lower_tile(f)]);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] *= since[i] * p.scale, beta[i] = row_factors(vectors, kBeta, i);
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) state[d] *= rest;
#pragma unroll
            for (int f = 0; f < kBlocks; ++f)
                if constexpr (WALK == kOutputs) scores[f] = block_terms<RANKS>(block + kBlocks * 3 * 256, f);
        }
        if constexpr (TRAIN) {
            now();
            Values::template write_terms<RANKS>(tile, delta, p.deltas + index * (RANKS * kChunk * padded_values(p.DV)) + mine * kChunk, padded_values(p.DV));
            now();
#pragma unroll
            for (int f = 0; f < kBlocks; ++f) scores[f] = block_terms<RANKS>(block + kBlocks * 3 * 256, f);
        }
        // What the steps read of each other, and the state behind them
        f32x4 until[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) until[i] = row_factors(vectors, kUntil, i), delta[i] *= beta[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) right[i] = delta[i];
        if (!finite) put_back(right, infinite);
        if (broken) {
#pragma unroll
            for (int i = 0; i < 4; ++i) drop(right[i], until[i]);
        }
        now();
        {
            Terms<TERMS> k[PIPE][2 * KS];
            const auto columns_of = [&](int half) {
#pragma unroll
                for (int d = 0; d < 2 * KS; ++d) k[half % PIPE][d] = Lds::columns(keys, d, half);
            };
            columns_of(0);
#pragma unroll
            for (int half = 0; half < 2 && !TRANSFER; ++half) {
                const Terms<RANKS> y = split<RANKS>(delta[2 * half], delta[2 * half + 1]);
#pragma unroll
                for (int rank = RANKS - 1; rank >= 0; --rank)
#pragma unroll
                    for (int j = 0; j <= rank; ++j)
#pragma unroll
                        for (int f = 0; f < kBlocks; ++f)
                            if (lower_half(f) == half) out[lower_tile(f)] = mfma(scores[f].t[j], y.t[rank - j], out[lower_tile(f)]);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (PIPE == 2 && half == 0) columns_of(1);
                if (PIPE == 1 && half == 1) columns_of(1);
                const Terms<3> y = split<3>(right[2 * half] * until[2 * half], right[2 * half + 1] * until[2 * half + 1]);
#pragma unroll
                for (int rank = 2; rank >= 0; --rank)
#pragma unroll
                    for (int j = 0; j <= rank; ++j)
                        if (j < TERMS) {
#pragma unroll
                            for (int d = 0; d < 2 * KS; ++d) state[d] = mfma(k[half % PIPE][d].t[j], y.t[rank - j], state[d]);
                        }
            }
            if (!TRANSFER && !finite) put_back(out, infinite);
            if constexpr (!TRANSFER) Values::turn_values(tile, out);
        }
        now();
        if constexpr (!TRANSFER) Values::write(tile, out_base + static_cast<int64_t>(chunk) * kChunk * p.out.step, p.out.step, p.T - chunk * kChunk, limit - chunk * kChunk, p.DV - mine, p.near_values);
    }
    if constexpr (TRANSFER) {
        float* to = p.transfers + static_cast<int64_t>(item) * transfer_floats(KS, p.DV);
        if (there) store_transfer<KS>(to, state, matrix, column, padded_values(p.DV));
        if (matrix && columns == value_parts && threadIdx.x == 0) to[transfer_floats(KS, p.DV) - 4] = forgotten ? 1.0f : 0.0f;
    } else if (segment == last) {
        for (int t = chunks * kChunk + wave * 4 + group; t < p.T; t += 4 * WAVES)      // padding
            for (int c = left + lane % 16; c < p.DV && c < left + Values::kColumns; c += 16) out_base[t * p.out.step + c - mine] = from_float<T>(0.0f);
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = head_element(d, r);
                if (there && row < p.DK) p.state_out[cell + static_cast<int64_t>(row) * p.DV] = state[d][r];
            }
    }
}

// The states between a head's segments, one after the other: 16 columns to a workgroup, 32 of the rows that are summed over to a wave. Products in float32, whose operands are what
// memory and accumulators hold: 64 a wave and step of 32 cycles each, 2.3 us with the exchange, the next segment's matrix on its way.
template <int KS>
__global__ __launch_bounds__(64 * KS) void delta_join_kernel(DeltaArgs p, int backward) {
    __shared__ f32x4 parts[2][KS][2 * KS][64];
    int head, tile;
    if (!part_of_head(p.N * p.HV, (p.DV + 15) / 16, &head, &tile)) return;
    const int n = head / p.HV, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, column = 16 * tile + lane % 16;
    const int chunks = (length_of(p, n) + kChunk - 1) / kChunk, last = chunks == 0 ? 0 : (chunks - 1) / p.per;
    const float* transfers = p.transfers + static_cast<int64_t>(head) * (p.segments - 1) * transfer_floats(KS, p.DV);
    float* between = p.between + static_cast<int64_t>(head) * p.segments * p.DK * p.DV;
    // Rows of the matrix as the accumulators have them, the wave's columns of it as they lie in the other operand; what the segment adds to the wave's own rows
    struct Segment {
        f32x4 matrix[2 * KS][2];
        f32x4 added[2];
        float forgotten;
    };
    const auto load = [&](Segment& x, int step) {
        step = step < last ? step : last - 1;
        const float* from = transfers + static_cast<int64_t>(backward ? last - 1 - step : step) * transfer_floats(KS, p.DV);
        x.forgotten = from[transfer_floats(KS, p.DV) - 4];
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
            for (int i = 0; i < 2; ++i) x.matrix[d][i] = *reinterpret_cast<const f32x4*>(from + (((wave * 2 * KS + d) * 2 + i) * 64 + lane) * 4);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) x.added[i][r] = from[transfer_matrix(KS) + head_element(2 * wave + i, r) * padded_values(p.DV) + column];
        now();
    };
    f32x4 state[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    const auto advance = [&](const Segment& x, int step) {
        if (step >= last) return;
        if (step > 0) {
            f32x4 sums[2 * KS];
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) sums[d] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float s = x.forgotten == 0.0f ? state[i][r] : 0.0f;       // an infinite state as well
#pragma unroll
                    for (int d = 0; d < 2 * KS; ++d) sums[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.matrix[d][i][r], s, sums[d], 0, 0, 0);
                }
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) parts[step % 2][wave][d][lane] = sums[d];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            state[i] = x.added[i];
            if (step > 0) {
#pragma unroll
                for (int w = 0; w < KS; ++w) state[i] += parts[step % 2][w][2 * wave + i][lane];
            }
            float* to = between + static_cast<int64_t>(backward ? last - 1 - step : step + 1) * p.DK * p.DV;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = head_element(2 * wave + i, r);
                if (row < p.DK && column < p.DV) to[row * p.DV + column] = state[i][r];
            }
        }
    };
    if (last == 0) return;
    Segment even, odd;
    load(even, 0);
    for (int step = 0; step < last; step += 2) {
        load(odd, step + 1);
        advance(even, step);
        load(even, step + 2);
        advance(odd, step + 1);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// A few steps
// ------------------------------------------------------------------------------------------------------------------
// Step by step, in float32: 64 columns of the state to a workgroup, 8 rows and 4 columns to a thread. k . S and q . S are summed over the rows in one
// exchange; out = scale (q . S + (q . k) beta delta). One step is bound by memory, 33.7 MB for 16 requests x 16 heads of 128 x 128 in 8.4 us (4.0 TB/s, a launch's start and end among them), each further one by the
// vector units, 0.9 us. 16 steps take 23.2 us and 17 as a chunk 29.7 (one request 16.8 and 19.6), so that 17 to some 20 would be faster step by step; they go in chunks since the steps' operands
// go to LDS at once, a piece of one step to a thread, of which there are as many as 16 steps have pieces.
// Of four numbers at once: row g of 16 lanes gets the sum of the g-th.
__device__ __forceinline__ float sums_of_rows(float a, float b, float c, float d) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(c), __float_as_uint(d), false, false);
    const float ab = __uint_as_float(x[0]) + __uint_as_float(x[1]), cd = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(ab), __float_as_uint(cd), false, false);
    return __uint_as_float(z[0]) + __uint_as_float(z[1]);
}

constexpr int kFewSteps = 16;

template <typename T, int KS>
__global__ __launch_bounds__(64 * KS) void delta_step_kernel(DeltaArgs p) {
    constexpr int PER = 4 * KS, COLUMNS = 64 / PER;     // pieces of 8 elements of a head, of which a thread has one of one step, and columns that it has of that
    static_assert(kFewSteps * PER == 64 * KS, "a thread to a piece");
    __shared__ alignas(16) float keys[kFewSteps][32 * KS], queries[kFewSteps][32 * KS], values[kFewSteps][64];
    __shared__ float decays[kFewSteps], rates[kFewSteps];
    __shared__ f32x4 sums[2][KS][16][3];
    int head, columns;
    if (!part_of_head(p.N * p.HV, (p.DV + 63) / 64, &head, &columns)) return;
    const int n = head / p.HV, hv = head % p.HV, h = hv / (p.HV / p.H), limit = length_of(p, n);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, column = columns * 64 + 4 * (lane % 16), row = 8 * (threadIdx.x / 16);
    const int left = p.DV - column;
    const int64_t cell = static_cast<int64_t>(head) * p.DK * p.DV + column;
    Raw<float, 4> state[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (p.state != nullptr && row + i < p.DK && left > 0) state[i].load(p.state + cell, static_cast<int64_t>(row + i) * p.DV, left);
        else state[i].clear();
    }
    // All steps' keys, queries, values and gates at once, to LDS
    {
        const int t = threadIdx.x / PER, piece = threadIdx.x % PER, at = 8 * piece, first = columns * 64 + COLUMNS * piece;
        Raw<T, 8> k, q;
        float v[COLUMNS];
        k.clear();
        q.clear();
        if (t < limit && at < p.DK) {
            k.load(static_cast<const T*>(p.k.data) + n * p.k.row + h * p.k.head, t * p.k.step + at, p.DK - at);
            q.load(static_cast<const T*>(p.q.data) + n * p.q.row + h * p.q.head, t * p.q.step + at, p.DK - at);
        }
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c)
            v[c] = t < limit && first + c < p.DV ? to_float(static_cast<const T*>(p.v.data)[n * p.v.row + hv * p.v.head + t * p.v.step + first + c]) : 0.0f;
        if (static_cast<int>(threadIdx.x) < limit) {
            const int64_t step = threadIdx.x;
            const float g = gate_value<T>(p.gate, p.gate_float, threadIdx.x, n, hv, 0.0f);
            const bool fresh = g < kForgotten || (p.starts != nullptr && p.starts[step * p.starts_step + n * p.starts_row] != 0);
            decays[threadIdx.x] = fresh ? 0.0f : expf(g);
            rates[threadIdx.x] = gate_value<T>(p.beta, p.gate_float, threadIdx.x, n, hv, 1.0f);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) keys[t][at + j] = k[j], queries[t][at + j] = q[j];
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) values[t][COLUMNS * piece + c] = v[c];
    }
    __syncthreads();
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][c] = state[i][c];
    T* outs = static_cast<T*>(const_cast<void*>(p.out.data)) + n * p.out.row + hv * p.out.head + column;
    for (int t = 0; t < limit; ++t) {
        const float a = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(decays[t]))), b = rates[t];
        float k[8], q[8], v[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = keys[t][row + i], q[i] = queries[t][row + i];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = values[t][4 * (lane % 16) + c];
        if (a == 0.0f) {                // infinities and NaN as well
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[i][c] = 0.0f;
        }
        float part[9];
#pragma unroll
        for (int c = 0; c < 9; ++c) part[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            part[8] = fmaf(k[i], q[i], part[8]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[i][c] *= a;
                part[c] = fmaf(k[i], s[i][c], part[c]);
                part[4 + c] = fmaf(q[i], s[i][c], part[4 + c]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) sums[t & 1][wave][lane % 16][i][lane / 16] = sums_of_rows(part[4 * i], part[4 * i + 1], part[4 * i + 2], part[4 * i + 3]);
        sums[t & 1][wave][lane % 16][2][0] = sum_of_rows(part[8]);
        __syncthreads();
        f32x4 all[KS][2];
        float dots[KS];
#pragma unroll
        for (int w = 0; w < KS; ++w) {
#pragma unroll
            for (int i = 0; i < 2; ++i) all[w][i] = sums[t & 1][w][lane % 16][i];
            dots[w] = sums[t & 1][w][lane % 16][2][0];
        }
#pragma unroll
        for (int c = 0; c < 9; ++c) {
            part[c] = c < 8 ? all[0][c / 4][c % 4] : dots[0];
#pragma unroll
            for (int w = 1; w < KS; ++w) part[c] += c < 8 ? all[w][c / 4][c % 4] : dots[w];
        }
        float u[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u[c] = b * (v[c] - part[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i][c] = fmaf(k[i], u[c], s[i][c]);
        }
        if (threadIdx.x < 16) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c < left) outs[t * p.out.step + c] = from_float<T>(p.scale * fmaf(part[8], u[c], part[4 + c]));
        }
    }
    for (int t = limit; t < p.T; ++t)
        if (threadIdx.x < 16) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c < left) outs[t * p.out.step + c] = from_float<T>(0.0f);
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        state[i].put(0, s[i][0], s[i][1]);
        state[i].put(2, s[i][2], s[i][3]);
        if (row + i < p.DK && left > 0) state[i].store(p.state_out + cell, static_cast<int64_t>(row + i) * p.DV, left);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------------------------
template <typename T, int KS, int WAVES, int RANKS, Walk WALK>
void launch_walk(const DeltaArgs& p, int segments, int parts, hipStream_t stream) {
    delta_walk_kernel<T, KS, WAVES, RANKS, WALK><<<head_grid(p.N * p.HV * segments, parts), dim3(walk_threads<T>(WAVES)), 0, stream>>>(p);
}

template <typename T, int KS, int RANKS, Walk WALK>
void launch_walks(const DeltaArgs& p, hipStream_t stream) {
    launch_chunks<T, KS, RANKS, false>(p, stream);
    if (p.segments > 1) {
        constexpr int WAVES = sizeof(T) == 2 ? 8 : 4;
        launch_walk<T, KS, WAVES, RANKS, kTransfer>(p, p.segments - 1, transfer_parts(WAVES, KS, p.DV), stream);
        launch_join<KS>(p, false, stream);
    }
    if constexpr (kTerms<T> == 1) {
        if (two_waves(p)) {
            launch_walk<T, KS, 2, RANKS, WALK>(p, p.segments, (p.DV + 31) / 32, stream);
            return;
        }
    }
    launch_walk<T, KS, 4, RANKS, WALK>(p, p.segments, (p.DV + 63) / 64, stream);
}

template <typename T, int KS>
void launch_forward(const DeltaArgs& p, int ranks, hipStream_t stream) {
    if (p.blocks == nullptr) delta_step_kernel<T, KS><<<head_grid(p.N * p.HV, (p.DV + 63) / 64), dim3(64 * KS), 0, stream>>>(p);
    else if (p.marks == nullptr) launch_walks<T, KS, kOutputRanks<T>, kOutputs>(p, stream);
    else if (ranks == 3) launch_walks<T, KS, 3, kTraining>(p, stream);
    else if constexpr (kOutputRanks<T> == 2) launch_walks<T, KS, 2, kTraining>(p, stream);
}

}  // namespace

template <int KS>
void launch_join(const DeltaArgs& p, bool backward, hipStream_t stream) {
    delta_join_kernel<KS><<<head_grid(p.N * p.HV, (p.DV + 15) / 16), dim3(64 * KS), 0, stream>>>(p, backward);
}
template void launch_join<2>(const DeltaArgs&, bool, hipStream_t);
template void launch_join<4>(const DeltaArgs&, bool, hipStream_t);

// As many as fill the chip on both walks, of 3 chunks at least, no more than the states between them are worth (a step there costs a third of a chunk), and 3 at least: with 2 the
// first walk takes the time that the second saves. Two more launches cost what 6 to 10 chunks of a walk do (16 heads of 128, with and without segments: bfloat16 16 chunks 67 and 66 us,
// 20 72 and 81, 32 82 and 115; float16 9 chunks 78 and 73, 12 82 and 93; float32 9 chunks 89 and 105).
int delta_segments(const snnf_delta_rule_call* c, bool backward) {
    const int64_t heads = static_cast<int64_t>(c->N) * c->value_heads, chunks = (c->T + kChunk - 1) / kChunk, units = compute_units();
    if (heads == 0 || heads > units || chunks <= (c->dtype == SNNF_BF16 ? 16 : 9)) return 1;
    const int waves = dtype_size(c->dtype) == 2 && !backward ? 8 : 4;
    int64_t segments = 1 + units / (heads * transfer_parts(waves, c->key_size <= 64 ? 2 : 4, c->value_size));
    segments = std::min(segments, units / (heads * ((c->value_size + 63) / 64)));
    segments = std::min(segments, chunks / 3);
    while (segments * segments > 8 * chunks) --segments;
    if (segments < 3) return 1;
    const int64_t per = (chunks + segments - 1) / segments;
    return static_cast<int>((chunks + per - 1) / per);
}
size_t delta_segment_floats(const snnf_delta_rule_call* c, bool backward) {
    const int64_t heads = static_cast<int64_t>(c->N) * c->value_heads, segments = delta_segments(c, backward);
    return segments == 1 ? 0 : static_cast<size_t>(heads * ((segments - 1) * transfer_floats(c->key_size <= 64 ? 2 : 4, c->value_size) + segments * c->key_size * c->value_size));
}
void set_segments(DeltaArgs& p, const snnf_delta_rule_call* c, bool backward, float* workspace) {
    p.segments = delta_segments(c, backward);
    p.per = (p.chunks + p.segments - 1) / p.segments;
    p.transfers = workspace;
    p.between = workspace + static_cast<int64_t>(p.N) * p.HV * (p.segments - 1) * transfer_floats(c->key_size <= 64 ? 2 : 4, p.DV);
}

template <typename T, int KS, int RANKS, bool BACKWARD>
void launch_chunks(const DeltaArgs& p, hipStream_t stream) {
    delta_chunk_kernel<T, KS, RANKS, BACKWARD><<<grid_of(static_cast<int64_t>(p.N) * p.HV * p.chunks), dim3(256), 0, stream>>>(p);
}
template void launch_chunks<float, 2, 3, true>(const DeltaArgs&, hipStream_t);
template void launch_chunks<float, 4, 3, true>(const DeltaArgs&, hipStream_t);
template void launch_chunks<bf16_t, 2, 3, true>(const DeltaArgs&, hipStream_t);
template void launch_chunks<bf16_t, 4, 3, true>(const DeltaArgs&, hipStream_t);
template void launch_chunks<f16_t, 2, 3, true>(const DeltaArgs&, hipStream_t);
template void launch_chunks<f16_t, 4, 3, true>(const DeltaArgs&, hipStream_t);

int check_delta(const char* name, const snnf_delta_rule_call* c) {
    if (c == nullptr) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: no call", name);
    if (c->T < 0 || c->N < 0 || c->heads < 0 || c->value_heads < 0 || c->key_size < 0 || c->value_size < 0)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: T=%d N=%d heads=%d value_heads=%d key_size=%d value_size=%d", name, c->T, c->N, c->heads, c->value_heads,
                    c->key_size, c->value_size);
    if (!valid_dtype(c->dtype) || (c->gate_dtype != c->dtype && c->gate_dtype != SNNF_F32))
        return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: dtype codes %d and, for gates, %d", name, c->dtype, c->gate_dtype);
    if (c->heads == 0 || c->value_heads % c->heads != 0)
        return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: value heads (%d) must be a multiple of heads (%d)", name, c->value_heads, c->heads);
    if (c->key_size < 1 || c->key_size > SNNF_DELTA_RULE_MAX_KEY || c->value_size < 1 || c->value_size > SNNF_DELTA_RULE_MAX_VALUE)
        return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: keys of 1 to %d and values of 1 to %d elements, got %d and %d", name, SNNF_DELTA_RULE_MAX_KEY,
                    SNNF_DELTA_RULE_MAX_VALUE, c->key_size, c->value_size);
    if (c->T > (1 << 30) || static_cast<int64_t>(c->N) * c->value_heads > (1 << 20) ||
        static_cast<int64_t>(c->N) * c->value_heads * ((c->T + kChunk - 1) / kChunk) > (1 << 30))
        return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: at most 2^20 heads of all sequences and 2^30 steps of 64 of them, got N=%d, %d heads, T=%d", name, c->N,
                    c->value_heads, c->T);
    return SNNF_OK;
}

DeltaArgs delta_args(const snnf_delta_rule_call* c) {
    const auto view = [](const snnf_heads& x) { return HeadView{x.data, x.step, x.row, x.head}; };
    DeltaArgs p = {};
    p.q = view(c->query), p.k = view(c->key), p.v = view(c->value), p.gate = view(c->gate), p.beta = view(c->beta);
    p.T = c->T, p.N = c->N, p.H = c->heads, p.HV = c->value_heads, p.DK = c->key_size, p.DV = c->value_size;
    p.chunks = (c->T + kChunk - 1) / kChunk;
    p.scale = c->scale;
    p.gate_float = c->gate_dtype == SNNF_F32;
    p.starts = static_cast<const uint8_t*>(c->starts), p.starts_step = c->starts_step, p.starts_row = c->starts_row;
    p.lengths = c->lengths;
    p.state = c->state;
    p.near_keys = c->key_size % 8 == 0 && near_by(p.q, c->dtype, true) && near_by(p.k, c->dtype, true);
    p.near_values = c->value_size % 8 == 0 && near_by(p.v, c->dtype, true);
    return p;
}

int delta_ranks(const snnf_delta_rule_call* c, bool training) { return c->dtype == SNNF_F32 || (training && c->gate_dtype == SNNF_F32) ? 3 : 2; }
int64_t delta_mark_elements(const snnf_delta_rule_call* c) { return mark_elements(delta_ranks(c, true), c->key_size <= 64 ? 2 : 4, c->value_size); }
int64_t delta_chunks(const snnf_delta_rule_call* c) {
    return static_cast<int64_t>(c->N) * c->value_heads * ((c->T + kChunk - 1) / kChunk);
}

}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_delta_rule_workspace_bytes(const snnf_delta_rule_call* call, int training) {
    if (check_delta("snnf_delta_rule_workspace_bytes", call) != SNNF_OK || (!training && call->T <= kFewSteps)) return 0;
    return static_cast<size_t>(delta_chunks(call)) * block_words(delta_ranks(call, training != 0)) * 4 + delta_segment_floats(call, false) * 4;
}

extern "C" size_t snnf_delta_rule_marks_bytes(const snnf_delta_rule_call* call) {
    if (check_delta("snnf_delta_rule_marks_bytes", call) != SNNF_OK) return 0;
    return static_cast<size_t>(delta_chunks(call)) * (delta_mark_elements(call) + delta_elements(delta_ranks(call, true), call->value_size)) * sizeof(uint16_t);
}

extern "C" int snnf_delta_rule(const snnf_delta_rule_call* call, const snnf_heads* out, float* state_out, void* marks, void* workspace, size_t workspace_bytes,
                               void* stream) {
    const int rc = check_delta("snnf_delta_rule", call);
    if (rc != SNNF_OK) return rc;
    if (call->T == 0 || call->N == 0) return SNNF_OK;
    if (call->query.data == nullptr || call->key.data == nullptr || call->value.data == nullptr || out == nullptr || out->data == nullptr || state_out == nullptr)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_delta_rule: query, key, value, out and state_out must be non-null");
    DeltaArgs p = delta_args(call);
    p.out = HeadView{out->data, out->step, out->row, out->head};
    p.state_out = state_out;
    const size_t need = snnf_delta_rule_workspace_bytes(call, marks != nullptr);
    if (need > 0) {
        if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
            return fail(SNNF_ERR_WORKSPACE, "snnf_delta_rule: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
        p.blocks = static_cast<uint32_t*>(workspace);
        set_segments(p, call, false, reinterpret_cast<float*>(p.blocks + delta_chunks(call) * block_words(delta_ranks(call, marks != nullptr))));
    }
    if (marks != nullptr) {
        if (!aligned_to(marks, 16)) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_delta_rule: marks must lie on 16 bytes");
        p.marks = static_cast<uint16_t*>(marks);
        p.deltas = p.marks + delta_chunks(call) * delta_mark_elements(call);
    }
    p.near_values = p.near_values && near_by(p.out, call->dtype, false);
    hipStream_t hs = as_stream(stream);
    const bool small = call->key_size <= 64;
    const int ranks = delta_ranks(call, marks != nullptr);
    if (call->dtype == SNNF_F32) small ? launch_forward<float, 2>(p, ranks, hs) : launch_forward<float, 4>(p, ranks, hs);
    else if (call->dtype == SNNF_BF16) small ? launch_forward<bf16_t, 2>(p, ranks, hs) : launch_forward<bf16_t, 4>(p, ranks, hs);
    else small ? launch_forward<f16_t, 2>(p, ranks, hs) : launch_forward<f16_t, 4>(p, ranks, hs);
    return check_launch("snnf_delta_rule");
}
