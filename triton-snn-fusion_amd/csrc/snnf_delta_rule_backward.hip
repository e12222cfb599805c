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
__global__ __launch_bounds__(256, 1) void delta_walk_back_kernel(DeltaArgs p) {
    using Lds = Rows<T, KS>;
    constexpr int BUFFERS = kTerms<T> == 1 ? 2 : 1;
    __shared__ uint16_t lds[BUFFERS][2][Lds::kSize];
    int head, columns;
    if (!part_of_head(p.N * p.HV, (p.DV + 63) / 64, &head, &columns)) return;
    const int n = head / p.HV, hv = head % p.HV, h = hv / (p.HV / p.H), limit = length_of(p, n), live = (limit + kChunk - 1) / kChunk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane / 16, column = columns * 64 + wave * 16 + lane % 16;
    const bool there = column < p.DV;
    const int64_t cell = static_cast<int64_t>(head) * p.DK * p.DV + column;
    f32x4 later[2 * KS];
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * d + 4 * group + r;
            later[d][r] = p.dstate != nullptr && there && row < p.DK ? p.dstate[cell + static_cast<int64_t>(row) * p.DV] : 0.0f;
        }
    const T* douts = static_cast<const T*>(p.dout.data) + n * p.dout.row + hv * p.dout.head + column;
    T* dvalues = static_cast<T*>(const_cast<void*>(p.dv.data)) + n * p.dv.row + hv * p.dv.head + column;
    T o[16];
    const auto fetch = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int t = chunk * kChunk + 16 * (i / 4) + 4 * group + i % 4;
            o[i] = there && t < limit ? douts[t * p.dout.step] : from_float<T>(0.0f);
        }
    };
    Staged<T, KS, 256> k_next, q_next;
    if (live > 0) {
        k_next.load(p.k, (live - 1) * kChunk, limit, n, h, p.DK);
        q_next.load(p.q, (live - 1) * kChunk, limit, n, h, p.DK);
        fetch(live - 1);
    }
    for (int chunk = live - 1; chunk >= 0; --chunk) {
        const int64_t index = static_cast<int64_t>(head) * p.chunks + chunk;
        uint16_t *keys = lds[chunk % BUFFERS][0], *queries = lds[chunk % BUFFERS][1];
        if constexpr (BUFFERS == 1) __syncthreads();
        k_next.store(keys);
        q_next.store(queries);
        __syncthreads();
        const uint32_t* blocks = p.blocks + index * block_words(3) + lane * 4;
        const float* vectors = p.vectors + index * 3 * kChunk + 4 * group;
        f32x4 since[4], until[4], beta[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            since[i] = *reinterpret_cast<const f32x4*>(vectors + 16 * i);
            until[i] = *reinterpret_cast<const f32x4*>(vectors + kChunk + 16 * i);
            beta[i] = *reinterpret_cast<const f32x4*>(vectors + 2 * kChunk + 16 * i);
        }
        const float rest = p.vectors[index * 3 * kChunk + kChunk - 1];
        f32x4 dout[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) dout[i / 4][i % 4] = to_float(o[i]);
        if (chunk > 0) {
            k_next.load(p.k, (chunk - 1) * kChunk, limit, n, h, p.DK);
            q_next.load(p.q, (chunk - 1) * kChunk, limit, n, h, p.DK);
            fetch(chunk - 1);
        }
        {
            float* marks = p.later + index * p.DK * p.DV + column;
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * d + 4 * group + r;
                    if (there && row < p.DK) marks[row * p.DV] = later[d][r];
                }
        }
        f32x4 pull[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pull[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const Terms<3> x = split<3>(later[2 * s], later[2 * s + 1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) pull[i] = product<3>(Lds::rows(keys, i, s), x, pull[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) pull[i][r] = kept(until[i][r], pull[i][r]);
        {
            const Terms<kTerms<T>> x[2] = {split<kTerms<T>>(dout[0], dout[1]), split<kTerms<T>>(dout[2], dout[3])};
#pragma unroll
            for (int f = 0; f < kBlocks; ++f) {
                Terms<3> scores;
#pragma unroll
                for (int i = 0; i < 3; ++i) scores.t[i] = *reinterpret_cast<const u32x4a*>(blocks + ((kBlocks + f) * 3 + i) * 256);
                pull[upper_tile(f)] = product<3>(scores, x[upper_half(f)], pull[upper_tile(f)]);
            }
        }
        f32x4 z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = f32x4{0, 0, 0, 0};
        {
            const Terms<3> x[2] = {split<3>(pull[0], pull[1]), split<3>(pull[2], pull[3])};
#pragma unroll
            for (int f = 0; f < kBlocks; ++f) {
                Terms<3> inverse;
#pragma unroll
                for (int i = 0; i < 3; ++i) inverse.t[i] = *reinterpret_cast<const u32x4a*>(blocks + (f * 3 + i) * 256);
                z[upper_tile(f)] = product<3>(inverse, x[upper_half(f)], z[upper_tile(f)]);
            }
        }
        float* pulls = p.pulls + index * kChunk * p.DV + column;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int at = 16 * (i / 4) + 4 * group + i % 4, t = chunk * kChunk + at;
            if (there) pulls[at * p.DV] = z[i / 4][i % 4];
            z[i / 4][i % 4] *= beta[i / 4][i % 4];
            if (there && t < p.T) dvalues[t * p.dv.step] = from_float<T>(t < limit ? z[i / 4][i % 4] : 0.0f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                z[i][r] = kept(since[i][r], -z[i][r]);
                dout[i][r] = kept(since[i][r] * p.scale, dout[i][r]);
            }
        {
            const Terms<3> x[2] = {split<3>(z[0], z[1]), split<3>(z[2], z[3])}, y[2] = {split<3>(dout[0], dout[1]), split<3>(dout[2], dout[3])};
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) {
#pragma unroll
                for (int r = 0; r < 4; ++r) later[d][r] = kept(rest, later[d][r]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    later[d] = product<3>(Lds::columns(keys, d, half), x[half], later[d]);
                    later[d] = product<3>(Lds::columns(queries, d, half), y[half], later[d]);
                }
            }
        }
    }
    for (int t = live * kChunk + wave * 4 + group; t < p.T; t += 16)      // padding
        for (int c = columns * 64 + lane % 16; c < p.DV && c < columns * 64 + 64; c += 16)
            dvalues[t * p.dv.step + c - column] = from_float<T>(0.0f);
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * d + 4 * group + r;
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
__device__ __forceinline__ void floats_of(float (&x)[8], const float* row, int at, int width, bool there) {
    Raw<float, 8> raw;
    if (there && at < width) raw.load(row, at, width - at);
    else raw.clear();
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = raw[j];
}
template <typename T>
__device__ __forceinline__ void store_four(T* to, int left, const f32x4& x) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < left) to[r] = from_float<T>(x[r]);
}

template <typename T, int KS>
__global__ __launch_bounds__(256, 1) void delta_gradient_kernel(DeltaArgs p) {
    using Lds = Rows<T, KS>;
    constexpr int RANKS = kOutputRanks<T>, TILES = 2 * KS;
    __shared__ uint16_t keys[Lds::kSize], queries[Lds::kSize];
    __shared__ double total[kChunk];
    __shared__ int part[kChunk];
    __shared__ float betas[kChunk], dsums[kChunk], tails[kChunk], dots[4];
    const uint32_t place = group_index();
    if (place >= static_cast<uint32_t>(p.N) * p.H * p.chunks) return;
    const int chunk = place % p.chunks, n = place / p.chunks / p.H, h = place / p.chunks % p.H, first = chunk * kChunk, limit = length_of(p, n);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane / 16, column = lane % 16, own = 16 * wave + column, t_own = first + own;
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
    if (first < limit) {
        Staged<T, KS, 256> k_rows, q_rows;
        k_rows.load(p.k, first, limit, n, h, p.DK);
        q_rows.load(p.q, first, limit, n, h, p.DK);
        k_rows.store(keys);
        q_rows.store(queries);
    }
    for (int member = 0; member < members; ++member) {
        const int hv = h * members + member;
        if (first >= limit) {
            if (group == 0 && t_own < p.T) store_gate(p.dgate, t_own, hv, 0.0f), store_gate(p.dbeta, t_own, hv, 0.0f);
            continue;
        }
        const int64_t index = (static_cast<int64_t>(n) * p.HV + hv) * p.chunks + chunk;
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
            betas[lane] = p.vectors[index * 3 * kChunk + 2 * kChunk + lane];
        }
        const float since = p.vectors[index * 3 * kChunk + own], until = p.vectors[index * 3 * kChunk + kChunk + own];
        const float beta = p.vectors[index * 3 * kChunk + 2 * kChunk + own];
        const float *marks = p.marks + index * p.DK * p.DV, *later = p.later + index * p.DK * p.DV;
        const float *deltas = p.deltas + index * kChunk * p.DV, *pulls = p.pulls + index * kChunk * p.DV;
        const T* douts = static_cast<const T*>(p.dout.data) + n * p.dout.row + hv * p.dout.head;
        const T* values = static_cast<const T*>(p.v.data) + n * p.v.row + hv * p.v.head;
        f32x4 score_row[4], score_column[4], pull_row[4], pull_column[4], dq[TILES], ds[TILES], dk[TILES];
#pragma unroll
        for (int j = 0; j < 4; ++j) score_row[j] = score_column[j] = pull_row[j] = pull_column[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < TILES; ++d) dq[d] = ds[d] = dk[d] = f32x4{0, 0, 0, 0};
        float dbeta = 0.0f, zv = 0.0f, dot = 0.0f;
        for (int s = 0; 32 * s < p.DV; ++s) {
            const int at = 32 * s + 8 * group;
            float z[8], delta[8];
            floats_of(z, pulls + own * p.DV, at, p.DV, true);
            floats_of(delta, deltas + own * p.DV, at, p.DV, true);
            const auto o_own = there && at < p.DV ? row_terms<T>(douts + t_own * p.dout.step, at, p.DV) : no_terms<kTerms<T>>();
            const Terms<RANKS> z_own = split<RANKS>(z), delta_own = split<RANKS>(delta);
            Raw<T, 8> v;
            if (there && at < p.DV) v.load(values + t_own * p.v.step, at, p.DV - at);
            else v.clear();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dbeta = fmaf(z[j], delta[j], dbeta);
                zv = fmaf(z[j], v[j], zv);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[8];
                if (j <= wave) {
                    floats_of(x, deltas + (16 * j + column) * p.DV, at, p.DV, true);
                    const Terms<RANKS> a = split<RANKS>(x);
                    score_row[j] = product<RANKS>(a, o_own, score_row[j]);
                    pull_row[j] = product<RANKS>(a, z_own, pull_row[j]);
                }
                if (j >= wave) {
                    const int t = first + 16 * j + column;
                    const auto o = t < limit && at < p.DV ? row_terms<T>(douts + t * p.dout.step, at, p.DV) : no_terms<kTerms<T>>();
                    score_column[j] = product<RANKS>(o, delta_own, score_column[j]);
                    floats_of(x, pulls + (16 * j + column) * p.DV, at, p.DV, true);
                    pull_column[j] = product<RANKS>(split<RANKS>(x), delta_own, pull_column[j]);
                }
            }
#pragma unroll
            for (int d = 0; d < TILES; ++d) {
                const int row = 16 * d + column;
                float x[8], y[8];
                floats_of(x, marks + row * p.DV, at, p.DV, row < p.DK);
                floats_of(y, later + row * p.DV, at, p.DV, row < p.DK);
                if (d % 4 == wave) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) dot = fmaf(x[j], y[j], dot);
                }
                const Terms<RANKS> a = split<RANKS>(x), b = split<RANKS>(y);
                dq[d] = product<RANKS>(a, o_own, dq[d]);
                ds[d] = product<RANKS>(a, z_own, ds[d]);
                dk[d] = product<RANKS>(b, delta_own, dk[d]);
            }
        }
        __syncthreads();
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
            dq_all[d] += dq[d];
            dk_all[d] += dk[d];
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
            const float rest = p.vectors[index * 3 * kChunk + kChunk - 1];
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
            const int at = 16 * d + 4 * group;
            store_four<T>(dquery + at, p.DK - at, dq_all[d]);
            store_four<T>(dkey + at, p.DK - at, dk_all[d]);
        }
    }
}

template <typename T, int KS>
void launch_backward(const DeltaArgs& p, hipStream_t stream) {
    launch_chunks<T, KS, true>(p, stream);
    delta_walk_back_kernel<T, KS><<<dim3(head_groups(p.N * p.HV, (p.DV + 63) / 64)), dim3(256), 0, stream>>>(p);
    delta_gradient_kernel<T, KS><<<grid_of(static_cast<int64_t>(p.N) * p.H * p.chunks), dim3(256), 0, stream>>>(p);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_delta_rule_backward_workspace_bytes(const snnf_delta_rule_call* call) {
    if (check_delta("snnf_delta_rule_backward_workspace_bytes", call) != SNNF_OK) return 0;
    return static_cast<size_t>(delta_chunks(call)) * (block_words(3) + 3 * kChunk + (call->key_size + kChunk) * call->value_size) * 4;
}

extern "C" int snnf_delta_rule_backward(const snnf_delta_rule_call* call, const float* marks, const snnf_heads* dout, const float* dstate, const snnf_heads* dquery,
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
    p.marks = const_cast<float*>(marks);
    p.deltas = p.marks + chunks * call->key_size * call->value_size;
    p.vectors = static_cast<float*>(workspace);
    p.blocks = reinterpret_cast<uint32_t*>(p.vectors + chunks * 3 * kChunk);
    p.later = reinterpret_cast<float*>(p.blocks + chunks * block_words(3));
    p.pulls = p.later + chunks * call->key_size * call->value_size;
    hipStream_t hs = as_stream(stream);
    const bool small = call->key_size <= 64;
    if (call->dtype == SNNF_F32) small ? launch_backward<float, 2>(p, hs) : launch_backward<float, 4>(p, hs);
    else if (call->dtype == SNNF_BF16) small ? launch_backward<bf16_t, 2>(p, hs) : launch_backward<bf16_t, 4>(p, hs);
    else small ? launch_backward<f16_t, 2>(p, hs) : launch_backward<f16_t, 4>(p, hs);
    return check_launch("snnf_delta_rule_backward");
}
