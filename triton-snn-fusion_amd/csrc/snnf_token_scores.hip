// Scores of given tokens: log probability, entropy of the row, the most likely alternatives, and the gradient of the first two.
//     M = max x, s = sum exp(x - M), t = sum exp(x - M) (x - M);   logprob = (x_token - M) - log s,   entropy = log s - t / s
//     d x_i = d_logprob (1[i = token] - p_i) - d_entropy p_i (log p_i + entropy)
// One pass over the logits: every thread keeps (M, s, t) of its elements, rescaled when a batch brings a larger maximum, and the workgroup joins
// them in a fixed order. Bound by memory: 8192 x 32000 bf16 97 us (5.4 TB/s) and its gradient, which reads and writes, 184 us (5.7). A few rows are
// bound by latency: 16 x 32000 bf16 5.2 us, with 8 alternatives 7.6.
// Alternatives: the threads' maxima, as 64 or 256 groups, give a value that at least k elements reach (their k-th largest), and only threads
// whose own maximum reaches it look through their elements again, which the caches still hold; a few dozen candidates are ranked by counting.
// Where a mask leaves fewer than k, or many share the bound, those above it are ranked and the rest taken from those at it in order of the index
// (500 x 50021 bf16 with 20 alternatives: 18 us, five elements left 24, with one maximum after the other 250; all of one value 24 and 281).
// Ties go to the lower index: an element's key is its value, in an order of unsigned numbers, above the complement of its index.
#include "snnf_sequence.h"

namespace snnf {
namespace {

constexpr int kMostAlternatives = 64;
constexpr int kCandidates = 1024;       // candidates that are ranked at once
constexpr int kEqual = 512;             // more than these at or above a bound: many may be equal to it
constexpr int kAtOnce = 4;              // elements a thread compares at once in the search for those equal to a bound
constexpr int kBatch = 2;               // vectors a thread works on while as many are on their way
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct ScoreArgs {
    const void* logits;
    int64_t row;                        // elements from one row to the next
    int64_t rows;
    int V, k;
    int splits, span;                   // workgroups to a row, elements of each
    const int64_t* tokens;
    float *logprob, *entropy, *top_logprob;
    int64_t* top_token;
    float2* stats;                      // M, s
    float4* parts;                      // [row][split] M, s, t
    uint64_t* keys;                     // [row][split][k]
    const float2* saved;
    const float *saved_entropy, *d_logprob, *d_entropy;
    void* d_logits;
};

// M, s and t (in powers of two: t = sum e z with e = 2^z) of some elements.
struct Stats {
    float M, s, t;
};
// (x - M) in powers of two, kept where 2^z is 0 and z times it as well: masked elements are minus infinity.
__device__ __forceinline__ float exponent(float x, float M) { return __builtin_elementwise_maximum((x - M) * kLog2e, -200.0f); }
// What is subtracted where nothing but minus infinity has been seen.
__device__ __forceinline__ float center(float M) { return M == -INFINITY ? 0.0f : M; }

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    const float M = fmaxf(a.M, b.M), c = center(M);
    const float za = exponent(a.M, c), zb = exponent(b.M, c);
    const float fa = __builtin_amdgcn_exp2f(za), fb = __builtin_amdgcn_exp2f(zb);
    return {M, a.s * fa + b.s * fb, fa * fmaf(za, a.s, a.t) + fb * fmaf(zb, b.s, b.t)};
}

// All threads' statistics as one, in every thread. A lane reads one wave's share, so that a few exchanges join 16 of them.
template <int BLOCK>
__device__ __forceinline__ Stats join_all(Stats v) {
    constexpr int WAVES = BLOCK / 64;
    __shared__ float largest[WAVES], sums[2][WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, other = lane % WAVES;
    float M = lane_max(v.M);
    if (lane == 0) largest[wave] = M;
    __syncthreads();
    M = lane_max(largest[other], WAVES);
    const float z = exponent(v.M, center(M)), f = __builtin_amdgcn_exp2f(z);
    const float s = lane_sum(v.s * f), t = lane_sum(f * fmaf(z, v.s, v.t));
    if (lane == 0) sums[0][wave] = s, sums[1][wave] = t;
    __syncthreads();
    return {M, lane_sum(sums[0][other], WAVES), lane_sum(sums[1][other], WAVES)};
}

__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t bits = __float_as_uint(x);
    if (x != x) return 0;               // a NaN comes last
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order == 0 ? 0x7fc00000u : (order & 0x80000000u ? order & 0x7fffffffu : ~order)); }
// Bits (an even one) from which on numbers of a type differ: those below are zeros in a 16-bit type's, ones where the order turns them.
template <typename T> inline constexpr int kLowest = sizeof(T) == 4 ? 0 : (dtype_of<T>::value == SNNF_BF16 ? 16 : 12);
// -0 and 0 are the same value.
__device__ __forceinline__ uint64_t key_of(float x, int index) { return static_cast<uint64_t>(order_of(x + 0.0f)) << 32 | static_cast<uint32_t>(~index); }

// Elements `at` to `end` - 1 of a row; minus infinity behind them.
template <typename T>
__device__ __forceinline__ void take(float (&v)[kVec<T>], const Raw<T, kVec<T>>& raw, int left) {
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) v[j] = raw[j];
    if (left < kVec<T>) {
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j) v[j] = j < left ? v[j] : -INFINITY;
    }
}

// The k largest keys among `count` in LDS, in order, to `out`.
template <int BLOCK>
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int count, int k, uint64_t* out) {
    for (int i = threadIdx.x; i < count; i += BLOCK) {
        const uint64_t mine = keys[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) rank += keys[j] > mine ? 1 : 0;
        if (rank < k) out[rank] = mine;
    }
}

// The k largest keys of a workgroup's elements. `most`: the thread's own largest value.
template <typename T, int BLOCK>
__device__ __forceinline__ void alternatives(const T* row, int begin, int end, int k, float most, uint64_t* out) {
    constexpr int VEC = kVec<T>, WAVES = BLOCK / 64;
    __shared__ float maxima[WAVES][64];
    __shared__ uint32_t reached;
    __shared__ int count;
    __shared__ uint64_t candidates[kCandidates];
    __shared__ int counts[kAtOnce][WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    maxima[wave][lane] = most;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    if (wave == 0) {
        // The k-th largest of 64 groups, or of 256 where 64 would be few for k (512 x 32000 bf16 with 64 alternatives 31 us, 102 by 64 groups, since
        // several hundred elements reach the smallest maximum; with 20 the four counts for a bit cost more, 20.2 and 19.8), by its bits: the largest number
        // that k of them reach, two bits at a time with one group to a lane.
        constexpr int kQuarters = 4;
        float group[kQuarters];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) group[w % kQuarters] = w < kQuarters ? maxima[w][lane] : fmaxf(group[w % kQuarters], maxima[w][lane]);
        uint32_t bound = 0;
        if (k <= 32) {
            const uint32_t mine = order_of(fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3])) + 0.0f);
#pragma unroll
            for (int bit = 30; bit >= kLowest<T>; bit -= 2) {
                const int one = __popcll(__ballot(mine >= (bound | 1u << bit))), two = __popcll(__ballot(mine >= (bound | 2u << bit)));
                const int three = __popcll(__ballot(mine >= (bound | 3u << bit)));
                bound |= static_cast<uint32_t>((one >= k) + (two >= k) + (three >= k)) << bit;
            }
        } else {
            uint32_t mine[kQuarters];
#pragma unroll
            for (int q = 0; q < kQuarters; ++q) mine[q] = order_of(group[q] + 0.0f);
#pragma unroll 4
            for (int bit = 31; bit >= kLowest<T>; --bit) {
                const uint32_t higher = bound | 1u << bit;
                int reach = 0;
#pragma unroll
                for (int q = 0; q < kQuarters; ++q) reach += __popcll(__ballot(mine[q] >= higher));
                if (reach >= k) bound = higher;
            }
        }
        if (lane == 0) reached = bound & 0x80000000u ? bound : bound | ((1u << kLowest<T>) - 1);
    }
    __syncthreads();
    const float bound = value_of(reached);
    // A wave looks through the elements of its threads that reach it (or pass it), one thread after the other, a lane to an element.
    const auto collect = [&](int room, auto counts) {
        uint64_t hot = __ballot(counts(most));
        while (hot != 0) {
            const int thread = wave * 64 + __builtin_ctzll(hot);
            hot &= hot - 1;
            for (int first = begin + thread * VEC; first < end; first += 64 * BLOCK) {
                const int at = first + lane / VEC * (BLOCK * VEC) + lane % VEC;
                if (at < end) {
                    const float v = to_float(row[at]);
                    if (counts(v)) {
                        const int to = atomicAdd(&count, 1);
                        if (to < kCandidates) candidates[to] = key_of(v, at);
                    }
                }
            }
            if (hot != 0 && *const_cast<volatile int*>(&count) > room) break;
        }
        __syncthreads();
        return count;
    };
    if (bound > -INFINITY) {
        const int found = collect(kEqual, [&](float v) { return v >= bound; });
        if (found >= k && found <= kEqual) {
            rank_keys<BLOCK>(candidates, found, k, out);
            return;
        }
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
    }
    // A mask leaves fewer than k, or many are equal (masked by a lowest value, say): those above the bound, then the first of those at it.
    const int above = collect(kCandidates, [&](float v) { return v > bound; });
    if (above <= kCandidates) {
        rank_keys<BLOCK>(candidates, above, k, out);
        int filled = above;
        for (int from = begin; from < end && filled < k; from += kAtOnce * BLOCK) {
            uint64_t same[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int at = from + u * BLOCK + static_cast<int>(threadIdx.x);
                same[u] = __ballot(at < end && to_float(row[at < end ? at : begin]) == bound);
                if (lane == 0) counts[u][wave] = __popcll(same[u]);
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                for (int w = 0; w < WAVES; ++w) {
                    const int to = filled + __popcll(same[u] & ((1ull << lane) - 1));
                    if (w == wave && (same[u] >> lane & 1) && to < k) out[to] = key_of(bound, from + u * BLOCK + static_cast<int>(threadIdx.x));
                    filled += counts[u][w];
                }
            }
            __syncthreads();
        }
        if (filled >= k) return;
    }
    // Anything else (more than fit above the bound, NaN among the few that count): the largest key below the last, k times.
    uint64_t last = ~0ull;
    for (int i = 0; i < k; ++i) {
        uint64_t best = 0;
        for (int at = begin + static_cast<int>(threadIdx.x) * VEC; at < end; at += BLOCK * VEC) {
            Raw<T, VEC> raw;
            float v[VEC];
            raw.load(row, at, end - at);
            take<T>(v, raw, end - at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint64_t key = key_of(v[j], at + j);
                if (at + j < end && key < last && key > best) best = key;
            }
        }
#pragma unroll
        for (int mask = 32; mask > 0; mask >>= 1) {
            const uint64_t other = static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(best >> 32), mask, 64)) << 32 | __shfl_xor(static_cast<uint32_t>(best), mask, 64);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) candidates[wave] = best;
        __syncthreads();
        for (int w = 0; w < WAVES; ++w) best = candidates[w] > best ? candidates[w] : best;
        if (threadIdx.x == 0) out[i] = best;
        last = best;
    }
}

// The given token's logit, which the first thread sends for before the row is read.
struct Given {
    bool there;
    float logit;
};
template <typename T>
__device__ __forceinline__ Given given_token(const ScoreArgs& p, int64_t r) {
    const int64_t token = p.tokens == nullptr ? -1 : p.tokens[r];
    const bool there = token >= 0 && token < p.V;
    return {there, there ? to_float(static_cast<const T*>(p.logits)[r * p.row + token]) : 0.0f};
}

// Scores of a row from its statistics and its k keys.
__device__ __forceinline__ void finish(const ScoreArgs& p, int64_t r, const Stats& v, const Given& given, const uint64_t* keys) {
    const bool none = v.s == 0.0f;              // nothing is left of the row
    const float log_s = none ? 0.0f : logf(v.s);
    if (threadIdx.x == 0) {
        p.logprob[r] = !given.there ? 0.0f : (none ? -INFINITY : (given.logit - v.M) - log_s);
        p.entropy[r] = none ? 0.0f : log_s - kLn2 * (v.t / v.s);
        if (p.stats != nullptr) p.stats[r] = make_float2(v.M, v.s);
    }
    if (static_cast<int>(threadIdx.x) < p.k) {
        const uint64_t key = keys[threadIdx.x];
        p.top_token[r * p.k + threadIdx.x] = static_cast<int64_t>(~static_cast<uint32_t>(key));
        p.top_logprob[r * p.k + threadIdx.x] = none ? -INFINITY : (value_of(static_cast<uint32_t>(key >> 32)) - v.M) - log_s;
    }
}

template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK, 8) void token_scores_kernel(ScoreArgs p) {
    constexpr int VEC = kVec<T>;
    __shared__ uint64_t top[kMostAlternatives];
    const uint32_t group = group_index();
    if (group >= p.rows * p.splits) return;
    const int64_t r = group / p.splits;
    const int split = static_cast<int>(group - r * p.splits), begin = split * p.span, end = begin + p.span < p.V ? begin + p.span : p.V;
    const T* row = static_cast<const T*>(p.logits) + r * p.row;
    Given given{false, 0.0f};
    if (p.splits == 1 && threadIdx.x == 0) given = given_token<T>(p, r);
    Stats mine{-INFINITY, 0.0f, 0.0f};
    Raw<T, VEC> now[kBatch], next[kBatch];
    const auto fetch = [&](int at) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) next[u].load(row, at + u * BLOCK * VEC, end - at - u * BLOCK * VEC);
    };
    int at = begin + static_cast<int>(threadIdx.x) * VEC;
    fetch(at);
    for (; at < end; at += kBatch * BLOCK * VEC) {
        float v[kBatch][VEC];
        float most = mine.M;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) now[u] = next[u];
        if (at + kBatch * BLOCK * VEC < end) fetch(at + kBatch * BLOCK * VEC);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) take<T>(v[u], now[u], end - at - u * BLOCK * VEC);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) most = fmaxf(most, v[u][j]);
        const float c = center(most), z = exponent(mine.M, c), f = __builtin_amdgcn_exp2f(z);
        mine.t = f * fmaf(z, mine.s, mine.t);
        mine.s *= f;
        mine.M = most;
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float zj = exponent(v[u][j], c), e = __builtin_amdgcn_exp2f(zj);
                mine.s += e;
                mine.t = fmaf(e, zj, mine.t);
            }
    }
    const Stats all = join_all<BLOCK>(mine);
    if (p.k > 0) {
        alternatives<T, BLOCK>(row, begin, end, p.k, mine.M, top);
        __syncthreads();
    }
    if (p.splits == 1) {
        finish(p, r, all, given, top);
        return;
    }
    if (threadIdx.x == 0) p.parts[group] = make_float4(all.M, all.s, all.t, 0.0f);
    if (static_cast<int>(threadIdx.x) < p.k) p.keys[static_cast<int64_t>(group) * p.k + threadIdx.x] = top[threadIdx.x];
}

// Joins the splits of a row: one workgroup of 256 threads.
constexpr int kMostSplits = 32;
template <typename T>
__global__ __launch_bounds__(256) void join_scores_kernel(ScoreArgs p) {
    __shared__ uint64_t candidates[kMostSplits * kMostAlternatives], top[kMostAlternatives];
    __shared__ int count;
    const int64_t r = group_index();
    if (r >= p.rows) return;
    Given given{false, 0.0f};
    if (threadIdx.x == 0) given = given_token<T>(p, r);
    const float4 first = p.parts[r * p.splits];
    Stats all{first.x, first.y, first.z};
    for (int i = 1; i < p.splits; ++i) {
        const float4 part = p.parts[r * p.splits + i];
        all = join(all, Stats{part.x, part.y, part.z});
    }
    if (p.k > 0) {
        // Whatever is smaller than some split's k-th key has k larger ones.
        const uint64_t* keys = p.keys + r * p.splits * p.k;
        uint64_t bound = 0;
        for (int i = 0; i < p.splits; ++i) bound = keys[i * p.k + p.k - 1] > bound ? keys[i * p.k + p.k - 1] : bound;
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < p.splits * p.k; i += 256)
            if (keys[i] >= bound) candidates[atomicAdd(&count, 1)] = keys[i];
        __syncthreads();
        rank_keys<256>(candidates, count, p.k, top);
        __syncthreads();
    }
    finish(p, r, all, given, top);
}

template <typename T>
__global__ __launch_bounds__(256) void token_scores_backward_kernel(ScoreArgs p) {
    constexpr int VEC = kVec<T>;
    const uint32_t group = group_index();
    if (group >= p.rows * p.splits) return;
    const int64_t r = group / p.splits;
    const int begin = static_cast<int>(group - r * p.splits) * p.span, end = begin + p.span < p.V ? begin + p.span : p.V;
    const T* row = static_cast<const T*>(p.logits) + r * p.row;
    T* out = static_cast<T*>(p.d_logits) + r * p.V;
    const float2 stats = p.saved[r];
    const int64_t token = p.tokens == nullptr ? -1 : p.tokens[r];
    const bool given = token >= 0 && token < p.V && p.d_logprob != nullptr;
    const float g = given ? p.d_logprob[r] : 0.0f, h = p.d_entropy != nullptr ? p.d_entropy[r] : 0.0f;
    const bool none = stats.y == 0.0f;
    const float c = center(stats.x), inverse = none ? 0.0f : 1.0f / stats.y;
    // -p (g + h (log p + entropy)) with log p = ln2 z - log s
    const float constant = none ? 0.0f : fmaf(h, p.saved_entropy[r] - logf(stats.y), g), slope = h * kLn2;
    for (int at = begin + static_cast<int>(threadIdx.x) * VEC; at < end; at += 256 * VEC) {
        Raw<T, VEC> raw;
        float v[VEC];
        raw.load(row, at, end - at);
        take<T>(v, raw, end - at);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float z = exponent(v[j], c), probability = __builtin_amdgcn_exp2f(z) * inverse;
            v[j] = -probability * fmaf(slope, z, constant);
            if (given && !none && at + j == token) v[j] += g;
        }
#pragma unroll
        for (int j = 0; j < VEC; j += 2) raw.put(j, v[j], v[j + 1]);
        raw.store(out, at, end - at);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------------------------
struct ScoreShape {
    int block, splits, span;
};

// A workgroup to a row: 256 threads where there are rows enough to fill the chip or few elements (8192 x 32000 bf16 97 us, with 1024 threads 117;
// 4096 x 6488 with 20 alternatives 28 and 60; 64 x 1000 float32 with 5 5.8 and 6.3), else 1024 (16 x 32000 bf16 with 8 alternatives 7.6 us, with 256
// threads 10.3; 500 x 50021 with 20 17.9 and 28.3). Few long rows are split over workgroups (1 x 200000 bf16 with 8 alternatives 14 us, in one
// piece 20; 4 x 500000 23 and 45; about even at 128 x 100000), pieces of 16384 elements at least: a second launch joins them.
ScoreShape score_shape(int64_t rows, int V) {
    const int64_t units = compute_units();
    ScoreShape s{rows >= units * 2 || V <= 8192 ? 256 : 1024, 1, V};
    if (rows < units && V > 64 * 1024) {
        int64_t splits = units / rows;
        const int64_t useful = V / (16 * 1024);
        splits = splits < useful ? splits : useful;
        splits = splits < kMostSplits ? splits : kMostSplits;
        if (splits > 1) {
            s.span = static_cast<int>(((V + splits - 1) / splits + 1023) / 1024 * 1024);
            s.splits = (V + s.span - 1) / s.span;
        }
    }
    return s;
}

int check_scores(const char* name, int64_t rows, int V, int dtype, int k) {
    if (rows < 0 || V < 1 || k < 0) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: rows=%lld V=%d top_k=%d", name, (long long)rows, V, k);
    if (V > (1 << 30)) return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: rows of at most 2^30 elements", name);
    if (k > V || k > kMostAlternatives)
        return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_top_k: at most %d alternatives and no more than elements, got %d of %d", name, kMostAlternatives, k, V);
    if (!valid_dtype(dtype)) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", name, dtype);
    return SNNF_OK;
}

template <typename T>
void launch_scores(const ScoreArgs& p, const ScoreShape& s, hipStream_t stream) {
    const dim3 grid = grid_of(p.rows * s.splits);
    if (s.block == 256) token_scores_kernel<T, 256><<<grid, dim3(256), 0, stream>>>(p);
    else token_scores_kernel<T, 1024><<<grid, dim3(1024), 0, stream>>>(p);
    if (s.splits > 1) join_scores_kernel<T><<<grid_of(p.rows), dim3(256), 0, stream>>>(p);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_token_scores_workspace_bytes(int64_t rows, int V, int top_k) {
    if (rows < 1 || V < 1 || top_k < 0) return 0;
    const ScoreShape s = score_shape(rows, V);
    return s.splits > 1 ? static_cast<size_t>(rows) * s.splits * (sizeof(float4) + sizeof(uint64_t) * top_k) : 0;
}

extern "C" int snnf_token_scores(const void* logits, int64_t row, int64_t rows, int V, int dtype, const int64_t* tokens, int top_k, float* logprob,
                                 float* entropy, float* top_logprob, int64_t* top_token, float* stats, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    const int rc = check_scores("snnf_token_scores", rows, V, dtype, top_k);
    if (rc != SNNF_OK) return rc;
    if (rows == 0) return SNNF_OK;
    if (logits == nullptr || logprob == nullptr || entropy == nullptr || (top_k > 0 && (top_logprob == nullptr || top_token == nullptr)))
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_token_scores: logits, logprob, entropy and what alternatives are written to must be non-null");
    const ScoreShape s = score_shape(rows, V);
    if (rows * s.splits > 0x7fffffffLL) return fail(SNNF_ERR_UNSUPPORTED, "snnf_token_scores: unsupported_shape: %lld rows", (long long)rows);
    ScoreArgs p = {};
    if (s.splits > 1) {
        const size_t need = snnf_token_scores_workspace_bytes(rows, V, top_k);
        if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
            return fail(SNNF_ERR_WORKSPACE, "snnf_token_scores: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
        p.parts = static_cast<float4*>(workspace);
        p.keys = reinterpret_cast<uint64_t*>(p.parts + rows * s.splits);
    }
    p.logits = logits, p.row = row, p.rows = rows;
    p.V = V, p.k = top_k;
    p.splits = s.splits, p.span = s.span;
    p.tokens = tokens;
    p.logprob = logprob, p.entropy = entropy, p.top_logprob = top_logprob, p.top_token = top_token;
    p.stats = reinterpret_cast<float2*>(stats);
    hipStream_t hs = as_stream(stream);
    if (dtype == SNNF_F32) launch_scores<float>(p, s, hs);
    else if (dtype == SNNF_BF16) launch_scores<bf16_t>(p, s, hs);
    else launch_scores<f16_t>(p, s, hs);
    return check_launch("snnf_token_scores");
}

extern "C" int snnf_token_scores_backward(const void* logits, int64_t row, int64_t rows, int V, int dtype, const int64_t* tokens, const float* stats,
                                          const float* entropy, const float* d_logprob, const float* d_entropy, void* d_logits, void* stream) {
    const int rc = check_scores("snnf_token_scores_backward", rows, V, dtype, 0);
    if (rc != SNNF_OK) return rc;
    if (rows == 0) return SNNF_OK;
    if (logits == nullptr || stats == nullptr || entropy == nullptr || d_logits == nullptr)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_token_scores_backward: logits, stats, entropy and d_logits must be non-null");
    ScoreArgs p = {};
    p.logits = logits, p.row = row, p.rows = rows;
    p.V = V;
    p.span = 8192;
    p.splits = (V + p.span - 1) / p.span;
    if (rows * p.splits > 0x7fffffffLL) return fail(SNNF_ERR_UNSUPPORTED, "snnf_token_scores_backward: unsupported_shape: %lld rows", (long long)rows);
    p.tokens = tokens;
    p.saved = reinterpret_cast<const float2*>(stats);
    p.saved_entropy = entropy;
    p.d_logprob = d_logprob, p.d_entropy = d_entropy;
    p.d_logits = d_logits;
    const dim3 grid = grid_of(rows * p.splits), block(256);
    hipStream_t hs = as_stream(stream);
    if (dtype == SNNF_F32) token_scores_backward_kernel<float><<<grid, block, 0, hs>>>(p);
    else if (dtype == SNNF_BF16) token_scores_backward_kernel<bf16_t><<<grid, block, 0, hs>>>(p);
    else token_scores_backward_kernel<f16_t><<<grid, block, 0, hs>>>(p);
    return check_launch("snnf_token_scores_backward");
}
