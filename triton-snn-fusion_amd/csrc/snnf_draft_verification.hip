// Verification of drafted tokens. With p = softmax(logits / temperature) of the target at a place and q that of the draft (1 at the drafted token where it has no
// distribution), token x is accepted while u q(x) < p(x); the place behind the accepted ones gets argmax_i r_i / e_i over exponential noise e, which draws i with
// probability r_i / sum r: r = p behind all drafts, max(p - q, 0) where one was turned down. So every token is distributed as p. The argmax is taken as it is written, whatever the noise: an
// entry of r = 0 has 0 and is the largest where no entry has noise above 0.
// Two launches: (r, s) = an r near the largest x / temperature and sum exp(x / temperature - r) of every row, then the decisions and one more pass over the row that is drawn from. Bound by
// memory; few rows are split over workgroups. 256 requests of 4 drafts x 128000 bfloat16 with both distributions take 167 us, of them 114 the first launch: 590 MB at 5.2 TB/s, next to what 295
// million exponents take of the vector units; one request of 4 x 32000 takes 12.9, the second launch's chain of statistics, drafted logits, verdicts, row and join.
// A decision is that of float64 on the given numbers: float32 gives each number with a bound of its error (`sum_doubt`, `share_doubt`), and where two cannot be told apart the workgroup goes
// over the rows again in float64. That takes several times as long as the rest (765 us in place of 164 at 256 x 4 x 128000, two of 150 calls on random numbers), so that the bounds matter. Exponents are powers of two, x * slope - r in one rounding; r is a whole number, so that
// sums for different r are brought together exactly; sums are compensated in a thread and float64 from there on.
#include "snnf_sequence.h"

namespace snnf {
namespace {

constexpr int kMostDrafts = 64;
constexpr int kMostSplits = 64;

struct VerifyArgs {
    const void *logits, *draft_logits;
    int64_t logits_row, logits_step, draft_row, draft_step, noise_row;      // row: of a request
    const int64_t* drafts;
    const float *uniforms, *noise, *temperatures;
    const int32_t* lengths;
    float temperature;
    int N, K, V, rows;                  // rows of a request: K + 1 of the target, then the draft's
    int splits, span;                   // of a row in the first launch
    int draw_splits, draw_span;         // and in the second
    float2* stats;                      // [request][row][split]: r, s
    uint64_t* largest;                  // [request][row][split]: key of the largest logit
    uint64_t* parts;                    // [request][split]: the two largest upper bounds; the largest lower bound, index; the lowest index of those that are 0
    uint32_t* arrived;                  // [request]
    int64_t* tokens;
    int32_t* accepted;
};

__device__ __forceinline__ float temperature_of(const VerifyArgs& p, int n) { return p.temperatures == nullptr ? p.temperature : p.temperatures[n]; }
__device__ __forceinline__ int drafts_of(const VerifyArgs& p, int n) {
    if (p.lengths == nullptr) return p.K;
    const int length = p.lengths[n];
    return length < 0 ? 0 : (length < p.K ? length : p.K);
}
template <typename T>
__device__ __forceinline__ const T* row_of(const VerifyArgs& p, int n, int row) {
    return row <= p.K ? static_cast<const T*>(p.logits) + n * p.logits_row + row * p.logits_step
                      : static_cast<const T*>(p.draft_logits) + n * p.draft_row + (row - p.K - 1) * p.draft_step;
}

// A key orders by value, equal ones by the lower index; 0: nothing that could be drawn (minus infinity and NaN).
__device__ __forceinline__ uint64_t key_of(float x, int index) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t bits = __float_as_uint(x + 0.0f), order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t lane_largest(uint64_t v) {
#pragma unroll
    for (int mask = 32; mask > 0; mask >>= 1)
        v = larger(v, static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(v >> 32), mask, 64)) << 32 | __shfl_xor(static_cast<uint32_t>(v), mask, 64));
    return v;
}

// Elements from `at` on, minus infinity behind the row's end.
template <typename T>
__device__ __forceinline__ void take(float (&v)[kVec<T>], const Raw<T, kVec<T>>& raw, int left) {
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) v[j] = left >= kVec<T> || j < left ? raw[j] : -INFINITY;
}
template <int VEC>
__device__ __forceinline__ float sum_of(const float (&v)[VEC]) {        // in pairs: a thread adds few of these
    if constexpr (VEC == 8) return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    else return (v[0] + v[1]) + (v[2] + v[3]);
}

// Temperatures whose slope and what it makes of logits float32 holds; those beyond are worked out in float64, with statistics of the nearest of these.
constexpr float kColdest = 1e-30f, kHottest = 1e30f;
__device__ __forceinline__ bool extreme(float temperature) { return temperature < kColdest || temperature > kHottest; }

// 1 / temperature in powers of two, as the sum of two numbers.
struct Slope {
    float high, low;
};
__device__ __forceinline__ Slope slope_of(float temperature) {
    const double slope = 1.4426950408889634074 / fminf(fmaxf(temperature, kColdest), kHottest);
    const float high = static_cast<float>(slope);
    return {high, static_cast<float>(slope - high)};
}
// 2^(x slope - r), with c = r / slope.high: what leaving out slope.low would change of it but not of the others it is compared with is put back. Off by `share_doubt`.
__device__ __forceinline__ float exponent_of(float x, float r, const Slope& slope) { return fmaf(x, slope.high, -r); }
__device__ __forceinline__ float share_of(float x, float r, float c, const Slope& slope) {
    constexpr float kLn2 = 0.69314718055994530942f;
    const float e = __builtin_amdgcn_exp2f(exponent_of(x, r, slope));
    return e == 0.0f ? 0.0f : fmaf(e, (x - c) * slope.low * kLn2, e);
}

// Statistics of several parts brought together: s of each times a power of two. r is infinite where the largest x * slope is beyond kLargest in magnitude; s is 0 then where all is masked, above 0
// where it is not, and in any case NaN where a number is NaN or infinite. Beyond kLargest c is too coarse, too; such rows are worked out in float64.
constexpr float kLargest = 4194304.0f;
__device__ __forceinline__ bool coarse(float r) { return !(fabsf(r) <= kLargest - 1024.0f); }      // or so near that parts of the row may be beyond and count
template <typename F>
__device__ __forceinline__ F brought(F s, float from, float to) {
    return from == to ? s : static_cast<F>(ldexp(s, static_cast<int>(fmaxf(from - to, -1000.0f))));
}
__device__ __forceinline__ bool something(const float2& stats) { return stats.y > 0.0f && stats.y < INFINITY; }
template <int MASK>
__device__ __forceinline__ double across(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t low = __float_as_uint(snnf::across<MASK>(__uint_as_float(static_cast<uint32_t>(bits)))), high = __float_as_uint(snnf::across<MASK>(__uint_as_float(static_cast<uint32_t>(bits >> 32))));
    return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}
__device__ __forceinline__ double lane_sum(double v) {
    v += across<1>(v);
    v += across<2>(v);
    v += across<4>(v);
    v += across<8>(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void verify_rows_kernel(VerifyArgs p) {
    constexpr int VEC = kVec<T>, WAVES = BLOCK / 64, BATCH = 2;
    __shared__ float maxima[WAVES];
    __shared__ double sums[WAVES];
    __shared__ uint64_t keys[WAVES];
    const uint32_t group = group_index();
    const int split = group % p.splits, place = group / p.splits, row = place % p.rows, n = place / p.rows;
    if (n >= p.N) return;
    if (row == 0 && split == 0 && threadIdx.x == 0) p.arrived[n] = 0;
    const int length = drafts_of(p, n);
    const float temperature = temperature_of(p, n);
    const bool greedy = !(temperature > 0.0f);
    if (row <= p.K ? row > length : greedy || row - p.K - 1 >= length) return;
    const T* x = row_of<T>(p, n, row);
    const int begin = split * p.span, end = begin + p.span < p.V ? begin + p.span : p.V, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Raw<T, VEC> now[BATCH], next[BATCH];
    const auto fetch = [&](int at) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u) next[u].load(x, at + u * BLOCK * VEC, end - at - u * BLOCK * VEC);
    };
    int at = begin + static_cast<int>(threadIdx.x) * VEC;
    fetch(at);
    if (greedy) {
        uint64_t best = 0;
        for (; at < end; at += BATCH * BLOCK * VEC) {
#pragma unroll
            for (int u = 0; u < BATCH; ++u) now[u] = next[u];
            if (at + BATCH * BLOCK * VEC < end) fetch(at + BATCH * BLOCK * VEC);
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                float v[VEC];
                take<T>(v, now[u], end - at - u * BLOCK * VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j) best = larger(best, key_of(v[j], at + u * BLOCK * VEC + j));
            }
        }
        best = lane_largest(best);
        if (lane == 0) keys[wave] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < WAVES; ++w) best = larger(best, keys[w]);
            p.largest[static_cast<int64_t>(place) * p.splits + split] = best;
        }
        return;
    }
    const Slope slope = slope_of(temperature);
    // r: rises as soon as an element would have more than 2 and stays a whole number, so that s is multiplied by powers of two.
    const int first = at;
    float M = -INFINITY, r = -INFINITY, s = 0.0f, lost = 0.0f;
    for (; at < end; at += BATCH * BLOCK * VEC) {
        float v[BATCH][VEC];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) now[u] = next[u];
        if (at + BATCH * BLOCK * VEC < end) fetch(at + BATCH * BLOCK * VEC);
#pragma unroll
        for (int u = 0; u < BATCH; ++u) take<T>(v[u], now[u], end - at - u * BLOCK * VEC);
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) M = fmaxf(M, v[u][j]);
        const float top = M * slope.high;
        if (!(top - r <= 1.0f) && fabsf(top) < kLargest) {
            const float higher = __builtin_rintf(top);
            s = brought(s, r, higher), lost = brought(lost, r, higher);
            r = higher;
        }
        const float subtracted = r == -INFINITY ? 0.0f : r;
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[u][j] = __builtin_amdgcn_exp2f(exponent_of(v[u][j], subtracted, slope));
            const float more = sum_of<VEC>(v[u]) - lost, now_s = s + more;
            lost = (now_s - s) - more;
            s = now_s;
        }
    }
    if (M > -INFINITY && !(fabsf(M * slope.high) < kLargest)) {
        bool broken = M == INFINITY;
        for (at = first; at < end; at += BATCH * BLOCK * VEC) {
            fetch(at);
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                float v[VEC];
                take<T>(v, next[u], end - at - u * BLOCK * VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j) broken = broken || v[j] != v[j];
            }
        }
        r = M > 0.0f ? INFINITY : -INFINITY, s = broken ? __builtin_nanf("") : 1.0f, lost = 0.0f;
    }
    const float most = lane_max(r);
    if (lane == 0) maxima[wave] = most;
    __syncthreads();
    const float all = lane_max(maxima[lane % WAVES], WAVES < 4 ? 4 : WAVES);
    const double sum = lane_sum(brought(static_cast<double>(s) - static_cast<double>(lost), r, all));
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double both = sums[0];
        for (int w = 1; w < WAVES; ++w) both += sums[w];
        p.stats[static_cast<int64_t>(place) * p.splits + split] = make_float2(all, static_cast<float>(both));
    }
}

// Bounds of relative errors, in units u = 2^-24. A share: ln 2 for each power of two of the exponent, which is rounded once, 2 for the power itself (1.43 measured over all exponents from -125
// to 126), 8 for the correction, three products, a quotient, a difference and the reciprocal of the noise. A sum: in the worst case all exponents are rounded the same way, as those of
// equal logits are, and slope.low is missing from all: ln 2 (1 + |slope.low / slope.high| / u) for each power of two. Weighted by the shares those are the row's entropy at most, log2 V, and 2
// for elements above r and r itself; then 2 for the powers, 3 for adding 8 of them, 3 for the compensated sum, 2 where it becomes float32.
__device__ __forceinline__ float share_doubt(float exponent) { return (10.0f + 0.7f * fminf(fabsf(exponent), 1000.0f)) * 0x1p-24f; }
__device__ __forceinline__ float sum_doubt(const Slope& slope, int V) {
    const float bits = static_cast<float>(32 - __builtin_clz(V));
    return (10.0f + 0.7f * (bits + 2.0f) * (1.0f + fabsf(slope.low / slope.high) * 0x1p24f)) * 0x1p-24f;
}

// ------------------------------------------------------------------------------------------------------------------
// In float64, by a workgroup
// ------------------------------------------------------------------------------------------------------------------
template <int BLOCK, typename V, typename Op>
__device__ __forceinline__ V over_block(V v, Op op) {
    __shared__ V shared[BLOCK];
    __syncthreads();
    shared[threadIdx.x] = v;
    __syncthreads();
    for (int half = BLOCK / 2; half > 0; half /= 2) {
        if (static_cast<int>(threadIdx.x) < half) shared[threadIdx.x] = op(shared[threadIdx.x], shared[threadIdx.x + half]);
        __syncthreads();
    }
    return shared[0];
}
__device__ __forceinline__ double exact_share(float x, float M, double temperature) {      // a masked entry has none at an infinite temperature either
    return x == -INFINITY ? 0.0 : exp((static_cast<double>(x) - M) / temperature);
}
template <typename T, int BLOCK>
__device__ float exact_top(const T* x, int V) {
    float M = -INFINITY;
    for (int i = threadIdx.x; i < V; i += BLOCK) M = fmaxf(M, to_float(x[i]));
    return over_block<BLOCK>(M, [](float a, float b) { return fmaxf(a, b); });
}
template <typename T, int BLOCK>
__device__ double exact_sum(const T* x, int V, float M, double temperature) {
    double s = 0.0;
    for (int i = threadIdx.x; i < V; i += BLOCK) s += exact_share(to_float(x[i]), M, temperature);
    return over_block<BLOCK>(s, [](double a, double b) { return a + b; });
}
struct Candidate {
    double value;
    int index;
};
template <typename T, int BLOCK>
__device__ int exact_draw(const T* x, const T* y, int passed, int V, double temperature, const float* noise) {
    const float M = exact_top<T, BLOCK>(x, V), M2 = y != nullptr ? exact_top<T, BLOCK>(y, V) : 0.0f;
    const double s = exact_sum<T, BLOCK>(x, V, M, temperature), s2 = y != nullptr ? exact_sum<T, BLOCK>(y, V, M2, temperature) : 1.0;
    for (int round = 0; round < 2; ++round) {       // where nothing is left beside the draft's share: from p
        Candidate best{0.0, -1};
        int some = 0;
        for (int i = threadIdx.x; i < V; i += BLOCK) {
            double r = exact_share(to_float(x[i]), M, temperature) / s;
            if (round == 0) r -= y != nullptr ? exact_share(to_float(y[i]), M2, temperature) / s2 : (i == passed ? 1.0 : 0.0);
            const double v = r > 0.0 ? r / static_cast<double>(noise[i]) : 0.0;
            some |= r > 0.0;
            if (best.index < 0 ? v == v : v > best.value) best = Candidate{v, i};
        }
        if (!__syncthreads_or(some)) continue;
        best = over_block<BLOCK>(best, [](const Candidate& a, const Candidate& b) {
            return b.index >= 0 && (a.index < 0 || b.value > a.value || (b.value == a.value && b.index < a.index)) ? b : a;
        });
        return best.index >= 0 ? best.index : -100;
    }
    return -100;
}

// ------------------------------------------------------------------------------------------------------------------
// Decisions and the draw
// ------------------------------------------------------------------------------------------------------------------
// Of the values r / e that are not known to be 0: the two largest upper bounds; the largest lower bound; index of the first, the lowest of equal ones. The lowest index of those that are.
constexpr int kNone = 0x7fffffff;
struct Race {
    float first, second, lower;
    int index, zero;
};
__device__ __forceinline__ Race nobody() { return {-INFINITY, -INFINITY, -INFINITY, kNone, kNone}; }
__device__ __forceinline__ Race join(const Race& a, const Race& b) {
    const bool other = b.first > a.first || (b.first == a.first && b.index < a.index);
    const Race& w = other ? b : a;
    return {w.first, fmaxf(w.second, other ? a.first : b.first), fmaxf(a.lower, b.lower), w.index, a.zero < b.zero ? a.zero : b.zero};
}
__device__ __forceinline__ Race lane_race(Race v) {
#pragma unroll
    for (int mask = 32; mask > 0; mask >>= 1)
        v = join(v, Race{__shfl_xor(v.first, mask, 64), __shfl_xor(v.second, mask, 64), __shfl_xor(v.lower, mask, 64), __shfl_xor(v.index, mask, 64), v.zero});
    if (__ballot(v.zero != kNone) != 0) {
#pragma unroll
        for (int mask = 32; mask > 0; mask >>= 1) {
            const int zero = __shfl_xor(v.zero, mask, 64);
            v.zero = zero < v.zero ? zero : v.zero;
        }
    }
    return v;
}
// The index of the largest value, the lowest of equal ones; -1: the bounds do not tell. An upper bound of 0 beside noise below 0 is one of a value that may be 0.
__device__ __forceinline__ int winner(const Race& v) {
    const bool zeros = v.zero != kNone;
    if (v.first > 0.0f) return v.second < v.lower && (v.lower > 0.0f || !zeros) ? v.index : -1;
    if (zeros) return v.first < 0.0f || v.index > v.zero ? v.zero : -1;
    return v.second < v.lower ? v.index : -1;
}
// Noise of a size for which bounds neither overflow nor vanish. Any other leaves the draw to float64.
constexpr float kLeastNoise = 1e-24f, kMostNoise = 1e12f;

__device__ __forceinline__ uint64_t two_words(float a, float b) { return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a); }

template <typename T>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs p) {
    constexpr int BLOCK = 256, VEC = kVec<T>;
    enum { kTaken, kRefused, kDoubtful };
    __shared__ float2 stats[2 * kMostDrafts + 1];
    __shared__ int verdicts[kMostDrafts];
    __shared__ uint64_t largest[kMostDrafts + 1];
    __shared__ Race races[4];
    __shared__ int last;
    const uint32_t group = group_index();
    const int split = group % p.draw_splits, n = group / p.draw_splits;
    if (n >= p.N) return;
    const int length = drafts_of(p, n), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float temperature = temperature_of(p, n);
    const bool greedy = !(temperature > 0.0f), beyond = extreme(temperature);
    const Slope slope = slope_of(greedy ? 1.0f : temperature);
    const float per_sum = sum_doubt(slope, p.V);
    // What the verdicts need of the drafts, sent for before the statistics.
    int64_t drafted_here = -1;
    float logit = 0.0f, theirs_logit = 0.0f, uniform = 0.0f;
    if (static_cast<int>(threadIdx.x) < length) {
        const int j = threadIdx.x;
        drafted_here = p.drafts[static_cast<int64_t>(n) * p.K + j];
        if (drafted_here >= 0 && drafted_here < p.V && !greedy) {
            uniform = p.uniforms[static_cast<int64_t>(n) * p.K + j];
            logit = to_float(row_of<T>(p, n, j)[drafted_here]);
            if (p.draft_logits != nullptr) theirs_logit = to_float(row_of<T>(p, n, p.K + 1 + j)[drafted_here]);
        }
    }
    // Statistics of the request's rows, a thread to a row.
    for (int row = threadIdx.x; row < p.rows; row += BLOCK) {
        if (row <= p.K ? row > length : greedy || row - p.K - 1 >= length) continue;
        const int64_t at = (static_cast<int64_t>(n) * p.rows + row) * p.splits;
        if (greedy) {
            uint64_t best = p.largest[at];
#pragma unroll 4
            for (int i = 1; i < p.splits; ++i) best = larger(best, p.largest[at + i]);
            largest[row] = best;
        } else {
            float r = -INFINITY;
            double s = 0.0;
#pragma unroll 4
            for (int i = 0; i < p.splits; ++i) r = fmaxf(r, p.stats[at + i].x);
#pragma unroll 4
            for (int i = 0; i < p.splits; ++i) s += brought(static_cast<double>(p.stats[at + i].y), p.stats[at + i].x, r);
            stats[row] = make_float2(r, static_cast<float>(s));
        }
    }
    __syncthreads();
    // The verdict on each draft.
    if (static_cast<int>(threadIdx.x) < length) {
        const int j = threadIdx.x;
        int verdict = kRefused;
        if (drafted_here >= 0 && drafted_here < p.V) {
            if (greedy) {
                verdict = largest[j] != 0 && static_cast<int64_t>(~static_cast<uint32_t>(largest[j])) == drafted_here ? kTaken : kRefused;
            } else {
                const float2 a = stats[j], b = p.draft_logits != nullptr ? stats[p.K + 1 + j] : make_float2(0.0f, 1.0f);
                const float mine = share_of(logit, a.x, a.x / slope.high, slope) / a.y;
                float theirs = uniform, unsure = per_sum + share_doubt(exponent_of(logit, a.x, slope));
                if (p.draft_logits != nullptr) {
                    theirs *= share_of(theirs_logit, b.x, b.x / slope.high, slope) / b.y;
                    unsure += per_sum + share_doubt(exponent_of(theirs_logit, b.x, slope));
                }
                verdict = something(a) && something(b) && theirs < mine ? kTaken : kRefused;
                // a bound, or numbers that vanish in float32
                if (something(a) && something(b) && (beyond || coarse(a.x) || coarse(b.x) || !(fabsf(theirs - mine) > unsure * (theirs + mine)) || fmaxf(theirs, mine) < 1e-30f))
                    verdict = uniform == uniform ? kDoubtful : kRefused;
            }
        }
        verdicts[j] = verdict;
    }
    __syncthreads();
    int taken = 0;
    for (; taken < length; ++taken) {
        int verdict = verdicts[taken];
        if (verdict == kDoubtful) {
            const int64_t x = p.drafts[static_cast<int64_t>(n) * p.K + taken];
            const T *a = row_of<T>(p, n, taken), *b = p.draft_logits == nullptr ? nullptr : row_of<T>(p, n, p.K + 1 + taken);
            const float M = exact_top<T, BLOCK>(a, p.V);
            const double mine = exact_share(to_float(a[x]), M, temperature) / exact_sum<T, BLOCK>(a, p.V, M, temperature);
            double theirs = p.uniforms[static_cast<int64_t>(n) * p.K + taken];
            if (b != nullptr) {
                const float M2 = exact_top<T, BLOCK>(b, p.V);
                theirs *= exact_share(to_float(b[x]), M2, temperature) / exact_sum<T, BLOCK>(b, p.V, M2, temperature);
            }
            verdict = theirs < mine ? kTaken : kRefused;
        }
        if (verdict != kTaken) break;
    }
    int64_t token = -100;
    const float* noise = p.noise + n * p.noise_row;
    if (greedy) {
        if (split != 0) return;
        if (largest[taken] != 0) {      // r is 1 there and 0 elsewhere
            token = static_cast<int64_t>(~static_cast<uint32_t>(largest[taken]));
            const float e = noise[token];
            if (fabsf(e) == INFINITY) token = 0;
            else if (!(e > 0.0f || __float_as_uint(e) == 0u) && (p.V > 1 || e != e)) token = p.V > 1 ? token == 0 : -100;
        }
    } else {
        const int64_t drafted = taken < length ? p.drafts[static_cast<int64_t>(n) * p.K + taken] : -1;
        const float2 a = stats[taken];
        const T *x = row_of<T>(p, n, taken), *y = taken < length && p.draft_logits != nullptr ? row_of<T>(p, n, p.K + 1 + taken) : nullptr;
        float2 b = y != nullptr ? stats[p.K + 1 + taken] : make_float2(0.0f, 1.0f);
        // A draft without a distribution that was turned down: p without it, since p is at most 1.
        const int passed = y == nullptr && drafted >= 0 && drafted < p.V ? static_cast<int>(drafted) : -1;
        const int begin = split * p.draw_span, end = begin + p.draw_span < p.V ? begin + p.draw_span : p.V;
        Race mine = nobody();
        Raw<T, VEC> raw, raw2;
        Raw<float, 4> e[VEC / 4];
        float bar = -INFINITY;
        int at = begin + static_cast<int>(threadIdx.x) * VEC;
        const auto fetch = [&](int from) {
            raw.load(x, from, end - from);
            if (y != nullptr) raw2.load(y, from, end - from);
#pragma unroll
            for (int u = 0; u < VEC / 4; ++u) e[u].load(noise, from + 4 * u, end - from - 4 * u);
        };
        fetch(at);
        if (!something(b)) y = nullptr, b = make_float2(0.0f, 1.0f);        // nothing of it is left to take from p
        const float c = a.x / slope.high, c2 = b.x / slope.high, part = 1.0f / a.y, part2 = 1.0f / b.y;
        const float of_sums = y != nullptr ? per_sum : 0.0f;        // what all of p have in common changes no order
        bool odd = beyond || coarse(a.x) || coarse(b.x);
        for (int from = begin; from < end; from += BLOCK * VEC, at += BLOCK * VEC) {        // together: the wave shares what it has seen
            float v[VEC], v2[VEC], inverse[VEC], rough[VEC];
            const int left = end - at;
            uint32_t least_bits = 0xffffffffu, most_bits = 0u;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float one = j < left ? e[j / 4][j % 4] : 1.0f;
                v[j] = j < left && at + j != passed ? raw[j] : -INFINITY;
                v2[j] = y != nullptr && j < left ? raw2[j] : -INFINITY;
                inverse[j] = __builtin_amdgcn_rcpf(one);
                const uint32_t bits = __float_as_uint(one);
                least_bits = least_bits < bits ? least_bits : bits, most_bits = most_bits > bits ? most_bits : bits;
            }
            // As whole numbers the bits of positive floats are in order, and those of negative ones and NaN behind.
            const bool usual = least_bits >= __float_as_uint(kLeastNoise) && most_bits <= __float_as_uint(kMostNoise);
            if (from + BLOCK * VEC < end) fetch(at + BLOCK * VEC);
            // What the wave has seen beats most elements by far, by their shares without corrections, off by less than 2^-14, and what vanishes in float32.
            constexpr float kRough = 6.2e-5f, kVanishing = 1e-37f;
            bool alive[VEC];            // may have more than 0
            if (__ballot(!usual) == 0) {
                float least = 0.0f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float share = __builtin_amdgcn_exp2f(exponent_of(v[j], a.x, slope)) * part, theirs = y != nullptr ? __builtin_amdgcn_exp2f(exponent_of(v2[j], b.x, slope)) * part2 : 0.0f;
                    const float middle = (share - theirs) * inverse[j], width = fmaf(share + theirs, kRough, kVanishing) * inverse[j];
                    least = fmaxf(least, middle - width);
                    rough[j] = fmaxf(middle + width, 0.0f);
                    alive[j] = rough[j] > 0.0f && v[j] > -INFINITY;
                }
                bar = fmaxf(bar, lane_max(least));
            } else {
                float least = -INFINITY;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float share = __builtin_amdgcn_exp2f(exponent_of(v[j], a.x, slope)) * part, theirs = y != nullptr ? __builtin_amdgcn_exp2f(exponent_of(v2[j], b.x, slope)) * part2 : 0.0f;
                    const float width = fmaf(share + theirs, kRough, kVanishing), most = fmaxf((share - theirs) + width, 0.0f), few = fmaxf((share - theirs) - width, 0.0f);
                    const bool negative = inverse[j] < 0.0f;
                    rough[j] = (negative ? few : most) * inverse[j];
                    if (j < left) least = fmaxf(least, (negative ? most : few) * inverse[j]);
                    alive[j] = most > 0.0f && v[j] > -INFINITY;
                    odd = odd || !(fabsf(inverse[j]) >= 0.999f / kMostNoise && fabsf(inverse[j]) <= 1.001f / kLeastNoise);
                }
                bar = fmaxf(bar, lane_max(least));
            }
            const bool none = mine.zero == kNone;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                // Of those that are 0 a lane's first one counts.
                if (rough[j] >= bar && (alive[j] || none)) {
                    const float p1 = share_of(v[j], a.x, c, slope) * part, p2 = y != nullptr ? share_of(v2[j], b.x, c2, slope) * part2 : 0.0f;
                    const float r = p1 - p2, unsure = fmaf(p1, of_sums + share_doubt(exponent_of(v[j], a.x, slope)), p2 > 0.0f ? p2 * (of_sums + share_doubt(exponent_of(v2[j], b.x, slope))) : 0.0f) + 1e-30f;
                    const float most = r + unsure, few = fmaxf(r - unsure, 0.0f);
                    if (v[j] == -INFINITY || most <= 0.0f) mine.zero = j < left && at + j < mine.zero ? at + j : mine.zero;
                    else mine = join(mine, Race{(inverse[j] < 0.0f ? few : most) * inverse[j], -INFINITY, (inverse[j] < 0.0f ? most : few) * inverse[j], at + j, kNone});
                }
            }
        }
        if (odd) mine.first = mine.second = INFINITY;
        mine = lane_race(mine);
        if (lane == 0) races[wave] = mine;
        __syncthreads();
        mine = join(join(races[0], races[1]), join(races[2], races[3]));
        if (p.draw_splits > 1) {
            // Parts are written and read past the dies' own caches and counted once they have arrived (a fence in place of that, which empties a die's cache, took 23 of 45 us a
            // workgroup at 256 x 128000).
            uint64_t* parts = p.parts + static_cast<int64_t>(n) * p.draw_splits * 3;
            if (threadIdx.x == 0) {
                __hip_atomic_store(parts + 3 * split, two_words(mine.first, mine.second), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(parts + 3 * split + 1, two_words(mine.lower, __int_as_float(mine.index)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(parts + 3 * split + 2, static_cast<uint64_t>(mine.zero), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
                last = __hip_atomic_fetch_add(p.arrived + n, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<uint32_t>(p.draw_splits - 1);
            }
            __syncthreads();
            if (!last) return;
            mine = nobody();
            if (lane < p.draw_splits) {
                const uint64_t one = __hip_atomic_load(parts + 3 * lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const uint64_t two = __hip_atomic_load(parts + 3 * lane + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const uint64_t three = __hip_atomic_load(parts + 3 * lane + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                mine = Race{__uint_as_float(static_cast<uint32_t>(one)), __uint_as_float(static_cast<uint32_t>(one >> 32)), __uint_as_float(static_cast<uint32_t>(two)),
                            static_cast<int>(two >> 32), static_cast<int>(three)};
            }
            mine = lane_race(mine);
        }
        if (something(a)) {
            token = winner(mine);
            if (token < 0) token = exact_draw<T, BLOCK>(x, y, passed, p.V, temperature, noise);
        }
    }
    if (static_cast<int>(threadIdx.x) <= p.K) {
        const int j = threadIdx.x;
        p.tokens[static_cast<int64_t>(n) * (p.K + 1) + j] = j < taken ? p.drafts[static_cast<int64_t>(n) * p.K + j] : (j == taken ? token : -100);
    }
    if (threadIdx.x == 0) p.accepted[n] = taken;
}

// ------------------------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------------------------
struct VerifyShape {
    int splits, span, draw_splits, draw_span;
};
void split_row(int64_t rows, int64_t wanted, int least, int V, int* splits, int* span) {
    int64_t pieces = (wanted + rows - 1) / rows;
    const int64_t useful = (V + least - 1) / least;
    pieces = pieces < useful ? pieces : useful;
    pieces = pieces < kMostSplits ? (pieces < 1 ? 1 : pieces) : kMostSplits;
    *span = static_cast<int>(((V + pieces - 1) / pieces + 1023) / 1024 * 1024);
    *splits = (V + *span - 1) / *span;
}
// Few rows are split until four workgroups to a CU have a piece each (32 x 8 x 32000 float32: 17.7 us, with two 19.2), but pieces are of some rounds of a workgroup at least: 4096 elements in
// the first launch (one request of 4 x 32000: 4096 12.8, 8192 13.0, 16384 13.9 us), 2048 in the second, whose pieces follow a chain of their own (2048 11.9, 4096 13.0, 8192 15.4; these and those above as measured when the draw had exponential noise alone, which made it 1 us shorter).
VerifyShape verify_shape(int64_t N, int rows, int V) {
    VerifyShape s;
    split_row(N * rows, compute_units() * 4, 4096, V, &s.splits, &s.span);
    split_row(N, compute_units() * 4, 2048, V, &s.draw_splits, &s.draw_span);
    return s;
}
int check_verification(const char* name, int N, int K, int V, int dtype) {
    if (N < 0 || K < 0 || V < 1) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: N=%d K=%d V=%d", name, N, K, V);
    if (!valid_dtype(dtype)) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", name, dtype);
    if (K > kMostDrafts || N > (1 << 20) || V > (1 << 30))
        return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: at most %d drafts of 2^20 requests and 2^30 logits, got K=%d N=%d V=%d", name, kMostDrafts, K, N, V);
    return SNNF_OK;
}
size_t rounded(size_t bytes) { return (bytes + 15) / 16 * 16; }

template <typename T>
void launch_verification(const VerifyArgs& p, hipStream_t stream) {
    verify_rows_kernel<T, 256><<<grid_of(static_cast<int64_t>(p.N) * p.rows * p.splits), dim3(256), 0, stream>>>(p);
    verify_draw_kernel<T><<<grid_of(static_cast<int64_t>(p.N) * p.draw_splits), dim3(256), 0, stream>>>(p);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_draft_verification_workspace_bytes(int N, int K, int V, int draft_logits) {
    if (check_verification("snnf_draft_verification_workspace_bytes", N, K, V, SNNF_F32) != SNNF_OK) return 0;
    const int rows = draft_logits ? 2 * K + 1 : K + 1;
    const VerifyShape s = verify_shape(N, rows, V);
    const size_t pieces = static_cast<size_t>(N) * rows * s.splits;
    return rounded(pieces * 8) + rounded(pieces * 8) + static_cast<size_t>(N) * s.draw_splits * 24 + rounded(static_cast<size_t>(N) * 4);
}

extern "C" int snnf_draft_verification(const void* logits, int64_t logits_row, int64_t logits_step, const void* draft_logits, int64_t draft_row, int64_t draft_step, int N,
                                       int K, int V, int dtype, const int64_t* drafts, const float* uniforms, const float* noise, int64_t noise_row, const int32_t* lengths,
                                       float temperature, const float* temperatures, int64_t* tokens, int32_t* accepted, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    const int rc = check_verification("snnf_draft_verification", N, K, V, dtype);
    if (rc != SNNF_OK) return rc;
    if (N == 0) return SNNF_OK;
    if (logits == nullptr || noise == nullptr || tokens == nullptr || accepted == nullptr || (K > 0 && (drafts == nullptr || uniforms == nullptr)))
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_draft_verification: logits, drafts, uniforms, noise, tokens and accepted must be non-null");
    if (K == 0) draft_logits = nullptr;
    const size_t need = snnf_draft_verification_workspace_bytes(N, K, V, draft_logits != nullptr);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
        return fail(SNNF_ERR_WORKSPACE, "snnf_draft_verification: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    VerifyArgs p = {};
    p.logits = logits, p.logits_row = logits_row, p.logits_step = logits_step;
    p.draft_logits = draft_logits, p.draft_row = draft_row, p.draft_step = draft_step;
    p.drafts = drafts, p.uniforms = uniforms, p.noise = noise, p.noise_row = noise_row;
    p.lengths = lengths, p.temperature = temperature, p.temperatures = temperatures;
    p.N = N, p.K = K, p.V = V, p.rows = draft_logits != nullptr ? 2 * K + 1 : K + 1;
    const VerifyShape s = verify_shape(N, p.rows, V);
    p.splits = s.splits, p.span = s.span, p.draw_splits = s.draw_splits, p.draw_span = s.draw_span;
    const size_t pieces = static_cast<size_t>(N) * p.rows * s.splits;
    char* space = static_cast<char*>(workspace);
    p.stats = reinterpret_cast<float2*>(space);
    p.largest = reinterpret_cast<uint64_t*>(space += rounded(pieces * 8));
    p.parts = reinterpret_cast<uint64_t*>(space += rounded(pieces * 8));
    p.arrived = reinterpret_cast<uint32_t*>(space + static_cast<size_t>(N) * s.draw_splits * 24);
    p.tokens = tokens, p.accepted = accepted;
    hipStream_t hs = as_stream(stream);
    if (dtype == SNNF_F32) launch_verification<float>(p, hs);
    else if (dtype == SNNF_BF16) launch_verification<bf16_t>(p, hs);
    else launch_verification<f16_t>(p, hs);
    return check_launch("snnf_draft_verification");
}
