// Gated linear recurrence over a sequence and its gradient: the neuron without threshold and reset, with a leak that is given per
// step and channel.
//     leaky :  a = sigmoid(g),  h_t = a h_{t-1} + (1 - a) x_t          linear:  a = g,  h_t = a h_{t-1} + x_t
// A step composes with the next one: a run of steps is h -> A h + H with A the product of its a and H its result from h = 0. So a
// sequence is cut into runs that are reduced to (A, H) at once and joined in order: a wave holds the elements of `S` steps of 64 * VEC
// channels in registers, the W waves of a workgroup hold consecutive runs (a tile of W * S steps) and join through LDS, and where
// there are too few channels to fill the chip, workgroups take chunks of whole tiles whose (A, H) a first kernel works out.
// Joining is the same chain of fused multiply-adds in every variant's order: results do not depend on timing.
//
// Gradient: with r_t the gradient that reaches h_t from later steps, s_t = dh_t + r_t and r_{t-1} = a_t s_t, the same recurrence
// backwards; dx = s (1 - a) or s, dg = s (h_{t-1} - x) a (1 - a) or s h_{t-1}. h_{t-1} is not read but worked out again from the
// float32 state that the forward pass leaves where each tile of the backward pass begins ("marks"): less to read than h itself, and no
// rounding of h to 16 bits enters the gradient.
#include "snnf_common.h"

namespace snnf {
namespace {

constexpr int kSteps = 16;              // steps of a wave's run, forward
constexpr int kBackSteps = 8;           // and backward, which holds twice the values for each

constexpr int kMostSteps = 1 << 30;

struct Series {                         // [T, N, D] with elements of a row next to each other
    const void* p;
    int64_t step, row;
};
struct Output {
    void* p;
    int64_t step, row;
};

struct Args {
    Series x, gate, dh;
    Output h, dx, dgate;
    const uint8_t* starts;
    int64_t starts_step, starts_row;
    const int32_t* lengths;
    const float* state;                 // forward: the state before the first step; backward: the gradient of the last state
    float* state_out;                   // the other way round
    float* marks;
    float* chunks;                      // [chunk][2][N * D]: what a chunk does to the value that enters it
    int T, N, D;
    int groups;                         // wave-wide groups of channels in a row
    int span;                           // steps from one mark to the next
    int tiles;                          // tiles of a chunk
    int n_chunks;
    int leaky;
};

template <typename XT> constexpr bool kPrecise = false;
template <> constexpr bool kPrecise<float> = true;

// a = sigmoid(g) and 1 - a, both to full relative accuracy: with e = exp(-|g|) the larger is 1 / (1 + e) and the smaller e / (1 + e).
// v_exp_f32 works on powers of two; for float32 tensors what the product with log2(e) loses is put back to first order.
template <bool PRECISE>
__device__ __forceinline__ void leak(float g, float& a, float& rest) {
    constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.925963033500e-8f, kLn2 = 0.69314718055994530942f;
    const float y = -fabsf(g);
    const float t = y * kLog2e;
    float e = __builtin_amdgcn_exp2f(t);
    if constexpr (PRECISE) {
        const float lost = fmaf(y, kLog2eLow, fmaf(y, kLog2e, -t));
        e = y < -126.0f ? e : fmaf(e, lost * kLn2, e);             // (far out e is 0 or next to it; -inf would make lost a NaN)
    }
    const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
    const bool positive = g >= 0.0f;
    a = positive ? big : small;
    rest = positive ? small : big;
    if (g != g) a = rest = g;
}

template <typename XT, int VEC>
__device__ __forceinline__ Pack<XT, VEC> load_at(const void* base, int64_t offset, int lane_offset) {
    return *reinterpret_cast<const Pack<XT, VEC>*>(static_cast<const XT*>(base) + offset + lane_offset);
}

// Bit i: the state is dropped before step `first` + i.
__device__ __forceinline__ uint32_t start_bits(const Args& p, int n, int first, int lim, int steps) {
    const int lane = threadIdx.x & 63;
    bool on = false;
    if (lane < steps && first + lane < lim) on = p.starts[static_cast<int64_t>(first + lane) * p.starts_step + static_cast<int64_t>(n) * p.starts_row] != 0;
    return static_cast<uint32_t>(__ballot(on));
}

// One link of the chain: what a run of steps makes of the value that enters it. A run that drops the value has A = 0, and must not multiply
// an infinity or NaN that belongs to what came before.
template <bool STARTS>
__device__ __forceinline__ float link(float A, float entering, float H) {
    const float v = fmaf(A, entering, H);
    if constexpr (STARTS) return A == 0.0f ? H : v;
    return v;
}

struct Place {
    int n, d, lim;                      // sequence, first channel of the lane, steps that count
    bool active;
    int64_t cell;                       // n * D + d
};
template <int VEC>
__device__ __forceinline__ Place place(const Args& p) {
    Place q;
    q.n = blockIdx.x / p.groups;
    q.d = ((blockIdx.x - q.n * p.groups) * 64 + (threadIdx.x & 63)) * VEC;
    q.active = q.d < p.D;
    q.cell = static_cast<int64_t>(q.n) * p.D + q.d;
    q.lim = p.T;
    if (p.lengths != nullptr) {
        const int len = p.lengths[q.n];
        q.lim = len < 0 ? 0 : (len < p.T ? len : p.T);
    }
    q.lim = __builtin_amdgcn_readfirstlane(q.lim);
    return q;
}

// The elements of S steps from `first` on, those that do not count left as they were.
template <typename XT, int VEC, int S>
__device__ __forceinline__ void fetch(Pack<XT, VEC> (&to)[S], const Series& from, const Place& q, int first) {
    if (!q.active) return;
    const XT* base = static_cast<const XT*>(from.p) + static_cast<int64_t>(q.n) * from.row + static_cast<int64_t>(first) * from.step;
    if (first + S <= q.lim) {
#pragma unroll
        for (int i = 0; i < S; ++i) to[i] = load_at<XT, VEC>(base, i * from.step, q.d);
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (first + i < q.lim) to[i] = load_at<XT, VEC>(base, i * from.step, q.d);
    }
}

// Value that enters chunk `c`: the chunks before it (forward) or behind it (backward) in their order.
template <int VEC, bool STARTS, bool BACKWARD>
__device__ __forceinline__ void entering(const Args& p, const Place& q, int c, float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = q.active && p.state != nullptr ? p.state[q.cell + j] : 0.0f;
    if (!q.active) return;
    const int64_t cells = static_cast<int64_t>(p.N) * p.D;
    const int many = BACKWARD ? p.n_chunks - 1 - c : c;
    constexpr int kBatch = 4;
    for (int i0 = 0; i0 < many; i0 += kBatch) {
        float A[kBatch][VEC], H[kBatch][VEC];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + u < many ? i0 + u : many - 1;
            const float* from = p.chunks + (BACKWARD ? p.n_chunks - 1 - i : i) * 2 * cells + q.cell;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                A[u][j] = from[j];
                H[u][j] = from[cells + j];
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (i0 + u < many) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = link<STARTS>(A[u][j], v[j], H[u][j]);
            }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Forward. REDUCE: only (A, H) of the chunk.
// ------------------------------------------------------------------------------------------------------------------
template <typename XT, int VEC, int W, int S, bool STARTS, bool REDUCE>
__global__ __launch_bounds__(64 * W) void recurrence_kernel(Args p) {
    constexpr int kLinks = W > 1 ? W : 1;
    __shared__ float links[2][kLinks][2 * VEC][64];
    const Place q = place<VEC>(p);
    const int lane = threadIdx.x & 63, wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int chunk = blockIdx.y;
    const int begin = chunk * p.tiles * W * S, end = begin + p.tiles * W * S < p.T ? begin + p.tiles * W * S : p.T;
    using XV = Pack<XT, VEC>;
    XV g[S], x[S];
    fetch<XT, VEC, S>(g, p.gate, q, begin + wave * S);
    fetch<XT, VEC, S>(x, p.x, q, begin + wave * S);
    float v[VEC], whole[VEC];           // the state that enters the tile; REDUCE: product of the chunk so far
    if constexpr (REDUCE) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 0.0f, whole[j] = 1.0f;
    } else {
        entering<VEC, STARTS, false>(p, q, chunk, v);
    }
    int buffer = 0;
    for (int t0 = begin; t0 < end; t0 += W * S) {
        const int first = t0 + wave * S;
        uint32_t drop = 0;
        if constexpr (STARTS) drop = start_bits(p, q.n, first, q.lim, S);
        float a[S][VEC], b[S][VEC];
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool counts = first + i < q.lim;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float ai = to_float(g[i].v[j]), bi = to_float(x[i].v[j]);
                if (p.leaky) {
                    float rest;
                    leak<kPrecise<XT>>(ai, ai, rest);
                    bi *= rest;
                }
                a[i][j] = counts ? ai : 1.0f;
                b[i][j] = counts ? bi : 0.0f;
            }
        }
        const bool more = t0 + W * S < end;
        if (more) {
            fetch<XT, VEC, S>(g, p.gate, q, first + W * S);
            fetch<XT, VEC, S>(x, p.x, q, first + W * S);
        }
        float enter[VEC];
        if constexpr (W > 1 || REDUCE) {
            float A[VEC], H[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) A[j] = 1.0f, H[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool dropped = STARTS && (drop >> i & 1u);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    H[j] = dropped ? b[i][j] : fmaf(a[i][j], H[j], b[i][j]);
                    A[j] = dropped ? 0.0f : A[j] * a[i][j];
                }
            }
            if constexpr (W > 1) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    links[buffer][wave][j][lane] = A[j];
                    links[buffer][wave][VEC + j][lane] = H[j];
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    if (w == wave) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) enter[j] = v[j];
                    }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float Aw = links[buffer][w][j][lane], Hw = links[buffer][w][VEC + j][lane];
                        v[j] = link<STARTS>(Aw, v[j], Hw);
                        if constexpr (REDUCE) whole[j] *= Aw;
                    }
                }
                buffer ^= 1;
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    v[j] = link<STARTS>(A[j], v[j], H[j]);
                    whole[j] *= A[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) enter[j] = v[j];
        }
        if constexpr (!REDUCE) {
            if (p.marks != nullptr && q.active && first % p.span == 0 && first < p.T) {
                float* mark = p.marks + static_cast<int64_t>(first / p.span) * p.N * p.D + q.cell;
#pragma unroll
                for (int j = 0; j < VEC; ++j) mark[j] = enter[j];
            }
            XT* out = static_cast<XT*>(p.h.p) + static_cast<int64_t>(q.n) * p.h.row + static_cast<int64_t>(first) * p.h.step + q.d;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool dropped = STARTS && (drop >> i & 1u);
                XV y;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    enter[j] = dropped ? b[i][j] : fmaf(a[i][j], enter[j], b[i][j]);
                    y.v[j] = from_float<XT>(first + i < q.lim ? enter[j] : 0.0f);
                }
                if (first + i < p.T && q.active) *reinterpret_cast<XV*>(out + i * p.h.step) = y;
            }
            if constexpr (W == 1) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = enter[j];
            }
        }
    }
    if (!q.active || wave != 0) return;
    if constexpr (REDUCE) {
        const int64_t cells = static_cast<int64_t>(p.N) * p.D;
        float* to = p.chunks + chunk * 2 * cells + q.cell;
#pragma unroll
        for (int j = 0; j < VEC; ++j) to[j] = whole[j], to[cells + j] = v[j];
    } else if (chunk == p.n_chunks - 1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.state_out[q.cell + j] = v[j];
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Backward: tiles from the last to the first. REDUCE: only (A, R) of the chunk.
// ------------------------------------------------------------------------------------------------------------------
template <typename XT, int VEC, int W, int S, bool STARTS, bool REDUCE>
__global__ __launch_bounds__(64 * W) void recurrence_backward_kernel(Args p) {
    constexpr int kParts = REDUCE ? 2 : 3;
    __shared__ float links[2][W][kParts * VEC][64];
    const Place q = place<VEC>(p);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.y + (REDUCE ? 1 : 0);           // nothing lies before the first chunk
    const int begin = chunk * p.tiles * W * S, end = begin + p.tiles * W * S < p.T ? begin + p.tiles * W * S : p.T;
    using XV = Pack<XT, VEC>;
    XV g[S], x[S], dh[S];
    float mark[VEC];
    int t0 = begin + (end - begin - 1) / (W * S) * (W * S);
    const auto fetch_tile = [&](int at) {
        const int first = at + wave * S;
        fetch<XT, VEC, S>(g, p.gate, q, first);
        fetch<XT, VEC, S>(dh, p.dh, q, first);
        if constexpr (!REDUCE) {
            fetch<XT, VEC, S>(x, p.x, q, first);
            const float* from = p.marks + static_cast<int64_t>(at / (W * S)) * p.N * p.D + q.cell;
#pragma unroll
            for (int j = 0; j < VEC; ++j) mark[j] = q.active ? from[j] : 0.0f;
        }
    };
    fetch_tile(t0);
    float r[VEC], whole[VEC];           // the gradient that enters the tile from behind
    if constexpr (REDUCE) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) r[j] = 0.0f, whole[j] = 1.0f;
    } else {
        entering<VEC, STARTS, true>(p, q, chunk, r);
    }
    int buffer = 0;
    for (; t0 >= begin; t0 -= W * S) {
        const int first = t0 + wave * S;
        uint32_t drop = 0;
        if constexpr (STARTS) drop = start_bits(p, q.n, first, q.lim, S);
        float a[S][VEC], rest[S][VEC], e[S][VEC], xi[S][VEC], h[VEC];
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool counts = first + i < q.lim;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float ai = to_float(g[i].v[j]), ri = 1.0f;
                if (p.leaky) leak<kPrecise<XT>>(ai, ai, ri);
                a[i][j] = counts ? ai : 1.0f;
                rest[i][j] = ri;
                e[i][j] = counts ? to_float(dh[i].v[j]) : 0.0f;
                if constexpr (!REDUCE) xi[i][j] = counts ? to_float(x[i].v[j]) : 0.0f;
            }
        }
        if constexpr (!REDUCE) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[j] = mark[j];
        }
        if (t0 > begin) fetch_tile(t0 - W * S);
        float A[VEC], H[VEC], R[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) A[j] = 1.0f, H[j] = R[j] = 0.0f;
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const bool dropped = STARTS && (drop >> i & 1u);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                R[j] = dropped ? 0.0f : a[i][j] * (R[j] + e[i][j]);
                A[j] = dropped ? 0.0f : A[j] * a[i][j];
            }
        }
        if constexpr (!REDUCE) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool dropped = STARTS && (drop >> i & 1u);
                const bool counts = first + i < q.lim;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float b = counts ? rest[i][j] * xi[i][j] : 0.0f;
                    H[j] = dropped ? b : fmaf(a[i][j], H[j], b);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            links[buffer][wave][j][lane] = A[j];
            links[buffer][wave][VEC + j][lane] = R[j];
            if constexpr (!REDUCE) links[buffer][wave][2 * VEC + j][lane] = H[j];
        }
        __syncthreads();
        float enter[VEC];
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
            if (w == wave) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) enter[j] = r[j];
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float Aw = links[buffer][w][j][lane];
                r[j] = link<STARTS>(Aw, r[j], links[buffer][w][VEC + j][lane]);
                if constexpr (REDUCE) whole[j] *= Aw;
            }
        }
        if constexpr (!REDUCE) {
#pragma unroll
            for (int w = 0; w < W - 1; ++w)
                if (w < wave) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) h[j] = link<STARTS>(links[buffer][w][j][lane], h[j], links[buffer][w][2 * VEC + j][lane]);
                }
            float before[S][VEC];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool dropped = STARTS && (drop >> i & 1u);
                const bool counts = first + i < q.lim;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    before[i][j] = dropped ? 0.0f : h[j];
                    h[j] = counts ? fmaf(a[i][j], before[i][j], rest[i][j] * xi[i][j]) : h[j];
                }
            }
            XT* dx = static_cast<XT*>(p.dx.p) + static_cast<int64_t>(q.n) * p.dx.row + static_cast<int64_t>(first) * p.dx.step + q.d;
            XT* dg = static_cast<XT*>(p.dgate.p) + static_cast<int64_t>(q.n) * p.dgate.row + static_cast<int64_t>(first) * p.dgate.step + q.d;
#pragma unroll
            for (int i = S - 1; i >= 0; --i) {
                const bool dropped = STARTS && (drop >> i & 1u);
                const bool counts = first + i < q.lim;
                XV ox, og;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float s = enter[j] + e[i][j];
                    const float gx = s * rest[i][j];
                    const float gg = p.leaky ? gx * (a[i][j] * (before[i][j] - xi[i][j])) : s * before[i][j];
                    ox.v[j] = from_float<XT>(counts ? gx : 0.0f);
                    og.v[j] = from_float<XT>(counts ? gg : 0.0f);
                    enter[j] = dropped ? 0.0f : a[i][j] * s;
                }
                if (first + i < p.T && q.active) {
                    *reinterpret_cast<XV*>(dx + i * p.dx.step) = ox;
                    *reinterpret_cast<XV*>(dg + i * p.dgate.step) = og;
                }
            }
        }
        buffer ^= 1;
    }
    if (!q.active || wave != 0) return;
    if constexpr (REDUCE) {
        const int64_t cells = static_cast<int64_t>(p.N) * p.D;
        float* to = p.chunks + chunk * 2 * cells + q.cell;
#pragma unroll
        for (int j = 0; j < VEC; ++j) to[j] = whole[j], to[cells + j] = r[j];
    } else if (chunk == 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.state_out[q.cell + j] = r[j];
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Which variant: waves of a tile, steps of a wave, chunks
// ------------------------------------------------------------------------------------------------------------------
struct Shape {
    int waves, steps, chunks, tiles;
};

// Waves of a backward tile. The marks lie where these tiles begin: the rule goes by what both passes know, not by alignment.
int back_waves(int T, int N, int D) { return T <= 32 || static_cast<int64_t>(N) * D >= compute_units() * 1024ll ? 4 : 16; }

Shape shape_of(int T, int N, int D, int64_t columns, bool backward) {
    Shape s;
    const int units = compute_units();
    if (!backward && T == 1) {
        s = {1, 1, 1, 1};
        return s;
    }
    s.steps = backward ? kBackSteps : kSteps;
    s.waves = backward ? back_waves(T, N, D) : T <= kSteps ? 1 : T <= 2 * kSteps || columns >= units * 8 ? 4 : 16;
    const int tile = s.waves * s.steps, tiles = (T + tile - 1) / tile;
    s.chunks = 1;
    if (s.waves == 16 && columns < units / 2) {
        const int64_t want = (units + columns - 1) / columns;
        s.chunks = static_cast<int>(want < tiles ? want : tiles);
    }
    s.tiles = (tiles + s.chunks - 1) / s.chunks;
    s.chunks = (tiles + s.tiles - 1) / s.tiles;
    return s;
}

// Channels of a lane: two 16-bit ones where rows allow 4-byte accesses, else one.
int vector_of(int D, int dtype) { return dtype != SNNF_F32 && D % 2 == 0 && D > 64 ? 2 : 1; }
int64_t columns_of(int N, int D, int vec) { return static_cast<int64_t>(N) * ((D + 64 * vec - 1) / (64 * vec)); }

size_t workspace_of(int T, int N, int D, int dtype, bool backward) {
    // One lane-width more than the call may take gives more chunks, never fewer: the larger of both is enough for either.
    size_t most = 0;
    for (int vec = 1; vec <= vector_of(D, dtype); ++vec) {
        const Shape s = shape_of(T, N, D, columns_of(N, D, vec), backward);
        const size_t bytes = s.chunks > 1 ? static_cast<size_t>(s.chunks) * 2 * N * D * sizeof(float) : 0;
        most = bytes > most ? bytes : most;
    }
    return most;
}

template <typename XT, int VEC, int W, int S, bool STARTS>
int run(Args& p, const Shape& s, int64_t columns, bool backward, hipStream_t stream) {
    const dim3 block(64 * W);
    if (backward) {
        if constexpr (S == kBackSteps) {
            if (s.chunks > 1) recurrence_backward_kernel<XT, VEC, W, S, STARTS, true><<<dim3(columns, s.chunks - 1), block, 0, stream>>>(p);
            recurrence_backward_kernel<XT, VEC, W, S, STARTS, false><<<dim3(columns, s.chunks), block, 0, stream>>>(p);
        }
    } else {
        if constexpr (S != kBackSteps) {
            if constexpr (W > 1)
                if (s.chunks > 1) recurrence_kernel<XT, VEC, W, S, STARTS, true><<<dim3(columns, s.chunks - 1), block, 0, stream>>>(p);
            recurrence_kernel<XT, VEC, W, S, STARTS, false><<<dim3(columns, s.chunks), block, 0, stream>>>(p);
        }
    }
    return check_launch(backward ? "snnf_gated_recurrence_backward" : "snnf_gated_recurrence");
}

template <typename XT, int VEC, bool STARTS>
int pick(Args& p, bool backward, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    p.groups = (p.D + 64 * VEC - 1) / (64 * VEC);
    const int64_t columns = static_cast<int64_t>(p.N) * p.groups;
    if (columns > 0x7fffffffLL) return fail(SNNF_ERR_UNSUPPORTED, "snnf_gated_recurrence: unsupported_shape: N=%d D=%d", p.N, p.D);
    const Shape s = shape_of(p.T, p.N, p.D, columns, backward);
    p.span = back_waves(p.T, p.N, p.D) * kBackSteps;
    p.tiles = s.tiles;
    p.n_chunks = s.chunks;
    if (s.chunks > 1) {
        const size_t need = static_cast<size_t>(s.chunks) * 2 * p.N * p.D * sizeof(float);
        if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 4))
            return fail(SNNF_ERR_WORKSPACE, "snnf_gated_recurrence: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
        p.chunks = static_cast<float*>(workspace);
    }
    if (backward) return s.waves == 16 ? run<XT, VEC, 16, kBackSteps, STARTS>(p, s, columns, true, stream) : run<XT, VEC, 4, kBackSteps, STARTS>(p, s, columns, true, stream);
    if (s.steps == 1) return run<XT, VEC, 1, 1, STARTS>(p, s, columns, false, stream);
    if (s.waves == 1) return run<XT, VEC, 1, kSteps, STARTS>(p, s, columns, false, stream);
    return s.waves == 16 ? run<XT, VEC, 16, kSteps, STARTS>(p, s, columns, false, stream) : run<XT, VEC, 4, kSteps, STARTS>(p, s, columns, false, stream);
}

template <typename XT>
int launch(Args& p, bool pairs, bool backward, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if constexpr (sizeof(XT) == 2) {
        if (pairs)
            return p.starts != nullptr ? pick<XT, 2, true>(p, backward, workspace, workspace_bytes, stream) : pick<XT, 2, false>(p, backward, workspace, workspace_bytes, stream);
    }
    return p.starts != nullptr ? pick<XT, 1, true>(p, backward, workspace, workspace_bytes, stream) : pick<XT, 1, false>(p, backward, workspace, workspace_bytes, stream);
}

bool pairs_fit(const void* p, int64_t step, int64_t row) { return aligned_to(p, 4) && step % 2 == 0 && row % 2 == 0; }

int dispatch(Args& p, int dtype, bool backward, void* workspace, size_t workspace_bytes, void* stream) {
    if (p.T > kMostSteps) return fail(SNNF_ERR_UNSUPPORTED, "snnf_gated_recurrence: unsupported_temporal_length: at most %d steps, got %d", kMostSteps, p.T);
    bool pairs = vector_of(p.D, dtype) == 2 && pairs_fit(p.x.p, p.x.step, p.x.row) && pairs_fit(p.gate.p, p.gate.step, p.gate.row);
    if (backward)
        pairs = pairs && pairs_fit(p.dh.p, p.dh.step, p.dh.row) && pairs_fit(p.dx.p, p.dx.step, p.dx.row) && pairs_fit(p.dgate.p, p.dgate.step, p.dgate.row);
    else
        pairs = pairs && pairs_fit(p.h.p, p.h.step, p.h.row);
    hipStream_t hs = as_stream(stream);
    if (dtype == SNNF_F32) return launch<float>(p, false, backward, workspace, workspace_bytes, hs);
    if (dtype == SNNF_BF16) return launch<bf16_t>(p, pairs, backward, workspace, workspace_bytes, hs);
    return launch<f16_t>(p, pairs, backward, workspace, workspace_bytes, hs);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_gated_recurrence_workspace_bytes(int T, int N, int D, int dtype, int backward) {
    if (T < 1 || N < 1 || D < 1 || !valid_dtype(dtype)) return 0;
    return workspace_of(T, N, D, dtype, backward != 0);
}

extern "C" size_t snnf_gated_recurrence_marks_bytes(int T, int N, int D) {
    if (T < 1 || N < 1 || D < 1) return 0;
    const int span = back_waves(T, N, D) * kBackSteps;
    return (static_cast<size_t>(T) + span - 1) / span * N * D * sizeof(float);
}

extern "C" int snnf_gated_recurrence(const void* x, int64_t x_step, int64_t x_row, const void* gate, int64_t gate_step, int64_t gate_row, int T, int N,
                                     int D, int dtype, int form, const void* starts, int64_t starts_step, int64_t starts_row, const int32_t* lengths,
                                     const float* state, void* h, int64_t h_step, int64_t h_row, float* state_out, float* marks, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    if (T < 1 || N < 0 || D < 0) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence: T=%d N=%d D=%d", T, N, D);
    if (!valid_dtype(dtype)) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence: unknown dtype code %d", dtype);
    if (form != SNNF_RECURRENCE_LEAKY && form != SNNF_RECURRENCE_LINEAR)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence: unknown form %d", form);
    if (N == 0 || D == 0) return SNNF_OK;
    if (x == nullptr || gate == nullptr || h == nullptr || state_out == nullptr)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence: x, gate, h and state_out must be non-null");
    Args p = {};
    p.x = {x, x_step, x_row};
    p.gate = {gate, gate_step, gate_row};
    p.h = {h, h_step, h_row};
    p.starts = static_cast<const uint8_t*>(starts);
    p.starts_step = starts_step;
    p.starts_row = starts_row;
    p.lengths = lengths;
    p.state = state;
    p.state_out = state_out;
    p.marks = marks;
    p.T = T, p.N = N, p.D = D;
    p.leaky = form == SNNF_RECURRENCE_LEAKY;
    return dispatch(p, dtype, false, workspace, workspace_bytes, stream);
}

extern "C" int snnf_gated_recurrence_backward(const void* x, int64_t x_step, int64_t x_row, const void* gate, int64_t gate_step, int64_t gate_row,
                                              const void* dh, int64_t dh_step, int64_t dh_row, int T, int N, int D, int dtype, int form,
                                              const void* starts, int64_t starts_step, int64_t starts_row, const int32_t* lengths, const float* marks,
                                              const float* dstate, void* dx, int64_t dx_step, int64_t dx_row, void* dgate, int64_t dgate_step,
                                              int64_t dgate_row, float* dstate_in, void* workspace, size_t workspace_bytes, void* stream) {
    if (T < 1 || N < 0 || D < 0) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence_backward: T=%d N=%d D=%d", T, N, D);
    if (!valid_dtype(dtype)) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence_backward: unknown dtype code %d", dtype);
    if (form != SNNF_RECURRENCE_LEAKY && form != SNNF_RECURRENCE_LINEAR)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence_backward: unknown form %d", form);
    if (N == 0 || D == 0) return SNNF_OK;
    if (x == nullptr || gate == nullptr || dh == nullptr || marks == nullptr || dx == nullptr || dgate == nullptr || dstate_in == nullptr)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence_backward: x, gate, dh, marks, dx, dgate and dstate_in must be non-null");
    Args p = {};
    p.x = {x, x_step, x_row};
    p.gate = {gate, gate_step, gate_row};
    p.dh = {dh, dh_step, dh_row};
    p.dx = {dx, dx_step, dx_row};
    p.dgate = {dgate, dgate_step, dgate_row};
    p.starts = static_cast<const uint8_t*>(starts);
    p.starts_step = starts_step;
    p.starts_row = starts_row;
    p.lengths = lengths;
    p.marks = const_cast<float*>(marks);
    p.state = dstate;
    p.state_out = dstate_in;
    p.T = T, p.N = N, p.D = D;
    p.leaky = form == SNNF_RECURRENCE_LEAKY;
    return dispatch(p, dtype, true, workspace, workspace_bytes, stream);
}
