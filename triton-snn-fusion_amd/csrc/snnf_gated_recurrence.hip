// Gated linear recurrence over a sequence and its gradient: the neuron without threshold and reset, with a leak that is given per
// step and channel.
//     leaky :  a = sigmoid(g),  h_t = a h_{t-1} + (1 - a) x_t          linear:  a = g,  h_t = a h_{t-1} + x_t
// A step composes with the next one: a run of steps is h -> A h + H with A the product of its a and H its result from h = 0. So a
// sequence is cut into runs that are reduced to (A, H) at once and joined in order: a wave holds the elements of `S` steps of 64 * VEC
// channels in registers, the W waves of a workgroup hold consecutive runs (a tile of W * S steps) and join through LDS. Where there are
// columns of channels enough to fill the chip, a workgroup walks over the tiles of its column. Where there are not, tiles are
// handed out in the order of time and each is joined with those before it through memory ("relay"): every element is still read once.
// The value that enters a tile is always the same chain of fused multiply-adds over the tiles before it: results do not depend on timing.
// A of a run with a long memory is worked out as 1 - c with c_t = c_{t-1} + (1 - a_t) (1 - c_{t-1}), which loses one rounding where the
// product of the a loses one per step: the last state of 4096 steps with memories of up to 2000 is then as exact as from a scan in
// which no value passes more than log2 T roundings.
//
// Gradient: with r_t the gradient that reaches h_t from later steps, s_t = dh_t + r_t and r_{t-1} = a_t s_t, the same recurrence
// backwards; dx = s (1 - a) or s, dg = s (h_{t-1} - x) a (1 - a) or s h_{t-1}. h_{t-1} is not read but worked out again from the
// float32 state that the forward pass leaves where each tile of the backward pass begins ("marks"): less to read than h itself, and no
// rounding of h to 16 bits enters the gradient.
#include <utility>

#include "snnf_sequence.h"

namespace snnf {
namespace {

// Waves of a tile and steps of a wave. Relay: the largest tile that 128 registers a lane and 16 waves allow (with the waves that relay), since
// each costs a trip through memory (16384 x 2 x 2048 bf16, forward: tiles of 224 steps 94 us, of 168 101, of 112 124). Walk: enough waves to
// cover the latency of memory by themselves where there are few columns (2048 x 16 x 2048: 8 waves 83 us, 4 85; 100 x 16 x 1024: 6.1 and
// 7.2), 4 where workgroups cover for each other (512 x 64 x 2048: 78 us, 8 waves 80).
constexpr int kRelayWaves = 14, kRelaySteps = 16, kRelayBackSteps = 8;
constexpr int kWalkWaves = 8, kWalkWavesMany = 4, kWalkSteps = 8;
// Marks are left by the wave whose run begins where a tile of the backward pass does.
static_assert(kRelayWaves * kRelayBackSteps % kRelaySteps == 0);
// Tiles that a relay looks back at in one go: more of them reach further where all tiles start at once, and cost their loads where most
// tiles in front are done (8192 x 1 x 1024: 2 28.6 us, 4 23.5, 8 22.4, 16 24.5; 16384 x 2 x 2048: 92, 94, 102, 111).
constexpr int kReach = 4;
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
    uint32_t* ticket;                   // relay: tiles handed out so far, less one
    uint64_t* runs;                     // relay: [tile][N * D] (A, H) of a tile, all ones while it is not known
    uint32_t* values;                   // relay: [tile][N * D] value behind a tile, all ones while it is not known
    int T, N, D;
    int groups;                         // wave-wide groups of channels in a row
    int columns;                        // N * groups
    int tiles;
    int span;                           // steps from one mark to the next
};

// Lane i: whether the state is dropped before step `first` + i.
__device__ __forceinline__ uint8_t start_of(const Args& p, int n, int first, int lim, int steps) {
    const int lane = threadIdx.x & 63;
    return lane < steps && first + lane < lim ? p.starts[static_cast<int64_t>(first + lane) * p.starts_step + static_cast<int64_t>(n) * p.starts_row] : 0;
}

// One link of the chain: what a run of steps makes of the value that enters it. A run that drops the value says so by A = -0, which no other run
// has, and must not multiply an infinity or NaN that belongs to what came before; A = 0 from a decay of 0 does.
constexpr uint32_t kDropped = 0x80000000u;
template <bool STARTS>
__device__ __forceinline__ bool dropped(float A) { return STARTS && __float_as_uint(A) == kDropped; }
template <bool STARTS>
__device__ __forceinline__ float link(float A, float entering, float H) {
    return dropped<STARTS>(A) ? H : fmaf(A, entering, H);
}
template <bool STARTS>
__device__ __forceinline__ float run_of(float A, bool drops) {
    if constexpr (STARTS) return drops ? __uint_as_float(kDropped) : A + 0.0f;      // -0 + 0 = 0
    return A;
}

// A run of the linear form with a gate beyond 1 in magnitude, unless it drops the value, gets an infinite A: its product, or its result from 0, may
// leave float32's range where the state itself does not. The runs of its tile then take the value one after the other, step by step, which costs little
// where columns fill the chip (2048 x 16 x 2048 bf16, such a gate in every tile: forward 81 -> 87 us, backward 138 -> 172) and a chain of tiles where they do
// not (8192 x 1 x 1024: 27 -> 145, 51 -> 350).
constexpr float kInTurn = INFINITY;

// What is left of the value that enters a run: the product of its decays, or for a long memory 1 - c. Where the product of decays other than 0 vanishes
// it is the smallest number there is: an infinite value stays infinite then, as it does step by step, and any other is off by 2^-149 of it at
// most either way. `least`: the smallest decay's magnitude; a sigmoid is never 0.
template <bool LEAKY>
__device__ __forceinline__ float left_over(float product, float c, float least) {
    constexpr float kSmallest = 0x1p-149f;
    const float left = c < 0.5f && c > -0.5f ? 1.0f - c : product;
    if constexpr (LEAKY) return __builtin_elementwise_maximum(left, kSmallest);
    return left == 0.0f && least > 0.0f ? __builtin_copysignf(kSmallest, left) : left;
}

struct Place {
    int n, d, lim;                      // sequence, first channel of the lane, steps that count
    bool active;
    int64_t cell;                       // n * D + d
};
template <int VEC>
__device__ __forceinline__ Place place(const Args& p, int column) {
    Place q;
    q.n = column / p.groups;
    q.d = ((column - q.n * p.groups) * 64 + (threadIdx.x & 63)) * VEC;
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

// A tensor from step `first` of a sequence on as a buffer, so that steps are a scalar offset and a lane behind the row's end, whose offset lies
// outside any buffer, reads 0 and stores nothing. Steps of a run and a row's bytes together stay below 2^31 (`dispatch`).
constexpr int kBufferBytes = 0x7fffffff;
__device__ __forceinline__ int lane_bytes(const Place& q, int size) { return q.active ? q.d * size : static_cast<int>(0x80000000u); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* p, int64_t step, int64_t row, const Place& q, int first, int size) {
    const char* base = static_cast<const char*>(p) + (static_cast<int64_t>(q.n) * row + static_cast<int64_t>(first) * step) * size;
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const uint64_t same = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32))) << 32 |
                          static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at)));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(same), 0, kBufferBytes, 0x00020000);
}
// VEC elements of a row in one register; as a word, not as a struct of 16-bit halves, which the compiler would take apart at every copy.
template <typename XT, int VEC>
__device__ __forceinline__ uint32_t read(__amdgpu_buffer_rsrc_t from, int lane_bytes, int step_bytes) {
    if constexpr (sizeof(XT) * VEC == 4) return __builtin_amdgcn_raw_buffer_load_b32(from, lane_bytes, step_bytes, 0);
    else return static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(from, lane_bytes, step_bytes, 0));
}
template <typename XT, int VEC>
__device__ __forceinline__ void write(__amdgpu_buffer_rsrc_t to, uint32_t word, int lane_bytes, int step_bytes) {
    if constexpr (sizeof(XT) * VEC == 4) __builtin_amdgcn_raw_buffer_store_b32(word, to, lane_bytes, step_bytes, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(word), to, lane_bytes, step_bytes, 0);
}
template <typename XT, int VEC>
__device__ __forceinline__ uint32_t word_of(const float (&v)[VEC]) {
    if constexpr (sizeof(XT) == 4) return __float_as_uint(v[0]);
    else if constexpr (VEC == 2) return pair_word<XT>(v[0], v[1]);
    else return from_float<XT>(v[0]).bits;
}

// The elements of S steps from `first` on. Steps that do not count are read from the last that does (from the first if there is none).
template <typename XT, int VEC, int S>
__device__ __forceinline__ void fetch(uint32_t (&to)[S], const Series& from, const Place& q, int first) {
    const int last = q.lim > 0 ? q.lim - 1 : 0, begin = first < last ? first : last;
    const auto rows = rows_at(from.p, from.step, from.row, q, begin, sizeof(XT));
    const int step = static_cast<int>(from.step) * static_cast<int>(sizeof(XT)), d = lane_bytes(q, sizeof(XT));
#pragma unroll
    for (int i = 0; i < S; ++i) to[i] = read<XT, VEC>(rows, d, (i < last - begin ? i : last - begin) * step);
}
template <typename XT, int VEC, int S>
__device__ __forceinline__ void idle(uint32_t (&x)[S], const Place& q, int first, float value) {
    if (first + S <= q.lim) return;
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = value;
    const uint32_t word = word_of<XT, VEC>(v);
#pragma unroll
    for (int i = 0; i < S; ++i)
        if (first + i >= q.lim) x[i] = word;
}
// What a gate is where a step does not count: a = 1 and nothing enters.
template <bool LEAKY> constexpr float kIdleGate = LEAKY ? INFINITY : 1.0f;

template <typename XT, int VEC, int S>
__device__ __forceinline__ void store(const Output& to, const Place& q, int first, int T, const uint32_t (&y)[S]) {
    const auto rows = rows_at(to.p, to.step, to.row, q, first, sizeof(XT));
    const int step = static_cast<int>(to.step) * static_cast<int>(sizeof(XT)), d = lane_bytes(q, sizeof(XT));
    if (first + S <= q.lim) {
#pragma unroll
        for (int i = 0; i < S; ++i) write<XT, VEC>(rows, y[i], d, i * step);
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (first + i < T) write<XT, VEC>(rows, first + i < q.lim ? y[i] : 0u, d, i * step);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Relay: a tile publishes its (A, H), takes the value that enters it from the tiles in front of it in the order of the scan, and publishes
// the value behind it. Each word says by itself whether it is known, so that relaxed accesses of the agent's scope are enough.
// Every wait ends whatever else shares the chip: a tile waits only for tiles that were handed out before it, and of those that are not done the one
// handed out first waits for none, since all before it have published their value. (A workgroup takes its next tile while its last one may still wait, so
// that a tile handed out need not have published anything yet.)
// ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t plain_bits(float v) { return v != v ? 0x7fc00000u : __float_as_uint(v); }      // never all ones

// One channel a lane; `cell` < 0: none. A tile whose runs have to be taken in turn publishes no (A, H): those behind it wait for its value, which
// `relay_value` publishes once the runs are done.
__device__ __forceinline__ void relay_value(const Args& p, int64_t cell, int order, float behind) {
    if (cell < 0) return;
    if (order == p.tiles - 1) p.state_out[cell] = behind;
    else __hip_atomic_store(p.values + order * (static_cast<int64_t>(p.N) * p.D) + cell, plain_bits(behind), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool STARTS>
__device__ __forceinline__ float relay(const Args& p, int64_t cell, int order, float A, float H, bool in_turn) {
    const int64_t cells = static_cast<int64_t>(p.N) * p.D;
    const bool active = cell >= 0, last = order == p.tiles - 1;
    uint64_t* runs = p.runs + order * cells + cell;
    uint32_t* values = p.values + order * cells + cell;
    if (active && !last && !in_turn)
        __hip_atomic_store(runs, static_cast<uint64_t>(plain_bits(A)) << 32 | plain_bits(H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    float from = active && p.state != nullptr ? p.state[cell] : 0.0f;
    if (order > 0) {
        const int reach = order < kReach ? order : kReach;
        uint64_t run[kReach];
        uint32_t value[kReach];
        int found;                      // tiles whose (A, H) lie between the value found and this tile
        for (;;) {
            found = -1;
            if (active) {
#pragma unroll
                for (int i = 0; i < kReach; ++i) {
                    const int64_t back = (i < reach ? i + 1 : reach) * cells;
                    run[i] = __hip_atomic_load(runs - back, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    value[i] = __hip_atomic_load(values - back, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            bool chained = true;        // every tile up to here has published its (A, H)
#pragma unroll
            for (int i = 0; i < kReach; ++i) {
                const bool all_value = __all(!active || value[i] != ~0u), all_run = __all(!active || run[i] != ~0ull);
                if (chained && found < 0 && i < reach && all_value) found = i;
                chained = chained && (i >= reach || all_run);
            }
            if (found < 0 && chained && order <= kReach) found = reach;         // all the way to the start
            if (found >= 0) break;
            __builtin_amdgcn_s_sleep(1);
        }
#pragma unroll
        for (int i = kReach - 1; i >= 0; --i) {
            if (i == found && i < reach) from = __uint_as_float(value[i]);
            if (i < found) from = link<STARTS>(__uint_as_float(static_cast<uint32_t>(run[i] >> 32)), from, __uint_as_float(static_cast<uint32_t>(run[i])));
        }
    }
    if (!in_turn) relay_value(p, cell, order, link<STARTS>(A, from, H));
    return from;
}

__global__ __launch_bounds__(256) void unknown_kernel(uint4* p, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) p[i] = uint4{~0u, ~0u, ~0u, ~0u};
}

// ------------------------------------------------------------------------------------------------------------------
// Steps of one wave
// ------------------------------------------------------------------------------------------------------------------
template <typename XT, int VEC, int S, bool LEAKY>
__device__ __forceinline__ void decode(const uint32_t (&g)[S], float (&a)[S][VEC], float (&rest)[S][VEC]) {
    if constexpr (LEAKY) {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) leak<kPrecise<XT>>(element<XT>(g[i], j), a[i][j], rest[i][j]);
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                a[i][j] = element<XT>(g[i], j);
                rest[i][j] = 1.0f - a[i][j];
            }
    }
}

// The same bits, of which the compiler knows nothing.
template <int S>
__device__ __forceinline__ void again(uint32_t (&x)[S]) {
#pragma unroll
    for (int i = 0; i < S; ++i) asm("" : "+v"(x[i]));
}

// The value that enters step i of a run whose bit says whether it is dropped.
template <bool STARTS>
__device__ __forceinline__ float kept(uint32_t drop, int i, float v) { return STARTS && (drop >> i & 1u) ? 0.0f : v; }

// A of the run and H: what it makes of 0.
template <int VEC, int S, bool STARTS, bool LEAKY>
__device__ __forceinline__ void reduce(const float (&a)[S][VEC], const float (&b)[S][VEC], const float (&c)[VEC], uint32_t drop, float (&A)[VEC], float (&H)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, H[j] = 0.0f;
    float least[VEC], most[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) least[j] = 1.0f, most[j] = 1.0f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            H[j] = fmaf(a[i][j], kept<STARTS>(drop, i, H[j]), b[i][j]);
            A[j] *= a[i][j];
            if constexpr (!LEAKY) most[j] = fmaxf(most[j], fabsf(a[i][j]));
        }
    if constexpr (!LEAKY) {
        if (__any(A[0] == 0.0f || A[VEC - 1] == 0.0f)) {       // seldom
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) least[j] = fminf(least[j], fabsf(a[i][j]));
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = run_of<STARTS>(most[j] > 1.0f ? kInTurn : left_over<LEAKY>(A[j], c[j], least[j]), drop != 0);
}

// Whether a run of the tile has to be taken in its turn.
template <int W>
__device__ __forceinline__ bool any_turn(const bool* turns) { return __any(turns[(threadIdx.x & 63) % W]); }
__device__ __forceinline__ void say_turn(bool* turns, int wave, bool turn) {
    turn = __any(turn);
    if ((threadIdx.x & 63) == 0) turns[wave] = turn;
}

// The W runs of a tile as one: A in row `w * rows`, H `second` rows behind it.
template <int W, bool STARTS, bool LEAKY>
__device__ __forceinline__ void join(float (*links)[64], int rows, int second, bool reversed, float& A, float& H) {
    const int lane = threadIdx.x & 63;
    float c = 0.0f, least = 1.0f;
    bool drops = false;
    A = 1.0f, H = 0.0f;
#pragma unroll 4
    for (int i = 0; i < W; ++i) {
        const int w = reversed ? W - 1 - i : i;
        const float Aw = links[w * rows][lane];
        H = link<STARTS>(Aw, H, links[w * rows + second][lane]);
        A *= Aw;
        c = fmaf(1.0f - Aw, 1.0f - c, c);
        if constexpr (!LEAKY) least = fminf(least, fabsf(Aw));
        drops = drops || dropped<STARTS>(Aw);
    }
    A = run_of<STARTS>(left_over<LEAKY>(A, c, least), drops);
}

// ------------------------------------------------------------------------------------------------------------------
// A tile in the hands of its W waves. Forward: read, reduce, and with the value that enters the wave's run, write.
// ------------------------------------------------------------------------------------------------------------------
template <typename XT, int VEC, int W, int S, bool STARTS, bool LEAKY>
struct ForwardTile {
    static constexpr int kParts = 2;
    static constexpr bool kLeaky = LEAKY;
    uint32_t g[S], x[S];
    uint8_t start;
    float a[S][VEC], b[S][VEC], c[VEC];
    uint32_t drop;                         // bit i: the state is dropped before step i of the run

    __device__ __forceinline__ static int at(const Args&, int order) { return order * W * S; }
    __device__ __forceinline__ void fetch_tile(const Args& p, const Place& q, int t0, int wave) {
        const int first = t0 + wave * S;
        fetch<XT, VEC, S>(g, p.gate, q, first);
        fetch<XT, VEC, S>(x, p.x, q, first);
        if constexpr (STARTS) start = start_of(p, q.n, first, q.lim, S);
    }
    __device__ __forceinline__ void decode_tile(const Place& q, int t0, int wave) {
        const int first = t0 + wave * S;
        idle<XT, VEC, S>(g, q, first, kIdleGate<LEAKY>);
        idle<XT, VEC, S>(x, q, first, 0.0f);
        float rest[S][VEC];
        decode<XT, VEC, S, LEAKY>(g, a, rest);
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) b[i][j] = LEAKY ? rest[i][j] * element<XT>(x[i], j) : element<XT>(x[i], j);
        drop = 0;
        if constexpr (STARTS) drop = static_cast<uint32_t>(__ballot(start != 0));
        if constexpr (W > 1) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) c[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) c[j] = fmaf(rest[i][j], 1.0f - c[j], c[j]);
        }
    }
    __device__ __forceinline__ void reduce_tile(float (*links)[64], bool* turns, int wave) {
        const int lane = threadIdx.x & 63;
        float A[VEC], H[VEC];
        reduce<VEC, S, STARTS, LEAKY>(a, b, c, drop, A, H);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            links[wave * 2 * VEC + j][lane] = A[j];
            links[(wave * 2 + 1) * VEC + j][lane] = H[j];
        }
        if constexpr (!LEAKY) say_turn(turns, wave, A[0] == kInTurn || A[VEC - 1] == kInTurn);
    }
    // What enters the run besides the value that travels: nothing.
    struct Entering {};
    __device__ __forceinline__ Entering entering(float (*)[64], int) const { return {}; }
    static constexpr int kTurns = 1;
    // v: the value that enters the run, then the one behind it
    __device__ __forceinline__ void step(int, float (&v)[VEC]) const {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = fmaf(a[i][j], kept<STARTS>(drop, i, v[j]), b[i][j]);
    }
    __device__ __forceinline__ void write_tile(const Args& p, const Place& q, int t0, int wave, Entering, float (&v)[VEC]) {
        const int first = t0 + wave * S;
        if (p.marks != nullptr && q.active && first % p.span == 0 && first < p.T) {
            float* mark = p.marks + static_cast<int64_t>(first / p.span) * p.N * p.D + q.cell;
#pragma unroll
            for (int j = 0; j < VEC; ++j) mark[j] = v[j];
        }
        uint32_t y[S];
#pragma unroll
        for (int i = 0; i < S; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = fmaf(a[i][j], kept<STARTS>(drop, i, v[j]), b[i][j]);
            y[i] = word_of<XT, VEC>(v);
        }
        store<XT, VEC, S>(p.h, q, first, p.T, y);
    }
    // Waves whose runs the value passes before it reaches wave `wave`.
    __device__ __forceinline__ static int passes(int wave) { return wave; }
    __device__ __forceinline__ static int wave_at(int k) { return k; }
};

// Backward, from the last tile to the first: the value that travels is the gradient, and h comes from the tile's mark.
template <typename XT, int VEC, int W, int S, bool STARTS, bool LEAKY>
struct BackwardTile {
    static constexpr int kParts = 3;       // A, R, H
    static constexpr bool kLeaky = LEAKY;
    uint32_t g[S], x[S], dh[S], xs[S], es[S];
    float next_mark[VEC], mark[VEC];
    uint8_t start;
    float a[S][VEC], rest[S][VEC];
    float A[VEC], H[VEC], R[VEC];
    uint32_t drop;

    __device__ __forceinline__ static int at(const Args& p, int order) { return (p.tiles - 1 - order) * W * S; }
    __device__ __forceinline__ void fetch_tile(const Args& p, const Place& q, int t0, int wave) {
        const int first = t0 + wave * S;
        fetch<XT, VEC, S>(g, p.gate, q, first);
        fetch<XT, VEC, S>(dh, p.dh, q, first);
        fetch<XT, VEC, S>(x, p.x, q, first);
        if constexpr (STARTS) start = start_of(p, q.n, first, q.lim, S);
        const float* from = p.marks + static_cast<int64_t>(t0 / p.span) * p.N * p.D + q.cell;
#pragma unroll
        for (int j = 0; j < VEC; ++j) next_mark[j] = q.active ? from[j] : 0.0f;
    }
    __device__ __forceinline__ float in(int i, int j) const { return LEAKY ? rest[i][j] * element<XT>(xs[i], j) : element<XT>(xs[i], j); }
    __device__ __forceinline__ void decode_tile(const Place& q, int t0, int wave) {
        const int first = t0 + wave * S;
        idle<XT, VEC, S>(g, q, first, kIdleGate<LEAKY>);
        idle<XT, VEC, S>(x, q, first, 0.0f);
        idle<XT, VEC, S>(dh, q, first, 0.0f);
        decode<XT, VEC, S, LEAKY>(g, a, rest);
        drop = 0;
        if constexpr (STARTS) drop = static_cast<uint32_t>(__ballot(start != 0));
        float b[S][VEC], c[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) mark[j] = next_mark[j], c[j] = 0.0f, R[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            xs[i] = x[i], es[i] = dh[i];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                b[i][j] = in(i, j);
                c[j] = fmaf(rest[i][j], 1.0f - c[j], c[j]);
            }
        }
        reduce<VEC, S, STARTS, LEAKY>(a, b, c, drop, A, H);
#pragma unroll
        for (int i = S - 1; i >= 0; --i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) R[j] = kept<STARTS>(drop, i, a[i][j] * (R[j] + element<XT>(es[i], j)));
        // From here on the elements are taken apart anew: kept apart, they would double the registers of the wait.
        again<S>(xs);
        again<S>(es);
    }
    __device__ __forceinline__ void reduce_tile(float (*links)[64], bool* turns, int wave) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            links[wave * 3 * VEC + j][lane] = A[j];
            links[(wave * 3 + 1) * VEC + j][lane] = R[j];
            links[(wave * 3 + 2) * VEC + j][lane] = H[j];
        }
        if constexpr (!LEAKY) say_turn(turns, wave, A[0] == kInTurn || A[VEC - 1] == kInTurn);
    }
    // h that enters the run
    struct Entering {
        float h[VEC];
    };
    __device__ __forceinline__ Entering entering(float (*links)[64], int wave) const {
        const int lane = threadIdx.x & 63;
        Entering e;
#pragma unroll
        for (int j = 0; j < VEC; ++j) e.h[j] = mark[j];
#pragma unroll 4
        for (int w = 0; w < wave; ++w) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) e.h[j] = link<STARTS>(links[w * 3 * VEC + j][lane], e.h[j], links[(w * 3 + 2) * VEC + j][lane]);
        }
        return e;
    }
    // Turn 0: the gradient, from the last step to the first; turn 1: h.
    static constexpr int kTurns = 2;
    __device__ __forceinline__ void step(int turn, float (&v)[VEC]) const {
        if (turn == 0) {
#pragma unroll
            for (int i = S - 1; i >= 0; --i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = kept<STARTS>(drop, i, a[i][j] * (v[j] + element<XT>(es[i], j)));
        } else {
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = fmaf(a[i][j], kept<STARTS>(drop, i, v[j]), in(i, j));
        }
    }
    __device__ __forceinline__ void write_tile(const Args& p, const Place& q, int t0, int wave, const Entering& e, float (&v)[VEC]) {
        const int first = t0 + wave * S;
        float h[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[j] = e.h[j];
        float before[S][VEC];
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                before[i][j] = kept<STARTS>(drop, i, h[j]);
                h[j] = fmaf(a[i][j], before[i][j], in(i, j));
            }
        uint32_t ox[S], og[S];
#pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            float gx[VEC], gg[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float s = v[j] + element<XT>(es[i], j);
                v[j] = kept<STARTS>(drop, i, a[i][j] * s);
                gx[j] = LEAKY ? s * rest[i][j] : s;
                gg[j] = LEAKY ? gx[j] * (a[i][j] * (before[i][j] - element<XT>(xs[i], j))) : s * before[i][j];
            }
            ox[i] = word_of<XT, VEC>(gx);
            og[i] = word_of<XT, VEC>(gg);
        }
        store<XT, VEC, S>(p.dx, q, first, p.T, ox);
        store<XT, VEC, S>(p.dgate, q, first, p.T, og);
    }
    __device__ __forceinline__ static int passes(int wave) { return W - 1 - wave; }
    __device__ __forceinline__ static int wave_at(int k) { return W - 1 - k; }
};

// The runs of a tile one after the other: in `enter` the value that enters this wave's, in v first the one that enters the tile, then the one behind it.
// With two buffers in turn a round costs one barrier. All threads of the workgroup call it, those of other waves with `wave` < 0.
template <typename Tile, int VEC, int W>
__device__ __forceinline__ void take_turns(Tile& tile, int wave, float (*passed)[VEC][64], float (&v)[VEC], float (&enter)[VEC], typename Tile::Entering& e) {
    static_assert(W % 2 == 0);          // the last round leaves the first buffer free
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int k = 0; k < W; ++k) {
        if (wave >= 0 && k == Tile::passes(wave)) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) enter[j] = v[j];
            tile.step(0, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) passed[k & 1][j][lane] = v[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = passed[k & 1][j][lane];
    }
    if constexpr (Tile::kTurns == 2) {
        float h[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[j] = tile.mark[j];
#pragma unroll 1
        for (int k = 0; k < W; ++k) {
            if (k == wave) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) e.h[j] = h[j];
                tile.step(1, h);
#pragma unroll
                for (int j = 0; j < VEC; ++j) passed[k & 1][j][lane] = h[j];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VEC; ++j) h[j] = passed[k & 1][j][lane];
        }
    }
}

// A workgroup to a column, from tile to tile.
template <typename Tile, int VEC, int W, bool STARTS>
__global__ __launch_bounds__(64 * W) void walk_kernel(Args p) {
    constexpr int kRows = Tile::kParts * VEC;
    __shared__ float links[2][W * kRows][64];
    __shared__ float passed[Tile::kLeaky ? 1 : 2][VEC][64];
    __shared__ bool turns[2][W];
    const uint32_t column = group_index();
    if (column >= static_cast<uint32_t>(p.columns)) return;
    const Place q = place<VEC>(p, column);
    const int lane = threadIdx.x & 63, wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    Tile tile;
    int t0 = Tile::at(p, 0);
    tile.fetch_tile(p, q, t0, wave);
    float v[VEC];                       // the value that enters the tile
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = q.active && p.state != nullptr ? p.state[q.cell + j] : 0.0f;
    for (int order = 0; order < p.tiles; ++order) {
        tile.decode_tile(q, t0, wave);
        const int now = t0;
        if (order + 1 < p.tiles) {
            t0 = Tile::at(p, order + 1);
            tile.fetch_tile(p, q, t0, wave);
        }
        float(*const shared)[64] = links[order & 1];
        if constexpr (W > 1) {
            tile.reduce_tile(shared, turns[order & 1], wave);
            __syncthreads();
            float enter[VEC];
            typename Tile::Entering e;
            if (Tile::kLeaky || !any_turn<W>(turns[order & 1])) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) enter[j] = v[j];
#pragma unroll 4
                for (int k = 0; k < W; ++k) {
                    if (k == Tile::passes(wave)) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) enter[j] = v[j];
                    }
                    const int w = Tile::wave_at(k);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] = link<STARTS>(shared[w * kRows + j][lane], v[j], shared[w * kRows + VEC + j][lane]);
                }
                e = tile.entering(shared, wave);
            } else {
                take_turns<Tile, VEC, W>(tile, wave, passed, v, enter, e);
            }
            tile.write_tile(p, q, now, wave, e, enter);
        } else {
            tile.write_tile(p, q, now, 0, tile.entering(shared, 0), v);
        }
    }
    if (q.active && wave == 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.state_out[q.cell + j] = v[j];
    }
}

// Workgroups that take tiles as they come, W waves for the elements and VEC more that relay: while those wait for the tiles in front, the
// others read the next tile.
template <typename Tile, int VEC, int W, bool STARTS>
__global__ __launch_bounds__(64 * (W + VEC)) void relay_kernel(Args p) {
    constexpr int kRows = Tile::kParts * VEC;
    __shared__ float links[2][W * kRows][64];
    __shared__ float values[VEC][64];
    __shared__ uint32_t next_ticket;
    __shared__ float passed[Tile::kLeaky ? 1 : 2][VEC][64];
    __shared__ bool turns[2][W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t total = static_cast<uint32_t>(p.tiles) * static_cast<uint32_t>(p.columns);
    if (threadIdx.x == 64 * W) next_ticket = atomicAdd(p.ticket, 1u) + 1u;
    __syncthreads();
    uint32_t ticket = __builtin_amdgcn_readfirstlane(next_ticket);
    __syncthreads();                    // before the next one is written
    int buffer = 0;
    if (wave >= W) {
        while (ticket < total) {
            if (threadIdx.x == 64 * W) next_ticket = atomicAdd(p.ticket, 1u) + 1u;
            const int order = ticket / p.columns, column = ticket - order * p.columns;
            const Place q = place<VEC>(p, column);
            __syncthreads();
            ticket = __builtin_amdgcn_readfirstlane(next_ticket);
            float A, H;
            join<W, STARTS, Tile::kLeaky>(&links[buffer][wave - W], kRows, VEC, Tile::wave_at(0) != 0, A, H);
            const bool turn = !Tile::kLeaky && any_turn<W>(turns[buffer]);
            const int64_t cell = q.active ? q.cell + wave - W : -1;
            values[wave - W][lane] = relay<STARTS>(p, cell, order, A, H, turn);
            buffer ^= 1;
            __syncthreads();
            if constexpr (!Tile::kLeaky) {
                if (turn) {
                    float v[VEC] = {}, enter[VEC];
                    typename Tile::Entering e;
                    Tile none;
                    take_turns<Tile, VEC, W>(none, -1, passed, v, enter, e);
                    relay_value(p, cell, order, wave == W ? v[0] : v[VEC - 1]);
                }
            }
        }
        return;
    }
    Tile tile;
    int order = ticket / p.columns;
    Place q = place<VEC>(p, ticket - order * p.columns);
    if (ticket < total) tile.fetch_tile(p, q, Tile::at(p, order), wave);
    while (ticket < total) {
        const int t0 = Tile::at(p, order);
        tile.decode_tile(q, t0, wave);
        tile.reduce_tile(links[buffer], turns[buffer], wave);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(next_ticket);
        const Place here = q;
        if (ticket < total) {
            order = ticket / p.columns;
            q = place<VEC>(p, ticket - order * p.columns);
            tile.fetch_tile(p, q, Tile::at(p, order), wave);
        }
        __syncthreads();
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = values[j][lane];
        const auto chain = [&] {
#pragma unroll 4
            for (int k = 0; k < Tile::passes(wave); ++k) {
                const int w = Tile::wave_at(k);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = link<STARTS>(links[buffer][w * kRows + j][lane], v[j], links[buffer][w * kRows + VEC + j][lane]);
            }
            return tile.entering(links[buffer], wave);
        };
        if constexpr (Tile::kLeaky) {
            const auto e = chain();
            tile.write_tile(p, here, t0, wave, e, v);
        } else {
            typename Tile::Entering e;
            if (any_turn<W>(turns[buffer])) {
                float enter[VEC];
                take_turns<Tile, VEC, W>(tile, wave, passed, v, enter, e);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = enter[j];
            } else {
                e = chain();
            }
            tile.write_tile(p, here, t0, wave, e, v);
        }
        buffer ^= 1;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Which variant
// ------------------------------------------------------------------------------------------------------------------
struct Shape {
    bool relay;
    int waves, steps;
    int tile() const { return waves * steps; }
};

// Relay where columns of 64 * VEC channels are fewer than three quarters of the compute units, and the sequence longer than its way through
// memory pays for (bf16: 4096 steps, 128 columns, walk 152 us, relay 107; 256 columns 83 and 104; 32 columns, 300 steps 11.3 and 11.6, 600 steps
// 21.2 and 12.4). The rule goes by what the forward and the backward pass both know, not by alignment: marks lie where backward tiles begin. It counts
// columns as if every lane had a channel, which sequences of few channels that starts or lengths keep apart do not come to.
Shape shape_of(int T, int N, int D, int dtype, bool backward) {
    const int units = compute_units();
    const int64_t columns = static_cast<int64_t>(N) * D / (dtype == SNNF_F32 ? 64 : 128);
    if (!backward && T == 1) return {false, 1, 1};
    if (!backward && T <= kWalkSteps) return {false, 1, kWalkSteps};
    if (T > 256 && columns * 4 < units * 3) return {true, kRelayWaves, backward ? kRelayBackSteps : kRelaySteps};
    return {false, columns < units * 4 ? kWalkWaves : kWalkWavesMany, kWalkSteps};
}
int64_t tiles_of(int T, const Shape& s) { return (static_cast<int64_t>(T) + s.tile() - 1) / s.tile(); }

// [ticket, in 64 bytes][tile][N * D] runs [tile][N * D] values
size_t workspace_of(int T, int N, int D, int dtype, bool backward) {
    const Shape s = shape_of(T, N, D, dtype, backward);
    if (!s.relay) return 0;
    const size_t words = static_cast<size_t>(tiles_of(T, s)) * N * D * (sizeof(uint64_t) + sizeof(uint32_t));
    return (words + 15) / 16 * 16 + 64;
}

template <typename XT, int VEC, bool STARTS, bool LEAKY, int W, int S>
void walk(const Args& p, bool backward, hipStream_t stream) {
    const dim3 grid = grid_of(p.columns), block(64 * W);
    if constexpr (W > 1) {
        if (backward) {
            walk_kernel<BackwardTile<XT, VEC, W, S, STARTS, LEAKY>, VEC, W, STARTS><<<grid, block, 0, stream>>>(p);
            return;
        }
    }
    walk_kernel<ForwardTile<XT, VEC, W, S, STARTS, LEAKY>, VEC, W, STARTS><<<grid, block, 0, stream>>>(p);
}

template <typename XT, int VEC, bool STARTS, bool LEAKY>
int pick(Args& p, bool backward, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    constexpr int dtype = dtype_of<XT>::value;
    const char* const name = backward ? "snnf_gated_recurrence_backward" : "snnf_gated_recurrence";
    const Shape s = shape_of(p.T, p.N, p.D, dtype, backward);
    p.groups = (p.D + 64 * VEC - 1) / (64 * VEC);
    const int64_t columns = static_cast<int64_t>(p.N) * p.groups, tiles = tiles_of(p.T, s);
    if (columns * (s.relay ? tiles : 1) > 0x7fffffffLL) return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: T=%d N=%d D=%d", name, p.T, p.N, p.D);
    p.columns = static_cast<int>(columns);
    p.tiles = static_cast<int>(tiles);
    p.span = shape_of(p.T, p.N, p.D, dtype, true).tile();
    if (s.relay) {
        const size_t need = workspace_of(p.T, p.N, p.D, dtype, backward);
        if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
            return fail(SNNF_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", name, need, workspace_bytes);
        p.ticket = static_cast<uint32_t*>(workspace);
        p.runs = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + 64);
        p.values = reinterpret_cast<uint32_t*>(p.runs + static_cast<size_t>(tiles) * p.N * p.D);
        const int64_t words = static_cast<int64_t>(need / 16), fill = (words + 255) / 256;
        unknown_kernel<<<dim3(static_cast<unsigned>(fill < 2048 ? fill : 2048)), dim3(256), 0, stream>>>(static_cast<uint4*>(workspace), words);
        // One workgroup to a compute unit: a second one, with half the steps to a tile, doubles the trips through memory.
        const int64_t units = compute_units();
        const dim3 grid(static_cast<unsigned>(columns * tiles < units ? columns * tiles : units)), block(64 * (kRelayWaves + VEC));
        if (backward) relay_kernel<BackwardTile<XT, VEC, kRelayWaves, kRelayBackSteps, STARTS, LEAKY>, VEC, kRelayWaves, STARTS><<<grid, block, 0, stream>>>(p);
        else relay_kernel<ForwardTile<XT, VEC, kRelayWaves, kRelaySteps, STARTS, LEAKY>, VEC, kRelayWaves, STARTS><<<grid, block, 0, stream>>>(p);
    } else if (s.waves == kWalkWaves) {
        walk<XT, VEC, STARTS, LEAKY, kWalkWaves, kWalkSteps>(p, backward, stream);
    } else if (s.waves == kWalkWavesMany) {
        walk<XT, VEC, STARTS, LEAKY, kWalkWavesMany, kWalkSteps>(p, backward, stream);
    } else if (s.steps == 1) {
        walk<XT, VEC, STARTS, LEAKY, 1, 1>(p, false, stream);
    } else {
        walk<XT, VEC, STARTS, LEAKY, 1, kWalkSteps>(p, false, stream);
    }
    return check_launch(name);
}

template <typename XT, int VEC>
int launch(Args& p, bool leaky, bool backward, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (leaky)
        return p.starts != nullptr ? pick<XT, VEC, true, true>(p, backward, workspace, workspace_bytes, stream)
                                   : pick<XT, VEC, false, true>(p, backward, workspace, workspace_bytes, stream);
    return p.starts != nullptr ? pick<XT, VEC, true, false>(p, backward, workspace, workspace_bytes, stream)
                               : pick<XT, VEC, false, false>(p, backward, workspace, workspace_bytes, stream);
}

bool pairs_fit(const void* p, int64_t step, int64_t row) { return aligned_to(p, 4) && step % 2 == 0 && row % 2 == 0; }

int dispatch(Args& p, int dtype, bool leaky, bool backward, void* workspace, size_t workspace_bytes, void* stream) {
    if (p.T > kMostSteps) return fail(SNNF_ERR_UNSUPPORTED, "snnf_gated_recurrence: unsupported_temporal_length: at most %d steps, got %d", kMostSteps, p.T);
    const int64_t size = dtype_size(dtype), run = p.T < kRelaySteps ? p.T : kRelaySteps;
    for (int64_t* step : {&p.x.step, &p.gate.step, &p.dh.step, &p.h.step, &p.dx.step, &p.dgate.step}) {
        if (p.T == 1) *step = 0;        // what the stride of a single step is says nothing
        if (*step < 0 || *step > kBufferBytes || (*step * (run - 1) + p.D) * size >= kBufferBytes)
            return fail(SNNF_ERR_UNSUPPORTED, "snnf_gated_recurrence: unsupported_stride: %d steps of %lld elements pass 2 GiB", static_cast<int>(run), (long long)*step);
    }
    // Sequences that lie next to each other at every step, with nothing that tells them apart, are one of more channels: few channels leave most
    // lanes of a wave idle (1024 x 256 x 40 bf16 forward 35 -> 23 us, backward 63 -> 35; 512 x 64 x 24 11.8 -> 11.0 and 17.1 -> 11.8).
    const int64_t wide = static_cast<int64_t>(p.N) * p.D;
    bool one = p.N > 1 && p.starts == nullptr && p.lengths == nullptr && wide <= (1 << 30);
    for (const auto& [step, row] : {std::pair(p.x.step, p.x.row), std::pair(p.gate.step, p.gate.row),
                                    backward ? std::pair(p.dh.step, p.dh.row) : std::pair(p.h.step, p.h.row),
                                    backward ? std::pair(p.dx.step, p.dx.row) : std::pair(p.h.step, p.h.row),
                                    backward ? std::pair(p.dgate.step, p.dgate.row) : std::pair(p.h.step, p.h.row)})
        one = one && row == p.D && (step * (run - 1) + wide) * size < kBufferBytes;
    if (one) p.D = static_cast<int>(wide), p.N = 1;
    // Two 16-bit channels to a lane where rows allow 4-byte accesses.
    bool pairs = dtype != SNNF_F32 && p.D % 2 == 0 && p.D > 64 && pairs_fit(p.x.p, p.x.step, p.x.row) && pairs_fit(p.gate.p, p.gate.step, p.gate.row);
    if (backward)
        pairs = pairs && pairs_fit(p.dh.p, p.dh.step, p.dh.row) && pairs_fit(p.dx.p, p.dx.step, p.dx.row) && pairs_fit(p.dgate.p, p.dgate.step, p.dgate.row);
    else
        pairs = pairs && pairs_fit(p.h.p, p.h.step, p.h.row);
    hipStream_t hs = as_stream(stream);
    if (dtype == SNNF_F32) return launch<float, 1>(p, leaky, backward, workspace, workspace_bytes, hs);
    if (dtype == SNNF_BF16)
        return pairs ? launch<bf16_t, 2>(p, leaky, backward, workspace, workspace_bytes, hs) : launch<bf16_t, 1>(p, leaky, backward, workspace, workspace_bytes, hs);
    return pairs ? launch<f16_t, 2>(p, leaky, backward, workspace, workspace_bytes, hs) : launch<f16_t, 1>(p, leaky, backward, workspace, workspace_bytes, hs);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" size_t snnf_gated_recurrence_workspace_bytes(int T, int N, int D, int dtype, int backward) {
    if (T < 1 || N < 1 || D < 1 || !valid_dtype(dtype)) return 0;
    return workspace_of(T, N, D, dtype, backward != 0);
}

extern "C" size_t snnf_gated_recurrence_marks_bytes(int T, int N, int D, int dtype) {
    if (T < 1 || N < 1 || D < 1 || !valid_dtype(dtype)) return 0;
    return static_cast<size_t>(tiles_of(T, shape_of(T, N, D, dtype, true))) * N * D * sizeof(float);
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
    if (state == state_out) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence: state and state_out must not be the same memory");
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
    return dispatch(p, dtype, form == SNNF_RECURRENCE_LEAKY, false, workspace, workspace_bytes, stream);
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
    if (dstate == dstate_in) return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_gated_recurrence_backward: dstate and dstate_in must not be the same memory");
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
    return dispatch(p, dtype, form == SNNF_RECURRENCE_LEAKY, true, workspace, workspace_bytes, stream);
}
