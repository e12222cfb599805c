// Norm of a block's output, its gate and scale, residual addition and the norm in front of the next block, and their gradient.
//     y = norm(branch) * branch_weight;   residual' = residual + factor * scale * act(gate) * y;   normed = norm(residual') * next_weight
// norm takes the mean out (LAYER) or not and divides by sqrt(mean of squares + eps); without a branch residual' is the residual. With unit = the
// divided row and r = 1 / sqrt(...), the gradient through a norm is r * (d - unit * mean(d * unit) [- mean(d)]).
// A row lies in the registers of P threads (8 elements each, 16 where rows pass 4096), so that every tensor is read once; its statistics are
// sums over them, and the backward pass reads the row statistics that the forward pass leaves. What a program's vectors get as gradients is
// summed over the rows a workgroup takes in registers, and over the workgroups by a second kernel, in a fixed order.
// Bound by memory: 5 tensors forward, 8 backward (32768 x 2048 bf16, gated: 128 us, 5.2 TB/s, and 224 us, 4.8 TB/s); few rows by the sums over
// workgroups (1000 x 1024 bf16: 4.6 and 14.6 us).
#include <type_traits>

#include "snnf_sequence.h"

namespace snnf {
namespace {

constexpr int kMostWidth = 16384;
constexpr int kPhases = 16;             // threads to a column in the sum over workgroups

struct Rows {
    const void* p;
    int64_t row;                        // elements from one row to the next
};

struct NormArgs {
    Rows residual, branch, gate, d_residual_out, d_normed;
    const void *branch_weight, *next_weight, *scale;
    void *residual_out, *normed;        // rows next to each other, as those of the gradients
    void *d_residual, *d_branch, *d_gate;
    float4* stats;                      // mean and 1 / sqrt of the branch, of residual'
    float* parts;                       // [part][3][D] gradients of branch_weight, next_weight, scale over the rows of a part
    int64_t rows;
    int D, per_row;                     // threads to a row
    int gate_form;
    float factor, eps;
};

template <typename T, int VEC>
__device__ __forceinline__ void save(void* base, int64_t at, int left, const float (&v)[VEC]) {
    Raw<T, VEC> raw;
#pragma unroll
    for (int j = 0; j < VEC; j += 2) raw.put(j, v[j], v[j + 1]);
    raw.store(base, at, left);
}

// What the gate lets through, and its slope. No gate is a sigmoid's at infinity: 1, and 0.
template <typename T>
__device__ __forceinline__ void gate_of(bool silu, float g, float& act, float& slope) {
    float s, rest;
    leak<kPrecise<T>>(g, s, rest);
    const float from = __builtin_elementwise_maximum(g, -86.0f);        // a gate at the type's lowest value lets nothing through
    act = s * (silu ? from : 1.0f);
    slope = s * (silu ? fmaf(__builtin_elementwise_minimum(from, 200.0f), rest, 1.0f) : rest);
}
template <typename T, int VEC>
__device__ __forceinline__ void open_gate(Raw<T, VEC>& g) {
#pragma unroll
    for (int i = 0; i < Raw<T, VEC>::kWords; ++i) {
        if constexpr (sizeof(T) == 4) g.w[i] = __float_as_uint(INFINITY);
        else g.w[i] = pair_word<T>(INFINITY, INFINITY);
    }
}
// Elements are worked out two at a time: all at once would hold more than the registers that are left.
#define SNNF_ELEMENT_DONE(j) \
    if ((j) % 2 == 1) __builtin_amdgcn_sched_barrier(0)

// Sums over the threads of a row: over the lanes of a wave, or of a part of one, and where a row takes several waves through LDS, two buffers in
// turn so that a sum costs one barrier. Always in the same order.
struct RowSum {
    float (*shared)[16][2];
    int lanes, waves, first_wave, wave;
    int buffer;
    template <int COUNT>
    __device__ __forceinline__ void operator()(float (&v)[COUNT]) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) v[i] = lane_sum(v[i], lanes);
        if (waves <= 1) return;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i) shared[buffer][wave][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < COUNT; ++i) v[i] = 0.0f;
        for (int w = 0; w < waves; ++w) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i) v[i] += shared[buffer][first_wave + w][i];
        }
        buffer ^= 1;
    }
};

// The thread's place in its row and its row's in the workgroup.
template <int K, int VEC>
struct Seat {
    int slots, slot, thread;
    int at[K], left[K];
    RowSum sum;
    __device__ __forceinline__ Seat(const NormArgs& p, float (*shared)[16][2]) {
        slots = blockDim.x / p.per_row;
        slot = threadIdx.x / p.per_row;
        thread = threadIdx.x - slot * p.per_row;
        const int waves = p.per_row >> 6;
        sum = RowSum{shared, p.per_row < 64 ? p.per_row : 64, waves, slot * waves, static_cast<int>(threadIdx.x >> 6), 0};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at[k] = (k * p.per_row + thread) * VEC;
            left[k] = p.D - at[k];
        }
    }
};

template <typename RT, typename XT, typename VT, int K, bool LAYER, int BLOCK>
__global__ __launch_bounds__(BLOCK) void block_norm_kernel(NormArgs p) {
    constexpr int VEC = kVec<XT>;
    __shared__ float shared[2][16][2];
    Seat<K, VEC> seat(p, shared);
    const int (&left)[K] = seat.left;
    const bool branch = p.branch.p != nullptr, gated = p.gate_form != SNNF_GATE_NONE, silu = p.gate_form == SNNF_GATE_SILU;
    const float part = 1.0f / p.D;
    Raw<VT, VEC> wb[K], wn[K], sc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        wn[k].load_vector(p.next_weight, seat.at[k], left[k]);
        wb[k].load_vector(branch ? p.branch_weight : nullptr, seat.at[k], left[k]);
        sc[k].load_vector(branch ? p.scale : nullptr, seat.at[k], left[k]);
    }
    const int64_t stride = static_cast<int64_t>(gridDim.x) * seat.slots;
    Raw<RT, VEC> r[K];
    Raw<XT, VEC> o[K], g[K];
#pragma unroll
    for (int k = 0; k < K; ++k) open_gate(g[k]);
    // The next row is on its way as soon as this one's elements are taken apart. (Slots behind the last row repeat it and write nothing.)
    const auto fetch = [&](int64_t row) {
        row = row < p.rows ? row : p.rows - 1;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (branch) o[k].load(p.branch.p, row * p.branch.row + seat.at[k], left[k]);
            if (gated) g[k].load(p.gate.p, row * p.gate.row + seat.at[k], left[k]);
            r[k].load(p.residual.p, row * p.residual.row + seat.at[k], left[k]);
        }
    };
    int64_t base = static_cast<int64_t>(blockIdx.x) * seat.slots;
    fetch(base + seat.slot);
    for (; base < p.rows; base += stride) {
        const int64_t row = base + seat.slot;
        const bool writes = row < p.rows;
        float total[K][VEC];
        float4 stats = {0.0f, 0.0f, 0.0f, 0.0f};
        if (branch) {
            if constexpr (LAYER) {
                float s[1] = {0.0f};
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) s[0] += o[k][j];
                seat.sum(s);
                stats.x = s[0] * part;
            }
            float s[1] = {0.0f};
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float v = LAYER && j >= left[k] ? 0.0f : o[k][j] - stats.x;
                    s[0] = fmaf(v, v, s[0]);
                }
            seat.sum(s);
            stats.y = 1.0f / sqrtf(s[0] * part + p.eps);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                o[k].again(), wb[k].again(), sc[k].again();
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float act, slope;
                    gate_of<XT>(silu, g[k][j], act, slope);
                    const float more = ((o[k][j] - stats.x) * stats.y * wb[k][j]) * (act * (sc[k][j] * p.factor));
                    total[k][j] = r[k][j] + (LAYER && j >= left[k] ? 0.0f : more);
                }
                if (writes) save<RT, VEC>(p.residual_out, row * p.D + seat.at[k], left[k], total[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) total[k][j] = r[k][j];
        }
        if (base + stride < p.rows) fetch(row + stride);
        if constexpr (LAYER) {
            float s[1] = {0.0f};
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[0] += total[k][j];
            seat.sum(s);
            stats.z = s[0] * part;
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                total[k][j] = LAYER && j >= left[k] ? 0.0f : total[k][j] - stats.z;
                s[0] = fmaf(total[k][j], total[k][j], s[0]);
            }
        seat.sum(s);
        stats.w = 1.0f / sqrtf(s[0] * part + p.eps);
        if (!writes) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            wn[k].again();
#pragma unroll
            for (int j = 0; j < VEC; ++j) total[k][j] = total[k][j] * stats.w * wn[k][j];
            save<XT, VEC>(p.normed, row * p.D + seat.at[k], left[k], total[k]);
        }
        if (p.stats != nullptr && seat.thread == 0) p.stats[row] = stats;
    }
}

// Sums over a workgroup's rows, of the columns that a thread owns: in LDS, each read and written by its owner (registers would cost half the
// waves: 32768 x 2048 bf16 250 -> 226 us), for the widest rows, whose sums LDS does not hold, in registers.
constexpr bool sums_in_lds(int block, int elements) { return block * elements * 3 * 4 <= 100 * 1024; }
typedef float Four __attribute__((ext_vector_type(4)));
template <int BLOCK, int ELEMENTS, bool IN_LDS = sums_in_lds(BLOCK, ELEMENTS)>
struct ColumnSums {
    static constexpr int kShared = 1;
    float v[3][ELEMENTS];
    __device__ __forceinline__ ColumnSums(Four*) {
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int e = 0; e < ELEMENTS; ++e) v[i][e] = 0.0f;
    }
    __device__ __forceinline__ void add(int i, int first, const float (&more)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][first + e] += more[e];
    }
};
template <int BLOCK, int ELEMENTS>
struct ColumnSums<BLOCK, ELEMENTS, true> {
    static constexpr int kShared = 3 * (ELEMENTS / 4) * BLOCK;         // [3][ELEMENTS / 4][BLOCK]
    Four* mine;
    __device__ __forceinline__ ColumnSums(Four* shared) : mine(shared + threadIdx.x) {
#pragma unroll
        for (int i = 0; i < 3 * (ELEMENTS / 4); ++i) mine[i * BLOCK] = Four{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void add(int i, int first, const float (&more)[4]) {
        Four& at = mine[(i * (ELEMENTS / 4) + first / 4) * BLOCK];
        at = at + Four{more[0], more[1], more[2], more[3]};
    }
};

// Elements stay as they lie in memory and are taken apart where they are needed, the gate among them twice: what a thread would have to hold
// otherwise costs the waves that cover the latency of memory.
template <typename RT, typename XT, typename VT, int K, bool LAYER, int BLOCK>
__global__ __launch_bounds__(BLOCK, BLOCK == 256 ? 3 : 1) void block_norm_backward_kernel(NormArgs p) {
    constexpr int VEC = kVec<XT>;
    __shared__ float shared[2][16][2];
    constexpr int kElements = K * VEC;
    __shared__ Four columns[ColumnSums<BLOCK, kElements>::kShared];
    ColumnSums<BLOCK, kElements> sums(columns);
    Seat<K, VEC> seat(p, shared);
    const int (&left)[K] = seat.left;
    const bool branch = p.branch.p != nullptr, gated = p.gate_form != SNNF_GATE_NONE, silu = p.gate_form == SNNF_GATE_SILU, from_out = p.d_residual_out.p != nullptr, from_normed = p.d_normed.p != nullptr;
    const float part = 1.0f / p.D;
    Raw<VT, VEC> wb[K], wn[K], sc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        wn[k].load_vector(p.next_weight, seat.at[k], left[k]);
        wb[k].load_vector(branch ? p.branch_weight : nullptr, seat.at[k], left[k]);
        sc[k].load_vector(branch ? p.scale : nullptr, seat.at[k], left[k]);
    }
    const int64_t stride = static_cast<int64_t>(gridDim.x) * seat.slots;
    Raw<RT, VEC> r[K], d_out[K];
    Raw<XT, VEC> o[K], g[K], dn[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {       // what is not there: a branch, whose statistics are 0 then, and gradients of 0
        open_gate(g[k]);
        o[k].clear(), dn[k].clear(), d_out[k].clear();
    }
    // The next row's elements are sent for as soon as this row's in their place are done with.
    const auto fetch_total = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            r[k].load(p.residual.p, row * p.residual.row + seat.at[k], left[k]);
            if (from_normed) dn[k].load(p.d_normed.p, row * p.d_normed.row + seat.at[k], left[k]);
        }
    };
    const auto fetch_gate = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (gated) g[k].load(p.gate.p, row * p.gate.row + seat.at[k], left[k]);
            if (from_out) d_out[k].load(p.d_residual_out.p, row * p.d_residual_out.row + seat.at[k], left[k]);
        }
    };
    const auto fetch_branch = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (branch) o[k].load(p.branch.p, row * p.branch.row + seat.at[k], left[k]);
    };
    const auto real = [&](int64_t row) { return row < p.rows ? row : p.rows - 1; };
    int64_t base = static_cast<int64_t>(blockIdx.x) * seat.slots;
    fetch_total(real(base + seat.slot));
    fetch_branch(real(base + seat.slot));
    fetch_gate(real(base + seat.slot));
    float4 next_stats = p.stats[real(base + seat.slot)];
    for (; base < p.rows; base += stride) {
        const int64_t row = base + seat.slot, next = real(row + stride);
        const bool writes = row < p.rows, more = base + stride < p.rows;
        const float counts = writes ? 1.0f : 0.0f;
        const float4 stats = next_stats;
        float unit2[K][VEC], d[K][VEC], s[2] = {0.0f, 0.0f};           // the unit row of the second norm, the gradient in front of its weight
#pragma unroll
        for (int k = 0; k < K; ++k) {
            wb[k].again(), wn[k].again(), sc[k].again();
            float more[4];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float act, slope;
                gate_of<XT>(silu, g[k][j], act, slope);
                const float total = r[k][j] + ((o[k][j] - stats.x) * stats.y * wb[k][j]) * (act * (sc[k][j] * p.factor));
                unit2[k][j] = LAYER && j >= left[k] ? 0.0f : (total - stats.z) * stats.w;
                more[j % 4] = dn[k][j] * counts * unit2[k][j];
                if (j % 4 == 3) sums.add(1, k * VEC + j - 3, more);
                d[k][j] = dn[k][j] * wn[k][j];
                s[0] = fmaf(d[k][j], unit2[k][j], s[0]);
                s[1] += d[k][j];
                SNNF_ELEMENT_DONE(j);
            }
        }
        if (more) fetch_total(next);
        seat.sum(s);
        s[0] *= part;
        s[1] = LAYER ? s[1] * part : 0.0f;
        float q[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[k][j] = LAYER && j >= left[k] ? 0.0f : stats.w * (d[k][j] - unit2[k][j] * s[0] - s[1]) + d_out[k][j];
            if (writes) save<RT, VEC>(p.d_residual, row * p.D + seat.at[k], left[k], d[k]);
            o[k].again(), g[k].again(), wb[k].again(), sc[k].again();
            float more_weight[4], more_scale[4], gates[2];
            Raw<XT, VEC> d_gate;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float act, slope;
                gate_of<XT>(silu, g[k][j], act, slope);
                const float unit = LAYER && j >= left[k] ? 0.0f : (o[k][j] - stats.x) * stats.y;
                const float through = d[k][j] * p.factor, y = unit * wb[k][j], du = through * sc[k][j] * act;
                more_scale[j % 4] = through * act * counts * y;
                more_weight[j % 4] = du * counts * unit;
                gates[j % 2] = through * sc[k][j] * y * slope;
                if (j % 2 == 1) d_gate.put(j - 1, gates[0], gates[1]);
                d[k][j] = du * wb[k][j];
                q[0] = fmaf(d[k][j], unit, q[0]);
                q[1] += d[k][j];
                if (j % 4 == 3) {
                    sums.add(0, k * VEC + j - 3, more_weight);
                    sums.add(2, k * VEC + j - 3, more_scale);
                }
                SNNF_ELEMENT_DONE(j);
            }
            if (gated && writes) d_gate.store(p.d_gate, row * p.D + seat.at[k], left[k]);
        }
        if (more) {
            fetch_gate(next);
            next_stats = p.stats[next];
        }
        seat.sum(q);
        q[0] *= part;
        q[1] = LAYER ? q[1] * part : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            o[k].again();
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[k][j] = stats.y * (d[k][j] - (o[k][j] - stats.x) * stats.y * q[0] - q[1]);
            if (branch && writes) save<XT, VEC>(p.d_branch, row * p.D + seat.at[k], left[k], d[k]);
        }
        if (more) fetch_branch(next);
    }
    // A workgroup's rows as one part, slot by slot.
    float* const to = p.parts + static_cast<int64_t>(blockIdx.x) * 3 * p.D;
    if constexpr (sums_in_lds(BLOCK, kElements)) {
        __syncthreads();
        for (int i = threadIdx.x; i < p.D; i += BLOCK) {
            const int chunk = i / VEC, owner = chunk % p.per_row, e = chunk / p.per_row * VEC + i % VEC;
#pragma unroll
            for (int v = 0; v < 3; ++v) {
                const float* const column = reinterpret_cast<const float*>(columns + (v * (kElements / 4) + e / 4) * BLOCK + owner) + e % 4;
                float total = 0.0f;
                for (int t = 0; t < seat.slots; ++t) total += column[t * p.per_row * 4];
                to[v * p.D + i] = total;
            }
        }
    } else {
#pragma unroll
        for (int v = 0; v < 3; ++v)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float total[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) total[j] = sums.v[v][k * VEC + j];
                save<float, VEC>(to + v * p.D, seat.at[k], left[k], total);
            }
    }
}

// Sum of the parts: 64 columns and kPhases parts at a time.
template <typename WT>
__global__ __launch_bounds__(64 * kPhases) void vector_gradient_kernel(const float* parts, int n_parts, int D, WT* d_branch_weight, WT* d_next_weight, WT* d_scale) {
    __shared__ float shared[kPhases][64];
    WT* const out = blockIdx.y == 0 ? d_branch_weight : (blockIdx.y == 1 ? d_next_weight : d_scale);
    if (out == nullptr) return;
    const int lane = threadIdx.x & 63, phase = threadIdx.x >> 6, column = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (column < D) {
#pragma unroll 8
        for (int i = phase; i < n_parts; i += kPhases) s += parts[(static_cast<int64_t>(i) * 3 + blockIdx.y) * D + column];
    }
    shared[phase][lane] = s;
    __syncthreads();
    if (phase != 0 || column >= D) return;
    for (int i = 1; i < kPhases; ++i) s += shared[i][lane];
    out[column] = from_float<WT>(s);
}

// ------------------------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------------------------
struct NormShape {
    int per_row, block, slots, chunks, grid;
};

// Threads to a row: 8 elements each up to 512 threads, 16 from there on (with 16 from 256 threads on 8192 x 4096 bf16 takes 70 us in place of 65,
// 4096 x 8192 107 in place of 63, and the backward pass no longer fits the registers). Workgroups: as many as are resident at once, which walk
// over the rows (four times as many: 8192 x 4096 65 -> 68 us forward, 131 -> 157 backward; 8192 x 2048 33 -> 31, 77 -> 86). Backward, a
// workgroup takes at least four rows to a slot where that leaves one for every compute unit: its sums over rows cost as much memory as a
// row does (1000 x 1024: 14.6 us, without 16.7; 1531 x 777 float32 19.2 and 21.0; the other way 2000 x 2048 28.3 and 25.2). Rows past 8192 take 1024 threads,
// whose 128 registers do not hold 16 elements of everything: all 18 backward kernels of that size keep up to 1032 bytes a lane in scratch memory, and 10 of the 18
// forward ones, whose vectors are float32, up to 304 (2048 x 12288 bf16 forward 67 us, of which 47 are its bytes, backward 870, of which 75 are).
NormShape norm_shape(int64_t rows, int D, bool backward, int vec) {
    NormShape s;
    s.per_row = 8;
    while (s.per_row < 512 && s.per_row * 8 < D) s.per_row *= 2;
    s.chunks = s.per_row * 8 < D ? 16 / vec : 8 / vec;
    if (s.per_row * 16 < D) s.per_row = 1024;
    s.block = s.per_row < 256 ? 256 : s.per_row;
    s.slots = s.block / s.per_row;
    const int64_t units = compute_units();
    const int64_t fit = s.block == 1024 ? 1 : (backward ? (s.block == 512 ? 1 : 3) : (s.block == 512 ? (s.chunks * vec == 8 ? 3 : 2) : 6));
    const int64_t resident = units * fit;
    int64_t grid = (rows + s.slots - 1) / s.slots;
    if (backward) {
        const int64_t few = (rows + s.slots * 4 - 1) / (s.slots * 4);
        grid = grid < units ? grid : (few < units ? units : few);
    }
    s.grid = static_cast<int>(grid < resident ? grid : resident);
    return s;
}

template <typename RT, typename XT, typename VT, int K>
void launch_norm(const NormArgs& p, const NormShape& s, bool layer, bool backward, hipStream_t stream) {
    const dim3 grid(s.grid), block(s.block);
    const auto go = [&](auto block_size) {
        constexpr int BLOCK = decltype(block_size)::value;
        if (backward) {
            if (layer) block_norm_backward_kernel<RT, XT, VT, K, true, BLOCK><<<grid, block, 0, stream>>>(p);
            else block_norm_backward_kernel<RT, XT, VT, K, false, BLOCK><<<grid, block, 0, stream>>>(p);
        } else {
            if (layer) block_norm_kernel<RT, XT, VT, K, true, BLOCK><<<grid, block, 0, stream>>>(p);
            else block_norm_kernel<RT, XT, VT, K, false, BLOCK><<<grid, block, 0, stream>>>(p);
        }
    };
    if constexpr (K * kVec<XT> == 8) {
        if (s.block == 512) go(std::integral_constant<int, 512>{});
        else go(std::integral_constant<int, 256>{});
    } else {
        if (s.block == 512) go(std::integral_constant<int, 512>{});
        else go(std::integral_constant<int, 1024>{});
    }
}

template <typename RT, typename XT, typename VT>
void launch_types(const NormArgs& p, const NormShape& s, bool layer, bool backward, hipStream_t stream) {
    constexpr int few = 8 / kVec<XT>;
    if (s.chunks == few) launch_norm<RT, XT, VT, few>(p, s, layer, backward, stream);
    else launch_norm<RT, XT, VT, 2 * few>(p, s, layer, backward, stream);
}

template <typename XT>
void launch_16(const NormArgs& p, const NormShape& s, bool wide_residual, bool wide_vectors, bool layer, bool backward, hipStream_t stream) {
    if (wide_residual) {
        if (wide_vectors) launch_types<float, XT, float>(p, s, layer, backward, stream);
        else launch_types<float, XT, XT>(p, s, layer, backward, stream);
    } else {
        if (wide_vectors) launch_types<XT, XT, float>(p, s, layer, backward, stream);
        else launch_types<XT, XT, XT>(p, s, layer, backward, stream);
    }
}

int check_norm(const char* name, int64_t rows, int D, int residual_dtype, int dtype, int vector_dtype, int kind, int gate_form, float eps) {
    if (rows < 0 || D < 1) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: rows=%lld D=%d", name, (long long)rows, D);
    if (D > kMostWidth) return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_shape: rows of at most %d elements, got %d", name, kMostWidth, D);
    if (!valid_dtype(dtype) || !valid_dtype(residual_dtype) || !valid_dtype(vector_dtype))
        return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: unknown dtype code", name);
    if ((residual_dtype != dtype && residual_dtype != SNNF_F32) || (vector_dtype != dtype && vector_dtype != SNNF_F32))
        return fail(SNNF_ERR_UNSUPPORTED, "%s: unsupported_dtype: the residual and the vectors are of the activations' type or float32", name);
    if (kind != SNNF_NORM_RMS && kind != SNNF_NORM_LAYER) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: unknown kind %d", name, kind);
    if (gate_form != SNNF_GATE_NONE && gate_form != SNNF_GATE_SIGMOID && gate_form != SNNF_GATE_SILU)
        return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: unknown gate form %d", name, gate_form);
    if (!(eps >= 0.0f)) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: eps must not be negative", name);
    return SNNF_OK;
}

int run_norm(const char* name, const NormArgs& p, int residual_dtype, int dtype, int vector_dtype, int kind, bool backward, const NormShape& s, hipStream_t stream) {
    const bool layer = kind == SNNF_NORM_LAYER, wide_residual = residual_dtype == SNNF_F32, wide_vectors = vector_dtype == SNNF_F32;
    if (dtype == SNNF_F32) launch_types<float, float, float>(p, s, layer, backward, stream);
    else if (dtype == SNNF_BF16) launch_16<bf16_t>(p, s, wide_residual, wide_vectors, layer, backward, stream);
    else launch_16<f16_t>(p, s, wide_residual, wide_vectors, layer, backward, stream);
    return check_launch(name);
}

}  // namespace
}  // namespace snnf

using namespace snnf;

extern "C" int snnf_block_norm(const void* residual, int64_t residual_row, const void* branch, int64_t branch_row, const void* gate, int64_t gate_row,
                               const void* branch_weight, const void* next_weight, const void* scale, float factor, int64_t rows, int D,
                               int residual_dtype, int dtype, int vector_dtype, int kind, int gate_form, float eps, void* residual_out, void* normed,
                               float* stats, void* stream) {
    const int rc = check_norm("snnf_block_norm", rows, D, residual_dtype, dtype, vector_dtype, kind, gate_form, eps);
    if (rc != SNNF_OK) return rc;
    if (rows == 0) return SNNF_OK;
    if (residual == nullptr || normed == nullptr || (branch != nullptr && residual_out == nullptr) || (gate_form != SNNF_GATE_NONE && (gate == nullptr || branch == nullptr)))
        return fail(SNNF_ERR_INVALID_ARGUMENT, "snnf_block_norm: residual, normed, with a branch residual_out, and a gate's operands must be non-null");
    NormArgs p = {};
    p.residual = {residual, residual_row};
    p.branch = {branch, branch_row};
    p.gate = {gate, gate_row};
    p.branch_weight = branch_weight, p.next_weight = next_weight, p.scale = scale;
    p.residual_out = residual_out, p.normed = normed;
    p.stats = reinterpret_cast<float4*>(stats);
    p.rows = rows, p.D = D;
    p.gate_form = gate_form;
    p.factor = factor, p.eps = eps;
    const NormShape s = norm_shape(rows, D, false, dtype == SNNF_F32 ? 4 : 8);
    p.per_row = s.per_row;
    return run_norm("snnf_block_norm", p, residual_dtype, dtype, vector_dtype, kind, false, s, as_stream(stream));
}

extern "C" size_t snnf_block_norm_backward_workspace_bytes(int64_t rows, int D) {
    if (rows < 1 || D < 1 || D > kMostWidth) return 0;
    const NormShape s = norm_shape(rows, D, true, 8);
    return static_cast<size_t>(s.grid) * 3 * D * sizeof(float);
}

extern "C" int snnf_block_norm_backward(const void* residual, int64_t residual_row, const void* branch, int64_t branch_row, const void* gate,
                                        int64_t gate_row, const void* branch_weight, const void* next_weight, const void* scale, float factor,
                                        const void* d_residual_out, int64_t d_residual_out_row, const void* d_normed, int64_t d_normed_row,
                                        const float* stats, int64_t rows, int D, int residual_dtype, int dtype, int vector_dtype, int kind,
                                        int gate_form, void* d_residual, void* d_branch, void* d_gate, void* d_branch_weight, void* d_next_weight,
                                        void* d_scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* const name = "snnf_block_norm_backward";
    const int rc = check_norm(name, rows, D, residual_dtype, dtype, vector_dtype, kind, gate_form, 0.0f);
    if (rc != SNNF_OK) return rc;
    if (rows == 0) return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: no rows", name);
    if (residual == nullptr || stats == nullptr || d_residual == nullptr || (branch != nullptr && d_branch == nullptr) ||
        (gate_form != SNNF_GATE_NONE && (gate == nullptr || branch == nullptr || d_gate == nullptr)))
        return fail(SNNF_ERR_INVALID_ARGUMENT, "%s: residual, stats and the gradients of the operands that are there must be non-null", name);
    const size_t need = snnf_block_norm_backward_workspace_bytes(rows, D);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
        return fail(SNNF_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", name, need, workspace_bytes);
    NormArgs p = {};
    p.residual = {residual, residual_row};
    p.branch = {branch, branch_row};
    p.gate = {gate, gate_row};
    p.d_residual_out = {d_residual_out, d_residual_out_row};
    p.d_normed = {d_normed, d_normed_row};
    p.branch_weight = branch_weight, p.next_weight = next_weight, p.scale = scale;
    p.d_residual = d_residual, p.d_branch = d_branch, p.d_gate = d_gate;
    p.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    p.parts = static_cast<float*>(workspace);
    p.rows = rows, p.D = D;
    p.gate_form = gate_form;
    p.factor = factor;
    const NormShape s = norm_shape(rows, D, true, dtype == SNNF_F32 ? 4 : 8);
    p.per_row = s.per_row;
    hipStream_t hs = as_stream(stream);
    const int status = run_norm(name, p, residual_dtype, dtype, vector_dtype, kind, true, s, hs);
    if (status != SNNF_OK || (d_branch_weight == nullptr && d_next_weight == nullptr && d_scale == nullptr)) return status;
    const dim3 grid((D + 63) / 64, 3), block(64 * kPhases);
    const int n_parts = s.grid;
    if (vector_dtype == SNNF_F32)
        vector_gradient_kernel<<<grid, block, 0, hs>>>(p.parts, n_parts, D, static_cast<float*>(d_branch_weight), static_cast<float*>(d_next_weight), static_cast<float*>(d_scale));
    else if (vector_dtype == SNNF_BF16)
        vector_gradient_kernel<<<grid, block, 0, hs>>>(p.parts, n_parts, D, static_cast<bf16_t*>(d_branch_weight), static_cast<bf16_t*>(d_next_weight), static_cast<bf16_t*>(d_scale));
    else
        vector_gradient_kernel<<<grid, block, 0, hs>>>(p.parts, n_parts, D, static_cast<f16_t*>(d_branch_weight), static_cast<f16_t*>(d_next_weight), static_cast<f16_t*>(d_scale));
    return check_launch(name);
}
