// Norm of a block's output, its gate and scale, residual addition and the norm in front of the next block, and their gradient.
//     y = norm(branch) * branch_weight;   residual' = residual + factor * scale * act(gate) * y;   normed = norm(residual') * next_weight
// norm takes the mean out (LAYER) or not and divides by sqrt(mean of squares + eps); without a branch residual' is the residual. With unit = the
// divided row and r = 1 / sqrt(...), the gradient through a norm is r * (d - unit * mean(d * unit) [- mean(d)]).
// A row lies in the registers of P threads (8 elements each, 16 where rows pass 8192), so that every tensor is read once; its statistics are
// sums over them, and the backward pass reads the row statistics that the forward pass leaves. What a program's vectors get as gradients is
// summed over the rows a workgroup takes in registers, and over the workgroups by a second kernel, in a fixed order.
// Bound by memory: 5 tensors forward, 8 backward.
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
    int vectors_f32;                    // the weights and the scale are float32
    float factor, eps;
};

template <typename T> constexpr int kVec = sizeof(T) == 4 ? 4 : 8;

template <typename T, int VEC>
__device__ __forceinline__ void load(float (&v)[VEC], const void* base, int64_t at, int left) {
    const T* p = static_cast<const T*>(base) + at;
    if (left >= VEC) {
        const auto w = *reinterpret_cast<const typename Words<T, VEC>::type*>(p);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (sizeof(T) == 4) v[j] = element<T>(w[j], 0);
            else v[j] = element<T>(w[j / 2], j % 2);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = j < left ? to_float(p[j]) : 0.0f;
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void save(void* base, int64_t at, int left, const float (&v)[VEC]) {
    T* p = static_cast<T*>(base) + at;
    if (left >= VEC) {
        typename Words<T, VEC>::type w;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[j] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) w[j / 2] = pair_word<T>(v[j], v[j + 1]);
        }
        *reinterpret_cast<typename Words<T, VEC>::type*>(p) = w;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < left) p[j] = from_float<T>(v[j]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void load_vector(float (&v)[VEC], const void* base, bool f32, int at, int left) {
    if (base == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 1.0f;
    } else if (f32) {
        load<float, VEC>(v, base, at, left);
    } else {
        load<T, VEC>(v, base, at, left);
    }
}

// What the gate lets through and its slope.
template <bool PRECISE>
__device__ __forceinline__ void gate_of(int form, float g, float& act, float& slope) {
    if (form == SNNF_GATE_NONE) {
        act = 1.0f, slope = 0.0f;
        return;
    }
    float s, rest;
    leak<PRECISE>(g, s, rest);
    if (form == SNNF_GATE_SIGMOID) {
        act = s, slope = s * rest;
    } else {
        const float from = __builtin_elementwise_maximum(g, -86.0f);        // a gate at the type's lowest value lets nothing through
        act = from * s;
        slope = s * fmaf(__builtin_elementwise_minimum(from, 200.0f), rest, 1.0f);
    }
}

// Sums over the threads of a row. Two buffers in turn, so that a sum costs one barrier.
struct RowSum {
    float (*shared)[16][2];
    int waves, first_wave, wave;
    int buffer;
    template <int COUNT>
    __device__ __forceinline__ void operator()(float (&v)[COUNT]) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) v[i] = wave_sum(v[i]);
        if (waves == 1) return;
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

// Takes the mean out where asked, returns it, and 1 / sqrt(mean of squares + eps).
template <bool LAYER, int K, int VEC>
__device__ __forceinline__ void whiten(float (&x)[K][VEC], const int (&left)[K], int D, float eps, RowSum& sum, float& mean, float& r) {
    mean = 0.0f;
    if constexpr (LAYER) {
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[0] += x[k][j];
        sum(s);
        mean = s[0] / D;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[k][j] = j < left[k] ? x[k][j] - mean : 0.0f;
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[0] = fmaf(x[k][j], x[k][j], s[0]);
    sum(s);
    r = 1.0f / sqrtf(s[0] / D + eps);
}

template <typename RT, typename XT, int K, bool LAYER>
__global__ __launch_bounds__(1024) void block_norm_kernel(NormArgs p) {
    constexpr int VEC = kVec<XT>;
    __shared__ float shared[2][16][2];
    const int slots = blockDim.x / p.per_row, slot = threadIdx.x / p.per_row, thread = threadIdx.x - slot * p.per_row;
    const int wave = threadIdx.x >> 6, waves = p.per_row >> 6;
    RowSum sum{shared, waves, slot * waves, wave, 0};
    int at[K], left[K];
    float wb[K][VEC], wn[K][VEC], sc[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        at[k] = (k * p.per_row + thread) * VEC;
        left[k] = p.D - at[k];
        load_vector<XT, VEC>(wn[k], p.next_weight, p.vectors_f32, at[k], left[k]);
        if (p.branch.p != nullptr) {
            load_vector<XT, VEC>(wb[k], p.branch_weight, p.vectors_f32, at[k], left[k]);
            load_vector<XT, VEC>(sc[k], p.scale, p.vectors_f32, at[k], left[k]);
        }
    }
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * slots; base < p.rows; base += static_cast<int64_t>(gridDim.x) * slots) {
        const int64_t row = base + slot < p.rows ? base + slot : p.rows - 1;       // (rows behind the last repeat it and are not written)
        const bool writes = base + slot < p.rows;
        float x[K][VEC], total[K][VEC], g[K][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) load<RT, VEC>(total[k], p.residual.p, row * p.residual.row + at[k], left[k]);
        float4 stats = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.branch.p != nullptr) {
#pragma unroll
            for (int k = 0; k < K; ++k) load<XT, VEC>(x[k], p.branch.p, row * p.branch.row + at[k], left[k]);
            if (p.gate_form != SNNF_GATE_NONE) {
#pragma unroll
                for (int k = 0; k < K; ++k) load<XT, VEC>(g[k], p.gate.p, row * p.gate.row + at[k], left[k]);
            }
            whiten<LAYER, K, VEC>(x, left, p.D, p.eps, sum, stats.x, stats.y);
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float act = 1.0f, slope;
                    if (p.gate_form != SNNF_GATE_NONE) gate_of<kPrecise<XT>>(p.gate_form, g[k][j], act, slope);
                    const float more = (x[k][j] * stats.y * wb[k][j]) * (act * (sc[k][j] * p.factor));
                    total[k][j] = j < left[k] ? total[k][j] + more : 0.0f;
                }
                if (writes) save<RT, VEC>(p.residual_out, row * p.D + at[k], left[k], total[k]);
            }
        }
        whiten<LAYER, K, VEC>(total, left, p.D, p.eps, sum, stats.z, stats.w);
        if (!writes) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) total[k][j] = total[k][j] * stats.w * wn[k][j];
            save<XT, VEC>(p.normed, row * p.D + at[k], left[k], total[k]);
        }
        if (p.stats != nullptr && thread == 0) p.stats[row] = stats;
    }
}

template <typename RT, typename XT, int K, bool LAYER, int BLOCK>
__global__ __launch_bounds__(BLOCK) void block_norm_backward_kernel(NormArgs p) {
    constexpr int VEC = kVec<XT>;
    __shared__ float shared[2][16][2];
    const int slots = blockDim.x / p.per_row, slot = threadIdx.x / p.per_row, thread = threadIdx.x - slot * p.per_row;
    const int wave = threadIdx.x >> 6, waves = p.per_row >> 6;
    RowSum sum{shared, waves, slot * waves, wave, 0};
    const bool branch = p.branch.p != nullptr, gated = p.gate_form != SNNF_GATE_NONE;
    int at[K], left[K];
    float wb[K][VEC], wn[K][VEC], sc[K][VEC], dwb[K][VEC], dwn[K][VEC], dsc[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        at[k] = (k * p.per_row + thread) * VEC;
        left[k] = p.D - at[k];
        load_vector<XT, VEC>(wn[k], p.next_weight, p.vectors_f32, at[k], left[k]);
        load_vector<XT, VEC>(wb[k], branch ? p.branch_weight : nullptr, p.vectors_f32, at[k], left[k]);
        load_vector<XT, VEC>(sc[k], branch ? p.scale : nullptr, p.vectors_f32, at[k], left[k]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) dwb[k][j] = dwn[k][j] = dsc[k][j] = 0.0f;
    }
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * slots; base < p.rows; base += static_cast<int64_t>(gridDim.x) * slots) {
        const bool writes = base + slot < p.rows;
        const int64_t row = writes ? base + slot : p.rows - 1;
        float total[K][VEC], unit[K][VEC], g[K][VEC], d[K][VEC], dn[K][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            load<RT, VEC>(total[k], p.residual.p, row * p.residual.row + at[k], left[k]);
            if (p.d_normed.p != nullptr) load<XT, VEC>(dn[k], p.d_normed.p, row * p.d_normed.row + at[k], left[k]);
            if (p.d_residual_out.p != nullptr) load<RT, VEC>(d[k], p.d_residual_out.p, row * p.d_residual_out.row + at[k], left[k]);
            if (branch) load<XT, VEC>(unit[k], p.branch.p, row * p.branch.row + at[k], left[k]);
            if (gated) load<XT, VEC>(g[k], p.gate.p, row * p.gate.row + at[k], left[k]);
        }
        const float4 stats = p.stats[row];
        float act[K][VEC], slope[K][VEC], s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const bool in = j < left[k];
                act[k][j] = 1.0f, slope[k][j] = 0.0f;
                if (branch) {
                    if (gated) gate_of<kPrecise<XT>>(p.gate_form, g[k][j], act[k][j], slope[k][j]);
                    unit[k][j] = in ? (unit[k][j] - stats.x) * stats.y : 0.0f;
                    total[k][j] += (unit[k][j] * wb[k][j]) * (act[k][j] * (sc[k][j] * p.factor));
                }
                total[k][j] = in ? (total[k][j] - stats.z) * stats.w : 0.0f;       // the unit row of the second norm
                if (p.d_normed.p == nullptr) dn[k][j] = 0.0f;
                if (p.d_residual_out.p == nullptr) d[k][j] = 0.0f;
                if (writes) dwn[k][j] = fmaf(dn[k][j], total[k][j], dwn[k][j]);
                dn[k][j] = in ? dn[k][j] * wn[k][j] : 0.0f;
                s[0] = fmaf(dn[k][j], total[k][j], s[0]);
                s[1] += dn[k][j];
            }
        sum(s);
        s[0] /= p.D;
        s[1] = LAYER ? s[1] / p.D : 0.0f;
        float q[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                d[k][j] += stats.w * (dn[k][j] - total[k][j] * s[0] - s[1]);
                if (branch) {
                    const float through = d[k][j] * p.factor, y = unit[k][j] * wb[k][j];
                    if (writes) dsc[k][j] = fmaf(through * act[k][j], y, dsc[k][j]);
                    slope[k][j] = through * sc[k][j] * y * slope[k][j];            // the gate's gradient
                    const float du = through * sc[k][j] * act[k][j];
                    if (writes) dwb[k][j] = fmaf(du, unit[k][j], dwb[k][j]);
                    dn[k][j] = j < left[k] ? du * wb[k][j] : 0.0f;
                    q[0] = fmaf(dn[k][j], unit[k][j], q[0]);
                    q[1] += dn[k][j];
                }
            }
            if (writes) {
                save<RT, VEC>(p.d_residual, row * p.D + at[k], left[k], d[k]);
                if (gated) save<XT, VEC>(p.d_gate, row * p.D + at[k], left[k], slope[k]);
            }
        }
        if (branch) {
            sum(q);
            q[0] /= p.D;
            q[1] = LAYER ? q[1] / p.D : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) dn[k][j] = stats.y * (dn[k][j] - unit[k][j] * q[0] - q[1]);
                if (writes) save<XT, VEC>(p.d_branch, row * p.D + at[k], left[k], dn[k]);
            }
        }
    }
    float* to = p.parts + (static_cast<int64_t>(blockIdx.x) * slots + slot) * 3 * p.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        save<float, VEC>(to, at[k], left[k], dwb[k]);
        save<float, VEC>(to + p.D, at[k], left[k], dwn[k]);
        save<float, VEC>(to + 2 * p.D, at[k], left[k], dsc[k]);
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

// Threads to a row: 8 elements each, up to 1024 threads. Backward, a workgroup takes at least four rows to a slot where that leaves one for every
// compute unit: its sums over rows cost as much memory as a row does.
NormShape norm_shape(int64_t rows, int D, bool backward, int vec) {
    NormShape s;
    s.per_row = 64;
    while (s.per_row < 1024 && s.per_row * 8 < D) s.per_row *= 2;
    s.chunks = s.per_row * 8 < D ? 16 / vec : 8 / vec;
    s.block = s.per_row < 256 ? 256 : s.per_row;
    s.slots = s.block / s.per_row;
    const int64_t units = compute_units(), resident = units * (backward ? (s.block == 256 ? 3 : 1) : 2048 / s.block);
    int64_t grid = (rows + s.slots - 1) / s.slots;
    if (backward) {
        const int64_t few = (rows + s.slots * 4 - 1) / (s.slots * 4);
        grid = grid < units ? grid : (few < units ? units : few);
    }
    s.grid = static_cast<int>(grid < resident ? grid : resident);
    return s;
}

template <typename RT, typename XT, int K>
void launch_norm(const NormArgs& p, const NormShape& s, bool layer, bool backward, hipStream_t stream) {
    const dim3 grid(s.grid), block(s.block);
    if (backward) {
        if (s.block > 512) {
            if (layer) block_norm_backward_kernel<RT, XT, K, true, 1024><<<grid, block, 0, stream>>>(p);
            else block_norm_backward_kernel<RT, XT, K, false, 1024><<<grid, block, 0, stream>>>(p);
        } else if constexpr (K * kVec<XT> == 8) {
            if (layer) block_norm_backward_kernel<RT, XT, K, true, 512><<<grid, block, 0, stream>>>(p);
            else block_norm_backward_kernel<RT, XT, K, false, 512><<<grid, block, 0, stream>>>(p);
        }
    } else {
        if (layer) block_norm_kernel<RT, XT, K, true><<<grid, block, 0, stream>>>(p);
        else block_norm_kernel<RT, XT, K, false><<<grid, block, 0, stream>>>(p);
    }
}

template <typename RT, typename XT>
void launch_types(const NormArgs& p, const NormShape& s, bool layer, bool backward, hipStream_t stream) {
    constexpr int few = 8 / kVec<XT>;
    if (s.chunks == few) launch_norm<RT, XT, few>(p, s, layer, backward, stream);
    else launch_norm<RT, XT, 2 * few>(p, s, layer, backward, stream);
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

int run_norm(const char* name, const NormArgs& p, int residual_dtype, int dtype, int kind, bool backward, const NormShape& s, hipStream_t stream) {
    const bool layer = kind == SNNF_NORM_LAYER;
    if (dtype == SNNF_F32) launch_types<float, float>(p, s, layer, backward, stream);
    else if (dtype == SNNF_BF16 && residual_dtype == SNNF_F32) launch_types<float, bf16_t>(p, s, layer, backward, stream);
    else if (dtype == SNNF_BF16) launch_types<bf16_t, bf16_t>(p, s, layer, backward, stream);
    else if (residual_dtype == SNNF_F32) launch_types<float, f16_t>(p, s, layer, backward, stream);
    else launch_types<f16_t, f16_t>(p, s, layer, backward, stream);
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
    p.vectors_f32 = vector_dtype == SNNF_F32;
    p.factor = factor, p.eps = eps;
    const NormShape s = norm_shape(rows, D, false, dtype == SNNF_F32 ? 4 : 8);
    p.per_row = s.per_row;
    return run_norm("snnf_block_norm", p, residual_dtype, dtype, kind, false, s, as_stream(stream));
}

extern "C" size_t snnf_block_norm_backward_workspace_bytes(int64_t rows, int D) {
    if (rows < 1 || D < 1 || D > kMostWidth) return 0;
    const NormShape s = norm_shape(rows, D, true, 8);
    return static_cast<size_t>(s.grid) * s.slots * 3 * D * sizeof(float);
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
    p.vectors_f32 = vector_dtype == SNNF_F32;
    p.factor = factor;
    const NormShape s = norm_shape(rows, D, true, dtype == SNNF_F32 ? 4 : 8);
    p.per_row = s.per_row;
    hipStream_t hs = as_stream(stream);
    const int status = run_norm(name, p, residual_dtype, dtype, kind, true, s, hs);
    if (status != SNNF_OK || (d_branch_weight == nullptr && d_next_weight == nullptr && d_scale == nullptr)) return status;
    const dim3 grid((D + 63) / 64, 3), block(64 * kPhases);
    const int n_parts = s.grid * s.slots;
    if (vector_dtype == SNNF_F32)
        vector_gradient_kernel<<<grid, block, 0, hs>>>(p.parts, n_parts, D, static_cast<float*>(d_branch_weight), static_cast<float*>(d_next_weight), static_cast<float*>(d_scale));
    else if (vector_dtype == SNNF_BF16)
        vector_gradient_kernel<<<grid, block, 0, hs>>>(p.parts, n_parts, D, static_cast<bf16_t*>(d_branch_weight), static_cast<bf16_t*>(d_next_weight), static_cast<bf16_t*>(d_scale));
    else
        vector_gradient_kernel<<<grid, block, 0, hs>>>(p.parts, n_parts, D, static_cast<f16_t*>(d_branch_weight), static_cast<f16_t*>(d_next_weight), static_cast<f16_t*>(d_scale));
    return check_launch(name);
}
