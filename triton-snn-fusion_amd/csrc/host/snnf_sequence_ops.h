// The sequence operators (gated recurrence, delta rule, block norm, token scores, verification of drafts) from C++: calls on tensors that the kernels read in place, with and without
// gradients. Included by snnf_dispatch.cpp, inside its namespace.
//
// A training step on a small batch is bound by the host: through the Python implementations forward and backward take 130 to 170 us of it, from
// here some 40. A call that is not plain (another layout, dtype or device, sizes of zero, arguments of the wrong kind) gets None, and the Python
// entry point, which judges and refuses, runs it. As there is no eager substitute, nothing is counted.
#pragma once

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Whether elements of the last dimension lie next to each other.
inline bool unit_rows(const Tensor& t) { return t.dim() > 0 && (t.size(-1) <= 1 || t.stride(-1) == 1); }
inline bool like_of(const Tensor& t, const Tensor& like, at::ScalarType dtype) { return t.is_cuda() && t.device() == like.device() && t.scalar_type() == dtype; }
inline bool activation(const Tensor& t) {
    int code;
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && dtype_code(t.scalar_type(), &code) && t.numel() > 0;
}
// Whether the kernels' work is all there is to a call: what traces torch's operations would record the outputs' allocation and nothing that fills them, a
// tangent of forward-mode differentiation would be lost, a tensor that a transform of torch.func wraps has no memory of its own, and a subclass may be a
// wrapper without an address.
inline bool traced() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    return torch::jit::tracer::isTracing() || (Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
}
inline bool unobserved(c10::ArrayRef<const Tensor*> tensors) {
    if (traced()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && (!t->has_storage() || t->unsafeGetTensorImpl()->is_python_dispatch() || t->_fw_grad(0).defined())) return false;
    return true;
}
// The same of the gradients that autograd hands over: there is no other implementation to refuse them.
inline void check_gradients(const char* name, const variable_list& grads) {
    TORCH_CHECK(!traced(), name, ": unsupported_tracing: torch.jit.trace and make_fx record torch's own operations only");
    for (const Tensor& d : grads) {
        if (!d.defined()) continue;
        TORCH_CHECK(d.has_storage(), name, ": unsupported_transform: a gradient is wrapped by a transform (torch.func, vmap) and has no memory of its own");
        TORCH_CHECK(d.const_data_ptr() != nullptr || d.numel() == 0, name, ": unsupported_subclass: a gradient wraps other tensors");
        TORCH_CHECK(!d._fw_grad(0).defined(), name, ": unsupported_forward_ad: a gradient has a tangent, and there is no forward-mode derivative");
    }
}
inline void* data_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline void check_status(int status) { TORCH_CHECK(status == 0, snnf_last_error()); }

// Operands that a call may lack are handed to autograd as absent ones, which have no edge: the edge of operand i is its place among those there.
using Maybe = std::optional<Tensor>;
inline Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
inline Tensor tensor_of(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

// The gradients are worked out by kernels that autograd does not see: a second differentiation has to fail, not to be silently zero.
inline variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list inputs;
    for (Tensor& g : grads) inputs.push_back(g.defined() ? g.detach().set_requires_grad(true) : Tensor());
    return torch::autograd::DelayedError("trying to differentiate twice an operator of libsnnf that is differentiable once", static_cast<int64_t>(grads.size()))
        .apply(std::move(inputs));
}

// [rows, D] with any stride between rows, without a copy; false: not such a tensor.
inline bool row_stride(const Tensor& t, int64_t* stride) {
    if (t.is_contiguous()) *stride = t.size(-1);
    else if (t.dim() == 2 && unit_rows(t)) *stride = t.stride(0);
    else return false;
    return true;
}
// A gradient as autograd hands it over, in rows that the kernels read.
inline Tensor readable(const Tensor& d, int64_t* stride) {
    if (!d.defined()) return d;
    if (row_stride(d, stride)) return d;
    Tensor c = d.contiguous();
    *stride = c.size(-1);
    return c;
}

// ------------------------------------------------------------------------------------------------------------------
// Gated recurrence
// ------------------------------------------------------------------------------------------------------------------
inline Tensor empty_steps(const Tensor& x) {
    const int64_t T = x.size(0), N = x.size(1), D = x.size(2);
    const bool batch_first = x.stride(1) > x.stride(0);
    return at::empty_strided({T, N, D}, batch_first ? std::array<int64_t, 3>{D, T * D, 1} : std::array<int64_t, 3>{N * D, D, 1}, x.options().requires_grad(false));
}

// The kernels reach the steps that a thread takes at once, up to 16, by offsets of 31 bits.
inline bool within_reach(const Tensor& t) {
    return (t.stride(0) * (std::min<int64_t>(t.size(0), 16) - 1) + t.size(2)) * static_cast<int64_t>(t.element_size()) < 0x7fffffff;
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list compute(const Tensor& x, const Tensor& gate, const Tensor& state, const Tensor& starts, const Tensor& lengths, int64_t form, Tensor* marks) {
        const c10::DeviceGuard guard(x.device());
        const int T = static_cast<int>(x.size(0)), N = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2)), code = code_of(x.scalar_type());
        Tensor h = empty_steps(x), last = empty({N, D}, at::kFloat, x);
        if (marks) *marks = empty({static_cast<int64_t>(snnf_gated_recurrence_marks_bytes(T, N, D, code) / 4)}, at::kFloat, x);
        const size_t bytes = snnf_gated_recurrence_workspace_bytes(T, N, D, code, 0);
        const Tensor space = bytes ? empty({static_cast<int64_t>(bytes)}, at::kByte, x) : Tensor();
        check_status(snnf_gated_recurrence(x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1), T, N, D, code,
                                           static_cast<int>(form), data_of(starts), starts.defined() ? starts.stride(0) : 0,
                                           starts.defined() ? starts.stride(1) : 0, static_cast<const int32_t*>(data_of(lengths)),
                                           static_cast<const float*>(data_of(state)), h.data_ptr(), h.stride(0), h.stride(1), last.data_ptr<float>(),
                                           marks ? marks->data_ptr<float>() : nullptr, data_of(space), bytes, stream_of(x)));
        return {std::move(h), std::move(last)};
    }
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor gate, Maybe state, Maybe starts, Maybe lengths, int64_t form) {
        Tensor marks;
        variable_list out = compute(x, gate, tensor_of(state), tensor_of(starts), tensor_of(lengths), form, &marks);
        ctx->set_materialize_grads(false);
        ctx->saved_data["form"] = form;
        ctx->saved_data["state"] = state.has_value();
        ctx->save_for_backward({x, gate, tensor_of(starts), tensor_of(lengths), marks});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_gradients("run_hip_gated_recurrence", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &gate = saved[1], &starts = saved[2], &lengths = saved[3], &marks = saved[4];
        const c10::DeviceGuard guard(x.device());
        const int T = static_cast<int>(x.size(0)), N = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2)), code = code_of(x.scalar_type());
        Tensor dh = grads[0].defined() ? grads[0] : at::zeros({D}, x.options().requires_grad(false)).expand({T, N, D});
        if (!unit_rows(dh) || !within_reach(dh)) {
            Tensor near_by = empty_steps(x);
            dh = near_by.copy_(dh);
        }
        const Tensor dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
        Tensor dx = empty_steps(x), dgate = empty_steps(x), dstate = empty({N, D}, at::kFloat, x);
        const size_t bytes = snnf_gated_recurrence_workspace_bytes(T, N, D, code, 1);
        const Tensor space = bytes ? empty({static_cast<int64_t>(bytes)}, at::kByte, x) : Tensor();
        check_status(snnf_gated_recurrence_backward(
            x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1), dh.data_ptr(), dh.stride(0), dh.stride(1), T, N, D,
            code, static_cast<int>(ctx->saved_data["form"].toInt()), data_of(starts), starts.defined() ? starts.stride(0) : 0,
            starts.defined() ? starts.stride(1) : 0, static_cast<const int32_t*>(data_of(lengths)), marks.data_ptr<float>(),
            static_cast<const float*>(data_of(dlast)), dx.data_ptr(), dx.stride(0), dx.stride(1), dgate.data_ptr(), dgate.stride(0), dgate.stride(1),
            dstate.data_ptr<float>(), data_of(space), bytes, stream_of(x)));
        if (!ctx->needs_input_grad(0)) dx = Tensor();
        if (!ctx->needs_input_grad(1)) dgate = Tensor();
        if (!ctx->saved_data["state"].toBool() || !ctx->needs_input_grad(2)) dstate = Tensor();
        return once({std::move(dx), std::move(dgate), std::move(dstate), Tensor(), Tensor(), Tensor()});
    }
};

// An argument that may be None; undefined then. Clears `fine` where it is neither None nor a tensor.
inline Tensor optional_tensor(Args& a, Py_ssize_t i) {
    if (a.v[i] == Py_None) return Tensor();
    const Tensor* t = a.tensor(i);
    return t ? *t : Tensor();
}
inline bool wants_gradient(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
inline PyObject* tuple_of(const variable_list& tensors) {
    PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    for (size_t i = 0; i < tensors.size(); ++i) {
        PyObject* item = tensors[i].defined() ? THPVariable_Wrap(tensors[i]) : none();
        PyTuple_SET_ITEM(tuple, static_cast<Py_ssize_t>(i), item);
    }
    return tuple;
}

// x_seq, gate_seq, state | None, starts | None, lengths | None, form
PyObject* gated_recurrence(Args& a) {
    const Tensor x = optional_tensor(a, 0), gate = optional_tensor(a, 1), state = optional_tensor(a, 2), starts = optional_tensor(a, 3), lengths = optional_tensor(a, 4);
    const int64_t form = a.number(5);
    if (!a.fine || !unobserved({&x, &gate, &state, &starts, &lengths}) || !activation(x) || x.dim() != 3 || !unit_rows(x) || !gate.defined()) return none();
    const int64_t T = x.size(0), N = x.size(1), D = x.size(2);
    if (std::max({T, N, D}) > (int64_t{1} << 30) || !like_of(gate, x, x.scalar_type()) || gate.sizes() != x.sizes() || !unit_rows(gate)) return none();
    if (state.defined() && (!like_of(state, x, at::kFloat) || state.dim() != 2 || state.size(0) != N || state.size(1) != D || !state.is_contiguous())) return none();
    if (starts.defined() && (!like_of(starts, x, at::kBool) || starts.dim() != 2 || starts.size(0) != T || starts.size(1) != N)) return none();
    if (lengths.defined() && (!like_of(lengths, x, at::kInt) || lengths.dim() != 1 || lengths.size(0) != N || !lengths.is_contiguous())) return none();
    variable_list out;
    unlocked([&] {
        out = wants_gradient({&x, &gate, &state}) ? Recurrence::apply(x, gate, maybe(state), maybe(starts), maybe(lengths), form)
                                                  : Recurrence::compute(x, gate, state, starts, lengths, form, nullptr);
        return true;
    });
    return tuple_of(out);
}

// ------------------------------------------------------------------------------------------------------------------
// Block norm
// ------------------------------------------------------------------------------------------------------------------
constexpr int64_t kWidestNorm = 16384;      // as the kernels take it; what follows divides by a width that fits an int

struct BlockNorm : torch::autograd::Function<BlockNorm> {
    struct Shape {
        int64_t rows, row[3];
        int D, residual_dtype, dtype, vector_dtype;
        // Of tensors whose rows are readable
        Shape(const Tensor& residual, const Tensor& branch, const Tensor& gate, const Tensor& vector) {
            D = static_cast<int>(residual.size(-1));
            rows = residual.numel() / D;
            const Tensor* all[3] = {&residual, &branch, &gate};
            for (int i = 0; i < 3; ++i) {
                row[i] = 0;
                if (all[i]->defined()) row_stride(*all[i], &row[i]);
            }
            residual_dtype = code_of(residual.scalar_type());
            dtype = code_of(branch.scalar_type());
            vector_dtype = vector.defined() ? code_of(vector.scalar_type()) : dtype;
        }
    };
    static const Tensor& some(const Tensor& a, const Tensor& b, const Tensor& c) { return a.defined() ? a : (b.defined() ? b : c); }
    static variable_list compute(const Tensor& residual, const Tensor& branch, const Tensor& gate, const Tensor& wb, const Tensor& wn, const Tensor& scale,
                                 double factor, int64_t kind, int64_t gate_form, double eps, Tensor* stats) {
        const c10::DeviceGuard guard(residual.device());
        const Shape s(residual, branch, gate, some(wb, wn, scale));
        Tensor out = empty(residual.sizes(), residual.scalar_type(), residual), normed = empty(residual.sizes(), branch.scalar_type(), residual);
        if (stats) *stats = empty({s.rows, 4}, at::kFloat, residual);
        check_status(snnf_block_norm(residual.data_ptr(), s.row[0], branch.data_ptr(), s.row[1], data_of(gate), s.row[2], data_of(wb), data_of(wn),
                                     data_of(scale), static_cast<float>(factor), s.rows, s.D, s.residual_dtype, s.dtype, s.vector_dtype,
                                     static_cast<int>(kind), gate.defined() ? static_cast<int>(gate_form) : 0, static_cast<float>(eps), out.data_ptr(),
                                     normed.data_ptr(), stats ? stats->data_ptr<float>() : nullptr, stream_of(residual)));
        return {std::move(out), std::move(normed)};
    }
    static variable_list forward(AutogradContext* ctx, Tensor residual, Tensor branch, Maybe gate, Maybe branch_weight, Maybe next_weight, Maybe learnt,
                                 double factor, int64_t kind, int64_t gate_form, double eps) {
        const Tensor g = tensor_of(gate), wb = tensor_of(branch_weight), wn = tensor_of(next_weight), scale = tensor_of(learnt);
        Tensor stats;
        variable_list out = compute(residual, branch, g, wb, wn, scale, factor, kind, gate_form, eps, &stats);
        ctx->set_materialize_grads(false);
        ctx->saved_data["factor"] = factor;
        ctx->saved_data["kind"] = kind;
        ctx->saved_data["gate_form"] = gate_form;
        ctx->save_for_backward({residual, branch, g, wb, wn, scale, stats});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_gradients("run_hip_block_norm", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &residual = saved[0], &branch = saved[1], &gate = saved[2], &wb = saved[3], &wn = saved[4], &scale = saved[5], &stats = saved[6];
        const c10::DeviceGuard guard(residual.device());
        const Shape s(residual, branch, gate, some(wb, wn, scale));
        int64_t out_row = 0, normed_row = 0;
        const Tensor d_out = readable(grads[0], &out_row), d_normed = readable(grads[1], &normed_row);
        variable_list d(10);
        for (int i = 0; i < 3; ++i)
            if (saved[i].defined()) d[i] = empty(saved[i].sizes(), saved[i].scalar_type(), residual);
        std::array<bool, 6> needed{};
        for (int i = 0, edge = 0; i < 6; ++i)
            if (saved[i].defined()) needed[i] = ctx->needs_input_grad(edge++);
        for (int i = 3; i < 6; ++i)
            if (needed[i]) d[i] = empty({s.D}, saved[i].scalar_type(), residual);
        const size_t bytes = snnf_block_norm_backward_workspace_bytes(s.rows, s.D);
        const Tensor space = empty({static_cast<int64_t>(bytes)}, at::kByte, residual);
        check_status(snnf_block_norm_backward(
            residual.data_ptr(), s.row[0], branch.data_ptr(), s.row[1], data_of(gate), s.row[2], data_of(wb), data_of(wn), data_of(scale),
            static_cast<float>(ctx->saved_data["factor"].toDouble()), data_of(d_out), out_row, data_of(d_normed), normed_row, stats.data_ptr<float>(), s.rows,
            s.D, s.residual_dtype, s.dtype, s.vector_dtype, static_cast<int>(ctx->saved_data["kind"].toInt()),
            gate.defined() ? static_cast<int>(ctx->saved_data["gate_form"].toInt()) : 0, d[0].data_ptr(), d[1].data_ptr(), data_of(d[2]), data_of(d[3]),
            data_of(d[4]), data_of(d[5]), space.data_ptr(), bytes, stream_of(residual)));
        for (int i = 0; i < 3; ++i)
            if (!needed[i]) d[i] = Tensor();
        return once(std::move(d));
    }
};

// residual, branch, gate | None, branch_weight | None, next_weight | None, scale | None, factor, kind, gate form, eps
PyObject* block_norm(Args& a) {
    const Tensor residual = optional_tensor(a, 0), branch = optional_tensor(a, 1), gate = optional_tensor(a, 2);
    const std::array<Tensor, 3> vectors{optional_tensor(a, 3), optional_tensor(a, 4), optional_tensor(a, 5)};
    const double factor = a.real(6), eps = a.real(9);
    const int64_t kind = a.number(7), gate_form = a.number(8);
    int64_t stride;
    if (!a.fine || !unobserved({&residual, &branch, &gate, &vectors[0], &vectors[1], &vectors[2]})) return none();
    if (!activation(residual) || !activation(branch) || residual.dim() < 1 || residual.size(-1) > kWidestNorm || !row_stride(residual, &stride)) return none();
    if (branch.device() != residual.device() || (residual.scalar_type() != branch.scalar_type() && residual.scalar_type() != at::kFloat)) return none();
    for (const Tensor* t : {&branch, &gate})
        if (t->defined() && (!like_of(*t, residual, branch.scalar_type()) || t->sizes() != residual.sizes() || !row_stride(*t, &stride))) return none();
    const Tensor& vector = BlockNorm::some(vectors[0], vectors[1], vectors[2]);
    for (const Tensor& t : vectors)
        if (t.defined() && (!like_of(t, residual, vector.scalar_type()) || (t.scalar_type() != at::kFloat && t.scalar_type() != branch.scalar_type()) || t.dim() != 1 ||
                            t.size(0) != residual.size(-1) || !t.is_contiguous()))
            return none();
    variable_list out;
    unlocked([&] {
        out = wants_gradient({&residual, &branch, &gate, &vectors[0], &vectors[1], &vectors[2]})
                  ? BlockNorm::apply(residual, branch, maybe(gate), maybe(vectors[0]), maybe(vectors[1]), maybe(vectors[2]), factor, kind, gate_form, eps)
                  : BlockNorm::compute(residual, branch, gate, vectors[0], vectors[1], vectors[2], factor, kind, gate_form, eps, nullptr);
        return true;
    });
    return tuple_of(out);
}

// ------------------------------------------------------------------------------------------------------------------
// Token scores
// ------------------------------------------------------------------------------------------------------------------
struct Scores : torch::autograd::Function<Scores> {
    // logprob, entropy and, with alternatives, top_logprob, top_token
    static variable_list compute(const Tensor& logits, const Tensor& tokens, int64_t top_k, Tensor* stats) {
        const c10::DeviceGuard guard(logits.device());
        const int64_t V = logits.size(-1), rows = logits.numel() / V;
        int64_t row = V;
        row_stride(logits, &row);
        const auto lead = logits.sizes().slice(0, logits.dim() - 1);
        variable_list out{empty(lead, at::kFloat, logits), empty(lead, at::kFloat, logits)};
        if (top_k > 0) {
            c10::SmallVector<int64_t, 6> shape(lead.begin(), lead.end());
            shape.push_back(top_k);
            out.push_back(empty(shape, at::kFloat, logits));
            out.push_back(empty(shape, at::kLong, logits));
        }
        if (stats) *stats = empty({rows, 2}, at::kFloat, logits);
        const size_t bytes = snnf_token_scores_workspace_bytes(rows, static_cast<int>(V), static_cast<int>(top_k));
        const Tensor space = bytes ? empty({static_cast<int64_t>(bytes)}, at::kByte, logits) : Tensor();
        check_status(snnf_token_scores(logits.data_ptr(), row, rows, static_cast<int>(V), code_of(logits.scalar_type()),
                                       static_cast<const int64_t*>(data_of(tokens)), static_cast<int>(top_k), out[0].data_ptr<float>(), out[1].data_ptr<float>(),
                                       top_k > 0 ? out[2].data_ptr<float>() : nullptr, top_k > 0 ? out[3].data_ptr<int64_t>() : nullptr,
                                       stats ? stats->data_ptr<float>() : nullptr, data_of(space), bytes, stream_of(logits)));
        return out;
    }
    static variable_list forward(AutogradContext* ctx, Tensor logits, Maybe tokens, int64_t top_k) {
        Tensor stats;
        variable_list out = compute(logits, tensor_of(tokens), top_k, &stats);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({logits, tensor_of(tokens), stats, out[1]});
        if (top_k > 0) ctx->mark_non_differentiable({out[2], out[3]});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_gradients("run_hip_token_scores", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2], &entropy = saved[3];
        const c10::DeviceGuard guard(logits.device());
        const int64_t V = logits.size(-1), rows = logits.numel() / V;
        int64_t row = V;
        row_stride(logits, &row);
        const Tensor d_logprob = grads[0].defined() ? grads[0].contiguous() : Tensor(), d_entropy = grads[1].defined() ? grads[1].contiguous() : Tensor();
        Tensor d = empty(logits.sizes(), logits.scalar_type(), logits);
        check_status(snnf_token_scores_backward(logits.data_ptr(), row, rows, static_cast<int>(V), code_of(logits.scalar_type()),
                                                static_cast<const int64_t*>(data_of(tokens)), stats.data_ptr<float>(), entropy.data_ptr<float>(),
                                                static_cast<const float*>(data_of(d_logprob)), static_cast<const float*>(data_of(d_entropy)), d.data_ptr(),
                                                stream_of(logits)));
        return once({std::move(d), Tensor(), Tensor()});
    }
};

// logits, tokens | None, top_k
PyObject* token_scores(Args& a) {
    const Tensor logits = optional_tensor(a, 0), tokens = optional_tensor(a, 1);
    const int64_t top_k = a.number(2);
    int64_t stride;
    if (!a.fine || !unobserved({&logits, &tokens}) || !activation(logits) || logits.dim() < 1 || logits.size(-1) > (int64_t{1} << 30) || !row_stride(logits, &stride)) return none();
    if (top_k < 0 || top_k > 64 || top_k > logits.size(-1)) return none();
    if (tokens.defined() && (!like_of(tokens, logits, at::kLong) || tokens.sizes() != logits.sizes().slice(0, logits.dim() - 1) || !tokens.is_contiguous())) return none();
    variable_list out;
    unlocked([&] {
        out = wants_gradient({&logits}) ? Scores::apply(logits, maybe(tokens), top_k) : Scores::compute(logits, tokens, top_k, nullptr);
        return true;
    });
    out.resize(4);
    return tuple_of(out);
}

// ------------------------------------------------------------------------------------------------------------------
// Gated delta rule
// ------------------------------------------------------------------------------------------------------------------
inline Tensor empty_heads(const Tensor& t) {     // steps and sequences in t's order in memory
    const int64_t T = t.size(0), N = t.size(1), inner = t.numel() / (T * N);
    c10::SmallVector<int64_t, 4> strides(t.dim(), 1);
    if (t.dim() == 4) strides[2] = t.size(3);
    strides[0] = t.stride(1) > t.stride(0) ? inner : N * inner;
    strides[1] = t.stride(1) > t.stride(0) ? T * inner : inner;
    return at::empty_strided(t.sizes(), strides, t.options().requires_grad(false));
}

struct DeltaRule : torch::autograd::Function<DeltaRule> {
    static snnf_heads heads(const Tensor& t) {
        return t.defined() ? snnf_heads{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)} : snnf_heads{nullptr, 0, 0, 0};
    }
    static snnf_delta_rule_call call_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& gate, const Tensor& beta, const Tensor& starts,
                                        const Tensor& lengths, double scale) {
        snnf_delta_rule_call c = {};
        c.T = static_cast<int>(q.size(0)), c.N = static_cast<int>(q.size(1)), c.heads = static_cast<int>(q.size(2)), c.value_heads = static_cast<int>(v.size(2));
        c.key_size = static_cast<int>(q.size(3)), c.value_size = static_cast<int>(v.size(3));
        c.dtype = code_of(q.scalar_type());
        c.gate_dtype = gate.defined() ? code_of(gate.scalar_type()) : (beta.defined() ? code_of(beta.scalar_type()) : c.dtype);
        c.scale = static_cast<float>(scale);
        c.query = heads(q), c.key = heads(k), c.value = heads(v), c.gate = heads(gate), c.beta = heads(beta);
        c.starts = data_of(starts);
        if (starts.defined()) c.starts_step = starts.stride(0), c.starts_row = starts.stride(1);
        c.lengths = static_cast<const int32_t*>(data_of(lengths));
        return c;
    }
    static variable_list compute(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& gate, const Tensor& beta, const Tensor& state, const Tensor& starts,
                                 const Tensor& lengths, double scale, const Tensor& state_out, Tensor* marks) {
        const c10::DeviceGuard guard(q.device());
        snnf_delta_rule_call c = call_of(q, k, v, gate, beta, starts, lengths, scale);
        c.state = static_cast<const float*>(data_of(state));
        Tensor out = empty_heads(v), last = state_out.defined() ? state_out : empty({v.size(1), v.size(2), q.size(3), v.size(3)}, at::kFloat, q);
        if (marks) *marks = empty({static_cast<int64_t>(snnf_delta_rule_marks_bytes(&c) / 4)}, at::kFloat, q);
        const size_t bytes = snnf_delta_rule_workspace_bytes(&c, marks != nullptr);
        const Tensor space = bytes ? empty({static_cast<int64_t>(bytes)}, at::kByte, q) : Tensor();
        const snnf_heads view = heads(out);
        check_status(snnf_delta_rule(&c, &view, last.data_ptr<float>(), marks ? marks->data_ptr<float>() : nullptr, data_of(space), bytes, stream_of(q)));
        if (state_out.defined() && !state_out.is_inference()) state_out.unsafeGetTensorImpl()->bump_version();      // a graph that kept what it held before has to notice
        return {std::move(out), std::move(last)};
    }
    static variable_list forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, Maybe gate, Maybe beta, Maybe state, Maybe starts, Maybe lengths, double scale) {
        const Tensor g = tensor_of(gate), b = tensor_of(beta), m = tensor_of(starts), l = tensor_of(lengths);
        Tensor marks;
        variable_list out = compute(q, k, v, g, b, tensor_of(state), m, l, scale, Tensor(), &marks);
        ctx->set_materialize_grads(false);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["state"] = state.has_value();
        ctx->save_for_backward({q, k, v, g, b, m, l, marks});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_gradients("run_hip_delta_rule", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &marks = saved[7];
        const c10::DeviceGuard guard(q.device());
        const snnf_delta_rule_call c = call_of(q, k, v, saved[3], saved[4], saved[5], saved[6], ctx->saved_data["scale"].toDouble());
        Tensor dout = grads[0].defined() ? grads[0] : at::zeros({v.size(3)}, v.options().requires_grad(false)).expand(v.sizes());
        if (!unit_rows(dout)) dout = dout.contiguous();
        const Tensor dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
        variable_list d(9);
        std::array<snnf_heads, 5> views;
        for (int i = 0; i < 5; ++i) {
            if (saved[i].defined()) d[i] = empty_heads(saved[i]);
            views[i] = heads(d[i]);
        }
        d[5] = empty({v.size(1), v.size(2), q.size(3), v.size(3)}, at::kFloat, q);
        const size_t bytes = snnf_delta_rule_backward_workspace_bytes(&c);
        const Tensor space = empty({static_cast<int64_t>(bytes)}, at::kByte, q);
        const snnf_heads dout_view = heads(dout);
        check_status(snnf_delta_rule_backward(&c, marks.data_ptr<float>(), &dout_view, static_cast<const float*>(data_of(dlast)), &views[0], &views[1], &views[2], &views[3],
                                              &views[4], d[5].data_ptr<float>(), space.data_ptr(), bytes, stream_of(q)));
        for (int i = 0, edge = 0; i < 6; ++i) {
            const bool there = i == 5 ? ctx->saved_data["state"].toBool() : saved[i].defined();
            if (!there || !ctx->needs_input_grad(edge)) d[i] = Tensor();
            edge += there;
        }
        return once(std::move(d));
    }
};

// query, key, value, gate | None, beta | None, state | None, scale | None, starts | None, lengths | None, state_out | None
PyObject* delta_rule(Args& a) {
    const Tensor q = optional_tensor(a, 0), k = optional_tensor(a, 1), v = optional_tensor(a, 2), gate = optional_tensor(a, 3), beta = optional_tensor(a, 4);
    const Tensor state = optional_tensor(a, 5), starts = optional_tensor(a, 7), lengths = optional_tensor(a, 8), state_out = optional_tensor(a, 9);
    if (!a.fine || !unobserved({&q, &k, &v, &gate, &beta, &state, &starts, &lengths, &state_out}) || !activation(q) || q.dim() != 4 || !unit_rows(q)) return none();
    if (a.v[6] != Py_None && !PyFloat_Check(a.v[6]) && !PyLong_Check(a.v[6])) return none();
    const int64_t T = q.size(0), N = q.size(1), H = q.size(2), DK = q.size(3);
    if (!k.defined() || !like_of(k, q, q.scalar_type()) || k.sizes() != q.sizes() || !unit_rows(k)) return none();
    if (!v.defined() || !like_of(v, q, q.scalar_type()) || v.dim() != 4 || v.size(0) != T || v.size(1) != N || !unit_rows(v)) return none();
    const int64_t HV = v.size(2), DV = v.size(3);
    if (HV < 1 || HV % H != 0 || DK > SNNF_DELTA_RULE_MAX_KEY || DV < 1 || DV > SNNF_DELTA_RULE_MAX_VALUE || T > (int64_t{1} << 30) || N > (int64_t{1} << 20) ||
        HV > (int64_t{1} << 20) || N * HV > (int64_t{1} << 20) || N * HV * ((T + 63) / 64) > (int64_t{1} << 30))
        return none();
    for (const Tensor* t : {&gate, &beta})
        if (t->defined() && (t->dim() != 3 || t->size(0) != T || t->size(1) != N || t->size(2) != HV || !(like_of(*t, q, q.scalar_type()) || like_of(*t, q, at::kFloat)))) return none();
    if (gate.defined() && beta.defined() && gate.scalar_type() != beta.scalar_type()) return none();
    for (const Tensor* t : {&state, &state_out})
        if (t->defined() && (!like_of(*t, q, at::kFloat) || t->dim() != 4 || t->size(0) != N || t->size(1) != HV || t->size(2) != DK || t->size(3) != DV || !t->is_contiguous()))
            return none();
    if (starts.defined() && (!like_of(starts, q, at::kBool) || starts.dim() != 2 || starts.size(0) != T || starts.size(1) != N)) return none();
    if (lengths.defined() && (!like_of(lengths, q, at::kInt) || lengths.dim() != 1 || lengths.size(0) != N || !lengths.is_contiguous())) return none();
    const bool gradient = wants_gradient({&q, &k, &v, &gate, &beta, &state});
    if (state_out.defined()) {
        if (gradient || state_out.requires_grad()) return none();
        for (const Tensor* t : {&q, &k, &v, &gate, &beta, &state, &starts, &lengths})
            if (t->defined() && t->is_alias_of(state_out) && !(t == &state && t->data_ptr() == state_out.data_ptr())) return none();
    }
    const double scale = a.v[6] == Py_None ? std::pow(static_cast<double>(DK), -0.5) : a.real(6);
    if (!a.fine) return none();
    variable_list out;
    unlocked([&] {
        out = gradient ? DeltaRule::apply(q, k, v, maybe(gate), maybe(beta), maybe(state), maybe(starts), maybe(lengths), scale)
                       : DeltaRule::compute(q, k, v, gate, beta, state, starts, lengths, scale, state_out, nullptr);
        return true;
    });
    return tuple_of(out);
}

// ------------------------------------------------------------------------------------------------------------------
// Verification of drafts
// ------------------------------------------------------------------------------------------------------------------
// logits, drafts, uniforms, noise, draft_logits | None, temperature, lengths | None
PyObject* verify_drafts(Args& a) {
    const bool number = PyFloat_Check(a.v[5]) || PyLong_Check(a.v[5]);
    const Tensor logits = optional_tensor(a, 0), drafts = optional_tensor(a, 1), uniforms = optional_tensor(a, 2), noise = optional_tensor(a, 3), theirs = optional_tensor(a, 4);
    const Tensor each = number ? Tensor() : optional_tensor(a, 5), lengths = optional_tensor(a, 6);
    if (!a.fine || !unobserved({&logits, &drafts, &uniforms, &noise, &theirs, &each, &lengths}) || !activation(logits) || logits.dim() != 3 || !unit_rows(logits)) return none();
    if (!number && !each.defined()) return none();
    const int64_t N = logits.size(0), K = logits.size(1) - 1, V = logits.size(2);
    if (K < 1 || K > 64 || N > (int64_t{1} << 20) || V > (int64_t{1} << 30)) return none();
    const auto rows = [&](const Tensor& t, at::ScalarType dtype) { return t.defined() && like_of(t, logits, dtype) && t.dim() == 2 && t.size(0) == N; };
    if (!rows(drafts, at::kLong) || drafts.size(1) != K || !drafts.is_contiguous() || !rows(uniforms, at::kFloat) || uniforms.size(1) != K || !uniforms.is_contiguous()) return none();
    if (!rows(noise, at::kFloat) || noise.size(1) != V || !unit_rows(noise)) return none();
    if (theirs.defined() && (!like_of(theirs, logits, logits.scalar_type()) || theirs.dim() != 3 || theirs.size(0) != N || theirs.size(1) != K || theirs.size(2) != V || !unit_rows(theirs)))
        return none();
    if (each.defined() && (!like_of(each, logits, at::kFloat) || each.dim() != 1 || each.size(0) != N || !each.is_contiguous())) return none();
    if (lengths.defined() && (!like_of(lengths, logits, at::kInt) || lengths.dim() != 1 || lengths.size(0) != N || !lengths.is_contiguous())) return none();
    const double temperature = number ? a.real(5) : 1.0;
    if (!a.fine) return none();
    variable_list out;
    unlocked([&] {
        const c10::DeviceGuard guard(logits.device());
        out = {empty({N, K + 1}, at::kLong, logits), empty({N}, at::kInt, logits)};
        const int n = static_cast<int>(N), k = static_cast<int>(K), v = static_cast<int>(V);
        const size_t bytes = snnf_draft_verification_workspace_bytes(n, k, v, theirs.defined());
        const Tensor space = empty({static_cast<int64_t>(bytes)}, at::kByte, logits);
        check_status(snnf_draft_verification(logits.data_ptr(), logits.stride(0), logits.stride(1), data_of(theirs), theirs.defined() ? theirs.stride(0) : 0,
                                             theirs.defined() ? theirs.stride(1) : 0, n, k, v, code_of(logits.scalar_type()), drafts.data_ptr<int64_t>(),
                                             uniforms.data_ptr<float>(), noise.data_ptr<float>(), noise.stride(0), static_cast<const int32_t*>(data_of(lengths)),
                                             static_cast<float>(temperature), static_cast<const float*>(data_of(each)), out[0].data_ptr<int64_t>(),
                                             out[1].data_ptr<int32_t>(), space.data_ptr(), bytes, stream_of(logits)));
        return true;
    });
    return tuple_of(out);
}

// Any number of arguments; what is no tensor counts for nothing
PyObject* are_unobserved(Args& a) {
    c10::SmallVector<const Tensor*, 8> tensors;
    for (Py_ssize_t i = 0; i < a.n; ++i) {
        if (THPVariable_Check(a.v[i])) tensors.push_back(&THPVariable_Unpack(a.v[i]));
    }
    return PyBool_FromLong(unobserved(tensors));
}
