"""Gated delta rule on libsnnf (`snnf_delta_rule`), with its gradient.

The gated recurrence with a matrix for a state: each value head keeps S of [Dk, Dv], which a step decays, corrects where its key points to, and reads with its query:

    S <- exp(gate) S,    S <- S + beta key (value - S^T key)^T,    out = scale S^T query

The reference has no operator for this. There is no eager substitute: what the kernels do not take raises RuntimeError("unsupported_...").
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._sequence_common import check_activation, check_operand, check_unobserved, native, on_device_of, recorded, refuse, refuse_observed, unit_rows, wants_gradient, workspace

MAX_KEY, MAX_VALUE = 128, 1024
OPERANDS = ("query", "key", "value", "gate", "beta", "state", "starts", "lengths", "state_out")


def check_delta_rule_support(query, key, value, gate=None, beta=None, state=None, scale=None, starts=None, lengths=None, state_out=None) -> List[str]:
    """Reasons why a call is refused; empty if the kernels take it."""
    reasons: List[str] = []
    check_unobserved(reasons, OPERANDS, query, key, value, gate, beta, state, starts, lengths, state_out)
    if not check_activation("query", query, reasons):
        return reasons
    if query.dim() != 4 or not isinstance(value, torch.Tensor) or value.dim() != 4:
        reasons.append("unsupported_rank: query and value must be [T, N, heads, size]")
        return reasons
    T, N, H, DK = (int(n) for n in query.shape)
    HV, DV = int(value.shape[2]), int(value.shape[3])
    device, dtype = query.device, query.dtype
    check_operand("key", key, device, (T, N, H, DK), (dtype,), reasons)
    check_operand("value", value, device, (T, N, HV, DV), (dtype,), reasons)
    if H < 1 or HV < 1 or HV % H:
        reasons.append(f"unsupported_shape: value heads ({HV}) must be a multiple of heads ({H})")
    if not 1 <= DK <= MAX_KEY or not 1 <= DV <= MAX_VALUE:
        reasons.append(f"unsupported_shape: keys of 1 to {MAX_KEY} and values of 1 to {MAX_VALUE} elements, got {DK} and {DV}")
    if T > 1 << 30 or N * HV > 1 << 20 or N * HV * ((T + 63) // 64) > 1 << 30:
        reasons.append(f"unsupported_shape: at most 2^20 heads of all sequences and 2^30 steps of 64 of them, got N={N}, {HV} heads, T={T}")
    gates = [t for t in (gate, beta) if isinstance(t, torch.Tensor)]
    for name, t in (("gate", gate), ("beta", beta)):
        if t is not None:
            check_operand(name, t, device, (T, N, HV), (gates[0].dtype,) if gates and gates[0].dtype in (dtype, torch.float32) else (dtype, torch.float32), reasons)
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None:
            check_operand(name, t, device, (N, HV, DK, DV), (torch.float32,), reasons)
    if starts is not None:
        check_operand("starts", starts, device, (T, N), (torch.bool,), reasons)
    if lengths is not None:
        check_operand("lengths", lengths, device, (N,), (torch.int32, torch.int64), reasons)
    if scale is not None and not isinstance(scale, (int, float)):
        reasons.append("scale must be a number")
    if state_out is not None and not reasons:
        if not state_out.is_contiguous():
            reasons.append("unsupported_stride: state_out must be contiguous")
        elif wants_gradient(query, key, value, gate, beta, state) or state_out.requires_grad:
            reasons.append("unsupported_gradient: state_out is for calls without gradients")
        elif any(_overlap(state_out, t) and not (t is state and state.is_contiguous() and state.data_ptr() == state_out.data_ptr())
                 for t in (query, key, value, gate, beta, state, starts, lengths) if t is not None):
            reasons.append("unsupported_overlap: state_out may be the state itself and overlap nothing else that is read")
    return reasons


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    if a.numel() == 0 or b.numel() == 0:
        return False
    ends = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (a, b)]
    return ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]


def _heads(t: Optional[torch.Tensor]) -> _lib.Heads:
    return _lib.Heads(None, 0, 0, 0) if t is None else _lib.Heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _empty_like_heads(t: torch.Tensor) -> torch.Tensor:
    """A tensor of t's shape with steps and sequences in t's order in memory. No view of another: autograd lets several outputs of a function be written over
    only if they are none."""
    T, N = t.shape[:2]
    inner = t[0, 0].numel()
    step, row = (inner, T * inner) if t.stride(1) > t.stride(0) else (N * inner, inner)
    rest = (t.shape[3], 1) if t.dim() == 4 else (1,)
    return torch.empty_strided(t.shape, (step, row, *rest), dtype=t.dtype, device=t.device)


def _call(query, key, value, gate, beta, state, scale: float, starts, lengths) -> _lib.DeltaRuleCall:
    T, N, H, DK = query.shape
    code = _lib.dtype_code(query.dtype)
    gates = gate if gate is not None else beta
    return _lib.DeltaRuleCall(T, N, H, value.shape[2], DK, value.shape[3], code, code if gates is None else _lib.dtype_code(gates.dtype), scale, _heads(query), _heads(key),
                              _heads(value), _heads(gate), _heads(beta), _lib.ptr(starts), 0 if starts is None else starts.stride(0),
                              0 if starts is None else starts.stride(1), _lib.ptr(lengths), _lib.ptr(state))


def _forward(query, key, value, gate, beta, state, scale, starts, lengths, state_out, keep_marks: bool):
    lib = _lib.lib()
    with on_device_of(query):
        call = _call(query, key, value, gate, beta, state, scale, starts, lengths)
        out = _empty_like_heads(value)
        N, HV, DK, DV = value.shape[1], value.shape[2], key.shape[3], value.shape[3]
        last = torch.empty((N, HV, DK, DV), dtype=torch.float32, device=query.device) if state_out is None else state_out
        marks = torch.empty(lib.snnf_delta_rule_marks_bytes(ctypes.byref(call)) // 4, dtype=torch.float32, device=query.device) if keep_marks else None
        nbytes = lib.snnf_delta_rule_workspace_bytes(ctypes.byref(call), int(keep_marks))
        space = workspace(nbytes, query)
        _lib.check("snnf_delta_rule", lib.snnf_delta_rule(ctypes.byref(call), ctypes.byref(_heads(out)), last.data_ptr(), _lib.ptr(marks), _lib.ptr(space), nbytes,
                                                          _lib.current_stream(query.device)))
    if state_out is not None and not state_out.is_inference():
        torch.autograd.graph.increment_version(state_out)      # a graph that kept what it held before has to notice
    return out, last, marks


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, gate, beta, state, scale, starts, lengths):
        out, last, marks = _forward(query, key, value, gate, beta, state, scale, starts, lengths, None, True)
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        ctx.save_for_backward(query, key, value, gate, beta, starts, lengths, marks)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        refuse_observed("run_hip_delta_rule", ("the gradient of out", "the gradient of the last state"), dout, dlast)
        query, key, value, gate, beta, starts, lengths, marks = ctx.saved_tensors
        lib = _lib.lib()
        with on_device_of(query):
            call = _call(query, key, value, gate, beta, None, ctx.scale, starts, lengths)
            if dout is None:
                dout = torch.zeros(value.shape[3], dtype=value.dtype, device=value.device).expand(value.shape)
            dout = unit_rows(dout)
            dlast = None if dlast is None else dlast.contiguous()
            dquery, dkey, dvalue = (_empty_like_heads(t) for t in (query, key, value))
            dgate, dbeta = (None if t is None else _empty_like_heads(t) for t in (gate, beta))
            dstate = torch.empty((value.shape[1], value.shape[2], key.shape[3], value.shape[3]), dtype=torch.float32, device=query.device)
            nbytes = lib.snnf_delta_rule_backward_workspace_bytes(ctypes.byref(call))
            space = workspace(nbytes, query)
            views = [_heads(t) for t in (dout, dquery, dkey, dvalue, dgate, dbeta)]
            _lib.check("snnf_delta_rule_backward", lib.snnf_delta_rule_backward(
                ctypes.byref(call), marks.data_ptr(), ctypes.byref(views[0]), _lib.ptr(dlast), *(ctypes.byref(v) for v in views[1:]), dstate.data_ptr(),
                _lib.ptr(space), nbytes, _lib.current_stream(query.device)))
        grads = (dquery, dkey, dvalue, dgate, dbeta, dstate)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def run_hip_delta_rule(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, gate: Optional[torch.Tensor] = None, beta: Optional[torch.Tensor] = None,
                       state: Optional[torch.Tensor] = None, scale: Optional[float] = None, starts: Optional[torch.Tensor] = None,
                       lengths: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [T, N, Hv, Dv], state [N, Hv, Dk, Dv] after the last step).

    query, key: [T, N, H, Dk], value: [T, N, Hv, Dv], float32, bfloat16 or float16, steps outermost; a batch-first tensor goes in as `t.transpose(0, 1)`, a slice of
        a wider projection as it is: nothing is copied unless neighbouring elements of a head lie apart, and out has value's order in memory. Hv is a
        multiple of H, and value head j works with key and query head j // (Hv // H). Dk is at most 128, Dv at most 1024.
    gate: [T, N, Hv], the logarithm of the decay (None: no decay), at most 0 in earnest. Below -104, where less than 2^-149 would be left, the state is dropped as by a start.
    beta: [T, N, Hv], how much of a step's correction is taken (None: 1). With keys of length 1 at most, states stay bounded for beta up to 2.
        gate and beta are both of query's type or both float32. Gradients of float32 ones are float32's own beside 16-bit queries, too: products of the
        training passes then have three bfloat16 terms in place of two (4096 steps x 4 x 16 heads of 128: 1.51 ms in place of 1.11, 604 MB kept in place of 403).
    state: [N, Hv, Dk, Dv] float32 before the first step (None: zeros). The returned state is float32 and, unless state_out is given, new memory.
    scale: of the outputs, 1 / sqrt(Dk) if None.
    starts: [T, N] bool. Where set, the state is dropped before the step (several documents packed into one sequence).
    lengths: [N] int32 or int64, clamped to 0..T. Steps from there on are padding: what the operands hold there does not matter, out is 0, the state stays. Drafted
        tokens that are not accepted are left out this way: lengths is their number and one.
    state_out: memory for the returned state, contiguous, without gradients; may be state itself. Written in place as by an operation of torch: a backward pass that
        needs what it held before raises.

    Up to 16 steps without gradients are taken one by one, others in chunks of 64. Infinities and NaN of states and values stay in their columns, reach no
    step before them and none behind a start; those of keys, beta and gates, and of any operand in the gradients, may reach every step of their chunk.
    Sums, states and decays are float32 or more, out is rounded once. Differentiable once, backwards, in query, key, value, gate, beta and state (forward
    mode, torch.func and tracing are refused); the gradients of a head's queries and keys are summed over its value heads in a fixed order. What a call with
    gradients keeps for its backward pass is 96 KB for 64 steps of a value head of 128 x 128 (144 KB for float32 heads or gates), in proportion below, and the
    backward pass takes 37 KB more than that for itself.
    """
    module = native(query)
    if module is not None:
        known = module.delta_rule(query, key, value, gate, beta, state, scale, starts, lengths, state_out)
        if known is not None:
            return known
    reasons = check_delta_rule_support(query, key, value, gate, beta, state, scale, starts, lengths, state_out)
    if reasons:
        node = recorded(run_hip_delta_rule, (query, key, value, gate, beta, state),
                        {"scale": scale, "starts": starts, "lengths": lengths, "state_out": state_out})
        if node is not None:
            return node
        refuse("run_hip_delta_rule", reasons)
    T, N, H, DK = (int(n) for n in query.shape)
    HV, DV = int(value.shape[2]), int(value.shape[3])
    scale = DK ** -0.5 if scale is None else float(scale)
    if T == 0 or N == 0:
        last = torch.zeros((N, HV, DK, DV), dtype=torch.float32, device=query.device) if state is None else state.clone()
        if state_out is not None:
            last = state_out.copy_(last)
        out = value * (query.sum() + key.sum())      # nothing, but differentiable
        for t in (gate, beta):
            out = out if t is None else out * t.to(value.dtype)[..., None]
        return out, last
    query, key, value = unit_rows(query), unit_rows(key), unit_rows(value)
    if state is not None:
        state = state.contiguous()
    if lengths is not None:
        lengths = lengths.clamp(0, T).to(torch.int32).contiguous() if lengths.dtype == torch.int64 else lengths.contiguous()
    if wants_gradient(query, key, value, gate, beta, state):
        return _DeltaRule.apply(query, key, value, gate, beta, state, scale, starts, lengths)
    return _forward(query, key, value, gate, beta, state, scale, starts, lengths, state_out, False)[:2]
