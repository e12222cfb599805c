"""Gated linear recurrence over a sequence on libsnnf (`snnf_gated_recurrence`), with its gradient.

The neuron of `fused_temporal_lif_state` without threshold and reset and with a leak of its own per step and channel, which is
what token models built from recurrences mix tokens with:

    form "leaky"    a = sigmoid(gate),  h_t = a h_{t-1} + (1 - a) x_t      (a constant gate is the charge rule of a neuron with
                                                                            1 / tau = 1 - sigmoid(gate))
    form "linear"   a = gate,           h_t = a h_{t-1} + x_t

The reference has no operator for this. There is no eager substitute: what the kernels do not take raises RuntimeError("unsupported_...").
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._sequence_common import check_activation, check_operand, check_unobserved, native, on_device_of, recorded, refuse, refuse_observed, unit_rows, unit_rows_in_place, wants_gradient, workspace

FORMS = {"leaky": 0, "linear": 1}
OPERANDS = ("x_seq", "gate_seq", "state", "starts", "lengths")


def check_gated_recurrence_support(x_seq, gate_seq, state=None, form: str = "leaky", starts=None, lengths=None) -> List[str]:
    """Reasons why a call is refused; empty if the kernels take it."""
    reasons: List[str] = []
    if form not in FORMS:
        reasons.append(f"unsupported_form: form must be one of {sorted(FORMS)}, got {form!r}")
    check_unobserved(reasons, OPERANDS, x_seq, gate_seq, state, starts, lengths)
    if not check_activation("x_seq", x_seq, reasons):
        return reasons
    if x_seq.dim() != 3:
        reasons.append(f"unsupported_rank: x_seq must be [T, N, D], got {x_seq.dim()} dimensions")
        return reasons
    T, N, D = (int(n) for n in x_seq.shape)
    if max(T, N, D) > 1 << 30:
        reasons.append(f"unsupported_shape: no dimension of x_seq may pass 2^30, got {(T, N, D)}")
    check_operand("gate_seq", gate_seq, x_seq.device, (T, N, D), (x_seq.dtype,), reasons)
    if state is not None:
        check_operand("state", state, x_seq.device, (N, D), (torch.float32,), reasons)
    if starts is not None:
        check_operand("starts", starts, x_seq.device, (T, N), (torch.bool,), reasons)
    if lengths is not None:
        check_operand("lengths", lengths, x_seq.device, (N,), (torch.int32, torch.int64), reasons)
    if not reasons:
        for name, step in (("x_seq", _step_of(x_seq)), ("gate_seq", _step_of(gate_seq)), ("h_seq", _steps_like(x_seq)[0])):
            if not _within_reach(x_seq, step):
                reasons.append(f"unsupported_stride: {name} has steps {step} elements apart, of which 16 may not pass 2 GiB")
    return reasons


def _steps_like(x: torch.Tensor) -> Tuple[int, int, int]:
    """Strides of a [T, N, D] tensor whose memory has steps and sequences in x's order: a batch-first tensor seen steps-first gives one again."""
    T, N, D = x.shape
    return (D, T * D, 1) if unit_rows_in_place(x) and x.stride(1) > x.stride(0) else (N * D, D, 1)


def _step_of(t: torch.Tensor) -> int:
    return t.stride(0) if unit_rows_in_place(t) else t.shape[1] * t.shape[2]        # of the copy


def _within_reach(x: torch.Tensor, step: int) -> bool:
    """The kernels reach the steps that a thread takes at once, up to 16, by offsets of 31 bits."""
    return (step * (min(x.shape[0], 16) - 1) + x.shape[2]) * x.element_size() < 0x7FFFFFFF


def _empty_like_steps(x: torch.Tensor) -> torch.Tensor:
    """A tensor of x's shape and order in memory. No view of another: autograd lets several outputs of a function be written over only if they are none."""
    return torch.empty_strided(x.shape, _steps_like(x), dtype=x.dtype, device=x.device)


def _series(t: torch.Tensor) -> Tuple[int, int, int]:
    return t.data_ptr(), t.stride(0), t.stride(1)


def _masks(starts, lengths) -> tuple:
    return (_lib.ptr(starts), 0 if starts is None else starts.stride(0), 0 if starts is None else starts.stride(1), _lib.ptr(lengths))


def _forward(x, gate, state, form: int, starts, lengths, keep_marks: bool):
    lib = _lib.lib()
    T, N, D = (int(n) for n in x.shape)
    code = _lib.dtype_code(x.dtype)
    with on_device_of(x):
        h = _empty_like_steps(x)
        last = torch.empty((N, D), dtype=torch.float32, device=x.device)
        marks = torch.empty(lib.snnf_gated_recurrence_marks_bytes(T, N, D, code) // 4, dtype=torch.float32, device=x.device) if keep_marks else None
        nbytes = lib.snnf_gated_recurrence_workspace_bytes(T, N, D, code, 0)
        space = workspace(nbytes, x)
        _lib.check("snnf_gated_recurrence", lib.snnf_gated_recurrence(
            *_series(x), *_series(gate), T, N, D, code, form, *_masks(starts, lengths), _lib.ptr(state), *_series(h), last.data_ptr(),
            _lib.ptr(marks), _lib.ptr(space), nbytes, _lib.current_stream(x.device)))
    return h, last, marks


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, form, starts, lengths):
        h, last, marks = _forward(x, gate, state, form, starts, lengths, True)
        ctx.set_materialize_grads(False)
        ctx.form = form
        ctx.save_for_backward(x, gate, starts, lengths, marks)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        refuse_observed("run_hip_gated_recurrence", ("the gradient of h_seq", "the gradient of the last state"), dh, dlast)
        x, gate, starts, lengths, marks = ctx.saved_tensors
        lib = _lib.lib()
        T, N, D = (int(n) for n in x.shape)
        code = _lib.dtype_code(x.dtype)
        with on_device_of(x):
            if dh is None:
                dh = torch.zeros(D, dtype=x.dtype, device=x.device).expand(T, N, D)
            elif not (unit_rows_in_place(dh) and _within_reach(dh, dh.stride(0))):
                dh = _empty_like_steps(x).copy_(dh)
            dlast = None if dlast is None else dlast.contiguous()
            dx, dgate = _empty_like_steps(x), _empty_like_steps(x)
            dstate = torch.empty((N, D), dtype=torch.float32, device=x.device)
            nbytes = lib.snnf_gated_recurrence_workspace_bytes(T, N, D, code, 1)
            space = workspace(nbytes, x)
            _lib.check("snnf_gated_recurrence_backward", lib.snnf_gated_recurrence_backward(
                *_series(x), *_series(gate), *_series(dh), T, N, D, code, ctx.form, *_masks(starts, lengths), marks.data_ptr(), _lib.ptr(dlast),
                *_series(dx), *_series(dgate), dstate.data_ptr(), _lib.ptr(space), nbytes, _lib.current_stream(x.device)))
        needs = ctx.needs_input_grad
        return dx if needs[0] else None, dgate if needs[1] else None, dstate if needs[2] else None, None, None, None


def run_hip_gated_recurrence(x_seq: torch.Tensor, gate_seq: torch.Tensor, state: Optional[torch.Tensor] = None, form: str = "leaky",
                             starts: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(h_seq [T, N, D], state [N, D] after the last step).

    x_seq, gate_seq: [T, N, D], float32, bfloat16 or float16, steps outermost as everywhere here; a batch-first tensor goes in as
        `t.transpose(0, 1)`, a slice of a wider projection or an expanded gate as it is: nothing is copied unless neighbouring channels lie
        apart, and h_seq has x_seq's order in memory. 16 steps may not pass 2 GiB: where sequences are that many, they go in batch-first.
    state: [N, D] float32 before the first step (None: zeros). The returned state is float32 and new memory; T = 0 returns it unchanged.
    starts: [T, N] bool. Where set, the state is dropped before the step (several documents packed into one sequence); what the state
        held, infinities and NaN among it, does not reach the steps from there on. Nothing else ends either.
    lengths: [N] int32 or int64, clamped to 0..T. Steps from there on are padding: what x_seq, gate_seq and starts hold there does not
        matter, h_seq is 0, the state stays.

    Gates of the linear form may pass 1 in magnitude: the 32 to 224 steps around such a gate are walked one by one, which takes up to seven times as long
    on a single long sequence. Other steps are joined by the products of their decays, and a product below 2^-149 leaves at most 2^-149 of the state.
    Arithmetic is float32 throughout, outputs are rounded once. Differentiable once, backwards, in x_seq, gate_seq and state
    (forward mode, torch.func and tracing are refused).
    """
    module = native(x_seq)
    if module is not None and form in FORMS:
        known = module.gated_recurrence(x_seq, gate_seq, state, starts, lengths, FORMS[form])
        if known is not None:
            return known
    reasons = check_gated_recurrence_support(x_seq, gate_seq, state, form, starts, lengths)
    if reasons:
        node = recorded(run_hip_gated_recurrence, (x_seq, gate_seq, state), {"form": form, "starts": starts, "lengths": lengths})
        if node is not None:
            return node
        refuse("run_hip_gated_recurrence", reasons)
    T, N, D = (int(n) for n in x_seq.shape)
    if T == 0:
        last = torch.zeros((N, D), dtype=torch.float32, device=x_seq.device) if state is None else state.clone()
        return x_seq * gate_seq, last        # nothing, but differentiable
    x, gate = unit_rows(x_seq), unit_rows(gate_seq)
    if state is not None:
        state = state.contiguous()
    if lengths is not None:
        lengths = lengths.clamp(0, T).to(torch.int32).contiguous() if lengths.dtype == torch.int64 else lengths.contiguous()
    if wants_gradient(x, gate, state):
        return _GatedRecurrence.apply(x, gate, state, FORMS[form], starts, lengths)
    h, last, _ = _forward(x, gate, state, FORMS[form], starts, lengths, False)
    return h, last
