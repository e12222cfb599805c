"""Norms behind and in front of a block, fused with its gate and residual scale, on libsnnf (`snnf_block_norm`), with gradients.

    residual' = residual + residual_scale * scale * act(gate) * norm(branch) * branch_weight
    normed    = norm(residual') * next_weight

is what lies between the block that gave `branch` (a recurrence, a feed-forward part) and the next one, which takes `normed`: for a
network of token-wise blocks what folded BatchNorm, residual and neuron are for the convolutions. One launch and one pass over the
tensors; without a branch it is the norm in front of the first block. The reference has no operator for this. There is no eager substitute:
what the kernels do not take raises RuntimeError("unsupported_...").
"""
from __future__ import annotations

from typing import List, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._sequence_common import SUPPORTED_DTYPES, check_activation, check_operand, check_unobserved, flat_rows, native, on_device_of, recorded, refuse, refuse_observed, wants_gradient, workspace

KINDS = {"rms": 0, "layer": 1}
GATE_FORMS = {"sigmoid": 1, "silu": 2}
MAX_WIDTH = 16384
OPERANDS = ("residual", "branch", "gate", "branch_weight", "next_weight", "scale")


def check_block_norm_support(residual, branch=None, gate=None, branch_weight=None, next_weight=None, scale=None, kind: str = "rms",
                             gate_form: str = "silu", eps: float = 1e-6) -> List[str]:
    """Reasons why a call is refused; empty if the kernels take it."""
    reasons: List[str] = []
    if kind not in KINDS:
        reasons.append(f"unsupported_kind: kind must be one of {sorted(KINDS)}, got {kind!r}")
    if gate_form not in GATE_FORMS:
        reasons.append(f"unsupported_gate: gate_form must be one of {sorted(GATE_FORMS)}, got {gate_form!r}")
    if not eps >= 0.0:
        reasons.append(f"unsupported_eps: eps must not be negative, got {eps}")
    check_unobserved(reasons, OPERANDS, residual, branch, gate, branch_weight, next_weight, scale)
    if not check_activation("residual", residual, reasons):
        return reasons
    if residual.dim() < 1 or not 1 <= residual.shape[-1] <= MAX_WIDTH:
        reasons.append(f"unsupported_shape: rows of 1 to {MAX_WIDTH} elements, got {tuple(residual.shape)}")
        return reasons
    shape, D, device = tuple(residual.shape), int(residual.shape[-1]), residual.device
    if branch is None:
        for name, t in (("gate", gate), ("branch_weight", branch_weight)):
            if t is not None:
                reasons.append(f"unsupported_gate: {name} without a branch")
        if isinstance(scale, torch.Tensor):
            reasons.append("unsupported_gate: scale without a branch")
        dtype = residual.dtype
    else:
        allowed = SUPPORTED_DTYPES if residual.dtype == torch.float32 else (residual.dtype,)
        check_operand("branch", branch, device, shape, allowed, reasons)
        dtype = getattr(branch, "dtype", residual.dtype)
        if gate is not None:
            check_operand("gate", gate, device, shape, (dtype,), reasons)
    vectors = [(n, t) for n, t in (("branch_weight", branch_weight), ("next_weight", next_weight), ("scale", scale)) if isinstance(t, torch.Tensor)]
    for name, t in vectors:
        check_operand(name, t, device, (D,), (dtype, torch.float32), reasons)
    if len({t.dtype for _, t in vectors}) > 1:
        reasons.append("unsupported_dtype: branch_weight, next_weight and scale must be of one dtype")
    return reasons


def _row(t: Optional[torch.Tensor]) -> Tuple[Optional[int], int]:
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


def _codes(residual, branch, vectors) -> Tuple[int, int, int]:
    dtype = residual.dtype if branch is None else branch.dtype
    vector = next((t.dtype for t in vectors if t is not None), dtype)
    return _lib.dtype_code(residual.dtype), _lib.dtype_code(dtype), _lib.dtype_code(vector)


def _forward(residual, branch, gate, vectors, factor, kind, gate_form, eps, keep_stats):
    rows, D = residual.shape
    like = residual if branch is None else branch
    with on_device_of(residual):
        out = None if branch is None else torch.empty((rows, D), dtype=residual.dtype, device=residual.device)
        normed = torch.empty((rows, D), dtype=like.dtype, device=residual.device)
        stats = torch.empty((rows, 4), dtype=torch.float32, device=residual.device) if keep_stats else None
        _lib.check("snnf_block_norm", _lib.lib().snnf_block_norm(
            *_row(residual), *_row(branch), *_row(gate), *(_lib.ptr(t) for t in vectors), factor, rows, D, *_codes(residual, branch, vectors),
            kind, gate_form if gate is not None else 0, eps, _lib.ptr(out), normed.data_ptr(), _lib.ptr(stats), _lib.current_stream(residual.device)))
    return out, normed, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, gate, branch_weight, next_weight, scale, factor, kind, gate_form, eps):
        vectors = (branch_weight, next_weight, scale)
        out, normed, stats = _forward(residual, branch, gate, vectors, factor, kind, gate_form, eps, True)
        ctx.set_materialize_grads(False)
        ctx.options = (factor, kind, gate_form)
        ctx.save_for_backward(residual, branch, gate, *vectors, stats)
        return (residual.new_empty(0) if out is None else out), normed

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_normed):
        refuse_observed("run_hip_block_norm", ("the gradient of residual'", "the gradient of normed"), d_out, d_normed)
        residual, branch, gate, *vectors, stats = ctx.saved_tensors
        factor, kind, gate_form = ctx.options
        rows, D = residual.shape
        lib = _lib.lib()
        with on_device_of(residual):
            d_out = None if branch is None or d_out is None else flat_rows(d_out)
            d_normed = None if d_normed is None else flat_rows(d_normed)
            grads = [None if t is None else torch.empty((rows, D), dtype=t.dtype, device=t.device) for t in (residual, branch, gate)]
            grads += [torch.empty_like(t) if t is not None and need else None for t, need in zip(vectors, ctx.needs_input_grad[3:6])]
            nbytes = lib.snnf_block_norm_backward_workspace_bytes(rows, D)
            space = workspace(nbytes, residual)
            _lib.check("snnf_block_norm_backward", lib.snnf_block_norm_backward(
                *_row(residual), *_row(branch), *_row(gate), *(_lib.ptr(t) for t in vectors), factor, *_row(d_out), *_row(d_normed),
                stats.data_ptr(), rows, D, *_codes(residual, branch, vectors), kind, gate_form if gate is not None else 0,
                *(_lib.ptr(t) for t in grads), space.data_ptr(), nbytes, _lib.current_stream(residual.device)))
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def run_hip_block_norm(residual: torch.Tensor, branch: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                       branch_weight: Optional[torch.Tensor] = None, next_weight: Optional[torch.Tensor] = None,
                       scale: Union[torch.Tensor, float, None] = None, kind: str = "rms", gate_form: str = "silu",
                       eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(residual', normed), both [..., D].

    residual: [..., D], D <= 16384; float32, bfloat16 or float16. A float32 residual may stand next to 16-bit branches: it stays float32,
        `normed` is of the branch's dtype.
    branch: the block's output, or None: residual' is the residual itself and normed its norm.
    gate: what the block's output is multiplied with after `gate_form`: "silu" (gate * sigmoid(gate)) or "sigmoid"; None: nothing.
    branch_weight, next_weight: [D], None: ones. scale: [D] (a learnt scale per channel), a number, or None. Vectors are float32 or of the
        branch's dtype, all of one.
    kind: "rms", or "layer" with the mean taken out.

    Leading dimensions that are one stride apart, slices of wider projections among them, go in without copies. Arithmetic is float32
    throughout (normed comes from residual' before its rounding), outputs are rounded once. Differentiable once, backwards, in all tensors
    (forward mode, torch.func and tracing are refused); the vectors' gradients are sums in a fixed order.
    """
    learnt = isinstance(scale, torch.Tensor)
    module = native(residual)
    if module is not None and kind in KINDS and gate_form in GATE_FORMS and eps >= 0.0:
        known = module.block_norm(residual, branch, gate, branch_weight, next_weight, scale if learnt else None,
                                  1.0 if learnt or scale is None else scale, KINDS[kind], GATE_FORMS[gate_form], eps)
        if known is not None:
            return known
    reasons = check_block_norm_support(residual, branch, gate, branch_weight, next_weight, scale, kind, gate_form, eps)
    if reasons:
        node = recorded(run_hip_block_norm, (residual, branch, gate, branch_weight, next_weight, scale), {"kind": kind, "gate_form": gate_form, "eps": eps})
        if node is not None:
            return node
        refuse("run_hip_block_norm", reasons)
    factor = 1.0
    if not learnt and scale is not None:
        factor, scale = float(scale), None
    shape = residual.shape
    like = residual if branch is None else branch
    if residual.numel() == 0:        # no rows, but differentiable in every operand
        none = like.clone()
        for t in (residual, gate, branch_weight, next_weight, scale):
            none = none if t is None else none * t.to(like.dtype)
        return (residual if branch is None else none.to(residual.dtype)), none
    rows = [None if t is None else flat_rows(t) for t in (residual, branch, gate)]
    vectors = [None if t is None else t.contiguous() for t in (branch_weight, next_weight, scale)]
    options = (factor, KINDS[kind], GATE_FORMS[gate_form], float(eps))
    if wants_gradient(*rows, *vectors):
        out, normed = _BlockNorm.apply(*rows, *vectors, *options)
    else:
        out, normed, _ = _forward(*rows, vectors, *options, False)
    return (residual if branch is None else out.view(shape)), normed.view(shape)
