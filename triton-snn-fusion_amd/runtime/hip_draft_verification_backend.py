"""Verification of drafted tokens on libsnnf (`snnf_draft_verification`): how many of a request's drafts stand, and the token behind them.

What follows the last projection of a token model that is served with drafts, next to `run_hip_token_scores`: the drafts of a smaller model (or of a look-up) are taken as far as the
target's distribution allows, so that every token is distributed as the target's own. The reference has no operator for this. There is no eager substitute:
what the kernels do not take raises RuntimeError("unsupported_...").
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Union

import torch

from .. import _lib
from ._sequence_common import check_activation, check_operand, check_unobserved, native, on_device_of, recorded, refuse, unit_rows, workspace

MAX_DRAFTS = 64
OPERANDS = ("logits", "drafts", "uniforms", "noise", "draft_logits", "temperature", "lengths")


class DraftVerification(NamedTuple):
    """tokens: [N, K + 1] int64, the accepted drafts, the token behind them, then -100. accepted: [N] int32."""

    tokens: torch.Tensor
    accepted: torch.Tensor


def check_draft_verification_support(logits, drafts, uniforms, noise, draft_logits=None, temperature: Union[float, torch.Tensor] = 1.0, lengths=None) -> List[str]:
    """Reasons why a call is refused; empty if the kernels take it."""
    reasons: List[str] = []
    check_unobserved(reasons, OPERANDS, logits, drafts, uniforms, noise, draft_logits, temperature, lengths)
    if not check_activation("logits", logits, reasons):
        return reasons
    if logits.dim() != 3 or logits.shape[1] < 1:
        reasons.append(f"unsupported_rank: logits must be [N, K + 1, V], got {tuple(logits.shape)}")
        return reasons
    N, K, V = int(logits.shape[0]), int(logits.shape[1]) - 1, int(logits.shape[2])
    if K > MAX_DRAFTS or N > 1 << 20 or not 1 <= V <= 1 << 30:
        reasons.append(f"unsupported_shape: at most {MAX_DRAFTS} drafts of 2^20 requests and 1 to 2^30 logits, got K={K}, N={N}, V={V}")
    check_operand("drafts", drafts, logits.device, (N, K), (torch.int64, torch.int32), reasons)
    check_operand("uniforms", uniforms, logits.device, (N, K), (torch.float32,), reasons)
    check_operand("noise", noise, logits.device, (N, V), (torch.float32,), reasons)
    if draft_logits is not None:
        check_operand("draft_logits", draft_logits, logits.device, (N, K, V), (logits.dtype,), reasons)
    if isinstance(temperature, torch.Tensor):
        check_operand("temperature", temperature, logits.device, (N,), (torch.float32,), reasons)
    elif not isinstance(temperature, (int, float)):
        reasons.append("temperature must be a number or a tensor")
    if lengths is not None:
        check_operand("lengths", lengths, logits.device, (N,), (torch.int32, torch.int64), reasons)
    return reasons


def run_hip_draft_verification(logits: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor, noise: torch.Tensor, draft_logits: Optional[torch.Tensor] = None,
                               temperature: Union[float, torch.Tensor] = 1.0, lengths: Optional[torch.Tensor] = None) -> DraftVerification:
    """Takes drafts as far as they stand and draws the token behind them.

    logits: [N, K + 1, V] float32, bfloat16 or float16, the target's at each draft and behind the last; rows may lie any distance apart. Minus infinity masks an entry.
    drafts: [N, K] int64 or int32; one outside [0, V) does not stand. K is at most 64 and may be 0 (a draw alone).
    uniforms: [N, K] float32 in [0, 1): draft x stands if uniform * q(x) < p(x), p = softmax(logits / temperature), q the draft's.
    noise: [N, V] float32, exponentially distributed (`torch.empty(N, V, device=...).exponential_()`): the token is the one of the largest
        r / noise, the lowest index where they are equal; r = p behind drafts that all stand, else max(p - q, 0) (p, should nothing be left). Taken as it is
        written whatever the noise: an entry of r = 0 (a masked one, too) has 0 and is the largest where no entry of r > 0 has noise above 0; r > 0 over NaN is left out.
    draft_logits: [N, K, V] of logits' type, what drafts were drawn from, at the same temperature. None: drafts without a distribution, q(x) = 1.
    temperature: a number, rounded to float32, or [N] float32; infinity makes what is not masked equal. Where it is not above 0 the request is answered greedily: drafts stand while they are the largest logit (the
        lowest index among equals), and p is 1 there and 0 elsewhere for the token behind them.
    lengths: [N] int32 or int64, clamped to 0..K, how many drafts each request has; what lies behind them is not read.

    Decisions are those of float64 on the given numbers: float32 comes with bounds of its error, and a request of which it cannot tell two numbers apart is
    worked out again in float64, which adds 0.6 ms at 128000 logits (on random numbers, in one call of 256 requests in a hundred). A target's row of
    which nothing is left (masked, or not finite) lets no draft stand, and its token is -100. A draft's row of which nothing is left stands for no
    distribution: its draft does not stand, and r = p. What a recurrent state takes of such a step is `lengths=accepted + 1`.
    Nothing is differentiable.
    """
    module = native(logits)
    if module is not None:
        known = module.verify_drafts(logits, drafts, uniforms, noise, draft_logits, temperature, lengths)
        if known is not None:
            return DraftVerification(*known)
    reasons = check_draft_verification_support(logits, drafts, uniforms, noise, draft_logits, temperature, lengths)
    if reasons:
        node = recorded(run_hip_draft_verification, (logits, drafts, uniforms, noise), {"draft_logits": draft_logits, "temperature": temperature, "lengths": lengths})
        if node is not None:
            return node
        refuse("run_hip_draft_verification", reasons)
    N, K, V = int(logits.shape[0]), int(logits.shape[1]) - 1, int(logits.shape[2])
    lib = _lib.lib()
    with on_device_of(logits), torch.no_grad():
        tokens = torch.empty((N, K + 1), dtype=torch.int64, device=logits.device)
        accepted = torch.empty(N, dtype=torch.int32, device=logits.device)
        if N == 0:
            return DraftVerification(tokens, accepted)
        logits, noise = unit_rows(logits), unit_rows(noise)
        draft_logits = None if draft_logits is None or K == 0 else unit_rows(draft_logits)
        drafts, uniforms = drafts.to(torch.int64).contiguous(), uniforms.contiguous()
        each = temperature.contiguous() if isinstance(temperature, torch.Tensor) else None
        if lengths is not None:
            lengths = lengths.clamp(0, K).to(torch.int32).contiguous() if lengths.dtype == torch.int64 else lengths.contiguous()
        nbytes = lib.snnf_draft_verification_workspace_bytes(N, K, V, int(draft_logits is not None))
        space = workspace(nbytes, logits)
        strides = (0, 0) if draft_logits is None else draft_logits.stride()[:2]
        _lib.check("snnf_draft_verification", lib.snnf_draft_verification(
            logits.data_ptr(), *logits.stride()[:2], _lib.ptr(draft_logits), *strides, N, K, V, _lib.dtype_code(logits.dtype), drafts.data_ptr(), uniforms.data_ptr(),
            noise.data_ptr(), noise.stride(0), _lib.ptr(lengths), 1.0 if each is not None else float(temperature), _lib.ptr(each), tokens.data_ptr(), accepted.data_ptr(),
            space.data_ptr(), nbytes, _lib.current_stream(logits.device)))
    return DraftVerification(tokens, accepted)
