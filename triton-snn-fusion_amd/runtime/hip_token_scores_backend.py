"""Scores of given tokens (or classes) on libsnnf (`snnf_token_scores`): log probability, entropy, the most likely alternatives, with gradient.

What follows the classifier (`fused_temporal_lif_avgpool_linear`, `spike_pool_linear`) or the last projection of a token model: logits
are read once, and nothing of their size is written but, in training, their gradient. The reference has no operator for this. There is no eager
substitute: what the kernels do not take raises RuntimeError("unsupported_...").
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._sequence_common import check_activation, check_operand, check_unobserved, flat_rows, native, on_device_of, recorded, refuse, refuse_observed, wants_gradient, workspace

MAX_ALTERNATIVES = 64


class TokenScores(NamedTuple):
    """logprob, entropy: [...] float32. top_logprob [..., top_k] float32, top_token [..., top_k] int64; None where top_k is 0."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_token: Optional[torch.Tensor]


def check_token_scores_support(logits, tokens=None, top_k: int = 0) -> List[str]:
    """Reasons why a call is refused; empty if the kernels take it."""
    reasons: List[str] = []
    check_unobserved(reasons, ("logits", "tokens"), logits, tokens)
    if not check_activation("logits", logits, reasons):
        return reasons
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= 1 << 30:
        reasons.append(f"unsupported_shape: rows of 1 to 2^30 logits, got {tuple(logits.shape)}")
        return reasons
    if tokens is not None:
        check_operand("tokens", tokens, logits.device, tuple(logits.shape[:-1]), (torch.int64, torch.int32), reasons)
    if not 0 <= top_k <= min(MAX_ALTERNATIVES, int(logits.shape[-1])):
        reasons.append(f"unsupported_top_k: 0 to {MAX_ALTERNATIVES} alternatives and no more than logits, got {top_k} of {int(logits.shape[-1])}")
    return reasons


def _forward(logits, tokens, top_k: int, keep_stats: bool):
    lib = _lib.lib()
    rows, V = logits.shape
    with on_device_of(logits):
        logprob, entropy = (torch.empty(rows, dtype=torch.float32, device=logits.device) for _ in range(2))
        top_logprob = torch.empty((rows, top_k), dtype=torch.float32, device=logits.device) if top_k else None
        top_token = torch.empty((rows, top_k), dtype=torch.int64, device=logits.device) if top_k else None
        stats = torch.empty((rows, 2), dtype=torch.float32, device=logits.device) if keep_stats else None
        nbytes = lib.snnf_token_scores_workspace_bytes(rows, V, top_k)
        space = workspace(nbytes, logits)
        _lib.check("snnf_token_scores", lib.snnf_token_scores(
            logits.data_ptr(), logits.stride(0), rows, V, _lib.dtype_code(logits.dtype), _lib.ptr(tokens), top_k, logprob.data_ptr(),
            entropy.data_ptr(), _lib.ptr(top_logprob), _lib.ptr(top_token), _lib.ptr(stats), _lib.ptr(space), nbytes,
            _lib.current_stream(logits.device)))
    return logprob, entropy, top_logprob, top_token, stats


class _TokenScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k):
        logprob, entropy, top_logprob, top_token, stats = _forward(logits, tokens, top_k, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, stats, entropy)
        if not top_k:
            return logprob, entropy
        ctx.mark_non_differentiable(top_logprob, top_token)
        return logprob, entropy, top_logprob, top_token

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprob, d_entropy, *_):
        refuse_observed("run_hip_token_scores", ("the gradient of logprob", "the gradient of entropy"), d_logprob, d_entropy)
        logits, tokens, stats, entropy = ctx.saved_tensors
        rows, V = logits.shape
        with on_device_of(logits):
            grads = [None if d is None else d.contiguous() for d in (d_logprob, d_entropy)]
            d_logits = torch.empty((rows, V), dtype=logits.dtype, device=logits.device)
            _lib.check("snnf_token_scores_backward", _lib.lib().snnf_token_scores_backward(
                logits.data_ptr(), logits.stride(0), rows, V, _lib.dtype_code(logits.dtype), _lib.ptr(tokens), stats.data_ptr(),
                entropy.data_ptr(), *(_lib.ptr(d) for d in grads), d_logits.data_ptr(), _lib.current_stream(logits.device)))
        return d_logits, None, None


def run_hip_token_scores(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0) -> TokenScores:
    """Scores of rows of logits.

    logits: [..., V] float32, bfloat16 or float16; rows may lie any distance apart. Minus infinity masks an entry; a row of nothing else has
        logprob -inf, entropy 0 and no gradient.
    tokens: [...] int64 or int32, the token given for each row; outside [0, V) (-100, say), or without tokens, logprob is 0 and passes no gradient.
    top_k: alternatives a row, up to 64: the most likely first, equal ones by the lower index. They carry no gradient.

    Arithmetic is float32; logprob and entropy are differentiable once, backwards, in the logits (forward mode, torch.func and tracing are refused).
    """
    module = native(logits)
    if module is not None:
        known = module.token_scores(logits, tokens, top_k)
        if known is not None:
            return TokenScores(*known)
    reasons = check_token_scores_support(logits, tokens, top_k)
    if reasons:
        node = recorded(run_hip_token_scores, (logits, tokens), {"top_k": top_k})
        if node is not None:
            return node
        refuse("run_hip_token_scores", reasons)
    lead = logits.shape[:-1]
    if logits.numel() == 0:
        zeros = logits.sum(-1, dtype=torch.float32)        # no rows, but differentiable
        return TokenScores(zeros, zeros.clone(), logits.new_zeros((*lead, top_k), dtype=torch.float32) if top_k else None,
                           logits.new_zeros((*lead, top_k), dtype=torch.int64) if top_k else None)
    rows = flat_rows(logits)
    if tokens is not None:
        tokens = tokens.reshape(-1).to(torch.int64).contiguous()
    if wants_gradient(rows):
        out = _TokenScores.apply(rows, tokens, top_k)
        logprob, entropy, top_logprob, top_token = out if top_k else (*out, None, None)
    else:
        logprob, entropy, top_logprob, top_token, _ = _forward(rows, tokens, top_k, False)
    return TokenScores(logprob.view(lead), entropy.view(lead), None if top_logprob is None else top_logprob.view(*lead, top_k),
                       None if top_token is None else top_token.view(*lead, top_k))
