"""What the sequence operators (gated recurrence, block norm, token scores) share on the host side."""
from __future__ import annotations

import contextlib
from typing import Iterable, List, Optional, Tuple

import torch
import torch.fx
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode
from torch.utils._python_dispatch import is_traceable_wrapper_subclass

from .. import _dispatch

SUPPORTED_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def recorded(function, operands: tuple, options: dict):
    """A call that the kernels do not take: None, or where torch.fx traces the program, which hands it stand-ins for tensors, the node that records it."""
    if any(isinstance(t, torch.fx.Proxy) for t in operands):
        return torch.overrides.handle_torch_function(function, operands, *operands, **options)
    return None


def refuse(operator: str, reasons: List[str]) -> None:
    if reasons:
        raise RuntimeError(f"{operator}: " + "; ".join(reasons))


def check_unobserved(reasons: List[str], names: Tuple[str, ...], *operands) -> None:
    """A tensor is its memory to the kernels, and their work is all there is to a call: what else travels with a tensor would be lost (a tangent silently),
    and a trace of torch's operations would hold the outputs' allocation and nothing that fills them."""
    module = native(next((t for t in operands if t is not None), None))
    if module is not None and module.unobserved(*operands):
        return
    if torch.jit.is_tracing() or get_proxy_mode() is not None:
        reasons.append("unsupported_tracing: torch.jit.trace and make_fx record torch's own operations only")
    for name, t in zip(names, operands):
        if not isinstance(t, torch.Tensor):
            continue
        if forward_ad.unpack_dual(t).tangent is not None:
            reasons.append(f"unsupported_forward_ad: {name} has a tangent, and there is no forward-mode derivative")
        try:
            t.untyped_storage()
        except (NotImplementedError, RuntimeError):
            reasons.append(f"unsupported_transform: {name} is wrapped by a transform (torch.func, vmap) and has no memory of its own")
        if is_traceable_wrapper_subclass(t):
            reasons.append(f"unsupported_subclass: {name} is a {type(t).__name__}, which wraps other tensors and has no address")


def refuse_observed(operator: str, names: Tuple[str, ...], *gradients) -> None:
    """The same of the gradients that autograd hands over."""
    reasons: List[str] = []
    check_unobserved(reasons, names, *gradients)
    refuse(operator, reasons)


def check_activation(name: str, t, reasons: List[str]) -> bool:
    """The tensor whose dtype and device the other operands have to match."""
    if not isinstance(t, torch.Tensor):
        reasons.append(f"{name} must be a tensor")
        return False
    if not t.is_cuda:
        reasons.append(f"unsupported_device: {name} is not on the GPU")
    if t.dtype not in SUPPORTED_DTYPES:
        reasons.append(f"unsupported_dtype: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    return not reasons


def check_operand(name: str, t, device: torch.device, shape: Tuple[int, ...], dtypes: Iterable[torch.dtype], reasons: List[str]) -> None:
    if not isinstance(t, torch.Tensor):
        reasons.append(f"{name} must be a tensor")
        return
    if t.device != device:
        reasons.append(f"unsupported_device: {name} is on {t.device}, not on {device}")
    if tuple(t.shape) != tuple(shape):
        reasons.append(f"unsupported_shape: {name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype not in tuple(dtypes):
        reasons.append(f"unsupported_dtype: {name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")


def native(t):
    """The dispatch module where a call on `t` may be plain enough for it (it answers None where it is not), else None."""
    return _dispatch.module() if isinstance(t, torch.Tensor) and t.is_cuda else None


def wants_gradient(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def on_device_of(t: torch.Tensor):
    """Kernels launch on the current HIP device: a context that makes it the tensor's."""
    if t.device.index is None or t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def unit_rows_in_place(t: torch.Tensor) -> bool:
    """Whether neighbouring elements of the last dimension lie next to each other."""
    return t.shape[-1] <= 1 or t.stride(-1) == 1


def unit_rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where they do, else a copy."""
    return t if unit_rows_in_place(t) else t.contiguous()


def workspace(nbytes: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    """Scratch memory from the caching allocator: of the current stream, and of the graph's own pool under capture, so that no two calls
    in flight share it."""
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def flat_rows(t: torch.Tensor) -> torch.Tensor:
    """[..., D] as [rows, D] with any stride between rows: a view where the leading dimensions allow one, else a copy."""
    t = unit_rows(t)
    if t.dim() == 2:
        return t
    if t.dim() == 1:
        return t.unsqueeze(0)
    lead = 1
    for n in t.shape[:-1]:
        lead *= int(n)
    try:
        return t.view(lead, t.shape[-1])
    except RuntimeError:
        return t.contiguous().view(lead, t.shape[-1])

