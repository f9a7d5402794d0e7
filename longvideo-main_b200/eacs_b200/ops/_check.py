"""Argument checks shared by the operator modules (raise RuntimeError, as the
reference's TORCH_CHECKs do)."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def cuda_tensors(name: str, *ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        require(isinstance(t, torch.Tensor), f"{name}: expects tensors")
        require(t.is_cuda, f"{name}: expects CUDA tensors (eacs_b200 has no CPU path)")
        if dev is None:
            dev = t.device
        require(t.device == dev, f"{name}: tensors must be on one device")
    return dev


def on(dev: torch.device):
    """torch.cuda.device(dev) where dev is not the current device, else nothing."""
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


_tracing, _transforms = torch._C._get_tracing_state, torch._C._functorch.peek_interpreter_stack


def is_plain(*ts: torch.Tensor | None) -> bool:
    """Whether these are tensors whose values alone are asked for: none has a
    forward-mode tangent, none belongs to a torch.func transform, and nothing
    is being traced.  Kernels called by pointer see the values only; what would
    have to be carried along or recorded would be lost."""
    if forward_ad._current_level < 0 and _tracing() is None and _transforms() is None:
        return True
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        return False
    if torch.compiler.is_compiling():  # (whose graph ends where the kernel is called)
        return True
    return _tracing() is None and _transforms() is None


def require_plain(name: str, *ts: torch.Tensor | None) -> None:
    if not is_plain(*ts):
        raise RuntimeError(f"{name}: has no forward-mode derivative and runs under no torch.func transform "
                           "or torch.jit.trace")


def one_device(name: str, first: torch.Tensor, *ts: torch.Tensor | None) -> torch.device:
    """cuda_tensors for tensors of which some may be None, without a loop's cost on the way that passes."""
    dev = first.device if isinstance(first, torch.Tensor) else None
    if dev is None or dev.type != "cuda" or any(t is not None and (not isinstance(t, torch.Tensor) or t.device != dev)
                                                for t in ts):
        return cuda_tensors(name, first, *(t for t in ts if t is not None))
    return dev
