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
    """cuda_tensors for tensors of which some may be None, without its cost on the way that passes."""
    if isinstance(first, torch.Tensor) and first.is_cuda:
        index = first.get_device()
        for t in ts:
            if t is not None and (not isinstance(t, torch.Tensor) or t.get_device() != index):
                break
        else:
            return first.device
    return cuda_tensors(name, first, *(t for t in ts if t is not None))


def wants_grad(*ts: torch.Tensor | None) -> bool:
    """Whether gradients are enabled and one of these wants one."""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def dense(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.contiguous()


def packed(t: torch.Tensor | None) -> torch.Tensor | None:
    """A saved tensor as a kernel that reads it by its pointer alone expects it: dense and on 16 bytes.  (Saved-tensor hooks
    may give back a copy that is neither.)"""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def new_like(t: torch.Tensor | None) -> torch.Tensor | None:
    """An uninitialised dense tensor of t's shape, dtype and device."""
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


class _Once(torch.autograd.Function):
    """Gradients as they are, behind the n tensors that they depend on, which may not be differentiated."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tuple(None if g is None else g.view_as(g) for g in tensors[n:])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("these gradients can be differentiated once only (create_graph is not supported here)")


def once(backward):
    """For a backward that cannot be differentiated itself: with create_graph its gradients are those of a plain backward, and
    a backward through any of them raises.  (Left without a graph they would count as constants, and a penalty on them among
    other terms would lose its gradient without a word.)  All inputs that may want a gradient have to be saved tensors."""
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        roots = [t for t in (*ctx.saved_tensors, *grads) if t is not None and t.requires_grad]
        return _Once.apply(len(roots), *roots, *out)
    return run


def dense_last(t: torch.Tensor | None) -> torch.Tensor | None:
    """t, copied if its last dimension is not dense."""
    if t is None or t.stride(-1) == 1 or t.shape[-1] == 1:
        return t
    return t.contiguous()
