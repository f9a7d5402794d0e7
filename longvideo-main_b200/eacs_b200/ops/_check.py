"""Argument checks shared by the operator modules (raise RuntimeError, as the
reference's TORCH_CHECKs do)."""
from __future__ import annotations

import contextlib

import torch


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


def one_device(name: str, first: torch.Tensor, *ts: torch.Tensor | None) -> torch.device:
    """cuda_tensors for tensors of which some may be None, without a loop's cost on the way that passes."""
    dev = first.device if isinstance(first, torch.Tensor) else None
    if dev is None or dev.type != "cuda" or any(t is not None and (not isinstance(t, torch.Tensor) or t.device != dev)
                                                for t in ts):
        return cuda_tensors(name, first, *(t for t in ts if t is not None))
    return dev
