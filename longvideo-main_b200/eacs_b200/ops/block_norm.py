"""The norms before and after a block, with its gate and its scaled residual (eacs_norm_*).

With rms(v) = v / sqrt(mean(v^2) + eps) over the last dimension:

    gated_norm:     y = rms(x) weight silu(gate)
    residual_norm:  u = x, or rms(x) post_weight;  u = u silu(gate) where there is a gate
                    s = residual + scale u,  y = rms(s) weight;  returns (y, s)

`gated_norm` follows a recurrence (the heads of gated_delta_rule, each normed by
itself as a last dimension of V; selective_ssm has its gate inside);
`residual_norm` adds a block's output to the residual stream and norms the sum
for the next block, in one pass over both.  They stand beside `layer_norm`.
Statistics and sums are float32 and each output is rounded once: the sum s is
normed before it is rounded.  Differentiable in every tensor, through y and s;
the backward takes everything again from the inputs, and the gradients of
weight, scale and post_weight are the same bits on every run.

Gradients are reverse mode, once; forward-mode, torch.func or traced calls are
refused.
"""
from __future__ import annotations

import torch
from torch import Tensor

from .. import _lib
from ._check import on, one_device, require_plain
from .layer_norm import MAX_D, _rows


def _args(x, gate, residual, weight, scale, post, post_norm, eps):
    """EacsNorm, and the tensors that it points into."""
    d = x.shape[-1]
    (xr, xs), (gr, gs), (rr, rs) = ((None, 0) if t is None else _rows(t, d) for t in (x, gate, residual))
    p = lambda t: 0 if t is None else t.data_ptr()
    w = next((t for t in (weight, scale, post) if t is not None), None)
    return _lib.NORM.pack(xr.data_ptr(), p(gr), p(rr), p(weight), p(scale), p(post), xs, gs, rs, x.numel() // d, d, eps,
                          _lib.DTYPE_CODES[x.dtype], 0 if w is None else _lib.DTYPE_CODES[w.dtype], int(post_norm)), (xr, gr, rr)


def _forward(x, gate, residual, weight, scale, post, post_norm, eps, dev):
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    s = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    if y.numel():
        p, held = _args(x, gate, residual, weight, scale, post, post_norm, eps)
        with on(dev):
            _lib.check(_lib.lib().eacs_norm_fwd(p, y.data_ptr(), _lib.ptr(s), _lib.raw_stream(dev.index)), "eacs_norm_fwd")
    return y, s


class BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, residual, weight, scale, post, post_norm, eps, dev):
        ctx.save_for_backward(x, gate, residual, weight, scale, post)
        ctx.post_norm, ctx.eps, ctx.dev = post_norm, eps, dev
        ctx.set_materialize_grads(False)
        y, s = _forward(x, gate, residual, weight, scale, post, post_norm, eps, dev)
        return y if s is None else (y, s)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds=None):
        x, gate, residual, weight, scale, post = ctx.saved_tensors
        if dy is None and ds is None:
            return (None,) * 9
        need, dev, d = ctx.needs_input_grad, ctx.dev, x.shape[-1]
        weight, scale, post = (None if t is None else t.contiguous() for t in (weight, scale, post))
        like = lambda t: torch.empty(t.shape, dtype=t.dtype, device=dev)
        dw, dc, dp = (like(t) if need[i] else None for i, t in ((3, weight), (4, scale), (5, post)))
        if x.numel() == 0:
            zero = lambda t: None if t is None else t.zero_()
            return like(x), None if gate is None else like(gate), None if residual is None else like(residual), zero(dw), zero(dc), \
                zero(dp), None, None, None
        p, held = _args(x, gate, residual, weight, scale, post, ctx.post_norm, ctx.eps)
        dx, dg = like(x), None if gate is None else like(gate)
        same = residual is not None and gate is None and scale is None and not ctx.post_norm  # as a sum's backward gives it
        dr = None if residual is None or same else like(residual)
        (gr, gs), (sr, ss) = ((None, 0) if t is None else _rows(t, d) for t in (dy, ds))
        L_ = _lib.lib()
        ws = None
        if dw is not None or dc is not None or dp is not None:
            ws = torch.empty(int(L_.eacs_norm_bwd_workspace_size(p)), dtype=torch.uint8, device=dev)
        with on(dev):
            _lib.check(L_.eacs_norm_bwd(p, _lib.ptr(gr), gs, _lib.ptr(sr), ss, dx.data_ptr(), _lib.ptr(dg), _lib.ptr(dr),
                                        _lib.ptr(dw), _lib.ptr(dc), _lib.ptr(dp), _lib.ptr(ws), 0 if ws is None else ws.numel(),
                                        _lib.raw_stream(dev.index)), "eacs_norm_bwd")
        return dx if need[0] else None, dg, dx if same and need[2] else dr, dw, dc, dp, None, None, None


def _run(name, x, gate, residual, weight, scale, post, post_norm, eps):
    dev = one_device(name, x, gate, residual, weight, scale, post)
    require_plain(name, x, gate, residual, weight, scale, post)
    if x.dim() < 1 or x.dtype not in _lib.DTYPE_CODES:
        raise RuntimeError(f"{name}: unsupported x, {x.dtype} of {x.dim()} dimensions")
    d = x.shape[-1]
    if not 1 <= d <= MAX_D:
        raise RuntimeError(f"{name}: d={d} must be 1 to {MAX_D}")
    for n, t in (("gate", gate), ("residual", residual)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise RuntimeError(f"{name}: {n} must have x's shape and dtype")
    dtypes = set()
    for t in (weight, scale, post):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != d or t.dtype not in _lib.DTYPE_CODES:
                raise RuntimeError(f"{name}: weight, scale and post_weight must be ({d},), float32, float16 or bfloat16")
            dtypes.add(t.dtype)
    if len(dtypes) > 1:
        raise RuntimeError(f"{name}: weight, scale and post_weight must have one dtype")
    weight, scale, post = (None if t is None else t.contiguous() for t in (weight, scale, post))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, residual, weight, scale, post)):
        out = BlockNormFunction.apply(x, gate, residual, weight, scale, post, post_norm, float(eps), dev)
        return out if residual is not None else (out, None)
    return _forward(x, gate, residual, weight, scale, post, post_norm, float(eps), dev)


def gated_norm(x: Tensor, gate: Tensor | None = None, weight: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """rms(x) weight silu(gate) over the last dimension, in x's dtype.

    x (..., d) float32 / float16 / bfloat16, d up to 8192; gate like x, or None
    (no gate); weight (d) of one of those dtypes, or None (ones)."""
    return _run("gated_norm", x, gate, None, weight, None, None, True, eps)[0]


def residual_norm(x: Tensor, residual: Tensor, weight: Tensor | None = None, scale: Tensor | None = None,
                  gate: Tensor | None = None, post_weight: Tensor | None = None, eps: float = 1e-5) -> tuple[Tensor, Tensor]:
    """(y, s) with s = residual + scale u and y = rms(s) weight, both in x's
    dtype; u is x, normed by itself where there is a post_weight, times
    silu(gate) where there is a gate.

    residual and gate like x; weight, scale and post_weight (d) of one dtype.
    Without weight or scale ones are taken."""
    if not isinstance(residual, Tensor):
        raise RuntimeError("residual_norm: expects a residual")
    return _run("residual_norm", x, gate, residual, weight, scale, post_weight, post_weight is not None, eps)
