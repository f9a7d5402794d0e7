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
from ._check import dense, new_like, on, once, one_device, require_plain, wants_grad
from .layer_norm import MAX_D, _rows


def _args(x, gate, residual, weight, scale, post, post_norm, eps):
    """EacsNorm, and the tensors that it points into."""
    d = x.shape[-1]
    xr, xs = _rows(x, d)
    gr, gs = (None, 0) if gate is None else _rows(gate, d)
    rr, rs = (None, 0) if residual is None else _rows(residual, d)
    w = weight if weight is not None else scale if scale is not None else post
    return _lib.NORM.pack(xr.data_ptr(), 0 if gr is None else gr.data_ptr(), 0 if rr is None else rr.data_ptr(),
                          0 if weight is None else weight.data_ptr(), 0 if scale is None else scale.data_ptr(),
                          0 if post is None else post.data_ptr(), xs, gs, rs, x.numel() // d, d, eps,
                          _lib.DTYPE_CODES[x.dtype], 0 if w is None else _lib.DTYPE_CODES[w.dtype], post_norm), (xr, gr, rr)


def _forward(x, gate, residual, weight, scale, post, post_norm, eps, dev):
    y = new_like(x)
    s = None if residual is None else new_like(x)
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
    @once
    def backward(ctx, dy, ds=None):
        x, gate, residual, weight, scale, post = ctx.saved_tensors
        if dy is None and ds is None:
            return (None,) * 9
        need, dev, d = ctx.needs_input_grad, ctx.dev, x.shape[-1]
        weight, scale, post = dense(weight), dense(scale), dense(post)
        dw = new_like(weight) if need[3] else None
        dc = new_like(scale) if need[4] else None
        dp = new_like(post) if need[5] else None
        same = residual is not None and gate is None and scale is None and not ctx.post_norm  # as a sum's backward gives it
        dx, dg = new_like(x), new_like(gate)
        dr = None if same else new_like(residual)
        if x.numel() == 0:
            zero = lambda t: None if t is None else t.zero_()
            return dx, dg, dx if same else dr, zero(dw), zero(dc), zero(dp), None, None, None
        p, held = _args(x, gate, residual, weight, scale, post, ctx.post_norm, ctx.eps)
        gr, gs = (None, 0) if dy is None else _rows(dy, d)
        sr, ss = (None, 0) if ds is None else _rows(ds, d)
        L_ = _lib.lib()
        ws = None
        if dw is not None or dc is not None or dp is not None:
            ws = x.new_empty(L_.eacs_norm_bwd_workspace_size(p), dtype=torch.uint8)
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
    for t in (gate, residual):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise RuntimeError(f"{name}: {'gate' if t is gate else 'residual'} must have x's shape and dtype")
    w = None
    for t in (weight, scale, post):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != d or t.dtype not in _lib.DTYPE_CODES:
                raise RuntimeError(f"{name}: weight, scale and post_weight must be ({d},), float32, float16 or bfloat16")
            if w is not None and t.dtype != w:
                raise RuntimeError(f"{name}: weight, scale and post_weight must have one dtype")
            w = t.dtype
    weight, scale, post = dense(weight), dense(scale), dense(post)
    if wants_grad(x, gate, residual, weight, scale, post):
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
