"""LayerNorm with its backward pass (eacs_layer_norm_fwd / eacs_layer_norm_bwd).

`layer_norm(x, weight, bias, eps, residual=None)` is
torch.nn.functional.layer_norm over the last dimension of x (+ residual): the
norm in front of an EACS layer's projections (cst_ssm/modules/eacs.py:334)
and, with the blended branches as the residual, MultiScaleEACS's
out_norm(x + fused) (cst_ssm/modules/multiscale.py:176-179).  Statistics and
sums are float32 and each output is rounded once, so x + residual is never
rounded (or written) itself.  Differentiable in x, residual, weight and bias;
the gradients of weight and bias are the same bits on every run.  A backward
with create_graph runs in torch operations, so that it can be differentiated.

`LayerNorm` is the nn.LayerNorm module that runs it (same parameters and state
dict), `use_norms(model)` turns the nn.LayerNorm modules of a model into it, and
eacs_b200.install(..., norms=True) does so for every EACSLayer,
ContinuousSSMLayer and MultiScaleEACS built afterwards.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn

from .. import _lib
from ._check import is_plain, on, one_device, require_plain

MAX_D = 8192


def _rows(t: Tensor, d: int) -> tuple[Tensor, int]:
    """t as (rows, d) with a dense last dimension, and its row stride."""
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= d:
        return t, t.stride(0)
    if t.is_contiguous():
        return t, d
    t = t.reshape(-1, d)
    if t.shape[0] > 1 and (t.stride(1) != 1 or t.stride(0) < d):
        t = t.contiguous()
    elif t.stride(1) != 1 and d > 1:
        t = t.contiguous()
    return t, max(t.stride(0), d)


def _forward(x, weight, bias, eps, residual, dev):
    d = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if y.numel():
        xr, xs = _rows(x, d)
        rr, rs = (None, 0) if residual is None else _rows(residual, d)
        w = weight if weight is not None else bias
        with on(dev):
            _lib.check(_lib.lib().eacs_layer_norm_fwd(
                xr.data_ptr(), xs, _lib.ptr(rr), rs, _lib.DTYPE_CODES[x.dtype], _lib.ptr(weight), _lib.ptr(bias),
                0 if w is None else _lib.DTYPE_CODES[w.dtype], eps, y.data_ptr(), y.numel() // d, d,
                _lib.raw_stream(dev.index)), "eacs_layer_norm_fwd")
    return y


def _recorded_gradients(x, weight, residual, dy, eps):
    """The gradients (ds, dweight, dbias) in torch operations: for a backward that is itself to be differentiated."""
    s = x.float() if residual is None else x.float() + residual.float()
    c = s - s.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    h, dy = c * rstd, dy.float()
    p = dy if weight is None else dy * weight.float()
    ds = rstd * (p - p.mean(-1, keepdim=True) - h * (p * h).mean(-1, keepdim=True))
    d = x.shape[-1]
    return ds.to(x.dtype), (dy * h).reshape(-1, d).sum(0), dy.reshape(-1, d).sum(0)


class LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, dev):
        ctx.save_for_backward(x, weight, residual)
        ctx.eps, ctx.dev = eps, dev
        ctx.bias_dtype = None if bias is None else bias.dtype
        return _forward(x, weight, bias, eps, residual, dev)

    @staticmethod
    def backward(ctx, dy):
        x, weight, residual = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r, _ = ctx.needs_input_grad
        dev, d = ctx.dev, x.shape[-1]
        wd = weight.dtype if weight is not None else ctx.bias_dtype
        if torch.is_grad_enabled():  # create_graph
            ds, dw, db = _recorded_gradients(x, weight, residual, dy, ctx.eps)
            return (ds if need_x else None, dw.to(wd) if need_w else None, db.to(wd) if need_b else None, None,
                    ds if need_r else None, None)
        dw = torch.empty(d, dtype=wd, device=dev) if need_w else None
        db = torch.empty(d, dtype=wd, device=dev) if need_b else None
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        rows = dx.numel() // d
        L = _lib.lib()
        ws = None
        if (need_w or need_b) and rows:
            ws = torch.empty(int(L.eacs_layer_norm_bwd_workspace_size(rows, d)), dtype=torch.uint8, device=dev)
        xr, xs = _rows(x, d)
        gr, gs = _rows(dy, d)
        rr, rs = (None, 0) if residual is None else _rows(residual, d)
        with on(dev):
            _lib.check(L.eacs_layer_norm_bwd(
                xr.data_ptr(), xs, _lib.ptr(rr), rs, gr.data_ptr(), gs, _lib.DTYPE_CODES[x.dtype], _lib.ptr(weight),
                0 if wd is None else _lib.DTYPE_CODES[wd], ctx.eps, dx.data_ptr(), _lib.ptr(dw), _lib.ptr(db),
                _lib.ptr(ws), 0 if ws is None else ws.numel(), rows, d, _lib.raw_stream(dev.index)), "eacs_layer_norm_bwd")
        # one gradient for both, as a sum's backward gives it
        return dx if need_x else None, dw, db, None, dx if need_r else None, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
               residual: Tensor | None = None) -> Tensor:
    """LayerNorm of x (+ residual) over the last dimension, in x's dtype.

    x (..., d) float32 / float16 / bfloat16, d up to 8192; residual like x;
    weight and bias (d), both of one of those dtypes, or None.  Gradients are
    reverse mode only, and forward-mode or traced inputs are refused."""
    dev = one_device("layer_norm", x, residual, weight, bias)
    require_plain("layer_norm", x, residual, weight, bias)
    dt = x.dtype
    if x.dim() < 1 or dt not in _lib.DTYPE_CODES:
        raise RuntimeError(f"layer_norm: unsupported x, {dt} of {x.dim()} dimensions")
    d = x.shape[-1]
    if not 1 <= d <= MAX_D:
        raise RuntimeError(f"layer_norm: d={d} must be 1 to {MAX_D}")
    grad = x.requires_grad
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != dt:
            raise RuntimeError("layer_norm: residual must have x's shape and dtype")
        grad = grad or residual.requires_grad
    for t in (weight, bias):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != d or t.dtype not in _lib.DTYPE_CODES:
                raise RuntimeError(f"layer_norm: weight and bias must be ({d},), float32, float16 or bfloat16")
            grad = grad or t.requires_grad
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("layer_norm: weight and bias must have one dtype")
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if grad and torch.is_grad_enabled():
        return LayerNormFunction.apply(x, weight, bias, float(eps), residual, dev)
    return _forward(x, weight, bias, float(eps), residual, dev)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension through `layer_norm`.

    In a float16 / bfloat16 autocast region the input is taken to float32
    first, as autocast runs layer norms.  CPU tensors and what `layer_norm`
    does not take (float64, several normalised dimensions, more than 8192
    features, forward-mode derivatives, torch.func and tracing) keep torch's
    own."""

    def forward(self, x: Tensor) -> Tensor:
        if (not x.is_cuda or len(self.normalized_shape) != 1 or self.normalized_shape[0] > MAX_D
                or not is_plain(x, self.weight, self.bias) or x.dtype not in _lib.DTYPE_CODES or x.shape[-1:] != self.normalized_shape
                or any(p is not None and p.dtype not in _lib.DTYPE_CODES for p in (self.weight, self.bias))):
            return super().forward(x)
        if x.dtype != torch.float32 and torch.is_autocast_enabled("cuda"):
            x = x.float()
        return layer_norm(x, self.weight, self.bias, self.eps)


def use_norms(model: nn.Module) -> int:
    """Turn the plain nn.LayerNorm modules of `model` into LayerNorm, keeping
    their parameters; returns how many."""
    n = 0
    for m in model.modules():
        if type(m) is nn.LayerNorm:
            m.__class__ = LayerNorm
            n += 1
    return n


def make_init(original):
    """A constructor whose own nn.LayerNorm modules become LayerNorm."""
    def init(self, *args, **kwargs):
        original(self, *args, **kwargs)
        use_norms(self)
    init.__wrapped__ = original
    return init
