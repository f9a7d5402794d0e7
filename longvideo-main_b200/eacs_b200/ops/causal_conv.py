"""The short causal convolution of each channel (eacs_conv_*).

    p_t = bias + sum_w weight[:, w] x_{t-W+1+w},   y_t = silu(p_t)

with W = 2 to 4 taps, as it stands in front of a recurrence (selective_ssm's x,
or the queries, keys and values of gated_delta_rule): each token sees itself and
the W - 1 tokens before it.  `causal_conv` runs sequences, differentiable, from
and to a state; `causal_conv_step` takes one token per row and moves the state
on in place, for streaming.

Layouts: x and y (B, L, D) of one dtype, weight (D, W) and bias (D) of one
dtype (an nn.Conv1d's weight with its middle dimension squeezed), up to 65535
rows (B), states (B, W - 1, D) of x's dtype: the last inputs, oldest first.  x
may be a view with a dense last dimension (a slice of a fused projection needs
no copy); rows that start on 16 bytes are fastest, then rows of an even number of
channels.  Sums are float32, an output is rounded once.  The same inputs give the
same bits.

Gradients are reverse mode, once; forward-mode, torch.func or traced calls are
refused.  A backward captured into a CUDA graph must not share its leaves with
an eager graph that is still alive (autograd's own rule).
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _lib
from ._check import dense, dense_last, new_like, on, once, one_device, require_plain, wants_grad

MIN_WIDTH, MAX_WIDTH = 2, 4


def _check(name, x, weight, bias, activation, lengths, state, lead):
    """Device of the arguments; lead: the dimensions in front of the channels."""
    if weight is None or (lead == 1 and state is None):
        raise RuntimeError(f"{name}: expects tensors for x{' and the weight' if lead == 2 else ', the weight and the state'}")
    dev = one_device(name, x, weight, bias, lengths, state)
    require_plain(name, x, weight, bias, state)
    xs = x.shape
    if x.dtype not in _lib.DTYPE_CODES or len(xs) != lead + 1 or xs[-1] < 1:
        raise RuntimeError(f"{name}: x must be float32, float16 or bfloat16 of {lead + 1} dimensions")
    if weight.dim() != 2 or weight.shape[0] != xs[-1] or weight.dtype not in _lib.DTYPE_CODES:
        raise RuntimeError(f"{name}: weight must be ({xs[-1]}, W), float32, float16 or bfloat16")
    W = weight.shape[1]
    if not MIN_WIDTH <= W <= MAX_WIDTH:
        raise RuntimeError(f"{name}: W={W} taps, not {MIN_WIDTH} to {MAX_WIDTH}")
    if bias is not None and (bias.shape != xs[-1:] or bias.dtype != weight.dtype):
        raise RuntimeError(f"{name}: bias must be ({xs[-1]},) of the weight's dtype")
    if activation not in ("silu", None):
        raise RuntimeError(f"{name}: activation must be 'silu' or None")
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != xs[:1]):
        raise RuntimeError(f"{name}: lengths must be int32 ({xs[0]},)")
    if state is not None and (state.dtype != x.dtype or state.shape != (xs[0], W - 1, xs[-1])):
        raise RuntimeError(f"{name}: the state must be ({xs[0]}, {W - 1}, {xs[-1]}) of x's dtype")
    return dev


def _args(x, weight, bias, activation, lengths, state) -> bytes:
    """EacsConv of sequences (B, L, D), or of one token a row (B, D)."""
    L, token = (x.shape[1], x.stride(1)) if x.dim() == 3 else (1, 0)
    return _lib.CONV.pack(x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
                          0 if state is None else state.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
                          x.stride(0), token, x.shape[0], L, x.shape[-1], weight.shape[1], _lib.DTYPE_CODES[x.dtype],
                          _lib.DTYPE_CODES[weight.dtype], int(activation is not None))


def _forward(x, weight, bias, activation, lengths, state, out_state, dev):
    y = new_like(x)
    final = x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2])) if out_state else None
    with on(dev):
        _lib.check(_lib.lib().eacs_conv_fwd(_args(x, weight, bias, activation, lengths, state), y.data_ptr(),
                                            _lib.ptr(final), _lib.raw_stream(dev.index)), "eacs_conv_fwd")
    return y, final


class CausalConvFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, lengths, initial, out_state, dev):
        y, final = _forward(x, weight, bias, activation, lengths, initial, out_state, dev)
        ctx.save_for_backward(x, weight, bias, lengths, initial)
        ctx.activation, ctx.dev = activation, dev
        ctx.set_materialize_grads(False)
        return (y, final) if out_state else y

    @staticmethod
    @once
    def backward(ctx, dy, dfinal=None):
        x, weight, bias, lengths, initial = ctx.saved_tensors
        dev = ctx.dev
        if dy is None and dfinal is None:
            return (None,) * 8
        # hooks may give saved tensors back in another layout
        x, weight, bias, lengths, initial = dense_last(x), dense(weight), dense(bias), dense(lengths), dense(initial)
        dy = torch.zeros(x.shape, dtype=x.dtype, device=dev) if dy is None else dense_last(dy)
        dfinal = dense(dfinal)
        p = _args(x, weight, bias, ctx.activation, lengths, initial)
        _, need_w, need_b, _, _, need_i, _, _ = ctx.needs_input_grad
        dx = new_like(x)
        dw = new_like(weight) if need_w else None
        db = new_like(bias) if need_b else None
        di = new_like(initial) if need_i else None
        L_ = _lib.lib()
        ws = x.new_empty(L_.eacs_conv_bwd_workspace_size(p), dtype=torch.uint8) if need_w or need_b else None
        with on(dev):
            _lib.check(L_.eacs_conv_bwd(p, dy.data_ptr(), (ctypes.c_int64 * 2)(*dy.stride()[:2]), _lib.ptr(dfinal),
                                        dx.data_ptr(), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(di), _lib.ptr(ws),
                                        0 if ws is None else ws.numel(), _lib.raw_stream(dev.index)), "eacs_conv_bwd")
        return dx, dw, db, None, None, di, None, None


def causal_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = "silu",
                initial_state: Tensor | None = None, output_final_state: bool = False, lengths: Tensor | None = None):
    """y (B, L, D) in x's dtype; with output_final_state also the state
    (B, W - 1, D) behind the last token.

    lengths (B) int32 on the device: row b has lengths[b] tokens (clamped to
    0..L); what lies behind is not read, its outputs and gradients are 0.
    Differentiable in x, weight, bias and initial_state, through y and the
    final state."""
    dev = _check("causal_conv", x, weight, bias, activation, lengths, initial_state, 2)
    x, weight, bias, lengths, state = dense_last(x), dense(weight), dense(bias), dense(lengths), dense(initial_state)
    if wants_grad(x, weight, bias, state):
        return CausalConvFunction.apply(x, weight, bias, activation, lengths, state, output_final_state, dev)
    y, final = _forward(x, weight, bias, activation, lengths, state, output_final_state, dev)
    return (y, final) if output_final_state else y


def causal_conv_step(x: Tensor, weight: Tensor, bias: Tensor | None, state: Tensor, activation: str | None = "silu") -> Tensor:
    """One token per row: x (B, D); `state` (B, W - 1, D), contiguous, is moved
    on in place.  Returns y (B, D).  No gradient: inputs that want one are
    refused where gradients are enabled."""
    dev = _check("causal_conv_step", x, weight, bias, activation, None, state, 1)
    if wants_grad(x, weight, bias):
        raise RuntimeError("causal_conv_step: has no gradient; call it under torch.no_grad() or with detached tensors")
    if not state.is_contiguous() or state.requires_grad:
        raise RuntimeError("causal_conv_step: the state is updated in place: it must be contiguous and without a gradient")
    x, weight, bias = dense_last(x), dense(weight), dense(bias)
    y = new_like(x)
    with on(dev):
        _lib.check(_lib.lib().eacs_conv_step(_args(x, weight, bias, activation, None, None), y.data_ptr(), state.data_ptr(),
                                             _lib.raw_stream(dev.index)), "eacs_conv_step")
    torch.autograd.graph.increment_version(state)
    return y
