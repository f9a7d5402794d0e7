"""The selective state space scan: a diagonal recurrence with a step per token and channel (eacs_selective_*).

For each channel d with N states (float32), per token with a step
s = softplus(dt + dt_bias) and the token's vectors B and C:

    h[n] = exp(s A[n]) h[n] + s x B[n],   y = (sum_n C[n] h[n] + skip x) silu(z)

It stands beside the ungated scan (ssm_forward: one step per frame, complex
rates, B and C per frame) and the gated delta rule: the same role in a layer,
with steps that each channel takes from the token.  `selective_ssm` runs
sequences, differentiable, from and to a state; `selective_ssm_step` takes one
token per row and updates the state in place, for streaming.  Its input comes
through causal_conv, as a rule.

Layouts: x, dt, z and y (B, L, D), the vectors B and C (B, L, N), all of one
dtype; A (D, N), skip and dt_bias (D) float32; states (B, D, N) float32.  N is 1
to 64; rows (B) up to 65535.  Views are taken with their strides (a slice of a
fused projection needs no copy) as long as their last dimension is dense; they
are fastest when their rows start on 16 bytes, and so do B's and C's: N a
multiple of 8 (float32: 4) is copied ahead, other N are read element by element
(B=8 L=8192 D=768 bfloat16 forward: N=8 takes 418 us, N=4 559, N=12 651, N=16
494).  A finite and <= 0 is meant, and steps >= 0.  Sums and states are float32,
an output is rounded once.  The same inputs give the same bits.

With gradients the forward keeps one state in 8 tokens (4 N bytes a channel,
N rounded up to 8, 16, 32 or 64) until the backward, and the backward takes
8 N P bytes a token of partial sums while it runs (N rounded up too): P, the
CTAs of a row, is N D / (128 G) rounded up, for the 1 to 8 groups of channels G
that leave the fewest rounds of CTAs.  One row of D=256, N=64 takes 64 KB a
token, eight of D=768, N=16 2 KB.  A NaN or an infinity of a token reaches what
follows it, never what lies before.

Gradients are reverse mode, once; forward-mode, torch.func or traced calls are
refused.  A backward captured into a CUDA graph must not share its leaves with
an eager graph that is still alive (autograd's own rule).
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _lib
from ._check import dense, dense_last, new_like, on, once, one_device, packed, require_plain, wants_grad

MAX_N = 64


def _check(name, x, dt, A, B, C, skip, z, dt_bias, lengths, state):
    lead = 1 if name.endswith("step") else 2
    if dt is None or A is None or B is None or C is None or (lead == 1 and state is None):
        raise RuntimeError(f"{name}: expects tensors for x, dt, A, B{' and C' if lead == 2 else ', C and the state'}")
    dev = one_device(name, x, dt, A, B, C, skip, z, dt_bias, lengths, state)
    require_plain(name, x, dt, A, B, C, skip, z, dt_bias, state)
    xs, ty = x.shape, x.dtype
    if ty not in _lib.DTYPE_CODES or dt.dtype != ty or B.dtype != ty or C.dtype != ty or (z is not None and z.dtype != ty):
        raise RuntimeError(f"{name}: x, dt, B, C and z must have one dtype, float32, float16 or bfloat16")
    if len(xs) != lead + 1 or dt.shape != xs or (z is not None and z.shape != xs):
        raise RuntimeError(f"{name}: x, dt and z must have one shape of {lead + 1} dimensions")
    if A.dim() != 2 or A.shape[0] != xs[-1] or A.dtype != torch.float32:
        raise RuntimeError(f"{name}: A must be float32 ({xs[-1]}, N)")
    N = A.shape[1]
    if not 1 <= N <= MAX_N or xs[-1] < 1:
        raise RuntimeError(f"{name}: N={N} must be 1 to {MAX_N}, and D at least 1")
    if B.shape != (*xs[:-1], N) or C.shape != B.shape:
        raise RuntimeError(f"{name}: B and C must be {(*xs[:-1], N)}")
    for t in (skip, dt_bias):
        if t is not None and (t.shape != xs[-1:] or t.dtype != torch.float32):
            raise RuntimeError(f"{name}: skip and dt_bias must be float32 ({xs[-1]},)")
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != xs[:1]):
        raise RuntimeError(f"{name}: lengths must be int32 ({xs[0]},)")
    if state is not None and (state.dtype != torch.float32 or state.shape != (xs[0], xs[-1], N)):
        raise RuntimeError(f"{name}: the state must be float32 ({xs[0]}, {xs[-1]}, {N})")
    return dev


def _args(x, dt, A, B, C, skip, z, dt_bias, softplus, lengths, state) -> bytes:
    """EacsSelective of sequences (B, L, D), or of one token a row (B, D)."""
    if x.dim() == 3:
        st = (*x.stride()[:2], *dt.stride()[:2], *((0, 0) if z is None else z.stride()[:2]), *B.stride()[:2], *C.stride()[:2])
        L = x.shape[1]
    else:
        st = (x.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0), 0, B.stride(0), 0, C.stride(0), 0)
        L = 1
    p = lambda t: 0 if t is None else t.data_ptr()
    return _lib.SELECTIVE.pack(x.data_ptr(), dt.data_ptr(), p(z), B.data_ptr(), C.data_ptr(), *st, A.data_ptr(), p(skip),
                               p(dt_bias), p(lengths), p(state), x.shape[0], L, x.shape[-1], A.shape[1],
                               _lib.DTYPE_CODES[x.dtype], int(softplus))


def _forward(args, out_state, training, dev):
    """(y, final state or None, checkpoints or None) of (x, dt, A, B, C, skip, z, dt_bias, softplus, lengths, initial)."""
    x, A = args[0], args[2]
    p = _args(*args)
    L_ = _lib.lib()
    y = new_like(x)
    final = A.new_empty((x.shape[0], *A.shape)) if out_state else None
    ck = x.new_empty(L_.eacs_selective_ckpt_size(p), dtype=torch.uint8) if training else None
    with on(dev):
        _lib.check(L_.eacs_selective_fwd(p, y.data_ptr(), _lib.ptr(final), _lib.ptr(ck), 0 if ck is None else ck.numel(),
                                         _lib.raw_stream(dev.index)), "eacs_selective_fwd")
    return y, final, ck


class SelectiveSSMFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, skip, z, dt_bias, softplus, lengths, initial, out_state, dev):
        y, final, ck = _forward((x, dt, A, B, C, skip, z, dt_bias, softplus, lengths, initial), out_state, True, dev)
        ctx.save_for_backward(x, dt, A, B, C, skip, z, dt_bias, lengths, initial, ck)
        ctx.softplus, ctx.dev = softplus, dev
        ctx.set_materialize_grads(False)
        return (y, final) if out_state else y

    @staticmethod
    @once
    def backward(ctx, dy, dfinal=None):
        x, dt, A, B, C, skip, z, dt_bias, lengths, initial, ck = ctx.saved_tensors
        dev = ctx.dev
        if dy is None and dfinal is None:
            return (None,) * 13
        # hooks may give saved tensors back in another layout
        x, dt, B, C, z = dense_last(x), dense_last(dt), dense_last(B), dense_last(C), dense_last(z)
        A, skip, dt_bias, lengths, initial = dense(A), dense(skip), dense(dt_bias), dense(lengths), dense(initial)
        ck = packed(ck)
        dy = torch.zeros(x.shape, dtype=x.dtype, device=dev) if dy is None else dense_last(dy)
        dfinal = dense(dfinal)
        p = _args(x, dt, A, B, C, skip, z, dt_bias, ctx.softplus, lengths, initial)
        dx, ddt, dA, dB, dC = new_like(x), new_like(dt), new_like(A), new_like(B), new_like(C)
        dskip, dz, dbias = new_like(skip), new_like(z), new_like(dt_bias)
        di = new_like(initial) if ctx.needs_input_grad[10] else None
        L_ = _lib.lib()
        ws = x.new_empty(L_.eacs_selective_bwd_workspace_size(p), dtype=torch.uint8)
        with on(dev):
            _lib.check(L_.eacs_selective_bwd(
                p, dy.data_ptr(), (ctypes.c_int64 * 2)(*dy.stride()[:2]), _lib.ptr(dfinal), dx.data_ptr(), ddt.data_ptr(),
                _lib.ptr(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _lib.ptr(dskip), _lib.ptr(dbias), _lib.ptr(di),
                ck.data_ptr(), ck.numel(), ws.data_ptr(), ws.numel(), _lib.raw_stream(dev.index)), "eacs_selective_bwd")
        return dx, ddt, dA, dB, dC, dskip, dz, dbias, None, None, di, None, None


def selective_ssm(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, skip: Tensor | None = None,
                  z: Tensor | None = None, dt_bias: Tensor | None = None, softplus: bool = True,
                  initial_state: Tensor | None = None, output_final_state: bool = False,
                  lengths: Tensor | None = None):
    """y (B, L, D) in x's dtype; with output_final_state also the state
    (B, D, N) float32 behind the last token.

    softplus=False takes dt (+ dt_bias) itself as the step; a softplus below
    e^-87.3 is 0, so that -inf or the dtype's lowest value in dt masks a token
    (its channel keeps its state).  lengths (B) int32
    on the device: row b has lengths[b] tokens (clamped to 0..L); what lies
    behind is not read, its outputs and gradients are 0.  Differentiable in
    every floating point input, through y and the final state."""
    dev = _check("selective_ssm", x, dt, A, B, C, skip, z, dt_bias, lengths, initial_state)
    x, dt, B, C, z = dense_last(x), dense_last(dt), dense_last(B), dense_last(C), dense_last(z)
    A, skip, dt_bias, lengths, state = dense(A), dense(skip), dense(dt_bias), dense(lengths), dense(initial_state)
    if wants_grad(x, dt, A, B, C, skip, z, dt_bias, state):
        return SelectiveSSMFunction.apply(x, dt, A, B, C, skip, z, dt_bias, bool(softplus), lengths, state,
                                          output_final_state, dev)
    y, final, _ = _forward((x, dt, A, B, C, skip, z, dt_bias, softplus, lengths, state), output_final_state, False, dev)
    return (y, final) if output_final_state else y


def selective_ssm_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, skip: Tensor | None = None,
                       z: Tensor | None = None, dt_bias: Tensor | None = None, softplus: bool = True) -> Tensor:
    """One token per row: x, dt, z (B, D), B and C (B, N); `state` (B, D, N)
    float32, contiguous, is updated in place.  Returns y (B, D) in x's dtype.
    No gradient: inputs that want one are refused where gradients are enabled."""
    dev = _check("selective_ssm_step", x, dt, A, B, C, skip, z, dt_bias, None, state)
    if wants_grad(x, dt, A, B, C, skip, z, dt_bias):
        raise RuntimeError("selective_ssm_step: has no gradient; call it under torch.no_grad() or with detached tensors")
    if not state.is_contiguous() or state.requires_grad:
        raise RuntimeError("selective_ssm_step: the state is updated in place: it must be contiguous and without a gradient")
    x, dt, B, C, z = dense_last(x), dense_last(dt), dense_last(B), dense_last(C), dense_last(z)
    A, skip, dt_bias = dense(A), dense(skip), dense(dt_bias)
    y = new_like(x)
    p = _args(x, dt, A, B, C, skip, z, dt_bias, softplus, None, None)
    with on(dev):
        _lib.check(_lib.lib().eacs_selective_step(p, y.data_ptr(), state.data_ptr(), _lib.raw_stream(dev.index)),
                   "eacs_selective_step")
    torch.autograd.graph.increment_version(state)
    return y
