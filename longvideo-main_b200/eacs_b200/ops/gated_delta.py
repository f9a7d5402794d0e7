"""The gated delta rule: a recurrence over a matrix state (eacs_delta_*).

For each head a state S (K x V, float32) and per token, with a decay's
logarithm g, a rate beta, a key k, a value v and a query q:

    S' = exp(g) S,  u = beta (v - S'^T k),  S = S' + k u^T,  o = scale S^T q

It stands beside the diagonal scans (selective_scan, ssm_forward): the same
role in a layer, with a state that is corrected towards v at key k instead of
summed.  `gated_delta_rule` runs sequences 64 tokens at a time on the tensor
cores, differentiable, from and to a state; `gated_delta_step` takes one token
per row and updates the state in place, for streaming.

Layouts: q, k (B, L, Hk, K), v (B, L, Hv, V), g and beta (B, L, Hv), states
(B, Hv, K, V) float32.  Hv is a multiple of Hk; value head h reads key head
h // (Hv // Hk).  Views are taken with their strides (a slice of a fused
projection needs no copy) as long as their last dimension is dense; 16-bit
ones are fastest when their rows start on 16 bytes (K, V and all strides
multiples of 8).  Sums and states are float32.  Operands of the products keep
22 significant bits, 16 for bfloat16 inputs; float16's states, values corrected
by them and gradients of them may be of any size that float32 holds.  The same
inputs give the same bits.  Where gradients are wanted beta is held 2^-64 away
from 0.

A NaN or an infinity of a token reaches what follows it, and up to 15 tokens
before it (the rest of its block of 16; in the backward pass, up to 15 behind an
upstream gradient's).  A forward at K = V = 128 takes 38 KB of workspace for each
chunk of 64 tokens of a head in the 16-bit kernels and 116 KB in the others;
with gradients 145 KB (float16 155, others 133) are kept until the backward,
which takes 106 KB (98) more.  A device wait that runs out leaves outputs unwritten and is reported by
eacs_device_status.

Gradients are reverse mode, once; forward-mode, torch.func or traced calls are
refused.  A backward that is captured into a graph must not share
leaves with an eager graph that is still alive (autograd's own rule).
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _lib
from ._check import dense_last, on, once, one_device, packed, require_plain

MAX_K = 128
MAX_V = 1024


def _check(name, q, k, v, g, beta, lengths, state, lead):
    """Device of the arguments; lead: the dimensions in front of the head's."""
    if k is None or v is None or g is None or beta is None or (lead == 1 and state is None):
        raise RuntimeError(f"{name}: expects tensors for q, k, v, g{' and beta' if lead == 2 else ', beta and the state'}")
    dev = one_device(name, q, k, v, g, beta, lengths, state)
    require_plain(name, q, k, v, g, beta, state)
    qs, vs, dt = q.shape, v.shape, q.dtype
    if len(qs) != lead + 2 or k.shape != qs:
        raise RuntimeError(f"{name}: q and k must have one shape of {lead + 2} dimensions")
    if len(vs) != lead + 2 or vs[:lead] != qs[:lead]:
        raise RuntimeError(f"{name}: v must have q's leading dimensions")
    Hk, K = qs[lead:]
    Hv, V = vs[lead:]
    if Hk < 1 or Hv < 1 or Hv % Hk:
        raise RuntimeError(f"{name}: {Hv} value heads are not a multiple of {Hk} key heads")
    if not (1 <= K <= MAX_K and 1 <= V <= MAX_V):
        raise RuntimeError(f"{name}: K={K}, V={V} must be 1 to {MAX_K}, 1 to {MAX_V}")
    if g.shape != vs[:-1] or beta.shape != g.shape:
        raise RuntimeError(f"{name}: g and beta must be {tuple(vs[:-1])}")
    if dt not in _lib.DTYPE_CODES or k.dtype != dt or v.dtype != dt:
        raise RuntimeError(f"{name}: q, k and v must have one dtype, float32, float16 or bfloat16")
    if g.dtype != beta.dtype or (g.dtype != dt and g.dtype != torch.float32):
        raise RuntimeError(f"{name}: g and beta must both be float32 or of q's dtype")
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != qs[:1]):
        raise RuntimeError(f"{name}: lengths must be int32 ({qs[0]},)")
    if state is not None and (state.dtype != torch.float32 or state.shape != (qs[0], Hv, K, V)):
        raise RuntimeError(f"{name}: the state must be float32 ({qs[0]}, {Hv}, {K}, {V})")
    return dev


def _args(q, k, v, g, beta, scale, lengths, state, path=0) -> bytes:
    """EacsDelta of a sequence (B, L, H, D), or of one token a row (B, H, D)."""
    qs, vs = q.shape, v.shape
    if len(qs) == 4:
        L = qs[1]
        st = (*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride(), *beta.stride())
    else:
        L = 1
        st = []
        for t in (q, k, v, g, beta):
            s = t.stride()
            st += (s[0], 0, s[1])
    return _lib.DELTA_PATH.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), *st,
                                0 if lengths is None else lengths.data_ptr(), 0 if state is None else state.data_ptr(),
                                qs[0], L, qs[-2], vs[-2], qs[-1], vs[-1], scale, _lib.DTYPE_CODES[q.dtype],
                                _lib.DTYPE_CODES[g.dtype], path)


def _forward(args, out_state, training, dev):
    """(o, final state or None, workspace, its path) of (q, k, v, g, beta, scale, lengths, initial)."""
    q, k, v = args[:3]
    p = _args(*args)
    L_ = _lib.lib()
    o = torch.empty(v.shape, dtype=q.dtype, device=dev)
    final = torch.empty(v.shape[0], v.shape[2], q.shape[3], v.shape[3], dtype=torch.float32, device=dev) if out_state else None
    ws = torch.empty(int(L_.eacs_delta_workspace_size(p, int(training))), dtype=torch.uint8, device=dev)
    with on(dev):
        _lib.check(L_.eacs_delta_fwd(p, o.data_ptr(), _lib.ptr(final), ws.data_ptr(), ws.numel(),
                                     int(training), _lib.raw_stream(dev.index)), "eacs_delta_fwd")
    return o, final, ws, L_.eacs_delta_path(p) if training else 0


class GatedDeltaFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, lengths, initial, out_state, dev):
        # what ws holds goes by where the inputs lie; hooks may give them back elsewhere
        o, final, ws, ctx.path = _forward((q, k, v, g, beta, scale, lengths, initial), out_state, True, dev)
        ctx.save_for_backward(q, k, v, g, beta, lengths, initial, ws)
        ctx.scale, ctx.dev = scale, dev
        ctx.set_materialize_grads(False)
        return (o, final) if out_state else o

    @staticmethod
    @once
    def backward(ctx, do, dfinal=None):
        q, k, v, g, beta, lengths, initial, ws = ctx.saved_tensors
        dev = ctx.dev
        if do is None and dfinal is None:
            return (None,) * 10
        do = torch.zeros(v.shape, dtype=q.dtype, device=dev) if do is None else do.contiguous()
        if do.data_ptr() % 16:  # a view that starts inside an allocation
            do = do.clone()
        dfinal = None if dfinal is None else dfinal.contiguous()
        q, k, v = dense_last(q), dense_last(k), dense_last(v)
        lengths, initial, ws = packed(lengths), packed(initial), packed(ws)
        L_ = _lib.lib()
        p = _args(q, k, v, g, beta, ctx.scale, lengths, initial, ctx.path)
        need = int(L_.eacs_delta_bwd_workspace_size(p))
        if need == 0 and do.numel():  # not as the path wants them
            q, k, v = (t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
            p = _args(q, k, v, g, beta, ctx.scale, lengths, initial, ctx.path)
            need = int(L_.eacs_delta_bwd_workspace_size(p))
        dq, dk, dv, dg, db = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v, g, beta))
        di = torch.empty(initial.shape, dtype=torch.float32, device=dev) if ctx.needs_input_grad[7] else None
        w2 = torch.empty(need, dtype=torch.uint8, device=dev)
        with on(dev):
            _lib.check(L_.eacs_delta_bwd(
                p, do.data_ptr(), (ctypes.c_int64 * 3)(*do.stride()[:3]), _lib.ptr(dfinal), dq.data_ptr(),
                dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), db.data_ptr(), _lib.ptr(di), ws.data_ptr(), ws.numel(),
                w2.data_ptr(), w2.numel(), _lib.raw_stream(dev.index)), "eacs_delta_bwd")
        return dq, dk, dv, dg, db, None, None, di, None, None


def gated_delta_rule(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: float | None = None,
                     initial_state: Tensor | None = None, output_final_state: bool = False,
                     lengths: Tensor | None = None):
    """o (B, L, Hv, V) in q's dtype; with output_final_state also the state
    (B, Hv, K, V) float32 behind the last token.

    scale defaults to K ** -0.5.  lengths (B) int32 on the device: row b has
    lengths[b] tokens (clamped to 0..L); what lies behind is not read, its
    outputs and gradients are 0.  Differentiable in q, k, v, g, beta and
    initial_state, through o and the final state."""
    dev = _check("gated_delta_rule", q, k, v, g, beta, lengths, initial_state, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v = dense_last(q), dense_last(k), dense_last(v)
    lengths = None if lengths is None else lengths.contiguous()
    state = None if initial_state is None else initial_state.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, state)):
        return GatedDeltaFunction.apply(q, k, v, g, beta, scale, lengths, state, output_final_state, dev)
    o, final, _, _ = _forward((q, k, v, g, beta, scale, lengths, state), output_final_state, False, dev)
    return (o, final) if output_final_state else o


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor,
                     scale: float | None = None) -> Tensor:
    """One token per row: q, k (B, Hk, K), v (B, Hv, V), g and beta (B, Hv);
    `state` (B, Hv, K, V) float32, contiguous, is updated in place.  Returns
    o (B, Hv, V) in q's dtype.  No gradient: inputs that want one are refused
    where gradients are enabled."""
    dev = _check("gated_delta_step", q, k, v, g, beta, None, state, 1)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta)):
        raise RuntimeError("gated_delta_step: has no gradient; call it under torch.no_grad() or with detached tensors")
    if not state.is_contiguous() or state.requires_grad:
        raise RuntimeError("gated_delta_step: the state is updated in place: it must be contiguous and without a gradient")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v = dense_last(q), dense_last(k), dense_last(v)
    o = torch.empty(v.shape, dtype=q.dtype, device=dev)
    p = _args(q, k, v, g, beta, scale, None, state)
    with on(dev):
        _lib.check(_lib.lib().eacs_delta_step(p, o.data_ptr(), state.data_ptr(), _lib.raw_stream(dev.index)),
                   "eacs_delta_step")
    torch.autograd.graph.increment_version(state)
    return o
