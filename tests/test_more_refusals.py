"""The selective scan, the causal convolution and the block norms on a machine without a GPU: refused arguments (before
anything touches the device), workspace sizes and empty calls."""
import ctypes

import pytest
import torch

from eacs_b200 import _lib

P = 256  # a pointer value that is never read
STRIDES = (ctypes.c_int64 * 2)(1, 1)
BIG = 1 << 40


def selective(rows=2, L=10, D=8, N=16, dtype=2, softplus=1, **ptr):
    p = [ptr.get(n, P) or 0 for n in ("x", "dt", "z", "B", "C")]
    q = [ptr.get(n, P) or 0 for n in ("A", "skip", "dt_bias")]
    return _lib.SELECTIVE.pack(*p, *[8] * 10, *q, 0, 0, rows, L, D, N, dtype, softplus)


def conv(rows=2, L=10, D=8, width=4, dtype=2, w_dtype=0, silu=1, **ptr):
    p = [ptr.get(n, P) or 0 for n in ("x", "weight", "bias")]
    return _lib.CONV.pack(*p, 0, 0, 80, 8, rows, L, D, width, dtype, w_dtype, silu)


def norm(rows=4, d=16, dtype=2, w_dtype=0, post=0, stride=16, **ptr):
    p = [ptr.get(n, P) or 0 for n in ("x", "gate", "residual", "weight", "scale", "post_weight")]
    return _lib.NORM.pack(*p, stride, stride, stride, rows, d, 1e-5, dtype, w_dtype, post)


def selective_bwd(p, dy=P, ck=BIG, ws=BIG, **kw):
    return _lib.lib().eacs_selective_bwd(p, dy, STRIDES, None, P, P, kw.get("dz", P), P, P, P, None, None, None, kw.get("ckp", P), ck,
                                         kw.get("wsp", P), ws, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(rows=-1), 1, "sizes"), (dict(L=-1), 1, "sizes"), (dict(D=0), 1, "sizes"), (dict(N=0), 1, "sizes"), (dict(dtype=3), 1, "dtype"),
    (dict(N=65), 5, "N=65"), (dict(rows=65536), 5, "65535"), (dict(D=(1 << 24) + 1), 5, "2^24"), (dict(L=(1 << 30) + 1), 5, "2^30"),
    (dict(x=None), 1, "null"), (dict(A=None), 1, "null"), (dict(C=None), 1, "null")])
def test_selective_rejects_bad_arguments_without_device(kw, code, word):
    L = _lib.lib()
    assert L.eacs_selective_fwd(selective(**kw), P, None, None, 0, None) == code and word in _lib.last_error()
    assert L.eacs_selective_step(selective(**kw), P, P, None) == code
    assert selective_bwd(selective(**kw)) == code
    assert L.eacs_selective_ckpt_size(selective(**kw)) == 0 and L.eacs_selective_bwd_workspace_size(selective(**kw)) == 0


def test_selective_workspaces_and_empty_calls_without_device():
    L = _lib.lib()
    ck, ws = L.eacs_selective_ckpt_size(selective()), L.eacs_selective_bwd_workspace_size(selective())
    assert ck == 2 * 2 * 8 * 16 * 4 and ws > 0  # a state in 8 tokens
    assert L.eacs_selective_ckpt_size(selective(N=17)) == 2 * ck  # N rounded up to 32
    assert L.eacs_selective_fwd(selective(), P, None, P, ck - 1, None) == _lib.EACS_ERR_WORKSPACE
    assert L.eacs_selective_fwd(selective(), P, None, P + 8, ck, None) == _lib.EACS_ERR_INVALID
    assert L.eacs_selective_fwd(selective(), None, None, None, 0, None) == _lib.EACS_ERR_INVALID
    assert selective_bwd(selective(), ck=ck - 1, ws=ws) == _lib.EACS_ERR_WORKSPACE
    assert selective_bwd(selective(), ck=ck, ws=ws - 1) == _lib.EACS_ERR_WORKSPACE
    assert selective_bwd(selective(), ck=ck, ws=ws, wsp=P + 4) == _lib.EACS_ERR_INVALID
    assert selective_bwd(selective(), dy=None) == _lib.EACS_ERR_INVALID
    assert selective_bwd(selective(), dz=None) == _lib.EACS_ERR_INVALID  # a gate without a place for its gradient
    assert L.eacs_selective_step(selective(), P, None, None) == _lib.EACS_ERR_INVALID
    assert L.eacs_selective_step(selective(rows=0), None, None, None) == _lib.EACS_OK
    for kw in (dict(rows=0), dict(L=0)):
        assert L.eacs_selective_fwd(selective(**kw), None, None, None, 0, None) == _lib.EACS_OK
    for f in (L.eacs_selective_ckpt_size, L.eacs_selective_bwd_workspace_size):
        assert f(None) == 0
    assert L.eacs_selective_fwd(None, P, None, None, 0, None) == _lib.EACS_ERR_INVALID
    assert L.eacs_selective_step(None, P, P, None) == _lib.EACS_ERR_INVALID


@pytest.mark.parametrize("kw,code,word", [
    (dict(rows=-1), 1, "sizes"), (dict(L=-1), 1, "sizes"), (dict(D=0), 1, "sizes"), (dict(dtype=3), 1, "dtype"), (dict(w_dtype=-1), 1, "dtype"),
    (dict(width=1), 5, "1 taps"), (dict(width=5), 5, "5 taps"), (dict(rows=65536), 5, "65535"), (dict(L=(1 << 30) + 1), 5, "2^30"),
    (dict(x=None), 1, "null"), (dict(weight=None), 1, "null")])
def test_conv_rejects_bad_arguments_without_device(kw, code, word):
    L = _lib.lib()
    assert L.eacs_conv_fwd(conv(**kw), P, None, None) == code and word in _lib.last_error()
    assert L.eacs_conv_step(conv(**kw), P, P, None) == code
    assert L.eacs_conv_bwd(conv(**kw), P, STRIDES, None, P, P, P, None, P, BIG, None) == code
    assert L.eacs_conv_bwd_workspace_size(conv(**kw)) == 0


@pytest.mark.parametrize("D", [1, 3, 33, 64, 1000, 4096])
def test_conv_workspaces_and_empty_calls_without_device(D):
    L = _lib.lib()
    for rows, length in ((1, 0), (1, 1), (2, 10), (65535, 1), (1, 1 << 20)):  # every grid has a size
        need = L.eacs_conv_bwd_workspace_size(conv(rows=rows, L=length, D=D))
        assert need > 0 and need % (D * 5 * 4) == 0
    need = L.eacs_conv_bwd_workspace_size(conv(D=D))
    bwd = lambda ws, p=P, dy=P: L.eacs_conv_bwd(conv(D=D), dy, STRIDES, None, P, P, P, None, p, ws, None)
    assert bwd(need - 1) == _lib.EACS_ERR_WORKSPACE and bwd(need, None) == _lib.EACS_ERR_WORKSPACE
    assert bwd(need, P + 4) == _lib.EACS_ERR_INVALID and bwd(need, P, None) == _lib.EACS_ERR_INVALID
    assert L.eacs_conv_fwd(conv(rows=0, D=D), None, None, None) == _lib.EACS_OK
    assert L.eacs_conv_fwd(conv(L=0, D=D), None, None, None) == _lib.EACS_OK
    assert L.eacs_conv_fwd(conv(D=D), None, None, None) == _lib.EACS_ERR_INVALID
    assert L.eacs_conv_step(conv(rows=0, D=D), None, None, None) == _lib.EACS_OK
    assert L.eacs_conv_step(conv(D=D), P, None, None) == _lib.EACS_ERR_INVALID
    assert L.eacs_conv_fwd(None, P, None, None) == _lib.EACS_ERR_INVALID and L.eacs_conv_bwd_workspace_size(None) == 0


@pytest.mark.parametrize("kw,code,word", [
    (dict(rows=-1), 1, "sizes"), (dict(d=0), 1, "sizes"), (dict(d=8193), 5, "8193"), (dict(dtype=3), 1, "dtype"), (dict(w_dtype=7), 1, "dtype"),
    (dict(x=None), 1, "null"), (dict(residual=None), 1, "scale without a residual"), (dict(stride=-1), 1, "stride")])
def test_norm_rejects_bad_arguments_without_device(kw, code, word):
    L = _lib.lib()
    assert L.eacs_norm_fwd(norm(**kw), P, P, None) == code and word in _lib.last_error()
    assert L.eacs_norm_bwd(norm(**kw), P, 16, P, 16, *[P] * 6, P, BIG, None) == code
    assert L.eacs_norm_bwd_workspace_size(norm(**kw)) == 0


def test_norm_workspaces_and_empty_calls_without_device():
    L = _lib.lib()
    need = L.eacs_norm_bwd_workspace_size(norm())
    assert need == 4 * 3 * 16 * 4 and L.eacs_norm_bwd_workspace_size(norm(rows=0)) == 0
    bwd = lambda ws, dx=P, dg=P, dr=P, dw=P: L.eacs_norm_bwd(norm(), P, 16, P, 16, dx, dg, dr, dw, P, None, P, ws, None)
    assert bwd(need - 1) == _lib.EACS_ERR_WORKSPACE
    assert bwd(need, dx=None) == _lib.EACS_ERR_INVALID and bwd(need, dg=None) == _lib.EACS_ERR_INVALID
    assert bwd(need, dr=None) == _lib.EACS_ERR_INVALID  # with a gate it is not dx
    assert L.eacs_norm_fwd(norm(), P, None, None) == _lib.EACS_ERR_INVALID  # a residual without a place for the sum
    assert L.eacs_norm_fwd(norm(rows=0), None, None, None) == _lib.EACS_OK
    assert L.eacs_norm_fwd(None, P, P, None) == _lib.EACS_ERR_INVALID and L.eacs_norm_bwd_workspace_size(None) == 0


def test_python_refusals_on_cpu_tensors():
    from eacs_b200.ops.block_norm import gated_norm, residual_norm
    from eacs_b200.ops.causal_conv import causal_conv, causal_conv_step
    from eacs_b200.ops.selective_ssm import selective_ssm, selective_ssm_step
    x, w, A, B = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(8, 16), torch.zeros(2, 5, 16)
    for f in (lambda: causal_conv(x, w), lambda: causal_conv_step(x[:, 0], w, None, torch.zeros(2, 3, 8)),
              lambda: selective_ssm(x, x, A, B, B), lambda: selective_ssm_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(2, 8, 16)),
              lambda: gated_norm(x, x), lambda: residual_norm(x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    for f in (lambda: causal_conv([1.0], w), lambda: selective_ssm(None, x, A, B, B), lambda: gated_norm(3.0)):
        with pytest.raises(RuntimeError, match="tensors"):
            f()
