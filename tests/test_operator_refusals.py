"""Layer norm and the gated delta rule on a machine without a GPU: refused
arguments (before anything touches the device), empty calls, and the modules
that fall back to torch on CPU tensors."""
import ctypes
import sys
import types

import pytest
import torch
from torch import nn

from eacs_b200 import _lib

P = 256  # a pointer value that is never read


def delta(B=2, L=10, Hk=2, Hv=4, K=16, V=8, dtype=2, gate=2, **pointers):
    p = [pointers.get(n, P) or 0 for n in ("q", "k", "v", "g", "beta")]
    return _lib.DELTA.pack(*p, *[0] * 15, 0, 0, B, L, Hk, Hv, K, V, 1.0, dtype, gate)


def test_layer_norm_rejects_bad_arguments_without_device():
    L = _lib.lib()

    def fwd(x=P, xs=16, r=None, rs=0, dt=2, wd=0, y=P, rows=4, d=16):
        return L.eacs_layer_norm_fwd(x, xs, r, rs, dt, P, P, wd, 1e-5, y, rows, d, None)
    assert fwd(rows=0) == _lib.EACS_OK
    assert fwd(d=0) == _lib.EACS_ERR_INVALID and fwd(rows=-1) == _lib.EACS_ERR_INVALID
    assert fwd(d=8193, xs=8193) == _lib.EACS_ERR_UNSUPPORTED and "8193" in _lib.last_error()
    assert fwd(dt=3) == _lib.EACS_ERR_INVALID and fwd(wd=-1) == _lib.EACS_ERR_INVALID
    assert fwd(x=None) == _lib.EACS_ERR_INVALID and fwd(y=None) == _lib.EACS_ERR_INVALID
    assert fwd(xs=15) == _lib.EACS_ERR_INVALID and "stride" in _lib.last_error()
    assert fwd(r=P, rs=3) == _lib.EACS_ERR_INVALID

    def bwd(dy=P, dw=P, db=P, ws=P, n=None, rows=4, d=16):
        need = L.eacs_layer_norm_bwd_workspace_size(rows, d)
        return L.eacs_layer_norm_bwd(P, d, None, 0, dy, d, 2, P, 0, 1e-5, P, dw, db, ws, need if n is None else n,
                                     rows, d, None)
    assert bwd(dy=None) == _lib.EACS_ERR_INVALID
    assert bwd(ws=None) == _lib.EACS_ERR_WORKSPACE
    assert bwd(n=L.eacs_layer_norm_bwd_workspace_size(4, 16) - 1) == _lib.EACS_ERR_WORKSPACE
    assert L.eacs_layer_norm_bwd_workspace_size(4, 8193) == 0


@pytest.mark.parametrize("kw,code,word", [
    (dict(B=-1), 1, "sizes"), (dict(K=0), 1, "sizes"), (dict(Hk=3), 1, "multiple"), (dict(dtype=3), 1, "dtype"),
    (dict(gate=9), 1, "dtype"), (dict(K=129), 5, "K=129"), (dict(V=1025), 5, "V=1025"), (dict(B=65536), 5, "65535"),
    (dict(q=None), 1, "null"), (dict(beta=None), 1, "null")])
def test_delta_rejects_bad_arguments_without_device(kw, code, word):
    L = _lib.lib()
    strides = (ctypes.c_int64 * 3)(1, 1, 1)
    big = 1 << 40
    assert L.eacs_delta_fwd(delta(**kw), P, None, P, big, 0, None) == code and word in _lib.last_error()
    assert L.eacs_delta_step(delta(**kw), P, P, None) == code
    assert L.eacs_delta_bwd(delta(**kw), P, strides, None, P, P, P, P, P, None, P, big, P, big, None) == code
    if code == 5 or "null" not in word:
        assert L.eacs_delta_workspace_size(delta(**kw), 1) == 0


def test_delta_workspaces_and_empty_calls_without_device():
    L = _lib.lib()
    strides = (ctypes.c_int64 * 3)(1, 1, 1)
    need, keep = L.eacs_delta_workspace_size(delta(), 0), L.eacs_delta_workspace_size(delta(), 1)
    back = L.eacs_delta_bwd_workspace_size(delta())
    assert 0 < need <= keep and back > 0
    assert L.eacs_delta_fwd(delta(), P, None, P, need - 1, 0, None) == _lib.EACS_ERR_WORKSPACE
    assert L.eacs_delta_fwd(delta(), P, None, None, 0, 0, None) == _lib.EACS_ERR_WORKSPACE
    assert L.eacs_delta_fwd(delta(), P, None, P + 8, keep, 1, None) == _lib.EACS_ERR_INVALID
    bwd = lambda saved, ws, do=P: L.eacs_delta_bwd(delta(), do, strides, None, P, P, P, P, P, None, P, saved, P, ws, None)
    assert bwd(keep - 1, back) == _lib.EACS_ERR_WORKSPACE and bwd(keep, back - 1) == _lib.EACS_ERR_WORKSPACE
    assert bwd(keep, back, None) == _lib.EACS_ERR_INVALID
    for kw in (dict(B=0), dict(L=0)):
        assert L.eacs_delta_fwd(delta(**kw), None, None, None, 0, 0, None) == _lib.EACS_OK
        assert L.eacs_delta_bwd(delta(**kw), None, strides, None, *[None] * 6, None, 0, None, 0, None) == _lib.EACS_OK
    assert L.eacs_delta_step(delta(B=0), None, None, None) == _lib.EACS_OK
    for f in (L.eacs_delta_fwd, ):
        assert f(None, P, None, P, 1, 0, None) == _lib.EACS_ERR_INVALID


def test_python_refusals():
    from eacs_b200.ops.gated_delta import gated_delta_rule, gated_delta_step
    from eacs_b200.ops.layer_norm import layer_norm
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x)
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_delta_rule(q, q, q, q[..., 0], q[..., 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_delta_step(q[:, 0], q[:, 0], q[:, 0], q[:, 0, :, 0], q[:, 0, :, 0], torch.zeros(1, 2, 8, 8))


def test_norm_module_on_cpu_and_use_norms():
    from eacs_b200.ops.layer_norm import LayerNorm, use_norms
    model = nn.Sequential(nn.LayerNorm(8), nn.Linear(8, 8), nn.LayerNorm((4, 8)))
    want = model(torch.randn(2, 4, 8, generator=torch.Generator().manual_seed(0)))
    keys = list(model.state_dict())
    assert use_norms(model) == 2 and use_norms(model) == 0
    assert type(model[0]) is LayerNorm and list(model.state_dict()) == keys
    assert torch.equal(model(torch.randn(2, 4, 8, generator=torch.Generator().manual_seed(0))), want)


def test_install_norms(monkeypatch):
    """install(norms=True) on a package with the reference's module names."""
    import eacs_b200
    from eacs_b200.ops.layer_norm import LayerNorm
    names = {"modules.eacs": "EACSLayer", "modules.continuous_ssm": "ContinuousSSMLayer", "modules.multiscale": "MultiScaleEACS"}
    mods = {}
    for n in ("", "ops", "modules", "ops.scan_cuda", "ops.eacs_gated_scan", "ops.eacs_cell_train", *names):
        mods[n] = types.ModuleType("fake_ssm" + ("." + n if n else ""))
        mods[n].__path__ = []
        monkeypatch.setitem(sys.modules, mods[n].__name__, mods[n])

    for n, cls in names.items():
        class Layer(nn.Module):
            def __init__(self, d):
                super().__init__()
                self.norm = nn.LayerNorm(d)
        setattr(mods[n], cls, Layer)
    patched = eacs_b200.install("fake_ssm", norms=True)
    eacs_b200.install("fake_ssm", norms=True)
    for n, cls in names.items():
        assert cls + ".__init__" in patched
        assert type(getattr(mods[n], cls)(8).norm) is LayerNorm
        assert not hasattr(getattr(mods[n], cls).__init__.__wrapped__, "__wrapped__")


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_delta_rejects_outputs_off_16_bytes_without_device(dtype):
    """Outputs and 16-bit gradients are written up to 16 bytes at a time."""
    L = _lib.lib()
    strides, big = (ctypes.c_int64 * 3)(1, 1, 1), 1 << 40
    off = P + (4 if dtype == 0 else 2)
    assert L.eacs_delta_fwd(delta(dtype=dtype, gate=dtype), off, None, P, big, 0, None) == _lib.EACS_ERR_INVALID
    assert "16 bytes" in _lib.last_error()
    for i in range(3):
        grads = [P] * 5
        grads[i] = off
        assert L.eacs_delta_bwd(delta(dtype=dtype, gate=dtype), P, strides, None, *grads, None, P, big, P, big,
                                None) == _lib.EACS_ERR_INVALID
        assert "16 bytes" in _lib.last_error()


def test_delta_path_named_by_the_caller_without_device():
    """A named path decides the layout; one that the inputs do not allow is refused."""
    L = _lib.lib()
    strides = (ctypes.c_int64 * 3)(64, 8, 8)

    def args(path, q=P, dtype=2, K=16):
        st = []
        for n in (K, K, 8, 1, 1):
            st += [640 * n, 64 * n, n]
        return _lib.DELTA_PATH.pack(q, P, P, P, P, *st, 0, 0, 2, 10, 4, 4, K, 8, 1.0, dtype, dtype, path)
    assert _lib.DELTA_PATH.size == _lib.DELTA.size
    assert L.eacs_delta_path(args(0)) == 2 and L.eacs_delta_path(args(0, q=P + 2)) == 1
    assert L.eacs_delta_path(args(0, K=12)) == 1 and L.eacs_delta_path(args(0, dtype=0)) == 1
    assert L.eacs_delta_path(args(0, dtype=1)) == 2 and L.eacs_delta_path(args(1)) == 1
    assert L.eacs_delta_path(None) == 0
    for size in (lambda a: L.eacs_delta_workspace_size(a, 1), L.eacs_delta_bwd_workspace_size):
        assert size(args(0)) == size(args(2)) != size(args(1)) == size(args(0, q=P + 2))
    big = 1 << 40
    for bad in (args(2, q=P + 2), args(2, dtype=0), args(3), args(-1)):
        assert L.eacs_delta_path(bad) == 0 and L.eacs_delta_workspace_size(bad, 1) == 0
        assert L.eacs_delta_fwd(bad, P, None, P, big, 1, None) == _lib.EACS_ERR_INVALID
        assert L.eacs_delta_bwd(bad, P, strides, None, P, P, P, P, P, None, P, big, P, big, None) == _lib.EACS_ERR_INVALID


def test_forward_mode_transforms_and_traces_are_seen():
    """What a kernel called by pointer would drop: tangents, transforms' wrappers, records of a trace."""
    from torch.autograd import forward_ad
    from eacs_b200.ops._check import is_plain, require_plain
    x, seen = torch.ones(3), []
    assert is_plain(x, None) and is_plain(x.clone().requires_grad_(True))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert is_plain(x) and not is_plain(x, None, dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            require_plain("op", dual)
    note = lambda t: seen.append(is_plain(t)) or t * 1
    torch.func.vmap(note)(torch.ones(2, 2))
    torch.func.jvp(note, (x,), (x,))
    torch.func.grad(lambda t: note(t).sum())(x)
    assert seen == [False] * 3 and is_plain(x)
    seen.clear()
    torch.jit.trace(note, x, check_trace=False)
    assert False in seen and is_plain(x)


@pytest.mark.parametrize("residual", [False, True])
def test_norm_gradients_that_are_differentiated_again(residual):
    """The recorded form of the norm's backward, its values and its own gradients, against torch's norm in 64 bits.  Sums of
    40 terms in float32, some ten operations deep: 2^-24 * 40 = 2.4e-6 of the norm at most, 1e-5 for the second step."""
    from eacs_b200.ops.layer_norm import _recorded_gradients
    g = torch.Generator().manual_seed(1)
    x, r, dy, up = (torch.randn(3, 7, 40, generator=g) for _ in range(4))
    w, b, uw, ub = (torch.randn(40, generator=g) for _ in range(4))
    res = []
    for dt in (torch.float32, torch.float64):
        leaves = [t.to(dt).requires_grad_(True) for t in (x, r, w, dy)]
        xx, rr, ww, dd = leaves
        if dt == torch.float32:
            first = _recorded_gradients(xx, ww, rr if residual else None, dd, 1e-5)
        else:
            bb = b.to(dt).requires_grad_(True)
            s = xx + rr if residual else xx + 0 * rr
            first = torch.autograd.grad(nn.functional.layer_norm(s, (40,), ww, bb, 1e-5), (xx, ww, bb), dd, create_graph=True)
        second = torch.autograd.grad(first, leaves, [t.to(dt) for t in (up, uw, ub)], allow_unused=True)
        res.append([*first, *second])
    for i, (a, c) in enumerate(zip(*res)):
        if a is None:  # without a residual
            assert i == 4 and not residual and float(c.abs().max()) == 0.0
            continue
        assert float((a.detach().double() - c.detach()).norm()) <= (2.4e-6 if i < 3 else 1e-5) * float(c.detach().norm()), i
