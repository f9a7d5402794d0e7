"""Calls of the scans, the convolution and the norms that autograd could divert: forward-mode tangents, torch.func transforms
and traces are refused before anything has changed, a backward with create_graph gives gradients that are not differentiated
again, and inference mode gives the same bits."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200.ops.block_norm import gated_norm, residual_norm
    from eacs_b200.ops.causal_conv import causal_conv, causal_conv_step
    from eacs_b200.ops.gated_delta import gated_delta_rule
    from eacs_b200.ops.selective_ssm import selective_ssm, selective_ssm_step


def calls():
    """name -> (function of its float tensors, those tensors); a step's state comes last."""
    g = torch.Generator(DEV).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, dt, z, Bs, Cs = rnd(2, 9, 24), rnd(2, 9, 24), rnd(2, 9, 24), rnd(2, 9, 16), rnd(2, 9, 16)
    A, skip, bias, h0 = -rnd(24, 16).abs(), rnd(24), rnd(24), rnd(2, 24, 16)
    w, b, c0, n = rnd(24, 4), rnd(24), rnd(2, 3, 24), rnd(24)
    t = lambda v: v[:, 0].contiguous()
    return {
        "scan": (lambda *a: selective_ssm(*a[:8], initial_state=a[8]), (x, dt, A, Bs, Cs, skip, z, bias, h0)),
        "scan step": (lambda x, dt, A, Bs, Cs, skip, z, bias, s: selective_ssm_step(x, dt, A, Bs, Cs, s, skip, z, bias),
                      (t(x), t(dt), A, t(Bs), t(Cs), skip, t(z), bias, h0)),
        "convolution": (lambda x, w, b, s: causal_conv(x, w, b, initial_state=s), (x, w, b, c0)),
        "convolution step": (lambda x, w, b, s: causal_conv_step(x, w, b, s), (t(x), w, b, c0)),
        "gated delta rule": (lambda q, k, v, g, b, s: gated_delta_rule(q, k, v, g, b, initial_state=s),
                             (rnd(2, 9, 2, 16), rnd(2, 9, 2, 16), rnd(2, 9, 2, 8), -rnd(2, 9, 2).abs(), torch.sigmoid(rnd(2, 9, 2)),
                              rnd(2, 2, 16, 8))),
        "gated norm": (gated_norm, (x, z, n)),
        "residual norm": (lambda x, r, w, c, g, p: residual_norm(x, r, w, c, g, p)[0], (x, dt, n, skip, z, bias)),
    }


NAMES = ["scan", "scan step", "convolution", "convolution step", "gated delta rule", "gated norm", "residual norm"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_and_traced_inputs_are_refused(name):
    f, args = calls()[name]
    before = args[-1].clone()
    with forward_ad.dual_level():
        for i in range(len(args)):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*dual)
    with torch.no_grad(), pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(f, args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="torch.func"):
        torch.func.vmap(lambda t: f(t, *args[1:]))(torch.stack([args[0]] * 2))
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda t: f(t, *args[1:]).sum())(args[0])
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.jvp(lambda t: f(t, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
    assert torch.equal(args[-1], before)


@pytest.mark.parametrize("name", [n for n in NAMES if "step" not in n])
def test_a_gradient_is_not_differentiated_again(name):
    f, args = calls()[name]
    leaves = [t.clone().requires_grad_(True) for t in args]
    plain = torch.autograd.grad(f(*leaves).sum(), leaves)
    first = torch.autograd.grad(f(*leaves).sum(), leaves, create_graph=True)
    for a, b in zip(plain, first):
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(b.sum(), leaves, allow_unused=True, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):  # a penalty among terms that do have a gradient
            torch.autograd.grad(b.square().sum() + leaves[0].square().sum(), leaves, allow_unused=True, retain_graph=True)


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(name):
    f, args = calls()[name]
    with torch.no_grad():
        state = args[-1].clone()
        want = f(*args[:-1], state)
    with torch.inference_mode():
        made = [t.clone() for t in args]  # tensors of inference mode
        assert torch.equal(f(*made), want)
        if "step" in name:
            assert torch.equal(made[-1], state)
    with torch.no_grad():  # and outside of it
        again = torch.inference_mode()(lambda: [t.clone() for t in args])()
        assert torch.equal(f(*again), want)
        if "step" in name:
            assert torch.equal(again[-1], state)


@pytest.mark.parametrize("name", [n for n in NAMES if "step" not in n])
def test_what_a_backward_needs_may_not_have_changed(name):
    f, args = calls()[name]
    for i in range(len(args)):
        leaves = [t.clone().requires_grad_(True) for t in args]
        loss = f(*leaves).sum()
        with torch.no_grad():
            leaves[i].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("name", ["scan step", "convolution step"])
def test_a_step_is_seen_by_autograd(name):
    """A state that a graph still needs may not be stepped: the backward says so."""
    f, args = calls()[name]
    state = args[-1].clone()
    w = torch.ones_like(state, requires_grad=True)
    loss = (w * state).sum()
    with torch.no_grad():
        f(*args[:-1], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("name", [n for n in NAMES if "step" not in n])
def test_a_graph_kept_and_run_twice(name):
    f, args = calls()[name]
    leaves = [t.clone().requires_grad_(True) for t in args]
    loss = f(*leaves).sum()
    loss.backward(retain_graph=True)
    once = [t.grad.clone() for t in leaves]
    loss.backward()
    for t, g in zip(leaves, once):
        assert torch.equal(t.grad, g + g)
