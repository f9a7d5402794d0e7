"""The exponentials inside the selective scan, the convolution and the gated norms, by themselves: inputs under which an
output is softplus(v), silu(v) or a derivative of them and nothing else, in float32, against 64 bits.

Bounds, relative.  The hardware's 2^v is off by 2^-22 and its quotient by 2^-22; a sum, a product and the rest of an
argument's rounding by 2^-24 each, at most eight of them: 2^-20 in all.  Silu's argument is rounded once, and log2(e) before it:
|v| (2^-24 + 2^-26) of e^-v more.  A derivative of silu takes the sigmoid twice: twice that of its terms' sizes
s + |v| s (1 - s).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, LOWEST = float("inf"), torch.finfo(torch.float32).min

if torch.cuda.is_available():
    from eacs_b200.ops.block_norm import gated_norm, residual_norm
    from eacs_b200.ops.causal_conv import causal_conv, causal_conv_step
    from eacs_b200.ops.selective_ssm import selective_ssm, selective_ssm_step


def ones(*s):
    return torch.ones(*s, device=DEV)


def row(lo, hi, n=40000):
    return torch.linspace(lo, hi, n, device=DEV)


def softplus_scan(v):
    """One token, x = B = C = 1 and a state of 0: y is the step."""
    n = v.numel()
    return selective_ssm(ones(1, 1, n), v.view(1, 1, n), torch.zeros(n, 1, device=DEV), ones(1, 1, 1), ones(1, 1, 1)).view(n)


def softplus_step(v):
    n = v.numel()
    return selective_ssm_step(ones(1, n), v.view(1, n), torch.zeros(n, 1, device=DEV), ones(1, 1), ones(1, 1),
                              torch.zeros(1, n, 1, device=DEV)).view(n)


def silu_scan(v):
    """y = skip x silu(z) with B = 0 and skip = x = 1."""
    n = v.numel()
    zero = torch.zeros(1, 1, 1, device=DEV)
    return selective_ssm(ones(1, 1, n), zero.expand(1, 1, n), -ones(n, 1), zero, zero, ones(n), v.view(1, 1, n)).view(n)


def silu_scan_step(v):
    n = v.numel()
    zero = torch.zeros(1, 1, device=DEV)
    return selective_ssm_step(ones(1, n), zero.expand(1, n), -ones(n, 1), zero, zero, torch.zeros(1, n, 1, device=DEV), ones(n),
                              v.view(1, n)).view(n)


def taps(n):
    return torch.tensor([0.0, 1.0], device=DEV).repeat(n, 1)


def silu_conv(v):
    return causal_conv(v.view(1, 1, -1), taps(v.numel())).view(-1)


def silu_conv_odd(v):
    """Odd rows: the kernels of one channel a thread."""
    v = torch.cat([v, v[:1]])
    return causal_conv(v.view(1, 1, -1), taps(v.numel())).view(-1)[:-1]


def silu_conv_step(v):
    return causal_conv_step(v.view(1, -1), taps(v.numel()), None, torch.zeros(1, 1, v.numel(), device=DEV)).view(-1)


def silu_norm(v):
    """Rows of ones with eps = 0: their norm is 1."""
    return gated_norm(ones(v.numel() // 16, 16), v.view(-1, 16), eps=0.0).view(-1)


def silu_residual(v):
    g = v.view(-1, 16)
    return residual_norm(torch.ones_like(g), torch.zeros_like(g), gate=g)[1].view(-1)


def grad(f, v):
    v = v.clone().requires_grad_(True)
    return torch.autograd.grad(f(v).sum(), v)[0]


SILUS = [silu_scan, silu_conv, silu_conv_odd, silu_norm, silu_residual]
STEPS = [silu_scan_step, silu_conv_step]


@pytest.mark.parametrize("f", [softplus_scan, softplus_step])
def test_softplus(f):
    for lo, hi in ((-86, -20), (-20, 0), (0, 3), (3, 50)):
        v = row(lo, hi)
        want = torch.nn.functional.softplus(v.double(), threshold=60)
        assert float(((f(v).double() - want).abs() / want).max()) <= 2.0 ** -20, (lo, hi)


def test_slope_of_softplus():
    for lo, hi in ((-86, -20), (-20, 0), (0, 3), (3, 50)):
        v = row(lo, hi)
        want = torch.sigmoid(v.double())
        assert float(((grad(softplus_scan, v).double() - want).abs() / want).max()) <= 2.0 ** -20, (lo, hi)


@pytest.mark.parametrize("f", [softplus_scan, softplus_step])
def test_steps_far_to_either_side(f):
    """A token masked by -inf, or by the type's lowest value, takes no step at all."""
    v = torch.tensor([-INF, LOWEST, -1e30, -1e5, -200.0, -120.0, 1e30, 1e5, 200.0, 88.0], device=DEV)
    want = [0.0] * 6 + [1e30, 1e5, 200.0, 88.0]
    got = f(v)
    assert torch.equal(got, torch.tensor(want, device=DEV)), got
    assert bool(torch.isnan(f(torch.full((4,), float("nan"), device=DEV))).all())
    edge = row(-110, -86)  # what float32 holds in fewer bits may be 0
    assert float((f(edge).double() - torch.exp(edge.double())).abs().max()) <= 2.0 ** -126 * 1.5


def test_slope_of_steps_far_to_either_side():
    v = torch.tensor([-INF, LOWEST, -1e5, -200.0, 1e30, 200.0, 88.0], device=DEV)
    assert torch.equal(grad(softplus_scan, v), torch.tensor([0.0, 0, 0, 0, 1, 1, 1], device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_masked_tokens_keep_the_state(dtype):
    """dt = -inf or the lowest value in some places of a sequence: the state passes them unchanged, and no gradient goes in."""
    g = torch.Generator(DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, dt, Bs, Cs = rnd(2, 24, 32).to(dtype), rnd(2, 24, 32).to(dtype), rnd(2, 24, 16).to(dtype), rnd(2, 24, 16).to(dtype)
    A, h0 = -rnd(32, 16).abs(), rnd(2, 32, 16)
    h0[0] = 0
    for low in (-INF, torch.finfo(dtype).min):
        dt[:, :] = low
        leaf = dt.clone().requires_grad_(True)
        y, last = selective_ssm(x, leaf, A, Bs, Cs, initial_state=h0, output_final_state=True)
        assert torch.equal(last, h0) and float(y[0].detach().abs().max()) == 0
        ddt = torch.autograd.grad((y, last), leaf, (torch.ones_like(y), torch.ones_like(last)))[0]
        assert float(ddt.abs().max()) == 0
        state = h0.clone()
        selective_ssm_step(x[:, 0], dt[:, 0], A, Bs[:, 0], Cs[:, 0], state)
        assert torch.equal(state, h0)


@pytest.mark.parametrize("f", SILUS + STEPS)
def test_silu(f):
    for lo, hi in ((-85, -40), (-40, -8), (-8, -1), (-1, -1e-6), (1e-6, 5), (5, 80)):
        v = row(lo, hi)
        want = torch.nn.functional.silu(v.double())
        tol = 2.0 ** -20 + v.double().abs() * (2.0 ** -24 + 2.0 ** -26)
        assert bool(((f(v).double() - want).abs() <= tol * want.abs()).all()), (lo, hi)


@pytest.mark.parametrize("f", SILUS)
def test_slope_of_silu(f):
    for lo, hi in ((-85, -40), (-40, -8), (-8, 0), (0, 5), (5, 80)):
        v = row(lo, hi)
        s = torch.sigmoid(v.double())
        want, mag = s + v.double() * s * (1 - s), s + v.double().abs() * s * (1 - s)
        tol = 2 * (2.0 ** -20 + v.double().abs() * (2.0 ** -24 + 2.0 ** -26))
        assert bool(((grad(f, v).double() - want).abs() <= tol * mag).all()), (lo, hi)


@pytest.mark.parametrize("f", SILUS + STEPS)
def test_silu_far_to_either_side(f):
    v = torch.tensor([1e2, 1e5, 1e30, 3e38, INF] + [1.0] * 11 + [-1e2, -1e5, -1e30, LOWEST] + [0.0] * 12, device=DEV)
    got = f(v)
    assert torch.equal(got[:5], v[:5]) and float(got[16:20].abs().max()) <= 1e-36 and float(got[20:].abs().max()) == 0
    assert bool(torch.isnan(f(torch.full((16,), float("nan"), device=DEV))).all())
