"""The gated delta rule (eacs_delta_*) against its token-by-token definition in 64 bits.

Tolerances are on |got - want| in the 2-norm over |want|.  Operands of the
matrix products keep at least 16 significant bits (2^-17 each), a token's way
from inputs to an output or gradient passes a handful of them and float32
sums, so computed values stay under 16 * 2^-17 = 1.3e-4 of their norm in the
worst case and, errors being of either sign, near 2^-17 * sqrt(16) = 3.1e-5:
TOL = 6.2e-5, twice that.  One rounding to the output's type adds eps / 2.

In the backward of 16-bit inputs one operand on a gradient's way, dV, is
rounded to one value of their type: off by up to half a step of an element,
2^-9 for bfloat16 and 2^-12 for float16.  That is what a float32 gradient
beside them may be off by (ONE); 16-bit ones have their own rounding, eps / 2,
and stay under it with both (each is 1 / sqrt(3) of its half step in the mean:
together 0.65 eps / 2).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 6.2e-5
ONE = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12, torch.float32: TOL}

if torch.cuda.is_available():
    from eacs_b200.ops.gated_delta import gated_delta_rule, gated_delta_step
    from eacs_b200.ops.layer_norm import layer_norm


def tol(dtype, inputs=torch.float32):
    """inputs: the type of q, k and v, for gradients."""
    if dtype != torch.float32:
        return TOL + torch.finfo(dtype).eps / 2
    return ONE[inputs]


def close(got, want, times=1.0, what="", inputs=torch.float32):
    assert got.shape == want.shape, what
    want = want.to(got.device)
    err, ref = float((got.double() - want).norm()), float(want.norm())
    assert err <= times * tol(got.dtype, inputs) * ref + 1e-12, (what, err / max(ref, 1e-30))


def oracle(q, k, v, g, beta, scale, initial=None, lengths=None):
    """(o, final state), differentiable, float64."""
    B, L, Hk, K = q.shape
    Hv, V = v.shape[2:]
    r = Hv // Hk
    q, k = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
    S = q.new_zeros(B, Hv, K, V) if initial is None else initial
    outs = []
    for t in range(L):
        Sd = S * g[:, t].exp()[..., None, None]
        u = beta[:, t][..., None] * (v[:, t] - (Sd * k[:, t][..., None]).sum(-2))
        Sn = Sd + k[:, t][..., None] * u[..., None, :]
        o = (Sn * q[:, t][..., None]).sum(-2) * scale
        if lengths is not None:
            live = (t < lengths).view(B, 1, 1)
            o = torch.where(live, o, torch.zeros_like(o))
            Sn = torch.where(live[..., None], Sn, S)
        S = Sn
        outs.append(o)
    return torch.stack(outs, 1) if outs else v.new_zeros(B, 0, Hv, V), S


def make(B, L, Hk, Hv, K, V, dtype, gate=None, seed=0, initial=True):
    gen = torch.Generator(DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    k = rnd(B, L, Hk, K) + 0.8 * rnd(B, 1, Hk, K)
    q = rnd(B, L, Hk, K)
    gate = dtype if gate is None else gate
    d = dict(q=(q / q.norm(dim=-1, keepdim=True)).to(dtype), k=(k / k.norm(dim=-1, keepdim=True)).to(dtype),
             v=rnd(B, L, Hv, V).to(dtype), g=(-torch.nn.functional.softplus(rnd(B, L, Hv)) * 0.2).to(gate),
             beta=torch.sigmoid(2 * rnd(B, L, Hv)).to(gate))
    if initial:
        d["initial"] = 0.5 * rnd(B, Hv, K, V)
    return d, rnd(B, L, Hv, V).to(dtype), rnd(B, Hv, K, V)


def both(d, do, dS, lengths=None, scale=None):
    """Kernel and oracle: outputs, final states and gradients by name."""
    scale = d["q"].shape[-1] ** -0.5 if scale is None else scale
    got, want = {}, {}
    for out, conv in ((got, lambda t: t.detach().clone()), (want, lambda t: t.detach().double().cpu())):
        x = {n: conv(t).requires_grad_(True) for n, t in d.items()}
        args = [x[n] for n in ("q", "k", "v", "g", "beta")]
        if out is got:
            o, S = gated_delta_rule(*args, scale=scale, initial_state=x.get("initial"), output_final_state=True, lengths=lengths)
            up = [do, dS]
        else:
            o, S = oracle(*args, scale, x.get("initial"), None if lengths is None else lengths.cpu())
            up = [do.double().cpu(), dS.double().cpu()]
        grads = torch.autograd.grad([o, S], list(x.values()), up, allow_unused=True)
        out.update(o=o.detach(), S=S.detach(), **{"d" + n: torch.zeros_like(t) if gr is None else gr
                                                  for (n, t), gr in zip(x.items(), grads)})
    return got, want


def compare(got, want, times=1.0):
    for n in want:
        assert bool(torch.isfinite(got[n]).all()), n
        close(got[n], want[n], times, n, got["dq"].dtype if n[0] == "d" else torch.float32)


SHAPES = [  # B, L, Hk, Hv, K, V
    (1, 1, 1, 1, 128, 128), (2, 2, 1, 2, 64, 64), (1, 63, 2, 2, 128, 64), (2, 64, 1, 1, 64, 128), (1, 65, 2, 4, 128, 128),
    (2, 130, 1, 3, 48, 40), (1, 257, 1, 1, 128, 200), (1, 90, 1, 2, 1, 1), (2, 70, 2, 2, 33, 17), (1, 129, 1, 1, 127, 130),
    (1, 100, 2, 2, 72, 24)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype):
    d, do, dS = make(*shape, dtype, seed=sum(shape))
    compare(*both(d, do, dS))


@pytest.mark.parametrize("shape", [(1, 130, 12, 24, 64, 200), (3, 130, 4, 16, 128, 128), (1, 130, 16, 64, 128, 104), (2, 193, 4, 32, 64, 128)])
def test_many_heads(shape):
    """Heads enough that a multiprocessor takes three or four groups of 16 value columns at once, the last ones partly
    filled; with what a backward reads kept and without."""
    d, do, dS = make(*shape, torch.bfloat16, seed=sum(shape))
    lengths = torch.tensor([shape[1], 66, 1][:shape[0]], dtype=torch.int32)
    got, want = both(d, do, dS, lengths.to(DEV))
    compare(got, want)
    with torch.no_grad():
        o, S = gated_delta_rule(*(d[n] for n in ("q", "k", "v", "g", "beta")), initial_state=d["initial"], output_final_state=True,
                                lengths=lengths.to(DEV))
    close(o, want["o"])
    close(S, want["S"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_gates_and_no_initial_state(dtype):
    d, do, dS = make(2, 150, 2, 4, 64, 96, dtype, torch.float32, seed=5, initial=False)
    got, want = both(d, do, dS, scale=0.7)
    assert got["dg"].dtype == torch.float32 and got["dbeta"].dtype == torch.float32
    compare(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_first_decay_of_an_empty_state_has_no_gradient(dtype):
    d, do, dS = make(3, 5, 1, 2, 64, 32, dtype, seed=30, initial=False)
    got, want = both(d, do, dS)
    assert float(want["dg"][:, 0].abs().max()) == 0.0 and float(got["dg"][:, 0].abs().max()) == 0.0
    compare(got, want)
    one, _ = both({n: t[:, :1] for n, t in d.items()}, do[:, :1], dS)
    assert float(one["dg"].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lengths(dtype):
    """Rows of no token, one token, up to a chunk's border and over L (clamped); what lies behind holds NaN and infinities."""
    lengths = [0, 1, 64, 100, 130, 500, -3]
    d, do, dS = make(len(lengths), 130, 1, 2, 64, 48, dtype, seed=6)
    dev = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    clean, want = both(d, do, dS, dev)
    compare(clean, want)
    for i, n in enumerate(lengths):
        n = min(max(n, 0), 130)
        assert float(clean["o"][i, n:].abs().sum()) == 0.0
        if n == 0:
            assert torch.equal(clean["S"][i], d["initial"][i]) and torch.equal(clean["dinitial"][i], dS[i])
        for name in ("q", "k", "v", "g", "beta"):
            assert float(clean["d" + name][i, n:].abs().sum()) == 0.0
            d[name][i, n:] = float("nan") if i % 2 else float("inf")
        do[i, n:] = float("nan")
    dirty, _ = both(d, do, dS, dev)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_resets_zero_and_double_rates(dtype):
    """g = -inf clears the state (and leaves the precision behind it), g = 0 keeps it; beta = 0 writes nothing,
    beta = 2 reflects."""
    d, do, dS = make(1, 140, 1, 2, 64, 64, dtype, seed=7)
    d["g"][0, 20], d["g"][0, 100, 0], d["g"][0, 30:60] = float("-inf"), -1e30, 0.0
    d["beta"][0, 10:14], d["beta"][0, 50], d["beta"][0, 51] = 0.0, 2.0, -0.5
    got, want = both(d, do, dS)
    want["dg"] = torch.nan_to_num(want["dg"])  # 0 * inf of the definition: the state before a reset has no weight
    for n in want:
        if n == "dg":
            # a reset's own gradient is a difference of terms of the size of its neighbours': of no sign, near 0
            live = torch.isfinite(d["g"]) & (d["g"] > -100)
            close(torch.where(live, got[n], torch.zeros_like(got[n])), torch.where(live.cpu(), want[n], torch.zeros_like(want[n])), 2.0, n)
            assert float(got[n][~live].abs().max()) <= 2 * tol(dtype) * float(want[n].abs().max()) * 8
        else:
            close(got[n], want[n], 1.0, n, dtype if n[0] == "d" else torch.float32)
    cut = {n: t[:, 20:] for n, t in d.items() if n != "initial"}  # from the reset on nothing of before is seen
    cut["g"] = cut["g"].clone()
    cut["g"][0, 0] = 0.0
    o = gated_delta_rule(*(cut[n] for n in ("q", "k", "v", "g", "beta")))
    close(got["o"][:, 20:], o.double(), 2.0)


def test_strong_decay_keeps_precision():
    """Decays of e^-60 and more a token: products of decays are formed from differences, not from quotients that overflow."""
    d, do, dS = make(1, 130, 1, 1, 64, 64, torch.float32, seed=8)
    d["g"] = d["g"] - 60.0 * (torch.rand(1, 130, 1, device=DEV, generator=torch.Generator(DEV).manual_seed(1)) < 0.3)
    got, want = both(d, do, dS)
    for n in want:
        if n != "dg":  # of decays near 0: products of numbers below 1e-26 beside rounding
            close(got[n], want[n], 1.0, n)
    assert float((got["dg"].double().cpu() - want["dg"]).abs().max()) <= 8 * TOL * float(want["dg"].abs().max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_views_of_a_fused_projection_and_broadcast(dtype):
    """Slices of one projection (aligned and not), a transposed layout, and keys shared by expansion."""
    B, L, H, K, V = 2, 100, 2, 64, 64
    d, do, _ = make(B, L, H, H, K, V, dtype, seed=9, initial=False)
    want, _ = oracle(*(d[n].double().cpu() for n in ("q", "k", "v", "g", "beta")), K ** -0.5)
    for pad in (0, 3):
        fused = torch.zeros(B, L, H * (2 * K + V + 2) + pad, dtype=dtype, device=DEV)
        parts, at = {}, pad
        for n in ("q", "k", "v", "g", "beta"):
            w = d[n].shape[-1] if d[n].dim() == 4 else 1
            view = fused[..., at:at + H * w].unflatten(-1, (H, w))
            view = view if d[n].dim() == 4 else view[..., 0]
            view.copy_(d[n])
            parts[n], at = view, at + H * w
        close(gated_delta_rule(*parts.values()), want)
    heads = {n: d[n].transpose(1, 2).contiguous().transpose(1, 2) for n in d}
    close(gated_delta_rule(*heads.values()), want)
    k = d["k"][:, :, :1].detach().clone().requires_grad_(True)  # one key head for all, by expansion
    args = lambda kk: (d["q"], kk.expand(B, L, H, K), d["v"], d["g"], d["beta"])
    dk = torch.autograd.grad(gated_delta_rule(*args(k)), k, do)[0]
    k64 = k.detach().double().cpu().requires_grad_(True)
    d64 = {n: t.double().cpu() for n, t in d.items()}
    o64, _ = oracle(d64["q"], k64.expand(B, L, H, K), d64["v"], d64["g"], d64["beta"], K ** -0.5)
    close(dk, torch.autograd.grad(o64, k64, do.double().cpu())[0], 2.0)  # rounded per head, then summed and rounded
    t = d["v"].detach().clone().transpose(-1, -2).contiguous().transpose(-1, -2)  # a value's elements apart
    close(gated_delta_rule(d["q"], d["k"], t, d["g"], d["beta"]), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(3, 7, 2, 4, 64, 40), (2, 5, 1, 1, 128, 128), (1, 6, 1, 2, 30, 37)])
def test_steps_continue_a_sequence(shape, dtype):
    """A prefill's state, then tokens one by one, give the whole sequence's outputs and state."""
    B, L, Hk, Hv, K, V = shape
    d, _, _ = make(B, 70 + L, Hk, Hv, K, V, dtype, seed=10)
    want, S_want = oracle(*(d[n].double().cpu() for n in ("q", "k", "v", "g", "beta")), K ** -0.5, d["initial"].double().cpu())
    head = [d[n][:, :70] for n in ("q", "k", "v", "g", "beta")]
    o, S = gated_delta_rule(*head, initial_state=d["initial"], output_final_state=True)
    outs, at = [o], S.data_ptr()
    for t in range(70, 70 + L):
        outs.append(gated_delta_step(*(d[n][:, t] for n in ("q", "k", "v", "g", "beta")), S)[:, None])
    assert S.data_ptr() == at
    close(torch.cat(outs, 1), want)
    close(S, S_want)


def test_step_state_past_32_bit_offsets():
    B, H, K, V = 4100, 32, 128, 128  # 2^31 state values and more
    gen = torch.Generator(DEV).manual_seed(11)
    q, k, v = (torch.randn(B, H, n, generator=gen, device=DEV).bfloat16() for n in (K, K, V))
    k = torch.nn.functional.normalize(k.float(), dim=-1).bfloat16()
    g, beta = -torch.rand(B, H, generator=gen, device=DEV), torch.rand(B, H, generator=gen, device=DEV)
    S = torch.zeros(B, H, K, V, device=DEV)
    S[-2:] = torch.randn(2, H, K, V, generator=gen, device=DEV)
    small = S[-2:].clone()
    o = gated_delta_step(q, k, v, g, beta, S)
    o2 = gated_delta_step(*(t[-2:] for t in (q, k, v, g, beta)), small)
    assert torch.equal(o[-2:], o2) and torch.equal(S[-2:], small)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_against_differences(dtype):
    """Directional fourth-order differences of the kernel's own forward.  h = 2^-4: truncation is h^4 = 1.5e-5 of a fifth
    derivative, and a forward off by up to TOL of |f| moves the slope by TOL |f| / h; float32 gates and state carry the
    directions exactly, bf16 tokens are left alone."""
    d, do, dS = make(1, 80, 1, 2, 64, 64, dtype, torch.float32, seed=12)
    names = ["g", "beta", "initial"] + (["q", "k", "v"] if dtype == torch.float32 else [])
    gen = torch.Generator(DEV).manual_seed(13)
    dirs = {n: 0.05 * torch.randn(d[n].shape, generator=gen, device=DEV) for n in names}
    up = torch.zeros_like(dS)

    def f(s):
        x = {n: t + s * dirs[n] if n in dirs else t for n, t in d.items()}
        S = gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)[1]
        return float((S.double() * dS.double()).sum())
    x = {n: t.detach().clone().requires_grad_(True) for n, t in d.items()}
    S = gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)[1]
    grads = torch.autograd.grad(S, [x[n] for n in names], dS)
    slope = float(sum((a.double() * dirs[n].double()).sum() for a, n in zip(grads, names)))
    h = 2.0 ** -4
    num = (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)
    size = float(S.detach().double().norm() * dS.double().norm())
    assert abs(num - slope) <= 4 * TOL * size / (h * size ** 0.5) + 2e-3 * abs(slope), (num, slope)
    assert up.shape == dS.shape


def test_only_some_gradients_and_only_one_output():
    d, do, dS = make(1, 70, 1, 1, 64, 64, torch.bfloat16, seed=14)
    full, _ = both(d, do, torch.zeros_like(dS))
    v = d["v"].detach().clone().requires_grad_(True)
    o, S = gated_delta_rule(d["q"], d["k"], v, d["g"], d["beta"], initial_state=d["initial"], output_final_state=True)
    assert torch.equal(torch.autograd.grad(o, v, do)[0], full["dv"])
    o, S = gated_delta_rule(d["q"], d["k"], v, d["g"], d["beta"], initial_state=d["initial"], output_final_state=True)
    gS = torch.autograd.grad(S, v, dS)[0]
    only, _ = both(d, torch.zeros_like(do), dS)
    assert torch.equal(gS, only["dv"])
    odd = torch.randn(1, 70, 64, 1, device=DEV).bfloat16().transpose(2, 3).expand(1, 70, 1, 64)  # an upstream gradient in another layout
    a = torch.autograd.grad(gated_delta_rule(d["q"], d["k"], v, d["g"], d["beta"]), v, odd)[0]
    b = torch.autograd.grad(gated_delta_rule(d["q"], d["k"], v, d["g"], d["beta"]), v, odd.contiguous())[0]
    assert torch.equal(a, b)


def test_same_bits_other_stream_and_graphs():
    d, do, dS = make(2, 200, 2, 4, 128, 128, torch.bfloat16, seed=15)
    x = {n: t.detach().clone().requires_grad_(True) for n, t in d.items()}
    state = torch.randn(2, 4, 128, 128, device=DEV)

    def step():
        o, S = gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)
        return (o.detach(), S.detach(), *torch.autograd.grad([o, S], list(x.values()), [do, dS]))
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    del side
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    with torch.no_grad():
        x["v"].mul_(0.5)
    want = step()
    for gr, _ in graphs:
        gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    first = state.clone()
    tok = [d[n][:, 0] for n in ("q", "k", "v", "g", "beta")]
    o1 = gated_delta_step(*tok, first)
    gr = torch.cuda.CUDAGraph()
    cap = state.clone()
    with torch.cuda.graph(gr):
        o2 = gated_delta_step(*tok, cap)
    cap.copy_(state)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(o1, o2) and torch.equal(first, cap)


def test_empty():
    q = torch.zeros(2, 0, 1, 64, device=DEV, requires_grad=True)
    v, g = torch.zeros(2, 0, 2, 32, device=DEV), torch.zeros(2, 0, 2, device=DEV)
    S0 = torch.randn(2, 2, 64, 32, device=DEV, requires_grad=True)
    o, S = gated_delta_rule(q, q, v, g, g, initial_state=S0, output_final_state=True)
    assert o.shape == (2, 0, 2, 32) and torch.equal(S, S0)
    up = torch.randn_like(S0)
    assert torch.equal(torch.autograd.grad(S, S0, up)[0], up)
    with torch.no_grad():
        assert float(gated_delta_rule(q, q, v, g, g, output_final_state=True)[1].abs().sum()) == 0.0
    assert gated_delta_rule(q[:0], q[:0], v[:0], g[:0], g[:0]).shape == (0, 0, 2, 32)
    assert gated_delta_step(*(torch.zeros(0, 2, 8, device=DEV) for _ in range(3)), torch.zeros(0, 2, device=DEV),
                            torch.zeros(0, 2, device=DEV), torch.zeros(0, 2, 8, 8, device=DEV)).shape == (0, 2, 8)


def test_norm_projection_delta_norm_together():
    """A pre-norm block, y = norm(x + proj(delta(norm(x)))): trained end to end, then streamed frame by frame."""
    B, L, D, H = 2, 75, 64, 2
    K = D // H
    gen = torch.Generator(DEV).manual_seed(16)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    P = dict(w1=1 + 0.1 * rnd(D), b1=0.1 * rnd(D), win=rnd(3 * D + 2 * H, D) * D ** -0.5, wo=rnd(D, D) * D ** -0.5,
             w2=1 + 0.1 * rnd(D), b2=0.1 * rnd(D))
    x, dy = rnd(B, L, D), rnd(B, L, D)

    def project(h, win):
        q, k, v, a, b = (h @ win.t()).split([D, D, D, H, H], -1)
        q, k, v = (t.unflatten(-1, (H, K)) for t in (q, k, v))
        return (torch.nn.functional.normalize(q, dim=-1), torch.nn.functional.normalize(k, dim=-1), v,
                torch.nn.functional.logsigmoid(a), torch.sigmoid(b))

    def block(x, p, norm, rule):
        o = rule(*project(norm(x, p["w1"], p["b1"], None), p["win"]))
        return norm(x, p["w2"], p["b2"], o.flatten(-2) @ p["wo"].t())
    ours = lambda x, w, b, r: layer_norm(x, w, b, 1e-5, residual=r)
    plain = lambda x, w, b, r: torch.nn.functional.layer_norm(x if r is None else x + r, (D,), w, b, 1e-5)
    got, want = {}, {}
    for out, conv in ((got, lambda t: t.clone()), (want, lambda t: t.double().cpu())):
        p = {n: conv(t).requires_grad_(True) for n, t in P.items()}
        xx = conv(x).requires_grad_(True)
        rule = gated_delta_rule if out is got else lambda *a: oracle(*a, K ** -0.5)[0]
        y = block(xx, p, ours if out is got else plain, rule)
        leaves = [xx, *p.values()]
        out.update(y=y.detach(), **dict(zip(["x", *p], torch.autograd.grad(y, leaves, conv(dy)))))
    for n in want:
        close(got[n], want[n], 2.0, n)  # two norms and two products around the rule
    with torch.no_grad():  # streaming: a prefill of 70 frames, then one frame at a time
        q, k, v, g, b = project(layer_norm(x, P["w1"], P["b1"]), P["win"])
        _, S = gated_delta_rule(q[:, :70], k[:, :70], v[:, :70], g[:, :70], b[:, :70], output_final_state=True)
        for t in range(70, L):
            q, k, v, g, b = project(layer_norm(x[:, t], P["w1"], P["b1"]), P["win"])
            o = gated_delta_step(q, k, v, g, b, S)
            y = layer_norm(x[:, t], P["w2"], P["b2"], residual=o.flatten(-2) @ P["wo"].t())
            close(y, want["y"][:, t], 2.0)


def test_refusals():
    d, _, _ = make(2, 8, 2, 4, 16, 8, torch.bfloat16, seed=17)
    q, k, v, g, b, S = (d[n] for n in ("q", "k", "v", "g", "beta", "initial"))
    ok = dict(q=q, k=k, v=v, g=g, beta=b)
    for bad in (dict(k=k[:, :7]), dict(v=v[:, :, :3]), dict(g=g[..., :2]), dict(beta=b.float()), dict(g=g.half(), beta=b.half()),
                dict(k=k.float()), dict(q=q.double(), k=k.double(), v=v.double()), dict(initial_state=S.half()),
                dict(initial_state=S[:1]), dict(lengths=torch.tensor([8, 8], device=DEV)),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(lengths=torch.zeros(2, dtype=torch.int32)),
                dict(q=q[..., :0], k=k[..., :0]), dict(v=v.cpu())):
        with pytest.raises(RuntimeError):
            gated_delta_rule(**{**ok, **bad})
    wide = torch.zeros(1, 2, 1, 129, device=DEV)
    with pytest.raises(RuntimeError, match="128"):
        gated_delta_rule(wide, wide, wide, wide[..., 0], wide[..., 0])
    tok = [t[:, 0] for t in (q, k, v, g, b)]
    for bad in (S.transpose(0, 1).contiguous().transpose(0, 1), S.half(), S[:1], S.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError):
            gated_delta_step(*tok, bad)
    leaf = S.clone()
    x = torch.ones(2, 4, 16, 8, device=DEV, requires_grad=True)
    y = (x * leaf).sum()  # autograd keeps leaf for its backward
    gated_delta_step(*tok, leaf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_step_refuses_inputs_that_want_a_gradient():
    d, _, _ = make(2, 1, 1, 2, 16, 8, torch.float32, seed=31)
    tok = [d[n][:, 0] for n in ("q", "k", "v", "g", "beta")]
    before = d["initial"].clone()
    for i in range(5):
        bad = [t.clone().requires_grad_(j == i) for j, t in enumerate(tok)]
        with pytest.raises(RuntimeError, match="no gradient"):
            gated_delta_step(*bad, d["initial"])
        assert torch.equal(d["initial"], before)
        with torch.no_grad():
            o = gated_delta_step(*bad, d["initial"].clone())
        assert torch.equal(o, gated_delta_step(*tok, d["initial"].clone()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_backward_twice_and_two_calls_at_once(dtype):
    """What a forward keeps serves every backward of it; calls on two streams share nothing."""
    runs = []
    for i in range(2):
        d, do, dS = make(2, 300, 2, 4, 128, 64, dtype, seed=32 + i)
        x = {n: t.detach().clone().requires_grad_(True) for n, t in d.items()}
        runs.append((x, do, dS))

    def forward(x):
        return gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)
    want = []
    for x, do, dS in runs:
        out = forward(x)
        first = torch.autograd.grad(out, list(x.values()), [do, dS], retain_graph=True)
        again = torch.autograd.grad(out, list(x.values()), [do, dS])
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        want.append([t.detach() for t in out] + list(first))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in runs], [[], []]
    for _ in range(3):
        for i, (x, do, dS) in enumerate(runs):
            with torch.cuda.stream(streams[i]):
                out = forward(x)
                got[i].append([t.detach() for t in out] + list(torch.autograd.grad(out, list(x.values()), [do, dS])))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_sequences_past_32_bit_offsets():
    """The last row of a batch with over 2^31 values, forward and backward, against that row alone (each within the
    tolerance of the truth)."""
    B, L, H, K, V = 2, 66000, 128, 64, 128
    gen = torch.Generator(DEV).manual_seed(34)
    rnd = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    x = dict(q=rnd(B, L, H, K).mul_(K ** -0.5), k=rnd(B, L, H, K).mul_(K ** -0.5), v=rnd(B, L, H, V),
             g=-0.1 * torch.rand(B, L, H, generator=gen, device=DEV), beta=torch.rand(B, L, H, generator=gen, device=DEV))
    do = rnd(B, L, H, V)
    res = []
    for rows in (slice(0, B), slice(B - 1, B)):
        leaves = [t[rows].detach().requires_grad_(True) for t in x.values()]
        o, S = gated_delta_rule(*leaves, output_final_state=True)
        grads = torch.autograd.grad(o, leaves, do[rows])
        res.append([t[-1].detach().clone() for t in (o, S, *grads)])
        del o, S, grads, leaves
    for n, a, b in zip(("o", "S", "dq", "dk", "dv", "dg", "dbeta"), *res):
        err, ref = float((a.float() - b.float()).norm()), float(b.float().norm())
        assert ref > 0 and err <= 2 * tol(a.dtype, torch.bfloat16) * ref, (n, err / ref)
    del x, do, res
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_and_infinity_of_a_token_reach_what_follows(dtype, pad, bad):
    """Also NaN with every bit set; rows that start on 16 bytes and not.  The chunks before are as they were."""
    d, _, _ = make(1, 200, 1, 2, 64, 64, dtype, seed=35)
    clean = {n: t.clone() for n, t in d.items()}
    d["k"][0, 70, 0, 5] = bad
    if bad != bad:
        bits = d["k"].view(torch.int16 if dtype.itemsize == 2 else torch.int32)
        bits[0, 70, 0, 5] = torch.iinfo(bits.dtype).max
    outs = []
    for x in (clean, d):
        args = []
        for n in ("q", "k", "v"):
            wide = torch.zeros(*x[n].shape[:-1], 64 + 8 + pad, dtype=dtype, device=DEV)
            wide[..., pad:pad + 64].copy_(x[n])
            args.append(wide[..., pad:pad + 64])
        outs.append(gated_delta_rule(*args, x["g"], x["beta"], initial_state=x["initial"], output_final_state=True))
    (o0, S0), (o1, S1) = outs
    assert bool(torch.isfinite(o0).all() and torch.isfinite(S0).all())
    assert torch.equal(o0[:, :64], o1[:, :64])
    assert not bool(torch.isfinite(o1[:, 128:]).any()) and not bool(torch.isfinite(S1).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 1e4, 1e6])
@pytest.mark.parametrize("K", [64, 128])
def test_small_rates_and_gradients_of_any_size(dtype, size, K):
    """Rates of 0, 1e-7 and 1e-4 among others, upstream gradients from 1e-6 to beyond float16's range (the final state's,
    in float32; the outputs' as far as their type goes).  A 16-bit gradient that is not a normal number of its type is off by half a
    step of the smallest (2^-25 in float16); one beyond its range is infinite.  Of a token whose rate is small, dbeta is
    the product of two vectors of V values that are off by TOL of their norms: by 2 TOL |a| |b|, which is 2 TOL sqrt(V) of
    the norm of the products' sums, as the vectors have nothing to do with each other."""
    B, L, V = 1, 140, 64
    d, do, dS = make(B, L, 1, 2, K, V, dtype, torch.float32, seed=40)
    rates = {10: 0.0, 11: 0.0, 12: 1e-7, 13: 1e-4, 63: 0.0, 64: 1e-7, 90: 1e-4, 139: 0.0}
    for t, x in rates.items():
        d["beta"][0, t] = x
    do = (do.float() * min(size, 1e4)).to(dtype)
    got, want = both(d, do, dS * size)
    step = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for n in want:
        a, w = got[n].double().cpu(), want[n]
        if got[n].dtype == torch.float16:
            inside = w.abs() < torch.finfo(torch.float16).max
            assert not bool(torch.isnan(a).any()), n
            a, w = torch.where(inside, a, 0.0), torch.where(inside, w, 0.0)
        assert bool(torch.isfinite(a).all()), n
        err = float((a - w).norm())
        assert err <= tol(got[n].dtype, dtype) * float(w.norm()) + step * a.numel() ** 0.5, (n, err / float(w.norm()))
    at = sorted(rates)
    a, w = got["dbeta"][0, at].double().cpu(), want["dbeta"][0, at]
    assert float((a - w).norm()) <= 2 * TOL * V ** 0.5 * float(w.norm()), (a, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 200, 1, 2, 64, 40), (1, 150, 2, 2, 128, 128), (1, 130, 16, 64, 128, 104)])
@pytest.mark.parametrize("rate,value,state,scale", [
    (1.0, 1.0, 1.0, 1.0), (1e-4, 1.0, 0.0, 1.0), (0.0, 1.0, 1e-3, 1e3), (1.0, 1e-3, 1e-3, 1e2), (1.0, 1.0, 1e6, 1e-6), (1e-20, 1.0, 0.0, 1e20),
    (1.0, 2e4, 1e9, 1e-9), (1e-30, 1.0, 1e-30, 1e30)])
def test_forward_without_gradients_of_any_size(dtype, shape, rate, value, state, scale):
    """Rates, values and states of very different sizes, with scales that bring the outputs near 1: the final state, which is
    float32, keeps TOL of every head's norm."""
    d, _, _ = make(*shape, dtype, torch.float32, seed=46)
    d["beta"] *= rate
    d["v"] = (d["v"].float() * value).clamp(-6e4, 6e4).to(dtype)  # (finite in float16)
    d["initial"] *= state
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    o, S = gated_delta_rule(*x, scale=scale, initial_state=d["initial"], output_final_state=True)
    want, S64 = oracle(*(t.double().cpu() for t in x), scale, d["initial"].double().cpu())
    assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(S).all())
    err, ref = (S.double().cpu() - S64).norm(dim=(2, 3)), S64.norm(dim=(2, 3))
    assert bool((err <= TOL * ref).all()), float((err / ref).max())
    err, ref = float((o.double().cpu() - want).norm()), float(want.norm())
    assert err <= tol(dtype) * ref + (2.0 ** -25 * o.numel() ** 0.5 if dtype == torch.float16 else 0.0), err / ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["off a boundary", "expanded", "aligned"])
def test_saved_tensors_that_come_back_in_another_layout(dtype, how):
    """Hooks that move what is saved give dense, aligned copies (or ones that are neither); the backward reads what the
    forward left all the same."""
    B, L, H, K, V = 2, 100, 2, 64, 64
    d, do, dS = make(B, L, H, H, K, V, dtype, seed=41)

    def run():
        leaves = {n: t.detach().clone().requires_grad_(True) for n, t in d.items()}
        x = dict(leaves)
        if how == "off a boundary":
            x["v"] = torch.nn.functional.pad(leaves["v"], (3, 5))[..., 3:3 + V]
        if how == "expanded":
            leaves["k"] = d["k"][:, :, :1].detach().clone().requires_grad_(True)
            x["k"] = leaves["k"].expand(B, L, H, K)
        o, S = gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)
        return o, S, list(leaves.values())

    def odd(t):  # one element off its old alignment
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        return flat.copy_(t.reshape(-1)).view(t.shape) if t.dtype == dtype else t
    o, S, leaves = run()
    want = torch.autograd.grad([o, S], leaves, [do, dS])
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(odd, lambda t: t)):
        with hooks:
            o, S, leaves = run()
        for a, b in zip(torch.autograd.grad([o, S], leaves, [do, dS]), want):
            assert torch.equal(a, b)


def test_forward_mode_and_traced_inputs_are_refused():
    from torch.autograd import forward_ad
    d, _, _ = make(1, 3, 1, 2, 16, 8, torch.bfloat16, seed=47)
    seq = [d[n] for n in ("q", "k", "v", "g", "beta")]
    tok, state = [t[:, 0] for t in seq], d["initial"]
    before = state.clone()
    with forward_ad.dual_level():
        for i in range(6):
            a = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate([*seq, state])]
            with pytest.raises(RuntimeError, match="forward-mode"):
                gated_delta_rule(*a[:5], initial_state=a[5])
            a = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate([*tok, state])]
            with pytest.raises(RuntimeError, match="forward-mode"):
                gated_delta_step(*a)
    with torch.no_grad(), pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda *a: gated_delta_rule(*a), seq)
    assert torch.equal(state, before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("training", [False, True])
@pytest.mark.parametrize("K,V", [(128, 128), (64, 40)])
def test_outputs_of_a_large_state_that_cancels(dtype, training, K, V):
    """A state whose columns sum to 0 under queries of equal elements: its operands' rounding (TOL of |q| |S|) shows, not
    the outputs'.  beta = 0 and g = 0 keep the state."""
    L = 130
    d, _, _ = make(1, L, 1, 2, K, V, dtype, torch.float32, seed=42)
    d["beta"].zero_()
    d["g"].zero_()
    d["q"] = (K ** -0.5 * (1 + 0.01 * d["q"].float())).to(dtype)
    S0 = 64 * (d["initial"] - d["initial"].mean(2, keepdim=True))
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    if training:
        x[2] = x[2].clone().requires_grad_(True)
    o, S = gated_delta_rule(*x, initial_state=S0, output_final_state=True)
    want, _ = oracle(*(t.detach().double().cpu() for t in x), K ** -0.5, S0.double().cpu())
    size = K ** -0.5 * L ** 0.5 * float(d["q"][0, 0].float().norm()) * float(S0.norm())
    err = float((o.detach().double().cpu() - want).norm())
    assert err <= TOL * size + torch.finfo(dtype).eps / 2 * float(want.norm()), err / size
    assert torch.equal(S.detach(), S0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 257, 2, 2, 128, 128), (1, 150, 1, 2, 64, 96), (1, 200, 2, 4, 128, 40)])
def test_float32_gradients_of_16_bit_tokens(dtype, shape):
    """The gradients of float32 gates and of the initial state are computed from operands of 16 bits or more, like the
    outputs: within TOL, whatever the tokens' type."""
    d, do, dS = make(*shape, dtype, torch.float32, seed=43)
    got, want = both(d, do, dS)
    for n in ("dg", "dbeta", "dinitial"):
        err, ref = float((got[n].double().cpu() - want[n]).norm()), float(want[n].norm())
        assert got[n].dtype == torch.float32 and err <= TOL * ref, (n, err / ref)


def test_lengths_and_resets_in_float16():
    test_lengths(torch.float16)
    test_resets_zero_and_double_rates(torch.float16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,V", [(64, 48), (128, 128)])
def test_lengths_and_resets_without_gradients(dtype, K, V):
    """The forward that keeps nothing: rows of any length with NaN and infinities behind them, resets, rates of 0 and 2."""
    lengths = [0, 1, 64, 100, 130, 500, -3]
    d, _, _ = make(len(lengths), 130, 1, 2, K, V, dtype, seed=48)
    d["g"][:, 20], d["g"][:, 100, 0], d["g"][:, 30:60] = float("-inf"), -60.0, 0.0
    d["beta"][:, 10:14], d["beta"][:, 50], d["beta"][:, 51] = 0.0, 2.0, -0.5
    dev = torch.tensor(lengths, dtype=torch.int32, device=DEV)

    def run():
        return gated_delta_rule(*(d[n] for n in ("q", "k", "v", "g", "beta")), initial_state=d["initial"], output_final_state=True,
                                lengths=dev)
    o, S = run()
    x = [d[n].double().cpu() for n in ("q", "k", "v", "g", "beta")]
    o64, S64 = oracle(*x, K ** -0.5, d["initial"].double().cpu(), dev.cpu())
    close(o, o64)
    close(S, S64)
    for i, n in enumerate(lengths):
        n = min(max(n, 0), 130)
        assert float(o[i, n:].abs().sum()) == 0.0
        if n == 0:
            assert torch.equal(S[i], d["initial"][i])
        for name in ("q", "k", "v", "g", "beta"):
            d[name][i, n:] = float("nan") if i % 2 else float("inf")
    again = run()
    assert torch.equal(o, again[0]) and torch.equal(S, again[1])


def test_without_gradients_on_another_stream_and_in_a_graph():
    d, _, _ = make(2, 200, 2, 4, 128, 128, torch.float16, seed=49)
    call = lambda: gated_delta_rule(*(d[n] for n in ("q", "k", "v", "g", "beta")), initial_state=d["initial"], output_final_state=True)
    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = call()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    del side
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call()
    d["v"].mul_(1e-4)
    d["initial"].mul_(1e5)
    want = call()
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.inference_mode():
        got = call()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "initial"])
def test_each_gradient_against_differences(name):
    """Each input by itself, f = <o, do> + <S, dS>, fourth-order differences of the kernel's forward along the input's own
    gradient, a tenth of the input's size.  float32 operands keep 22 bits and not 16, which leaves 2^-6 of TOL; with the
    float32 sums 2^-4.  A forward off by that much of |o| |do| + |S| |dS| moves the slope by 18 / 12 of it over h = 2^-4.
    Truncation is h^4 / 30 = 5e-7 of a fifth derivative, less than a tenth of that."""
    d, do, dS = make(1, 80, 1, 2, 64, 64, torch.float32, seed=44)

    def run(x):
        return gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)
    x = d[name].clone().requires_grad_(True)
    o, S = run({**d, name: x})
    grad = torch.autograd.grad([o, S], x, [do, dS])[0].double()
    way = (0.1 * d[name].double().norm() / grad.norm() * grad).float()

    def f(s):
        o, S = run({**d, name: d[name] + s * way})
        return float((o.double() * do.double()).sum() + (S.double() * dS.double()).sum())
    slope, h = float((grad * way.double()).sum()), 2.0 ** -4
    num = (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)
    size = float(o.detach().norm() * do.norm() + S.detach().norm() * dS.norm())
    allowed = 1.5 * TOL / 16 * size / h
    assert abs(num - slope) <= allowed and slope > 10 * allowed, (num, slope, allowed)


@pytest.mark.parametrize("shape", [(1, 130, 12, 24, 64, 200), (3, 130, 4, 16, 128, 128), (1, 130, 16, 64, 128, 104), (2, 193, 4, 32, 64, 128)])
def test_many_heads_in_float16(shape):
    d, do, dS = make(*shape, torch.float16, torch.float32, seed=sum(shape))
    lengths = torch.tensor([shape[1], 66, 1][:shape[0]], dtype=torch.int32)
    compare(*both(d, do, dS, lengths.to(DEV)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value,state,scale", [(1.0, 1.0, 1.0), (1e-3, 1e-3, 1e2), (1.0, 1e6, 1e-6), (1e4, 1e9, 1e-9), (1.0, 0.0, 1.0)])
def test_forward_with_and_without_gradients_has_the_same_bits(dtype, value, state, scale):
    d, _, _ = make(2, 200, 2, 4, 128, 72, dtype, torch.float32, seed=50)
    d["v"] = (d["v"].float() * value).clamp(-6e4, 6e4).to(dtype)
    d["initial"] *= state
    call = lambda q: gated_delta_rule(q, *(d[n] for n in ("k", "v", "g", "beta")), scale=scale, initial_state=d["initial"],
                                      output_final_state=True)
    for a, b in zip(call(d["q"].clone().requires_grad_(True)), call(d["q"])):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


@pytest.mark.parametrize("K,V", [(64, 64), (128, 48)])
def test_float16_gradients_of_groups_of_different_sizes(K, V):
    """Value columns (and so the tiles of a state) from 1e-4 to 1e4 of one another, forward and backward."""
    d, do, dS = make(1, 150, 1, 2, K, V, torch.float16, torch.float32, seed=51)
    sizes = torch.logspace(-2, 2, V, device=DEV)
    d["v"], d["initial"] = (d["v"].float() * sizes).half(), d["initial"] * sizes
    do, dS = (do.float() / sizes).half(), dS / sizes
    got, want = both(d, do, dS)
    compare(got, want)
    for n in ("S", "dinitial"):  # column by column
        err, ref = (got[n].double().cpu() - want[n]).norm(dim=2), want[n].norm(dim=2)
        assert bool((err <= TOL * ref).all()), (n, float((err / ref).max()))


def test_float16_backward_twice_streams_and_graphs():
    test_backward_twice_and_two_calls_at_once(torch.float16)
    d, do, dS = make(2, 200, 2, 4, 64, 64, torch.float16, seed=52)
    x = {n: t.detach().clone().requires_grad_(True) for n, t in d.items()}

    def step():
        o, S = gated_delta_rule(*(x[n] for n in ("q", "k", "v", "g", "beta")), initial_state=x["initial"], output_final_state=True)
        return (o.detach(), S.detach(), *torch.autograd.grad([o, S], list(x.values()), [do, dS]))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    with torch.no_grad():
        x["v"].mul_(0.01)
        do.mul_(0.01)
    want = step()
    for gr, _ in graphs:
        gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
