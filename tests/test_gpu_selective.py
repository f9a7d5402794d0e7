"""The selective state space scan (eacs_selective_*) against its formulas in 64 bits, token by token.

Tolerances are element by element, against `mag`: the same sums with every term's absolute value.  A decay
e^(s A) = 2^(s log2(e) A) is off by 2^-22 of itself (the hardware's exponential) and by the rounding of its argument
(at most 2^-22 for |s A| <= 4; a decay below e^-4 is that much smaller), a step by 2^-20 (softplus: an exponential, a
quotient, a series), and a term that is carried over n tokens collects n of them: a sum whose terms are carried over at
most L tokens is off by (L 2^-21 + 2^-18) mag, with the sums' own roundings.  Outputs are rounded once: half a step of
their type, eps / 2 of the value (float16: at least half of its smallest step, 2^-25).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200 import _lib
    from eacs_b200.ops.selective_ssm import selective_ssm, selective_ssm_step

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAMES = ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias")


def oracle(i, dy=None, dfinal=None, magnitudes=False):
    """Outputs and gradients in 64 bits; with `magnitudes` of the terms' absolute values."""
    f = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    d = lambda t: None if t is None else t.detach().double()
    x, B, C = f(d(i["x"])), f(d(i["B"])), f(d(i["C"]))
    A, dt = d(i["A"]), d(i["dt"])
    b, L, D = x.shape
    raw = dt + (0 if i["dt_bias"] is None else d(i["dt_bias"]))
    step = torch.nn.functional.softplus(raw, threshold=40) if i["softplus"] else raw  # (log1p(e^-40) is 2^-62 of 40)
    slope = torch.sigmoid(raw) if i["softplus"] else torch.ones_like(raw)
    len_ = torch.full((b,), L, device=x.device) if i["lengths"] is None else i["lengths"].long().clamp(0, L)
    live = (torch.arange(L, device=x.device) < len_[:, None])[..., None]
    nil = torch.zeros_like(x)
    step, x = torch.where(live, step, nil), torch.where(live, x, nil)
    B, C = torch.where(live, B, torch.zeros_like(B)), torch.where(live, C, torch.zeros_like(C))
    skip = torch.zeros(D, device=x.device, dtype=torch.float64) if i["skip"] is None else f(d(i["skip"]))
    h = torch.zeros(b, D, A.shape[1], device=x.device, dtype=torch.float64) if i["initial"] is None else f(d(i["initial"]))
    a = torch.exp(step[..., None] * A)
    olds, hs = [], []
    for t in range(L):
        olds.append(a[:, t] * h)
        h = olds[-1] + (step[:, t] * x[:, t])[..., None] * B[:, t, None]
        hs.append(h)
    hs, olds = torch.stack(hs, 1), torch.stack(olds, 1)
    o = (hs * C[:, :, None]).sum(-1) + skip * x
    z = d(i["z"])
    gain = torch.ones_like(x) if z is None else torch.nn.functional.silu(z)
    out = {"y": torch.where(live, o * f(gain), nil), "final": h}
    if dy is None:
        return out
    g0 = torch.where(live, f(dy.double()), nil)
    do = g0 * f(gain)
    g = torch.zeros_like(h) if dfinal is None else f(dfinal.double())
    gs = [None] * L
    for t in reversed(range(L)):
        gs[t] = g + do[:, t, :, None] * C[:, t, None]
        g = a[:, t] * gs[t]
    gs = torch.stack(gs, 1)
    w = gs * olds
    dv = (gs * B[:, :, None]).sum(-1)
    ds = (w * f(A)).sum(-1) + x * dv
    ddt = torch.where(live, ds * slope, nil)
    out.update(dx=torch.where(live, step * dv + skip * do, nil), ddt=ddt, dA=(w * step[..., None]).sum((0, 1)),
               dB=(gs * (step * x)[..., None]).sum(2), dC=(hs * do[..., None]).sum(2), dskip=(do * x).sum((0, 1)),
               ddt_bias=ddt.sum((0, 1)), dinitial=g)
    if z is not None:
        s = torch.sigmoid(z)
        # silu' is a sum of two terms of opposite signs for z < 0: with each off by 2^-24 of itself, it is off by that much
        # of s + |z| s (1 - s), however close to its zero at z = -1.28 it is
        out["dz"] = g0 * o * (s + f(z) * s * (1 - s))
    return out


def inputs(b, L, D, N, dtype, seed=0, gate=True, ragged=False, initial=False, skip=True, bias=True, softplus=True):
    g = torch.Generator(DEV).manual_seed(seed * 1009 + b * 7 + L * 13 + D * 17 + N)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    i = {"x": rnd(b, L, D).to(dtype), "B": rnd(b, L, N).to(dtype), "C": rnd(b, L, N).to(dtype),
         "A": -(1 + torch.arange(N, device=DEV)).float() * torch.exp(0.1 * rnd(D, N)) / N * 8,
         "z": rnd(b, L, D).to(dtype) if gate else None, "skip": rnd(D) if skip else None, "softplus": softplus,
         "dt_bias": -3 + rnd(D) if bias else None, "lengths": None, "initial": rnd(b, D, N) if initial else None}
    i["dt"] = (rnd(b, L, D) if softplus else 0.3 * torch.rand(b, L, D, generator=g, device=DEV)).to(dtype)
    if not softplus and bias:
        i["dt_bias"] = 0.1 * torch.rand(D, generator=g, device=DEV)
    if ragged:
        i["lengths"] = torch.randint(0, L + 1, (b,), generator=g, device=DEV).int()
        i["lengths"][0] = L
        if b > 1:
            i["lengths"][1] = 0
    return i, rnd


def call(i, **kw):
    return selective_ssm(i["x"], i["dt"], i["A"], i["B"], i["C"], i["skip"], i["z"], i["dt_bias"], softplus=i["softplus"],
                         initial_state=i["initial"], lengths=i["lengths"], **kw)


def close(name, got, want, mag, L, dtype):
    assert got.dtype == dtype and got.shape == want.shape, name
    assert bool(torch.isfinite(got).all()), name
    tol = (L * 2.0 ** -21 + 2.0 ** -18) * mag + 1e-30
    if dtype != F32:
        tol = tol + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == F16 else 0.0)
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0 if over.numel() else True, (name, float(over.max()), int(over.argmax()))


def check(i, L, dy=None, dfinal=None, leaves=()):
    """Forward (and backward) of i against the oracle; returns what the kernels gave."""
    for n in leaves:
        i[n] = i[n].detach().requires_grad_(True) if i[n] is not None else None
    y, final = call(i, output_final_state=True)
    want, mag = oracle(i, dy, dfinal), oracle(i, dy, dfinal, True)
    close("y", y.detach(), want["y"], mag["y"], L, i["x"].dtype)
    close("final", final.detach(), want["final"], mag["final"], L, F32)
    if dy is None:
        return y, final
    names = [n for n in leaves if i[n] is not None]
    outs, ups = ([y, final], [dy, dfinal]) if dfinal is not None else ([y], [dy])
    grads = torch.autograd.grad(outs, [i[n] for n in names], ups, retain_graph=True)
    for n, t in zip(names, grads):
        close("d" + n, t, want["d" + n], mag["d" + n], L, i[n].dtype)
    for t, u in zip(grads, torch.autograd.grad(outs, [i[n] for n in names], ups)):  # the same bits again
        assert torch.equal(t, u)
    return y, final, dict(zip(names, grads))


SIZES = [(1, 1, 1, 1), (2, 3, 5, 4), (3, 16, 8, 16), (2, 17, 33, 16), (1, 64, 64, 8), (2, 65, 24, 12), (1, 129, 100, 32),
         (2, 100, 12, 24), (2, 40, 20, 64), (1, 33, 7, 33), (3, 200, 72, 16), (1, 9, 520, 16)]


@pytest.mark.parametrize("b,L,D,N", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_forward(b, L, D, N, dtype):
    for k, kw in enumerate([dict(), dict(gate=False, ragged=True, initial=True), dict(skip=False, bias=False, softplus=False, initial=True)]):
        i, _ = inputs(b, L, D, N, dtype, k, **kw)
        check(i, L)


@pytest.mark.parametrize("b,L,D,N", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients(b, L, D, N, dtype):
    for k, kw in enumerate([dict(), dict(gate=False, ragged=True, initial=True, bias=False), dict(ragged=True, skip=False, softplus=False)]):
        i, rnd = inputs(b, L, D, N, dtype, 10 + k, **kw)
        check(i, L, rnd(b, L, D).to(dtype), rnd(b, D, N) if k == 1 else None, NAMES + ("initial",))


@pytest.mark.parametrize("b,D,N,dtype", [(1, 1, 1, F32), (3, 40, 16, BF16), (2, 33, 12, F16), (5, 70, 64, F32), (4, 17, 7, BF16),
                                         (300, 512, 16, BF16), (9, 8, 32, F16)])
def test_step(b, D, N, dtype):
    for kw in (dict(), dict(gate=False, softplus=False), dict(skip=False, bias=False)):
        i, _ = inputs(b, 1, D, N, dtype, 3, initial=True, **kw)
        want, mag = oracle(i), oracle(i, magnitudes=True)
        state = i["initial"].clone()
        one = {n: i[n][:, 0] if n in ("x", "dt", "B", "C", "z") and i[n] is not None else i[n] for n in NAMES}
        y = selective_ssm_step(one["x"], one["dt"], i["A"], one["B"], one["C"], state, i["skip"], one["z"], i["dt_bias"],
                               softplus=i["softplus"])
        close("y", y[:, None], want["y"], mag["y"], 1, dtype)
        close("state", state, want["final"], mag["final"], 1, F32)


def test_sequence_in_parts_and_by_steps():
    i, _ = inputs(2, 50, 40, 16, F32, 5)
    y, final = call(i, output_final_state=True)
    part = lambda lo, hi: {n: t[:, lo:hi] if n in ("x", "dt", "B", "C", "z") else t for n, t in i.items()}
    y0, s0 = call(part(0, 23), output_final_state=True)
    y1, s1 = call({**part(23, 50), "initial": s0}, output_final_state=True)
    state = torch.zeros(2, 40, 16, device=DEV)
    ys = [selective_ssm_step(*(i[n][:, t] if n in ("x", "dt", "B", "C") else i[n] for n in ("x", "dt", "A", "B", "C")), state,
                             i["skip"], i["z"][:, t], i["dt_bias"]) for t in range(50)]
    mag = oracle(i, magnitudes=True)
    for got in (torch.cat([y0, y1], 1), torch.stack(ys, 1)):
        close("y", got, y.double(), 2 * mag["y"], 50, F32)
    for got in (s1, state):
        close("state", got, final.double(), 2 * mag["final"], 50, F32)


def test_gradient_against_differences():
    i, rnd = inputs(2, 21, 9, 5, F32, 6, initial=True, ragged=True)
    dy, dfinal = rnd(2, 21, 9), rnd(2, 9, 5)
    names = [n for n in NAMES] + ["initial"]
    _, _, grads = check(i, 21, dy, dfinal, names)
    for n in names:  # every gradient by itself
        v = rnd(*i[n].shape)
        v = v / v.abs().max() * (0.05 if n in ("A", "dt_bias") else 1.0)
        h = 2.0 ** -4

        def f(s):
            w = oracle({**i, n: i[n].detach().double() + s * h * v.double()})
            return float((w["y"] * dy.double()).sum() + (w["final"] * dfinal.double()).sum())
        diff = (8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * h)  # of a 64-bit function: off by h^4 times its fifth derivative
        slope = float((grads[n].double() * v.double()).sum())
        size = float((grads[n].double() * v.double()).abs().sum()) + 1.0
        assert abs(diff - slope) <= 2e-4 * size, (n, diff, slope)


def test_masked_places_are_not_read_and_causality():
    i, rnd = inputs(3, 70, 40, 16, BF16, 7, ragged=True)
    y, final = call(i, output_final_state=True)
    j = dict(i)
    for n in ("x", "dt", "B", "C", "z"):
        j[n] = i[n].clone()
        for b in range(3):
            j[n][b, int(i["lengths"][b]):] = float("nan")
    leaves = ("x", "dt", "B", "C", "z", "A")
    for n in leaves:
        j[n] = j[n].detach().requires_grad_(True)
    y2, final2 = call(j, output_final_state=True)
    assert torch.equal(y2, y) and torch.equal(final2, final)
    dy = torch.full_like(y, float("nan"))
    for b in range(3):
        dy[b, :int(i["lengths"][b])] = 1
    for t in torch.autograd.grad(y2, [j[n] for n in leaves], dy):
        assert bool(torch.isfinite(t).all())
    for n in ("x", "dt", "B", "C", "z"):  # a NaN stays in its row and reaches no token before it
        j = {**i, "lengths": None, n: i[n].clone()}
        j[n][1, 37, 3] = float("nan")
        clean = call({**i, "lengths": None})
        got = call(j)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2]) and torch.equal(got[1, :37], clean[1, :37])
        assert bool(torch.isnan(got[1, 37]).any())


def test_lengths_outside_the_range():
    i, _ = inputs(3, 20, 16, 16, F32, 8)
    full = call(i)
    got, state = call({**i, "lengths": torch.tensor([-5, 99, 20], device=DEV, dtype=torch.int32)}, output_final_state=True)
    assert float(got[0].abs().max()) == 0 and float(state[0].abs().max()) == 0 and torch.equal(got[1:], full[1:])


def test_extreme_steps():
    """Steps of 0 and of thousands, decays that underflow, a softplus far to either side."""
    i, _ = inputs(2, 40, 16, 16, F32, 9, bias=False)
    i["dt"] = torch.linspace(-120, 3000, 2 * 40 * 16, device=DEV).reshape(2, 40, 16)[:, torch.randperm(40)].contiguous()
    y, final = call(i, output_final_state=True)
    want, mag = oracle(i), oracle(i, magnitudes=True)
    assert bool(torch.isfinite(y).all())
    # a step of 3000 has a decay's argument of 24000, whose rounding is 2^-24 of it: no decay of that size is left
    close("y", y, want["y"], mag["y"], 40, F32)
    i["A"] = torch.zeros_like(i["A"])  # nothing decays: a running sum
    close("y", call(i), oracle(i)["y"], oracle(i, magnitudes=True)["y"], 40, F32)


def test_views_broadcast_and_shared_inputs():
    g = torch.Generator(DEV).manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    base, _ = inputs(2, 37, 48, 16, BF16, 12)
    big, small = rnd(2, 37, 48 * 3 + 5).bfloat16(), rnd(2, 37, 16 * 2 + 3).bfloat16()
    for off in (0, 1, 8):  # slices of wider projections, on 16 bytes and off them
        i = {**base, "x": big[..., off:off + 48], "z": big[..., 48 + off:96 + off], "B": small[..., off % 3:16 + off % 3],
             "C": small[..., 16:32]}
        y = call(i)
        assert torch.equal(y, call({**i, **{n: i[n].contiguous() for n in ("x", "z", "B", "C")}}))
        check(i, 37, rnd(2, 37, 48).bfloat16(), None, ("x", "z", "B", "C", "dt"))
    i = {**base, "x": rnd(2, 48, 37).bfloat16().transpose(1, 2), "lengths": None}  # a last dimension that is not dense
    check(i, 37, rnd(2, 37, 48).bfloat16(), None, ("x",))
    # one row's B and C for all rows, one token's x for all tokens: gradients are summed
    one = rnd(1, 37, 16).requires_grad_(True)
    tok = rnd(2, 1, 48).requires_grad_(True)
    i = {**inputs(2, 37, 48, 16, F32, 13)[0], "B": one.expand(2, 37, 16), "C": one.expand(2, 37, 16), "x": tok.expand(2, 37, 48)}
    dy = rnd(2, 37, 48)
    got = torch.autograd.grad(call(i), (one, tok), dy)
    want, mag = oracle(i, dy), oracle(i, dy, magnitudes=True)
    close("one", got[0], (want["dB"] + want["dC"]).sum(0, keepdim=True), (mag["dB"] + mag["dC"]).sum(0, keepdim=True), 37, F32)
    close("tok", got[1], want["dx"].sum(1, keepdim=True), mag["dx"].sum(1, keepdim=True), 37, F32)
    dy1 = rnd(48).expand(2, 37, 48)  # an upstream gradient with strides of 0
    got = torch.autograd.grad(call(i), tok, dy1)[0]
    close("tok", got, oracle(i, dy1)["dx"].sum(1, keepdim=True), oracle(i, dy1, magnitudes=True)["dx"].sum(1, keepdim=True), 37, F32)


def test_needed_gradients_only_and_final_state_alone():
    i, rnd = inputs(2, 30, 20, 16, F32, 14, initial=True)
    for n in ("dt", "initial", "A"):
        j = {**i, n: i[n].clone().requires_grad_(True)}
        y, final = call(j, output_final_state=True)
        dfinal = rnd(2, 20, 16)
        got = torch.autograd.grad(final, j[n], dfinal)[0]
        zero = torch.zeros_like(y)
        close(n, got, oracle(j, zero, dfinal)["d" + n], oracle(j, zero, dfinal, True)["d" + n], 30, F32)


def test_empty():
    i, _ = inputs(2, 4, 8, 16, F32, 15, initial=True)
    cut = {**i, **{n: i[n][:, :0] for n in ("x", "dt", "B", "C", "z")}}
    cut["A"] = i["A"].clone().requires_grad_(True)
    cut["initial"] = i["initial"].clone().requires_grad_(True)
    y, final = call(cut, output_final_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(final, i["initial"])
    dA, di = torch.autograd.grad((y.sum() + (final * 2).sum()), (cut["A"], cut["initial"]))
    assert float(dA.abs().max()) == 0 and torch.equal(di, torch.full_like(di, 2))
    none = {**i, **{n: i[n][:0] for n in ("x", "dt", "B", "C", "z", "initial")}}
    y, final = call(none, output_final_state=True)
    assert y.shape == (0, 4, 8) and final.shape == (0, 8, 16)
    y = selective_ssm_step(none["x"][:, 0], none["dt"][:, 0], i["A"], none["B"][:, 0], none["C"][:, 0], none["initial"].clone())
    assert y.shape == (0, 8)


def test_long_rows_and_many_channels():
    """Longer than what a ring of warps holds, with more channels than a round of CTAs: parts against parts."""
    i, rnd = inputs(2, 3000, 1200, 16, BF16, 16, ragged=True)
    i["lengths"] = torch.tensor([3000, 1777], device=DEV, dtype=torch.int32)
    dy = rnd(2, 3000, 1200).bfloat16()
    leaves = ("x", "dt", "B", "C", "z", "A", "skip", "dt_bias")
    for n in leaves:
        i[n] = i[n].detach().requires_grad_(True)
    y = call(i)
    g = dict(zip(leaves, torch.autograd.grad(y, [i[n] for n in leaves], dy)))
    sub = [0, 7, 640, 1199]  # channels do not meet but in dB and dC
    cut = lambda t: t[..., sub]
    j = {**i, **{n: cut(i[n]) for n in ("x", "dt", "z", "skip", "dt_bias")}, "A": i["A"][sub]}
    want, mag = oracle(j, cut(dy)), oracle(j, cut(dy), magnitudes=True)
    close("y", cut(y.detach()), want["y"], mag["y"], 3000, BF16)
    for n in ("x", "dt", "z", "skip", "dt_bias"):
        close(n, cut(g[n]), want["d" + n], mag["d" + n], 3000, i[n].dtype)
    close("A", g["A"][sub], want["dA"], mag["dA"], 3000, F32)
    assert float(g["B"][1, 1777:].abs().max()) == 0 and float(g["x"][1, 1777:].abs().max()) == 0
    assert _lib.device_status() == 0


def test_streams_graphs_and_two_calls_at_once():
    i, rnd = inputs(2, 90, 64, 16, BF16, 17)
    want = call(i)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for st in s:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs += [call(i) for _ in range(3)]
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    leaves = [i[n].detach().requires_grad_(True) for n in ("x", "dt", "B", "C")]
    dy = rnd(2, 90, 64).bfloat16()

    def step():
        y = call({**i, **dict(zip(("x", "dt", "B", "C"), leaves))})
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for t in got:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    for t, u in zip(got, eager):
        assert torch.equal(t, u)


def test_refusals():
    i, _ = inputs(2, 6, 8, 16, F32, 18)
    args = [i[n] for n in ("x", "dt", "A", "B", "C")]
    state = torch.zeros(2, 8, 16, device=DEV)

    def bad(match, **kw):
        a = dict(zip(("x", "dt", "A", "B", "C"), args)) | kw
        with pytest.raises(RuntimeError, match=match):
            selective_ssm(**a)
    bad("one dtype", dt=args[1].half())
    bad("one shape", dt=args[1][:, :5])
    bad("one shape", z=args[0][..., :4])
    bad("A must be", A=args[2].half())
    bad("A must be", A=args[2][:4])
    bad("N=65", A=torch.zeros(8, 65, device=DEV))
    bad("B and C", C=args[4][..., :8])
    bad("skip and dt_bias", skip=torch.zeros(8, device=DEV, dtype=F16))
    bad("skip and dt_bias", dt_bias=torch.zeros(4, device=DEV))
    bad("lengths", lengths=torch.zeros(2, device=DEV, dtype=torch.int64))
    bad("the state", initial_state=state[:1])
    bad("CUDA", dt=args[1].cpu())
    bad("one dtype", x=args[0].double(), dt=args[1].double(), B=args[3].double(), C=args[4].double())
    one = [t[:, 0] if t.dim() == 3 else t for t in args]
    with pytest.raises(RuntimeError, match="no gradient"):
        selective_ssm_step(one[0].clone().requires_grad_(True), *one[1:], state)
    with pytest.raises(RuntimeError, match="in place"):
        selective_ssm_step(*one, torch.zeros(2, 16, 8, device=DEV).transpose(1, 2))
    v = state._version
    selective_ssm_step(*one, state)
    assert state._version > v
    y = selective_ssm(args[0].clone().requires_grad_(True), *args[1:])
    gx = torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    import torch.autograd.forward_ad as fwd_ad
    with fwd_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        selective_ssm(fwd_ad.make_dual(args[0], torch.ones_like(args[0])), *args[1:])
