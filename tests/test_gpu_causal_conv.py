"""The short causal convolution (eacs_conv_*) against its formulas in 64 bits.

Tolerances are element by element, against `mag`, the same sums with every term's absolute value.  A sum of at most 4 + 1
terms in float32, a sigmoid (the hardware's exponential, 2^-22, whose argument is off by 2^-23 |p| <= 2^-19, and a quotient,
2^-22) and their products are off by at most 2^-18 of it; sums over tokens (each in runs, then over runs) by 2^-14 in all.
Outputs are rounded once: half a step of their type (float16: at least 2^-25).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200.ops.causal_conv import causal_conv, causal_conv_step

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def oracle(i, dy=None, dfinal=None, magnitudes=False):
    f = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    d = lambda t: None if t is None else t.detach().double()
    x, w, bias = d(i["x"]), d(i["weight"]), d(i["bias"])
    b, L, D = x.shape
    W = w.shape[1]
    n = torch.full((b,), L, device=x.device) if i["lengths"] is None else i["lengths"].long().clamp(0, L)
    live = (torch.arange(L, device=x.device) < n[:, None])[..., None]
    x = torch.where(live, x, torch.zeros_like(x))
    h0 = torch.zeros(b, W - 1, D, device=x.device, dtype=torch.float64) if i["initial"] is None else d(i["initial"])
    row = torch.cat([h0, x], 1)

    def conv(g):
        return sum(g(row)[:, k:k + L] * g(w)[:, k] for k in range(W)) + (0 if bias is None else g(bias))
    p, same = conv(lambda t: t), lambda t: t
    pm = conv(f)
    s = torch.sigmoid(p) if i["activation"] else torch.ones_like(p)
    last = torch.stack([row[r, int(n[r]):int(n[r]) + W - 1] for r in range(b)]) if b else h0
    out = {"y": torch.where(live, pm * s, torch.zeros_like(p)), "final": last}
    if dy is None:
        return out
    slope = s + f(p) * s * (1 - s) if i["activation"] else s  # (two terms that cancel near p = -1.28)
    if magnitudes and i["activation"]:
        slope = slope + pm * 2  # an error of p moves silu' by at most half of it, of the terms' sum pm at most
    dp = torch.where(live, f(dy.double()) * slope, torch.zeros_like(p))
    g = torch.zeros_like(row)
    dw = torch.empty_like(w)
    for k in range(W):
        g[:, k:k + L] += f(w)[:, k] * dp
        dw[:, k] = (dp * f(row)[:, k:k + L]).sum((0, 1))
    if dfinal is not None:
        for r in range(b):
            g[r, int(n[r]):int(n[r]) + W - 1] += f(dfinal[r].double())
    dx = torch.where(live, g[:, W - 1:], torch.zeros_like(x))
    out.update(dx=dx, dweight=dw, dbias=dp.sum((0, 1)), dinitial=g[:, :W - 1])
    return out


def inputs(b, L, D, W, dtype, wdtype, seed=0, bias=True, ragged=False, initial=False, activation="silu"):
    g = torch.Generator(DEV).manual_seed(seed * 1009 + b * 7 + L * 13 + D * 17 + W)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    i = {"x": rnd(b, L, D).to(dtype), "weight": rnd(D, W).to(wdtype), "bias": rnd(D).to(wdtype) if bias else None,
         "initial": rnd(b, W - 1, D).to(dtype) if initial else None, "lengths": None, "activation": activation}
    if ragged:
        i["lengths"] = torch.randint(0, L + 1, (b,), generator=g, device=DEV).int()
        i["lengths"][0] = L
        if b > 1:
            i["lengths"][1] = 0
        if b > 2:
            i["lengths"][2] = min(1, L)
    return i, rnd


def call(i, **kw):
    return causal_conv(i["x"], i["weight"], i["bias"], i["activation"], initial_state=i["initial"], lengths=i["lengths"], **kw)


def close(name, got, want, mag, dtype, sums=False):
    assert got.dtype == dtype and got.shape == want.shape, name
    assert bool(torch.isfinite(got).all()), name
    tol = 2.0 ** (-14 if sums else -18) * mag + 1e-30
    if dtype != F32:
        tol = tol + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == F16 else 0.0)
    over = (got.double() - want).abs() - tol
    assert over.numel() == 0 or float(over.max()) <= 0, (name, float(over.max()), int(over.argmax()))


def check(i, dy=None, dfinal=None, leaves=("x", "weight", "bias", "initial")):
    if dy is not None:
        for n in leaves:
            i[n] = None if i[n] is None else i[n].detach().requires_grad_(True)
    y, final = call(i, output_final_state=True)
    want, mag = oracle(i, dy, dfinal), oracle(i, dy, dfinal, True)
    close("y", y.detach(), want["y"], mag["y"], i["x"].dtype)
    assert torch.equal(final.detach().double(), want["final"])
    if dy is None:
        return
    names = [n for n in leaves if i[n] is not None]
    outs, ups = ([y, final], [dy, dfinal]) if dfinal is not None else ([y], [dy])
    grads = torch.autograd.grad(outs, [i[n] for n in names], ups, retain_graph=True)
    for n, t in zip(names, grads):
        close("d" + n, t, want["d" + n], mag["d" + n], i[n].dtype, n in ("weight", "bias"))
    for t, u in zip(grads, torch.autograd.grad(outs, [i[n] for n in names], ups)):
        assert torch.equal(t, u)


SIZES = [(1, 1, 1, 2), (2, 2, 3, 4), (3, 5, 8, 3), (3, 40, 33, 4), (2, 65, 64, 4), (1, 300, 130, 2), (4, 97, 1024, 4), (5, 1, 16, 3),
         (2, 1000, 24, 4)]


@pytest.mark.parametrize("b,L,D,W", SIZES)
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
def test_forward_and_gradients(b, L, D, W, dtype, wdtype):
    for k, kw in enumerate([dict(), dict(ragged=True, initial=True), dict(bias=False, activation=None, initial=True)]):
        i, rnd = inputs(b, L, D, W, dtype, wdtype, k, **kw)
        check(i)
        check(i, rnd(b, L, D).to(dtype), rnd(b, W - 1, D).to(dtype) if k else None)


@pytest.mark.parametrize("L,D,W", [(70, 50, 4), (40, 98, 3), (300, 6, 4), (33, 202, 2), (9, 2, 4)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_even_rows_and_offsets(L, D, W, dtype):
    i, rnd = inputs(3, L, D, W, dtype, F32, 7, ragged=True, initial=True)  # rows aligned to pairs of channels only
    check(i, rnd(3, L, D).to(dtype), rnd(3, W - 1, D).to(dtype))
    wide = rnd(3, L, 2 * D + 6).to(dtype)
    for at in (2, 1, 4, D + 6):  # aligned to pairs, and not
        check({**i, "x": wide[..., at:at + D]}, wide.flip(1)[..., at:at + D])


@pytest.mark.parametrize("b,D,W,dtype", [(1, 1, 2, F32), (3, 40, 4, BF16), (2, 33, 3, F16), (300, 512, 4, BF16), (2, 6, 4, F32)])
def test_step(b, D, W, dtype):
    for kw in (dict(), dict(bias=False, activation=None)):
        i, _ = inputs(b, 1, D, W, dtype, dtype, 3, initial=True, **kw)
        want, mag, state = oracle(i), oracle(i, magnitudes=True), i["initial"].clone()
        y = causal_conv_step(i["x"][:, 0], i["weight"], i["bias"], state, i["activation"])
        close("y", y[:, None], want["y"], mag["y"], dtype)
        assert torch.equal(state.double(), want["final"])


def test_sequence_in_parts_and_by_steps():
    i, _ = inputs(2, 50, 40, 4, BF16, F32, 5)
    y, final = call(i, output_final_state=True)
    cut = lambda lo, hi: {**i, "x": i["x"][:, lo:hi]}
    y0, s0 = call(cut(0, 2), output_final_state=True)  # shorter than the state
    y1, s1 = call({**cut(2, 23), "initial": s0}, output_final_state=True)
    y2, s2 = call({**cut(23, 50), "initial": s1}, output_final_state=True)
    state = torch.zeros(2, 3, 40, device=DEV, dtype=BF16)
    ys = [causal_conv_step(i["x"][:, t], i["weight"], i["bias"], state) for t in range(50)]
    assert torch.equal(torch.cat([y0, y1, y2], 1), y) and torch.equal(s2, final)
    assert torch.equal(torch.stack(ys, 1), y) and torch.equal(state, final)


def test_gradient_against_differences():
    i, rnd = inputs(3, 21, 9, 4, F32, F32, 6, initial=True, ragged=True)
    dy, dfinal = rnd(3, 21, 9), rnd(3, 3, 9)
    for n in ("x", "weight", "bias", "initial"):
        j = {**i, n: i[n].clone().requires_grad_(True)}
        y, final = call(j, output_final_state=True)
        g = torch.autograd.grad((y, final), j[n], (dy, dfinal), allow_unused=True)[0]
        v, h = rnd(*i[n].shape), 2.0 ** -6

        def f(s):
            w = oracle({**i, n: i[n].double() + s * h * v.double()})
            return float((w["y"] * dy.double()).sum() + (w["final"] * dfinal.double()).sum())
        diff = (8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * h)  # off by h^4 = 6e-8 times fifth derivatives
        terms = g.double() * v.double()
        assert abs(diff - float(terms.sum())) <= 1e-4 * (float(terms.abs().sum()) + 1), n


def test_masked_places_are_not_read_and_causality():
    i, rnd = inputs(3, 70, 40, 4, BF16, F32, 7)
    i["lengths"] = torch.tensor([70, 0, 33], device=DEV, dtype=torch.int32)
    y, final = call(i, output_final_state=True)
    x = i["x"].clone()
    for b in range(3):
        x[b, int(i["lengths"][b]):] = float("nan")
    j = {**i, "x": x.requires_grad_(True), "weight": i["weight"].clone().requires_grad_(True)}
    y2, final2 = call(j, output_final_state=True)
    assert torch.equal(y2, y) and torch.equal(final2, final)
    dy = torch.full_like(y, float("nan"))
    for b in range(3):
        dy[b, :int(i["lengths"][b])] = 1
    for t in torch.autograd.grad(y2, (j["x"], j["weight"]), dy):
        assert bool(torch.isfinite(t).all())
    x = i["x"].clone()
    x[0, 20, 3] = float("inf")  # reaches its channel of the next three tokens, nothing else
    got = call({**i, "x": x})
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[0, 20:24, 3] = False
    assert torch.equal(got[keep], y[keep]) and not bool(torch.isfinite(got[0, 20, 3]))
    full, _ = call({**i, "lengths": torch.tensor([99, -3, 33], device=DEV, dtype=torch.int32)}, output_final_state=True)
    assert torch.equal(full, y)


def test_views_broadcast_streams_and_graphs():
    g = torch.Generator(DEV).manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    base, _ = inputs(2, 37, 48, 4, BF16, BF16, 12)
    big = rnd(2, 37, 48 * 2 + 13).bfloat16()
    for off in (0, 1, 4, 8):
        i = {**base, "x": big[..., off:off + 48]}
        assert torch.equal(call(i), call({**i, "x": i["x"].contiguous()}))
        check(i, rnd(2, 37, 48).bfloat16(), None, ("x", "weight"))
    check({**base, "x": rnd(2, 48, 37).bfloat16().transpose(1, 2)}, rnd(2, 48, 37).bfloat16().transpose(1, 2), None, ("x", "weight"))
    tok = rnd(1, 1, 48).requires_grad_(True)  # one token for all, and an upstream gradient with strides of 0
    i = {**inputs(2, 37, 48, 4, F32, F32, 13)[0], "x": tok.expand(2, 37, 48)}
    dy = rnd(48).expand(2, 37, 48)
    got = torch.autograd.grad(call(i), tok, dy)[0]
    close("tok", got, oracle(i, dy)["dx"].sum((0, 1), keepdim=True), oracle(i, dy, magnitudes=True)["dx"].sum((0, 1), keepdim=True), F32)
    want, outs = call(base), []
    for st in (torch.cuda.Stream(), torch.cuda.Stream()):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs += [call(base) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    leaves = [base["x"].detach().requires_grad_(True), base["weight"].detach().requires_grad_(True)]

    def step():
        y = causal_conv(leaves[0], leaves[1], base["bias"])
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]
    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t, u) for t, u in zip(got, eager))


def test_empty():
    i, _ = inputs(2, 4, 8, 4, F32, F32, 15, initial=True)
    cut = {**i, "x": i["x"][:, :0], "weight": i["weight"].clone().requires_grad_(True), "initial": i["initial"].clone().requires_grad_(True)}
    y, final = call(cut, output_final_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(final, i["initial"])
    dw, di = torch.autograd.grad((y.sum() + (final * 2).sum()), (cut["weight"], cut["initial"]))
    assert float(dw.abs().max()) == 0 and torch.equal(di, torch.full_like(di, 2))
    y, final = call({**i, "x": i["x"][:0], "initial": i["initial"][:0]}, output_final_state=True)
    assert y.shape == (0, 4, 8) and final.shape == (0, 3, 8)
    assert causal_conv_step(i["x"][:0, 0], i["weight"], i["bias"], i["initial"][:0].clone()).shape == (0, 8)


def test_refusals():
    i, _ = inputs(2, 6, 8, 4, F32, F32, 18)
    x, w, b = i["x"], i["weight"], i["bias"]
    for match, args, kw in (("x must be", (x.double(), w), {}), ("x must be", (x[0], w), {}), ("weight must be", (x, w[:4]), {}),
                            ("W=1", (x, w[:, :1]), {}), ("W=5", (x, torch.zeros(8, 5, device=DEV)), {}),
                            ("bias must be", (x, w, b.half()), {}), ("bias must be", (x, w, b[:3]), {}),
                            ("activation", (x, w, b, "relu"), {}), ("lengths", (x, w), dict(lengths=torch.zeros(2, device=DEV))),
                            ("the state", (x, w), dict(initial_state=x[:, :2])), ("CUDA", (x, w.cpu()), {})):
        with pytest.raises(RuntimeError, match=match):
            causal_conv(*args, **kw)
    state = torch.zeros(2, 3, 8, device=DEV)
    with pytest.raises(RuntimeError, match="no gradient"):
        causal_conv_step(x[:, 0].clone().requires_grad_(True), w, b, state)
    with pytest.raises(RuntimeError, match="in place"):
        causal_conv_step(x[:, 0], w, b, torch.zeros(2, 8, 3, device=DEV).transpose(1, 2))
    v = state._version
    causal_conv_step(x[:, 0], w, b, state)
    assert state._version > v
    import torch.autograd.forward_ad as fwd_ad
    with fwd_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        causal_conv(fwd_ad.make_dual(x, torch.ones_like(x)), w)
