"""The norms around a block (eacs_norm_*) against the formulas in 64 bits.

Tolerances: each value is a few products of float32 results, each off by at most 2^-20 (a norm's sum of up to 8192
squares in runs and over threads 2^-20, a root, a quotient, a sigmoid 2^-19), 2^-16 in all, of the largest term that
enters it: element by element `mag`, the sum of the terms' absolute values, with the sums over a row inside at their
largest (sums of absolute values).  Sums over rows: 2^-14.  Outputs are rounded once: half a step of their type (float16:
at least 2^-25).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200.ops.block_norm import gated_norm, residual_norm

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def oracle(i, dy=None, ds=None, magnitudes=False):
    f = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    d = lambda n: None if i.get(n) is None else i[n].detach().double()
    x, gate, res, weight, scale, post = (d(n) for n in ("x", "gate", "residual", "weight", "scale", "post"))
    one = torch.ones(x.shape[-1], device=x.device, dtype=torch.float64)
    eps, minus = i["eps"], 1 if magnitudes else -1
    r = lambda v: ((v * v).mean(-1, keepdim=True) + eps).rsqrt()
    first = i["residual"] is None or post is not None
    pw = (weight if res is None else post)
    pw = one if pw is None else pw
    r1 = r(x)
    u1s = x * r1 * pw if first else x
    sg = torch.sigmoid(gate) if gate is not None else None
    gain = one if gate is None else gate * sg
    u2s, u2 = u1s * gain, f(u1s) * f(gain)
    sc = one if scale is None else scale
    out = {}
    if res is None:
        out["y"] = u2
    else:
        ss = res + sc * u2s
        s = f(res) + f(sc) * u2
        r2 = r(ss)
        w = one if weight is None else weight
        out["s"], out["y"] = s, s * r2 * f(w)
    if dy is None:
        return out
    back = lambda q, v, rr: rr * (q + minus * v * rr * rr * (q * v).mean(-1, keepdim=True))
    dy = f(dy.double())
    rows = tuple(range(x.dim() - 1))
    if res is None:
        du2 = dy
    else:
        dv = f(ds.double()) + back(dy * f(w), s, r2)
        out["dresidual"], out["dweight"], out["dscale"] = dv, (dy * s * r2).sum(rows), (dv * u2).sum(rows)
        du2 = dv * f(sc)
    u1 = f(u1s)
    if gate is not None:
        out["dgate"] = du2 * u1 * (sg + f(gate) * sg * (1 - sg))
    du1 = du2 * f(gain)
    if first:
        out["dx"] = back(du1 * f(pw), f(x), r1)
        out["dweight" if res is None else "dpost"] = (du1 * f(x) * r1).sum(rows)
    else:
        out["dx"] = du1
    return out


def inputs(shape, dtype, wdtype, kind, seed=0, **kw):
    g = torch.Generator(DEV).manual_seed(seed * 1009 + shape[-1] * 17 + shape[0])
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    d = shape[-1]
    i = {"x": (rnd(*shape) * 1.7 + 0.3).to(dtype), "gate": rnd(*shape).to(dtype) if kw.get("gate") else None,
         "residual": rnd(*shape).to(dtype) if kind == "residual" else None, "weight": (1 + 0.3 * rnd(d)).to(wdtype),
         "scale": (0.5 * rnd(d)).to(wdtype) if kw.get("scale") else None, "post": (1 + 0.3 * rnd(d)).to(wdtype) if kw.get("post") else None,
         "eps": kw.get("eps", 1e-5)}
    if kw.get("bare"):
        i["weight"] = None
    return i, rnd


def call(i):
    if i["residual"] is None:
        return (gated_norm(i["x"], i["gate"], i["weight"], i["eps"]),)
    return residual_norm(i["x"], i["residual"], i["weight"], i["scale"], i["gate"], i["post"], i["eps"])


def close(name, got, want, mag, dtype, sums=False):
    assert got.dtype == dtype and got.shape == want.shape, name
    assert bool(torch.isfinite(got).all()), name
    tol = 2.0 ** (-14 if sums else -16) * mag + 1e-30
    if dtype != F32:
        tol = tol + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == F16 else 0.0)
    over = (got.double() - want).abs() - tol
    assert over.numel() == 0 or float(over.max()) <= 0, (name, float(over.max()), int(over.argmax()))


LEAVES = ("x", "gate", "residual", "weight", "scale", "post")


def check(i, dy, ds):
    for n in LEAVES:
        i[n] = None if i[n] is None else i[n].detach().requires_grad_(True)
    outs = call(i)
    want, mag = oracle(i, dy, ds), oracle(i, dy, ds, True)
    for n, t in zip(("y", "s"), outs):
        close(n, t.detach(), want[n], mag[n], i["x"].dtype)
    names = [n for n in LEAVES if i[n] is not None]
    ups = [dy, ds][:len(outs)]
    grads = torch.autograd.grad(outs, [i[n] for n in names], ups, retain_graph=True)
    for n, t in zip(names, grads):
        close("d" + n, t, want["d" + n], mag["d" + n], i[n].dtype, n in ("weight", "scale", "post"))
    for t, u in zip(grads, torch.autograd.grad(outs, [i[n] for n in names], ups)):
        assert torch.equal(t, u)
    with torch.no_grad():
        for t, u in zip(call(i), outs):
            assert torch.equal(t, u)


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 33), (70, 64), (301, 128), (7, 250), (1300, 513), (33, 768), (9, 999), (5, 1024),
                                    (600, 1504), (17, 2048), (4, 4096), (4, 4099), (3, 8191), (5, 8192)])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (BF16, F32)])
def test_norms(rows, d, dtype, wdtype):
    for k, (kind, kw) in enumerate([("gated", dict(gate=True)), ("gated", {}), ("residual", {}), ("residual", dict(scale=True)),
                                    ("residual", dict(gate=True, scale=True, post=True)), ("residual", dict(post=True, bare=True))]):
        i, rnd = inputs((rows, d), dtype, wdtype, kind, k, **kw)
        check(i, rnd(rows, d).to(dtype), rnd(rows, d).to(dtype))


@pytest.mark.parametrize("rows,d", [(1, 7), (300, 31), (33, 50), (1301, 63), (65, 127), (40, 190), (700, 255), (9, 411), (301, 509)])
def test_narrow_rows_element_by_element(rows, d):
    for k, kw in enumerate([dict(gate=True, scale=True, post=True), dict(scale=True)]):
        i, rnd = inputs((rows, d), F16, F32, "residual", k, **kw)
        check(i, rnd(rows, d).half(), rnd(rows, d).half())
    i, rnd = inputs((rows, d), BF16, BF16, "gated", 3, gate=True)
    check(i, rnd(rows, d).bfloat16(), None)


def test_heads_views_and_broadcast():
    i, rnd = inputs((2, 7, 3, 96), BF16, BF16, "gated", 1, gate=True)  # (B, L, heads, V): each head by itself
    check(i, rnd(2, 7, 3, 96).bfloat16(), None)
    big = rnd(2, 7, 3 * 96 + 40).bfloat16()
    for off in (0, 8, 3):
        v = big[..., off:off + 288]
        j = {**i, "x": v[..., :96], "gate": v[..., 96:192], "residual": v[..., 192:], "scale": i["weight"] * 0.5}
        check(j, rnd(2, 7, 96).bfloat16(), rnd(96).bfloat16().expand(2, 7, 96))
    one = rnd(1, 64).requires_grad_(True)  # one row for all: its gradient is summed
    i, rnd = inputs((9, 64), F32, F32, "residual", 2, scale=True)
    i["residual"] = one.expand(9, 64)
    dy, ds = rnd(9, 64), rnd(9, 64)
    got = torch.autograd.grad(call(i), one, (dy, ds))[0]
    close("one", got, oracle(i, dy, ds)["dresidual"].sum(0, keepdim=True), oracle(i, dy, ds, True)["dresidual"].sum(0, keepdim=True), F32)
    both = rnd(4, 64).requires_grad_(True)  # the same tensor twice
    y, s = residual_norm(both, both)
    g = torch.autograd.grad((y, s), both, (dy[:4], ds[:4]))[0]
    j = {**i, "x": both, "residual": both, "scale": None, "weight": None}
    w, m = oracle(j, dy[:4], ds[:4]), oracle(j, dy[:4], ds[:4], True)
    close("both", g, w["dx"] + w["dresidual"], m["dx"] + m["dresidual"], F32)


def test_one_output_alone_and_needed_gradients_only():
    i, rnd = inputs((37, 96), F32, F32, "residual", 3, scale=True, gate=True)
    dy, nil = rnd(37, 96), torch.zeros(37, 96, device=DEV)
    for which, ups in ((0, (dy, nil)), (1, (nil, dy))):
        for n in ("x", "weight", "scale", "residual"):
            if which == 1 and n == "weight":
                continue
            j = {**i, n: i[n].clone().requires_grad_(True)}
            got = torch.autograd.grad(call(j)[which], j[n], dy)[0]
            close(n, got, oracle(j, *ups)["d" + n], oracle(j, *ups, True)["d" + n], F32, n in ("weight", "scale"))
    for n in ("x", "residual"):  # nothing between them: one gradient for both
        j = {**i, "gate": None, "scale": None, n: i[n].clone().requires_grad_(True)}
        got = torch.autograd.grad(call(j), j[n], (dy, dy))[0]
        close(n, got, oracle(j, dy, dy)["d" + n], oracle(j, dy, dy, True)["d" + n], F32)


def test_zero_rows_nan_rows_and_empty():
    i, rnd = inputs((8, 777), F32, F32, "residual", 4, gate=True, post=True, scale=True)
    i["x"][2] = 0
    i["residual"][2] = 0
    y, s = call(i)
    assert float(y[2].abs().max()) == 0 and float(s[2].abs().max()) == 0
    x = i["x"].clone()
    x[3, 5] = float("nan")
    y2, s2 = call({**i, "x": x})
    keep = [0, 1, 2, 4, 5, 6, 7]
    assert bool(torch.isnan(y2[3]).all()) and torch.equal(y2[keep], y[keep]) and torch.equal(s2[keep], s[keep])
    small, rnd = inputs((40, 24), F32, F32, "gated", 5, gate=True)  # rows that share a warp
    small["x"][7] = float("inf")
    got = gated_norm(small["x"], small["gate"], small["weight"])
    rest = [k for k in range(40) if k != 7]
    assert bool(torch.isfinite(got[rest]).all()) and not bool(torch.isfinite(got[7]).any())
    w = i["weight"].clone().requires_grad_(True)
    e = torch.zeros(0, 777, device=DEV, requires_grad=True)
    y, s = residual_norm(e, e, w)
    assert y.shape == (0, 777) and float(torch.autograd.grad(y.sum() + s.sum(), w)[0].abs().max()) == 0.0


def test_gradient_against_differences():
    i, rnd = inputs((5, 129), F32, F32, "residual", 6, gate=True, post=True, scale=True)
    dy, ds = rnd(5, 129), rnd(5, 129)
    for n in LEAVES:
        j = {**i, n: i[n].clone().requires_grad_(True)}
        g = torch.autograd.grad(call(j), j[n], (dy, ds))[0]
        v, h = rnd(*i[n].shape), 2.0 ** -7

        def f(t):
            o = oracle({**i, n: i[n].double() + t * h * v.double()})
            return float((o["y"] * dy.double()).sum() + (o["s"] * ds.double()).sum())
        diff = (8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * h)
        terms = g.double() * v.double()
        assert abs(diff - float(terms.sum())) <= 1e-4 * (float(terms.abs().sum()) + 1), n


def test_streams_and_graphs():
    i, rnd = inputs((300, 256), BF16, F32, "residual", 7, gate=True, post=True, scale=True)
    want, outs = call(i), []
    for st in (torch.cuda.Stream(), torch.cuda.Stream()):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs += [call(i) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], want[0]) and torch.equal(o[1], want[1]) for o in outs)
    leaves = [i[n].detach().requires_grad_(True) for n in LEAVES]
    dy = rnd(300, 256).bfloat16()

    def step():
        y, s = call({**i, **dict(zip(LEAVES, leaves))})
        return [y.detach(), s.detach(), *torch.autograd.grad((y, s), leaves, (dy, dy))]
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


def test_refusals():
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for match, f in (("unsupported x", lambda: gated_norm(x.double())), ("d=8193", lambda: gated_norm(torch.zeros(1, 8193, device=DEV))),
                     ("gate must", lambda: gated_norm(x, x[:2])), ("gate must", lambda: gated_norm(x, x.half())),
                     ("residual must", lambda: residual_norm(x, x[:, :4])), ("expects a residual", lambda: residual_norm(x, None)),
                     ("weight, scale", lambda: gated_norm(x, x, w[:4])), ("one dtype", lambda: residual_norm(x, x, w, w.half())),
                     ("CUDA", lambda: gated_norm(x, x.cpu())), ("CUDA", lambda: gated_norm(x.cpu()))):
        with pytest.raises(RuntimeError, match=match):
            f()
    import torch.autograd.forward_ad as fwd_ad
    with fwd_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        gated_norm(fwd_ad.make_dual(x, torch.ones_like(x)), x, w)
