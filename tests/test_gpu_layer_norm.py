"""LayerNorm forward and backward (eacs_layer_norm_*) against the formulas in 64 bits.

Tolerances, max |got - want| / (row or column scale): a value is computed in
float32 from sums of at most d (or `rows`) terms added pairwise or in runs of a
few hundred, so its error stays under 2^-16 of the largest value, and it is
rounded once to its type (half a step, eps / 2 of the value).  The gradient of x is a
difference, rstd (p - mean(p) - h mean(p h)), whose terms are each off by
2^-24 of their own size however much they cancel (a row of two values has a
gradient of eps / variance of them): its float32 error is measured against
max |rstd p|.
"""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

if torch.cuda.is_available():
    from eacs_b200.ops.layer_norm import LayerNorm, layer_norm


def tol(dtype):
    return 2.0 ** -16 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0)


def close(got, want, dtype, terms=0.0):
    """terms: the size of what a difference is taken of."""
    got, want = got.detach(), want.detach().to(got.device)
    scale = float(want.abs().max()) + 1e-30
    assert got.dtype == dtype and got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    assert float((got.double() - want).abs().max()) <= tol(dtype) * scale + 2.0 ** -16 * terms


def terms_of(x, w, eps, r, dy):
    s = x.detach().double() if r is None else x.detach().double() + r.detach().double()
    rstd = ((s - s.mean(-1, keepdim=True)) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return float((rstd * dy.double() * (1 if w is None else w.detach().double())).abs().max())


def oracle(x, w, b, eps, r, dy):
    x, w, b, r = (None if t is None else t.detach().double().cpu().requires_grad_(True) for t in (x, w, b, r))
    s = x if r is None else x + r
    m = s.mean(-1, keepdim=True)
    h = (s - m) / (((s - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    y = h * (1 if w is None else w) + (0 if b is None else b)
    leaves = [t for t in (x, w, b, r) if t is not None]
    return y.detach(), dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None],
                                torch.autograd.grad(y, leaves, dy.double().cpu())))


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 33), (7, 250), (70, 256), (1300, 513), (33, 768), (9, 999),
                                    (5, 1024), (600, 1500), (17, 2048), (4, 4099), (3, 8191), (5, 8192)])
@pytest.mark.parametrize("dtype,wdtype,residual", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.float32, True),
                                                   (torch.float16, torch.float16, False), (torch.bfloat16, torch.bfloat16, False)])
def test_layer_norm(rows, d, dtype, wdtype, residual):
    g = torch.Generator(DEV).manual_seed(rows * 10007 + d)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = (rnd(rows, d) * 1.7 + 0.5).to(dtype).requires_grad_(True)
    r = rnd(rows, d).to(dtype).requires_grad_(True) if residual else None
    w, b = (1 + 0.3 * rnd(d)).to(wdtype).requires_grad_(True), rnd(d).to(wdtype).requires_grad_(True)
    dy = rnd(rows, d).to(dtype)
    y = layer_norm(x, w, b, 1e-5, residual=r)
    want, grads = oracle(x, w, b, 1e-5, r, dy)
    close(y, want, dtype)
    leaves = [x, w, b] + ([r] if residual else [])
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for n, t, gt in zip("xwbr", leaves, got):
        close(gt, grads[n], t.dtype, terms_of(x, w, 1e-5, r, dy) if n in "xr" else 0.0)
    for a, c in zip(got, torch.autograd.grad(y, leaves, dy)):  # the same bits again
        assert torch.equal(a, c)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, 1e-5, residual=r), y)


def test_without_weight_or_bias_and_needed_gradients_only():
    g = torch.Generator(DEV).manual_seed(1)
    x = torch.randn(37, 96, generator=g, device=DEV)
    w, b, dy = torch.rand(96, generator=g, device=DEV), torch.randn(96, generator=g, device=DEV), torch.randn(37, 96, generator=g, device=DEV)
    for ww, bb in ((None, None), (w, None), (None, b)):
        xx = x.clone().requires_grad_(True)
        y = layer_norm(xx, ww, bb)
        want, grads = oracle(x, ww, bb, 1e-5, None, dy)
        close(y, want, x.dtype)
        close(torch.autograd.grad(y, xx, dy)[0], grads["x"], x.dtype)
    bb = b.clone().requires_grad_(True)  # a bias's gradient alone, without a weight
    close(torch.autograd.grad(layer_norm(x, None, bb), bb, dy)[0], dy.double().sum(0), x.dtype)
    ww = w.clone().requires_grad_(True)
    close(torch.autograd.grad(layer_norm(x, ww, b), ww, dy)[0], oracle(x, w, b, 1e-5, None, dy)[1]["w"], x.dtype)


def test_views_broadcast_and_empty():
    g = torch.Generator(DEV).manual_seed(2)
    big = torch.randn(6, 5, 200, generator=g, device=DEV).half()
    w, b = torch.rand(64, generator=g, device=DEV), torch.randn(64, generator=g, device=DEV)
    for x in (big[..., 8:72], big[..., 3:67], big[:, 2, :64], big[0].t()[:, :1].expand(200, 64), big[:, :, ::3][..., :64],
              big[0, 0, :64], big[0, 0, :64].expand(9, 64)):
        y = layer_norm(x, w, b)
        close(y, oracle(x, w, b, 1e-5, None, torch.zeros_like(x))[0], x.dtype)
    leaf = torch.randn(64, generator=g, device=DEV, requires_grad=True)  # one row for all: its gradient is summed
    dy = torch.randn(9, 64, generator=g, device=DEV)
    other = torch.randn(9, 64, generator=g, device=DEV)
    y = layer_norm(leaf.expand(9, 64), w, b, residual=other)
    want = oracle(leaf.expand(9, 64), w, b, 1e-5, other, dy)[1]["x"].sum(0)
    close(torch.autograd.grad(y, leaf, dy)[0], want, torch.float32)
    both = torch.randn(4, 64, generator=g, device=DEV, requires_grad=True)  # the same tensor twice
    gb = torch.autograd.grad(layer_norm(both, w, b, residual=both), both, dy[:4])[0]
    close(gb, 2 * oracle(both, w, b, 1e-5, both, dy[:4])[1]["x"], torch.float32)
    e = torch.zeros(0, 64, device=DEV, requires_grad=True)
    we = w.clone().requires_grad_(True)
    y = layer_norm(e, we, b)
    assert y.shape == (0, 64) and float(torch.autograd.grad(y.sum(), we)[0].abs().max()) == 0.0


def test_constant_rows_large_means_and_nan_rows():
    x = torch.full((4, 100), 3.0, device=DEV)
    w, b = torch.full((100,), 2.0, device=DEV), torch.full((100,), 0.25, device=DEV)
    assert torch.equal(layer_norm(x, w, b), torch.full_like(x, 0.25))
    g = torch.Generator(DEV).manual_seed(3)
    x = torch.randn(8, 777, generator=g, device=DEV) + 4096.0  # E[x^2] - E[x]^2 would lose the variance
    y = layer_norm(x, None, None)
    want = oracle(x, None, None, 1e-5, None, torch.zeros_like(x))[0].to(DEV)
    # a sum of 777 values of 4096 is off by at most 2^-24 * log2-depth 10 of its size: 4096 * 10 * 2^-24 = 2.4e-3 in the mean
    assert float((y.double() - want).abs().max()) < 2.5e-3
    x[3, 5] = float("nan")
    y2 = layer_norm(x, None, None)
    keep = [i for i in range(8) if i != 3]
    assert bool(torch.isnan(y2[3]).all()) and torch.equal(y2[keep], y[keep])


def test_gradient_against_differences():
    g = torch.Generator(DEV).manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, w, b, dy = rnd(5, 129).requires_grad_(True), rnd(129).requires_grad_(True), rnd(129).requires_grad_(True), rnd(5, 129)
    grads = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    dirs, h = [rnd(*t.shape) for t in (x, w, b)], 2.0 ** -6
    f = lambda s: (layer_norm(*(t.detach() + s * h * v for t, v in zip((x, w, b), dirs))).double() * dy.double()).sum()
    slope = float(sum((a.double() * v.double()).sum() for a, v in zip(grads, dirs)))
    # 4th-order differences: truncation of order h^4 = 6e-8, rounding 2^-22 * |f| / h, |f| about 100: under 2e-3
    num = float((8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * h))
    assert abs(num - slope) < 5e-3 * max(1.0, abs(slope))


def test_other_stream_and_graph_replay():
    g = torch.Generator(DEV).manual_seed(5)
    x = torch.randn(300, 768, generator=g, device=DEV).bfloat16().requires_grad_(True)
    w, b = torch.rand(768, generator=g, device=DEV).requires_grad_(True), torch.randn(768, generator=g, device=DEV).requires_grad_(True)
    dy = torch.randn(300, 768, generator=g, device=DEV).bfloat16()

    def step():
        y = layer_norm(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(side, want))
    del side
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    with torch.no_grad():
        x.mul_(0.5)
    want = step()
    for gr, _ in graphs:
        gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_rows_past_32_bit_offsets():
    d = 1024
    rows = (1 << 31) // d + 5
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(DEV).manual_seed(6)
    x[-3:] = torch.randn(3, d, generator=g, device=DEV).bfloat16()
    y = layer_norm(x)
    assert torch.equal(y[-3:], layer_norm(x[-3:].clone())) and float(y[rows // 2].abs().max()) == 0.0


def test_module_matches_torch_and_autocast():
    m = LayerNorm(768).to(DEV)
    ref = nn.LayerNorm(768).to(DEV)
    x = torch.randn(4, 30, 768, device=DEV)
    close(m(x), ref(x).double(), torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, want = m(x.bfloat16()), ref(x.bfloat16())
    assert y.dtype == want.dtype == torch.float32
    close(y, want.double(), torch.float32)
    big = LayerNorm(9000).to(DEV)  # wider than the kernel takes
    xb = torch.randn(2, 9000, device=DEV)
    assert torch.equal(big(xb), nn.functional.layer_norm(xb, (9000,), big.weight, big.bias))


def test_refusals():
    x = torch.zeros(4, 16, device=DEV)
    w = torch.ones(16, device=DEV)
    for args, kw in (((x, w[:8]), {}), ((x.double(), None), {}), ((x, w, w.half()), {}), ((x, w), dict(residual=x[:2])),
                     ((x, w), dict(residual=x.half())), ((torch.zeros(1, 8193, device=DEV),), {}),
                     ((x, w.cpu()), {}), ((torch.zeros(3, 0, device=DEV),), {})):
        with pytest.raises(RuntimeError):
            layer_norm(*args, **kw)


def test_forward_mode_and_traced_inputs():
    """The function refuses what it would drop a derivative of; the module runs torch's own norm there."""
    from torch.autograd import forward_ad
    g = torch.Generator(DEV).manual_seed(7)
    x, t = (torch.randn(6, 48, generator=g, device=DEV) for _ in range(2))
    ours, ref = LayerNorm(48).to(DEV), nn.LayerNorm(48).to(DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        for kw in (dict(), dict(residual=x)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                layer_norm(dual, **kw)
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(x, residual=dual)
        got, want = (forward_ad.unpack_dual(m(dual)) for m in (ours, ref))
        assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent)
        close(layer_norm(x), ref(x).double(), torch.float32)  # (a tensor without a tangent)
    assert torch.equal(torch.func.jvp(ours, (x,), (t,))[1], torch.func.jvp(ref, (x,), (t,))[1])
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda a: layer_norm(a), x)
        traced = torch.jit.trace(ours, x)
        assert torch.equal(traced(t), ref(t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_of_the_backward(dtype):
    """A gradient penalty through the module, against torch's norm in 64 bits: first gradients rounded to the type once, the
    penalty's made of them and rounded again (half a step each, and 1e-5 for float32 sums)."""
    g = torch.Generator(DEV).manual_seed(8)
    x, dy = (torch.randn(5, 9, 64, generator=g, device=DEV).to(dtype) for _ in range(2))
    m = LayerNorm(64).to(DEV)
    nn.init.normal_(m.weight)
    ref = nn.LayerNorm(64).double()
    ref.load_state_dict({n: t.double().cpu() for n, t in m.state_dict().items()})
    res = []
    for norm, conv in ((m, lambda t: t.clone()), (ref, lambda t: t.double().cpu())):
        xx = conv(x).requires_grad_(True)
        dx, dw = torch.autograd.grad(norm(xx), (xx, norm.weight), conv(dy), create_graph=True)
        res.append([dx, dw, *torch.autograd.grad(dx.square().sum() + dw.square().sum(), (xx, norm.weight))])
    for a, c in zip(*res):
        err = float((a.detach().double().cpu() - c.detach()).norm())
        assert err <= (1e-5 + (torch.finfo(dtype).eps if dtype != torch.float32 else 0.0)) * float(c.detach().norm())
